// What the host side hands to the paged attention kernels (paged_attention.hip, compiled once per element type).
#pragma once
#include "packed_attention.h"

struct PagedDims {
  int n, H, Hk, D, causal;
  DivBy by;                          // G = H / Hk
  int page_shift, cols, pages;       // log2 of the tokens per page, columns of the table, pages of the pool
  long ldq, hq;                      // element strides of q's tokens and heads
  long page_ld, ld, hd;              // of the pages, of their tokens and heads (keys and values alike)
  long q_rows;                       // tokens of q
  int max_rows;                      // rows (token, head of the group) of the longest chunk
  int part_keys, parts;              // keys per part of a sequence, parts of the longest one
  float scale;
  int line_heads;                    // heads of a token that share 128 bytes of the cache
};
