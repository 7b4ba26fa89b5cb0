// What the host side hands to the rotary kernel (rotary.hip).
#pragma once
struct RotaryDims {
  long rows;                                   // tokens
  int H, Hk, D, R, interleaved, tokens;        // tokens: per workgroup, chosen at launch
  long ldq, hq, ldk, hk, ldv, hv;              // element strides of tokens and heads
  float multiplier, sign;                      // sign -1: the gradient
  int n, max_new, page_shift, cols, pages;     // paged form: sequences, their longest chunk, as in PagedDims
  long page_ld, ld, hd;
};
