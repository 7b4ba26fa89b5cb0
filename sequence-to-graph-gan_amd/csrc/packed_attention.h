// What the host side hands to the packed attention kernels (packed_attention.hip, compiled once per element type).
#pragma once
#include "frag.h"

// One tile of a sequence: 128 rows (query side) or 128 keys (key side).  Mirrors S2GPackedTile of include/s2g.h.
struct PackedTile {
  int q_start, q_len;      // the sequence's tokens in Q, out and dO
  int k_start, k_len;      // and in K and V
  int tile;                // which 128 rows / keys of the sequence
  int row_lo, row_hi;      // key side: the rows to go through, of all that the kv head has
  int slot;                // key side: -1, or where in the workspace these rows' share goes
};

struct PackedDims {
  int H, Hk, D, causal;
  DivBy by;                // G = H / Hk
  long ldq, hq, ldk, hk, ldv, hv, ldo, ho;       // element strides of tokens and heads; ldo, ho: of dO
  long q_rows, k_rows;     // tokens of Q and of K
  float scale;
};

// the element type this translation unit is compiled for: 0 fp32, 1 bf16, 2 fp16
#if PACKED_TYPE == 0
#define PACKED_T float
#define PACKED_NAME(n) n##_f32
#elif PACKED_TYPE == 1
#define PACKED_T __bf16
#define PACKED_NAME(n) n##_bf16
#elif PACKED_TYPE == 2
#define PACKED_T _Float16
#define PACKED_NAME(n) n##_f16
#endif

// F<T, width>(...) for the feature width that holds dm.D
#define PER_DIM(F, T, ...)                          \
  (dm.D <= 16   ? F<T, 16>(__VA_ARGS__)             \
   : dm.D <= 32 ? F<T, 32>(__VA_ARGS__)             \
   : dm.D <= 64 ? F<T, 64>(__VA_ARGS__)             \
   : dm.D <= 96 ? F<T, 96>(__VA_ARGS__)             \
                : F<T, 128>(__VA_ARGS__))
