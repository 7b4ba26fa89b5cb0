// Host side of the causal-transformer operators: argument checks behind the C ABI of include/s2g.h.
#include "packed_attention.h"
#include "paged_attention.h"
#include "rotary.h"
#include <math.h>
#include <algorithm>
#include <initializer_list>

// mirror include/s2g.h
struct S2GPackedTile {
  int q_start, q_len, k_start, k_len, tile, row_lo, row_hi, slot;
};
struct S2GPacked {
  int type, heads, kv_heads, dim, causal;
  float scale;
  long q_ld, q_hd, k_ld, k_hd, v_ld, v_hd, do_ld, do_hd, q_rows, k_rows;
};
struct S2GPaged {
  int type, sequences, heads, kv_heads, dim, causal, page_size, pages, table_cols, max_new, max_length, part_keys, parts, by_rows;
  float scale;
  long q_rows, q_ld, q_hd, page_ld, token_ld, head_ld;
};
struct S2GRotary {
  int type, heads, kv_heads, dim, rotary, interleaved, backward;
  float multiplier;
  long rows, q_ld, q_hd, k_ld, k_hd, v_ld, v_hd;
};

static_assert(sizeof(S2GPackedTile) == sizeof(PackedTile) && sizeof(PackedTile) == 32, "S2GPackedTile");

#define DECLARE(sfx)                                                                                                    \
  extern "C" int s2g_launch_packed_fwd_##sfx(const void*, const void*, const void*, void*, void*, float*, const PackedTile*, int, PackedDims, hipStream_t); \
  extern "C" int s2g_launch_packed_bwd_##sfx(const void*, const void*, const void*, const void*, const void*, const void*, const float*, float*, void*, void*, \
                                             void*, float*, const PackedTile*, int, const PackedTile*, int, const PackedTile*, int, PackedDims, hipStream_t); \
  extern "C" int s2g_launch_paged_##sfx(const void*, const void*, const void*, const int*, const int*, const int*, void*, float*, int, PagedDims, hipStream_t);
DECLARE(f32)
DECLARE(bf16)
DECLARE(f16)
extern "C" int s2g_launch_rotary(int, const void*, const void*, const void*, const int*, const double*, const int*, const int*,
                                 const int*, void*, void*, void*, int, RotaryDims, hipStream_t);
#define BY_TYPE(t, name, ...) \
  ((t) == 0 ? name##_f32(__VA_ARGS__) : (t) == 1 ? name##_bf16(__VA_ARGS__) : (t) == 2 ? name##_f16(__VA_ARGS__) : -1)

static inline int elem_size(int type) { return type == 0 ? 4 : 2; }
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// heads of D elements, 16-byte units throughout, the offsets of a tile of rows (of G heads side by side) within 31 bits
static bool wide_rows(long ld, long hd, int D, int es, int G = 1) {
  const int u = 16 / es;
  return ld >= 0 && hd >= 0 && ld % u == 0 && hd % u == 0 && D % u == 0 && ld < (1L << 22) && hd < (1L << 22) &&
         (64 * ld + G * hd) * es < 0x7ffffe00L;
}

static int packed_dims(const S2GPacked* a, PackedDims* d) {
  if (!a || a->type < 0 || a->type > 2 || a->heads <= 0 || a->kv_heads <= 0 || a->heads % a->kv_heads) return -1;
  if (a->dim <= 0 || a->dim > 128 || a->dim % 8 || !(a->scale > 0.0f) || !(a->scale < INFINITY)) return -1;
  if (a->q_rows < 0 || a->k_rows < 0 || a->q_rows * a->heads >= (1L << 30) || a->k_rows >= (1L << 30)) return -1;
  const int es = elem_size(a->type), G = a->heads / a->kv_heads;
  if (G > 128 || !wide_rows(a->q_ld, a->q_hd, a->dim, es, G) || !wide_rows(a->k_ld, a->k_hd, a->dim, es) ||
      !wide_rows(a->v_ld, a->v_hd, a->dim, es) || !wide_rows(a->do_ld, a->do_hd, a->dim, es, G))
    return -1;
  *d = PackedDims{a->heads, a->kv_heads, a->dim, a->causal != 0, div_by(G), a->q_ld, a->q_hd, a->k_ld, a->k_hd, a->v_ld, a->v_hd,
                  a->do_ld, a->do_hd, a->q_rows, a->k_rows, a->scale};
  return 0;
}

extern "C" {

int s2g_packed_attention_fwd(const void* Q, const void* K, const void* V, void* out, void* rest, float* lse, const S2GPackedTile* tiles,
                             int n_tiles, const S2GPacked* dims, void* stream) {
  PackedDims d;
  if (!Q || !K || !V || !out || !tiles || n_tiles <= 0 || packed_dims(dims, &d) != 0) return -1;
  if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(out) || !aligned16(rest) || (long)n_tiles * d.Hk >= (1L << 31)) return -1;
  return BY_TYPE(dims->type, s2g_launch_packed_fwd, Q, K, V, out, rest, lse, reinterpret_cast<const PackedTile*>(tiles), n_tiles, d, (hipStream_t)stream);
}

long s2g_packed_attention_bwd_workspace(const S2GPacked* dims, int slots) {
  PackedDims d;
  if (packed_dims(dims, &d) != 0 || slots < 0) return -1;
  return 256L * slots * d.Hk * d.D;
}

int s2g_packed_attention_bwd(const void* Q, const void* K, const void* V, const void* out, const void* rest, const void* dO, const float* lse,
                             float* delta, void* dQ, void* dK, void* dV, float* work, const S2GPackedTile* q_tiles,
                             int n_q_tiles, const S2GPackedTile* k_tiles, int n_k_tiles, const S2GPackedTile* cut_tiles,
                             int n_cut_tiles, const S2GPacked* dims, void* stream) {
  PackedDims d;
  if (!Q || !K || !V || !out || !dO || !lse || !delta || !dQ || !dK || !dV || packed_dims(dims, &d) != 0) return -1;
  if (n_q_tiles < 0 || n_k_tiles < 0 || n_cut_tiles < 0 || (n_q_tiles && !q_tiles) || (n_k_tiles && !k_tiles) || (n_cut_tiles && (!cut_tiles || !work))) return -1;
  if ((long)n_q_tiles * d.Hk >= (1L << 31) || (long)n_k_tiles * d.Hk >= (1L << 31) || (long)n_cut_tiles * d.Hk >= (1L << 31)) return -1;
  if (dims->type != 0 && !rest) return -1;
  const void* all[] = {Q, K, V, out, rest, dO, dQ, dK, dV, work};
  for (const void* p : all)
    if (!aligned16(p)) return -1;
  return BY_TYPE(dims->type, s2g_launch_packed_bwd, Q, K, V, out, rest, dO, lse, delta, dQ, dK, dV, work,
                 reinterpret_cast<const PackedTile*>(q_tiles), n_q_tiles, reinterpret_cast<const PackedTile*>(k_tiles), n_k_tiles,
                 reinterpret_cast<const PackedTile*>(cut_tiles), n_cut_tiles, d, (hipStream_t)stream);
}

static int page_shift(int page_size) {
  for (int s = 4; s <= 16; ++s)
    if (page_size == 1 << s) return s;
  return -1;
}

static int paged_dims(const S2GPaged* a, PagedDims* d) {
  if (!a || a->type < 0 || a->type > 2 || a->sequences <= 0 || a->sequences > 65535 || a->heads <= 0 || a->kv_heads <= 0 ||
      a->heads % a->kv_heads || a->dim <= 0 || a->dim > 128 || a->dim % 8 || !(a->scale > 0.0f) || !(a->scale < INFINITY))
    return -1;
  const int G = a->heads / a->kv_heads, es = elem_size(a->type), shift = page_shift(a->page_size);
  if (shift < 0 || a->pages <= 0 || a->table_cols <= 0 || (long)a->table_cols * a->page_size >= (1L << 30) || G > 128) return -1;
  if (a->q_rows <= 0 || a->q_rows * a->heads >= (1L << 30) || a->max_new <= 0 || a->max_new > a->q_rows || a->max_length < 0) return -1;
  if (!wide_rows(a->q_ld, a->q_hd, a->dim, es) || !wide_rows(a->token_ld, a->head_ld, a->dim, es) || a->page_ld % (16 / es) || a->page_ld < 0) return -1;
  // a page's offset is its number times 32 bits of 16-byte units, a token's within its page has 32 bits
  if (a->page_ld >= (1L << 36) / es || a->page_size * a->token_ld * es >= (1L << 32)) return -1;
  if (a->part_keys <= 0 || a->part_keys % 128 || a->parts <= 0 || (long)a->part_keys * a->parts < a->max_length || a->parts > 4096 ||
      (long)a->part_keys * a->parts >= (1L << 31))
    return -1;
  *d = PagedDims{a->sequences, a->heads, a->kv_heads, a->dim, a->causal != 0, div_by(G), shift, a->table_cols, a->pages,
                 a->q_ld, a->q_hd, a->page_ld, a->token_ld, a->head_ld, a->q_rows, a->max_new * G, a->part_keys, a->parts, a->scale,
                 (int)(a->head_ld > 0 ? std::max(1L, 128 / (a->head_ld * es)) : 1)};
  return 0;
}

long s2g_paged_attention_workspace(const S2GPaged* dims) {
  PagedDims d;
  if (paged_dims(dims, &d) != 0) return -1;
  return d.parts == 1 ? 0 : d.q_rows * d.H * d.parts * (d.D + 2L);
}

int s2g_paged_attention(const void* Q, const void* keys, const void* values, const int* table, const int* lengths,
                        const int* starts, void* out, float* work, const S2GPaged* dims, void* stream) {
  PagedDims d;
  if (!Q || !keys || !values || !table || !lengths || !starts || !out || paged_dims(dims, &d) != 0 || (d.parts > 1 && !work)) return -1;
  if (!aligned16(Q) || !aligned16(keys) || !aligned16(values) || !aligned16(out) || !aligned16(work)) return -1;
  const int tile = dims->by_rows ? 128 : 32;
  if ((d.max_rows + tile - 1) / tile > 65535 || (long)d.Hk * d.parts >= (1L << 31) || (long)d.Hk * d.max_rows >= (1L << 31)) return -1;
  return BY_TYPE(dims->type, s2g_launch_paged, Q, keys, values, table, lengths, starts, out, work, dims->by_rows, d, (hipStream_t)stream);
}

static int rotary_dims(const S2GRotary* a, RotaryDims* d) {
  if (!a || a->type < 0 || a->type > 2 || a->rows <= 0 || a->rows >= (1L << 31) || a->heads < 0 || a->kv_heads < 0 || a->heads + a->kv_heads <= 0) return -1;
  if (a->dim <= 0 || a->dim > 256 || a->rotary < 0 || a->rotary > a->dim || a->rotary % 2 || !(fabsf(a->multiplier) < INFINITY)) return -1;
  *d = RotaryDims{a->rows, a->heads, a->kv_heads, a->dim, a->rotary, a->interleaved != 0, 1, a->q_ld, a->q_hd, a->k_ld, a->k_hd,
                  a->v_ld, a->v_hd, a->multiplier, a->backward ? -1.0f : 1.0f, 0, 0, 0, 0, 0, 0, 0, 0};
  return 0;
}
// 16-byte units fit: every size and stride a multiple, every address aligned
static int rotary_wide(const S2GRotary* a, std::initializer_list<const void*> ps, std::initializer_list<long> strides) {
  const int u = a->type == 0 ? 4 : 8;
  if (a->dim % u || (a->interleaved ? a->rotary : a->rotary / 2) % u || (a->dim - a->rotary) % u) return 0;
  for (const void* p : ps)
    if (!aligned16(p)) return 0;
  for (long s : strides)
    if (s % u) return 0;
  return 1;
}

int s2g_rotary(const void* q, const void* k, const int* positions, const double* frequencies, void* q_out, void* k_out,
               const S2GRotary* dims, void* stream) {
  RotaryDims d;
  if (rotary_dims(dims, &d) != 0 || !positions || (d.R && !frequencies) || (d.H && (!q || !q_out)) || (d.Hk && (!k || !k_out))) return -1;
  const int wide = rotary_wide(dims, {q, k, q_out, k_out}, {d.ldq, d.hq, d.ldk, d.hk});
  return s2g_launch_rotary(dims->type, q, k, nullptr, positions, frequencies, nullptr, nullptr, nullptr, q_out, k_out, nullptr, wide, d, (hipStream_t)stream);
}

int s2g_rotary_append(const void* q, const void* k, const void* v, const double* frequencies, void* q_out, void* keys,
                      void* values, const int* table, const int* lengths, const int* starts, const S2GRotary* dims,
                      const S2GPaged* paged, void* stream) {
  RotaryDims d;
  if (rotary_dims(dims, &d) != 0 || !q || !k || !v || !q_out || !keys || !values || !table || !lengths || !starts || !paged) return -1;
  if ((d.R && !frequencies) || d.H <= 0 || d.Hk <= 0 || paged->sequences <= 0 || paged->sequences > 65535 || paged->max_new <= 0 || paged->max_new > d.rows) return -1;
  d.page_shift = page_shift(paged->page_size);
  if (d.page_shift < 0 || paged->pages <= 0 || paged->table_cols <= 0 || (long)paged->table_cols * paged->page_size >= (1L << 30)) return -1;
  d.n = paged->sequences, d.max_new = paged->max_new, d.cols = paged->table_cols, d.pages = paged->pages;
  d.page_ld = paged->page_ld, d.ld = paged->token_ld, d.hd = paged->head_ld;
  const int wide = rotary_wide(dims, {q, k, v, q_out, keys, values}, {d.ldq, d.hq, d.ldk, d.hk, d.ldv, d.hv, d.page_ld, d.ld, d.hd});
  return s2g_launch_rotary(dims->type, q, k, v, nullptr, frequencies, table, lengths, starts, q_out, keys, values, wide, d, (hipStream_t)stream);
}

}  // extern "C"
