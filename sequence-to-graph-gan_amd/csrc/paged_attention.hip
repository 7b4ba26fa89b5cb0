// Attention of the last few tokens of every sequence over its keys and values in a paged cache.
//
// Sequence s has lens[s] tokens in the cache, the newest starts[s + 1] - starts[s] of which bring queries; query i of n
// sees keys j <= len - n + i.  Token t of s lies in page table[s][t >> shift].  Rows are (token, head of the group), as
// in packed_attention.hip, so the G query heads of a kv head read its keys and values once.
//
// Single tokens are bound by reading K and V: a workgroup takes 32 rows and a part of the keys, each wave streams tiles
// of 32 keys of its own through LDS without ever waiting for the others, and the waves join at the end.  Chunks of new
// tokens are bound by the products: a workgroup takes 128 rows, its waves share tiles of 64 keys.  Either way a long
// axis is cut into parts of part_keys keys so that few rows still fill the chip; parts leave (O, m, l) in 32 bits and
// s2g_k_paged_join_few / _many add them in order.  A sequence with a single part is written at once.
//
// Measured (8 kv heads of 128 bf16, 32 query heads): one token of 64 sequences of 300 to 8200, 213 us and 4 to join, 5.2 TB/s
// of keys and values (a copy: 4.8); chunks of 512, 301, 777 and 5 new tokens over up to 16001, 349 us with 16 to join (profiled
// 365 and 16, the matrix units busy 35 % of the time at 2.1 GHz): by the chain of scores, weights and sums of the two waves of a
// SIMD.  (The packed forward pass hides weights behind the next keys' scores; here the second list of pages which that takes
// costs more: 388 us for 370.)  One token of 131071 and of 90001 (2 kv heads of 96 fp16): 37 us and 5, 4.6 TB/s.  One token of
// 777 fp32: 8 us and 3, latency.
//
// Lengths and pages come from device memory (a captured decoding loop updates them there), so nothing read from it is
// trusted: keys beyond what the table covers are not there, a page number outside the pool is a page that is not there.
#include "attn_rows.h"
#include "paged_attention.h"

struct PagedSeq {
  int n, len, start, rows;
  int first;                         // position of the first query: it sees keys up to itself
};
__device__ __forceinline__ PagedSeq paged_seq(const int* lens, const int* starts, int s, const PagedDims& dm) {
  PagedSeq q;
  const int a = min(max(uniform(starts[s]), 0), (int)dm.q_rows), b = min(max(uniform(starts[s + 1]), a), (int)dm.q_rows);
  q.start = a;
  q.n = b - a;
  const int len = min(max(uniform(lens[s]), 0), 1 << 30);
  q.first = len - q.n;
  q.len = (int)min((long)len, (long)dm.cols << dm.page_shift);
  q.len = min(q.len, dm.part_keys * dm.parts);
  q.rows = min(q.n * dm.by.G, dm.max_rows);
  return q;
}
// keys that the rows [row0, row0 + count) of a sequence see, at most
__device__ __forceinline__ int keys_seen(const PagedSeq& q, int row, const PagedDims& dm) {
  if (!dm.causal) return q.len;
  return max(0, min(q.len, divide(min(row, q.rows - 1), dm.by) + q.first + 1));
}

// What the table says of key `key`'s page.  The load is unconditional (of a key that exists, or the first) and is looked
// at only when its tile is fetched, an iteration later: a test here would wait for it, and for every load before it.
__device__ __forceinline__ int page_of(const int* table, int key, int len, const PagedDims& dm) {
  return table[key < len ? key >> dm.page_shift : 0];
}
__device__ __forceinline__ bool in_pool(int page, const PagedDims& dm) { return (unsigned)page < (unsigned)dm.pages; }
// One tile of keys from k0 on, and of values behind it: wave instruction after wave instruction, each within one page (whose
// 16 tokens or more it never crosses).  Keys beyond the length and of absent pages come as zeros.  Where a page's rows lie is
// made by the vector unit, lane l for key k0 + l, all of a tile at once, and read from there: made for one instruction after
// another by the scalar unit it is a wave's longest path (chunks over 16001 tokens of 128 bf16: 176 scalar operations a tile).
template <typename LT, int WAVES, bool KEYS = true, bool VALUES = true, typename T>
__device__ __forceinline__ void fetch_pages(char* lds, const T* keys, const T* values, int page, int k0, int len, const int* off,
                                            int wave, int lane, const PagedDims& dm) {
  const unsigned to = lds_address(lds), ld = (unsigned)dm.ld * (unsigned)sizeof(T), units = (unsigned)((dm.page_ld * (long)sizeof(T)) >> 4);
  const int key = k0 + lane, n = min(LT::RPI, len - key);
  const unsigned long at = (((unsigned long)(unsigned)page * units) << 4) + ((unsigned)key & ((1u << dm.page_shift) - 1u)) * ld;
  const int bytes = in_pool(page, dm) && n > 0 ? (n - 1) * (int)ld + dm.D * (int)sizeof(T) : 0;       // 0: nothing is touched
  const int lo = (int)(unsigned)at, hi = (int)(unsigned)(at >> 32);
#pragma unroll
  for (int i = 0; i < LT::NI; ++i) {
    const int r = (i * WAVES + wave) * LT::RPI;
    const unsigned long row = (unsigned long)(unsigned)__builtin_amdgcn_readlane(lo, r) | (unsigned long)(unsigned)__builtin_amdgcn_readlane(hi, r) << 32;
    const int b = __builtin_amdgcn_readlane(bytes, r);
    if constexpr (KEYS) load_to_lds(buffer_of(reinterpret_cast<const char*>(keys) + row, b), to + (i * WAVES + wave) * 1024, off[i]);
    if constexpr (VALUES) load_to_lds(buffer_of(reinterpret_cast<const char*>(values) + row, b), to + LT::BYTES + (i * WAVES + wave) * 1024, off[i]);
  }
}
template <typename LT, typename T>
__device__ __forceinline__ void page_offsets(int* off, int wave, int lane, const PagedDims& dm) {
#pragma unroll
  for (int i = 0; i < LT::NI; ++i) {
    const int c = LT::chunk_of(i, wave, lane);
    off[i] = c * 16 < dm.D * (int)sizeof(T) ? (int)((lane / LT::CH) * dm.ld * (long)sizeof(T)) + c * 16 : OUT_OF_BUFFER;
  }
}

// rows of a wave: O = sum over their keys among lo .. lo + width - 1, lo + step .., up to hi, of 2^(c s - base) V, times f
template <typename T, int DP, typename U>
__device__ __attribute__((noinline)) void slow_pages(const T* q, const T* keys, const T* values, const int* table, int lo, int width, int step, int hi,
                                                     int last, float c, float base, float f, U* to, bool live, int D, int page_shift,
                                                     int pages, long page_ld, long ld) {
  const int half = (threadIdx.x >> 5) & 1;
  for (int from = 16 * half; from < DP + 16 * half; from += 32) {                // both halves take every turn: their dots are one
    float acc[16] = {};
    for (int k0 = lo; k0 < hi; k0 += step)
      for (int key = k0; key < min(k0 + width, hi); ++key) {
        const int page = uniform(table[key >> page_shift]);
        if ((unsigned)page >= (unsigned)pages) continue;
        const long at = page * page_ld + (key & ((1 << page_shift) - 1)) * ld;
        const float w = __builtin_amdgcn_exp2f(fmaf(slow_dot<T, DP / 16>(q, keys + at, D, half), c, -base));
        if (key <= last) slow_add(acc, w, values + at, from, D);
      }
    slow_store(to, acc, f, from, D, live);
  }
}

// The part that the i-th workgroup of a sequence takes: turned by one from sequence to sequence.  Workgroups are dealt to
// the XCDs and their engines in turn, so the parts that short sequences lack would otherwise all fall to the same ones
// (64 sequences of 300 to 8200 tokens in 8 parts: 300 us, turned 250).
__device__ __forceinline__ int part_of(int i, int by, int parts) { return (i + by) % parts; }

// The order of a sequence's (part, kv head) pairs, heads fastest.  Workgroups are dealt to the 8 XCDs in turn, so neighbouring
// heads would be read by different caches, and where several share a 128-byte line each would fetch it whole (one token of 64
// sequences of 8000, 8 heads of 16 bf16: 162 us, so 93; 4000, of 32: 82, so 46): such heads lie 8 apart.
__device__ __forceinline__ int shared_lines(int b, int blocks, int line_heads) {
  const int all = 8 * line_heads, r = b % all;
  return line_heads == 1 || b - r + all > blocks ? b : b - r + r % 8 * line_heads + r / 8;
}

// Where a row's result goes: the output if its sequence has one part, else part `part` of the workspace
// ([row of all kv heads][part][D] sums, then [row][part] (m, l)).
struct Joined {
  float* sums;
  float* ml;
};
__device__ __forceinline__ Joined workspace(float* ws, const PagedDims& dm) {
  return {ws, ws + (long)dm.Hk * dm.q_rows * dm.by.G * dm.parts * dm.D};
}
__device__ __forceinline__ long ws_row(const PagedSeq& q, int kvh, int row, const PagedDims& dm) {
  return ((long)kvh * dm.q_rows + q.start) * dm.by.G + row;
}

// --------------------------------------------------------------------------------------------------------- single tokens
template <typename T, int DP>
__global__ __launch_bounds__(64 * (WaveTiles<T, DP>::NW)) void s2g_k_paged_attn_keys(
    const T* __restrict__ Q, const T* __restrict__ keys, const T* __restrict__ values, const int* __restrict__ table,
    const int* __restrict__ lens, const int* __restrict__ starts, T* __restrict__ out, float* __restrict__ ws, PagedDims dm) {
  typedef WaveTiles<T, DP> KT;
  typedef typename KT::LT LT;
  constexpr int KEYS = KT::KEYS, STEP = KEYS * KT::NW;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int pair = shared_lines(blockIdx.x, gridDim.x, dm.line_heads);
  const int kvh = pair % dm.Hk, tile = blockIdx.y, s = blockIdx.z, part = part_of(pair / dm.Hk, s + tile, dm.parts);
  const PagedSeq sq = paged_seq(lens, starts, s, dm);
  if (tile * 32 >= sq.rows) return;
  const int seen = keys_seen(sq, tile * 32 + 31, dm);
  const int lo = part * dm.part_keys, hi = min(seen, lo + dm.part_keys);
  if (lo >= hi && part > 0) return;
  const bool alone = seen <= dm.part_keys;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int row = tile * 32 + (lane & 31), rr = min(row, sq.rows - 1);
  const bool live = row < sq.rows;
  const int tok = divide(rr, dm.by), head = kvh * dm.by.G + rr - tok * dm.by.G;
  const int last = live ? (dm.causal ? min(sq.first + tok, sq.len - 1) : sq.len - 1) : -1;
  const int w_lo = keys_seen(sq, tile * 32, dm) - 1;           // every row sees the keys up to here
  table += (long)s * dm.cols;
  const T* kb = keys + kvh * dm.hd;
  const T* vb = values + kvh * dm.hd;

  int off[LT::NI];
  page_offsets<LT, T>(off, 0, lane, dm);
  char* mine = lds + wave * (KT::ONCE ? 2 : 4) * LT::BYTES;
  // tiles lo + KEYS wave + STEP t, the pages of the one after next on their way with the next
  int k0 = lo + KEYS * wave;
  const int at = lane & (KEYS - 1);
  int page = page_of(table, k0 + at, hi, dm);
  Rows<T, DP> r;
  if (k0 < hi) fetch_pages<LT, 1>(mine, kb, vb, page, k0, hi, off, 0, lane, dm);
  int next = page_of(table, k0 + STEP + at, hi, dm);
  const T* qp = Q + ((long)sq.start + tok) * dm.ldq + head * dm.hq;
  r.begin(qp, dm.D, live, half, dm.scale);
  for (int t = 0; k0 < hi; ++t, k0 += STEP) {
    char* kt = mine + (KT::ONCE ? 0 : (t & 1) * 2 * LT::BYTES);
    wait_loads();
    const unsigned long long gone = __ballot(!in_pool(page, dm) && k0 + at < hi), absent = KEYS == 32 ? (unsigned)gone : gone;
    page = next;
    const bool edge = k0 + KEYS - 1 > min(w_lo, hi - 1), more = k0 + STEP < hi;
    const int end = min(last, hi - 1) - k0;
    if constexpr (KT::ONCE) {
      fx16 st[KT::KB];
      r.template scores<KT::KB>(st, kt, lane, [](int) {});
      wait_reads();
      if (more) fetch_pages<LT, 1, true, false>(kt, kb, vb, page, k0 + STEP, hi, off, 0, lane, dm);
      r.template add<KT::KB, false>(st, nullptr, nullptr, kt + LT::BYTES, edge, end, absent, lane);
      wait_reads();
      if (more) fetch_pages<LT, 1, false, true>(kt, kb, vb, page, k0 + STEP, hi, off, 0, lane, dm);
    } else {
      if (more) fetch_pages<LT, 1>(mine + ((t + 1) & 1) * 2 * LT::BYTES, kb, vb, page, k0 + STEP, hi, off, 0, lane, dm);
    }
    if (more) next = page_of(table, k0 + 2 * STEP + at, hi, dm);
    if constexpr (!KT::ONCE) r.template step<KT::KB, true>(kt, kt + LT::BYTES, edge, end, absent, lane);
  }
  // what rounding left of a weight may be zero, and makes NaN of an infinite value then: such rows are made anew
  if constexpr (sizeof(T) == 2) {
    bool none = false;
#pragma unroll
    for (int d = 0; d < Shape<T, DP>::DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) none = none || r.o[d][i] != r.o[d][i];
    r.tainted = r.tainted || __any(none && r.l == r.l);
  }
  const Joined j = workspace(ws, dm);
  const auto slow = [&](float f, float* to) {
    slow_pages<T, DP>(qp, kb, vb, table, lo + KT::KEYS * wave, KT::KEYS, STEP, hi, last, r.c, r.base(), f, to, true, dm.D, dm.page_shift, dm.pages, dm.page_ld, dm.ld);
  };
  const auto statistics = [&](float m, float sum) {
    if (!alone && live) {
      float* p = j.ml + (ws_row(sq, kvh, row, dm) * dm.parts + part) * 2;
      p[0] = m;
      p[1] = sum;
    }
  };
  join_waves<KT>(lds, r, min(32, sq.rows - tile * 32), alone, dm.D, wave, lane, slow, statistics, [&](int y, int d, const fx4& a) {
    const int ry = tile * 32 + y;
    if (alone) {
      const int tk = divide(ry, dm.by);
      put4(out + (((long)sq.start + tk) * dm.H + kvh * dm.by.G + ry - tk * dm.by.G) * dm.D + d, a);
    } else {
      *reinterpret_cast<fx4*>(j.sums + (ws_row(sq, kvh, ry, dm) * dm.parts + part) * dm.D + d) = a;
    }
  });
}

// ---------------------------------------------------------------------------------------------------------------- chunks
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void s2g_k_paged_attn_rows(
    const T* __restrict__ Q, const T* __restrict__ keys, const T* __restrict__ values, const int* __restrict__ table,
    const int* __restrict__ lens, const int* __restrict__ starts, T* __restrict__ out, float* __restrict__ ws, PagedDims dm) {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int kvh = blockIdx.x % dm.Hk, tile = blockIdx.x / dm.Hk, s = blockIdx.z, part = part_of(blockIdx.y, s, dm.parts);
  const PagedSeq sq = paged_seq(lens, starts, s, dm);
  if (tile * 128 >= sq.rows) return;
  const int seen = keys_seen(sq, tile * 128 + 127, dm);
  const int lo = part * dm.part_keys, hi = min(seen, lo + dm.part_keys);
  if (lo >= hi && part > 0) return;
  const bool alone = seen <= dm.part_keys;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int w_row = tile * 128 + 32 * wave, row = w_row + (lane & 31), rr = min(row, sq.rows - 1);
  const bool live = row < sq.rows;
  const int tok = divide(rr, dm.by), head = kvh * dm.by.G + rr - tok * dm.by.G;
  const int last = live ? (dm.causal ? min(sq.first + tok, sq.len - 1) : sq.len - 1) : -1;
  const int w_lo = keys_seen(sq, w_row, dm) - 1, w_hi = w_row < sq.rows ? keys_seen(sq, w_row + 31, dm) - 1 : -1;
  table += (long)s * dm.cols;
  const T* kb = keys + kvh * dm.hd;
  const T* vb = values + kvh * dm.hd;
  int off[LT::NI];
  page_offsets<LT, T>(off, wave, lane, dm);

  const int kl = lane & (S::KT - 1);
  int k0 = lo, page = page_of(table, k0 + kl, hi, dm);
  if (k0 < hi) {
    fetch_pages<LT, 4>(lds, kb, vb, page, k0, hi, off, wave, lane, dm);
  }
  int next = page_of(table, k0 + S::KT + kl, hi, dm);
  Rows<T, DP> r;
  const T* qp = Q + ((long)sq.start + tok) * dm.ldq + head * dm.hq;
  r.begin(qp, dm.D, live, half, dm.scale);
  for (int t = 0; k0 < hi; ++t, k0 += S::KT) {
    const char* kt = lds + (t & 1) * 2 * LT::BYTES;
    wait_loads();
    const unsigned long long absent = __ballot(!in_pool(page, dm) && k0 + kl < hi);
    page = next;
    __syncthreads();
    if (k0 + S::KT < hi) {
      fetch_pages<LT, 4>(lds + ((t + 1) & 1) * 2 * LT::BYTES, kb, vb, page, k0 + S::KT, hi, off, wave, lane, dm);
      next = page_of(table, k0 + 2 * S::KT + kl, hi, dm);
    }
    if (k0 > w_hi) continue;
    const bool edge = k0 + S::KT - 1 > min(w_lo, hi - 1);
    r.template step<S::KB>(kt, kt + LT::BYTES, edge, min(last, hi - 1) - k0, absent, lane);
  }
  S::whole(r.o, lane);
  const float l = both_sum(r.l);
  if (alone) {
    T* to = out + (((long)sq.start + tok) * dm.H + head) * dm.D;
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (r.tainted) slow_pages<T, DP>(qp, kb, vb, table, lo, 32, 32, hi, last, r.c, r.base(), f, to, live, dm.D, dm.page_shift, dm.pages, dm.page_ld, dm.ld);
    else store_rows<T, S::DB>(to, r.o, f, dm.D, half, live);
  } else {
    const Joined j = workspace(ws, dm);
    const long at = ws_row(sq, kvh, rr, dm) * dm.parts + part;
    float* to = j.sums + at * dm.D;
    if (r.tainted) slow_pages<T, DP>(qp, kb, vb, table, lo, 32, 32, hi, last, r.c, r.base(), 1.0f, to, live, dm.D, dm.page_shift, dm.pages, dm.page_ld, dm.ld);
    else store_rows<T, S::DB>(to, r.o, 1.0f, dm.D, half, live);
    if (live && half == 0) {
      j.ml[2 * at] = r.m;
      j.ml[2 * at + 1] = l;
    }
  }
}

// The parts of a row brought to its maximum and added.  Up to 32 parts: half a wave to a row, lane p of the half holding
// part p's factor, each lane four features.
template <typename T>
__global__ __launch_bounds__(256) void s2g_k_paged_join_few(const float* __restrict__ ws, const int* __restrict__ lens,
                                                            const int* __restrict__ starts, T* __restrict__ out, int tile_rows,
                                                            PagedDims dm) {
  const int l32 = threadIdx.x & 31, kvh = blockIdx.x % dm.Hk, row = blockIdx.x / dm.Hk * 8 + (threadIdx.x >> 5);
  const PagedSeq sq = paged_seq(lens, starts, blockIdx.z, dm);
  if (row >= sq.rows) return;
  const int seen = keys_seen(sq, row / tile_rows * tile_rows + tile_rows - 1, dm);     // as the row's workgroup saw it
  const int parts = (seen + dm.part_keys - 1) / dm.part_keys;
  if (parts <= 1) return;
  const Joined j = workspace(const_cast<float*>(ws), dm);
  const long at = ws_row(sq, kvh, row, dm) * dm.parts;
  const float* sums = j.sums + at * dm.D;
  const int p0 = min(l32, parts - 1), d = min(4 * l32, dm.D - 4);
  const float2 ml = *reinterpret_cast<const float2*>(j.ml + 2 * (at + p0));
  fx4 a = {0.0f, 0.0f, 0.0f, 0.0f};
  fx4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const fx4*>(sums + (long)min(i, parts - 1) * dm.D + d);
  float m = ml.x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float f = ml.x == m ? 1.0f : __builtin_amdgcn_exp2f((ml.x - m) * dm.scale * LOG2E);
  float l = l32 < parts ? ml.y * f : 0.0f;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) l += __shfl_xor(l, o);
  for (int p = 0; p < parts; p += 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float w = __shfl(f, p + i, 32);
      if (p + i < parts) {
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = fmaf(x[i][k], w, a[k]);
      }
      x[i] = *reinterpret_cast<const fx4*>(sums + (long)min(p + 4 + i, parts - 1) * dm.D + d);
    }
  }
  if (4 * l32 >= dm.D) return;
  const int tk = divide(row, dm.by);
  typename Vec<T>::v4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = (T)(l == 0.0f ? 0.0f : a[k] / l);
  *reinterpret_cast<typename Vec<T>::v4*>(out + (((long)sq.start + tk) * dm.H + kvh * dm.by.G + row - tk * dm.by.G) * dm.D + d) = v;
}

// Many parts: a workgroup to a row, the parts dealt to its four waves, eight loads of each on their way at a time (a loop of
// single loads would wait for memory at every part), the waves' sums added in order.
template <typename T>
__global__ __launch_bounds__(256) void s2g_k_paged_join_many(const float* __restrict__ ws, const int* __restrict__ lens,
                                                             const int* __restrict__ starts, T* __restrict__ out, int tile_rows,
                                                             PagedDims dm) {
  __shared__ float sum[4][132];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int kvh = blockIdx.x % dm.Hk, row = blockIdx.x / dm.Hk;
  const PagedSeq sq = paged_seq(lens, starts, blockIdx.z, dm);
  const int seen = row < sq.rows ? keys_seen(sq, row / tile_rows * tile_rows + tile_rows - 1, dm) : 0;
  const int parts = (seen + dm.part_keys - 1) / dm.part_keys;
  if (parts <= 1) return;                       // the whole workgroup
  const Joined j = workspace(const_cast<float*>(ws), dm);
  const long at = ws_row(sq, kvh, row, dm) * dm.parts;
  const float* ml = j.ml + 2 * at;
  const float* sums = j.sums + at * dm.D;
  const float c = dm.scale * LOG2E;
  float m = -INFINITY;
  for (int p = lane; p < parts; p += 64) m = fmaxf(m, ml[2 * p]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  const int f0 = min(lane, dm.D - 1), f1 = min(lane + 64, dm.D - 1);
  float l = 0.0f, a0 = 0.0f, a1 = 0.0f;
  for (int p0 = wave; p0 < parts; p0 += 32) {
    float mp[8], lp[8], x0[8], x1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = min(p0 + 4 * i, parts - 1);
      mp[i] = ml[2 * p];
      lp[i] = ml[2 * p + 1];
      x0[i] = sums[(long)p * dm.D + f0];
      x1[i] = sums[(long)p * dm.D + f1];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (p0 + 4 * i < parts) {
        const float f = mp[i] == m ? 1.0f : __builtin_amdgcn_exp2f((mp[i] - m) * c);
        l = fmaf(lp[i], f, l);
        a0 = fmaf(x0[i], f, a0);
        a1 = fmaf(x1[i], f, a1);
      }
  }
  sum[wave][lane] = a0;
  sum[wave][lane + 64] = a1;
  if (lane == 0) sum[wave][128] = l;
  __syncthreads();
  if (wave != 0) return;
  a0 = (sum[0][lane] + sum[1][lane]) + (sum[2][lane] + sum[3][lane]);
  a1 = (sum[0][lane + 64] + sum[1][lane + 64]) + (sum[2][lane + 64] + sum[3][lane + 64]);
  l = (sum[0][128] + sum[1][128]) + (sum[2][128] + sum[3][128]);
  const int tk = divide(row, dm.by);
  T* o = out + (((long)sq.start + tk) * dm.H + kvh * dm.by.G + row - tk * dm.by.G) * dm.D;
  if (lane < dm.D) o[lane] = (T)(l == 0.0f ? 0.0f : a0 / l);
  if (lane + 64 < dm.D) o[lane + 64] = (T)(l == 0.0f ? 0.0f : a1 / l);
}

// ----------------------------------------------------------------------------------------------------------------- host
template <typename T, int DP>
static int launch_paged(const void* Q, const void* keys, const void* values, const int* table, const int* lens,
                        const int* starts, void* out, float* ws, int by_rows, const PagedDims& dm, hipStream_t st) {
  static S2GLdsCap rcap, kcap;
  const int tile_rows = by_rows ? 128 : 32, tiles = (dm.max_rows + tile_rows - 1) / tile_rows;
  const dim3 grid((unsigned)dm.Hk * dm.parts, tiles, dm.n);
  if (by_rows) {
    const auto kernel = s2g_k_paged_attn_rows<T, DP>;
    const int bytes = 4 * Shape<T, DP>::LT::BYTES;
    if (s2g_lds_cap(rcap, reinterpret_cast<const void*>(kernel), bytes) != 0) return -2;
    hipLaunchKernelGGL(kernel, dim3((unsigned)dm.Hk * tiles, dm.parts, dm.n), dim3(256), bytes, st, (const T*)Q, (const T*)keys, (const T*)values, table, lens, starts, (T*)out, ws, dm);
  } else {
    const auto kernel = s2g_k_paged_attn_keys<T, DP>;
    typedef WaveTiles<T, DP> KT;
    const int join = KT::NW * (64 + 32 * (32 * Shape<T, DP>::DB + 4)) * (int)sizeof(float), bytes = KT::BYTES > join ? KT::BYTES : join;
    if (s2g_lds_cap(kcap, reinterpret_cast<const void*>(kernel), bytes) != 0) return -2;
    hipLaunchKernelGGL(kernel, grid, dim3(64 * KT::NW), bytes, st, (const T*)Q, (const T*)keys, (const T*)values, table, lens, starts, (T*)out, ws, dm);
  }
  if (dm.parts > 32)
    hipLaunchKernelGGL(s2g_k_paged_join_many<T>, dim3((unsigned)dm.Hk * dm.max_rows, 1, dm.n), dim3(256), 0, st, ws, lens, starts, (T*)out, tile_rows, dm);
  else if (dm.parts > 1)
    hipLaunchKernelGGL(s2g_k_paged_join_few<T>, dim3((unsigned)dm.Hk * ((dm.max_rows + 7) / 8), 1, dm.n), dim3(256), 0, st, ws, lens, starts, (T*)out, tile_rows, dm);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int PACKED_NAME(s2g_launch_paged)(const void* Q, const void* keys, const void* values, const int* table,
                                             const int* lens, const int* starts, void* out, float* ws, int by_rows,
                                             PagedDims dm, hipStream_t st) {
  return PER_DIM(launch_paged, PACKED_T, Q, keys, values, table, lens, starts, out, ws, by_rows, dm, st);
}
