// Attention over packed sequences of different lengths, grouped heads, causal or not, and its gradient.
//
//   S = scale Q K^T,  P = softmax over the keys a row sees,  O = P V            (row i of n_q sees keys j <= i + n_k - n_q)
//   D = rowsum(dO o O),  dS = P o (dO V^T - D),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// No matrix of scores is stored: the forward pass keeps the running maximum and sum of every row and leaves their
// logarithm L (base 2) behind, the backward pass makes P = 2^(S log2(e) - L) again.
//
// Rows.  The G query heads of one kv head read the same keys, so they are rows of one problem: row r of a sequence
// and kv head j is token r / G, head j G + r % G.  A tile of 128 rows is then 128 / G tokens, which wastes less of a
// short sequence and of the causal diagonal than one head at a time.
//
// Work list.  The host knows the lengths, so it lays out one entry per (sequence, tile), longest first, and the
// kernels bring nothing but that entry: no search, no empty workgroups.  Workgroup b takes kv head b % Hk of entry
// b / Hk: with 8 kv heads each XCD (workgroups are dealt to the 8 XCDs in turn) keeps to one head's K and V.
#include "attn_rows.h"
#include "packed_attention.h"

// rows of a wave: O = sum over their keys among lo .. lo + width - 1, lo + step .., up to `keys`, of 2^(c s - base) V, times f
template <typename T, int DP, typename U>
__device__ __attribute__((noinline)) void slow_out(const T* q, const T* k, long ldk, const T* v, long ldv, int lo, int width, int step,
                                                   int keys, int last, float c, float base, float f, U* out, T* rest, int D, bool live) {
  const int half = (threadIdx.x >> 5) & 1;
  for (int from = 16 * half; from < DP + 16 * half; from += 32) {                // both halves take every turn: their dots are one
    float acc[16] = {};
    for (int k0 = lo; k0 < keys; k0 += step)
      for (int key = k0; key < min(k0 + width, keys); ++key) {
        const float w = __builtin_amdgcn_exp2f(fmaf(slow_dot<T, DP / 16>(q, k + key * ldk, D, half), c, -base));
        if (key <= last) slow_add(acc, w, v + key * ldv, from, D);
      }
    slow_store(out, acc, f, from, D, live);
    if (rest) {
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[j] = acc[j] * f - (float)(T)(acc[j] * f);
      slow_store(rest, acc, 1.0f, from, D, live);
    }
  }
}
// dQ of a wave's rows over the same keys
template <typename T, int DP, typename U>
__device__ __attribute__((noinline)) void slow_dq(const T* q, const T* g, const T* k, long ldk, const T* v, long ldv, int lo, int width,
                                                  int step, int keys, int last, float c, float scale, float L, float delta, U* dq, int D, bool live) {
  const int half = (threadIdx.x >> 5) & 1;
  for (int from = 16 * half; from < DP + 16 * half; from += 32) {
    float acc[16] = {};
    for (int k0 = lo; k0 < keys; k0 += step)
      for (int key = k0; key < min(k0 + width, keys); ++key) {
        const float p = __builtin_amdgcn_exp2f(fmaf(slow_dot<T, DP / 16>(q, k + key * ldk, D, half), c, -L));
        const float ds = last == 0 ? 0.0f : p * (slow_dot<T, DP / 16>(g, v + key * ldv, D, half) - delta);
        if (key <= last) slow_add(acc, ds, k + key * ldk, from, D);
      }
    slow_store(dq, acc, scale, from, D, live);
  }
}
// dK (which 0) or dV (1) of a wave's keys, over the rows lo .. hi of their kv head
template <typename T, int DP, typename U>
__device__ __attribute__((noinline)) void slow_key(int which, const T* k, const T* v, const T* Q, const T* dO, const float* lse,
                                                   const float* delta, int lo, int hi, int first, float c, float f, U* to, bool live,
                                                   int D, DivBy by, long ldq, long hq, long ldo, long ho) {
  const int half = (threadIdx.x >> 5) & 1;
  for (int from = 16 * half; from < DP + 16 * half; from += 32) {
    float acc[16] = {};
    for (int r = lo; r < hi; ++r) {
      const int tk = divide(r, by), h = r - tk * by.G;
      const T* q = Q + tk * ldq + h * hq;
      const T* g = dO + tk * ldo + h * ho;
      const float p = __builtin_amdgcn_exp2f(fmaf(slow_dot<T, DP / 16>(k, q, D, half), c, -lse[r]));
      const float ds = p * (slow_dot<T, DP / 16>(v, g, D, half) - delta[r]);
      if (r >= first) slow_add(acc, which ? p : ds, which ? g : q, from, D);
    }
    slow_store(to, acc, f, from, D, live);
  }
}

// Rounding dS and P to 16 bits adds as much to dQ, dK and dV as rounding those results does (1.44 times the error, all
// told), and more where a row's few slopes, which add up to zero, nearly cancel (1.5 to 1.9 times, over short sequences).
// So for rows that see at most this many keys the products of the backward pass take what rounding left, too: 1.05 to 1.25
// times, over long sequences 1.3.  They are the first rows of a long sequence or all of short ones; it costs 3 % of a
// training step on sequences up to 4096 and 9 us of 80 on 96 of up to 203 tokens (12 heads of 64).
// fp16 slopes are not raised as the weights are (by 2^11 in the forward pass, by 2^14 on the key side): how large they get is
// up to dO and V, so nothing says how far they may be.  Those below 2^-14 lose bits and those beyond 65504 are infinite, like dO,
// dQ, dK and dV of that size themselves: fp16 training scales its loss.
#define FEW_KEYS 128
template <typename T>
__device__ __forceinline__ fx16 left_by_rounding(const fx16& x) {
  fx16 y;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float d = x[i] - (float)(T)x[i];
    y[i] = fabsf(d) < INFINITY ? d : 0.0f;           // infinities stay what they are
  }
  return y;
}

// -------------------------------------------------------------------------------------------------------------- forward
// 128 rows to a workgroup of four waves, 64 keys to a tile; K and V twice in LDS (64 KB at 128 features), so that two
// workgroups share a compute unit and one's 2^x stand beside the other's products.  Bound by the matrix units, and at long
// prompts by power: 8191 + 1025 + 5000 bf16 tokens, 32 query and 8 kv heads of 128, 748 to 765 us, 1020 to 1000 TFLOP/s, the units busy half
// of the time at 1.8 GHz (one 8192^3 product of the library: 1140 TFLOP/s).  64 fp32 sequences up to 512, 4 heads of 16: 28 us
// (query side of the gradient 38), the units busy 26 (28) % of the time and the waves waiting 40 %.  It is not the longest
// sequences' chain of products: a quarter of it (s2g_k_packed_attn_fwd_few) takes as long.
template <typename T, int DP, bool TRAIN>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void s2g_k_packed_attn_fwd(const T* __restrict__ Q, const T* __restrict__ K,
                                                             const T* __restrict__ V, T* __restrict__ out,
                                                             T* __restrict__ rest, float* __restrict__ lse, const PackedTile* __restrict__ tiles,
                                                             PackedDims dm) {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int rows = w.q_len * dm.by.G, row = w.tile * 128 + 32 * wave + (lane & 31);
  const bool live = row < rows;
  const int tok = divide(min(row, rows - 1), dm.by), head = kvh * dm.by.G + (min(row, rows - 1) - tok * dm.by.G);
  const long qrow = (long)w.q_start + tok;
  const T* qp = Q + qrow * dm.ldq + head * dm.hq;
  const T* kp = K + (long)w.k_start * dm.ldk + kvh * dm.hk;
  const T* vp = V + (long)w.k_start * dm.ldv + kvh * dm.hv;

  Rows<T, DP, TRAIN> r;
  r.begin(qp, dm.D, live, half, dm.scale);
  // the last key this row sees; of this wave's rows, and of the workgroup's
  const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
  const int last = live ? min(w.k_len - 1, tok + shift) : -1;
  const int w_lo = min(w.k_len - 1, divide(min(w.tile * 128 + 32 * wave, rows - 1), dm.by) + shift);
  const int w_hi = w.tile * 128 + 32 * wave < rows ? min(w.k_len - 1, divide(min(w.tile * 128 + 32 * wave + 31, rows - 1), dm.by) + shift) : -1;
  const int b_hi = min(w.k_len - 1, divide(min(w.tile * 128 + 127, rows - 1), dm.by) + shift);
  const int nt = b_hi < 0 ? 0 : b_hi / S::KT + 1;

  int ko[LT::NI], vo[LT::NI];
  tile_offsets<LT, T>(ko, dm.ldk, dm.D, wave, lane);
  tile_offsets<LT, T>(vo, dm.ldv, dm.D, wave, lane);
  // 32 keys at a time: while one half of a tile is summed, the scores of the next half are made.  So the tiles of K lie 32
  // keys ahead of those of V.  LDS: K even, K odd, V even, V odd; two turns of the loop, so that every LDS address is a
  // register and a constant.
  const auto fetch = [&](const T* p, long ld, int key, int place, const int* off) {
    fetch_rows<LT>(lds + place * LT::BYTES, p + (long)key * ld, ld, dm.D, min(S::KT, w.k_len - key), off, wave);
  };
  constexpr int HALF = 32 * S::PITCH * (int)sizeof(T);
  fx16 one, two;
  const int mine = w_hi < 0 ? 0 : w_hi / S::KT + 1;         // tiles that some row of this wave sees
  if (nt > 0) {
    fetch(kp, dm.ldk, 0, 1, ko);                            // the first 32 keys
    fetch(kp, dm.ldk, 32, 0, ko);
    fetch(vp, dm.ldv, 0, 2, vo);
    wait_loads();
    __syncthreads();
    r.template scores<1>(&one, lds + LT::BYTES, lane, [](int) {});
  }
  const auto turn = [&](int t, auto parity) {
    constexpr int P = decltype(parity)::value;
    wait_loads();
    __syncthreads();            // this turn's K and V are here; everyone is done with the last turn's
    const int k0 = t * S::KT;
    if (t + 1 < nt) {
      fetch(kp, dm.ldk, k0 + S::KT + 32, 1 - P, ko);
      fetch(vp, dm.ldv, k0 + S::KT, 3 - P, vo);
    }
    if (t >= mine) return;
    const char* kt = lds + P * LT::BYTES;                   // behind the last key: scores that nobody takes
    const char* vt = lds + (2 + P) * LT::BYTES;
    r.template add<1, true>(&one, &two, kt, vt, k0 + 31 > w_lo, last - k0, 0, lane);
    if constexpr (S::KB == 2) r.template add<1, true>(&two, &one, kt + HALF, vt + HALF, k0 + 63 > w_lo, last - k0 - 32, 0, lane);
    else one = two;
  };
  for (int t = 0; t < nt; t += 2) {
    turn(t, std::integral_constant<int, 0>{});
    if (t + 1 < nt) turn(t + 1, std::integral_constant<int, 1>{});
  }
  S::whole(r.o, lane);
  const float l = both_sum(r.l), f = l == 0.0f ? 0.0f : 1.0f / l, sum = TRAIN ? both_sum(r.whole) : l;
  const long orow = (qrow * dm.H + head) * dm.D;
  // a row that sees no key gives zeros, and L = +inf makes its P zero in the backward pass
  if (lse && live && half == 0)
    lse[((long)kvh * dm.q_rows + w.q_start) * dm.by.G + row] = l == 0.0f ? INFINITY : r.log_sum(sum);
  if (r.tainted) {
    slow_out<T, DP>(qp, kp, dm.ldk, vp, dm.ldv, 0, 32, 32, w_hi + 1, last, r.c, r.base(), f,
                    out + orow, sizeof(T) == 2 && rest ? rest + orow : nullptr, dm.D, live);
    return;
  }
  store_rows<T, S::DB>(out + orow, r.o, f, dm.D, half, live);
  // what rounding took from O: with it the backward pass has D = dO . O nearly exactly where dP - D is a small difference.
  // Only rows of few keys need it: of n like keys, D's error is 1 / sqrt(n) of what rounding dS adds.  (Without it dQ and dK
  // of short fp16 sequences are off by 1.57 times the result's own rounding, with it by 1.45.)
  if (sizeof(T) == 2 && rest && w_lo < FEW_KEYS) {
#pragma unroll
    for (int d = 0; d < S::DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) r.o[d][i] = r.o[d][i] * f - (float)(T)(r.o[d][i] * f);
    store_rows<T, S::DB>(rest + orow, r.o, 1.0f, dm.D, half, live && last < FEW_KEYS);
  }
}

// The same for few tiles, which would leave most compute units idle: 32 rows to a workgroup (blockIdx.y: which of the tile's
// 128), every wave over 32-key tiles of its own, joined at the end as in the paged cache's single tokens.  4444 fp16 tokens,
// 3 / 1 heads of 128: 85 -> 61 us; 1000 bf16 tokens, 8 heads of 128: 25 -> 15; 8 fp32 sequences up to 722, 2 heads of 96:
// 90 -> 30.  (few_tiles() says when.)
template <typename T, int DP, bool TRAIN>
__global__ __launch_bounds__(64 * (WaveTiles<T, DP>::NW)) void s2g_k_packed_attn_fwd_few(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, T* __restrict__ out, T* __restrict__ rest,
    float* __restrict__ lse, const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef WaveTiles<T, DP> WT;
  typedef typename WT::LT LT;
  constexpr int STEP = WT::KEYS * WT::NW;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int rows = w.q_len * dm.by.G, row0 = w.tile * 128 + 32 * blockIdx.y;
  if (row0 >= rows) return;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int row = row0 + (lane & 31);
  const bool live = row < rows;
  const int tok = divide(min(row, rows - 1), dm.by), head = kvh * dm.by.G + (min(row, rows - 1) - tok * dm.by.G);
  const T* qp = Q + ((long)w.q_start + tok) * dm.ldq + head * dm.hq;
  const T* kp = K + (long)w.k_start * dm.ldk + kvh * dm.hk;
  const T* vp = V + (long)w.k_start * dm.ldv + kvh * dm.hv;
  const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
  const int last = live ? min(w.k_len - 1, tok + shift) : -1;
  const int w_lo = min(w.k_len - 1, divide(row0, dm.by) + shift);
  const int hi = max(0, min(w.k_len, divide(min(row0 + 31, rows - 1), dm.by) + shift + 1));       // the keys that some row sees
  int ko[LT::NI], vo[LT::NI];
  tile_offsets<LT, T>(ko, dm.ldk, dm.D, 0, lane);
  tile_offsets<LT, T>(vo, dm.ldv, dm.D, 0, lane);
  char* mine = lds + wave * (WT::ONCE ? 2 : 4) * LT::BYTES;
  const auto fetch_k = [&](int k0, char* to) { fetch_rows<LT, T, 1>(to, kp + (long)k0 * dm.ldk, dm.ldk, dm.D, min(WT::KEYS, w.k_len - k0), ko, 0); };
  const auto fetch_v = [&](int k0, char* to) { fetch_rows<LT, T, 1>(to, vp + (long)k0 * dm.ldv, dm.ldv, dm.D, min(WT::KEYS, w.k_len - k0), vo, 0); };
  const int first = WT::KEYS * wave;
  if (first < hi) {
    fetch_k(first, mine);
    fetch_v(first, mine + LT::BYTES);
  }
  Rows<T, DP, TRAIN> r;
  r.begin(qp, dm.D, live, half, dm.scale);
  for (int t = 0, k0 = first; k0 < hi; ++t, k0 += STEP) {
    char* kt = mine + (WT::ONCE ? 0 : (t & 1) * 2 * LT::BYTES);
    const bool edge = k0 + WT::KEYS - 1 > w_lo, more = k0 + STEP < hi;
    wait_loads();
    if constexpr (WT::ONCE) {
      fx16 st[WT::KB];
      r.template scores<WT::KB>(st, kt, lane, [](int) {});
      wait_reads();
      if (more) fetch_k(k0 + STEP, kt);
      r.template add<WT::KB, false>(st, nullptr, nullptr, kt + LT::BYTES, edge, last - k0, 0, lane);
      wait_reads();
      if (more) fetch_v(k0 + STEP, kt + LT::BYTES);
    } else {
      if (more) {
        char* to = mine + ((t + 1) & 1) * 2 * LT::BYTES;
        fetch_k(k0 + STEP, to);
        fetch_v(k0 + STEP, to + LT::BYTES);
      }
      r.template step<WT::KB>(kt, kt + LT::BYTES, edge, last - k0, 0, lane);
    }
  }
  const auto slow = [&](float f, float* to) {
    slow_out<T, DP>(qp, kp, dm.ldk, vp, dm.ldv, first, WT::KEYS, STEP, hi, last, r.c, r.base(), f, to, (T*)nullptr, dm.D, true);
  };
  const auto statistics = [&](float m, float sum) {
    if (lse && live)
      lse[((long)kvh * dm.q_rows + w.q_start) * dm.by.G + row] = sum == 0.0f ? INFINITY : fmaf(m, r.c, __builtin_amdgcn_logf(sum)) - Weights<T>::RAISE;
  };
  join_waves<WT>(lds, r, min(32, rows - row0), true, dm.D, wave, lane, slow, statistics, [&](int y, int d, const fx4& a) {
    const int tk = divide(row0 + y, dm.by);
    const long at = (((long)w.q_start + tk) * dm.H + kvh * dm.by.G + row0 + y - tk * dm.by.G) * dm.D + d;
    put4(out + at, a);
    if (sizeof(T) == 2 && rest && min(w.k_len - 1, tk + shift) < FEW_KEYS)
      put4(rest + at, (fx4){a[0] - (float)(T)a[0], a[1] - (float)(T)a[1], a[2] - (float)(T)a[2], a[3] - (float)(T)a[3]});
  });
}

// ------------------------------------------------------------------------------------------------- backward, query side
// D of every row, and dQ: lanes are rows, as in the forward pass.  Three products (S, dP, dQ) to the forward's two.  8 bf16
// sequences up to 4096, 16 query and 4 kv heads of 128: 302 to 324 us, 1015 to 950 TFLOP/s.  Making dQ here and not with atomics from the
// key side costs S and dP twice (two products of seven) and keeps every bit the same from run to run.  FEW: few tiles, as in
// s2g_k_packed_attn_fwd_few (4444 fp16 tokens, 3 / 1 heads of 128: 96 -> 74 us).
template <typename T, int DP, bool FEW>
__global__ __launch_bounds__(FEW ? 64 * (WaveTiles<T, DP>::NW) : 256, FEW || sizeof(T) == 4 ? 1 : 2) void s2g_k_packed_attn_bwd_q(const T* __restrict__ Q, const T* __restrict__ K,
                                                               const T* __restrict__ V, const T* __restrict__ out,
                                                               const T* __restrict__ rest, const T* __restrict__ dO, const float* __restrict__ lse,
                                                               float* __restrict__ delta, T* __restrict__ dQ,
                                                               const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef Shape<T, DP> S;
  typedef WaveTiles<T, DP> WT;
  typedef typename std::conditional<FEW, typename WT::LT, typename S::LT>::type LT;
  constexpr int KT = FEW ? WT::KEYS : S::KT, KB = KT / 32, STEP = FEW ? KT * WT::NW : KT, LOADERS = FEW ? 1 : 4;
  constexpr bool ONCE = FEW && WT::ONCE;
  typedef typename Vec<T>::v8 v8;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int rows = w.q_len * dm.by.G, row0 = w.tile * 128 + 32 * (FEW ? (int)blockIdx.y : wave), row = row0 + (lane & 31);
  if (FEW && row0 >= rows) return;
  const bool live = row < rows;
  const int tok = divide(min(row, rows - 1), dm.by), head = kvh * dm.by.G + (min(row, rows - 1) - tok * dm.by.G);
  const long qrow = (long)w.q_start + tok, orow = (qrow * dm.H + head) * dm.D, lrow = ((long)kvh * dm.q_rows + w.q_start) * dm.by.G + row;
  const T* qp = Q + qrow * dm.ldq + head * dm.hq;
  const T* gp = dO + qrow * dm.ldo + head * dm.ho;
  const T* kp = K + (long)w.k_start * dm.ldk + kvh * dm.hk;
  const T* vp = V + (long)w.k_start * dm.ldv + kvh * dm.hv;

  const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
  const int last = live ? min(w.k_len - 1, tok + shift) : -1;
  const int w_lo = min(w.k_len - 1, divide(min(row0, rows - 1), dm.by) + shift);
  const int w_hi = row0 < rows ? min(w.k_len - 1, divide(min(row0 + 31, rows - 1), dm.by) + shift) : -1;
  const int b_hi = FEW ? w_hi : min(w.k_len - 1, divide(min(w.tile * 128 + 127, rows - 1), dm.by) + shift);
  const int first = FEW ? KT * wave : 0;                         // this wave's first tile of keys

  v8 q[S::KS], g[S::KS];
  float dl = 0.0f;
  {
    v8 y[S::KS], x[S::KS];
    const bool few = sizeof(T) == 2 && w_lo < FEW_KEYS;
#pragma unroll
    for (int s = 0; s < S::KS; ++s) {
      const int at = 16 * s + 8 * half;
      q[s] = row8(qp, at, dm.D, live);
      g[s] = row8(gp, at, dm.D, live);
      y[s] = row8(out + orow, at, dm.D, live);
    }
    if (few)
#pragma unroll
      for (int s = 0; s < S::KS; ++s) x[s] = row8(rest + orow, 16 * s + 8 * half, dm.D, live && last < FEW_KEYS);
#pragma unroll
    for (int s = 0; s < S::KS; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) dl = fmaf((float)g[s][j], (float)y[s][j], dl);
    if (few)
#pragma unroll
      for (int s = 0; s < S::KS; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) dl = fmaf((float)g[s][j], (float)x[s][j], dl);
  }
  dl = both_sum(dl);
  const float L = live ? lse[lrow] : INFINITY, c = dm.scale * LOG2E;

  int ko[LT::NI], vo[LT::NI];
  tile_offsets<LT, T>(ko, dm.ldk, dm.D, FEW ? 0 : wave, lane);
  tile_offsets<LT, T>(vo, dm.ldv, dm.D, FEW ? 0 : wave, lane);
  bool tainted = false;            // a tile with hidden keys held an infinity or a NaN in K
  fx16 dq[S::DB];
#pragma unroll
  for (int d = 0; d < S::DB; ++d) dq[d] = zero16();
  char* mine = lds + (FEW ? wave * (ONCE ? 2 : 4) * LT::BYTES : 0);
  const auto place = [&](int t) { return mine + (ONCE ? 0 : (t & 1) * 2 * LT::BYTES); };
  const auto fetch_k = [&](int k0, int t) {
    fetch_rows<LT, T, LOADERS>(place(t), kp + (long)k0 * dm.ldk, dm.ldk, dm.D, min(KT, w.k_len - k0), ko, FEW ? 0 : wave);
  };
  const auto fetch_v = [&](int k0, int t) {
    fetch_rows<LT, T, LOADERS>(place(t) + LT::BYTES, vp + (long)k0 * dm.ldv, dm.ldv, dm.D, min(KT, w.k_len - k0), vo, FEW ? 0 : wave);
  };
  if (first <= b_hi) {
    fetch_k(first, 0);
    fetch_v(first, 0);
  }
  for (int t = 0, k0 = first; k0 <= b_hi; ++t, k0 += STEP) {
    const char* kt = place(t);
    const char* vt = kt + LT::BYTES;
    const bool more = k0 + STEP <= b_hi;
    wait_loads();
    if (!FEW) __syncthreads();
    if (!ONCE && more) {
      fetch_k(k0 + STEP, t + 1);
      fetch_v(k0 + STEP, t + 1);
    }
    if (k0 > w_hi) continue;
    const bool edge = k0 + KT - 1 > w_lo;
    // 32 keys at a time, 2^x beside the products of dP, dS beside those of the next keys' S
    fx16 st = zero16(), next;
    products<T, S::KS, S::AHEAD>([&](int i) { return LT::along(kt, lane & 31, i, half); },
                                 [&](int i, const v8& a) { st = mma(a, q[i], st); }, [](int) {});
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      fx16 dp = zero16();
      products<T, S::KS, S::AHEAD>([&](int i) { return LT::along(vt, 32 * b + (lane & 31), i, half); },
                                   [&](int i, const v8& a) { dp = mma(a, g[i], dp); },
                                   [&](int i) {
#pragma unroll
                                     for (int e = 16 * i / S::KS; e < 16 * (i + 1) / S::KS; ++e) st[e] = __builtin_amdgcn_exp2f(fmaf(st[e], c, -L));
                                   });
      if constexpr (ONCE) {                       // (32 keys)
        wait_reads();
        if (more) fetch_v(k0 + STEP, 0);
      }
      // a row that sees one key only has D = dP there, to the last bit: its scores have no gradient
      if (b == 0 && k0 == 0 && last == 0) dl = dp[0];
      const auto slope = [&](int i) {
#pragma unroll
        for (int e = 16 * i / S::KS; e < 16 * (i + 1) / S::KS; ++e) st[e] *= dp[e] - dl;
      };
      if (b + 1 < KB) {
        next = zero16();
        products<T, S::KS, S::AHEAD>([&](int i) { return LT::along(kt, 32 * (b + 1) + (lane & 31), i, half); },
                                     [&](int i, const v8& a) { next = mma(a, q[i], next); }, slope);
      } else {
#pragma unroll
        for (int i = 0; i < S::KS; ++i) slope(i);
      }
      if (edge) {
        tainted = tainted || not_finite<T>(kt + 32 * b * S::PITCH * (int)sizeof(T), 32 * S::PITCH * (int)sizeof(T), lane);
        const int at = hidden(last - k0 - 32 * b - 4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (reg_row(i) > at) st[i] = 0.0f;
      }
      const v8 ds[2] = {operand<T>(st, 0), operand<T>(st, 1)};
      products<T, 2 * S::DB, S::AHEAD>([&](int i) { return LT::across(kt, i % S::DB, 2 * b + i / S::DB, lane); },
                                       [&](int i, const v8& a) { dq[i % S::DB] = S::sum(a, ds[i / S::DB], dq[i % S::DB]); }, [](int) {});
      if (sizeof(T) == 2 && __builtin_expect(w_lo < FEW_KEYS, 0)) {
        const fx16 z = left_by_rounding<T>(st);
        const v8 ds[2] = {operand<T>(z, 0), operand<T>(z, 1)};
        products<T, 2 * S::DB, S::AHEAD>([&](int i) { return LT::across(kt, i % S::DB, 2 * b + i / S::DB, lane); },
                                         [&](int i, const v8& a) { dq[i % S::DB] = S::sum(a, ds[i / S::DB], dq[i % S::DB]); }, [](int) {});
      }
      st = next;
    }
    if constexpr (ONCE) {
      wait_reads();
      if (more) fetch_k(k0 + STEP, 0);
    }
  }
  if (live && half == 0 && (!FEW || wave == 0)) delta[lrow] = dl;          // (the first wave has seen the first key)
  if constexpr (FEW) {
    S::whole(dq, lane);
    __syncthreads();
    float* os = reinterpret_cast<float*>(lds);
    float* to = os + (wave * 32 + (lane & 31)) * WT::PAD;
    if (tainted) slow_dq<T, DP>(qp, gp, kp, dm.ldk, vp, dm.ldv, first, KT, STEP, w_hi + 1, last, c, dm.scale, L, dl, to, dm.D, true);
    else store_rows<T, S::DB>(to, dq, dm.scale, 32 * S::DB, half, true);
    __syncthreads();
    add_waves<WT>(os, min(32, rows - row0), dm.D, [&](int y, int d, const fx4& a) {
      const int tk = divide(row0 + y, dm.by);
      put4(dQ + (((long)w.q_start + tk) * dm.H + kvh * dm.by.G + row0 + y - tk * dm.by.G) * dm.D + d, a);
    });
  } else {
    if (tainted) {
      slow_dq<T, DP>(qp, gp, kp, dm.ldk, vp, dm.ldv, 0, 32, 32, w_hi + 1, last, c, dm.scale, L, dl, dQ + orow, dm.D, live);
      return;
    }
    S::whole(dq, lane);
    store_rows<T, S::DB>(dQ + orow, dq, dm.scale, dm.D, half, live);
  }
}

// --------------------------------------------------------------------------------------------------- backward, key side
// dK and dV of 128 keys: lanes are keys, the rows of the kv head's G query heads come by in tiles.  The first keys of a
// long sequence are seen by all its rows: where such a tile is more than its share of the work, or the tiles are too few
// for the chip, the host cuts a tile's rows into ranges, each leaving a 32-bit partial result in a slot of its own that
// s2g_k_packed_attn_sum adds in a fixed order: no atomics, the same bits every time.
//
// Four products (S, dP, dK, dV).  8 bf16 sequences up to 4096, 16 query and 4 kv heads of 128: 510 to 547 us, 805 to 750
// TFLOP/s, and 15 us for the sums of cut tiles.  96 fp16 sequences up to 203, 12 heads of 64: 33 us and 7.  64 fp32 sequences up
// to 512, 4 heads of 16: 37 to 40 us, the matrix units busy 35 % of the time and the waves waiting 37 %; as long with a third
// workgroup to a compute unit.
//
// Two forms.  Up to 64 16-bit features, and in fp32, a wave takes 32 keys.  Beyond, the sums of dK and dV of 32 keys with
// their K and V leave room for only one wave to a SIMD, which keeps the matrix unit idle while it makes P and dS; so there
// two waves share 32 keys (s2g_k_packed_attn_bwd_kv2).
template <typename T, int DP>
struct KeySums {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  typedef typename Vec<T>::v8 v8;
  // fp16 weights below 2^-14 lose bits, and a long row's are that small: the products of dV take them 2^14 times as large, as in
  // PairSums (of 90000 like keys, dV off by 2^-8.8 of itself without it; 8 sequences up to 4096, 16 / 4 heads of 64: 299 -> 307 us).
  static constexpr float RAISE = std::is_same<T, _Float16>::value ? 16384.0f : 1.0f;
  v8 k[S::KS], v[S::KS];
  fx16 dv[S::DB], dk[S::DB];
  bool tainted;                // a tile with rows that do not see some key held an infinity or a NaN

  __device__ __forceinline__ void begin(const T* kp, const T* vp, int D, bool live, int half) {
#pragma unroll
    for (int s = 0; s < S::KS; ++s) {
      k[s] = row8(kp, 16 * s + 8 * half, D, live);
      v[s] = row8(vp, 16 * s + 8 * half, D, live);
    }
#pragma unroll
    for (int d = 0; d < S::DB; ++d) {
      dv[d] = zero16();
      dk[d] = zero16();
      tainted = false;
    }
  }
  // a tile of rows: Q, dO, (L, D); edge: some of them do not see some of the wave's keys (`first`: the first that sees this
  // lane's, counted from the tile's first); few: some of them see few keys
  __device__ __forceinline__ void step(const char* qt, const char* gt, const float* sl, float c, bool few, bool edge, int first, int lane) {
    const int half = lane >> 5, col = lane & 31;
    if (edge) tainted = tainted || not_finite<T>(qt, 2 * LT::BYTES, lane);        // Q and dO, side by side
#pragma unroll
    for (int b = 0; b < S::KB; ++b) {
      fx16 p = zero16(), ds = zero16();
#pragma unroll
      for (int s = 0; s < S::KS; ++s) p = mma(LT::along(qt, 32 * b + col, s, half), k[s], p);
#pragma unroll
      for (int s = 0; s < S::KS; ++s) ds = mma(LT::along(gt, 32 * b + col, s, half), v[s], ds);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const fx4 L = *reinterpret_cast<const fx4*>(sl + 32 * b + 8 * g + 4 * half);
        const fx4 D = *reinterpret_cast<const fx4*>(sl + S::KT + 32 * b + 8 * g + 4 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * g + j;
          p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c, -L[j]));
          ds[i] = p[i] * (ds[i] - D[j]);
          if constexpr (RAISE != 1.0f) p[i] *= RAISE;
        }
      }
      if (edge) {
        const int at = hidden(first - 4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + reg_row(i) < at) p[i] = 0.0f, ds[i] = 0.0f;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const v8 pt = operand<T>(p, s), dt = operand<T>(ds, s);
#pragma unroll
        for (int d = 0; d < S::DB; ++d) dv[d] = S::sum(LT::across(gt, d, 2 * b + s, lane), pt, dv[d]);
#pragma unroll
        for (int d = 0; d < S::DB; ++d) dk[d] = S::sum(LT::across(qt, d, 2 * b + s, lane), dt, dk[d]);
      }
      if (sizeof(T) == 2 && __builtin_expect(few, 0)) {
        const fx16 y = left_by_rounding<T>(p), z = left_by_rounding<T>(ds);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const v8 yt = operand<T>(y, s), zt = operand<T>(z, s);
#pragma unroll
          for (int d = 0; d < S::DB; ++d) dv[d] = mma(LT::across(gt, d, 2 * b + s, lane), yt, dv[d]);
#pragma unroll
          for (int d = 0; d < S::DB; ++d) dk[d] = mma(LT::across(qt, d, 2 * b + s, lane), zt, dk[d]);
        }
      }
    }
  }
};

// What both forms know of a wave's 32 keys and of the rows that see them
struct KeyWork {
  PackedTile w;
  int kvh, rows, few, first, w_lo, w_hi, t0, t1;
  bool live, ragged;
  long krow, lrow;
  // ROWS rows to a tile; `group`: which 32 of the tile's 128 keys
  template <int ROWS>
  __device__ __forceinline__ void begin(const PackedTile* tiles, int group, int lane, const PackedDims& dm) {
    kvh = blockIdx.x % dm.Hk;
    w = tiles[blockIdx.x / dm.Hk];
    const int G = dm.by.G, w_key = w.tile * 128 + 32 * group, key = w_key + (lane & 31);
    rows = w.q_len * G;
    live = key < w.k_len;
    krow = (long)w.k_start + min(key, w.k_len - 1);
    lrow = ((long)kvh * dm.q_rows + w.q_start) * G;
    // the first row that sees this key, the wave's first and last, the tiles of rows that see some key of the workgroup
    const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
    first = !live ? 0x7fffffff : max(0, key - shift) * G;
    w_lo = w_key < w.k_len ? max(0, w_key - shift) * G : 0x7fffffff;
    w_hi = max(0, min(w_key + 31, w.k_len - 1) - shift) * G;
    few = w.k_len <= FEW_KEYS ? rows : dm.causal ? (FEW_KEYS - shift) * G : 0;          // rows before this one see few keys
    ragged = w_key + 31 >= w.k_len;
    t0 = max(max(0, w.tile * 128 - shift) * G, w.row_lo) / ROWS;           // row_lo, row_hi: whole tiles
    t1 = (min(rows, w.row_hi) + ROWS - 1) / ROWS;
  }
  // Q and dO of a tile of rows from r0 on, side by side: the group's heads of a token, then the next token.  Where whole
  // tokens fill the tiles (`off`, made once by offsets()) a tile is fetched as the one before; other groups divide anew.
  // Behind the last row come its Q again, zeros of dO and an infinite L, so that they weigh nothing: zeros of Q would make NaN of
  // a key that is minus infinity, whose weight every row that there is takes for zero.
  template <typename LT, typename T>
  __device__ __forceinline__ void offsets(int* off, long ld, long hd, int wave, int lane, const PackedDims& dm) const {
#pragma unroll
    for (int i = 0; i < LT::NI; ++i) {
      const int r = LT::row_of(i, wave, lane), tk = divide(r, dm.by), ch = LT::chunk_of(i, wave, lane) * 16;
      off[i] = ch < dm.D * (int)sizeof(T) ? (int)((tk * ld + (r - tk * dm.by.G) * hd) * (long)sizeof(T)) + ch : OUT_OF_BUFFER;
    }
  }
  template <typename LT, int WAVES, int ROWS, typename T>
  __device__ __forceinline__ void fetch(unsigned to, int r0, const T* Q, const T* dO, const int* qoff, const int* goff, int wave,
                                        int lane, const PackedDims& dm) const {
    const int G = dm.by.G, tok0 = divide(r0, dm.by);
    const ix4 qr = buffer_of(Q + ((long)w.q_start + tok0) * dm.ldq + kvh * G * dm.hq, 0x7ffffe00);
    const ix4 gr = buffer_of(dO + ((long)w.q_start + tok0) * dm.ldo + kvh * G * dm.ho, 0x7ffffe00);
    if (ROWS % G == 0 && r0 + ROWS <= rows) {
#pragma unroll
      for (int i = 0; i < LT::NI; ++i) {
        load_to_lds(qr, to + (i * WAVES + wave) * 1024, qoff[i]);
        load_to_lds(gr, to + LT::BYTES + (i * WAVES + wave) * 1024, goff[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < LT::NI; ++i) {
        const int at = r0 + LT::row_of(i, wave, lane), r = min(at, rows - 1), tk = divide(r, dm.by), hd = r - tk * G;
        const int ch = LT::chunk_of(i, wave, lane) * 16;
        const bool ok = ch < dm.D * (int)sizeof(T);
        load_to_lds(qr, to + (i * WAVES + wave) * 1024, ok ? (int)(((tk - tok0) * dm.ldq + hd * dm.hq) * (long)sizeof(T)) + ch : OUT_OF_BUFFER);
        load_to_lds(gr, to + LT::BYTES + (i * WAVES + wave) * 1024,
                    ok && at < rows ? (int)(((tk - tok0) * dm.ldo + hd * dm.ho) * (long)sizeof(T)) + ch : OUT_OF_BUFFER);
      }
    }
  }
  // where this lane's key's dK (second 0) or dV (1) goes
  template <typename T>
  __device__ __forceinline__ T* row_of(T* out, const PackedDims& dm) const { return out + (krow * dm.Hk + kvh) * dm.D; }
  __device__ __forceinline__ float* slot_of(float* partial, int second, int group, int lane, const PackedDims& dm) const {
    return partial + (((long)w.slot * dm.Hk + kvh) * 256 + 128 * second + 32 * group + (lane & 31)) * dm.D;
  }
  template <typename T, int DB>
  __device__ __forceinline__ void store(T* out, float* partial, int second, const fx16* acc, float f, int group, int lane, const PackedDims& dm) const {
    if (w.slot < 0) store_rows<T, DB>(row_of(out, dm), acc, f, dm.D, lane >> 5, live);
    else store_rows<T, DB>(slot_of(partial, second, group, lane, dm), acc, f, dm.D, lane >> 5, live);
  }
  template <typename T, int DP>
  __device__ __forceinline__ void slow(int second, const T* Q, const T* K, const T* V, const T* dO, const float* lse, const float* delta,
                                       T* out, float* partial, int rows_per_tile, int group, int lane, const PackedDims& dm) const {
    const T* k = K + krow * dm.ldk + kvh * dm.hk;
    const T* v = V + krow * dm.ldv + kvh * dm.hv;
    const T* q = Q + (long)w.q_start * dm.ldq + kvh * dm.by.G * dm.hq;
    const T* g = dO + (long)w.q_start * dm.ldo + kvh * dm.by.G * dm.ho;
    const int lo = t0 * rows_per_tile, hi = min(rows, t1 * rows_per_tile);
    const float c = dm.scale * LOG2E, f = second ? 1.0f : dm.scale;
    if (w.slot < 0) slow_key<T, DP>(second, k, v, q, g, lse + lrow, delta + lrow, lo, hi, first, c, f, row_of(out, dm), live, dm.D, dm.by, dm.ldq, dm.hq, dm.ldo, dm.ho);
    else slow_key<T, DP>(second, k, v, q, g, lse + lrow, delta + lrow, lo, hi, first, c, f, slot_of(partial, second, group, lane, dm), live, dm.D, dm.by, dm.ldq, dm.hq, dm.ldo, dm.ho);
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void s2g_k_packed_attn_bwd_kv(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ dO,
    const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dK, T* __restrict__ dV,
    float* __restrict__ partial, const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  extern __shared__ __attribute__((aligned(1024))) char lds[];       // Q, dO, Q, dO, then 2 x (L, D)
  float* stats = reinterpret_cast<float*>(lds + 4 * LT::BYTES);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  KeyWork kw;
  kw.begin<S::KT>(tiles, wave, lane, dm);
  int qoff[LT::NI], goff[LT::NI];
  kw.offsets<LT, T>(qoff, dm.ldq, dm.hq, wave, lane, dm);
  kw.offsets<LT, T>(goff, dm.ldo, dm.ho, wave, lane, dm);
  const auto fetch = [&](int t) {
    kw.fetch<LT, 4, S::KT>(lds_address(lds) + (t & 1) * 2 * LT::BYTES, t * S::KT, Q, dO, qoff, goff, wave, lane, dm);
  };
  float st_next = 0.0f;
  const auto stat = [&](int t) {                                      // threads 0 .. 2 KT: L, then D of the tile's rows
    const int r = t * S::KT + (threadIdx.x & (S::KT - 1));
    st_next = threadIdx.x < S::KT ? INFINITY : 0.0f;
    if (threadIdx.x < 2 * S::KT && r < kw.rows) st_next = (threadIdx.x < S::KT ? lse : delta)[kw.lrow + r];
  };
  const float c = dm.scale * LOG2E;
  if (kw.t0 < kw.t1) {
    stat(kw.t0);
    fetch(kw.t0);
  }
  KeySums<T, DP> sums;
  sums.begin(K + kw.krow * dm.ldk + kw.kvh * dm.hk, V + kw.krow * dm.ldv + kw.kvh * dm.hv, dm.D, kw.live, lane >> 5);
  for (int t = kw.t0; t < kw.t1; ++t) {
    const char* qt = lds + (t & 1) * 2 * LT::BYTES;
    float* sl = stats + (t & 1) * 2 * S::KT;
    wait_loads();
    if (threadIdx.x < 2 * S::KT) sl[threadIdx.x] = st_next;
    __syncthreads();
    if (t + 1 < kw.t1) {
      stat(t + 1);
      fetch(t + 1);
    }
    const int r0 = t * S::KT;
    if (r0 + S::KT <= kw.w_lo) continue;                              // none of these rows sees this wave's keys
    sums.step(qt, qt + LT::BYTES, sl, c, r0 < kw.few, kw.ragged || r0 < kw.w_hi, kw.first - r0, lane);
  }
  if (sums.tainted) {
    kw.slow<T, DP>(0, Q, K, V, dO, lse, delta, dK, partial, S::KT, wave, lane, dm);
    kw.slow<T, DP>(1, Q, K, V, dO, lse, delta, dV, partial, S::KT, wave, lane, dm);
    return;
  }
  S::whole(sums.dk, lane);
  S::whole(sums.dv, lane);
  kw.store<T, S::DB>(dK, partial, 0, sums.dk, dm.scale, wave, lane, dm);
  kw.store<T, S::DB>(dV, partial, 1, sums.dv, 1.0f / sums.RAISE, wave, lane, dm);
}

// Two waves to 32 keys: wave g of the first four makes S, P and dV, wave 4 + g dP, dS and dK.  P goes from one to the other
// through LDS.  For bf16 it goes as the upper 24 bits of a float: its range, as a key that no row weighs much has weights of any
// size and dK made of them (as fp16 they would end at 2^-38), and 2^-15 of a weight, a hundredth of what rounding dS to bf16
// takes (two instructions a weight: 497 -> 510 us).  fp16 has dS in more bits, so there it goes whole, and a tile is half as many
// rows; the weights are raised by 2^14, as dV's products take them.
// The first four are a tile ahead, so that neither waits for the other within one.
template <typename T, int DP>
struct PairSums {
  typedef Shape<T, DP> S;
  static constexpr bool WIDE = std::is_same<T, _Float16>::value;
  static constexpr int BLOCKS = WIDE ? 1 : 2, ROWS = 32 * BLOCKS;
  typedef Tile<T, S::PITCH, ROWS, 8> LT;
  typedef typename Vec<T>::v8 v8;
  static constexpr int UNITS = WIDE ? 4 : 3, SHARE = BLOCKS * UNITS * 64;      // 16-byte units of P of 32 rows per lane; of a tile
  static constexpr int BYTES = 6 * LT::BYTES + 8 * SHARE * 16 + 3 * 2 * ROWS * (int)sizeof(float);
  static_assert(BYTES <= 163840, "LDS");
  static constexpr float RAISE = WIDE ? 14.0f : 0.0f, LOWER = WIDE ? 1.0f / 16384.0f : 1.0f;
  v8 k[S::KS];                                     // K of the first four, V of the others
  fx16 sum[S::DB];
  bool tainted;                                    // a tile with rows that do not see some key held an infinity or a NaN

  __device__ __forceinline__ void begin(const T* p, int D, bool live, int half) {
#pragma unroll
    for (int s = 0; s < S::KS; ++s) k[s] = row8(p, 16 * s + 8 * half, D, live);
#pragma unroll
    for (int d = 0; d < S::DB; ++d) sum[d] = zero16();
    tainted = false;
  }
  template <typename B>
  __device__ __forceinline__ void rows_by_keys(const char* tile, int b, fx16& to, int lane, B beside) const {
    to = zero16();
    products<T, S::KS, S::AHEAD>([&](int i) { return LT::along(tile, 32 * b + (lane & 31), i, lane >> 5); },
                                 [&](int i, const v8& a) { to = mma(a, k[i], to); }, beside);
  }
  __device__ __forceinline__ void add(const char* tile, int b, const v8* x, int lane) {
    products<T, 2 * S::DB, S::AHEAD>([&](int i) { return LT::across(tile, i % S::DB, 2 * b + i / S::DB, lane); },
                                     [&](int i, const v8& a) { sum[i % S::DB] = mma(a, x[i / S::DB], sum[i % S::DB]); }, [](int) {});
  }
  // f(0 .. 3) over the S::KS products that they stand beside
  template <typename F>
  static __device__ __forceinline__ auto spread(F f) {
    return [f](int i) {
#pragma unroll
      for (int g = 4 * i / S::KS; g < 4 * (i + 1) / S::KS; ++g) f(g);
    };
  }
  static __device__ __forceinline__ void mask(fx16& x, int first, int lane) {
    const int at = hidden(first - 4 * (lane >> 5));
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (reg_row(i) < at) x[i] = 0.0f;
  }
  static __device__ __forceinline__ void give(fx4* share, const fx16& p, int lane) {
    if constexpr (WIDE) {
#pragma unroll
      for (int u = 0; u < 4; ++u) share[u * 64 + lane] = (fx4){p[4 * u], p[4 * u + 1], p[4 * u + 2], p[4 * u + 3]};
    } else {
      unsigned w[12];                              // four floats' upper three bytes in three words
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const unsigned x0 = bits(p[4 * g]), x1 = bits(p[4 * g + 1]), x2 = bits(p[4 * g + 2]), x3 = bits(p[4 * g + 3]);
        w[3 * g] = __builtin_amdgcn_perm(x1, x0, 0x05030201u);
        w[3 * g + 1] = __builtin_amdgcn_perm(x2, x1, 0x06050302u);
        w[3 * g + 2] = __builtin_amdgcn_perm(x3, x2, 0x07060503u);
      }
#pragma unroll
      for (int u = 0; u < 3; ++u)
        share[u * 64 + lane] = (fx4){flt(w[4 * u]), flt(w[4 * u + 1]), flt(w[4 * u + 2]), flt(w[4 * u + 3])};
    }
  }
  static __device__ __forceinline__ unsigned bits(float x) { return __builtin_bit_cast(unsigned, x); }
  static __device__ __forceinline__ float flt(unsigned x) { return __builtin_bit_cast(float, x); }
  // P of register i out of what was given
  static __device__ __forceinline__ float given(const fx4* x, int i) {
    if constexpr (WIDE) return x[i >> 2][i & 3];
    else {
      const auto w = [&](int k) { const float y = x[k >> 2][k & 3]; return bits(y); };
      const int k = 3 * (i >> 2);
      switch (i & 3) {
        case 0: return flt(w(k) << 8);
        case 1: return flt(__builtin_amdgcn_perm(w(k + 1), w(k), 0x0504030cu));
        case 2: return flt(__builtin_amdgcn_perm(w(k + 2), w(k + 1), 0x0403020cu));
        default: return flt(w(k + 2) & 0xffffff00u);
      }
    }
  }
  // a tile of rows: P to `share` ([block][unit][lane] of 16 bytes), dV^T += dO^T P
  __device__ __forceinline__ void weights(const char* qt, const char* gt, const float* L, fx4* share, float c, bool few, bool edge, int first, int lane) {
    fx16 p, next;
    if (edge) tainted = tainted || not_finite<T>(gt, LT::BYTES, lane);
    rows_by_keys(qt, 0, p, lane, [](int) {});
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      const auto weigh = [&](int g) {
        const fx4 l = *reinterpret_cast<const fx4*>(L + 32 * b + 8 * g + 4 * (lane >> 5));
#pragma unroll
        for (int i = 4 * g; i < 4 * g + 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c, l[i & 3]));
      };
      if (b + 1 < BLOCKS) rows_by_keys(qt, 1, next, lane, spread(weigh));
      else
#pragma unroll
        for (int g = 0; g < 4; ++g) weigh(g);
      if (edge) mask(p, first - 32 * b, lane);
      give(share + b * UNITS * 64, p, lane);
      const v8 x[2] = {operand<T>(p, 0), operand<T>(p, 1)};
      add(gt, b, x, lane);
      if (__builtin_expect(few, 0)) {
        const fx16 y = left_by_rounding<T>(p);
        const v8 x[2] = {operand<T>(y, 0), operand<T>(y, 1)};
        add(gt, b, x, lane);
      }
      p = next;
    }
  }
  // the same rows, P taken from `share`: dK^T += Q^T dS
  __device__ __forceinline__ void slopes(const char* qt, const char* gt, const float* D, const fx4* share, bool few, bool edge, int first, int lane) {
    fx16 ds, next;
    if (edge) tainted = tainted || not_finite<T>(qt, LT::BYTES, lane);
    rows_by_keys(gt, 0, ds, lane, [](int) {});
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
      fx4 x[UNITS];
#pragma unroll
      for (int u = 0; u < UNITS; ++u) x[u] = share[(b * UNITS + u) * 64 + lane];
      const auto slope = [&](int g) {
        const fx4 d = *reinterpret_cast<const fx4*>(D + 32 * b + 8 * g + 4 * (lane >> 5));
#pragma unroll
        for (int i = 4 * g; i < 4 * g + 4; ++i) ds[i] = given(x, i) * (WIDE ? fmaf(ds[i], LOWER, d[i & 3]) : ds[i] + d[i & 3]);
      };
      if (b + 1 < BLOCKS) rows_by_keys(gt, 1, next, lane, spread(slope));
      else
#pragma unroll
        for (int g = 0; g < 4; ++g) slope(g);
      if (edge) mask(ds, first - 32 * b, lane);
      const v8 y[2] = {operand<T>(ds, 0), operand<T>(ds, 1)};
      add(qt, b, y, lane);
      if (__builtin_expect(few, 0)) {
        const fx16 z = left_by_rounding<T>(ds);
        const v8 y[2] = {operand<T>(z, 0), operand<T>(z, 1)};
        add(qt, b, y, lane);
      }
      ds = next;
    }
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void s2g_k_packed_attn_bwd_kv2(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ dO,
    const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dK, T* __restrict__ dV,
    float* __restrict__ partial, const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef PairSums<T, DP> P;
  typedef typename P::LT LT;
  constexpr int DB = Shape<T, DP>::DB, ROWS = P::ROWS;
  extern __shared__ __attribute__((aligned(1024))) char lds[];       // 3 x (Q, dO), 2 x 4 x P, 3 x (L, D)
  fx4* shares = reinterpret_cast<fx4*>(lds + 6 * LT::BYTES);
  float* stats = reinterpret_cast<float*>(shares + 8 * P::SHARE);
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), group = wave & 3;
  KeyWork kw;
  kw.begin<ROWS>(tiles, group, lane, dm);
  const int t0 = kw.t0, t1 = kw.t1;
  int qoff[LT::NI], goff[LT::NI];
  kw.offsets<LT, T>(qoff, dm.ldq, dm.hq, wave, lane, dm);
  kw.offsets<LT, T>(goff, dm.ldo, dm.ho, wave, lane, dm);
  const auto fetch = [&](int t, int place) {
    kw.fetch<LT, 8, ROWS>(lds_address(lds) + place * 2 * LT::BYTES, t * ROWS, Q, dO, qoff, goff, wave, lane, dm);
  };
  float st_next = 0.0f;
  const auto stat = [&](int t) {                                      // threads 0 .. 2 ROWS: RAISE - L, then -LOWER D of the tile's rows
    const int r = t * ROWS + (threadIdx.x & (ROWS - 1));
    st_next = threadIdx.x < ROWS ? -INFINITY : 0.0f;
    if (threadIdx.x < 2 * ROWS && r < kw.rows) st_next = threadIdx.x < ROWS ? P::RAISE - lse[kw.lrow + r] : -P::LOWER * delta[kw.lrow + r];
  };
  const float c = dm.scale * LOG2E;
  if (t0 < t1) {
    stat(t0);
    fetch(t0, 0);
  }
  P sums;
  if (wave < 4) sums.begin(K + kw.krow * dm.ldk + kw.kvh * dm.hk, dm.D, kw.live, lane >> 5);
  else sums.begin(V + kw.krow * dm.ldv + kw.kvh * dm.hv, dm.D, kw.live, lane >> 5);
  // turn t: the first four at tile t, the others at tile t - 1, tile t + 1 on its way
  const auto turns = [&](auto first_four) {
    int at = 0;                                                       // (t - t0) % 3
    for (int t = t0; t < t1 + (t0 < t1); ++t) {
      const int next = at == 2 ? 0 : at + 1, before = at == 0 ? 2 : at - 1;
      wait_loads();
      if (threadIdx.x < 2 * ROWS && t < t1) stats[at * 2 * ROWS + threadIdx.x] = st_next;
      __syncthreads();
      if (t + 1 < t1) {
        stat(t + 1);
        fetch(t + 1, next);
      }
      const int mine = first_four.value ? t : t - 1, r0 = mine * ROWS, place = first_four.value ? at : before;
      at = next;
      if (mine < t0 || mine >= t1 || r0 + ROWS <= kw.w_lo) continue;   // none of these rows sees this wave's keys
      const char* qt = lds + place * 2 * LT::BYTES;
      const float* st = stats + place * 2 * ROWS;
      fx4* share = shares + ((mine & 1) * 4 + group) * P::SHARE;
      const bool edge = kw.ragged || r0 < kw.w_hi;
      if constexpr (first_four.value) sums.weights(qt, qt + LT::BYTES, st, share, c, r0 < kw.few, edge, kw.first - r0, lane);
      else sums.slopes(qt, qt + LT::BYTES, st + ROWS, share, r0 < kw.few, edge, kw.first - r0, lane);
    }
  };
  if (wave < 4) turns(std::true_type{});
  else turns(std::false_type{});
  if (sums.tainted) {
    kw.slow<T, DP>(wave < 4, Q, K, V, dO, lse, delta, wave < 4 ? dV : dK, partial, ROWS, group, lane, dm);
    return;
  }
  if (wave < 4) kw.store<T, DB>(dV, partial, 1, sums.sum, P::LOWER, group, lane, dm);
  else kw.store<T, DB>(dK, partial, 0, sums.sum, dm.scale, group, lane, dm);
}

// one cut tile (its entry's row_lo: the number of its slots) and kv head: blockIdx.y / 4 0 dK, 1 dV, and 32 of its keys
template <typename T>
__global__ __launch_bounds__(256) void s2g_k_packed_attn_sum(const float* __restrict__ partial, T* __restrict__ dK,
                                                             T* __restrict__ dV, const PackedTile* __restrict__ tiles,
                                                             PackedDims dm) {
  typedef typename Vec<T>::v4 v4;
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int n4 = dm.D >> 2, y0 = 32 * (blockIdx.y & 3), count = min(32, w.k_len - w.tile * 128 - y0) * n4;
  const long next = (long)dm.Hk * 256 * dm.D;
  const float* from = partial + (((long)w.slot * dm.Hk + kvh) * 256 + 32 * blockIdx.y) * dm.D;
  T* to = blockIdx.y >> 2 ? dV : dK;
  for (int e = threadIdx.x; e < count; e += 256) {
    const int y = e / n4, d = (e - y * n4) * 4;
    fx4 s = *reinterpret_cast<const fx4*>(from + y * dm.D + d);
#pragma unroll 4
    for (int p = 1; p < w.row_lo; ++p) {
      const fx4 x = *reinterpret_cast<const fx4*>(from + p * next + y * dm.D + d);
      s[0] += x[0]; s[1] += x[1]; s[2] += x[2]; s[3] += x[3];
    }
    v4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = (T)s[j];
    *reinterpret_cast<v4*>(to + (((long)w.k_start + w.tile * 128 + y0 + y) * dm.Hk + kvh) * dm.D + d) = r;
  }
}

// ----------------------------------------------------------------------------------------------------------------- host
// Whether 128-row tiles are too few for 256 compute units, so that 32 rows to a workgroup and keys dealt to its waves, at less
// a rate, end sooner.  Measured with tiles / with the keys dealt, forward and query side of the gradient (us):
// bf16, 8 heads of 128, 1000 tokens (64 tiles) 25 + 29 / 15 + 19; 2000 (128) 43 + 49 / 40 + 49; 16 / 4 heads of 64, 1500 (192) 19 +
// 22 / 18 + 23; 32 / 8 of 128, 700 (176) 20 + 25 / 29 + 37.  fp32, whose products take eight times as long: 8 / 4 heads of 128,
// 2630 tokens (168) 386 + 564 / 189 + 277; twice those (336) 394 + 568 / 323 + 474; 4 heads of 32, 8 x 1500 (384) 84 + 110 / 60 + 81;
// 32 x 500 (512) 35 + 47 / 40 + 55; 4 of 16, 64 up to 512 (700) 26 + 35 / 27 + 40.
template <typename T>
static bool few_tiles(int nt, const PackedDims& dm) { return (long)nt * dm.Hk <= (sizeof(T) == 4 ? 384 : 128); }

template <typename T, int DP, bool TRAIN>
static int launch_fwd_for(const void* Q, const void* K, const void* V, void* out, void* rest, float* lse, const PackedTile* tiles, int nt,
                          const PackedDims& dm, hipStream_t st) {
  static S2GLdsCap cap, few_cap;
  const auto launch = [&](auto kernel, S2GLdsCap& c, dim3 grid, int threads, int bytes) {
    if (s2g_lds_cap(c, reinterpret_cast<const void*>(kernel), bytes) != 0) return -2;
    hipLaunchKernelGGL(kernel, grid, dim3(threads), bytes, st, (const T*)Q, (const T*)K, (const T*)V, (T*)out, (T*)rest, lse, tiles, dm);
    return 0;
  };
  const int rc = few_tiles<T>(nt, dm) ? launch(s2g_k_packed_attn_fwd_few<T, DP, TRAIN>, few_cap, dim3((unsigned)nt * dm.Hk, 4), 64 * WaveTiles<T, DP>::NW, WaveTiles<T, DP>::BYTES)
                                      : launch(s2g_k_packed_attn_fwd<T, DP, TRAIN>, cap, dim3((unsigned)nt * dm.Hk), 256, 4 * Shape<T, DP>::LT::BYTES);
  if (rc != 0) return rc;
  return hipGetLastError() == hipSuccess ? 0 : -2;
}
template <typename T, int DP>
static int launch_fwd(const void* Q, const void* K, const void* V, void* out, void* rest, float* lse, const PackedTile* tiles, int nt,
                      const PackedDims& dm, hipStream_t st) {
  if constexpr (std::is_same<T, __bf16>::value)          // fp32 and fp16 sum the weights as they were anyway
    if (lse) return launch_fwd_for<T, DP, true>(Q, K, V, out, rest, lse, tiles, nt, dm, st);
  return launch_fwd_for<T, DP, false>(Q, K, V, out, rest, lse, tiles, nt, dm, st);
}
template <typename T, int DP>
static int launch_bwd(const void* Q, const void* K, const void* V, const void* out, const void* rest, const void* dO, const float* lse,
                      float* delta, void* dQ, void* dK, void* dV, float* partial, const PackedTile* qt, int nqt,
                      const PackedTile* kt, int nkt, const PackedTile* cut, int ncut, const PackedDims& dm, hipStream_t st) {
  typedef typename Shape<T, DP>::LT LT;
  constexpr bool PAIR = sizeof(T) == 2 && DP > 64;
  static S2GLdsCap qcap, few_cap, kcap;
  const auto query_side = [&](auto kq, S2GLdsCap& c, dim3 grid, int threads, int bytes) {
    if (s2g_lds_cap(c, reinterpret_cast<const void*>(kq), bytes) != 0) return -2;
    if (nqt > 0)
      hipLaunchKernelGGL(kq, grid, dim3(threads), bytes, st, (const T*)Q, (const T*)K, (const T*)V, (const T*)out, (const T*)rest,
                         (const T*)dO, lse, delta, (T*)dQ, qt, dm);
    return 0;
  };
  const auto key_side = [&](auto kk, int threads, int bytes) {
    if (s2g_lds_cap(kcap, reinterpret_cast<const void*>(kk), bytes) != 0) return -2;
    if (nkt > 0)
      hipLaunchKernelGGL(kk, dim3((unsigned)nkt * dm.Hk), dim3(threads), bytes, st, (const T*)Q, (const T*)K, (const T*)V,
                         (const T*)dO, lse, delta, (T*)dK, (T*)dV, partial, kt, dm);
    return 0;
  };
  int rc = few_tiles<T>(nqt, dm) ? query_side(s2g_k_packed_attn_bwd_q<T, DP, true>, few_cap, dim3((unsigned)nqt * dm.Hk, 4), 64 * WaveTiles<T, DP>::NW, WaveTiles<T, DP>::BYTES)
                                 : query_side(s2g_k_packed_attn_bwd_q<T, DP, false>, qcap, dim3((unsigned)nqt * dm.Hk), 256, 4 * LT::BYTES);
  if (rc != 0) return rc;
  if constexpr (PAIR) rc = key_side(s2g_k_packed_attn_bwd_kv2<T, DP>, 512, PairSums<T, DP>::BYTES);
  else rc = key_side(s2g_k_packed_attn_bwd_kv<T, DP>, 256, 4 * LT::BYTES + 4 * Shape<T, DP>::KT * (int)sizeof(float));
  if (rc != 0) return rc;
  if (ncut > 0)
    hipLaunchKernelGGL(s2g_k_packed_attn_sum<T>, dim3((unsigned)ncut * dm.Hk, 8), dim3(256), 0, st, partial, (T*)dK, (T*)dV, cut, dm);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int PACKED_NAME(s2g_launch_packed_fwd)(const void* Q, const void* K, const void* V, void* out, void* rest, float* lse,
                                                  const PackedTile* tiles, int nt, PackedDims dm, hipStream_t st) {
  return PER_DIM(launch_fwd, PACKED_T, Q, K, V, out, rest, lse, tiles, nt, dm, st);
}
extern "C" int PACKED_NAME(s2g_launch_packed_bwd)(const void* Q, const void* K, const void* V, const void* out,
                                                  const void* rest, const void* dO, const float* lse, float* delta, void* dQ, void* dK,
                                                  void* dV, float* partial, const PackedTile* qt, int nqt,
                                                  const PackedTile* kt, int nkt, const PackedTile* cut, int ncut,
                                                  PackedDims dm, hipStream_t st) {
  return PER_DIM(launch_bwd, PACKED_T, Q, K, V, out, rest, dO, lse, delta, dQ, dK, dV, partial, qt, nqt, kt, nkt, cut, ncut, dm, st);
}
