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
#include <type_traits>

// -------------------------------------------------------------------------------------------------------------- forward
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void s2g_k_packed_attn_fwd(const T* __restrict__ Q, const T* __restrict__ K,
                                                             const T* __restrict__ V, T* __restrict__ out,
                                                             float* __restrict__ lse, const PackedTile* __restrict__ tiles,
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

  Rows<T, DP> r;
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
  const float l = both_sum(r.l);
  store_rows<T, S::DB>(out + (qrow * dm.H + head) * dm.D, r.o, l == 0.0f ? 0.0f : 1.0f / l, dm.D, half, live);
  // a row that sees no key gives zeros, and L = +inf makes its P zero in the backward pass
  if (lse && live && half == 0)
    lse[((long)kvh * dm.q_rows + w.q_start) * dm.by.G + row] = l == 0.0f ? INFINITY : r.log_sum(l);
}

// ------------------------------------------------------------------------------------------------- backward, query side
// D of every row, and dQ: lanes are rows, as in the forward pass
template <typename T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void s2g_k_packed_attn_bwd_q(const T* __restrict__ Q, const T* __restrict__ K,
                                                               const T* __restrict__ V, const T* __restrict__ out,
                                                               const T* __restrict__ dO, const float* __restrict__ lse,
                                                               float* __restrict__ delta, T* __restrict__ dQ,
                                                               const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  typedef typename Vec<T>::v8 v8;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int rows = w.q_len * dm.by.G, row = w.tile * 128 + 32 * wave + (lane & 31);
  const bool live = row < rows;
  const int tok = divide(min(row, rows - 1), dm.by), head = kvh * dm.by.G + (min(row, rows - 1) - tok * dm.by.G);
  const long qrow = (long)w.q_start + tok, orow = (qrow * dm.H + head) * dm.D, lrow = ((long)kvh * dm.q_rows + w.q_start) * dm.by.G + row;
  const T* qp = Q + qrow * dm.ldq + head * dm.hq;
  const T* gp = dO + qrow * dm.ldo + head * dm.ho;
  const T* kp = K + (long)w.k_start * dm.ldk + kvh * dm.hk;
  const T* vp = V + (long)w.k_start * dm.ldv + kvh * dm.hv;

  v8 q[S::KS], g[S::KS];
  float dl = 0.0f;
#pragma unroll
  for (int s = 0; s < S::KS; ++s) {
    const int at = 16 * s + 8 * half;
    q[s] = row8(qp, at, dm.D, live);
    g[s] = row8(gp, at, dm.D, live);
    const v8 y = row8(out + orow, at, dm.D, live);
#pragma unroll
    for (int j = 0; j < 8; ++j) dl = fmaf((float)g[s][j], (float)y[j], dl);
  }
  dl = both_sum(dl);
  if (live && half == 0) delta[lrow] = dl;
  const float L = live ? lse[lrow] : INFINITY, c = dm.scale * LOG2E;

  const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
  const int last = live ? min(w.k_len - 1, tok + shift) : -1;
  const int w_lo = min(w.k_len - 1, divide(min(w.tile * 128 + 32 * wave, rows - 1), dm.by) + shift);
  const int w_hi = w.tile * 128 + 32 * wave < rows ? min(w.k_len - 1, divide(min(w.tile * 128 + 32 * wave + 31, rows - 1), dm.by) + shift) : -1;
  const int b_hi = min(w.k_len - 1, divide(min(w.tile * 128 + 127, rows - 1), dm.by) + shift);
  const int nt = b_hi < 0 ? 0 : b_hi / S::KT + 1;

  int ko[LT::NI], vo[LT::NI];
  tile_offsets<LT, T>(ko, dm.ldk, dm.D, wave, lane);
  tile_offsets<LT, T>(vo, dm.ldv, dm.D, wave, lane);
  fx16 dq[S::DB];
#pragma unroll
  for (int d = 0; d < S::DB; ++d) dq[d] = zero16();
  if (nt > 0) {
    fetch_rows<LT>(lds, kp, dm.ldk, dm.D, min(S::KT, w.k_len), ko, wave);
    fetch_rows<LT>(lds + LT::BYTES, vp, dm.ldv, dm.D, min(S::KT, w.k_len), vo, wave);
  }
  for (int t = 0; t < nt; ++t) {
    char* kt = lds + (t & 1) * 2 * LT::BYTES;
    const char* vt = kt + LT::BYTES;
    wait_loads();
    __syncthreads();
    if (t + 1 < nt) {
      char* nx = lds + ((t + 1) & 1) * 2 * LT::BYTES;
      const int k1 = (t + 1) * S::KT, n = min(S::KT, w.k_len - k1);
      fetch_rows<LT>(nx, kp + (long)k1 * dm.ldk, dm.ldk, dm.D, n, ko, wave);
      fetch_rows<LT>(nx + LT::BYTES, vp + (long)k1 * dm.ldv, dm.ldv, dm.D, n, vo, wave);
    }
    const int k0 = t * S::KT;
    if (k0 > w_hi) continue;
    const bool edge = k0 + S::KT - 1 > w_lo;
#pragma unroll
    for (int b = 0; b < S::KB; ++b) {
      fx16 st = zero16(), dp = zero16();
#pragma unroll
      for (int s = 0; s < S::KS; ++s) st = mma(LT::along(kt, 32 * b + (lane & 31), s, half), q[s], st);
#pragma unroll
      for (int s = 0; s < S::KS; ++s) dp = mma(LT::along(vt, 32 * b + (lane & 31), s, half), g[s], dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) st[i] = __builtin_amdgcn_exp2f(fmaf(st[i], c, -L)) * (dp[i] - dl);
      if (edge) {
        const int at = hidden(last - k0 - 4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + reg_row(i) > at) st[i] = 0.0f;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const v8 ds = operand<T>(st, s);
#pragma unroll
        for (int d = 0; d < S::DB; ++d) dq[d] = mma(LT::across(kt, d, 2 * b + s, lane), ds, dq[d]);
      }
    }
  }
  store_rows<T, S::DB>(dQ + orow, dq, dm.scale, dm.D, half, live);
}

// --------------------------------------------------------------------------------------------------- backward, key side
// dK and dV of 128 keys: lanes are keys, the rows of the kv head's G query heads come by in tiles.  The first keys of a
// long sequence are seen by all its rows: where such a tile is more than its share of the work, or the tiles are too few
// for the chip, the host cuts a tile's rows into ranges, each leaving a 32-bit partial result in a slot of its own that
// s2g_k_packed_attn_sum adds in a fixed order: no atomics, the same bits every time.
//
// The sums of dK and dV of 32 keys, with their K and V, leave room for one wave to a SIMD at 96 or 128 16-bit features,
// and one wave alone keeps the matrix unit idle while it makes P and dS.  There 8 waves share the work: waves 0 .. 3 take
// S and dV, waves 4 .. 7 S, dP and dK of the same keys, 40 products where 32 would do, but two waves to a SIMD
// (DKV_SPLIT_FIGURES).
template <typename T, int DP>
struct KeySide {
  static constexpr bool SPLIT = sizeof(T) == 2 && DP > 64;
  static constexpr int WAVES = SPLIT ? 8 : 4;
  typedef Tile<T, Shape<T, DP>::PITCH, Shape<T, DP>::KT, WAVES> LT;
};

template <typename T, int DP, bool DV, bool DK>
struct KeySums {
  typedef Shape<T, DP> S;
  typedef typename KeySide<T, DP>::LT LT;
  typedef typename Vec<T>::v8 v8;
  v8 k[S::KS], v[DK ? S::KS : 1];
  fx16 dv[DV ? S::DB : 1], dk[DK ? S::DB : 1];

  __device__ __forceinline__ void begin(const T* kp, const T* vp, int D, bool live, int half) {
#pragma unroll
    for (int s = 0; s < S::KS; ++s) {
      k[s] = row8(kp, 16 * s + 8 * half, D, live);
      if constexpr (DK) v[s] = row8(vp, 16 * s + 8 * half, D, live);
    }
#pragma unroll
    for (int d = 0; d < S::DB; ++d) {
      if constexpr (DV) dv[d] = zero16();
      if constexpr (DK) dk[d] = zero16();
    }
  }
  // a tile of rows: Q, dO, (L, D); edge: some of them do not see some of the wave's keys (`first`: the first that sees this
  // lane's, counted from the tile's first)
  __device__ __forceinline__ void step(const char* qt, const char* gt, const float* sl, float c, bool edge, int first, int lane) {
    const int half = lane >> 5, col = lane & 31;
#pragma unroll
    for (int b = 0; b < S::KB; ++b) {
      fx16 p = zero16(), ds = zero16();
#pragma unroll
      for (int s = 0; s < S::KS; ++s) p = mma(LT::along(qt, 32 * b + col, s, half), k[s], p);
      if constexpr (DK)
#pragma unroll
        for (int s = 0; s < S::KS; ++s) ds = mma(LT::along(gt, 32 * b + col, s, half), v[s], ds);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const fx4 L = *reinterpret_cast<const fx4*>(sl + 32 * b + 8 * g + 4 * half);
        fx4 D;
        if constexpr (DK) D = *reinterpret_cast<const fx4*>(sl + S::KT + 32 * b + 8 * g + 4 * half);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = 4 * g + j;
          p[i] = __builtin_amdgcn_exp2f(fmaf(p[i], c, -L[j]));
          if constexpr (DK) ds[i] = p[i] * (ds[i] - D[j]);
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
        if constexpr (DV) {
          const v8 pt = operand<T>(p, s);
#pragma unroll
          for (int d = 0; d < S::DB; ++d) dv[d] = mma(LT::across(gt, d, 2 * b + s, lane), pt, dv[d]);
        }
        if constexpr (DK) {
          const v8 dt = operand<T>(ds, s);
#pragma unroll
          for (int d = 0; d < S::DB; ++d) dk[d] = mma(LT::across(qt, d, 2 * b + s, lane), dt, dk[d]);
        }
      }
    }
  }
};

template <typename T, int DP>
__global__ __launch_bounds__(64 * (KeySide<T, DP>::WAVES), sizeof(T) == 2 ? 2 : 1) void s2g_k_packed_attn_bwd_kv(
    const T* __restrict__ Q, const T* __restrict__ K, const T* __restrict__ V, const T* __restrict__ dO,
    const float* __restrict__ lse, const float* __restrict__ delta, T* __restrict__ dK, T* __restrict__ dV,
    float* __restrict__ partial, const PackedTile* __restrict__ tiles, PackedDims dm) {
  typedef Shape<T, DP> S;
  typedef typename KeySide<T, DP>::LT LT;
  constexpr int WAVES = KeySide<T, DP>::WAVES;
  extern __shared__ __attribute__((aligned(1024))) char lds[];       // Q, dO, Q, dO, then 2 x (L, D)
  float* stats = reinterpret_cast<float*>(lds + 4 * LT::BYTES);
  const int kvh = blockIdx.x % dm.Hk;
  const PackedTile w = tiles[blockIdx.x / dm.Hk];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), half = lane >> 5;
  const int G = dm.by.G, rows = w.q_len * G, w_key = w.tile * 128 + 32 * (wave & 3), key = w_key + (lane & 31);
  const bool live = key < w.k_len;
  const long krow = (long)w.k_start + min(key, w.k_len - 1);
  // the first row that sees this key, the wave's first and last, the workgroup's first
  const int shift = dm.causal ? w.k_len - w.q_len : 0x40000000;
  const int first = !live ? 0x7fffffff : max(0, key - shift) * G;
  const int w_lo = w_key < w.k_len ? max(0, w_key - shift) * G : 0x7fffffff, w_hi = max(0, min(w_key + 31, w.k_len - 1) - shift) * G;
  const bool ragged = w_key + 31 >= w.k_len;
  const int b_lo = max(max(0, w.tile * 128 - shift) * G, w.row_lo);
  const int t0 = b_lo / S::KT, t1 = (min(rows, w.row_hi) + S::KT - 1) / S::KT;     // row_lo, row_hi: whole tiles

  const T* qb = Q + (long)w.q_start * dm.ldq + kvh * G * dm.hq;
  const T* gb = dO + (long)w.q_start * dm.ldo + kvh * G * dm.ho;
  const long lb = ((long)kvh * dm.q_rows + w.q_start) * G;
  auto fetch = [&](int t, int into) {
    const unsigned to = lds_address(lds) + into * 2 * LT::BYTES;
    const int r0 = t * S::KT, tok0 = divide(r0, dm.by);
    const ix4 qr = buffer_of(qb + tok0 * dm.ldq, 0x7ffffe00), gr = buffer_of(gb + tok0 * dm.ldo, 0x7ffffe00);
#pragma unroll
    for (int i = 0; i < LT::NI; ++i) {
      const int r = r0 + LT::row_of(i, wave, lane), tk = divide(r, dm.by), hd = r - tk * G, ch = LT::chunk_of(i, wave, lane) * 16;
      const bool ok = r < rows && ch < dm.D * (int)sizeof(T);
      load_to_lds(qr, to + (i * WAVES + wave) * 1024, ok ? (int)(((tk - tok0) * dm.ldq + hd * dm.hq) * (long)sizeof(T)) + ch : OUT_OF_BUFFER);
      load_to_lds(gr, to + LT::BYTES + (i * WAVES + wave) * 1024, ok ? (int)(((tk - tok0) * dm.ldo + hd * dm.ho) * (long)sizeof(T)) + ch : OUT_OF_BUFFER);
    }
  };
  float st_next = 0.0f;
  auto stat = [&](int t) {                                            // threads 0 .. 2 KT: L, then D of the tile's rows
    const int r = t * S::KT + (threadIdx.x & (S::KT - 1));
    st_next = 0.0f;
    if (threadIdx.x < 2 * S::KT && r < rows) st_next = (threadIdx.x < S::KT ? lse : delta)[lb + r];
  };
  const float c = dm.scale * LOG2E;
  const T* kp = K + krow * dm.ldk + kvh * dm.hk;
  const T* vp = V + krow * dm.ldv + kvh * dm.hv;
  const long orow = (krow * dm.Hk + kvh) * dm.D;
  float* slot = partial + (((long)w.slot * dm.Hk + kvh) * 256 + 32 * (wave & 3) + (lane & 31)) * dm.D;    // dK, then dV
  if (t0 < t1) {
    stat(t0);
    fetch(t0, t0 & 1);
  }
  // every wave goes through the same tiles and barriers, whichever of the sums are its own
  auto all_tiles = [&](auto& sums, auto dk_mine, auto dv_mine) {
    sums.begin(kp, vp, dm.D, live, half);
    for (int t = t0; t < t1; ++t) {
      const char* qt = lds + (t & 1) * 2 * LT::BYTES;
      float* sl = stats + (t & 1) * 2 * S::KT;
      wait_loads();
      if (threadIdx.x < 2 * S::KT) sl[threadIdx.x] = st_next;
      __syncthreads();
      if (t + 1 < t1) {
        stat(t + 1);
        fetch(t + 1, (t + 1) & 1);
      }
      const int r0 = t * S::KT;
      if (r0 + S::KT <= w_lo) continue;                              // none of these rows sees this wave's keys
      sums.step(qt, qt + LT::BYTES, sl, c, ragged || r0 < w_hi, first - r0, lane);
    }
    if constexpr (dk_mine.value) {
      if (w.slot < 0) store_rows<T, S::DB>(dK + orow, sums.dk, dm.scale, dm.D, half, live);
      else store_rows<T, S::DB>(slot, sums.dk, dm.scale, dm.D, half, live);
    }
    if constexpr (dv_mine.value) {
      if (w.slot < 0) store_rows<T, S::DB>(dV + orow, sums.dv, 1.0f, dm.D, half, live);
      else store_rows<T, S::DB>(slot + 128 * dm.D, sums.dv, 1.0f, dm.D, half, live);
    }
  };
  if constexpr (KeySide<T, DP>::SPLIT) {
    if (wave < 4) {
      KeySums<T, DP, true, false> sums;
      all_tiles(sums, std::false_type{}, std::true_type{});
    } else {
      KeySums<T, DP, false, true> sums;
      all_tiles(sums, std::true_type{}, std::false_type{});
    }
  } else {
    KeySums<T, DP, true, true> sums;
    all_tiles(sums, std::true_type{}, std::true_type{});
  }
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
template <typename T, int DP>
static int launch_fwd(const void* Q, const void* K, const void* V, void* out, float* lse, const PackedTile* tiles, int nt,
                      const PackedDims& dm, hipStream_t st) {
  const int bytes = 4 * Shape<T, DP>::LT::BYTES;
  static S2GLdsCap cap;
  const auto kernel = s2g_k_packed_attn_fwd<T, DP>;
  if (s2g_lds_cap(cap, reinterpret_cast<const void*>(kernel), bytes) != 0) return -2;
  hipLaunchKernelGGL(kernel, dim3((unsigned)nt * dm.Hk), dim3(256), bytes, st, (const T*)Q, (const T*)K, (const T*)V, (T*)out, lse, tiles, dm);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}
template <typename T, int DP>
static int launch_bwd(const void* Q, const void* K, const void* V, const void* out, const void* dO, const float* lse,
                      float* delta, void* dQ, void* dK, void* dV, float* partial, const PackedTile* qt, int nqt,
                      const PackedTile* kt, int nkt, const PackedTile* cut, int ncut, const PackedDims& dm, hipStream_t st) {
  typedef typename Shape<T, DP>::LT LT;
  const int qb = 4 * LT::BYTES, kb = 4 * LT::BYTES + 4 * Shape<T, DP>::KT * (int)sizeof(float);
  static S2GLdsCap qcap, kcap;
  const auto kq = s2g_k_packed_attn_bwd_q<T, DP>;
  const auto kk = s2g_k_packed_attn_bwd_kv<T, DP>;
  if (s2g_lds_cap(qcap, reinterpret_cast<const void*>(kq), qb) != 0 || s2g_lds_cap(kcap, reinterpret_cast<const void*>(kk), kb) != 0) return -2;
  if (nqt > 0)
    hipLaunchKernelGGL(kq, dim3((unsigned)nqt * dm.Hk), dim3(256), qb, st, (const T*)Q, (const T*)K, (const T*)V, (const T*)out,
                       (const T*)dO, lse, delta, (T*)dQ, qt, dm);
  if (nkt > 0)
    hipLaunchKernelGGL(kk, dim3((unsigned)nkt * dm.Hk), dim3(64 * KeySide<T, DP>::WAVES), kb, st, (const T*)Q, (const T*)K,
                       (const T*)V, (const T*)dO, lse, delta, (T*)dK, (T*)dV, partial, kt, dm);
  if (ncut > 0)
    hipLaunchKernelGGL(s2g_k_packed_attn_sum<T>, dim3((unsigned)ncut * dm.Hk, 8), dim3(256), 0, st, partial, (T*)dK, (T*)dV, cut, dm);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int PACKED_NAME(s2g_launch_packed_fwd)(const void* Q, const void* K, const void* V, void* out, float* lse,
                                                  const PackedTile* tiles, int nt, PackedDims dm, hipStream_t st) {
  return PER_DIM(launch_fwd, PACKED_T, Q, K, V, out, lse, tiles, nt, dm, st);
}
extern "C" int PACKED_NAME(s2g_launch_packed_bwd)(const void* Q, const void* K, const void* V, const void* out,
                                                  const void* dO, const float* lse, float* delta, void* dQ, void* dK,
                                                  void* dV, float* partial, const PackedTile* qt, int nqt,
                                                  const PackedTile* kt, int nkt, const PackedTile* cut, int ncut,
                                                  PackedDims dm, hipStream_t st) {
  return PER_DIM(launch_bwd, PACKED_T, Q, K, V, out, dO, lse, delta, dQ, dK, dV, partial, qt, nqt, kt, nkt, cut, ncut, dm, st);
}
