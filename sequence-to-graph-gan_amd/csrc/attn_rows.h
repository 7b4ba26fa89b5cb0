// What the packed and the paged attention kernels share: tile shapes, row loads and stores, the running softmax.
#pragma once
#include "frag.h"

// DP: the feature width the kernels are compiled for; rows in LDS are a power of two of 16-byte chunks, four at least
template <typename T, int DP>
struct Shape {
  static constexpr int PITCH = DP == 96 ? 128 : DP == 16 && sizeof(T) == 2 ? 32 : DP;
  static constexpr int KT = sizeof(T) == 2 || DP == 16 ? 64 : 32;      // keys (rows, in the key-side backward pass) per LDS tile
  static constexpr int KS = DP / 16, DB = (DP + 31) / 32, KB = KT / 32;
  static constexpr int AHEAD = 2;
  typedef Tile<T, PITCH, KT, 4> LT;
  typedef typename Vec<T>::v8 v8;
  // Sums over rows (keys) of 16 fp32 features: a 32 x 32 step would fill half of its result for nothing, so the same
  // operands go through v_mfma_f32_16x16x1_4b, four 16 x 16 products at once: columns 0 .. 15 and 16 .. 31 with the lower
  // half's contraction slots, and again with the upper half's, which whole() adds at the end.  (Training on 64 sequences up
  // to 512, 4 heads: 122 -> 102 us.)
  static constexpr bool NARROW = sizeof(T) == 4 && DP == 16;
  static __device__ __forceinline__ fx16 sum(const v8& a, const v8& b, fx16 c) {
    if constexpr (NARROW) {
#pragma unroll
      for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x1f32(a[j], b[j], c, 0, 0, 0);
      return c;
    } else {
      return mma(a, b, c);
    }
  }
  // Register i of lane l: column l % 16 of block i / 4, feature 4 (l / 16) + i % 4; made the 32 x 32 result it stands for
  static __device__ __forceinline__ void whole(fx16* c, int lane) {
    if constexpr (NARROW) {
      fx16 r = zero16();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int from = (lane & 15) + 16 * (2 * (i >> 2) + (lane >> 5)), j = i & 3;
        const float x = __shfl(c[0][j] + c[0][8 + j], from), y = __shfl(c[0][4 + j] + c[0][12 + j], from);
        r[i] = lane & 16 ? y : x;
      }
      c[0] = r;
    }
  }
  // sums times a factor of every column (lane l: column l % 32)
  static __device__ __forceinline__ void scaled(fx16* c, float f, int lane) {
    const float x = NARROW ? __shfl(f, lane & 15) : f, y = NARROW ? __shfl(f, 16 + (lane & 15)) : f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) c[d][i] *= i & 4 ? y : x;
  }
};

// Offsets of this lane's chunks of a tile whose rows lie `ld` elements apart, and the buffer over the tile's rows
template <typename LT, typename T>
__device__ __forceinline__ void tile_offsets(int* off, long ld, int D, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < LT::NI; ++i) {
    const int c = LT::chunk_of(i, wave, lane);
    off[i] = c * 16 < D * (int)sizeof(T) ? (int)(LT::row_of(i, wave, lane) * ld * (long)sizeof(T)) + c * 16 : OUT_OF_BUFFER;
  }
}
template <typename LT, typename T, int WAVES = 4>
__device__ __forceinline__ void fetch_rows(char* lds, const T* p, long ld, int D, int rows, const int* off, int wave) {
  const ix4 b = buffer_of(p, rows > 0 ? (int)(((rows - 1) * ld + D) * (long)sizeof(T)) : 0);
  const unsigned to = lds_address(lds);
#pragma unroll
  for (int i = 0; i < LT::NI; ++i) load_to_lds(b, to + (i * WAVES + wave) * 1024, off[i]);
}

// 8 elements of a row straight from memory: zeros beyond the row's D elements or where !ok.  The loads are unconditional (of
// the row's beginning where there is nothing to load; the row itself always exists), so that many are on their way at once.
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 row8(const T* p, int at, int D, bool ok) {
  typename Vec<T>::v8 r;
  if constexpr (sizeof(T) == 2) {
    r = load8(p + (at < D ? at : 0));
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = ok && at < D ? r[j] : (T)0.0f;
  } else {                                          // fp32 rows come in fours
    const fx4 a = *reinterpret_cast<const fx4*>(p + (at < D ? at : 0)), b = *reinterpret_cast<const fx4*>(p + (at + 4 < D ? at + 4 : 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      r[j] = ok && at < D ? a[j] : 0.0f;
      r[j + 4] = ok && at + 4 < D ? b[j] : 0.0f;
    }
  }
  return r;
}

// writes a transposed result (lane = row, registers = features) times f
template <typename T, int DB, typename U>
__device__ __forceinline__ void store_rows(U* p, const fx16* acc, float f, int D, int half, bool ok) {
  if (!ok) return;
#pragma unroll
  for (int d = 0; d < DB; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = 32 * d + 8 * g + 4 * half;
      if (at < D) {
        typename Vec<U>::v4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (U)(acc[d][4 * g + j] * f);
        *reinterpret_cast<typename Vec<U>::v4*>(p + at) = v;
      }
    }
}

// Infinities and NaN.  A product takes 0 x NaN for NaN, so a tile that holds one, and a row (key) that does not see it, cannot
// go through the matrix unit together.  Where a tile with hidden pairs holds one, a wave makes its 32 rows (keys) anew: pair
// by pair, straight from memory, 16 features at a time, and only the pairs that see each other: all of their pairs, those of clean
// tiles too.  That is slow (8 bf16 sequences up to 4096, 16 / 4 heads of 128: the gradient 0.8 -> 97 ms for one infinity in dO and
// 242 for all of it, the forward pass 0.2 -> 52 for one value in a hundred tokens; 96 fp16 ones up to 203, 12 heads of 64: 0.06 -> 2.4
// and 3.3).  Functions of their own, never inlined: their registers would be the main loops' (packed attention, query side of the
// gradient: 297 -> 330 us).
template <typename T, int N>
__device__ __forceinline__ float slow_dot(const T* a, const T* b, int D, int half) {
  float s = 0.0f;
#pragma unroll 1
  for (int i = 0; i < N; ++i) s = dot8(row8(a, 16 * i + 8 * half, D, true), row8(b, 16 * i + 8 * half, D, true), s);
  return both_sum(s);
}
template <typename T>
__device__ __forceinline__ void slow_add(float* acc, float f, const T* p, int from, int D) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int at = from + 4 * g;
    const typename Vec<T>::v4 x = *reinterpret_cast<const typename Vec<T>::v4*>(p + (at < D ? at : 0));
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[4 * g + j] = fmaf(f, (float)x[j], acc[4 * g + j]);
  }
}
template <typename T>
__device__ __forceinline__ void slow_store(T* p, const float* acc, float f, int from, int D, bool ok) {
#pragma unroll
  for (int j = 0; j < 16; ++j)
    if (ok && from + j < D) p[from + j] = (T)(acc[j] * f);
}

// fp16 weights below 2^-14 lose bits, and a long row's weights are that small: there all of them are taken 2^RAISE times
// as large (the sums alike, so it cancels), as much as the largest term, 2^SLACK, leaves room for.
template <typename T> struct Weights { static constexpr float RAISE = 0.0f, SLACK = 8.0f; };
template <> struct Weights<_Float16> { static constexpr float RAISE = 11.0f, SLACK = 4.0f; };

// The running softmax of 32 rows of one wave: lane l holds row l % 32 (both halves of the wave; each its own keys).
// TRAIN: bf16 rows whose sums go into the backward pass.  O is divided by the sum of the rounded weights, whose errors cancel
// those of a row's few large ones; the weights of the backward pass are not rounded, and by that sum they would be off by half a
// step all alike: the sum of the weights as they were is kept beside it (8 sequences up to 4096, 16 / 4 heads of 128: 229 -> 239 us;
// of 64: 128 -> 135).
template <typename T, int DP, bool TRAIN = false>
struct Rows {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  typedef typename Vec<T>::v8 v8;
  v8 q[S::KS];
  fx16 o[S::DB];
  float m, l, c, slack;
  float whole;               // TRAIN: the sum of the weights before they are rounded
  bool tainted;              // a tile with hidden keys held an infinity or a NaN in V: o is not to be used (slow_out, slow_pages)

  __device__ __forceinline__ void begin(const T* qp, int D, bool live, int half, float scale) {
#pragma unroll
    for (int s = 0; s < S::KS; ++s) q[s] = row8(qp, 16 * s + 8 * half, D, live);
#pragma unroll
    for (int d = 0; d < S::DB; ++d) o[d] = zero16();
    m = -INFINITY, l = 0.0f, whole = 0.0f, c = scale * LOG2E, slack = Weights<T>::SLACK / c, tainted = false;
  }
  // S^T = K Q^T of KB blocks of 32 keys: a lane holds one row's scores, so a row's maximum and sum are taken over a lane's
  // own registers and one exchange between the halves
  template <int KB, typename F>
  __device__ __forceinline__ void scores(fx16* st, const char* kt, int lane, F beside) const {
#pragma unroll
    for (int b = 0; b < KB; ++b) st[b] = zero16();
    products<T, KB * S::KS, S::AHEAD>([&](int i) { return LT::along(kt, (lane & 31) + 32 * (i / S::KS), i % S::KS, lane >> 5); },
                            [&](int i, const v8& a) { st[i / S::KS] = mma(a, q[i % S::KS], st[i / S::KS]); }, beside);
  }
  // Scores st into sums.  edge: some row of the wave does not see all of the keys (`last`: the last one that this lane's
  // row sees, counted from the tile's first); absent: keys (bits) that are not there.  NEXT: the scores of the next tile,
  // kt, are made meanwhile, so that the matrix unit has work while this tile's 2^x are taken.
  // The matrix unit takes 16-bit weights, and rounding them to those costs the result as much as its own rounding does: errors of
  // 2.0e-3 for 1.6e-3 (bf16).  WHOLE: products of what rounding left as well, for kernels in which the unit is idle (single tokens
  // over a paged cache: 64 sequences of 300 to 8200, 8 heads of 128, 215 -> 216 us; 2 of 131071 and 90001, 2 of 96, 36.8 -> 37.7;
  // 64 of 8000, 8 of 16, 92 -> 94); where it is the bound (prompts, chunks, training) they would be a third product beside two.
  template <int KB, bool NEXT, bool WHOLE = false>
  __device__ __forceinline__ void add(fx16* st, fx16* next, const char* kt, const char* vt, bool edge, int last,
                                      unsigned long long absent, int lane) {
    const int half = lane >> 5;
    if (edge) {
      tainted = tainted || not_finite<T>(vt, 32 * KB * S::PITCH * (int)sizeof(T), lane);
      const int at = hidden(last - 4 * half);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + reg_row(i) > at) st[b][i] = -INFINITY;
    }
    if (absent) {
#pragma unroll
      for (int b = 0; b < KB; ++b) {
        const unsigned bits = (unsigned)(absent >> (32 * b)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((bits >> reg_row(i)) & 1) st[b][i] = -INFINITY;
      }
    }
    float mx = st[0][0];
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[b][i]);
    mx = both_max(mx);
    // the sums are rescaled only where a row's maximum has grown by a factor of 2^SLACK: until then its terms stay below
    // that and nothing is lost, every term being rounded relative to its own size
    if (__any(mx > m + slack)) {
      const float mn = fmaxf(m, mx), a = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= a;
      if constexpr (TRAIN) whole *= a;
      S::scaled(o, a, lane);
    }
    const float low = base();
    constexpr bool LEFT = WHOLE && sizeof(T) == 2;
    v8 p[2 * KB], left[LEFT ? 2 * KB : 1];
    const auto weigh = [&](int e) {                      // two weights; four pairs make an operand
      const int b = e >> 3, i = 2 * (e & 7);
      st[b][i] = __builtin_amdgcn_exp2f(fmaf(st[b][i], c, -low));
      st[b][i + 1] = __builtin_amdgcn_exp2f(fmaf(st[b][i + 1], c, -low));
      p[e >> 2][i & 7] = (T)st[b][i];
      p[e >> 2][(i & 7) + 1] = (T)st[b][i + 1];
      if constexpr (LEFT) {
        left[e >> 2][i & 7] = (T)(st[b][i] - (float)p[e >> 2][i & 7]);
        left[e >> 2][(i & 7) + 1] = (T)(st[b][i + 1] - (float)p[e >> 2][(i & 7) + 1]);
        l += st[b][i] + st[b][i + 1];
      } else {
        l = add_two(l, p[e >> 2], st[b], i);
        if constexpr (TRAIN) whole += st[b][i] + st[b][i + 1];
      }
    };
    constexpr int PAIRS = 8 * KB, N = KB * S::KS;
    if constexpr (NEXT) {
      scores<KB>(next, kt, lane, [&](int i) {
#pragma unroll
        for (int e = i * PAIRS / N; e < (i + 1) * PAIRS / N; ++e) weigh(e);
      });
    } else {
#pragma unroll
      for (int e = 0; e < PAIRS; ++e) weigh(e);
    }
    // O^T += V^T P^T, the weights straight from the registers they are in
    products<T, 2 * KB * S::DB, S::AHEAD>([&](int i) { return LT::across(vt, i % S::DB, i / S::DB, lane); },
                                [&](int i, const v8& a) {
                                  o[i % S::DB] = S::sum(a, p[i / S::DB], o[i % S::DB]);
                                  if constexpr (LEFT) o[i % S::DB] = S::sum(a, left[i / S::DB], o[i % S::DB]);
                                }, [](int) {});
  }
  template <int KB, bool WHOLE = false>
  __device__ __forceinline__ void step(const char* kt, const char* vt, bool edge, int last, unsigned long long absent, int lane) {
    fx16 st[KB];
    scores<KB>(st, kt, lane, [](int) {});
    add<KB, false, WHOLE>(st, nullptr, nullptr, vt, edge, last, absent, lane);
  }
  // what weigh() takes from a score (times c) to make a weight
  __device__ __forceinline__ float base() const { return (m == -INFINITY ? 0.0f : m * c) - Weights<T>::RAISE; }
  // log2 of the row's sum of exponentials, given the sum over both halves
  __device__ __forceinline__ float log_sum(float sum) const { return fmaf(m, c, __builtin_amdgcn_logf(sum)) - Weights<T>::RAISE; }

 private:
  // a row's sum is that of the rounded weights, as its products take them, where one instruction (v_dot2) does it
  static __device__ __forceinline__ float add_two(float l, bx8 p, const fx16&, int i) {
    typedef __bf16 bx2 __attribute__((ext_vector_type(2)));
    const bx2 one = {(__bf16)1.0f, (__bf16)1.0f}, two = {p[i & 7], p[(i & 7) + 1]};
    return __builtin_amdgcn_fdot2_f32_bf16(two, one, l, false);
  }
  static __device__ __forceinline__ float add_two(float l, hx8, const fx16& st, int i) { return l + st[i] + st[i + 1]; }
  static __device__ __forceinline__ float add_two(float l, fx8, const fx16& st, int i) { return l + st[i] + st[i + 1]; }
};

// A wave's own tiles of 32 keys (K and V, twice), and what joins the waves of a workgroup.  Four waves' rows of 512 bytes leave
// room for one tile of each only, which is filled again as it has been read (ONCE): two waves with two tiles of each leave half
// the matrix units idle (one fp32 token of 32 sequences of 4000, 32 / 8 heads of 128: 379 -> 268 us).
template <typename T, int DP>
struct WaveTiles {
  typedef Shape<T, DP> S;
  static constexpr int KEYS = 32, KB = KEYS / 32, NW = 4;
  typedef Tile<T, S::PITCH, KEYS, 1> LT;
  static constexpr bool ONCE = 4 * NW * LT::BYTES > 131072;
  static constexpr int PAD = 32 * S::DB + 4;                   // floats of a row of sums
  static constexpr int TILES = (ONCE ? 2 : 4) * NW * LT::BYTES, JOIN = NW * (96 + 32 * PAD) * (int)sizeof(float);
  static constexpr int BYTES = TILES > JOIN ? TILES : JOIN;
};
template <typename T>
__device__ __forceinline__ void put4(T* p, const fx4& a) {
  typename Vec<T>::v4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = (T)a[i];
  *reinterpret_cast<typename Vec<T>::v4*>(p) = v;
}
// 32 rows' sums of every wave (float [wave][row][PAD] in LDS) added; store(row, feature, four of them)
template <typename W, typename Store>
__device__ __forceinline__ void add_waves(const float* os, int rows, int D, Store store) {
  const int n4 = D >> 2, count = rows * n4;
  for (int e = threadIdx.x; e < count; e += 64 * W::NW) {
    const int y = e / n4, d = (e - y * n4) * 4;
    fx4 a = *reinterpret_cast<const fx4*>(os + y * W::PAD + d);
#pragma unroll
    for (int w = 1; w < W::NW; ++w) {
      const fx4 b = *reinterpret_cast<const fx4*>(os + (w * 32 + y) * W::PAD + d);
      a[0] += b[0]; a[1] += b[1]; a[2] += b[2]; a[3] += b[3];
    }
    store(y, d, a);
  }
}
// The running softmaxes of 32 rows, each wave's over its own keys, joined: maxima and sums through LDS, then O scaled to the
// common maximum (and by its sum if `divided`).  slow(f, to): a wave's O times f made anew; statistics(m, sum): of this lane's row
// (TRAIN: of its weights before they are rounded).
template <typename W, typename T, int DP, bool TRAIN, typename Slow, typename Statistics, typename Store>
__device__ __forceinline__ void join_waves(char* lds, Rows<T, DP, TRAIN>& r, int rows, bool divided, int D, int wave, int lane, Slow slow,
                                           Statistics statistics, Store store) {
  constexpr int N = TRAIN ? 3 : 2;
  const int half = lane >> 5;
  float* ml = reinterpret_cast<float*>(lds);                   // [wave][row] (m, l, TRAIN: whole)
  const float l = both_sum(r.l), all = TRAIN ? both_sum(r.whole) : 0.0f;
  Shape<T, DP>::whole(r.o, lane);
  __syncthreads();
  if (half == 0) {
    ml[(wave * 32 + lane) * N] = r.m;
    ml[(wave * 32 + lane) * N + 1] = l;
    if (TRAIN) ml[(wave * 32 + lane) * N + 2] = all;
  }
  __syncthreads();
  float m = -INFINITY, sum = 0.0f, whole = 0.0f;
#pragma unroll
  for (int w = 0; w < W::NW; ++w) m = fmaxf(m, ml[(w * 32 + (lane & 31)) * N]);
#pragma unroll
  for (int w = 0; w < W::NW; ++w) {
    const float mw = ml[(w * 32 + (lane & 31)) * N], f = mw == m ? 1.0f : __builtin_amdgcn_exp2f((mw - m) * r.c);
    sum += ml[(w * 32 + (lane & 31)) * N + 1] * f;
    if (TRAIN) whole += ml[(w * 32 + (lane & 31)) * N + 2] * f;
  }
  const float f = r.m == m ? 1.0f : __builtin_amdgcn_exp2f((r.m - m) * r.c), scaled = divided ? (sum == 0.0f ? 0.0f : f / sum) : f;
  float* os = ml + W::NW * 32 * N;
  float* mine = os + (wave * 32 + (lane & 31)) * W::PAD;
  if (r.tainted) slow(scaled, mine);
  else store_rows<T, Shape<T, DP>::DB>(mine, r.o, scaled, 32 * Shape<T, DP>::DB, half, true);
  if (wave == 0 && half == 0) statistics(m, TRAIN ? whole : sum);
  __syncthreads();
  add_waves<W>(os, rows, D, store);
}
