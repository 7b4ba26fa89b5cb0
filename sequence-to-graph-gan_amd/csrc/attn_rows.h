// What the packed and the paged attention kernels share: tile shapes, row loads and stores, the running softmax.
#pragma once
#include "frag.h"

template <typename T, int DP>
struct Shape {
  static constexpr int PITCH = DP == 96 ? 128 : DP;
  static constexpr int KT = sizeof(T) == 2 ? 64 : 32;        // keys (rows, in the key-side backward pass) per LDS tile
  static constexpr int KS = DP / 16, DB = DP / 32, KB = KT / 32;
  typedef Tile<T, PITCH, KT, 4> LT;
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
template <typename LT, typename T>
__device__ __forceinline__ void fetch_rows(char* lds, const T* p, long ld, int D, int rows, const int* off, int wave) {
  const ix4 b = buffer_of(p, (int)(((rows - 1) * ld + D) * (long)sizeof(T)));
  const unsigned to = lds_address(lds);
#pragma unroll
  for (int i = 0; i < LT::NI; ++i) load_to_lds(b, to + (i * 4 + wave) * 1024, off[i]);
}

// 8 elements of a row straight from memory: zeros beyond the row's D elements or where !ok
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 row8(const T* p, int at, int D, bool ok) {
  if (sizeof(T) == 2 || at + 8 <= D) return ok && at < D ? load8(p + at) : zero8<T>();
  typename Vec<T>::v8 r = zero8<T>();              // fp32 rows come in fours
  if (ok && at < D) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = p[at + j];
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

// The running softmax of 32 rows of one wave: lane l holds row l % 32 (both halves of the wave; each its own keys).
template <typename T, int DP>
struct Rows {
  typedef Shape<T, DP> S;
  typedef typename S::LT LT;
  typename Vec<T>::v8 q[S::KS];
  fx16 o[S::DB];
  float m, l, c, slack;

  __device__ __forceinline__ void begin(const T* qp, int D, bool live, int half, float scale) {
#pragma unroll
    for (int s = 0; s < S::KS; ++s) q[s] = row8(qp, 16 * s + 8 * half, D, live);
#pragma unroll
    for (int d = 0; d < S::DB; ++d) o[d] = zero16();
    m = -INFINITY, l = 0.0f, c = scale * LOG2E, slack = 8.0f / c;
  }
  // KB blocks of 32 keys from LDS.  edge: some row of the wave does not see all of them (`last`: the last one that this
  // lane's row sees, counted from the tile's first); absent: keys (bits) that are not there.
  template <int KB>
  __device__ __forceinline__ void step(const char* kt, const char* vt, bool edge, int last, unsigned long long absent, int lane) {
    const int half = lane >> 5;
    // S^T = K Q^T: a lane holds one row's scores, so a row's maximum and sum are taken over a lane's own registers and
    // one exchange between the halves
    fx16 st[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      st[b] = zero16();
#pragma unroll
      for (int s = 0; s < S::KS; ++s) st[b] = mma(LT::along(kt, 32 * b + (lane & 31), s, half), q[s], st[b]);
    }
    if (edge) {
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + reg_row(i) + 4 * half > last) st[b][i] = -INFINITY;
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
    // the sums are rescaled only where a row's maximum has grown by a factor of 2^8: until then its terms stay below
    // 2^8 and nothing is lost, every term being rounded relative to its own size
    if (__any(mx > m + slack)) {
      const float mn = fmaxf(m, mx), a = m == mn ? 1.0f : __builtin_amdgcn_exp2f((m - mn) * c);
      m = mn;
      l *= a;
#pragma unroll
      for (int d = 0; d < S::DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] *= a;
    }
    const float base = m == -INFINITY ? 0.0f : m * c;
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        st[b][i] = __builtin_amdgcn_exp2f(fmaf(st[b][i], c, -base));
        l += st[b][i];
      }
    // O^T += V^T P^T, the weights (rounded to the inputs' type) straight from the registers they are in
#pragma unroll
    for (int s = 0; s < 2 * KB; ++s) {
      const typename Vec<T>::v8 p = operand<T>(st[s >> 1], s & 1);
#pragma unroll
      for (int d = 0; d < S::DB; ++d) o[d] = mma(LT::across(vt, d, s, lane), p, o[d]);
    }
  }
};
