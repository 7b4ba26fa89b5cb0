// Rotary positions: pair i of a head's first R features is turned by the angle t_i = position * frequency_i,
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),
// the pairs lying side by side (2i, 2i + 1) or in halves (i, i + R / 2); features R .. D pass through.  The gradient is
// the turn by -t.  One launch turns q and k, or, for a paged cache, turns q, writes turned k and plain v into their pages.
//
// Bound by memory: every element once in, once out.  16383 bf16 tokens, 32 + 8 heads of 128: 69.6 us, 4.8 TB/s, as a copy;
// 4451 such tokens into pages of 64: 21 us; 32768 fp32 tokens of 4 + 4 heads of 16: 10.3 us; one token of 48 sequences into
// the cache: 4 us, a launch.  A token's R / 2 angles serve all its heads, so a workgroup first
// makes them for its tokens, one per thread, and leaves cos and sin in LDS; a thread then keeps those of one 16-byte
// unit in registers and walks over heads with 16-byte loads and stores.  The angle is a product in 64 bits, reduced to
// an eighth of a turn before it is rounded to 32: at position 10^6 a 32-bit angle would be off by 0.03 radians.
#include "attn_rows.h"
#include "packed_attention.h"
#include "paged_attention.h"
#include "rotary.h"

// cos and sin of 2 pi x
__device__ __forceinline__ float2 turn_cos_sin(double x) {
  x -= rint(x);
  const double k = rint(4.0 * x);
  const float r = (float)(2.0 * x - 0.5 * k);              // in half turns, |r| <= 1/4
  float s, c;
  sincospif(r, &s, &c);
  switch ((int)k & 3) {
    case 1: return make_float2(-s, c);
    case 2: return make_float2(-c, -s);
    case 3: return make_float2(s, -c);
  }
  return make_float2(c, s);
}

template <typename T, int N>
struct Unit {
  typedef T type __attribute__((ext_vector_type(N)));
};
template <typename T>
struct Unit<T, 1> {
  typedef T type;
};
template <typename T, int N>
__device__ __forceinline__ void get(float* x, const T* p) {
  const typename Unit<T, N>::type v = *reinterpret_cast<const typename Unit<T, N>::type*>(p);
  if constexpr (N == 1) x[0] = (float)v;
  else
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = (float)v[i];
}
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float* x) {
  typename Unit<T, N>::type v;
  if constexpr (N == 1) v = (T)x[0];
  else
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (T)x[i];
  *reinterpret_cast<typename Unit<T, N>::type*>(p) = v;
}

// N features per unit: 16 bytes where sizes, strides and addresses allow it, else 1 (a pair, side by side)
template <typename T, int N, bool INTER, bool PAGED>
__global__ __launch_bounds__(256) void s2g_k_rotary(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                    const int* __restrict__ positions, const double* __restrict__ freq,
                                                    const int* __restrict__ table, const int* __restrict__ lens,
                                                    const int* __restrict__ starts, T* __restrict__ qo, T* __restrict__ ko,
                                                    T* __restrict__ vo, RotaryDims dm) {
  extern __shared__ float2 cs[];                           // [tokens of the workgroup][R / 2]
  const int P = dm.R >> 1, tid = threadIdx.x;
  int count, row0, pos0 = 0, len = 0;
  if constexpr (PAGED) {
    const int s = blockIdx.y, a = min(max(starts[s], 0), (int)dm.rows), b = min(max(starts[s + 1], a), (int)dm.rows);
    const int n = min(b - a, dm.max_new), t = blockIdx.x * dm.tokens;
    if (t >= n) return;
    const int all = min(max(lens[s], 0), 1 << 30);
    len = (int)min((long)all, (long)dm.cols << dm.page_shift);            // positions from there on have no page
    count = min(dm.tokens, n - t);
    row0 = a + t;
    pos0 = all - (b - a) + t;
    table += (long)s * dm.cols;
  } else {
    const long first = (long)blockIdx.x * dm.tokens;
    row0 = (int)first;
    count = (int)min((long)dm.tokens, dm.rows - first);
  }
  for (int e = tid; e < count * P; e += 256) {
    const int t = e / P, i = e - t * P;
    const int pos = PAGED ? pos0 + t : positions[row0 + t];
    const float2 y = turn_cos_sin((double)pos * freq[i] * 0.15915494309189533577);
    cs[e] = make_float2(y.x * dm.multiplier, y.y * dm.multiplier * dm.sign);
  }
  __syncthreads();
  const int per = 256 / dm.tokens, t = tid / per, at = tid - t * per;
  if (t >= count) return;
  constexpr int W = INTER && N == 1 ? 2 : N;               // features of a turning unit's first part
  const int turning = INTER ? dm.R / W : P / N, units = turning + (dm.D - dm.R) / N;
  const int u = at % units, lanes = per / units;
  if (at >= lanes * units) return;
  const long row = row0 + t;
  float c[N], s[N];
  constexpr int PAIRS = INTER ? W / 2 : N;
  const bool turns = u < turning;
  if (turns)
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const float2 y = cs[t * P + u * PAIRS + i];
      c[i] = y.x;
      s[i] = y.y;
    }
  T* kt = nullptr;
  T* vt = nullptr;
  if constexpr (PAGED) {
    const int pos = pos0 + t;
    if (pos >= 0 && pos < len) {
      const int page = table[pos >> dm.page_shift];
      if ((unsigned)page < (unsigned)dm.pages) {
        const long o = page * dm.page_ld + (pos & ((1 << dm.page_shift) - 1)) * dm.ld;
        kt = ko + o;
        vt = vo + o;
      }
    }
  } else {
    kt = ko ? ko + row * dm.Hk * dm.D : nullptr;
  }
  const long ohd = PAGED ? dm.hd : dm.D;
  for (int h = at / units; h < dm.H + (kt ? dm.Hk : 0); h += lanes) {
    const T* in = h < dm.H ? q + row * dm.ldq + h * dm.hq : k + row * dm.ldk + (h - dm.H) * dm.hk;
    T* out = h < dm.H ? qo + (row * dm.H + h) * dm.D : kt + (h - dm.H) * ohd;
    if (!turns) {
      const int f = dm.R + (u - turning) * N;
      float x[N];
      get<T, N>(x, in + f);
      put<T, N>(out + f, x);
    } else if constexpr (INTER) {
      float x[W], y[W];
      if constexpr (N == 1) {                              // a pair may not be aligned as a pair
        x[0] = (float)in[2 * u];
        x[1] = (float)in[2 * u + 1];
      } else {
        get<T, W>(x, in + u * W);
      }
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        y[2 * i] = x[2 * i] * c[i] - x[2 * i + 1] * s[i];
        y[2 * i + 1] = x[2 * i] * s[i] + x[2 * i + 1] * c[i];
      }
      if constexpr (N == 1) {
        out[2 * u] = (T)y[0];
        out[2 * u + 1] = (T)y[1];
      } else {
        put<T, W>(out + u * W, y);
      }
    } else {
      float a[N], b[N], y[N], z[N];
      get<T, N>(a, in + u * N);
      get<T, N>(b, in + P + u * N);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        y[i] = a[i] * c[i] - b[i] * s[i];
        z[i] = a[i] * s[i] + b[i] * c[i];
      }
      put<T, N>(out + u * N, y);
      put<T, N>(out + P + u * N, z);
    }
  }
  if constexpr (PAGED) {
    if (vt)
      for (int h = at / units; h < dm.Hk; h += lanes)
        for (int f = u; f < dm.D / N; f += units) {
          float x[N];
          get<T, N>(x, v + row * dm.ldv + h * dm.hv + f * N);
          put<T, N>(vt + h * dm.hd + f * N, x);
        }
  }
}

template <typename T, int N, bool INTER, bool PAGED>
static int launch_rotary(const void* q, const void* k, const void* v, const int* positions, const double* freq,
                         const int* table, const int* lens, const int* starts, void* qo, void* ko, void* vo, RotaryDims dm,
                         hipStream_t st) {
  constexpr int W = INTER && N == 1 ? 2 : N;
  const int units = (INTER ? dm.R / W : dm.R / 2 / N) + (dm.D - dm.R) / N;
  const long most = PAGED ? dm.max_new : dm.rows, groups = PAGED ? dm.n : 1;
  // tokens per workgroup: as many as leave every token a lane per unit, and two workgroups to every compute unit
  dm.tokens = 1;
  while (dm.tokens < 8 && units * dm.tokens * 2 <= 256 && groups * ((most + 2 * dm.tokens - 1) / (2 * dm.tokens)) >= 512) dm.tokens *= 2;
  const dim3 grid((unsigned)((most + dm.tokens - 1) / dm.tokens), (unsigned)groups);
  hipLaunchKernelGGL((s2g_k_rotary<T, N, INTER, PAGED>), grid, dim3(256), dm.tokens * (dm.R / 2) * sizeof(float2), st,
                     (const T*)q, (const T*)k, (const T*)v, positions, freq, table, lens, starts, (T*)qo, (T*)ko, (T*)vo, dm);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

extern "C" int s2g_launch_rotary(int type, const void* q, const void* k, const void* v, const int* positions,
                                 const double* freq, const int* table, const int* lens, const int* starts, void* qo, void* ko,
                                 void* vo, int wide, RotaryDims dm, hipStream_t st) {
#define ROTARY(T, N)                                                                                                           \
  (dm.interleaved ? (table ? launch_rotary<T, N, true, true>(q, k, v, positions, freq, table, lens, starts, qo, ko, vo, dm, st)  \
                           : launch_rotary<T, N, true, false>(q, k, v, positions, freq, table, lens, starts, qo, ko, vo, dm, st)) \
                  : (table ? launch_rotary<T, N, false, true>(q, k, v, positions, freq, table, lens, starts, qo, ko, vo, dm, st) \
                           : launch_rotary<T, N, false, false>(q, k, v, positions, freq, table, lens, starts, qo, ko, vo, dm, st)))
  switch (type) {
    case 0: return wide ? ROTARY(float, 4) : ROTARY(float, 1);
    case 1: return wide ? ROTARY(__bf16, 8) : ROTARY(__bf16, 1);
    case 2: return wide ? ROTARY(_Float16, 8) : ROTARY(_Float16, 1);
  }
  return -1;
}
