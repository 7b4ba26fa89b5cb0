// Matrix fragments shared by the packed and the paged attention kernels: element types, the 32 x 32 x 16 matrix step,
// tiles in LDS and the direct loads that fill them.
//
// One matrix step multiplies a 32 x 16 by a 16 x 32 operand; lane l holds 8 elements of row (column) l % 32, the
// contraction slots 8 (l / 32) .. + 7.  bf16 and fp16 use one v_mfma_f32_32x32x16; fp32 stays exact in eight
// v_mfma_f32_32x32x2_f32, the j-th taking every lane's element j, so one body serves all three types.  The 16 result
// registers of lane l are column l % 32, rows (i & 3) + 8 (i >> 2) + 4 (l / 32).
//
// A result can therefore be the next product's operand without leaving its registers: eight of its registers ARE
// eight contraction slots, standing for rows 4 half + {0..3, 8..11} of a 16-row step, as long as the other operand is
// read in that same order (Tile::across).
#pragma once
#include "s2g_common.h"
#include <type_traits>

typedef float fx16 __attribute__((ext_vector_type(16)));
typedef float fx8 __attribute__((ext_vector_type(8)));
typedef float fx4 __attribute__((ext_vector_type(4)));
typedef _Float16 hx8 __attribute__((ext_vector_type(8)));
typedef _Float16 hx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bx8 __attribute__((ext_vector_type(8)));
typedef __bf16 bx4 __attribute__((ext_vector_type(4)));
typedef short sx4 __attribute__((ext_vector_type(4)));
typedef int ix4 __attribute__((ext_vector_type(4)));

#define LOG2E 1.4426950408889634f

template <typename T> struct Vec;
template <> struct Vec<float> { typedef fx8 v8; typedef fx4 v4; };
template <> struct Vec<_Float16> { typedef hx8 v8; typedef hx4 v4; };
template <> struct Vec<__bf16> { typedef bx8 v8; typedef bx4 v4; };

__device__ __forceinline__ fx16 mma(bx8 a, bx8 b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ fx16 mma(hx8 a, hx8 b, fx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ fx16 mma(fx8 a, fx8 b, fx16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// registers 8 s .. 8 s + 7 of a result as the operand of the next product (rounded to nearest for 16-bit types)
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 operand(const fx16& c, int s) {
  typename Vec<T>::v8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)c[8 * s + j];
  return r;
}

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 zero8() {
  typename Vec<T>::v8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (T)0.0f;
  return r;
}

template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 load8(const T* p) {      // 16-byte aligned
  return *reinterpret_cast<const typename Vec<T>::v8*>(p);
}
template <>
__device__ __forceinline__ fx8 load8<float>(const float* p) {
  const fx4 a = *reinterpret_cast<const fx4*>(p), b = *reinterpret_cast<const fx4*>(p + 4);
  return (fx8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

__device__ __forceinline__ fx16 zero16() {
  fx16 r;
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = 0.0f;
  return r;
}
// the result row of register i
__device__ __forceinline__ constexpr int reg_row(int i) { return (i & 3) + 8 * (i >> 2); }

// x, of which the compiler knows nothing: comparing it with constants stays that (it would rather move x to the constants'
// side and keep the 32 sums in registers throughout a loop)
__device__ __forceinline__ int hidden(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// a value of this lane and of lane ^ 32: v_permlane32_swap leaves the lower half's in one register, the upper half's in
// the other
struct Halves {
  float lo, hi;
};
__device__ __forceinline__ Halves halves(float x) {
  const unsigned u = __builtin_bit_cast(unsigned, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned lo = r[0], hi = r[1];          // (a bit cast of a vector's element takes the vector's first)
  return {__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)};
}
__device__ __forceinline__ float both_max(float x) {
  const Halves h = halves(x);
  return fmaxf(h.lo, h.hi);
}
__device__ __forceinline__ float both_sum(float x) {
  const Halves h = halves(x);
  return h.lo + h.hi;
}

// r / G for 0 <= r < 2^31 with magic = ceil(2^32 / G) (G >= 2): the product overshoots by at most one
struct DivBy {
  int G;
  unsigned magic;
};
__host__ __device__ inline DivBy div_by(int G) { return {G, G > 1 ? (unsigned)((0x100000000ull + G - 1) / G) : 0u}; }
__device__ __forceinline__ int divide(int r, DivBy d) {
  if (d.G == 1) return r;
  int q = (int)__umulhi((unsigned)r, d.magic);
  if (q * (long)d.G > r) --q;
  return q;
}

// A tile of ROWS rows of PITCH elements in LDS, filled by buffer_load ... lds of 16 bytes per lane.  One wave instruction
// fills 1 KB of consecutive LDS, so the layout is [row][chunk of 16 bytes] without padding, and bank conflicts are
// kept away by WHERE a chunk sits: chunk c of row r is stored at c ^ key(r).  Rows read in step with each other
// (32 rows, same chunk) then cover all banks, and so do the 4 x 4-element blocks of a transposed read, whose rows
// differ in their low two bits (those move a row by whole 64-byte groups).
template <typename T, int PITCH, int ROWS, int WAVES>
struct Tile {
  static constexpr int ES = sizeof(T), CH = PITCH * ES / 16, BYTES = ROWS * PITCH * ES;
  static constexpr int RPI = 64 / CH;                     // rows that one wave instruction fills
  static constexpr int NI = ROWS / RPI / WAVES;           // instructions per wave
  static_assert(CH >= 4 && CH <= 32 && RPI * CH == 64 && NI * RPI * WAVES == ROWS, "tile shape");

  static __device__ __forceinline__ int key(int r) {
    if (CH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    if (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);      // two rows fill the 64 banks
    return (r >> 2) & 3;                                              // four do
  }
  // row of this lane within instruction i of wave w, and the 16-byte chunk of the row that it fetches
  static __device__ __forceinline__ int row_of(int i, int w, int lane) { return (i * WAVES + w) * RPI + lane / CH; }
  static __device__ __forceinline__ int chunk_of(int i, int w, int lane) { return (lane % CH) ^ key(row_of(i, w, lane)); }

  // contraction along a row: row r, step s (elements 16 s + 8 half ..)
  static __device__ __forceinline__ typename Vec<T>::v8 along(const char* lds, int r, int s, int half) {
    const char* p = lds + r * (PITCH * ES);
    if constexpr (ES == 2) {
      return *reinterpret_cast<const typename Vec<T>::v8*>(p + (((2 * s + half) ^ key(r)) << 4));
    } else {
      const int c = 4 * s + 2 * half;
      const fx4 a = *reinterpret_cast<const fx4*>(p + ((c ^ key(r)) << 4));
      const fx4 b = *reinterpret_cast<const fx4*>(p + (((c + 1) ^ key(r)) << 4));
      return (fx8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
  }
  // contraction across rows: column 32 d + lane % 32 (of a 16-column tile: columns 16 .. 31 repeat 0 .. 15, nobody takes
  // them), rows 16 s + 4 half + {0..3, 8..11}
  static __device__ __forceinline__ typename Vec<T>::v8 across(const char* lds, int d, int s, int lane) {
    const int half = lane >> 5;
    if constexpr (ES == 2) {
      // ds_read_b64_tr_b16: 16 lanes fetch a 4-row x 16-column block, lane i gets column i of it
      const int i = lane & 15, col = 32 * d + (lane & 16) + 4 * (i & 3);
      union { sx4 h[2]; typename Vec<T>::v8 v; } u;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 16 * s + 8 * j + 4 * half + (i >> 2);
        const char* p = lds + r * (PITCH * 2) + ((((col >> 3) ^ key(r)) << 4) | ((col & 4) << 1));
        u.h[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) sx4*)p);
      }
      return u.v;
    } else {
      const int col = (32 * d + (lane & 31)) % PITCH;
      fx8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int r = 16 * s + 8 * (j >> 2) + 4 * half + (j & 3);
        v[j] = *reinterpret_cast<const float*>(lds + r * (PITCH * 4) + ((((col >> 2) ^ key(r)) << 4) | ((col & 3) << 2)));
      }
      return v;
    }
  }
};

// A raw buffer over `bytes` bytes at p (both the same in all lanes): lanes whose offset lies beyond it fetch zeros.
__device__ __forceinline__ ix4 buffer_of(const void* p, int bytes) {
  const unsigned long a = (unsigned long)p;
  return (ix4){__builtin_amdgcn_readfirstlane((int)a), __builtin_amdgcn_readfirstlane((int)(a >> 32)),
               __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
#define OUT_OF_BUFFER 0x7fffff00       // an offset beyond every buffer made here
// 16 bytes per lane to consecutive LDS from `lds` on (an LDS byte address).  In assembly because the compiler, which
// cannot tell the tile being filled from the one being read, waits for the loads of the builtin before every transposed
// read: the next tile would never be in flight.  No register is written; wait_loads() is the wait.  The compiler does not look
// into the assembly for hazards: five wait states (the move and the s_nop) after whatever vector instruction wrote `b`.
__device__ __forceinline__ void load_to_lds(ix4 b, unsigned lds, int lane_offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds), "v"(lane_offset), "s"(b) : "memory", "m0");
}
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return __builtin_amdgcn_readfirstlane((int)(unsigned long)(const __attribute__((address_space(3))) void*)p);
}
// this wave's LDS reads are done: what they read may be filled again
__device__ __forceinline__ void wait_reads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// this wave's loads have arrived, and its LDS reads are done (the next loads may take the place of what they read).  The
// builtin, not assembly: the compiler then knows that its own loads have arrived too, and waits no second time in the loop.
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);      // vmcnt(0) lgkmcnt(0)
  asm volatile("" ::: "memory");
}

// N products in a row: load(i) fetches the LDS operand of product i, use(i, a) makes it, beside(i) is arithmetic that fills
// the 32 cycles a 16-bit product takes.  For 16-bit types the order is laid down here, LDS reads AHEAD products ahead: left
// to itself the compiler reads one ahead, or hoists so many that registers spill.  fp32 products take eight times as long.
template <typename T, int N, int AHEAD, typename L, typename U, typename B>
__device__ __forceinline__ void products(L load, U use, B beside) {
  if constexpr (sizeof(T) == 2) {
    typename Vec<T>::v8 a[AHEAD + 1];
#pragma unroll
    for (int i = 0; i < AHEAD && i < N; ++i) a[i] = load(i);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i + AHEAD < N) a[(i + AHEAD) % (AHEAD + 1)] = load(i + AHEAD);
      use(i, a[i % (AHEAD + 1)]);
      beside(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      use(i, load(i));
      beside(i);
    }
  }
}

// Whether `bytes` (a multiple of 1024) of LDS hold an infinity or a NaN; the same in all lanes.  A product takes 0 x NaN for
// NaN, so where a tile holds one, what a row (or key) does not see has to be kept from it some other way.
template <typename T>
__device__ __forceinline__ bool not_finite(const char* lds, int bytes, int lane) {
  constexpr unsigned EXP = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, _Float16>::value ? 0x7c007c00u : 0x7f807f80u;
  constexpr unsigned ONE = sizeof(T) == 4 ? 0x00800000u : std::is_same<T, _Float16>::value ? 0x04000400u : 0x00800080u;
  unsigned any = 0;
  for (int at = lane * 16; at < bytes; at += 1024) {
    const ix4 x = *reinterpret_cast<const ix4*>(lds + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) any |= ((unsigned)x[i] & EXP) + ONE;      // an exponent of ones carries into the sign
  }
  return __any(any & (sizeof(T) == 4 ? 0x80000000u : 0x80008000u));
}
// sum over 8 elements, in fp32
template <typename V>
__device__ __forceinline__ float dot8(const V& a, const V& b, float s) {
#pragma unroll
  for (int j = 0; j < 8; ++j) s = fmaf((float)a[j], (float)b[j], s);
  return s;
}

// wave-uniform values: tells the compiler to keep them in scalar registers
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
