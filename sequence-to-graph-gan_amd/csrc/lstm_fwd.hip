// Forward-in-time sweeps of the critic's 2-layer LSTM (reference: nn.LSTM(175, 50, 2) inside
// Discriminator.forward, wgan_gp.py:189,217): sweep A (primal states) and sweep C (tangent
// states along an input direction, used by the gradient penalty's second-order term,
// wgan_gp.py:247-256).
//
// A sweep is a chain of 512 dependent steps, so its time is (cycles per step) x 512.  A SIMD
// issues one wave64 VALU instruction per 4 cycles whatever the number of resident waves, so the
// design minimises VALU instructions per SIMD per step and spreads them evenly over the 4 SIMDs.
// ONE workgroup of EIGHT waves per sequence; the three 200x50 mat-vecs of a step run
// concurrently on different time steps, with a single barrier per step:
//   waves 0,1  t = tau      a0 = xproj_t + W_hh0 h0_{t-1}  -> gates, c0, h0_t, y_t = mask*h0_t
//   waves 4..7 t = tau-1    p1 = b1 + W_ih1 y_t             -> LDS
//   waves 2,3  t = tau-2    a1 = p1 + W_hh1 h1_{t-1}        -> gates, c1, h1_t
// (wave i sits on SIMD i%4: every SIMD gets one cell wave and one projection wave).
// Cell waves: lane = (unit u, half s); it holds the 4 gate rows of u over columns 25s..25s+24 in
// 100 registers, as pairs -> 100 v_fma_f32 per step, the state slice coming from LDS in
// 7 16-byte reads.  A 2-lane reduce-scatter (2 DPP adds) leaves gates (i,f) in lane s=0 and
// (g,o) in lane s=1; each lane activates and stores its pair, lane 1 fetches (i,f) by DPP and
// advances the cell.  Projection waves: lane = (unit, quarter s) with 13 columns, 52 v_fma_f32
// and a 4-lane reduce-scatter (3 DPP adds) that leaves gate s in lane s.
// Per-step inputs are prefetched PF steps ahead into a register ring by UNCONDITIONAL loads from
// clamped addresses (a load under a branch makes the compiler drain vmcnt to 0 at the join: one
// full memory round trip on each of the 512 sequential steps).
#include "s2g_common.h"

#define PF 6
#ifndef PFC
#define PFC 6                  // ring depth of sweep C's cell waves
#endif
#define FWD_THREADS 512
#define HV 56                  // LDS state vector: 2 slices of 25 units, each padded to 28 floats
#define FWD_LDS_FLOATS 864     // h0buf[2][HV] h1buf[2][HV] ybuf[2][64] p1buf[2][256]

__device__ __forceinline__ int pos25(int k) { return 28 * (k / 25) + (k % 25); }

// Cell-wave weights of lane (u, s): columns 25s..25s+24 of unit u's gate rows in a torch-layout
// [4H, H] matrix.  wk = the gate pair this lane keeps (2s, 2s+1), wx = the pair it hands over.
__device__ __forceinline__ void load_w_half(const float* W, int u, int s, f2 wk[25], f2 wx[25]) {
  const int qk = 2 * s, qx = 2 * (s ^ 1);
#pragma unroll
  for (int k = 0; k < 25; ++k) {
    const int col = 25 * s + k;
    wk[k] = (f2){W[((qk + 0) * S2G_H + u) * S2G_H + col], W[((qk + 1) * S2G_H + u) * S2G_H + col]};
    wx[k] = (f2){W[((qx + 0) * S2G_H + u) * S2G_H + col], W[((qx + 1) * S2G_H + u) * S2G_H + col]};
  }
}

// this lane's 28-float slice of an LDS state vector
__device__ __forceinline__ void load_slice28(const float* slice, float v[28]) {
  const float4* p = reinterpret_cast<const float4*>(slice);
#pragma unroll
  for (int i = 0; i < 7; ++i) {
    const float4 a = p[i];
    v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
  }
}

// pre-activations of gates (2s, 2s+1) of unit u = init + W . v
__device__ __forceinline__ f2 matvec_half(const f2 wk[25], const f2 wx[25], const float v[28], f2 init) {
  f2 ak = init, ax = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 25; ++k) {
    const f2 vv = {v[k], v[k]};
    ak = __builtin_elementwise_fma(wk[k], vv, ak);
    ax = __builtin_elementwise_fma(wx[k], vv, ax);
  }
  ak.x += dpp_mov<DPP_QUAD(1, 0, 3, 2)>(ax.x);
  ak.y += dpp_mov<DPP_QUAD(1, 0, 3, 2)>(ax.y);
  return ak;
}

// Projection-wave weights of lane (u, s): columns 13s..13s+12, slot q = gate (s ^ q)
__device__ __forceinline__ void load_w_quarter(const float* W, int u, int s, f2 w01[13], f2 w23[13]) {
#pragma unroll
  for (int k = 0; k < 13; ++k) {
    const int col = 13 * s + k;
    const bool ok = col < S2G_H;
    const int cc = ok ? col : 0;
    float v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float x = W[((s ^ q) * S2G_H + u) * S2G_H + cc];
      v[q] = ok ? x : 0.0f;
    }
    w01[k] = (f2){v[0], v[1]};
    w23[k] = (f2){v[2], v[3]};
  }
}

// gate s of unit u: (W . v) summed over the quad; slice = this lane's 16-float slice (pos13 layout)
__device__ __forceinline__ float matvec_quarter(const f2 w01[13], const f2 w23[13], const float* slice) {
  float v[16];
  const float4* p = reinterpret_cast<const float4*>(slice);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 a = p[i];
    v[4 * i] = a.x; v[4 * i + 1] = a.y; v[4 * i + 2] = a.z; v[4 * i + 3] = a.w;
  }
  f2 a01 = {0.f, 0.f}, a23 = {0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 13; ++k) {
    const f2 vv = {v[k], v[k]};
    a01 = __builtin_elementwise_fma(w01[k], vv, a01);
    a23 = __builtin_elementwise_fma(w23[k], vv, a23);
  }
  return quad_reduce_scatter(a01.x, a01.y, a23.x, a23.y);
}

// value of the even lane of each lane pair
__device__ __forceinline__ float from_even(float v) { return dpp_mov<DPP_QUAD(0, 0, 2, 2)>(v); }

// ------------------------------------------------------------------------------------------
// Sweep A.  Saves per (row = ws_row + t): gates{0,1}[row][4u+q] = activated gate q of unit u;
// cell0[row][4u+{0,1,2,3}] = (c, tanh c, h, mask*h); cell1 likewise with the 4th slot 0;
// hT[n][u] = final hidden state of layer 1.
// Dynamic LDS: FWD_LDS_FLOATS floats + max_len ints.
// ------------------------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(FWD_THREADS) void s2g_k_lstm2_fwd(
    const S2GSeq* __restrict__ seqs, const int* __restrict__ tokens, const float* __restrict__ WT0,
    const float* __restrict__ P, const float* __restrict__ mask, const float* __restrict__ b0,
    const float* __restrict__ b1, const float* __restrict__ whh0, const float* __restrict__ wih1,
    const float* __restrict__ whh1, float* __restrict__ gates0, float* __restrict__ cell0,
    float* __restrict__ gates1, float* __restrict__ cell1, float* __restrict__ hT, int vocab, int max_len) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  float* h0buf = reinterpret_cast<float*>(smem);   // [2][HV]
  float* h1buf = h0buf + 2 * HV;                    // [2][HV]
  float* ybuf = h1buf + 2 * HV;                     // [2][64], pos13 layout
  float* p1buf = ybuf + 128;                        // [2][256]
  int* tok_lds = reinterpret_cast<int*>(p1buf + 512);

  const int n = blockIdx.x;
  const S2GSeq sq = seqs[n];
  const int tid = threadIdx.x;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);   // wave-uniform: role tests and row pointers stay scalar
  const int lane = tid & 63;
  const int len = min(sq.len, max_len);      // the token stage in LDS holds max_len entries
  const bool has_tok = sq.tok_off >= 0 && sq.ca != 0.0f;
  const bool has_p = sq.p_off >= 0 && sq.cp != 0.0f && sq.p_len > 0;
  const bool has_mask = sq.mask_off >= 0 && mask != nullptr;

  if (len <= 0) {
    if (tid < S2G_H) hT[(size_t)n * S2G_H + tid] = 0.0f;
    return;
  }
  for (int i = tid; i < FWD_LDS_FLOATS; i += FWD_THREADS) h0buf[i] = 0.0f;
  // a token outside [0, vocab) would index past the V rows of WT0: the host wrappers reject such batches
  // where they see them on the CPU; here the row index is clamped so that no access leaves the table
  for (int i = tid; i < len; i += FWD_THREADS)
    tok_lds[i] = has_tok ? min(max(tokens[sq.tok_off + i], 0), vocab - 1) : 0;
  const int nit = len + 2;                    // pipeline iterations (= barriers) of every wave

  if (wv >= 4) {
    // ---------------- projection waves: p1 = b1 + W_ih1 y_{tau-1} ----------------
    const int u = 16 * (wv - 4) + (lane >> 2), s = lane & 3;
    const bool valid = u < S2G_H;
    const int uc = valid ? u : S2G_H - 1;
    f2 w01[13], w23[13];
    load_w_quarter(wih1, uc, s, w01, w23);
    const float bias = b1[4 * uc + s];
    __syncthreads();
    for (int tau = 0; tau < nit; ++tau) {
      const int t = tau - 1;
      if (t >= 0 && t < len) {
        const float r = matvec_quarter(w01, w23, ybuf + (t & 1) * 64 + 16 * s) + bias;
        if (valid) p1buf[(t & 1) * 256 + 4 * u + s] = r;
      }
      __syncthreads();
    }
    return;
  }

  // ---------------- cell waves ----------------
  // Global addresses are (wave-uniform row pointer) + (constant per-lane offset): the row pointer
  // lives in scalar registers and the per-step address arithmetic costs no vector instructions.
  const bool l0 = wv < 2;
  const int u = 32 * (wv & 1) + (lane >> 1), s = lane & 1;
  const bool valid = u < S2G_H;
  const int uc = valid ? u : S2G_H - 1;
  const bool owner = valid && s == 1;
  f2 wk[25], wx[25];
  load_w_half(l0 ? whh0 : whh1, uc, s, wk, wx);
  const unsigned lo4 = 4 * uc, lo2 = 4 * uc + 2 * s;          // lane offsets inside a 200-float row
  const size_t row0 = (size_t)sq.ws_row * S2G_G;
  const float kact = s ? -2.8853900817779268f : -1.4426950408889634f;   // lane 1's first gate is the tanh one
  const float actA = s ? 2.0f : 1.0f, actB = s ? -1.0f : 0.0f;
  const int hp = pos25(uc), yp = pos13(uc);

  if (l0) {
    const float2 bias = *reinterpret_cast<const float2*>(b0 + lo2);
    // absent inputs read b0 (always 200 valid floats) with stride 0 and coefficient 0
    const float* pa = has_tok ? WT0 : b0;
    const int sa = has_tok ? S2G_G : 0;
    const float* pp = has_p ? P + (size_t)sq.p_off * S2G_G : b0;
    const int sp = has_p ? S2G_G : 0;
    const float* pm = has_mask ? mask + (size_t)sq.mask_off * S2G_MASKW : b0;
    const int sm = has_mask ? S2G_MASKW : 0;
    const float ca = has_tok ? sq.ca : 0.0f;
    const float cp = has_p ? sq.cp : 0.0f;
    const int plast = sq.p_len > 0 ? sq.p_len - 1 : 0;
    float* gout = gates0 + row0;
    float* cout = cell0 + row0;
    __syncthreads();
    float2 xa[PF], xp[PF];
    float mk[PF];
#define ISSUE_A(j, t, token)                                                                 \
    {                                                                                        \
      const int tc_ = min((t), len - 1);                                                     \
      const int tok_ = __builtin_amdgcn_readfirstlane(token);                                \
      xa[j] = *reinterpret_cast<const float2*>(pa + (unsigned)(tok_ * sa) + lo2);            \
      xp[j] = *reinterpret_cast<const float2*>(pp + (unsigned)(min(tc_, plast) * sp) + lo2); \
      mk[j] = (pm + (unsigned)(tc_ * sm))[uc];                                               \
    }
#pragma unroll
    for (int j = 0; j < PF; ++j) ISSUE_A(j, j, tok_lds[min(j, len - 1)])
    int tk = tok_lds[min(PF, len - 1)];      // token of the next step to prefetch, read one step early
    // Order inside a step: the LDS reads of h_{t-1} go first (they head the step's critical path);
    // their latency is filled with work that is off it -- the global stores of step t-1 (kept in
    // registers for one step) and the refill of the ring slot step t-1 consumed.
    float c = 0.0f;
    float2 sg = make_float2(0.f, 0.f);
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int base = 0; base < len; base += PF) {
#pragma unroll
      for (int j = 0; j < PF; ++j) {
        const int t = base + j;
        if (t < len) {
          float hv[28];
          load_slice28(h0buf + ((t + 1) & 1) * HV + 28 * s, hv);
          if (t >= 1) {
            float* grow = gout + (unsigned)((t - 1) * S2G_G);
            float* crow = cout + (unsigned)((t - 1) * S2G_G);
            if (valid) *reinterpret_cast<float2*>(grow + lo2) = sg;
            if (owner) *reinterpret_cast<float4*>(crow + lo4) = sc;
            ISSUE_A((j + PF - 1) % PF, t - 1 + PF, tk)
            tk = tok_lds[min(t + PF, len - 1)];
          }
          const float cpt = (t < sq.p_len) ? cp : 0.0f;
          const f2 x = {fmaf(cpt, xp[j].x, fmaf(ca, xa[j].x, bias.x)), fmaf(cpt, xp[j].y, fmaf(ca, xa[j].y, bias.y))};
          const f2 a = matvec_half(wk, wx, hv, x);
          const float v0 = fmaf(__builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(kact * a.x)), actA, actB);
          const float v1 = fast_sigmoid(a.y);
          const float gi = from_even(v0), gf = from_even(v1);      // lane 1: (i, f); its own v0, v1 = (g, o)
          c = fmaf(gf, c, gi * v0);
          const float tc = fast_tanh(c);
          const float h = v1 * tc;
          const float y = has_mask ? mk[j] * h : h;
          if (owner) {
            h0buf[(t & 1) * HV + hp] = h;
            ybuf[(t & 1) * 64 + yp] = y;
          }
          sg = make_float2(v0, v1);
          sc = make_float4(c, tc, h, y);
          __syncthreads();
        }
      }
    }
    {
      float* grow = gout + (unsigned)((len - 1) * S2G_G);
      float* crow = cout + (unsigned)((len - 1) * S2G_G);
      if (valid) *reinterpret_cast<float2*>(grow + lo2) = sg;
      if (owner) *reinterpret_cast<float4*>(crow + lo4) = sc;
    }
    __syncthreads();      // the two pipeline-drain iterations of the other waves
    __syncthreads();
  } else {
    float* gout = gates1 + row0;
    float* cout = cell1 + row0;
    __syncthreads();
    __syncthreads();      // pipeline fill: layer 1 starts two steps behind layer 0
    __syncthreads();
    float c = 0.0f;
    float2 sg = make_float2(0.f, 0.f);
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int t = 0; t < len; ++t) {
      float hv[28];
      load_slice28(h1buf + ((t + 1) & 1) * HV + 28 * s, hv);
      const float2 pin = *reinterpret_cast<const float2*>(p1buf + (t & 1) * 256 + lo2);
      if (t >= 1) {
        float* grow = gout + (unsigned)((t - 1) * S2G_G);
        float* crow = cout + (unsigned)((t - 1) * S2G_G);
        if (valid) *reinterpret_cast<float2*>(grow + lo2) = sg;
        if (owner) *reinterpret_cast<float4*>(crow + lo4) = sc;
      }
      const f2 a = matvec_half(wk, wx, hv, (f2){pin.x, pin.y});
      const float v0 = fmaf(__builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(kact * a.x)), actA, actB);
      const float v1 = fast_sigmoid(a.y);
      const float gi = from_even(v0), gf = from_even(v1);
      c = fmaf(gf, c, gi * v0);
      const float tc = fast_tanh(c);
      const float h = v1 * tc;
      if (owner) h1buf[(t & 1) * HV + hp] = h;
      sg = make_float2(v0, v1);
      sc = make_float4(c, tc, h, 0.0f);
      __syncthreads();
    }
    {
      float* grow = gout + (unsigned)((len - 1) * S2G_G);
      float* crow = cout + (unsigned)((len - 1) * S2G_G);
      if (valid) *reinterpret_cast<float2*>(grow + lo2) = sg;
      if (owner) {
        *reinterpret_cast<float4*>(crow + lo4) = sc;
        hT[(size_t)n * S2G_H + u] = sc.z;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------
// Sweep C: tangent states.  adot_t = xdot_t + W_hh hdot_{t-1}, gate tangents from the saved
// primal gates, cdot_t = fdot c_{t-1} + f cdot_{t-1} + idot g + i gdot,
// hdot_t = odot tanh(c) + o (1 - tanh^2 c) cdot.  Saves adot{0,1}[row][4u+q],
// celld0[row][4u+{0,1,2,3}] = (cdot, hdot, mask*hdot, 0), celld1 = (cdot, hdot, 0, 0), hdotT.
// Xdot holds the projected input direction rows [ws_row + t][200] (no bias).
// Same eight-wave pipeline as sweep A; the cell waves prefetch the saved primal gates / cell values.
// ------------------------------------------------------------------------------------------
extern "C" __global__ __launch_bounds__(FWD_THREADS) void s2g_k_lstm2_tangent(
    const S2GSeq* __restrict__ seqs, const float* __restrict__ Xdot, const float* __restrict__ mask,
    const float* __restrict__ whh0, const float* __restrict__ wih1, const float* __restrict__ whh1,
    const float* __restrict__ gates0, const float* __restrict__ cell0, const float* __restrict__ gates1,
    const float* __restrict__ cell1, float* __restrict__ adot0, float* __restrict__ celld0,
    float* __restrict__ adot1, float* __restrict__ celld1, float* __restrict__ hdotT,
    const float* __restrict__ gp_partial, float gp_upstream, float gp_n_batch) {
  __shared__ __attribute__((aligned(16))) float lds[FWD_LDS_FLOATS];
  float* h0buf = lds;                 // hdot of layer 0 [2][HV]
  float* h1buf = lds + 2 * HV;        // hdot of layer 1 [2][HV]
  float* ybuf = h1buf + 2 * HV;       // mask * hdot0    [2][64], pos13 layout
  float* p1buf = ybuf + 128;          // W_ih1 ydot      [2][256]

  const int n = blockIdx.x;
  const S2GSeq sq = seqs[n];
  const int tid = threadIdx.x;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int len = sq.len;
  const bool has_mask = sq.mask_off >= 0 && mask != nullptr;

  if (len <= 0) {
    if (tid < S2G_H) hdotT[(size_t)n * S2G_H + tid] = 0.0f;
    return;
  }
  for (int i = tid; i < FWD_LDS_FLOATS; i += FWD_THREADS) lds[i] = 0.0f;
  const int nit = len + 2;

  if (wv >= 4) {
    const int u = 16 * (wv - 4) + (lane >> 2), s = lane & 3;
    const bool valid = u < S2G_H;
    const int uc = valid ? u : S2G_H - 1;
    f2 w01[13], w23[13];
    load_w_quarter(wih1, uc, s, w01, w23);
    __syncthreads();
    for (int tau = 0; tau < nit; ++tau) {
      const int t = tau - 1;
      if (t >= 0 && t < len) {
        const float r = matvec_quarter(w01, w23, ybuf + (t & 1) * 64 + 16 * s);
        if (valid) p1buf[(t & 1) * 256 + 4 * u + s] = r;
      }
      __syncthreads();
    }
    return;
  }

  // cell waves: 0,1 = layer 0 (lag 0), 2,3 = layer 1 (lag 2); shared element-wise code
  const bool l0 = wv < 2;
  const int lag = l0 ? 0 : 2;
  const int u = 32 * (wv & 1) + (lane >> 1), s = lane & 1;
  const bool valid = u < S2G_H;
  const int uc = valid ? u : S2G_H - 1;
  const bool owner = valid && s == 1;
  f2 wk[25], wx[25];
  load_w_half(l0 ? whh0 : whh1, uc, s, wk, wx);
  // wave-uniform row pointers + constant per-lane offsets (see sweep A)
  const unsigned lo4 = 4 * uc, lo2 = 4 * uc + 2 * s;
  const size_t row0 = (size_t)sq.ws_row * S2G_G;
  const float* pg = (l0 ? gates0 : gates1) + row0;
  const float* pc = (l0 ? cell0 : cell1) + row0;
  const float* px = l0 ? Xdot + row0 : whh0;          // absent inputs read whh0 (2500 floats) with stride 0
  const int sx = l0 ? S2G_G : 0;
  const float* pm = (l0 && has_mask) ? mask + (size_t)sq.mask_off * S2G_MASKW : whh0;
  const int sm = (l0 && has_mask) ? S2G_MASKW : 0;
  float* adot = (l0 ? adot0 : adot1) + row0;
  float* celld = (l0 ? celld0 : celld1) + row0;
  float* hb = l0 ? h0buf : h1buf;
  const int hp = pos25(uc), yp = pos13(uc);
  __syncthreads();

  float4 rg[PFC];
  float2 rx[PFC], rc[PFC];
  float mk[PFC];
#define ISSUE_C(j, t)                                                        \
  {                                                                          \
    const int tc_ = max(min((t), len - 1), 0);                               \
    rg[j] = *reinterpret_cast<const float4*>(pg + (unsigned)(tc_ * S2G_G) + lo4);  \
    rc[j] = *reinterpret_cast<const float2*>(pc + (unsigned)(tc_ * S2G_G) + lo4);  \
    rx[j] = *reinterpret_cast<const float2*>(px + (unsigned)(tc_ * sx) + lo2);     \
    mk[j] = (pm + (unsigned)(tc_ * sm))[uc];                                       \
  }
  // ring slot tau % PFC holds step tau - lag
#pragma unroll
  for (int j = 0; j < PFC; ++j) ISSUE_C(j, j - lag)

  // gp_partial (optional): Xdot holds the UNSCALED projected direction M2 delta of the gradient
  // penalty; its per-sample factor comes from the four partial sums of |g|^2 (s2g_k_gp_dots), so no
  // scaling pass over Xdot sits between the reverse sweep and this one
  const float seed_scale =
      gp_partial ? gp_coef_from_partials(gp_partial + 4 * blockIdx.x, gp_upstream, gp_n_batch) : 1.0f;
  float cd = 0.0f;      // cdot carried
  float cprev = 0.0f;   // primal c_{t-1} carried
  for (int base = 0; base < nit; base += PFC) {
#pragma unroll
    for (int j = 0; j < PFC; ++j) {
      const int tau = base + j;
      if (tau < nit) {
        const int t = tau - lag;
        if (t >= 0 && t < len) {
          f2 init;
          if (l0) init = (f2){seed_scale * rx[j].x, seed_scale * rx[j].y};
          else {
            const float2 pin = *reinterpret_cast<const float2*>(p1buf + (t & 1) * 256 + lo2);
            init = (f2){pin.x, pin.y};
          }
          const f2 ad = matvec_half(wk, wx, hb + ((t + 1) & 1) * HV + 28 * s, init);
          const float gi = rg[j].x, gf = rg[j].y, gg = rg[j].z, go = rg[j].w, tc = rc[j].y;
          const float g0 = s ? gg : gi, g1 = s ? go : gf;              // this lane's gate pair
          const float d0 = fmaf(-g0, g0, s ? 1.0f : g0) * ad.x;      // sigma' = g(1-g), tanh' = 1-g^2
          const float d1 = fmaf(-g1, g1, g1) * ad.y;
          const float di = from_even(d0), df = from_even(d1);          // lane 1: its own d0, d1 = (dg, do)
          cd = df * cprev + gf * cd + di * gg + gi * d0;
          cprev = rc[j].x;
          const float hd = d1 * tc + go * (1.0f - tc * tc) * cd;
          const float yd = (l0 && has_mask) ? mk[j] * hd : hd;
          float* arow = adot + (unsigned)(t * S2G_G);
          float* crow = celld + (unsigned)(t * S2G_G);
          if (valid) *reinterpret_cast<float2*>(arow + lo2) = make_float2(ad.x, ad.y);
          if (owner) {
            *reinterpret_cast<float4*>(crow + lo4) = make_float4(cd, hd, l0 ? yd : 0.0f, 0.0f);
            hb[(t & 1) * HV + hp] = hd;
            if (l0) ybuf[(t & 1) * 64 + yp] = yd;
            if (!l0 && t == len - 1) hdotT[(size_t)n * S2G_H + u] = hd;
          }
        }
        __syncthreads();
      }
      ISSUE_C(j, tau + PFC - lag)     // refill after the slot's last use: it keeps its registers
    }
  }
}
