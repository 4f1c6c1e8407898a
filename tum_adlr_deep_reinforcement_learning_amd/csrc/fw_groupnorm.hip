// fw_groupnorm.hip -- group norm with an activation over channels-last rows (include/fwrollout.h).
//
// A unit is one sample's group: L rows of cg = C / G adjacent channels, read as vectors of VW channels.  The kernels, by a unit's size:
//   k_gn_wave   a unit fits 64 lanes x 4 vectors: 2^k lanes per unit, several units per wave; for one row per sample
//               (a policy's features) this is a plain stream over the tensor (524288 x 64 float32 in 4 groups, tanh:
//               forward 52 us, 5100 GB/s; backward 86 us, 4700 GB/s)
//   k_gn_block  a unit fits a block's registers: read once, written once (16 x 4096 x 512 bfloat16 in 32 groups, silu:
//               39 us, 3500 GB/s; all blocks run at once, so loading, sums and storing follow each other)
//   k_gn_bundle several neighbouring units do, where one has too few channels for 16-byte accesses (64 x 900 x 320
//               bfloat16 in 32 groups, gelu: forward 44 us, 1700 GB/s, backward 67 us)
//   k_gn_stream_*  larger: two passes over the tensor
// All statistics are sums of deviations from a mean, so a large mean does not cancel.  Memory bound: x in, y out (and
// dy in, dx out); the gradients of weight and bias are column sums of per-unit partial sums, in a fixed order.
#include <algorithm>
#include <type_traits>

#include "fw_seq_common.hpp"

using namespace fwseq;

namespace {

struct Rows {
  void* p;
  int64_t sn, sl;
};
struct GnArgs {
  Rows x, y, dy, dx;
  const void *w, *b;
  int64_t N, L;
  int32_t G, cg, wdt, act, split, lanes_log2;
  float eps;
  float* stats;  // [N][G][2] or NULL
  float* dw;     // partial sums [R][C], or NULL
  float* db;
  float* sums;   // streams: [N][split][G][3]
};

__device__ __forceinline__ float param(const void* p, int dt, int c, float none) {
  if (!p) return none;
  if (dt == FW_DT_F32) return ((const float*)p)[c];
  if (dt == FW_DT_BF16) return to_f32(((const bf16*)p)[c]);
  return to_f32(((const f16*)p)[c]);
}

// Activations from the hardware's exp2 and reciprocal (an ulp each), with no division and no branch.  In float32 what the
// exponent rounds off is carried along and the reciprocal gets a step of Newton's; the 16-bit types do not see either.
template <typename T>
__device__ __forceinline__ float exp_fast(float x) {
  const float h = x * 1.44269504f;
  if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(h);
  const float rest = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -h));  // log2(e) in two parts
  return __builtin_amdgcn_exp2f(h) * fmaf(fabsf(h) < 256.f ? rest : 0.f, 0.693147181f, 1.f);
}
template <typename T>
__device__ __forceinline__ float reciprocal(float x) {  // x >= 1
  const float r = __builtin_amdgcn_rcpf(x);
  if constexpr (sizeof(T) == 2) return r;
  return x < 1e38f ? fmaf(fmaf(-x, r, 1.f), r, r) : r;
}
template <typename T>
__device__ __forceinline__ float sigmoid(float z) {
  return reciprocal<T>(1.f + exp_fast<T>(-z));
}
template <typename T>
__device__ __forceinline__ float tanh_fast(float z) {
  // near 0 the difference below loses what it has; there z + z^3 times a polynomial in z^2, fitted to tanh up to 5/8 (4e-9)
  const float t = z * z;
  const float p = fmaf(t * z, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.00570498453f, 0.0206390843f), -0.0537397154f), 0.133314416f),
                                   -0.333332807f), z);
  const float q = fmaf(-2.f, reciprocal<T>(1.f + exp_fast<T>(2.f * z)), 1.f);
  return fabsf(z) < 0.625f ? p : q;
}
// Phi(-|z|), and e = exp(-z^2 / 2) beside it.  float32: the library's erfc.  16-bit types: e times a polynomial in t = 1 / (1 +
// 0.3041 |z|), fitted to Phi(-|z|) / e so that its largest relative error up to z = 13.6 (where float32 ends) is least:
// 9e-8, which a bias's gradient, a float32 sum of many slopes, needs; far out the exponential's argument adds 1e-5, against
// half a step of 5e-4 (float16) and 4e-3 (bfloat16).
template <typename T>
__device__ __forceinline__ float normal_tail(float z, float& e) {
  if constexpr (sizeof(T) == 4) {
    // z^2 / 2 and |z| / sqrt(2) round to 2^-24 of numbers that the tail has as exponents: what they lose is carried along
    const float a = fabsf(z) > 64.f ? 64.f : fabsf(z), s = a * a, x = a * 0.707106769f;
    e = exp_fast<T>(-0.5f * s) * fmaf(-0.5f, fmaf(a, a, -s), 1.f);
    const float rest = fmaf(a, 1.21016175e-8f, fmaf(a, 0.707106769f, -x));  // 1 / sqrt(2) in two parts
    return fmaf(-0.564189584f * rest, e, 0.5f * erfcf(x));
  } else {
    e = __builtin_amdgcn_exp2f(z * -0.72134752f * z);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3041f, fabsf(z), 1.f));
    const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.0368336476f, -0.1550304f), 0.191474333f), -0.0425504558f), 0.123265989f);
    return t * e * fmaf(t, fmaf(t, fmaf(t, p, 0.102532998f), 0.122198641f), 0.121275306f);
  }
}

template <typename T>
__device__ __forceinline__ float act_value(float z, int act) {
  float e;
  switch (act) {
    case FW_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case FW_ACT_SILU: return z * sigmoid<T>(z);
    case FW_ACT_GELU: {  // z Phi(z) from the tail on z's own side: no difference of near numbers
      const float q = normal_tail<T>(z, e);
      return fmaf(-fminf(fabsf(z), 64.f), q, fmaxf(z, 0.f));  // (an infinity times no tail is no tail)
    }
    case FW_ACT_TANH: return tanh_fast<T>(z);
  }
  return z;
}
template <typename T>
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case FW_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case FW_ACT_SILU: {
      const float s = sigmoid<T>(z);
      return s * fmaf(z, 1.f - s, 1.f);
    }
    case FW_ACT_GELU: {
      float e;
      const float q = normal_tail<T>(z, e);
      return fmaf(z * 0.39894228f, e, z < 0.f ? q : 1.f - q);
    }
    case FW_ACT_TANH: {
      const float s = sigmoid<T>(-2.f * fabsf(z));  // 1 - tanh^2, without the difference
      return 4.f * s * (1.f - s);
    }
  }
  return 1.f;
}
// 1 / sqrt(x): the hardware's estimate and one step of Newton's, which small numbers and an infinite one (a variance beyond
// float32: 0, so that y is the bias) would leave with 0 x inf
__device__ __forceinline__ float inv_sqrt(float x) {
  const float r = __builtin_amdgcn_rsqf(x);
  return x < 1e-30f || x > 1e38f ? 1.f / sqrtf(x) : r * fmaf(-0.5f * x * r, r, 1.5f);
}

// ------------------------------------------------------------------ units of a few lanes
// Slot = a run of 2^lanes_log2 lanes.  The number of slots is a multiple of G, so a slot keeps its group (and its
// weights, and its weight gradients) while n runs.
template <typename T, int VW, int VPL, bool BWD>
__global__ __launch_bounds__(256) void k_gn_wave(GnArgs A) {
  const int lane = threadIdx.x & 63, lg = 1 << A.lanes_log2, sub = lane & (lg - 1);
  const int64_t slot = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * (64 >> A.lanes_log2) + (lane >> A.lanes_log2);
  const int64_t slots = (int64_t)gridDim.x * 4 * (64 >> A.lanes_log2);
  const int g = (int)(slot % A.G);
  const int64_t dn = slots / A.G;
  const int cgv = A.cg / VW, total = (int)A.L * cgv;
  const float count = (float)(A.L * A.cg), inv = 1.f / count;
  bool ok[VPL];
  int row[VPL], col[VPL];
  float w[VPL][VW], b[VPL][VW], dw[VPL][VW], db[VPL][VW];
#pragma unroll
  for (int i = 0; i < VPL; i++) {
    const int e = sub + lg * i;
    ok[i] = e < total;
    row[i] = ok[i] ? e / cgv : 0;
    col[i] = ok[i] ? (e - row[i] * cgv) * VW : 0;
#pragma unroll
    for (int k = 0; k < VW; k++) {
      w[i][k] = param(A.w, A.wdt, g * A.cg + col[i] + k, 1.f);
      b[i][k] = param(A.b, A.wdt, g * A.cg + col[i] + k, 0.f);
      dw[i][k] = db[i][k] = 0.f;
    }
  }
  auto total_of = [&](float s) {
    for (int m = 1; m < lg; m <<= 1) s += __shfl_xor(s, m);
    return s;
  };
  for (int64_t n = slot / A.G; __any(n < A.N); n += dn) {
    const bool live = n < A.N;
    const int64_t nn = live ? n : 0;
    float x[VPL][VW], dy[VPL][VW];
#pragma unroll
    for (int i = 0; i < VPL; i++) {
      load_vec<T, VW>((const T*)A.x.p + nn * A.x.sn + row[i] * A.x.sl + g * A.cg + col[i], x[i]);
      if constexpr (BWD) load_vec<T, VW>((const T*)A.dy.p + nn * A.dy.sn + row[i] * A.dy.sl + g * A.cg + col[i], dy[i]);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++)
#pragma unroll
      for (int k = 0; k < VW; k++) s += ok[i] ? x[i][k] : 0.f;
    const float mean = total_of(s) / count;  // (of equal numbers: that number)
    s = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++)
#pragma unroll
      for (int k = 0; k < VW; k++) {
        x[i][k] -= mean;
        s += ok[i] ? x[i][k] * x[i][k] : 0.f;
      }
    const float r = inv_sqrt(total_of(s) * inv + A.eps);
    if constexpr (!BWD) {
      if (A.stats && live && sub == 0) {
        A.stats[2 * (n * A.G + g)] = mean;
        A.stats[2 * (n * A.G + g) + 1] = r;
      }
#pragma unroll
      for (int i = 0; i < VPL; i++) {
#pragma unroll
        for (int k = 0; k < VW; k++) x[i][k] = act_value<T>(fmaf(x[i][k] * r, w[i][k], b[i][k]), A.act);
        if (ok[i] && live) store_vec<T, VW>((T*)A.y.p + n * A.y.sn + row[i] * A.y.sl + g * A.cg + col[i], x[i]);
      }
    } else {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; i++)
#pragma unroll
        for (int k = 0; k < VW; k++) {
          x[i][k] *= r;
          const float dz = ok[i] && live ? dy[i][k] * act_slope<T>(fmaf(x[i][k], w[i][k], b[i][k]), A.act) : 0.f;
          db[i][k] += dz;
          dw[i][k] += ok[i] && live ? dz * x[i][k] : 0.f;
          dy[i][k] = dz * w[i][k];
          s1 += dy[i][k];
          s2 += ok[i] ? dy[i][k] * x[i][k] : 0.f;
        }
      s1 = total_of(s1) * inv;
      s2 = total_of(s2) * inv;
#pragma unroll
      for (int i = 0; i < VPL; i++) {
#pragma unroll
        for (int k = 0; k < VW; k++) x[i][k] = r * (dy[i][k] - s1 - x[i][k] * s2);
        if (ok[i] && live) store_vec<T, VW>((T*)A.dx.p + n * A.dx.sn + row[i] * A.dx.sl + g * A.cg + col[i], x[i]);
      }
    }
  }
  if constexpr (BWD) {
    // The block's sums: over its rows, and over its slots of equal group where it holds every group equally often.
    extern __shared__ float sl[];  // [slots of the block][L][cg]
    const int spb = 4 * (64 >> A.lanes_log2), myslot = (int)(threadIdx.x >> A.lanes_log2), unit = (int)A.L * A.cg;
    const int classes = spb % A.G == 0 ? A.G : spb;
#pragma unroll
    for (int which = 0; which < 2; which++) {
      float* part = which ? A.db : A.dw;
      if (!part) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < VPL; i++)
        if (ok[i])
#pragma unroll
          for (int k = 0; k < VW; k++) sl[myslot * unit + row[i] * A.cg + col[i] + k] = which ? db[i][k] : dw[i][k];
      __syncthreads();
      for (int o = threadIdx.x; o < classes * A.cg; o += 256) {
        const int j = o / A.cg, c = o - j * A.cg;
        float s = 0.f;
        for (int q = j; q < spb; q += classes)
          for (int l = 0; l < (int)A.L; l++) s += sl[q * unit + l * A.cg + c];
        part[(int64_t)blockIdx.x * classes * A.cg + o] = s;
      }
    }
  }
}

// ------------------------------------------------------------------ block helpers
template <int NV>
__device__ __forceinline__ void block_sum(float* v, float (*lds)[NV]) {  // every thread gets the sums, fixed order
#pragma unroll
  for (int k = 0; k < NV; k++)
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v[k] += __shfl_xor(v[k], m);
  const int waves = (blockDim.x + 63) >> 6;
  __syncthreads();
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < NV; k++) lds[threadIdx.x >> 6][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NV; k++) {
    float s = 0.f;
    for (int q = 0; q < waves; q++) s += lds[q][k];
    v[k] = s;
  }
}

// Per channel (VW of a column, thread = row * cols + column, `rows` rows): the sums of NA values over its rows, in a fixed
// order, each handed to sink(channel, sums) by one thread.  Many rows: a wave per channel; few: a thread.  (A tree over
// the rows with a barrier a step takes 7 us more: map of 64 x 900 x 320 bfloat16, forward.)
template <int VW, int NA, typename Sink>
__device__ __forceinline__ void channel_sums(const float (&v)[NA][VW], int t, int rows, int cols, bool on, float* lds, Sink sink) {
  const int threads = (int)blockDim.x, lane = t & 63;
  __syncthreads();
  if (on)
#pragma unroll
    for (int a = 0; a < NA; a++)
#pragma unroll
      for (int k = 0; k < VW; k++) lds[(a * VW + k) * threads + t] = v[a][k];
  __syncthreads();
  float s[NA];
  if (rows >= 32) {
    for (int ch = __builtin_amdgcn_readfirstlane(t >> 6); ch < cols * VW; ch += threads >> 6) {
#pragma unroll
      for (int a = 0; a < NA; a++) s[a] = 0.f;
      for (int r = lane; r < rows; r += 64)
#pragma unroll
        for (int a = 0; a < NA; a++) s[a] += lds[(a * VW + ch % VW) * threads + r * cols + ch / VW];
#pragma unroll
      for (int m = 1; m < 64; m <<= 1)
#pragma unroll
        for (int a = 0; a < NA; a++) s[a] += __shfl_xor(s[a], m);
      if (lane == 0) sink(ch, s);
    }
  } else {
    for (int ch = t; ch < cols * VW; ch += threads) {
#pragma unroll
      for (int a = 0; a < NA; a++) s[a] = 0.f;
      for (int r = 0; r < rows; r++)
#pragma unroll
        for (int a = 0; a < NA; a++) s[a] += lds[(a * VW + ch % VW) * threads + r * cols + ch / VW];
      sink(ch, s);
    }
  }
}

// Blocks are dealt to the 8 XCDs in turn; neighbouring groups share memory lines, so they are given to one XCD.
__device__ __forceinline__ int64_t xcd_unit(int64_t b, int64_t total) {
  const int64_t per = total / 8;
  return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}

// ------------------------------------------------------------------ units held by one block
// A thread holds up to `hold` vectors; with 8 channels a vector the backward kernel needs 6 x (4 + 4 + 8) registers and
// as much for the channels' constants and sums: a few more than the 168 that 768 threads have (it spills 40 bytes a lane, the
// bundles' 80), and far more than the 128 of 1024.
constexpr int max_threads(bool bwd, int vw) { return bwd && vw == 8 ? 768 : 1024; }
constexpr int max_hold(bool bwd, int vw) { return vw == 8 ? (bwd ? 6 : 8) : bwd ? 8 : 16; }

template <typename T, int VW, int VPT, bool BWD>
__global__ __launch_bounds__(max_threads(BWD, VW)) void k_gn_block(GnArgs A) {
  __shared__ float red[16][2];
  extern __shared__ float cols[];  // 2 VW floats a thread in the backward kernel
  const int64_t u = xcd_unit(blockIdx.x, A.N * A.G);
  const int64_t n = u / A.G;
  const int g = (int)(u % A.G), t = threadIdx.x;
  const int cgv = A.cg / VW, rp = (int)blockDim.x / cgv;
  const bool on = t < rp * cgv;
  const int r0 = t / cgv, col = (on ? t - r0 * cgv : 0) * VW, c = g * A.cg + col;
  const float count = (float)A.L * (float)A.cg, inv = 1.f / count;
  Pack<T, VW> xv[VPT], dv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++) {
    const int64_t row = r0 + (int64_t)rp * i;
    if (on && row < A.L) {
      xv[i] = *(const Pack<T, VW>*)((const T*)A.x.p + n * A.x.sn + row * A.x.sl + c);
      if constexpr (BWD) dv[i] = *(const Pack<T, VW>*)((const T*)A.dy.p + n * A.dy.sn + row * A.dy.sl + c);
    }
  }
  auto have = [&](int i) { return on && r0 + (int64_t)rp * i < A.L; };
  float w[VW], b[VW];
#pragma unroll
  for (int k = 0; k < VW; k++) {
    w[k] = param(A.w, A.wdt, c + k, 1.f);
    b[k] = param(A.b, A.wdt, c + k, 0.f);
  }
  float v[2] = {0.f, 0.f}, mean, r;
  if (BWD && A.stats) {
    mean = A.stats[2 * u];
    r = A.stats[2 * u + 1];
  } else {
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) v[0] += to_f32(xv[i].e[k]);
    block_sum<2>(v, red);
    mean = v[0] / count;  // (of equal numbers: that number)
    v[0] = v[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float d = to_f32(xv[i].e[k]) - mean;
          v[0] = fmaf(d, d, v[0]);
        }
    block_sum<2>(v, red);
    r = inv_sqrt(v[0] * inv + A.eps);
    if (A.stats && t == 0) {
      A.stats[2 * u] = mean;
      A.stats[2 * u + 1] = r;
    }
  }
  if constexpr (!BWD) {  // z = (x - mean) (r w) + b; never x (r w) + (b - mean r w): r is up to 1 / sqrt(eps)
#pragma unroll
    for (int k = 0; k < VW; k++) w[k] *= r;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++)
          y[k] = act_value<T>(fmaf(to_f32(xv[i].e[k]) - mean, w[k], b[k]), A.act);
        store_vec<T, VW>((T*)A.y.p + n * A.y.sn + (r0 + (int64_t)rp * i) * A.y.sl + c, y);
      }
  } else {
    float sum[2][VW], d[VPT][VW];  // of dweight and dbias
#pragma unroll
    for (int k = 0; k < VW; k++) sum[0][k] = sum[1][k] = 0.f;
    v[0] = v[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float xh = (to_f32(xv[i].e[k]) - mean) * r;
          const float dz = to_f32(dv[i].e[k]) * act_slope<T>(fmaf(xh, w[k], b[k]), A.act);
          sum[1][k] += dz;
          sum[0][k] = fmaf(dz, xh, sum[0][k]);
          d[i][k] = dz * w[k];
          v[0] += d[i][k];
          v[1] = fmaf(d[i][k], xh, v[1]);
        }
    block_sum<2>(v, red);
    const float s1 = -r * (v[0] * inv), s2 = -r * (v[1] * inv);
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++)
          y[k] = fmaf(d[i][k], r, fmaf((to_f32(xv[i].e[k]) - mean) * r, s2, s1));
        store_vec<T, VW>((T*)A.dx.p + n * A.dx.sn + (r0 + (int64_t)rp * i) * A.dx.sl + c, y);
      }
    if (A.dw || A.db)
      channel_sums<VW, 2>(sum, t, rp, cgv, on, cols, [&](int ch, const float* s) {
        if (A.dw) A.dw[u * A.cg + ch] = s[0];
        if (A.db) A.db[u * A.cg + ch] = s[1];
      });
  }
}

// ------------------------------------------------------------------ several units held by one block
// Where a group's channels do not fill 16-byte vectors, a block takes `bundle` neighbouring groups that together do.  A
// vector's channels may then belong to different groups, so sums are kept per channel and joined per group at the end;
// the backward pass needs the sums per channel anyway.
template <typename T, int VPT, bool BWD>
__global__ __launch_bounds__(max_threads(BWD, 16 / sizeof(T))) void k_gn_bundle(GnArgs A, int bundle) {
  constexpr int VW = 16 / sizeof(T);
  extern __shared__ float lds[];  // VW (backward 2 VW) floats a thread
  __shared__ float chan[2][1024], group[2][64];
  const int64_t u = xcd_unit(blockIdx.x, A.N * A.G / bundle);
  const int64_t n = u / (A.G / bundle);
  const int g0 = (int)(u % (A.G / bundle)) * bundle, t = threadIdx.x, width = bundle * A.cg;
  const int cols = width / VW, rp = (int)blockDim.x / cols;
  const bool on = t < rp * cols;
  const int r0 = t / cols, col = (on ? t - r0 * cols : 0) * VW, c = g0 * A.cg + col;
  const float count = (float)A.L * (float)A.cg, inv = 1.f / count;
  auto have = [&](int i) { return on && r0 + (int64_t)rp * i < A.L; };
  Pack<T, VW> xv[VPT], dv[VPT];
#pragma unroll
  for (int i = 0; i < VPT; i++)
    if (have(i)) {
      const int64_t row = r0 + (int64_t)rp * i;
      xv[i] = *(const Pack<T, VW>*)((const T*)A.x.p + n * A.x.sn + row * A.x.sl + c);
      if constexpr (BWD) dv[i] = *(const Pack<T, VW>*)((const T*)A.dy.p + n * A.dy.sn + row * A.dy.sl + c);
    }
  int gi[VW];
#pragma unroll
  for (int k = 0; k < VW; k++) gi[k] = (col + k) / A.cg;
  // the channels' sums, and on every thread the groups' from them (weighted: of w times the channel's)
  auto group_sums = [&](const auto& v, int first, bool weighted) {
    constexpr int NA = std::extent_v<std::remove_reference_t<decltype(v)>, 0>;
    channel_sums<VW, NA>(v, t, rp, cols, on, lds, [&](int ch, const float* s) {
#pragma unroll
      for (int a = 0; a < NA; a++) chan[first + a][ch] = s[a];
    });
    __syncthreads();
    if (t < bundle * NA) {
      const int a = first + t / bundle, g = t % bundle;
      float s = 0.f;
      for (int k = g * A.cg; k < (g + 1) * A.cg; k++)
        s = fmaf(chan[a][k], weighted ? param(A.w, A.wdt, g0 * A.cg + k, 1.f) : 1.f, s);
      group[a][g] = s;
    }
    __syncthreads();
  };
  float v[1][VW], mean[VW], r[VW], w[VW], b[VW];
#pragma unroll
  for (int k = 0; k < VW; k++) {
    w[k] = param(A.w, A.wdt, c + k, 1.f);
    b[k] = param(A.b, A.wdt, c + k, 0.f);
  }
  if (BWD && A.stats) {
#pragma unroll
    for (int k = 0; k < VW; k++) {
      mean[k] = A.stats[2 * (n * A.G + g0 + gi[k])];
      r[k] = A.stats[2 * (n * A.G + g0 + gi[k]) + 1];
    }
  } else {
#pragma unroll
    for (int k = 0; k < VW; k++) v[0][k] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) v[0][k] += to_f32(xv[i].e[k]);
    group_sums(v, 0, false);
#pragma unroll
    for (int k = 0; k < VW; k++) {
      mean[k] = group[0][gi[k]] / count;  // (of equal numbers: that number)
      v[0][k] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float d = to_f32(xv[i].e[k]) - mean[k];
          v[0][k] = fmaf(d, d, v[0][k]);
        }
    group_sums(v, 1, false);
#pragma unroll
    for (int k = 0; k < VW; k++) r[k] = inv_sqrt(group[1][gi[k]] * inv + A.eps);
    if (A.stats && t < bundle) {
      A.stats[2 * (n * A.G + g0 + t)] = group[0][t] / count;
      A.stats[2 * (n * A.G + g0 + t) + 1] = inv_sqrt(group[1][t] * inv + A.eps);
    }
  }
  if constexpr (!BWD) {
#pragma unroll
    for (int k = 0; k < VW; k++) w[k] *= r[k];  // z = (x - mean) (r w) + b
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++)
          y[k] = act_value<T>(fmaf(to_f32(xv[i].e[k]) - mean[k], w[k], b[k]), A.act);
        store_vec<T, VW>((T*)A.y.p + n * A.y.sn + (r0 + (int64_t)rp * i) * A.y.sl + c, y);
      }
  } else {
    float sum[2][VW], d[VPT][VW];  // of dbias and dweight
#pragma unroll
    for (int k = 0; k < VW; k++) sum[0][k] = sum[1][k] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float xh = (to_f32(xv[i].e[k]) - mean[k]) * r[k];
          d[i][k] = to_f32(dv[i].e[k]) * act_slope<T>(fmaf(xh, w[k], b[k]), A.act);
          sum[0][k] += d[i][k];
          sum[1][k] = fmaf(d[i][k], xh, sum[1][k]);
        }
    group_sums(sum, 0, true);  // sum dxh = sum w db, sum dxh xh = sum w dw
    for (int ch = t; ch < width; ch += (int)blockDim.x) {
      if (A.db) A.db[n * A.G * A.cg + g0 * A.cg + ch] = chan[0][ch];
      if (A.dw) A.dw[n * A.G * A.cg + g0 * A.cg + ch] = chan[1][ch];
    }
    float s1[VW], s2[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      s1[k] = -r[k] * (group[0][gi[k]] * inv);
      s2[k] = -r[k] * (group[1][gi[k]] * inv);
      w[k] *= r[k];
    }
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++)
          y[k] = fmaf(d[i][k], w[k], fmaf((to_f32(xv[i].e[k]) - mean[k]) * r[k], s2[k], s1[k]));
        store_vec<T, VW>((T*)A.dx.p + n * A.dx.sn + (r0 + (int64_t)rp * i) * A.dx.sl + c, y);
      }
  }
}

// ------------------------------------------------------------------ streams over whole rows
// Two passes over the tensor, each a plain stream: a block takes some rows of a sample and all its channels (256 vectors
// at a time, so that a thread keeps its channels), and leaves sums per group (and, backward, per channel); these are
// joined, and the second pass applies them.

// (count, mean, sum of squared deviations) of two sets joined
__device__ __forceinline__ void join(float& n, float& m, float& q, float n2, float m2, float q2) {
  if (n2 == 0.f) return;
  const float t = n + n2, d = m2 - m, f = n2 * __builtin_amdgcn_rcpf(t);
  m = fmaf(d, f, m);
  q += q2 + d * (d * (n * f));  // (n may be 0, and d d infinite)
  n = t;
}

struct Part {
  int64_t n, l0, l1;
  int s;
};
__device__ __forceinline__ Part part_of(const GnArgs& A) {
  Part p;
  p.n = blockIdx.x / A.split;
  p.s = blockIdx.x % A.split;
  const int64_t per = (A.L + A.split - 1) / A.split;
  p.l0 = min(A.L, p.s * per);
  p.l1 = min(A.L, p.l0 + per);
  return p;
}
// this thread's place in a chunk of columns that begins with vector c0
struct Place {
  int cols, rp, r0, v;  // columns of the chunk, rows at a time, first row, vector
  bool on;
};
__device__ __forceinline__ Place place_of(int vectors, int c0) {
  Place p;
  p.cols = min(256, vectors - c0);
  p.rp = 256 / p.cols;
  p.r0 = (int)threadIdx.x / p.cols;
  p.on = p.r0 < p.rp;
  p.v = c0 + (int)threadIdx.x % p.cols;
  return p;
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_stream_stats(GnArgs A) {
  __shared__ float lds[3][VW][256];
  const Part p = part_of(A);
  const int C = A.G * A.cg, t = threadIdx.x;
  float* out = A.sums + (p.n * A.split + p.s) * A.G * 3;
  for (int c0 = 0; c0 < C / VW; c0 += 256) {
    const Place at = place_of(C / VW, c0);
    // per channel and thread: running mean and squared deviations
    float n = 0.f, m[VW], q[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) m[k] = q[k] = 0.f;
    const T* x = (const T*)A.x.p + p.n * A.x.sn + at.v * VW;
    if (at.on) {
      constexpr int B = 4;  // rows in flight
      for (int64_t l = p.l0 + at.r0; l < p.l1; l += (int64_t)at.rp * B) {
        float v[B][VW];
#pragma unroll
        for (int i = 0; i < B; i++) load_vec<T, VW>(x + min(l + (int64_t)at.rp * i, p.l1 - 1) * A.x.sl, v[i]);
#pragma unroll
        for (int i = 0; i < B; i++)
          if (l + (int64_t)at.rp * i < p.l1) {
            n += 1.f;
            const float f = __builtin_amdgcn_rcpf(n);
#pragma unroll
            for (int k = 0; k < VW; k++) {
              const float d = v[i][k] - m[k];
              m[k] = fmaf(d, f, m[k]);
              q[k] = fmaf(d, v[i][k] - m[k], q[k]);
            }
          }
      }
    }
    // over the threads of a column, in a fixed order
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VW; k++) {
      lds[0][k][t] = n;
      lds[1][k][t] = m[k];
      lds[2][k][t] = q[k];
    }
    __syncthreads();
    for (int rows = at.rp; rows > 1; rows = (rows + 1) >> 1) {
      const int other = t + ((rows + 1) >> 1) * at.cols;
      if (at.on && t < (rows >> 1) * at.cols)
#pragma unroll
        for (int k = 0; k < VW; k++)
          join(lds[0][k][t], lds[1][k][t], lds[2][k][t], lds[0][k][other], lds[1][k][other], lds[2][k][other]);
      __syncthreads();
    }
    // over the channels of a group; a group that began in the chunk before goes on
    const int g0 = c0 * VW / A.cg, g1 = ((c0 + at.cols) * VW - 1) / A.cg;
    for (int g = g0 + t; g <= g1; g += 256) {
      float n = 0.f, m = 0.f, q = 0.f;
      if (g * A.cg < c0 * VW) {
        n = out[3 * g];
        m = out[3 * g + 1];
        q = out[3 * g + 2];
      }
      const int first = max(g * A.cg, c0 * VW), last = min((g + 1) * A.cg, (c0 + at.cols) * VW);
      for (int c = first; c < last; c++) {
        const int v = c / VW - c0, k = c % VW;
        join(n, m, q, lds[0][k][v], lds[1][k][v], lds[2][k][v]);
      }
      out[3 * g] = n;
      out[3 * g + 1] = m;
      out[3 * g + 2] = q;
    }
    __syncthreads();
  }
}

// The parts of a sample's group joined, one wave each, in a fixed order: its mean and 1 / sqrt(var + eps), or (BWD) the
// means of dxh and of dxh xh.
template <bool BWD>
__global__ __launch_bounds__(256) void k_gn_stream_join(GnArgs A, float* out) {
  const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (u >= A.N * A.G) return;
  float n = 0.f, m = 0.f, q = 0.f;
  for (int s = lane; s < A.split; s += 64) {
    const float* o = A.sums + ((u / A.G * A.split + s) * A.G + u % A.G) * 3;
    if constexpr (BWD) {
      m += o[0];
      q += o[1];
    } else {
      join(n, m, q, o[0], o[1], o[2]);
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const float n2 = __shfl_down(n, d), m2 = __shfl_down(m, d), q2 = __shfl_down(q, d);
    if constexpr (BWD) {
      m += m2;
      q += q2;
    } else {
      join(n, m, q, n2, m2, q2);
    }
  }
  if (lane == 0) {
    const float inv = 1.f / ((float)A.L * (float)A.cg);
    out[2 * u] = BWD ? m * inv : m;
    out[2 * u + 1] = BWD ? q * inv : inv_sqrt(q * inv + A.eps);
  }
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_stream_apply(GnArgs A) {
  const Part p = part_of(A);
  const int C = A.G * A.cg;
  for (int c0 = 0; c0 < C / VW; c0 += 256) {
    const Place at = place_of(C / VW, c0);
    if (!at.on) continue;
    const int c = at.v * VW;
    float m[VW], w[VW], b[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      const int64_t g = p.n * A.G + (c + k) / A.cg;
      m[k] = A.stats[2 * g];
      w[k] = A.stats[2 * g + 1] * param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
    }
    const T* x = (const T*)A.x.p + p.n * A.x.sn + c;
    T* y = (T*)A.y.p + p.n * A.y.sn + c;
    constexpr int B = 4;
    for (int64_t l = p.l0 + at.r0; l < p.l1; l += (int64_t)at.rp * B) {
      float v[B][VW];
#pragma unroll
      for (int i = 0; i < B; i++) load_vec<T, VW>(x + min(l + (int64_t)at.rp * i, p.l1 - 1) * A.x.sl, v[i]);
#pragma unroll
      for (int i = 0; i < B; i++)
        if (l + (int64_t)at.rp * i < p.l1) {
#pragma unroll
          for (int k = 0; k < VW; k++)
            v[i][k] = act_value<T>(fmaf(v[i][k] - m[k], w[k], b[k]), A.act);
          store_vec<T, VW>(y + (l + (int64_t)at.rp * i) * A.y.sl, v[i]);
        }
    }
  }
}

// backward: the sums of dz and dz xh per channel of a part, and of w dz and w dz xh per group
template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_stream_sums(GnArgs A) {
  __shared__ float lds[2][VW][256];
  const Part p = part_of(A);
  const int C = A.G * A.cg, t = threadIdx.x;
  float* out = A.sums + (p.n * A.split + p.s) * A.G * 3;
  for (int c0 = 0; c0 < C / VW; c0 += 256) {
    const Place at = place_of(C / VW, c0);
    const int c = at.v * VW;
    float m[VW], r[VW], w[VW], b[VW], dw[VW], db[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      const int64_t g = p.n * A.G + (c + k) / A.cg;
      m[k] = A.stats[2 * g];
      r[k] = A.stats[2 * g + 1];
      w[k] = param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
      dw[k] = db[k] = 0.f;
    }
    const T* x = (const T*)A.x.p + p.n * A.x.sn + c;
    const T* dy = (const T*)A.dy.p + p.n * A.dy.sn + c;
    if (at.on) {
      constexpr int B = 2;
      for (int64_t l = p.l0 + at.r0; l < p.l1; l += (int64_t)at.rp * B) {
        float v[B][VW], d[B][VW];
#pragma unroll
        for (int i = 0; i < B; i++) {
          const int64_t row = min(l + (int64_t)at.rp * i, p.l1 - 1);
          load_vec<T, VW>(x + row * A.x.sl, v[i]);
          load_vec<T, VW>(dy + row * A.dy.sl, d[i]);
        }
#pragma unroll
        for (int i = 0; i < B; i++)
          if (l + (int64_t)at.rp * i < p.l1)
#pragma unroll
            for (int k = 0; k < VW; k++) {
              const float xh = (v[i][k] - m[k]) * r[k], dz = d[i][k] * act_slope<T>(fmaf(xh, w[k], b[k]), A.act);
              db[k] += dz;
              dw[k] = fmaf(dz, xh, dw[k]);
            }
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < VW; k++) {
      lds[0][k][t] = db[k];
      lds[1][k][t] = dw[k];
    }
    __syncthreads();
    for (int rows = at.rp; rows > 1; rows = (rows + 1) >> 1) {
      const int other = t + ((rows + 1) >> 1) * at.cols;
      if (at.on && t < (rows >> 1) * at.cols)
#pragma unroll
        for (int k = 0; k < VW; k++) {
          lds[0][k][t] += lds[0][k][other];
          lds[1][k][t] += lds[1][k][other];
        }
      __syncthreads();
    }
    if (t < at.cols)
#pragma unroll
      for (int k = 0; k < VW; k++) {
        const int64_t o = (p.n * A.split + p.s) * C + c + k;
        if (A.db) A.db[o] = lds[0][k][t];
        if (A.dw) A.dw[o] = lds[1][k][t];
        lds[0][k][t] *= w[k];
        lds[1][k][t] *= w[k];
      }
    __syncthreads();
    const int g0 = c0 * VW / A.cg, g1 = ((c0 + at.cols) * VW - 1) / A.cg;
    for (int g = g0 + t; g <= g1; g += 256) {
      const bool begun = g * A.cg < c0 * VW;
      float s1 = begun ? out[3 * g] : 0.f, s2 = begun ? out[3 * g + 1] : 0.f;
      const int first = max(g * A.cg, c0 * VW), last = min((g + 1) * A.cg, (c0 + at.cols) * VW);
      for (int ch = first; ch < last; ch++) {
        s1 += lds[0][ch % VW][ch / VW - c0];
        s2 += lds[1][ch % VW][ch / VW - c0];
      }
      out[3 * g] = s1;
      out[3 * g + 1] = s2;
    }
    __syncthreads();
  }
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_stream_dx(GnArgs A, const float* means) {
  const Part p = part_of(A);
  const int C = A.G * A.cg;
  for (int c0 = 0; c0 < C / VW; c0 += 256) {
    const Place at = place_of(C / VW, c0);
    if (!at.on) continue;
    const int c = at.v * VW;
    float m[VW], r[VW], w[VW], b[VW], s1[VW], s2[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      const int64_t g = p.n * A.G + (c + k) / A.cg;
      m[k] = A.stats[2 * g];
      r[k] = A.stats[2 * g + 1];
      s1[k] = means[2 * g];
      s2[k] = means[2 * g + 1];
      w[k] = param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
    }
    const T* x = (const T*)A.x.p + p.n * A.x.sn + c;
    const T* dy = (const T*)A.dy.p + p.n * A.dy.sn + c;
    T* dx = (T*)A.dx.p + p.n * A.dx.sn + c;
    constexpr int B = 2;
    for (int64_t l = p.l0 + at.r0; l < p.l1; l += (int64_t)at.rp * B) {
      float v[B][VW], d[B][VW];
#pragma unroll
      for (int i = 0; i < B; i++) {
        const int64_t row = min(l + (int64_t)at.rp * i, p.l1 - 1);
        load_vec<T, VW>(x + row * A.x.sl, v[i]);
        load_vec<T, VW>(dy + row * A.dy.sl, d[i]);
      }
#pragma unroll
      for (int i = 0; i < B; i++)
        if (l + (int64_t)at.rp * i < p.l1) {
#pragma unroll
          for (int k = 0; k < VW; k++) {
            const float xh = (v[i][k] - m[k]) * r[k];
            const float dxh = d[i][k] * act_slope<T>(fmaf(xh, w[k], b[k]), A.act) * w[k];
            v[i][k] = r[k] * (dxh - s1[k] - xh * s2[k]);
          }
          store_vec<T, VW>(dx + (l + (int64_t)at.rp * i) * A.dx.sl, v[i]);
        }
    }
  }
}

// dweight / dbias: part [R][C] -> [C].  A block takes 16 channels with 64 threads each, in a fixed order.
__global__ __launch_bounds__(1024) void k_gn_params(const float* dw, const float* db, int64_t R, int C, void* ow,
                                                    void* ob, int wdt) {
  __shared__ double lds[64][17];
  const float* part = blockIdx.y ? db : dw;
  void* out = blockIdx.y ? ob : ow;
  if (!out) return;
  const int k = threadIdx.x & 15, q = threadIdx.x >> 4, c = blockIdx.x * 16 + k;
  double s = 0.0;
  if (c < C) {
#pragma unroll 4
    for (int64_t a = q; a < R; a += 64) s += part[a * C + c];
  }
  lds[q][k] = s;
  __syncthreads();
  if (q == 0 && c < C) {
    s = 0.0;
    for (int i = 0; i < 64; i++) s += lds[i][k];
    if (wdt == FW_DT_F32)
      ((float*)out)[c] = (float)s;
    else if (wdt == FW_DT_BF16)
      ((bf16*)out)[c] = from_f32<bf16>((float)s);
    else
      ((f16*)out)[c] = from_f32<f16>((float)s);
  }
}

// ------------------------------------------------------------------ host side
enum { WAVE, BLOCK, BUNDLE, STREAM };
struct Plan {
  int kind, vw, per, lanes_log2, threads, split, bundle;
  int64_t grid, R;  // R: rows of partial sums
};

// the widest vector that fits runs of `cg` channels and every tensor's alignment
int vector_width(const fw_group_norm* a, bool backward, int64_t cg) {
  const int e = a->dtype == FW_DT_F32 ? 4 : 2;
  int vw = 16 / e;
  auto fits = [&](const fw_rows& r) {
    return (uintptr_t)r.p % (vw * e) == 0 && (r.sn % vw == 0 || a->N < 2) && (r.sl % vw == 0 || a->L < 2);
  };
  while (vw > 1 && !(cg % vw == 0 && fits(a->x) && (backward ? fits(a->dy) && fits(a->dx) : fits(a->y)))) vw /= 2;
  return vw;
}
int64_t gcd64(int64_t a, int64_t b) { return b ? gcd64(b, a % b) : a; }

// Statistics are kept wherever a unit may be too large for a block (with vectors of one channel: 1024 columns, or 8
// rows of more than 512); their traffic is nothing beside such a unit's.
bool needs_stats(const fw_group_norm* a) { return a->L * (a->C / a->G) > 1024; }

Plan plan(const fw_group_norm* a, bool backward) {
  Plan p{};
  const int64_t cg = a->C / a->G, units = a->N * a->G;
  p.vw = vector_width(a, backward, cg);
  const int64_t cgv = cg / p.vw, vecs = a->L * cgv;
  if (vecs <= 64 * 4) {
    p.kind = WAVE;
    while ((int64_t)1 << p.lanes_log2 < vecs && p.lanes_log2 < 6) p.lanes_log2++;
    const int64_t per_lane = (vecs + (1 << p.lanes_log2) - 1) >> p.lanes_log2;
    p.per = per_lane <= 1 ? 1 : per_lane <= 2 ? 2 : 4;
    const int64_t slots_per_block = 4 * (64 >> p.lanes_log2);
    const int64_t quantum = a->G / gcd64(a->G, slots_per_block);  // blocks whose slots are a multiple of G
    const int64_t want = std::min<int64_t>((units + slots_per_block - 1) / slots_per_block, backward ? 1024 : 2048);
    p.grid = std::max<int64_t>(quantum, (want + quantum - 1) / quantum * quantum);
    p.R = slots_per_block % a->G == 0 ? p.grid : p.grid * slots_per_block / a->G;
    return p;
  }
  // the fewest threads that hold `cols` columns of vectors, with at most `hold` each; 0 if none do
  auto block_of = [&](int64_t cols, int vw, int hold) {
    for (int threads : {256, 512, 768, 1024})
      if (threads <= max_threads(backward, vw) && cols <= threads && (a->L + threads / cols - 1) / (threads / cols) <= hold) {
        p.threads = threads;
        const int64_t per = (a->L + threads / cols - 1) / (threads / cols);
        p.per = 2 * per <= hold ? hold / 2 : hold;
        return true;
      }
    return false;
  };
  // a block for the fewest neighbouring groups that fill 16-byte vectors, where one group does not
  const int full = a->dtype == FW_DT_F32 ? 4 : 8;
  if (p.vw < full)
    for (int64_t q = 2; q <= 32 && q * cg <= 1024; q++)
      if (a->G % q == 0 && q * cg % full == 0) {
        if (vector_width(a, backward, q * cg) < full || !block_of(q * cg / full, full, backward && full == 8 ? 6 : 8)) break;
        p.kind = BUNDLE;
        p.bundle = (int)q;
        p.grid = units / q;
        p.R = a->N;
        return p;
      }
  if (block_of(cgv, p.vw, max_hold(backward, p.vw))) {
    p.kind = BLOCK;
    p.grid = units;
    p.R = a->N;
    return p;
  }
  p.kind = STREAM;
  p.vw = vector_width(a, backward, a->C);
  // about 1024 blocks of at least 16 KB each
  const int64_t bytes = a->L * a->C * (a->dtype == FW_DT_F32 ? 4 : 2);
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>({(1024 + a->N - 1) / a->N, bytes / 16384, a->L, 256}));
  p.grid = a->N * p.split;
  p.R = a->N * p.split;
  return p;
}
size_t part_floats(const fw_group_norm* a, const Plan& p) { return (size_t)p.R * a->C; }
size_t sum_floats(const fw_group_norm* a, const Plan& p) {
  return p.kind == STREAM ? (size_t)a->N * a->G * (p.split * 3 + 2) : 0;
}

template <typename T, int VW, bool BWD>
int launch(const GnArgs& A, const Plan& p, hipStream_t s) {
  if (p.grid > UINT32_MAX / (p.kind == BLOCK || p.kind == BUNDLE ? p.threads : 256))  // threads of a launch
    return fw::set_error(FW_E_INVALID, "group norm: too many groups for one call");
  const dim3 grid((unsigned)p.grid);
  if (p.kind == WAVE) {
    const size_t lds = BWD ? (size_t)4 * (64 >> p.lanes_log2) * A.L * A.cg * sizeof(float) : 0;  // at most 32 KB
    if (p.per == 1)
      hipLaunchKernelGGL((k_gn_wave<T, VW, 1, BWD>), grid, dim3(256), lds, s, A);
    else if (p.per == 2)
      hipLaunchKernelGGL((k_gn_wave<T, VW, 2, BWD>), grid, dim3(256), lds, s, A);
    else
      hipLaunchKernelGGL((k_gn_wave<T, VW, 4, BWD>), grid, dim3(256), lds, s, A);
  } else if (p.kind == BLOCK) {
    const size_t lds = BWD ? 2 * VW * p.threads * sizeof(float) : 0;  // at most 48 KB
    constexpr int HOLD = max_hold(BWD, VW);
    if (p.per < HOLD)
      hipLaunchKernelGGL((k_gn_block<T, VW, HOLD / 2, BWD>), grid, dim3(p.threads), lds, s, A);
    else
      hipLaunchKernelGGL((k_gn_block<T, VW, HOLD, BWD>), grid, dim3(p.threads), lds, s, A);
  } else if (p.kind == BUNDLE) {
    const size_t lds = (BWD ? 2 : 1) * 16 / sizeof(T) * p.threads * sizeof(float);  // at most 48 KB
    constexpr int HOLD = BWD && sizeof(T) == 2 ? 6 : 8;
    if (p.per < HOLD)
      hipLaunchKernelGGL((k_gn_bundle<T, HOLD / 2, BWD>), grid, dim3(p.threads), lds, s, A, p.bundle);
    else
      hipLaunchKernelGGL((k_gn_bundle<T, HOLD, BWD>), grid, dim3(p.threads), lds, s, A, p.bundle);
  } else {
    const dim3 joins((unsigned)((A.N * A.G + 3) / 4));
    float* pairs = A.sums + A.N * A.G * A.split * 3;  // [N][G][2]
    if constexpr (!BWD) {
      GnArgs B = A;
      if (!B.stats) B.stats = pairs;
      hipLaunchKernelGGL((k_gn_stream_stats<T, VW>), grid, dim3(256), 0, s, A);
      FW_HIP(hipGetLastError());
      hipLaunchKernelGGL((k_gn_stream_join<false>), joins, dim3(256), 0, s, A, B.stats);
      FW_HIP(hipGetLastError());
      hipLaunchKernelGGL((k_gn_stream_apply<T, VW>), grid, dim3(256), 0, s, B);
    } else {
      hipLaunchKernelGGL((k_gn_stream_sums<T, VW>), grid, dim3(256), 0, s, A);
      FW_HIP(hipGetLastError());
      hipLaunchKernelGGL((k_gn_stream_join<true>), joins, dim3(256), 0, s, A, pairs);
      FW_HIP(hipGetLastError());
      hipLaunchKernelGGL((k_gn_stream_dx<T, VW>), grid, dim3(256), 0, s, A, (const float*)pairs);
    }
  }
  FW_HIP(hipGetLastError());
  return FW_OK;
}
template <typename T, bool BWD>
int launch_vw(const GnArgs& A, const Plan& p, hipStream_t s) {
  if (p.vw == 1) return launch<T, 1, BWD>(A, p, s);
  if (p.vw == 2) return launch<T, 2, BWD>(A, p, s);
  if (p.vw == 4) return launch<T, 4, BWD>(A, p, s);
  if constexpr (sizeof(T) == 2) return launch<T, 8, BWD>(A, p, s);
  return fw::set_error(FW_E_INVALID, "group norm: vector width");
}
template <bool BWD>
int launch_dt(const fw_group_norm* a, const GnArgs& A, const Plan& p, hipStream_t s) {
  if (a->dtype == FW_DT_F32) return launch_vw<float, BWD>(A, p, s);
  if (a->dtype == FW_DT_BF16) return launch_vw<bf16, BWD>(A, p, s);
  return launch_vw<f16, BWD>(A, p, s);
}

int check(const fw_group_norm* a, const char* who) {
  auto bad = [&](const char* m) { return fw::set_error(FW_E_INVALID, std::string(who) + ": " + m); };
  if (!a) return bad("NULL arguments");
  if (a->N < 0 || a->L < 0 || a->C < 1 || a->G < 1 || a->C % a->G) return bad("C must be a positive multiple of G >= 1");
  if (a->dtype < FW_DT_F32 || a->dtype > FW_DT_F16) return bad("dtype must be float32, bfloat16 or float16");
  if (a->wdtype != FW_DT_F32 && a->wdtype != a->dtype) return bad("wdtype must be float32 or dtype");
  if (a->act < FW_ACT_NONE || a->act > FW_ACT_TANH) return bad("unknown activation");
  if (!(a->eps >= 0.0)) return bad("eps must be >= 0");
  if (a->N > INT32_MAX / a->G) return bad("too many groups for one call");
  return FW_OK;
}
GnArgs base(const fw_group_norm* a, const Plan& p) {
  GnArgs A{};
  auto rows = [](const fw_rows& r) { return Rows{r.p, r.sn, r.sl}; };
  A.x = rows(a->x);
  A.y = rows(a->y);
  A.dy = rows(a->dy);
  A.dx = rows(a->dx);
  A.w = a->weight;
  A.b = a->bias;
  A.N = a->N;
  A.L = a->L;
  A.G = a->G;
  A.cg = a->C / a->G;
  A.wdt = a->wdtype;
  A.act = a->act;
  A.split = p.split;
  A.lanes_log2 = p.lanes_log2;
  A.eps = (float)a->eps;
  A.stats = a->stats;
  A.sums = (float*)a->workspace;
  return A;
}

}  // namespace

extern "C" {

int fw_group_norm_stats(const fw_group_norm* a) { return a && a->G > 0 && needs_stats(a); }

size_t fw_group_norm_workspace_bytes(const fw_group_norm* a, int32_t backward) {
  if (!a || a->N < 1 || a->L < 1 || a->C < 1 || a->G < 1 || a->C % a->G) return 0;
  const Plan p = plan(a, backward);
  return sizeof(float) * (sum_floats(a, p) + (backward ? 2 * part_floats(a, p) : 0));
}

int fw_group_norm_forward(const fw_group_norm* a, void* stream) {
  if (int rc = check(a, "fw_group_norm_forward")) return rc;
  if (a->N == 0 || a->L == 0) return FW_OK;
  if (!a->x.p || !a->y.p) return fw::set_error(FW_E_INVALID, "fw_group_norm_forward: NULL x or y");
  const Plan p = plan(a, false);
  const size_t need = fw_group_norm_workspace_bytes(a, 0);
  if (need && (!a->workspace || a->workspace_bytes < need))
    return fw::set_error(FW_E_INVALID, "fw_group_norm_forward: workspace too small");
  return launch_dt<false>(a, base(a, p), p, (hipStream_t)stream);
}

int fw_group_norm_backward(const fw_group_norm* a, void* stream) {
  if (int rc = check(a, "fw_group_norm_backward")) return rc;
  if (a->N == 0 || a->L == 0) return fw::set_error(FW_E_INVALID, "fw_group_norm_backward: empty");
  if (!a->x.p || !a->dy.p || !a->dx.p) return fw::set_error(FW_E_INVALID, "fw_group_norm_backward: NULL x, dy or dx");
  const Plan p = plan(a, true);
  if (p.kind == STREAM && !a->stats) return fw::set_error(FW_E_INVALID, "fw_group_norm_backward: stats needed");
  const size_t need = fw_group_norm_workspace_bytes(a, 1);
  if (need && (!a->workspace || a->workspace_bytes < need))
    return fw::set_error(FW_E_INVALID, "fw_group_norm_backward: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  GnArgs A = base(a, p);
  if (p.kind == WAVE) A.stats = nullptr;
  float* part = A.sums + sum_floats(a, p);
  A.dw = a->dweight ? part : nullptr;
  A.db = a->dbias ? part + part_floats(a, p) : nullptr;
  if (int rc = launch_dt<true>(a, A, p, s)) return rc;
  if (!A.dw && !A.db) return FW_OK;
  hipLaunchKernelGGL(k_gn_params, dim3((a->C + 15) / 16, 2), dim3(1024), 0, s, A.dw, A.db, p.R, a->C, a->dweight,
                     a->dbias, a->wdtype);
  FW_HIP(hipGetLastError());
  return FW_OK;
}

}  // extern "C"
