// fw_groupnorm.hip -- group norm with an activation over channels-last rows (include/fwrollout.h).
//
// A unit is one sample's group: L rows of cg = C / G adjacent channels, read as vectors of VW channels.  Three sizes:
//   k_gn_wave   a unit fits 64 lanes x 4 vectors: 2^k lanes per unit, several units per wave; for one row per sample
//               (a policy's features) this is a plain stream over the tensor
//   k_gn_block  a unit fits a block's registers: read once, written once
//   k_gn_*big   larger: statistics per part of the rows, joined by the blocks that apply them
// All statistics are sums of deviations from a mean, so a large mean does not cancel.  Memory bound: x in, y out (and
// dy in, dx out); the gradients of weight and bias are column sums of per-unit partial sums, in a fixed order.
#include <algorithm>

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
  float* sums;   // big: [N][G][split][3]
};

__device__ __forceinline__ float param(const void* p, int dt, int c, float none) {
  if (!p) return none;
  if (dt == FW_DT_F32) return ((const float*)p)[c];
  if (dt == FW_DT_BF16) return to_f32(((const bf16*)p)[c]);
  return to_f32(((const f16*)p)[c]);
}

constexpr float RSQRT2 = 0.70710678118654752f, RSQRT2PI = 0.39894228040143268f;

__device__ __forceinline__ float act_value(float z, int act) {
  switch (act) {
    case FW_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
    case FW_ACT_SILU: return z / (1.f + expf(-z));
    case FW_ACT_GELU: return 0.5f * z * erfcf(-z * RSQRT2);
    case FW_ACT_TANH: return tanhf(z);
  }
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case FW_ACT_RELU: return z > 0.f ? 1.f : 0.f;
    case FW_ACT_SILU: {
      const float s = 1.f / (1.f + expf(-z));
      return s * (1.f + z * (1.f - s));
    }
    case FW_ACT_GELU: return 0.5f * erfcf(-z * RSQRT2) + z * RSQRT2PI * expf(-0.5f * z * z);
    case FW_ACT_TANH: {
      const float t = tanhf(z);
      return 1.f - t * t;
    }
  }
  return 1.f;
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
  const float inv = 1.f / (float)(A.L * A.cg);
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
    const float mean = total_of(s) * inv;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; i++)
#pragma unroll
      for (int k = 0; k < VW; k++) {
        x[i][k] -= mean;
        s += ok[i] ? x[i][k] * x[i][k] : 0.f;
      }
    const float r = 1.f / sqrtf(total_of(s) * inv + A.eps);
    if constexpr (!BWD) {
      if (A.stats && live && sub == 0) {
        A.stats[2 * (n * A.G + g)] = mean;
        A.stats[2 * (n * A.G + g) + 1] = r;
      }
#pragma unroll
      for (int i = 0; i < VPL; i++) {
#pragma unroll
        for (int k = 0; k < VW; k++) x[i][k] = act_value(fmaf(x[i][k] * r, w[i][k], b[i][k]), A.act);
        if (ok[i] && live) store_vec<T, VW>((T*)A.y.p + n * A.y.sn + row[i] * A.y.sl + g * A.cg + col[i], x[i]);
      }
    } else {
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; i++)
#pragma unroll
        for (int k = 0; k < VW; k++) {
          x[i][k] *= r;
          const float dz = ok[i] && live ? dy[i][k] * act_slope(fmaf(x[i][k], w[i][k], b[i][k]), A.act) : 0.f;
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

// Sums v over the threads of equal column (thread = row * cols + column, `rows` rows), result on row 0.
template <int VW>
__device__ __forceinline__ void column_sum(float* v, int t, int rows, int cols, bool on, float* lds) {
  __syncthreads();
  if (on)
#pragma unroll
    for (int k = 0; k < VW; k++) lds[k * 1024 + t] = v[k];
  __syncthreads();
  while (rows > 1) {
    const int half = (rows + 1) >> 1;
    if (on && t < (rows - half) * cols)
#pragma unroll
      for (int k = 0; k < VW; k++) lds[k * 1024 + t] += lds[k * 1024 + t + half * cols];
    rows = half;
    __syncthreads();
  }
  if (on && t < cols)
#pragma unroll
    for (int k = 0; k < VW; k++) v[k] = lds[k * 1024 + t];
}

// Blocks are dealt to the 8 XCDs in turn; neighbouring groups share memory lines, so they are given to one XCD.
__device__ __forceinline__ int64_t xcd_unit(int64_t b, int64_t total) {
  const int64_t per = total / 8;
  return b < per * 8 ? (b & 7) * per + (b >> 3) : b;
}

// ------------------------------------------------------------------ units held by one block
template <typename T, int VW, int VPT, bool BWD>
__global__ __launch_bounds__(1024) void k_gn_block(GnArgs A) {
  __shared__ float red[16][2];
  extern __shared__ float cols[];  // VW * 1024 floats in the backward kernel
  const int64_t u = xcd_unit(blockIdx.x, A.N * A.G);
  const int64_t n = u / A.G;
  const int g = (int)(u % A.G), t = threadIdx.x;
  const int cgv = A.cg / VW, rp = (int)blockDim.x / cgv;
  const bool on = t < rp * cgv;
  const int r0 = t / cgv, col = (on ? t - r0 * cgv : 0) * VW, c = g * A.cg + col;
  const float inv = 1.f / ((float)A.L * (float)A.cg);
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
    mean = v[0] * inv;
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
    r = 1.f / sqrtf(v[0] * inv + A.eps);
    if (A.stats && t == 0) {
      A.stats[2 * u] = mean;
      A.stats[2 * u + 1] = r;
    }
  }
  float w[VW], b[VW];
#pragma unroll
  for (int k = 0; k < VW; k++) {
    w[k] = param(A.w, A.wdt, c + k, 1.f);
    b[k] = param(A.b, A.wdt, c + k, 0.f);
  }
  if constexpr (!BWD) {
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++) y[k] = act_value(fmaf((to_f32(xv[i].e[k]) - mean) * r, w[k], b[k]), A.act);
        store_vec<T, VW>((T*)A.y.p + n * A.y.sn + (r0 + (int64_t)rp * i) * A.y.sl + c, y);
      }
  } else {
    float dw[VW], db[VW], d[VPT][VW];
#pragma unroll
    for (int k = 0; k < VW; k++) dw[k] = db[k] = 0.f;
    v[0] = v[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i))
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float xh = (to_f32(xv[i].e[k]) - mean) * r;
          const float dz = to_f32(dv[i].e[k]) * act_slope(fmaf(xh, w[k], b[k]), A.act);
          db[k] += dz;
          dw[k] = fmaf(dz, xh, dw[k]);
          d[i][k] = dz * w[k];
          v[0] += d[i][k];
          v[1] = fmaf(d[i][k], xh, v[1]);
        }
    block_sum<2>(v, red);
    const float s1 = v[0] * inv, s2 = v[1] * inv;
#pragma unroll
    for (int i = 0; i < VPT; i++)
      if (have(i)) {
        float y[VW];
#pragma unroll
        for (int k = 0; k < VW; k++) y[k] = r * (d[i][k] - s1 - (to_f32(xv[i].e[k]) - mean) * r * s2);
        store_vec<T, VW>((T*)A.dx.p + n * A.dx.sn + (r0 + (int64_t)rp * i) * A.dx.sl + c, y);
      }
    if (A.dw) {
      column_sum<VW>(dw, t, rp, cgv, on, cols);
      if (t < cgv)
#pragma unroll
        for (int k = 0; k < VW; k++) A.dw[u * A.cg + col + k] = dw[k];
    }
    if (A.db) {
      column_sum<VW>(db, t, rp, cgv, on, cols);
      if (t < cgv)
#pragma unroll
        for (int k = 0; k < VW; k++) A.db[u * A.cg + col + k] = db[k];
    }
  }
}

// ------------------------------------------------------------------ units of any size
// (count, mean, sum of squared deviations) of two sets joined
__device__ __forceinline__ void join(float& n, float& m, float& q, float n2, float m2, float q2) {
  if (n2 == 0.f) return;
  const float t = n + n2, d = m2 - m;
  m = fmaf(d, n2 / t, m);
  q += q2 + d * d * (n * n2 / t);
  n = t;
}
// the same over a block, in a fixed order; the result on every thread
__device__ __forceinline__ void block_join(float& n, float& m, float& q, float (*lds)[3]) {
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) {
    const float n2 = __shfl_xor(n, s), m2 = __shfl_xor(m, s), q2 = __shfl_xor(q, s);
    // the lower lane's set first on both sides, so that both get the same bits
    if (threadIdx.x & s) {
      float a = n2, b = m2, c = q2;
      join(a, b, c, n, m, q);
      n = a;
      m = b;
      q = c;
    } else {
      join(n, m, q, n2, m2, q2);
    }
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lds[threadIdx.x >> 6][0] = n;
    lds[threadIdx.x >> 6][1] = m;
    lds[threadIdx.x >> 6][2] = q;
  }
  __syncthreads();
  n = m = q = 0.f;
  for (int w = 0; w < (int)blockDim.x / 64; w++) join(n, m, q, lds[w][0], lds[w][1], lds[w][2]);
}

// The part's rows [l0, l1), and for each column chunk f(row, column, i) with the column fixed for a thread.
struct Part {
  int64_t n, u, l0, l1;
  int g, s;
};
__device__ __forceinline__ Part part_of(const GnArgs& A) {
  Part p;
  const int64_t b = xcd_unit(blockIdx.x, A.N * A.G * A.split);
  // parts of neighbouring groups are neighbours: (n, s, g)
  p.g = (int)(b % A.G);
  p.s = (int)(b / A.G % A.split);
  p.n = b / A.G / A.split;
  p.u = p.n * A.G + p.g;
  const int64_t per = (A.L + A.split - 1) / A.split;
  p.l0 = min(A.L, p.s * per);
  p.l1 = min(A.L, p.l0 + per);
  return p;
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_big_stats(GnArgs A) {
  __shared__ float lds[4][3];
  const Part p = part_of(A);
  const int cgv = A.cg / VW, t = threadIdx.x;
  float n = 0.f, m = 0.f, q = 0.f;
  const int step = min(cgv, 256), rp = 256 / step;
  for (int c0 = 0; c0 < cgv; c0 += step) {
    const int cv = c0 + t % step;
    if (t >= rp * step || cv >= cgv) continue;
    const T* x = (const T*)A.x.p + p.n * A.x.sn + p.g * A.cg + cv * VW;
    constexpr int B = 4;  // rows at a time: exact deviations within, joined outside
    for (int64_t l = p.l0 + t / step; l < p.l1; l += (int64_t)rp * B) {
      float v[B][VW], s = 0.f, d2 = 0.f, cnt = 0.f;
#pragma unroll
      for (int i = 0; i < B; i++) {
        const int64_t row = l + (int64_t)rp * i;
        load_vec<T, VW>(x + min(row, p.l1 - 1) * A.x.sl, v[i]);
        if (row < p.l1) {
          cnt += VW;
#pragma unroll
          for (int k = 0; k < VW; k++) s += v[i][k];
        }
      }
      const float mm = s / cnt;
#pragma unroll
      for (int i = 0; i < B; i++)
        if (l + (int64_t)rp * i < p.l1)
#pragma unroll
          for (int k = 0; k < VW; k++) d2 = fmaf(v[i][k] - mm, v[i][k] - mm, d2);
      join(n, m, q, cnt, mm, d2);
    }
  }
  block_join(n, m, q, lds);
  if (t == 0) {
    float* o = A.sums + (p.u * A.split + p.s) * 3;
    o[0] = n;
    o[1] = m;
    o[2] = q;
  }
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_big_apply(GnArgs A) {
  const Part p = part_of(A);
  float n = 0.f, m = 0.f, q = 0.f;
  for (int s = 0; s < A.split; s++) {
    const float* o = A.sums + (p.u * A.split + s) * 3;
    join(n, m, q, o[0], o[1], o[2]);
  }
  const float r = 1.f / sqrtf(q / n + A.eps);
  const int cgv = A.cg / VW, t = threadIdx.x;
  if (A.stats && p.s == 0 && t == 0) {
    A.stats[2 * p.u] = m;
    A.stats[2 * p.u + 1] = r;
  }
  const int step = min(cgv, 256), rp = 256 / step;
  for (int c0 = 0; c0 < cgv; c0 += step) {
    const int cv = c0 + t % step;
    if (t >= rp * step || cv >= cgv) continue;
    const int c = p.g * A.cg + cv * VW;
    float w[VW], b[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      w[k] = param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
    }
    for (int64_t l = p.l0 + t / step; l < p.l1; l += rp) {
      float x[VW];
      load_vec<T, VW>((const T*)A.x.p + p.n * A.x.sn + l * A.x.sl + c, x);
#pragma unroll
      for (int k = 0; k < VW; k++) x[k] = act_value(fmaf((x[k] - m) * r, w[k], b[k]), A.act);
      store_vec<T, VW>((T*)A.y.p + p.n * A.y.sn + l * A.y.sl + c, x);
    }
  }
}

// backward: the two sums of a unit and the partial sums of the parameter gradients
template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_big_sums(GnArgs A) {
  __shared__ float red[16][2];
  extern __shared__ float cols[];
  const Part p = part_of(A);
  const int cgv = A.cg / VW, t = threadIdx.x;
  const float m = A.stats[2 * p.u], r = A.stats[2 * p.u + 1];
  float v[2] = {0.f, 0.f};
  const int step = min(cgv, 256), rp = 256 / step;
  for (int c0 = 0; c0 < cgv; c0 += step) {
    const int cv = c0 + t % step;
    const bool on = t < rp * step && cv < cgv;
    const int c = p.g * A.cg + (on ? cv : 0) * VW;
    float w[VW], b[VW], dw[VW], db[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      w[k] = param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
      dw[k] = db[k] = 0.f;
    }
    if (on)
      for (int64_t l = p.l0 + t / step; l < p.l1; l += rp) {
        float x[VW], dy[VW];
        load_vec<T, VW>((const T*)A.x.p + p.n * A.x.sn + l * A.x.sl + c, x);
        load_vec<T, VW>((const T*)A.dy.p + p.n * A.dy.sn + l * A.dy.sl + c, dy);
#pragma unroll
        for (int k = 0; k < VW; k++) {
          const float xh = (x[k] - m) * r, dz = dy[k] * act_slope(fmaf(xh, w[k], b[k]), A.act);
          db[k] += dz;
          dw[k] = fmaf(dz, xh, dw[k]);
        }
      }
    // the unit's sums, from the columns' sums: sum dxh = sum w db, sum dxh xh = sum w dw
#pragma unroll
    for (int k = 0; k < VW; k++) {
      v[0] = fmaf(w[k], db[k], v[0]);
      v[1] = fmaf(w[k], dw[k], v[1]);
    }
    const int64_t o = ((p.n * A.split + p.s) * A.G + p.g) * A.cg + cv * VW;
    if (A.dw) {
      column_sum<VW>(dw, t, rp, step, t < rp * step, cols);
      if (t < step && cv < cgv)
#pragma unroll
        for (int k = 0; k < VW; k++) A.dw[o + k] = dw[k];
    }
    if (A.db) {
      column_sum<VW>(db, t, rp, step, t < rp * step, cols);
      if (t < step && cv < cgv)
#pragma unroll
        for (int k = 0; k < VW; k++) A.db[o + k] = db[k];
    }
  }
  block_sum<2>(v, red);
  if (t == 0) {
    float* o = A.sums + (p.u * A.split + p.s) * 3;
    o[0] = v[0];
    o[1] = v[1];
  }
}

template <typename T, int VW>
__global__ __launch_bounds__(256) void k_gn_big_dx(GnArgs A) {
  const Part p = part_of(A);
  const float m = A.stats[2 * p.u], r = A.stats[2 * p.u + 1];
  float s1 = 0.f, s2 = 0.f;
  for (int s = 0; s < A.split; s++) {
    const float* o = A.sums + (p.u * A.split + s) * 3;
    s1 += o[0];
    s2 += o[1];
  }
  const float inv = 1.f / ((float)A.L * (float)A.cg);
  s1 *= inv;
  s2 *= inv;
  const int cgv = A.cg / VW, t = threadIdx.x;
  const int step = min(cgv, 256), rp = 256 / step;
  for (int c0 = 0; c0 < cgv; c0 += step) {
    const int cv = c0 + t % step;
    if (t >= rp * step || cv >= cgv) continue;
    const int c = p.g * A.cg + cv * VW;
    float w[VW], b[VW];
#pragma unroll
    for (int k = 0; k < VW; k++) {
      w[k] = param(A.w, A.wdt, c + k, 1.f);
      b[k] = param(A.b, A.wdt, c + k, 0.f);
    }
    for (int64_t l = p.l0 + t / step; l < p.l1; l += rp) {
      float x[VW], dy[VW];
      load_vec<T, VW>((const T*)A.x.p + p.n * A.x.sn + l * A.x.sl + c, x);
      load_vec<T, VW>((const T*)A.dy.p + p.n * A.dy.sn + l * A.dy.sl + c, dy);
#pragma unroll
      for (int k = 0; k < VW; k++) {
        const float xh = (x[k] - m) * r;
        x[k] = r * (dy[k] * act_slope(fmaf(xh, w[k], b[k]), A.act) * w[k] - s1 - xh * s2);
      }
      store_vec<T, VW>((T*)A.dx.p + p.n * A.dx.sn + l * A.dx.sl + c, x);
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
enum { WAVE, BLOCK, BIG };
struct Plan {
  int kind, vw, per, lanes_log2, threads, split;
  int64_t grid, R;  // R: rows of partial sums
};

int vector_width(const fw_group_norm* a, bool backward) {
  const int e = a->dtype == FW_DT_F32 ? 4 : 2, cg = a->C / a->G;
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
  p.vw = vector_width(a, backward);
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
  const int hold = backward || p.vw == 8 ? 8 : 16;  // vectors a thread holds: 64 floats of 128 registers
  if (cgv <= 1024 && (a->L + 1024 / cgv - 1) / (1024 / cgv) <= hold) {
    p.kind = BLOCK;
    p.threads = 256;  // the fewest threads whose registers hold the unit with at most `hold` vectors each
    while (p.threads < 1024 && (cgv > p.threads || (a->L + p.threads / cgv - 1) / (p.threads / cgv) > hold)) p.threads *= 2;
    const int64_t per = (a->L + p.threads / cgv - 1) / (p.threads / cgv);
    p.per = per <= 4 ? 4 : per <= 8 ? 8 : 16;
    p.grid = units;
    p.R = a->N;
    return p;
  }
  p.kind = BIG;
  const int64_t want = std::max<int64_t>(1, 2048 / units);  // blocks per unit
  p.split = (int)std::max<int64_t>(1, std::min<int64_t>({want, (vecs + 1023) / 1024, a->L, 256}));
  p.grid = units * p.split;
  p.R = a->N * p.split;
  return p;
}
size_t part_floats(const fw_group_norm* a, const Plan& p) { return (size_t)p.R * a->C; }
size_t sum_floats(const fw_group_norm* a, const Plan& p) {
  return p.kind == BIG ? (size_t)a->N * a->G * p.split * 3 : 0;
}

template <typename T, int VW, bool BWD>
int launch(const GnArgs& A, const Plan& p, hipStream_t s) {
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
    const size_t lds = BWD ? VW * 1024 * sizeof(float) : 0;
    if (p.per == 4)
      hipLaunchKernelGGL((k_gn_block<T, VW, 4, BWD>), grid, dim3(p.threads), lds, s, A);
    else if (p.per == 8)
      hipLaunchKernelGGL((k_gn_block<T, VW, 8, BWD>), grid, dim3(p.threads), lds, s, A);
    else if constexpr (!BWD && VW < 8)
      hipLaunchKernelGGL((k_gn_block<T, VW, 16, BWD>), grid, dim3(p.threads), lds, s, A);
  } else if constexpr (!BWD) {
    hipLaunchKernelGGL((k_gn_big_stats<T, VW>), grid, dim3(256), 0, s, A);
    FW_HIP(hipGetLastError());
    hipLaunchKernelGGL((k_gn_big_apply<T, VW>), grid, dim3(256), 0, s, A);
  } else {
    hipLaunchKernelGGL((k_gn_big_sums<T, VW>), grid, dim3(256), VW * 1024 * sizeof(float), s, A);
    FW_HIP(hipGetLastError());
    hipLaunchKernelGGL((k_gn_big_dx<T, VW>), grid, dim3(256), 0, s, A);
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
  if (a->N > 0 && a->N * (int64_t)a->G > INT32_MAX) return bad("too many groups for one call");
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
  if (p.kind == BIG && !a->stats) return fw::set_error(FW_E_INVALID, "fw_group_norm_backward: stats needed");
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
