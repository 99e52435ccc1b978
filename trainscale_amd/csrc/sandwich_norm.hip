// The norms before and after a block, fused with the block's gate and residual, for gfx950:
//   yhat = y * ry,  ry = 1 / sqrt(mean(y^2) + eps)           y: the block's output
//   h    = a x + g * yhat * (o + post)                       x: the residual stream
//   n    = h * rh * (o + pre),  rh = 1 / sqrt(mean(h^2) + eps)
// a: residual scale, g: gate (none, one row of channels, or one row for each group of rows),
// o: weight offset (1 for weights stored as their difference from 1). fp32 throughout; h and n
// are rounded once, and n comes from the unrounded h.
//
// Backward, from dn and dh:
//   e = dn (o + pre),  t = dh + rh (e - hhat mean(e hhat)),  hhat = h rh
//   dx = a t,  q = t g (o + post),  dy = ry (q - yhat mean(q yhat))
//   dpre = sum over rows of dn hhat,  A = sum over a group's rows of t yhat:
//   dgate = (o + post) A,  dpost = sum over groups of g A
// With t put in, mean(q yhat) = mean((dh + rh e) u) - rh mean(e hhat) mean(hhat u), where
// u = g (o + post) yhat: the row's three means come out of one reduction, one barrier, instead
// of two that wait for each other. h is formed again from x and y as the forward formed it, so
// the backward reads x instead of h (the same bytes) and sees no rounding of h.
//
// HBM-bound: 4 tensors of traffic forward (x, y in; h, n out), 6 backward (dn, dh, x, y in; dx,
// dy out): [8192, 4096] bf16 50 us (5.3 TB/s) and 65 us (6.2 TB/s) + 7 us for the parameters' sums;
// [4095, 8192] 55 and 75 us, where one workgroup of 1024 threads fills a CU and no other computes
// while it waits. Inputs are read through the caches, where what the layer before has written may
// still be (both directions 6 to 8 us faster than streaming loads when it is). A row is owned by
// TPR threads (whole waves), KV 16-byte vectors each, and stays in registers between its reductions
// and its outputs. The backward's workgroups walk rows of one group a fixed distance apart and keep
// t yhat and dn hhat of their columns in fp32 registers; one partial row each per workgroup, summed
// in a fixed order afterwards, so the parameters' gradients do not depend on timing.
//
// Rows of any length and address: vectors are loaded at element alignment, the elements behind
// the last whole vector by one lane.
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

// Vector v of a row, or the row's last elements (v == nvec), or zeros behind them.
template <typename T>
__device__ inline u32x4 load_raw(const T* __restrict__ row, int v, int nvec, int tail) {
  constexpr int V = Elt<T>::kVec;
  if (v < nvec) return ld16_any(row + (int64_t)v * V);
  float f[V];
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = v == nvec && i < tail ? Elt<T>::load1(row + (int64_t)v * V + i) : 0.f;
  return Elt<T>::pack(f);
}
template <typename T>
__device__ inline void store_part(T* __restrict__ row, int v, int nvec, int tail,
                                  const float (&f)[Elt<T>::kVec]) {
  constexpr int V = Elt<T>::kVec;
  if (v < nvec) {
    st16_any_stream(row + (int64_t)v * V, Elt<T>::pack(f));
  } else if (v == nvec) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < tail) Elt<T>::store1(row + (int64_t)v * V + i, f[i]);
  }
}

// A row of parameters (weights or a gate), of the data type or fp32.
struct Param {
  const void* p;
  int f32;
};
template <typename W, int V>
__device__ inline void load_values(const W* __restrict__ p, int v, int nvec, int tail,
                                   float (&f)[V]) {
  if (v < nvec) {
#pragma unroll
    for (int i = 0; i < V; i += Elt<W>::kVec)
      Elt<W>::unpack(ld16_any(p + (int64_t)v * V + i), f + i);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = v == nvec && i < tail ? Elt<W>::load1(p + (int64_t)v * V + i) : 0.f;
  }
}
template <typename T>
__device__ inline void load_param(const Param& w, int64_t row, int cols, int v, int nvec, int tail,
                                  float (&f)[Elt<T>::kVec]) {
  if (w.f32)
    load_values<float>(static_cast<const float*>(w.p) + row * cols, v, nvec, tail, f);
  else
    load_values<T>(static_cast<const T*>(w.p) + row * cols, v, nvec, tail, f);
}

template <typename T>
struct Io {  // a [rows, cols] tensor with its row stride; p may be NULL where the text says so
  T* p;
  int64_t ld;
};

struct Shape {
  int64_t rows, group_rows;  // row r belongs to group r / group_rows
  int cols, nvec, tail;
  float fcols, eps, scale, offset;
};

// Sums of kN values over the TPR threads of a row; `red` is this reduction's own.
template <int TPR, int kBlock, int kN>
__device__ inline void row_sums(float (&v)[kN], float (*red)[kBlock / kWave]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) v[j] = wave_sum(v[j]);
  if constexpr (TPR > kWave) {
    constexpr int kWaves = TPR / kWave;
    const int wid = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) {
#pragma unroll
      for (int j = 0; j < kN; ++j) red[j][wid] = v[j];
    }
    __syncthreads();
    const int first = wid / kWaves * kWaves;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kWaves; ++i) t += red[j][first + i];
      v[j] = t;
    }
  }
}

__device__ inline float rstd_of(float sum, const Shape& s) {
  return 1.0f / __builtin_sqrtf(sum / s.fcols + s.eps);
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <typename T, int TPR, int KV>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void sandwich_fwd(
    Io<const T> y, Io<const T> x, Param post, Param pre, Param gate, Io<T> n, Io<T> h,
    float* __restrict__ ry_out, float* __restrict__ rh_out, Shape s) {
  constexpr int V = Elt<T>::kVec;
  constexpr int kBlock = TPR > 256 ? TPR : 256;
  __shared__ float red[2][1][kBlock / kWave];
  const int t = threadIdx.x % TPR;
  const int64_t row =
      (int64_t)blockIdx.x * (kBlock / TPR) + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const bool valid = row < s.rows;
  const int64_t r = valid ? row : 0;
  u32x4 yq[KV], xq[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    yq[k] = load_raw(y.p + r * y.ld, t + k * TPR, s.nvec, s.tail);
    xq[k] = load_raw(x.p + r * x.ld, t + k * TPR, s.nvec, s.tail);
  }
  float sum[1] = {0.f};
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    float f[V];
    Elt<T>::unpack(yq[k], f);
#pragma unroll
    for (int i = 0; i < V; ++i) sum[0] = __builtin_fmaf(f[i], f[i], sum[0]);
  }
  row_sums<TPR, kBlock>(sum, red[0]);
  const float ry = rstd_of(sum[0], s);
  float hf[KV][V];
  // (The weights loaded with the row instead of here: 55 us for 50 at [8192, 4096] bf16, their
  // registers cost more than the round trip to L2 that they save.)
  sum[0] = 0.f;
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    float yf[V], xf[V], w[V];
    Elt<T>::unpack(yq[k], yf);
    Elt<T>::unpack(xq[k], xf);
    load_param<T>(post, 0, s.cols, t + k * TPR, s.nvec, s.tail, w);
#pragma unroll
    for (int i = 0; i < V; ++i) hf[k][i] = (yf[i] * ry) * (w[i] + s.offset);
    if (gate.p != nullptr) {
      load_param<T>(gate, r / s.group_rows, s.cols, t + k * TPR, s.nvec, s.tail, w);
#pragma unroll
      for (int i = 0; i < V; ++i) hf[k][i] *= w[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      hf[k][i] = __builtin_fmaf(xf[i], s.scale, hf[k][i]);
      sum[0] = __builtin_fmaf(hf[k][i], hf[k][i], sum[0]);
    }
    if (valid) store_part(h.p + r * h.ld, t + k * TPR, s.nvec, s.tail, hf[k]);
  }
  row_sums<TPR, kBlock>(sum, red[1]);
  const float rh = rstd_of(sum[0], s);
  if (!valid) return;
  if (t == 0) {
    ry_out[r] = ry;
    rh_out[r] = rh;
  }
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    float w[V];
    load_param<T>(pre, 0, s.cols, t + k * TPR, s.nvec, s.tail, w);
#pragma unroll
    for (int i = 0; i < V; ++i) hf[k][i] = (hf[k][i] * rh) * (w[i] + s.offset);
    store_part(n.p + r * n.ld, t + k * TPR, s.nvec, s.tail, hf[k]);
  }
}

// ---------------------------------------------------------------------------
// Backward: dx, dy and the parameters' partial rows. Workgroup g * per_group + p takes rows
// (p + st * per_group) * kRpb + sub of group g, st < steps.
// ---------------------------------------------------------------------------
template <typename T, int TPR, int KV>
__global__ __launch_bounds__(TPR > 512 ? TPR : 512) void sandwich_bwd(
    Io<const T> dn, Io<const T> dh, Io<const T> y, Io<const T> x, Param post, Param pre,
    Param gate, const float* __restrict__ ry_in, const float* __restrict__ rh_in, Io<T> dy,
    Io<T> dx, float* __restrict__ partial, int64_t ldp, int64_t per_group, int64_t steps, Shape s) {
  constexpr int V = Elt<T>::kVec;
  constexpr int kBlock = TPR > 512 ? TPR : 512;
  constexpr int kRpb = kBlock / TPR;
  __shared__ float red[2][3][kBlock / kWave];
  __shared__ float4 slots[kRpb > 1 ? kBlock * KV * V / 4 : 1];
  const int t = threadIdx.x % TPR;
  const int sub = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);  // a wave's: rows in SGPRs
  const int64_t group = blockIdx.x / per_group, p = blockIdx.x % per_group;
  const int64_t row0 = group * s.group_rows;
  const int64_t row1 = row0 + s.group_rows < s.rows ? row0 + s.group_rows : s.rows;

  // u0 = g (o + post) and o + pre of this thread's columns, in registers, or in LDS where a thread
  // has several vectors (the widest rows; registers would spill)
  constexpr bool kHold = KV == 1;
  __shared__ float4 pars[kHold ? 1 : 2 * KV * V / 4 * TPR];
  float u0[V], wq[V], acc_a[KV][V], acc_b[KV][V];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = 1.f;
    load_param<T>(post, 0, s.cols, t + k * TPR, s.nvec, s.tail, u0);
    load_param<T>(pre, 0, s.cols, t + k * TPR, s.nvec, s.tail, wq);
    if (gate.p != nullptr) load_param<T>(gate, group, s.cols, t + k * TPR, s.nvec, s.tail, g);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      u0[i] = (u0[i] + s.offset) * g[i];
      wq[i] += s.offset;
      acc_a[k][i] = acc_b[k][i] = 0.f;
    }
    if constexpr (!kHold) {
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        pars[(2 * (k * (V / 4) + q)) * TPR + t] =
            make_float4(u0[4 * q], u0[4 * q + 1], u0[4 * q + 2], u0[4 * q + 3]);
        pars[(2 * (k * (V / 4) + q) + 1) * TPR + t] =
            make_float4(wq[4 * q], wq[4 * q + 1], wq[4 * q + 2], wq[4 * q + 3]);
      }
    }
  }
  auto params_of = [&](int k) {  // the thread's own entries: no barrier
    if constexpr (!kHold) {
#pragma unroll
      for (int q = 0; q < V / 4; ++q) {
        const float4 a = pars[(2 * (k * (V / 4) + q)) * TPR + t];
        const float4 b = pars[(2 * (k * (V / 4) + q) + 1) * TPR + t];
        u0[4 * q] = a.x, u0[4 * q + 1] = a.y, u0[4 * q + 2] = a.z, u0[4 * q + 3] = a.w;
        wq[4 * q] = b.x, wq[4 * q + 1] = b.y, wq[4 * q + 2] = b.z, wq[4 * q + 3] = b.w;
      }
    }
  };
  for (int64_t st = 0; st < steps; ++st) {  // uniform over the workgroup
    const int64_t at = row0 + (p + st * per_group) * kRpb + sub;
    const bool valid = at < row1;
    const int64_t r = valid ? at : row0;  // (past the group: its first row, for nothing)
    u32x4 yq[KV], xq[KV], nq[KV], hq[KV];
    const u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int k = 0; k < KV; ++k) {
      const int v = t + k * TPR;
      yq[k] = load_raw(y.p + r * y.ld, v, s.nvec, s.tail);
      xq[k] = load_raw(x.p + r * x.ld, v, s.nvec, s.tail);
      nq[k] = dn.p != nullptr ? load_raw(dn.p + r * dn.ld, v, s.nvec, s.tail) : zero;
      hq[k] = dh.p != nullptr ? load_raw(dh.p + r * dh.ld, v, s.nvec, s.tail) : zero;
    }
    const float ry = ry_in[r], rh = rh_in[r];
    float sum[3] = {0.f, 0.f, 0.f};  // e hhat, (dh + rh e) u, hhat u
    // what the outputs need of the row, unpacked and scaled once: with each vector unpacked again
    // after the reduction (fewer registers) the kernel issued 48 operations an element, 41 of its
    // 70 us at [8192, 4096] bf16. Loading a row ahead does not help: 68 us against 66.
    float yh[KV][V], hh[KV][V], d[KV][V];  // yhat, hhat, dh + rh e
#pragma unroll
    for (int k = 0; k < KV; ++k) {
      float xf[V], nf[V];
      Elt<T>::unpack(yq[k], yh[k]);
      Elt<T>::unpack(xq[k], xf);
      Elt<T>::unpack(nq[k], nf);
      Elt<T>::unpack(hq[k], d[k]);
      params_of(k);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        yh[k][i] *= ry;
        const float u = yh[k][i] * u0[i];
        hh[k][i] = __builtin_fmaf(xf[i], s.scale, u) * rh;
        const float e = nf[i] * wq[i];
        d[k][i] = __builtin_fmaf(rh, e, d[k][i]);
        sum[0] = __builtin_fmaf(e, hh[k][i], sum[0]);
        sum[1] = __builtin_fmaf(d[k][i], u, sum[1]);
        sum[2] = __builtin_fmaf(hh[k][i], u, sum[2]);
      }
      if (valid) {
#pragma unroll
        for (int i = 0; i < V; ++i) acc_b[k][i] = __builtin_fmaf(nf[i], hh[k][i], acc_b[k][i]);
      }
    }
    row_sums<TPR, kBlock>(sum, red[st & 1]);
    const float c1 = sum[0] / s.fcols;
    const float c2 = (sum[1] - (rh * c1) * sum[2]) / s.fcols;
    const float rc1 = rh * c1, rc2 = ry * c2;
    if (valid) {
#pragma unroll
      for (int k = 0; k < KV; ++k) {
        params_of(k);
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[k][i] = __builtin_fmaf(-hh[k][i], rc1, d[k][i]);  // t
          acc_a[k][i] = __builtin_fmaf(d[k][i], yh[k][i], acc_a[k][i]);
          o[i] = __builtin_fmaf(d[k][i] * u0[i], ry, -(yh[k][i] * rc2));
          d[k][i] *= s.scale;
        }
        if (dx.p != nullptr) store_part(dx.p + r * dx.ld, t + k * TPR, s.nvec, s.tail, d[k]);
        if (dy.p != nullptr) store_part(dy.p + r * dy.ld, t + k * TPR, s.nvec, s.tail, o);
      }
    }
  }

  if (partial == nullptr) return;  // no parameter wants a gradient
  const int parts = s.nvec + (s.tail > 0);
  float* rows[2] = {partial + 2 * (int64_t)blockIdx.x * ldp,
                    partial + (2 * (int64_t)blockIdx.x + 1) * ldp};
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[KV][V] = which ? acc_b : acc_a;
    if constexpr (kRpb > 1) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < KV; ++k)
#pragma unroll
        for (int q = 0; q < V / 4; ++q)
          slots[(sub * KV + k) * TPR * (V / 4) + t * (V / 4) + q] =
              make_float4(acc[k][4 * q], acc[k][4 * q + 1], acc[k][4 * q + 2], acc[k][4 * q + 3]);
      __syncthreads();
      if (sub == 0) {
#pragma unroll
        for (int k = 0; k < KV; ++k)
#pragma unroll
          for (int q = 0; q < V / 4; ++q)
            for (int j = 1; j < kRpb; ++j) {
              const float4 f = slots[(j * KV + k) * TPR * (V / 4) + t * (V / 4) + q];
              acc[k][4 * q] += f.x;
              acc[k][4 * q + 1] += f.y;
              acc[k][4 * q + 2] += f.z;
              acc[k][4 * q + 3] += f.w;
            }
      }
    }
    if (sub == 0) {
#pragma unroll
      for (int k = 0; k < KV; ++k) {
        const int v = t + k * TPR;
        if (v < parts) {
#pragma unroll
          for (int q = 0; q < V / 4; ++q)
            *reinterpret_cast<float4*>(rows[which] + (int64_t)v * V + 4 * q) =
                make_float4(acc[k][4 * q], acc[k][4 * q + 1], acc[k][4 * q + 2], acc[k][4 * q + 3]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Gradients of the parameters from the partial rows
// ---------------------------------------------------------------------------
// Columns of a workgroup: 8 quads (128 bytes of a row) by 32 row groups.
constexpr int kCols = 32;
constexpr int kQuads = kCols / 4, kGroups = 256 / kQuads;
static_assert(ts_plan::kSandwichReduceCols == kCols, "columns of a reducing workgroup");

// Sum over rows i < nrows of the quad at rows + i * stride + c, in a fixed order; valid in the
// first kQuads threads (g == 0), one for each quad.
__device__ inline float4 sum_rows(const float* __restrict__ rows, int64_t stride, int64_t nrows,
                                  int64_t c, bool in, float4 (*red)[kQuads]) {
  const int cq = threadIdx.x % kQuads, g = threadIdx.x / kQuads;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  if (in) {
    for (int64_t i = g; i < nrows; i += kGroups) {
      const float4 v = *reinterpret_cast<const float4*>(rows + i * stride + c);
      a.x += v.x;
      a.y += v.y;
      a.z += v.z;
      a.w += v.w;
    }
  }
  red[g][cq] = a;
  __syncthreads();
#pragma unroll
  for (int h = kGroups / 2; h >= 1; h >>= 1) {
    if (g < h) {
      const float4 o = red[g + h][cq];
      float4 m = red[g][cq];
      m.x += o.x;
      m.y += o.y;
      m.z += o.z;
      m.w += o.w;
      red[g][cq] = m;
    }
    __syncthreads();
  }
  return red[0][cq];
}

template <typename T>
__device__ inline float param1(const Param& w, int64_t i) {
  return w.f32 ? static_cast<const float*>(w.p)[i] : Elt<T>::load1(static_cast<const T*>(w.p) + i);
}
template <typename T>
__device__ inline void store_param(void* p, int f32, int64_t i, float v) {
  if (f32)
    static_cast<float*>(p)[i] = v;
  else
    Elt<T>::store1(static_cast<T*>(p) + i, v);
}

// blockIdx.y = 2 * group + which: the group's A (which 0) or its part of dpre (1), from its
// workgroups' partial rows. With one group these are the gradients; with more, dgate is written
// and g A and dpre's part go to rows 2 * group + which of `mid`.
template <typename T>
__global__ __launch_bounds__(256) void sandwich_params(const float* __restrict__ partial,
                                                       int64_t ldp, int64_t per_group,
                                                       int64_t groups, int cols, Param post,
                                                       Param gate, float offset, void* dpost,
                                                       void* dpre, void* dgate, int post_f32,
                                                       int pre_f32, int gate_f32,
                                                       float* __restrict__ mid) {
  __shared__ float4 red[kGroups][kQuads];
  const int64_t blocks_x = (ldp + kCols - 1) / kCols;
  const int64_t group = blockIdx.x / blocks_x / 2;
  const int which = (int)(blockIdx.x / blocks_x & 1);
  const int64_t c = blockIdx.x % blocks_x * kCols + (threadIdx.x % kQuads) * 4;
  const float4 a = sum_rows(partial + (group * per_group * 2 + which) * ldp, 2 * ldp, per_group, c,
                            c < ldp, red);
  if (threadIdx.x >= kQuads) return;
  const float f[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (c + i >= cols) break;
    if (which == 0) {
      if (dgate != nullptr)
        store_param<T>(dgate, gate_f32, group * cols + c + i,
                       (param1<T>(post, c + i) + offset) * f[i]);
      const float ga = gate.p != nullptr ? param1<T>(gate, group * cols + c + i) * f[i] : f[i];
      if (groups > 1)
        mid[2 * group * ldp + c + i] = ga;
      else if (dpost != nullptr)
        store_param<T>(dpost, post_f32, c + i, ga);
    } else if (groups > 1) {
      mid[(2 * group + 1) * ldp + c + i] = f[i];
    } else if (dpre != nullptr) {
      store_param<T>(dpre, pre_f32, c + i, f[i]);
    }
  }
}

// dpost and dpre (blockIdx.y) over the groups' rows of `mid`.
template <typename T>
__global__ __launch_bounds__(256) void sandwich_params_groups(const float* __restrict__ mid,
                                                              int64_t ldp, int64_t groups,
                                                              int cols, void* dpost, void* dpre,
                                                              int post_f32, int pre_f32) {
  __shared__ float4 red[kGroups][kQuads];
  const int64_t c = (int64_t)blockIdx.x * kCols + (threadIdx.x % kQuads) * 4;
  const float4 a = sum_rows(mid + blockIdx.y * ldp, 2 * ldp, groups, c, c < ldp, red);
  void* out = blockIdx.y ? dpre : dpost;
  if (threadIdx.x >= kQuads || out == nullptr) return;
  const float f[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < cols) store_param<T>(out, blockIdx.y ? pre_f32 : post_f32, c + i, f[i]);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Call {
  const void *dn, *dh, *y, *x;
  int64_t lddn, lddh, ldy, ldx;
  ts_dtype dtype;
  Param post, pre, gate;
  int64_t groups, rows, cols;
  float scale, offset, eps;
};

template <typename T>
Shape shape_of(const Call& c) {
  Shape s;
  s.rows = c.rows;
  s.group_rows = c.rows / c.groups;
  s.cols = (int)c.cols;
  s.nvec = (int)(c.cols / Elt<T>::kVec);
  s.tail = (int)(c.cols % Elt<T>::kVec);
  s.fcols = (float)c.cols;
  s.eps = c.eps;
  s.scale = c.scale;
  s.offset = c.offset;
  return s;
}

template <typename T>
ts_status fwd_typed(const Call& c, void* n, int64_t ldn, void* h, int64_t ldh, float* ry, float* rh,
                    hipStream_t st) {
  const Shape s = shape_of<T>(c);
  const ts_plan::SandwichPlan p = ts_plan::sandwich_fwd_plan(s.nvec + (s.tail > 0));
  const int64_t blocks = (c.rows + p.rpb - 1) / p.rpb;
  if (blocks > ts_plan::max_blocks(p.tpr > 256 ? p.tpr : 256))
    return ts_host::fail(TS_ERR_SHAPE, "sandwich_norm_fwd: too many rows");
  const Io<const T> y{static_cast<const T*>(c.y), c.ldy}, x{static_cast<const T*>(c.x), c.ldx};
  const Io<T> no{static_cast<T*>(n), ldn}, ho{static_cast<T*>(h), ldh};
#define TS_FWD(R, K)                                                                              \
  hipLaunchKernelGGL((sandwich_fwd<T, R, K>), dim3((unsigned)blocks), dim3(R > 256 ? R : 256), 0, \
                     st, y, x, c.post, c.pre, c.gate, no, ho, ry, rh, s)
  switch (p.tpr * 8 + p.kv) {
    case 64 * 8 + 1: TS_FWD(64, 1); break;
    case 64 * 8 + 2: TS_FWD(64, 2); break;
    case 128 * 8 + 2: TS_FWD(128, 2); break;
    case 256 * 8 + 2: TS_FWD(256, 2); break;
    case 512 * 8 + 2: TS_FWD(512, 2); break;
    case 512 * 8 + 4: TS_FWD(512, 4); break;
    default: return ts_host::fail(TS_ERR_SHAPE, "sandwich_norm_fwd: no plan");
  }
#undef TS_FWD
  return ts_host::check_launch("sandwich_fwd");
}

template <typename T>
ts_status bwd_typed(const Call& c, const float* ry, const float* rh, void* dy, int64_t lddy,
                    void* dx, int64_t lddx, void* dpost, void* dpre, void* dgate, float* ws,
                    hipStream_t st) {
  const Shape s = shape_of<T>(c);
  const int parts = s.nvec + (s.tail > 0);
  const ts_plan::SandwichBwdPlan p =
      ts_plan::sandwich_bwd_plan(c.rows, c.groups, c.cols, Elt<T>::kVec);
  const int64_t ldp = (int64_t)parts * Elt<T>::kVec;
  const int64_t blocks = c.groups * p.per_group;
  const int64_t reduce = (ldp + kCols - 1) / kCols * c.groups * 2;
  if (blocks > ts_plan::max_blocks(p.row.tpr > 512 ? p.row.tpr : 512) ||
      reduce > ts_plan::max_blocks(256))
    return ts_host::fail(TS_ERR_SHAPE, "sandwich_norm_bwd: too many groups");
  const Io<const T> dn{static_cast<const T*>(c.dn), c.lddn}, dh{static_cast<const T*>(c.dh), c.lddh},
      y{static_cast<const T*>(c.y), c.ldy}, x{static_cast<const T*>(c.x), c.ldx};
  const Io<T> dyo{static_cast<T*>(dy), lddy}, dxo{static_cast<T*>(dx), lddx};
  const bool params = dpost != nullptr || dpre != nullptr || dgate != nullptr;
  float* partial = params ? ws : nullptr;
#define TS_BWD(R, K)                                                                              \
  hipLaunchKernelGGL((sandwich_bwd<T, R, K>), dim3((unsigned)blocks), dim3(R > 512 ? R : 512), 0, \
                     st, dn, dh, y, x, c.post, c.pre, c.gate, ry, rh, dyo, dxo, partial, ldp,     \
                     p.per_group, p.steps, s)
  switch (p.row.tpr * 8 + p.row.kv) {
    case 64 * 8 + 1: TS_BWD(64, 1); break;
    case 128 * 8 + 1: TS_BWD(128, 1); break;
    case 256 * 8 + 1: TS_BWD(256, 1); break;
    case 512 * 8 + 1: TS_BWD(512, 1); break;
    case 1024 * 8 + 1: TS_BWD(1024, 1); break;
    case 512 * 8 + 4: TS_BWD(512, 4); break;
    default: return ts_host::fail(TS_ERR_SHAPE, "sandwich_norm_bwd: no plan");
  }
#undef TS_BWD
  ts_status status = ts_host::check_launch("sandwich_bwd");
  if (status != TS_OK || !params) return status;
  float* mid = ws + 2 * blocks * ldp;
  hipLaunchKernelGGL(sandwich_params<T>, dim3((unsigned)reduce), dim3(256), 0, st, partial, ldp,
                     p.per_group, c.groups, s.cols, c.post, c.gate, s.offset, dpost, dpre, dgate,
                     c.post.f32, c.pre.f32, c.gate.f32, mid);
  status = ts_host::check_launch("sandwich_params");
  if (status != TS_OK || c.groups == 1 || (dpost == nullptr && dpre == nullptr)) return status;
  hipLaunchKernelGGL(sandwich_params_groups<T>, dim3((unsigned)((ldp + kCols - 1) / kCols), 2),
                     dim3(256), 0, st, mid, ldp, c.groups, s.cols, dpost, dpre, c.post.f32,
                     c.pre.f32);
  return ts_host::check_launch("sandwich_params_groups");
}

bool misaligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

// The checks both directions share. The tensors may be NULL only where there are no rows.
ts_status check_call(const char* what, const Call& c, ts_dtype w_dtype, ts_dtype gate_dtype) {
  using ts_host::fail;
  if (!ts_host::valid_dtype(c.dtype) || !ts_host::valid_dtype(w_dtype))
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: bad dtype", what);
  if (w_dtype != c.dtype && w_dtype != TS_F32)
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: weights are neither fp32 nor of the data's dtype",
                what);
  if (c.rows < 0 || c.cols <= 0) return fail(TS_ERR_SHAPE, "%s: bad sizes", what);
  if (c.cols > ts_plan::sandwich_max_cols((int)ts_host::dtype_size(c.dtype)))
    return fail(TS_ERR_SHAPE, "%s: rows longer than %lld elements", what,
                (long long)ts_plan::sandwich_max_cols((int)ts_host::dtype_size(c.dtype)));
  if (c.groups < 1 || (c.rows > 0 && c.rows % c.groups != 0))
    return fail(TS_ERR_SHAPE, "%s: the rows do not divide into the gate's groups", what);
  if (c.gate.p == nullptr && c.groups != 1)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: groups without a gate", what);
  if (c.gate.p != nullptr) {
    if (!ts_host::valid_dtype(gate_dtype) || (gate_dtype != c.dtype && gate_dtype != TS_F32))
      return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: the gate is neither fp32 nor of the data's dtype",
                  what);
    if (misaligned(c.gate.p, ts_host::dtype_size(gate_dtype)))
      return fail(TS_ERR_INVALID_ARGUMENT, "%s: a tensor is not aligned to its elements", what);
  }
  if (!(c.eps >= 0.f)) return fail(TS_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", what);
  if (c.rows == 0) return TS_OK;
  if (c.x == nullptr || c.y == nullptr || c.post.p == nullptr || c.pre.p == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
  if (c.ldx < c.cols || c.ldy < c.cols)
    return fail(TS_ERR_SHAPE, "%s: row stride below the row's length", what);
  const size_t e = ts_host::dtype_size(c.dtype), w = ts_host::dtype_size(w_dtype);
  if (misaligned(c.x, e) || misaligned(c.y, e) || misaligned(c.post.p, w) || misaligned(c.pre.p, w))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: a tensor is not aligned to its elements", what);
  return TS_OK;
}

// A fp32 row is read as fp32 also where that is the data's own type.
Param param_of(const void* p, ts_dtype t) { return Param{p, t == TS_F32 ? 1 : 0}; }

}  // namespace

extern "C" ts_status ts_sandwich_norm_fwd(const void* y, int64_t ldy, const void* x, int64_t ldx,
                                          ts_dtype dtype, const void* post, const void* pre,
                                          ts_dtype w_dtype, const void* gate, ts_dtype gate_dtype,
                                          int64_t gate_groups, void* n, int64_t ldn, void* h,
                                          int64_t ldh, float* rstd_y, float* rstd_h, int64_t rows,
                                          int64_t cols, float residual_scale, float weight_offset,
                                          float eps, ts_stream_t stream) {
  using ts_host::fail;
  const Call c{nullptr, nullptr, y, x, 0, 0, ldy, ldx, dtype, param_of(post, w_dtype),
               param_of(pre, w_dtype), param_of(gate, gate_dtype), gate_groups, rows, cols,
               residual_scale, weight_offset, eps};
  const ts_status s = check_call("sandwich_norm_fwd", c, w_dtype, gate_dtype);
  if (s != TS_OK || rows == 0) return s;
  if (n == nullptr || h == nullptr || rstd_y == nullptr || rstd_h == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "sandwich_norm_fwd: NULL pointer");
  if (ldn < cols || ldh < cols)
    return fail(TS_ERR_SHAPE, "sandwich_norm_fwd: row stride below the row's length");
  if (misaligned(n, ts_host::dtype_size(dtype)) || misaligned(h, ts_host::dtype_size(dtype)))
    return fail(TS_ERR_INVALID_ARGUMENT,
                "sandwich_norm_fwd: a tensor is not aligned to its elements");
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_BF16: return fwd_typed<__bf16>(c, n, ldn, h, ldh, rstd_y, rstd_h, st);
    case TS_F16: return fwd_typed<_Float16>(c, n, ldn, h, ldh, rstd_y, rstd_h, st);
    case TS_F32: return fwd_typed<float>(c, n, ldn, h, ldh, rstd_y, rstd_h, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "sandwich_norm_fwd: bad dtype");
}

extern "C" size_t ts_sandwich_norm_bwd_workspace_size(int64_t rows, int64_t cols,
                                                      int64_t gate_groups) {
  if (rows <= 0 || cols <= 0 || gate_groups < 1 || gate_groups > rows) return 0;
  return (size_t)ts_plan::sandwich_workspace(rows, gate_groups, cols);
}

extern "C" ts_status ts_sandwich_norm_bwd(
    const void* dn, int64_t lddn, const void* dh, int64_t lddh, const void* y, int64_t ldy,
    const void* x, int64_t ldx, ts_dtype dtype, const void* post, const void* pre,
    ts_dtype w_dtype, const void* gate, ts_dtype gate_dtype, int64_t gate_groups,
    const float* rstd_y, const float* rstd_h, void* dy, int64_t lddy, void* dx, int64_t lddx,
    void* dpost, void* dpre, void* dgate, int64_t rows, int64_t cols, float residual_scale,
    float weight_offset, void* workspace, size_t workspace_bytes, ts_stream_t stream) {
  using ts_host::fail;
  const Call c{dn, dh, y, x, lddn, lddh, ldy, ldx, dtype, param_of(post, w_dtype),
               param_of(pre, w_dtype), param_of(gate, gate_dtype), gate_groups, rows, cols,
               residual_scale, weight_offset, 0.f};
  const ts_status s = check_call("sandwich_norm_bwd", c, w_dtype, gate_dtype);
  if (s != TS_OK) return s;
  if (rows == 0) return fail(TS_ERR_SHAPE, "sandwich_norm_bwd: no rows");
  if (rstd_y == nullptr || rstd_h == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "sandwich_norm_bwd: NULL pointer");
  if (dgate != nullptr && gate == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "sandwich_norm_bwd: a gate's gradient without a gate");
  if ((dn != nullptr && lddn < cols) || (dh != nullptr && lddh < cols) ||
      (dy != nullptr && lddy < cols) || (dx != nullptr && lddx < cols))
    return fail(TS_ERR_SHAPE, "sandwich_norm_bwd: row stride below the row's length");
  const size_t e = ts_host::dtype_size(dtype), w = ts_host::dtype_size(w_dtype);
  if (misaligned(dn, e) || misaligned(dh, e) || misaligned(dy, e) || misaligned(dx, e) ||
      misaligned(dpost, w) || misaligned(dpre, w) ||
      (dgate != nullptr && misaligned(dgate, ts_host::dtype_size(gate_dtype))))
    return fail(TS_ERR_INVALID_ARGUMENT,
                "sandwich_norm_bwd: a tensor is not aligned to its elements");
  if (dpost != nullptr || dpre != nullptr || dgate != nullptr) {
    if (workspace == nullptr || !ts_host::aligned16(workspace) ||
        workspace_bytes < ts_sandwich_norm_bwd_workspace_size(rows, cols, gate_groups))
      return fail(TS_ERR_WORKSPACE,
                  "sandwich_norm_bwd: workspace missing, too small or unaligned");
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* ws = static_cast<float*>(workspace);
  switch (dtype) {
    case TS_BF16:
      return bwd_typed<__bf16>(c, rstd_y, rstd_h, dy, lddy, dx, lddx, dpost, dpre, dgate, ws, st);
    case TS_F16:
      return bwd_typed<_Float16>(c, rstd_y, rstd_h, dy, lddy, dx, lddx, dpost, dpre, dgate, ws, st);
    case TS_F32:
      return bwd_typed<float>(c, rstd_y, rstd_h, dy, lddy, dx, lddx, dpost, dpre, dgate, ws, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "sandwich_norm_bwd: bad dtype");
}
