// Dropout from a counter-based generator for gfx950, its mask never stored: alone, with the
// residual sum, and with the residual sum and the next RMSNorm, forward and backward.
//   D(x) = kept ? x / (1 - q) : 0,  q = drop / 65536
//   out = residual + D(x);   h = residual + D(x), y = h rstd(h) w
//   backward of the norm: e = dy w, t = dh + rstd (e - hat mean(e hat)), hat = h rstd,
//   dresidual = t, dx = D(t), dw = sum over rows of dy hat
//
// Random bits: Philox 4x32 with 10 rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", 2011) under key `seed`. Counter (r ceil(cols / 8) + c / 8, offset),
// 64 bits each, serves elements c / 8 * 8 .. + 7 of row r with 16 bits each, the low halves of its
// four words first; an element is dropped where its 16 bits are below `drop`. So the mask follows
// from (seed, offset, row, column) alone, whatever the type, strides or launch shape, and the
// backward forms it again.
//
// Every kernel gives a lane groups of 8 elements, one counter each: a group is one 16-byte access
// (two for fp32), at any element address; a row's last, shorter group goes element by element.
//
// Bound by HBM, with the generator's 20 products a group nearly hidden under it. Measured on MI355X,
// [8192, 14336] bf16: 75 us (6.3 TB/s) back to back; between events 80.3, 76.5 without a mask, and
// 83.4 with exclusive ors in pairs, each 16 bits taken apart and a division for the row. With the norm,
// [16384, 4096] bf16 94 us forward (5.8 TB/s) and 129 + 5 us
// backward (5.4 TB/s; much the same without the mask or dw, so what is left is memory latency), [8191,
// 768] fp32 26 and 29 + 4 us.
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

struct Rng {
  uint64_t seed, offset;
  const int64_t* state;  // device [2] (seed, offset), or NULL
  int32_t drop;          // 0 .. 65536
  float scale;           // 1 / (1 - q), 0 where everything is dropped
};

struct Key {
  uint32_t k0, k1, o0, o1;
};
__device__ inline Key key_of(const Rng& r) {
  uint64_t s = r.seed, o = r.offset;
  if (r.state != nullptr) {
    s = (uint64_t)r.state[0];
    o = (uint64_t)r.state[1];
  }
  return Key{(uint32_t)s, (uint32_t)(s >> 32), (uint32_t)o, (uint32_t)(o >> 32)};
}

// Four random words of counter (n, offset).
__device__ inline u32x4 philox(uint64_t n, Key k) {
  uint32_t c0 = (uint32_t)n, c1 = (uint32_t)(n >> 32), c2 = k.o0, c3 = k.o1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
    c0 = __builtin_amdgcn_bitop3_b32((uint32_t)(p1 >> 32), c1, k.k0, 0x96);  // exclusive or of 3
    c1 = (uint32_t)p1;
    c2 = __builtin_amdgcn_bitop3_b32((uint32_t)(p0 >> 32), c3, k.k1, 0x96);
    c3 = (uint32_t)p0;
    k.k0 += 0x9E3779B9u;
    k.k1 += 0xBB67AE85u;
  }
  return u32x4{c0, c1, c2, c3};
}

// f[i] = kept ? f[i] * scale : 0 over the 8 elements of group n, drop > 0. An element's 16 bits are
// compared from the top of a word: at or above drop if the word is above 65536 drop - 1, which fits
// 32 bits up to drop = 65536 (nothing kept).
__device__ inline void apply_mask(float (&f)[8], uint64_t n, const Key& k, int drop, float scale) {
  const u32x4 w = philox(n, k);
  const uint32_t limit = ((uint32_t)drop << 16) - 1u;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t top = i & 1 ? w[i / 2] : w[i / 2] << 16;
    f[i] = top > limit ? f[i] * scale : 0.f;
  }
}

// Eight elements from p, or the first n of them (the others 0).
template <typename T>
__device__ inline void load8(const T* p, float (&f)[8], int n) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      Elt<T>::unpack(ld16_any_stream(p), f);
    } else {
      const u32x4 a = ld16_any_stream(p), b = ld16_any_stream(p + 4);
      Elt<T>::unpack(a, f);
      Elt<T>::unpack(b, f + 4);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? Elt<T>::load1(p + i) : 0.f;
  }
}
template <typename T>
__device__ inline void store8(T* p, const float (&f)[8], int n) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      st16_any_stream(p, Elt<T>::pack(f));
    } else {
      st16_any_stream(p, Elt<T>::pack(f));
      st16_any_stream(p + 4, Elt<T>::pack(f + 4));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) Elt<T>::store1(p + i, f[i]);
  }
}

// ---------------------------------------------------------------------------
// out = [residual +] D(x): one group a thread
// ---------------------------------------------------------------------------
struct DropArgs {
  const void* x;
  int64_t ldx;
  const void* res;
  int64_t ldr;
  void* out;
  int64_t ldo;
  int64_t cols, groups, total;  // groups a row, groups in all
  uint64_t magic;               // ts_plan::magic64_for(groups)
  int32_t one_row;
  Rng rng;
};

template <typename T, bool kRes>
__global__ __launch_bounds__(256) void dropout_kernel(const DropArgs a) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= a.total) return;
  const int64_t r = a.one_row ? 0 : a.magic == 0 ? v : (int64_t)__umul64hi((uint64_t)v, a.magic);
  const int64_t c = (v - r * a.groups) * 8;
  const int n = a.cols - c < 8 ? (int)(a.cols - c) : 8;
  float f[8], res[8];
  load8(static_cast<const T*>(a.x) + r * a.ldx + c, f, n);
  if constexpr (kRes) load8(static_cast<const T*>(a.res) + r * a.ldr + c, res, n);
  if (a.rng.drop > 0) apply_mask(f, (uint64_t)v, key_of(a.rng), a.rng.drop, a.rng.scale);
  if constexpr (kRes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] += res[i];
  }
  store8(static_cast<T*>(a.out) + r * a.ldo + c, f, n);
}

// ---------------------------------------------------------------------------
// With the norm: a row on kTpr threads (a power of two: lanes of a wave, or whole waves) of kKv
// groups each, kTpr groups apart
// ---------------------------------------------------------------------------
struct NormArgs {
  const void* x;    // forward: x and residual in, y and h out
  int64_t ldx;
  const void* res;
  int64_t ldr;
  const void* dy;   // backward: dy, dh and h in, dx and dres out
  int64_t lddy;
  const void* dh;
  int64_t lddh;
  const void* w;
  void* y;
  void* h;
  int64_t ldh;
  float* rstd;
  void* dx;
  void* dres;
  float* part;      // [workgroups][cols] of dw
  int64_t rows, cols, groups;
  float eps;
  Rng rng;
};

// Sum over the kTpr threads of a row; `lds` holds a float for each wave of the workgroup.
template <int kTpr, int kBlock>
__device__ inline float row_total(float v, float* lds) {
  if constexpr (kTpr <= 64) {
#pragma unroll
    for (int m = 1; m < kTpr; m <<= 1) v += __shfl_xor(v, m);
    return v;
  } else {
    constexpr int kWaves = kTpr / 64;
    v = wave_sum(v);
    const int wid = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[wid] = v;
    __syncthreads();
    const int w0 = wid / kWaves * kWaves;
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) t += lds[w0 + i];
    __syncthreads();
    return t;
  }
}

template <typename W>
__device__ inline void load_w(const void* w, int64_t c, int n, float (&f)[8]) {
  load8(static_cast<const W*>(w) + c, f, n);
}

template <typename T, typename W, int kTpr, int kKv, int kBlock>
__global__ __launch_bounds__(kBlock) void dropout_norm_fwd(const NormArgs a) {
  __shared__ float lds[kBlock / 64];
  constexpr int kRows = kBlock / kTpr;
  const int t = threadIdx.x % kTpr;
  const int64_t r = (int64_t)blockIdx.x * kRows + threadIdx.x / kTpr;
  const bool live = r < a.rows;
  const int64_t row = live ? r : 0;
  float f[kKv][8], res[kKv][8];
  int n[kKv];
#pragma unroll
  for (int k = 0; k < kKv; ++k) {
    const int64_t c = ((int64_t)t + k * kTpr) * 8;
    const int64_t left = live ? a.cols - c : 0;
    n[k] = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    load8(static_cast<const T*>(a.x) + row * a.ldx + c, f[k], n[k]);
    load8(static_cast<const T*>(a.res) + row * a.ldr + c, res[k], n[k]);
  }
  float sq = 0.f;
#pragma unroll
  for (int k = 0; k < kKv; ++k) {
    if (a.rng.drop > 0 && n[k] > 0)
      apply_mask(f[k], (uint64_t)row * a.groups + t + k * kTpr, key_of(a.rng), a.rng.drop,
                 a.rng.scale);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      f[k][i] += res[k][i];
      sq += f[k][i] * f[k][i];
    }
    if (n[k] > 0)
      store8(static_cast<T*>(a.h) + row * a.cols + ((int64_t)t + k * kTpr) * 8, f[k], n[k]);
  }
  const float s = row_total<kTpr, kBlock>(sq, lds);
  const float rstd = 1.f / sqrtf(s / (float)a.cols + a.eps);
  if (live && t == 0) a.rstd[r] = rstd;
#pragma unroll
  for (int k = 0; k < kKv; ++k) {
    if (n[k] == 0) continue;
    const int64_t c = ((int64_t)t + k * kTpr) * 8;
    float w[8];
    load_w<W>(a.w, c, n[k], w);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[k][i] = f[k][i] * rstd * w[i];
    store8(static_cast<T*>(a.y) + row * a.cols + c, f[k], n[k]);
  }
}

// Workgroups walk the row groups b, b + grid, ...; dw's terms of a thread's columns stay in its
// registers, are added over the workgroup's row slots in LDS and written as one partial row.
template <typename T, typename W, int kTpr, int kKv, int kBlock>
__global__ __launch_bounds__(kBlock) void dropout_norm_bwd(const NormArgs a) {
  constexpr int kRows = kBlock / kTpr;
  __shared__ float lds[kBlock / 64];
  const int t = threadIdx.x % kTpr, slot = threadIdx.x / kTpr;
  const Key key = key_of(a.rng);
  float w[kKv][8], dw[kKv][8];
  int n[kKv];
#pragma unroll
  for (int k = 0; k < kKv; ++k) {
    const int64_t c = ((int64_t)t + k * kTpr) * 8;
    const int64_t left = a.cols - c;
    n[k] = left >= 8 ? 8 : left > 0 ? (int)left : 0;
    load_w<W>(a.w, c, n[k], w[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[k][i] = 0.f;
  }
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < a.rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t r = r0 + slot;
    const bool live = r < a.rows;
    const int64_t row = live ? r : r0;
    float e[kKv][8], hat[kKv][8], t0[kKv][8];
    const float rstd = a.rstd[row];
    float dot = 0.f;
#pragma unroll
    for (int k = 0; k < kKv; ++k) {
      const int64_t c = ((int64_t)t + k * kTpr) * 8;
      const int m = live ? n[k] : 0;
      if (a.dy != nullptr) load8(static_cast<const T*>(a.dy) + row * a.lddy + c, e[k], m);
      load8(static_cast<const T*>(a.h) + row * a.ldh + c, hat[k], m);
      if (a.dh != nullptr) load8(static_cast<const T*>(a.dh) + row * a.lddh + c, t0[k], m);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (a.dy == nullptr) e[k][i] = 0.f;
        if (a.dh == nullptr) t0[k][i] = 0.f;
        hat[k][i] *= rstd;
        dw[k][i] += e[k][i] * hat[k][i];
        e[k][i] *= w[k][i];
        dot += e[k][i] * hat[k][i];
      }
    }
    const float c1 = row_total<kTpr, kBlock>(dot, lds) / (float)a.cols;
    if (!live) continue;  // nothing to write; its terms were zeros
#pragma unroll
    for (int k = 0; k < kKv; ++k) {
      if (n[k] == 0) continue;
      const int64_t c = ((int64_t)t + k * kTpr) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) t0[k][i] += rstd * (e[k][i] - hat[k][i] * c1);
      if (a.dres != nullptr) store8(static_cast<T*>(a.dres) + row * a.cols + c, t0[k], n[k]);
      if (a.dx != nullptr) {
        if (a.rng.drop > 0)
          apply_mask(t0[k], (uint64_t)row * a.groups + t + k * kTpr, key, a.rng.drop, a.rng.scale);
        store8(static_cast<T*>(a.dx) + row * a.cols + c, t0[k], n[k]);
      }
    }
  }
  if (a.part == nullptr) return;
  float* out = a.part + (int64_t)blockIdx.x * a.cols;
  if constexpr (kRows == 1) {
#pragma unroll
    for (int k = 0; k < kKv; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n[k]) out[((int64_t)t + k * kTpr) * 8 + i] = dw[k][i];
  } else {
    // row slots in LDS, a group of 8 at a time, added in slot order
    __shared__ float sums[kBlock][9];
#pragma unroll
    for (int k = 0; k < kKv; ++k) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 8; ++i) sums[threadIdx.x][i] = dw[k][i];
      __syncthreads();
      for (int j = threadIdx.x; j < kTpr * 8; j += kBlock) {
        const int64_t c = ((int64_t)(j >> 3) + k * kTpr) * 8 + (j & 7);
        float s = 0.f;
        for (int q = 0; q < kRows; ++q) s += sums[q * kTpr + (j >> 3)][j & 7];
        if (c < a.cols) out[c] = s;
      }
    }
  }
}

// dw[c] = sum of the partial rows in a fixed order: 32 columns x 32 slices of rows a workgroup, 8
// rows' loads in flight. 64 columns x 16 slices, with half the workgroups, took 9.6 us for 512 rows
// of 4096 and 10.4 us of 768.
constexpr int kSumCols = 32, kSumSlices = 32, kSumUnroll = 8;
template <typename W>
__global__ __launch_bounds__(kSumCols * kSumSlices) void dropout_dw_sum(
    const float* __restrict__ part, int64_t nparts, int64_t cols, W* __restrict__ dw) {
  __shared__ float lds[kSumSlices][kSumCols + 1];
  const int lane = threadIdx.x % kSumCols, slice = threadIdx.x / kSumCols;
  const int64_t c = (int64_t)blockIdx.x * kSumCols + lane;
  float s = 0.f;
  if (c < cols) {
    for (int64_t p0 = slice; p0 < nparts; p0 += kSumSlices * kSumUnroll) {
      float v[kSumUnroll];
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u) {
        const int64_t p = p0 + u * kSumSlices;
        v[u] = p < nparts ? part[p * cols + c] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < kSumUnroll; ++u) s += v[u];
    }
  }
  lds[slice][lane] = s;
  __syncthreads();
  if (slice == 0 && c < cols) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < kSumSlices; ++i) t += lds[i][lane];
    Elt<W>::store1(dw + c, t);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
ts_status rng_of(const char* who, const ts_dropout_rng* in, Rng& r) {
  using ts_host::fail;
  if (in == nullptr) return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL rng", who);
  if (in->drop < 0 || in->drop > 65536)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: drop must be 0 to 65536, got %d", who,
                (int)in->drop);
  if ((reinterpret_cast<uintptr_t>(in->state) & 7u) != 0)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: rng state must be 8-byte aligned", who);
  r.seed = in->seed;
  r.offset = in->offset;
  r.state = in->state;
  r.drop = in->drop;
  r.scale = in->drop >= 65536 ? 0.f : (float)(65536.0 / (65536 - in->drop));
  return TS_OK;
}

ts_status check_rows(const char* who, int dtype, int64_t rows, int64_t cols) {
  using ts_host::fail;
  if (!ts_host::valid_dtype(dtype)) return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: bad dtype", who);
  if (rows < 0 || cols < 0)
    return fail(TS_ERR_SHAPE, "%s: bad shape [%lld, %lld]", who, (long long)rows,
                (long long)cols);
  return TS_OK;
}

template <typename T>
ts_status launch_dropout(const DropArgs& a, hipStream_t st) {
  const int64_t blocks = (a.total + 255) / 256;
  if (blocks > ts_plan::max_blocks(256))
    return ts_host::fail(TS_ERR_SHAPE, "dropout: tensor too large");
  if (a.res != nullptr)
    hipLaunchKernelGGL((dropout_kernel<T, true>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), dim3((unsigned)blocks), dim3(256), 0, st, a);
  return ts_host::check_launch("dropout_kernel");
}

template <typename T, typename W, int kTpr, int kKv, int kBlock>
ts_status launch_shape(const NormArgs& a, bool backward, int64_t grid, hipStream_t st) {
  if (grid > ts_plan::max_blocks(kBlock))
    return ts_host::fail(TS_ERR_SHAPE, "dropout_add_rmsnorm: too many rows");
  if (backward)
    hipLaunchKernelGGL((dropout_norm_bwd<T, W, kTpr, kKv, kBlock>), dim3((unsigned)grid),
                       dim3(kBlock), 0, st, a);
  else
    hipLaunchKernelGGL((dropout_norm_fwd<T, W, kTpr, kKv, kBlock>), dim3((unsigned)grid),
                       dim3(kBlock), 0, st, a);
  return ts_host::check_launch("dropout_norm");
}

template <typename T, typename W>
ts_status launch_norm(const NormArgs& a, bool backward, hipStream_t st) {
  constexpr int esize = sizeof(T);
  const ts_plan::DropNormPlan p =
      backward ? ts_plan::drop_norm_bwd_plan(a.groups, esize) : ts_plan::drop_norm_plan(a.groups);
  const int64_t steps = (a.rows + p.rows - 1) / p.rows;
  const int64_t grid = backward ? ts_plan::drop_norm_bwd_grid(a.rows, a.groups) : steps;
  switch (p.tpr * 8 + p.kv) {
    case 8 * 8 + 1: return launch_shape<T, W, 8, 1, 256>(a, backward, grid, st);
    case 32 * 8 + 1: return launch_shape<T, W, 32, 1, 256>(a, backward, grid, st);
    case 64 * 8 + 1: return launch_shape<T, W, 64, 1, 256>(a, backward, grid, st);
    case 64 * 8 + 2: return launch_shape<T, W, 64, 2, 256>(a, backward, grid, st);
    case 256 * 8 + 1: return launch_shape<T, W, 256, 1, 256>(a, backward, grid, st);
    case 256 * 8 + 2:
      if constexpr (esize == 2) return launch_shape<T, W, 256, 2, 256>(a, backward, grid, st);
      break;
    case 512 * 8 + 1: return launch_shape<T, W, 512, 1, 512>(a, backward, grid, st);
    case 512 * 8 + 2: return launch_shape<T, W, 512, 2, 512>(a, backward, grid, st);
    case 512 * 8 + 4: return launch_shape<T, W, 512, 4, 512>(a, backward, grid, st);
  }
  return ts_host::fail(TS_ERR_SHAPE, "dropout_add_rmsnorm: more than %d columns",
                       (int)ts_plan::kDropNormMaxCols);
}

template <typename T>
ts_status launch_norm_w(const NormArgs& a, bool backward, bool wide, hipStream_t st) {
  return wide ? launch_norm<T, float>(a, backward, st) : launch_norm<T, T>(a, backward, st);
}

ts_status dispatch_norm(const NormArgs& a, ts_dtype dtype, ts_dtype wdtype, bool backward,
                        hipStream_t st) {
  const bool wide = wdtype == TS_F32;
  switch (dtype) {
    case TS_BF16: return launch_norm_w<__bf16>(a, backward, wide, st);
    case TS_F16: return launch_norm_w<_Float16>(a, backward, wide, st);
    case TS_F32: return launch_norm<float, float>(a, backward, st);
  }
  return ts_host::fail(TS_ERR_UNSUPPORTED_DTYPE, "dropout_add_rmsnorm: bad dtype");
}

ts_status check_norm(const char* who, ts_dtype dtype, const void* weight, ts_dtype wdtype,
                     int64_t rows, int64_t cols) {
  using ts_host::fail;
  const ts_status s = check_rows(who, dtype, rows, cols);
  if (s != TS_OK) return s;
  if (wdtype != dtype && wdtype != TS_F32)
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: the weight must have x's dtype or fp32", who);
  if (cols < 1 || cols > ts_plan::kDropNormMaxCols)
    return fail(TS_ERR_SHAPE, "%s: 1 to %d columns, got %lld", who,
                (int)ts_plan::kDropNormMaxCols, (long long)cols);
  if (weight == nullptr) return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL weight", who);
  return TS_OK;
}

#define TS_TRY(x)                  \
  do {                             \
    const ts_status s_ = (x);      \
    if (s_ != TS_OK) return s_;    \
  } while (0)

}  // namespace

extern "C" ts_status ts_dropout_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                                    void* out, int64_t ldo, ts_dtype dtype, int64_t rows,
                                    int64_t cols, const ts_dropout_rng* rng, ts_stream_t stream) {
  using ts_host::fail;
  DropArgs a{};
  TS_TRY(check_rows("dropout_fwd", dtype, rows, cols));
  TS_TRY(rng_of("dropout_fwd", rng, a.rng));
  if (rows == 0 || cols == 0) return TS_OK;
  if (x == nullptr || out == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "dropout_fwd: NULL pointer");
  if (ldx < cols || ldo < cols || (residual != nullptr && ldr < cols))
    return fail(TS_ERR_SHAPE, "dropout_fwd: row stride shorter than a row");
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldr = ldr;
  a.out = out;
  a.ldo = ldo;
  a.cols = cols;
  a.groups = (cols + 7) / 8;
  if (rows > ((int64_t)1 << 34) / a.groups)
    return fail(TS_ERR_SHAPE, "dropout_fwd: tensor too large");
  a.total = rows * a.groups;
  // whole groups without gaps between rows are one row of the same groups: no division
  if (cols % 8 == 0 && ldx == cols && ldo == cols && (residual == nullptr || ldr == cols)) {
    a.cols = rows * cols;
    a.groups = a.total;
  }
  a.one_row = a.groups == a.total;
  a.magic = ts_plan::magic64_for((uint64_t)a.groups);  // total * groups < 2^64
  if (!a.one_row && !ts_plan::magic64_exact((uint64_t)a.total, (uint64_t)a.groups))
    return fail(TS_ERR_SHAPE, "dropout_fwd: tensor too large");
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_BF16: return launch_dropout<__bf16>(a, st);
    case TS_F16: return launch_dropout<_Float16>(a, st);
    case TS_F32: return launch_dropout<float>(a, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "dropout_fwd: bad dtype");
}

extern "C" ts_status ts_dropout_add_rmsnorm_fwd(const void* x, int64_t ldx, const void* residual,
                                                int64_t ldr, ts_dtype dtype, const void* weight,
                                                ts_dtype wdtype, void* y, void* h, float* rstd,
                                                int64_t rows, int64_t cols, float eps,
                                                const ts_dropout_rng* rng, ts_stream_t stream) {
  using ts_host::fail;
  NormArgs a{};
  TS_TRY(check_norm("dropout_add_rmsnorm_fwd", dtype, weight, wdtype, rows, cols));
  TS_TRY(rng_of("dropout_add_rmsnorm_fwd", rng, a.rng));
  if (!(eps >= 0.f))
    return fail(TS_ERR_INVALID_ARGUMENT, "dropout_add_rmsnorm_fwd: eps must be >= 0");
  if (rows == 0) return TS_OK;
  if (x == nullptr || residual == nullptr || y == nullptr || h == nullptr || rstd == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "dropout_add_rmsnorm_fwd: NULL pointer");
  if (ldx < cols || ldr < cols)
    return fail(TS_ERR_SHAPE, "dropout_add_rmsnorm_fwd: row stride shorter than a row");
  a.x = x;
  a.ldx = ldx;
  a.res = residual;
  a.ldr = ldr;
  a.w = weight;
  a.y = y;
  a.h = h;
  a.rstd = rstd;
  a.rows = rows;
  a.cols = cols;
  a.groups = (cols + 7) / 8;
  a.eps = eps;
  return dispatch_norm(a, dtype, wdtype, false, static_cast<hipStream_t>(stream));
}

extern "C" size_t ts_dropout_add_rmsnorm_bwd_workspace_size(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || cols > ts_plan::kDropNormMaxCols) return 0;
  return (size_t)ts_plan::drop_norm_bwd_grid(rows, (cols + 7) / 8) * cols * sizeof(float);
}

extern "C" ts_status ts_dropout_add_rmsnorm_bwd(
    const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh,
    ts_dtype dtype, const void* weight, ts_dtype wdtype, const float* rstd, void* dx, void* dres,
    void* dw, int64_t rows, int64_t cols, const ts_dropout_rng* rng, void* workspace,
    size_t workspace_bytes, ts_stream_t stream) {
  using ts_host::fail;
  NormArgs a{};
  TS_TRY(check_norm("dropout_add_rmsnorm_bwd", dtype, weight, wdtype, rows, cols));
  TS_TRY(rng_of("dropout_add_rmsnorm_bwd", rng, a.rng));
  if (rows == 0)
    return fail(TS_ERR_SHAPE, "dropout_add_rmsnorm_bwd: no rows (dw is zero)");
  if (h == nullptr || rstd == nullptr || (dy == nullptr && dh == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "dropout_add_rmsnorm_bwd: NULL pointer");
  if ((dy != nullptr && lddy < cols) || (dh != nullptr && lddh < cols) || ldh < cols)
    return fail(TS_ERR_SHAPE, "dropout_add_rmsnorm_bwd: row stride shorter than a row");
  const size_t need = ts_dropout_add_rmsnorm_bwd_workspace_size(rows, cols);
  if (dw != nullptr && (workspace == nullptr || workspace_bytes < need ||
                        !ts_host::aligned16(workspace)))
    return fail(TS_ERR_WORKSPACE, "dropout_add_rmsnorm_bwd: workspace of %zu bytes, need %zu",
                workspace_bytes, need);
  a.dy = dy;
  a.lddy = lddy;
  a.dh = dh;
  a.lddh = lddh;
  a.h = const_cast<void*>(h);
  a.ldh = ldh;
  a.w = weight;
  a.rstd = const_cast<float*>(rstd);
  a.dx = dx;
  a.dres = dres;
  a.part = dw != nullptr ? static_cast<float*>(workspace) : nullptr;
  a.rows = rows;
  a.cols = cols;
  a.groups = (cols + 7) / 8;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TS_TRY(dispatch_norm(a, dtype, wdtype, true, st));
  if (dw == nullptr) return TS_OK;
  const int64_t nparts = ts_plan::drop_norm_bwd_grid(rows, a.groups);
  const dim3 grid((unsigned)((cols + kSumCols - 1) / kSumCols)), block(kSumCols * kSumSlices);
  switch (wdtype) {
    case TS_BF16:
      hipLaunchKernelGGL(dropout_dw_sum<__bf16>, grid, block, 0, st, a.part, nparts, cols,
                         static_cast<__bf16*>(dw));
      break;
    case TS_F16:
      hipLaunchKernelGGL(dropout_dw_sum<_Float16>, grid, block, 0, st, a.part, nparts, cols,
                         static_cast<_Float16*>(dw));
      break;
    default:
      hipLaunchKernelGGL(dropout_dw_sum<float>, grid, block, 0, st, a.part, nparts, cols,
                         static_cast<float*>(dw));
  }
  return ts_host::check_launch("dropout_dw_sum");
}
