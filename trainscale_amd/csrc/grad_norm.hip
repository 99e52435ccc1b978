// Global gradient norm over many tensors and clipping, for gfx950:
//   norm = sqrt(sum over all tensors of x^2),  out = x * min(1, max_norm / (norm + 1e-6))
//
// HBM-bound: the norm reads every gradient once, the scaling reads it again and writes it; the
// scale depends on all of the data, so no order of the work saves the second read (walking back
// through what the 256 MB last-level cache might still hold measured no gain at 0.5 and 2.8 GB).
// A model has hundreds of tensors of very different sizes, so one launch takes up to kTensors of
// one type pair: their pointers and sizes travel in the kernel's arguments (no table in device
// memory to allocate, copy or keep alive, and a captured graph holds its own copy). The tensors
// are cut into chunks of one step of a workgroup, numbered through.
//
// Norm: at most 8 workgroups a CU, workgroup b takes chunks b, b + G, b + 2G, ...: the running
// workgroups work on a compact window of memory whatever the tensors' sizes. 2.8 GB of bf16 in
// 37 tensors: 407 us, 6.9 TB/s (through the caches instead of streaming: 466 us).
// Scaling: one short chunk a workgroup, all in flight at once; 2.8 GB of bf16 into 5.6 GB of fp32
// 1326 us, 6.3 TB/s, where a 4 GiB copy reaches 6.5 (2048 workgroups that walk chunks: 1556 us;
// 16-byte loads, which make each store instruction skip every other 16 bytes: 2091 us).
//
// Sums: the squares of one 16-byte vector are added in fp32 and that sum goes into a double.
// Where the vector's sum leaves [2^-80, 2^100] (values whose squares overflow or underflow fp32,
// zeros, NaN) its squares are formed in double instead, so the norm is the double one's for any
// finite gradients. Every workgroup writes one double; they are added in a fixed order, so the
// norm does not depend on timing.
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

constexpr int kThreads = ts_plan::kGradThreads;
constexpr int kGrid = ts_plan::kGradGrid;
constexpr int kTensors = ts_plan::kGradTensors;
// 16-byte vectors each thread has in flight: those of a chunk
constexpr int kNormVecs = ts_plan::kGradNormPieces;
constexpr int kScaleVecs = ts_plan::kGradScalePieces;

struct Table {
  const void* src[kTensors];
  void* dst[kTensors];
  int64_t numel[kTensors];
  int32_t chunk_end[kTensors];  // chunks of tensors 0 .. t
};
static_assert(sizeof(Table) <= 3840, "kernel arguments stay below 4 KB");

constexpr float kSumMin = 0x1p-80f, kSumMax = 0x1p100f;

// Sum of squares of V values as a double.
template <int V>
__device__ inline double vec_squares(const float (&f)[V]) {
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < V; ++i) s = __builtin_fmaf(f[i], f[i], s);
  if (s >= kSumMin && s <= kSumMax) return (double)s;
  double d = 0.;
#pragma unroll
  for (int i = 0; i < V; ++i) d += (double)f[i] * (double)f[i];
  return d;
}

// Sum over the workgroup in a fixed order; every thread gets it. Two barriers.
template <int kT>
__device__ inline double block_sum_f64(double v, double* lds) {
#pragma unroll
  for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  const int wid = threadIdx.x / kWave;
  if ((threadIdx.x & (kWave - 1)) == 0) lds[wid] = v;
  __syncthreads();
  double t = 0.;
#pragma unroll
  for (int i = 0; i < kT / kWave; ++i) t += lds[i];
  __syncthreads();
  return t;
}

__device__ inline int find_tensor(const Table& tab, int count, int chunk) {
  return ts_plan::grad_find_tensor(tab.chunk_end, count, chunk);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void grad_squares(Table tab, int count, int chunks,
                                                         double* __restrict__ partial) {
  constexpr int V = Elt<T>::kVec;
  constexpr int64_t kChunk = ts_plan::grad_chunk(sizeof(T), kNormVecs);
  __shared__ double lds[kThreads / kWave];
  double acc = 0.;
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int t = find_tensor(tab, count, c);
    const int64_t first = (int64_t)(c - (t ? tab.chunk_end[t - 1] : 0)) * kChunk;
    const T* x = static_cast<const T*>(tab.src[t]) + first;
    const int64_t left = tab.numel[t] - first;
    const int n = (int)(left < kChunk ? left : kChunk);
    const int nvec = n / V;
    if (n == kChunk) {
      u32x4 q[kNormVecs];
#pragma unroll
      for (int k = 0; k < kNormVecs; ++k)
        q[k] = ld16_any_stream(x + (threadIdx.x + k * kThreads) * V);
#pragma unroll
      for (int k = 0; k < kNormVecs; ++k) {
        float f[V];
        Elt<T>::unpack(q[k], f);
        acc += vec_squares<V>(f);
      }
      continue;
    }
    for (int v = threadIdx.x; v < nvec; v += kThreads) {
      float f[V];
      Elt<T>::unpack(ld16_any_stream(x + v * V), f);
      acc += vec_squares<V>(f);
    }
    const int e = nvec * V + threadIdx.x;  // fewer than V values behind the last vector
    if (e < n) {
      const double d = (double)Elt<T>::load1(x + e);
      acc += d * d;
    }
  }
  const double s = block_sum_f64<kThreads>(acc, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The partial sums' total, in the same order in every workgroup that asks for it. The scaling's
// workgroups form it themselves while it is short, which saves a launch between the two passes;
// past kOwnParts partial sums (8 MB of gradients in one launch) a launch of its own forms the norm.
// In place below the limit, bf16: 1 partial sum 4.0 us against 5.9 with the launch, 128 5.1 and 6.7,
// 512 6.6 and 7.1, 1024 8.4 and 8.0, 4096 23.5 and 17.0.
constexpr int kOwnParts = 512;
constexpr int kFinalThreads = 1024;

template <int kT>
__device__ inline double total_squares(const double* __restrict__ partial, int nparts,
                                       double* lds) {
  double s = 0.;
  for (int i = threadIdx.x; i < nparts; i += kT) s += partial[i];
  return block_sum_f64<kT>(s, lds);
}

__global__ __launch_bounds__(kFinalThreads) void grad_norm_final(const double* __restrict__ partial,
                                                            int nparts, float* __restrict__ norm) {
  __shared__ double lds[kFinalThreads / kWave];
  const double s = total_squares<kFinalThreads>(partial, nparts, lds);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// min(1, max_norm / (norm + 1e-6)); NaN stays NaN (the gradients of such a step are lost, and
// show it)
__device__ inline float clip_coef(double norm, float max_norm) {
  const double c = (double)max_norm / (norm + 1e-6);
  return c >= 1. ? 1.f : (float)c;
}

// N elements of T at any element address: 16 bytes, or 8 for 16-bit gradients that go to fp32,
// so that every lane of a wave stores 16 bytes next to its neighbour's.
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
template <typename T, int N>
struct Piece {
  u32x4 q;
  __device__ inline void load(const T* x) {
    if constexpr (N == Elt<T>::kVec) {
      q = ld16_any_stream(x);
    } else {
      const u32x2_any h = __builtin_nontemporal_load(reinterpret_cast<const u32x2_any*>(x));
      q = u32x4{h[0], h[1], 0u, 0u};
    }
  }
  __device__ inline void unpack(float (&f)[N]) const {
    float all[Elt<T>::kVec];
    Elt<T>::unpack(q, all);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = all[i];
  }
};

// The norm comes from `partial` (nparts > 0; workgroup 0 of the first launch writes it to
// norm_out) or from *norm_in.
template <typename T, typename D>
__global__ __launch_bounds__(kThreads) void grad_scale(Table tab, int count, int chunks,
                                                       const double* __restrict__ partial,
                                                       int nparts, const float* norm_in,
                                                       float* norm_out, float max_norm,
                                                       int in_place) {
  constexpr int V = Elt<D>::kVec;
  constexpr int64_t kChunk = ts_plan::grad_chunk(sizeof(D), kScaleVecs);
  __shared__ double lds[kThreads / kWave];
  double norm;
  if (nparts > 0) {
    // rounded as the norm that is returned: the factor is the same whoever forms it, and 0 for
    // norms beyond fp32's range
    const float rounded = (float)sqrt(total_squares<kThreads>(partial, nparts, lds));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = rounded;
    norm = (double)rounded;
  } else {
    norm = (double)*norm_in;
  }
  const float coef = clip_coef(norm, max_norm);
  if (coef == 1.f && in_place) return;  // every gradient stays as it is
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {  // one chunk, but for 64 GB and more
    const int t = find_tensor(tab, count, c);
    if (coef == 1.f && tab.src[t] == tab.dst[t]) continue;
    const int64_t first = (int64_t)(c - (t ? tab.chunk_end[t - 1] : 0)) * kChunk;
    const T* x = static_cast<const T*>(tab.src[t]) + first;
    D* o = static_cast<D*>(tab.dst[t]) + first;
    const int64_t left = tab.numel[t] - first;
    const int n = (int)(left < kChunk ? left : kChunk);
    const int nvec = n / V;
    Piece<T, V> q[kScaleVecs];
#pragma unroll
    for (int k = 0; k < kScaleVecs; ++k) {
      const int v = threadIdx.x + k * kThreads;
      if (v < nvec) q[k].load(x + v * V);
    }
#pragma unroll
    for (int k = 0; k < kScaleVecs; ++k) {
      const int v = threadIdx.x + k * kThreads;
      if (v < nvec) {
        float f[V];
        q[k].unpack(f);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] *= coef;
        st16_any_stream(o + v * V, Elt<D>::pack(f));
      }
    }
    const int e = nvec * V + threadIdx.x;
    if (e < n) Elt<D>::store1(o + e, Elt<T>::load1(x + e) * coef);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

struct Lists {
  const void* const* src;
  void* const* dst;
  const int64_t* numel;
  const int32_t* dtype;
  const int32_t* dst_dtype;
  int64_t count;
};

ts_status check_lists(const char* what, const Lists& l, bool dst) {
  using ts_host::fail;
  if (l.count < 0) return fail(TS_ERR_SHAPE, "%s: negative tensor count", what);
  if (l.count == 0) return TS_OK;
  if (l.src == nullptr || l.numel == nullptr || l.dtype == nullptr ||
      (dst && (l.dst == nullptr || l.dst_dtype == nullptr)))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL list", what);
  int64_t chunks = 0;
  for (int64_t i = 0; i < l.count; ++i) {
    if (l.numel[i] < 0) return fail(TS_ERR_SHAPE, "%s: tensor %lld has a negative size", what,
                                    (long long)i);
    if (!ts_host::valid_dtype(l.dtype[i]) || (dst && !ts_host::valid_dtype(l.dst_dtype[i])))
      return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: tensor %lld has a bad dtype", what, (long long)i);
    if (dst && l.dst_dtype[i] != l.dtype[i] && l.dst_dtype[i] != TS_F32)
      return fail(TS_ERR_UNSUPPORTED_DTYPE,
                  "%s: output %lld is neither fp32 nor of its gradient's dtype", what,
                  (long long)i);
    if (l.numel[i] == 0) continue;
    if (l.src[i] == nullptr || (dst && l.dst[i] == nullptr))
      return fail(TS_ERR_INVALID_ARGUMENT, "%s: tensor %lld is NULL", what, (long long)i);
    const uintptr_t size = ts_host::dtype_size((ts_dtype)l.dtype[i]);
    const uintptr_t dsize = dst ? ts_host::dtype_size((ts_dtype)l.dst_dtype[i]) : 1;
    if (reinterpret_cast<uintptr_t>(l.src[i]) % size != 0 ||
        (dst && reinterpret_cast<uintptr_t>(l.dst[i]) % dsize != 0))
      return fail(TS_ERR_INVALID_ARGUMENT, "%s: tensor %lld is not aligned to its elements", what,
                  (long long)i);
    // the shorter of the two kernels' chunks
    const int64_t c = ts_plan::grad_chunks(l.numel[i], ts_plan::grad_chunk(4, 2));
    if (c > ts_plan::kGradMaxChunks - chunks)
      return fail(TS_ERR_SHAPE, "%s: tensors too large", what);
    chunks += c;
  }
  return TS_OK;
}

int64_t norm_chunk(int32_t t) {
  return ts_plan::grad_chunk((int)ts_host::dtype_size((ts_dtype)t), kNormVecs);
}
int64_t scale_chunk(int32_t t) {
  return ts_plan::grad_chunk((int)ts_host::dtype_size((ts_dtype)t), kScaleVecs);
}

// Calls f(table, tensors, chunks, dtype, dst dtype) for groups of up to kTensors tensors of one
// type pair, in a fixed order.
template <typename F>
ts_status for_groups(const Lists& l, bool dst, F f) {
  static const int32_t pairs[5][2] = {
      {TS_F32, TS_F32}, {TS_BF16, TS_BF16}, {TS_F16, TS_F16}, {TS_BF16, TS_F32}, {TS_F16, TS_F32}};
  Table tab;
  for (int p = 0; p < (dst ? 5 : 3); ++p) {
    int n = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i <= l.count; ++i) {
      if (n == kTensors || (i == l.count && n > 0)) {
        const ts_status s = f(tab, n, (int)chunks, pairs[p][0], pairs[p][1]);
        if (s != TS_OK) return s;
        n = 0;
        chunks = 0;
      }
      if (i == l.count) break;
      if (l.dtype[i] != pairs[p][0] || (dst && l.dst_dtype[i] != pairs[p][1]) || l.numel[i] == 0)
        continue;
      chunks += ts_plan::grad_chunks(l.numel[i], dst ? scale_chunk(pairs[p][1]) : norm_chunk(pairs[p][0]));
      tab.src[n] = l.src[i];
      tab.dst[n] = dst ? l.dst[i] : nullptr;
      tab.numel[n] = l.numel[i];
      tab.chunk_end[n] = (int32_t)chunks;
      ++n;
    }
  }
  return TS_OK;
}

ts_status launch_squares(const Lists& l, double* partial, int64_t capacity, int* nparts,
                         hipStream_t st) {
  *nparts = 0;
  return for_groups(l, false, [&](const Table& tab, int n, int chunks, int32_t t, int32_t) {
    const unsigned g = (unsigned)(chunks < kGrid ? chunks : kGrid);
    if (*nparts + (int64_t)g > capacity)
      return ts_host::fail(TS_ERR_WORKSPACE, "grad_norm: workspace too small");
    double* out = partial + *nparts;
    *nparts += (int)g;
    const dim3 grid(g), block(kThreads);
    switch (t) {
      case TS_BF16:
        hipLaunchKernelGGL(grad_squares<__bf16>, grid, block, 0, st, tab, n, chunks, out);
        break;
      case TS_F16:
        hipLaunchKernelGGL(grad_squares<_Float16>, grid, block, 0, st, tab, n, chunks, out);
        break;
      default:
        hipLaunchKernelGGL(grad_squares<float>, grid, block, 0, st, tab, n, chunks, out);
    }
    return ts_host::check_launch("grad_squares");
  });
}

ts_status launch_scale(const Lists& l, const double* partial, int nparts, const float* norm_in,
                       float* norm_out, float max_norm, hipStream_t st) {
  return for_groups(l, true, [&](const Table& tab, int n, int chunks, int32_t t, int32_t d) {
    const dim3 grid((unsigned)(chunks < ts_plan::kGradScaleGrid ? chunks : ts_plan::kGradScaleGrid)),
        block(kThreads);
    int in_place = 1;
    for (int i = 0; i < n; ++i) in_place &= tab.src[i] == tab.dst[i];
#define TS_SCALE(T, D)                                                                         \
  hipLaunchKernelGGL((grad_scale<T, D>), grid, block, 0, st, tab, n, chunks, partial, nparts, \
                     norm_in, norm_out, max_norm, in_place)
    if (t == TS_F32) {
      TS_SCALE(float, float);
    } else if (t == TS_BF16) {
      if (d == TS_BF16) TS_SCALE(__bf16, __bf16); else TS_SCALE(__bf16, float);
    } else {
      if (d == TS_F16) TS_SCALE(_Float16, _Float16); else TS_SCALE(_Float16, float);
    }
#undef TS_SCALE
    norm_out = nullptr;  // the first launch has written it
    return ts_host::check_launch("grad_scale");
  });
}

ts_status check_max_norm(const char* what, float max_norm) {
  if (!(max_norm >= 0.f))
    return ts_host::fail(TS_ERR_INVALID_ARGUMENT, "%s: max_norm must be >= 0", what);
  return TS_OK;
}

ts_status check_workspace(const char* what, const void* ws, size_t bytes, int64_t count) {
  if (bytes < ts_grad_norm_workspace_size(count))
    return ts_host::fail(TS_ERR_WORKSPACE, "%s: workspace too small", what);
  if (ws == nullptr || reinterpret_cast<uintptr_t>(ws) % 8 != 0)
    return ts_host::fail(TS_ERR_WORKSPACE, "%s: workspace missing or not 8-byte aligned", what);
  return TS_OK;
}

ts_status launch_final(const double* partial, int nparts, float* norm, hipStream_t st) {
  hipLaunchKernelGGL(grad_norm_final, dim3(1), dim3(kFinalThreads), 0, st, partial, nparts, norm);
  return ts_host::check_launch("grad_norm_final");
}

}  // namespace

extern "C" size_t ts_grad_norm_workspace_size(int64_t count) {
  return (size_t)ts_plan::grad_norm_parts(count) * sizeof(double);
}

extern "C" ts_status ts_grad_norm(const void* const* tensors, const int64_t* numels,
                                  const int32_t* dtypes, int64_t count, float* norm,
                                  void* workspace, size_t workspace_bytes, ts_stream_t stream) {
  const Lists l{tensors, nullptr, numels, dtypes, nullptr, count};
  ts_status s = check_lists("grad_norm", l, false);
  if (s != TS_OK) return s;
  if (norm == nullptr) return ts_host::fail(TS_ERR_INVALID_ARGUMENT, "grad_norm: NULL norm");
  s = check_workspace("grad_norm", workspace, workspace_bytes, count);
  if (s != TS_OK) return s;
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int nparts = 0;
  s = launch_squares(l, partial, (int64_t)(workspace_bytes / sizeof(double)), &nparts, st);
  if (s != TS_OK) return s;
  return launch_final(partial, nparts, norm, st);
}

extern "C" ts_status ts_grad_scale(const void* const* tensors, void* const* outs,
                                   const int64_t* numels, const int32_t* dtypes,
                                   const int32_t* out_dtypes, int64_t count, const float* norm,
                                   float max_norm, ts_stream_t stream) {
  const Lists l{tensors, outs, numels, dtypes, out_dtypes, count};
  ts_status s = check_lists("grad_scale", l, true);
  if (s != TS_OK) return s;
  if (norm == nullptr) return ts_host::fail(TS_ERR_INVALID_ARGUMENT, "grad_scale: NULL norm");
  s = check_max_norm("grad_scale", max_norm);
  if (s != TS_OK) return s;
  return launch_scale(l, nullptr, 0, norm, nullptr, max_norm, static_cast<hipStream_t>(stream));
}

extern "C" ts_status ts_grad_clip(const void* const* tensors, void* const* outs,
                                  const int64_t* numels, const int32_t* dtypes,
                                  const int32_t* out_dtypes, int64_t count, float max_norm,
                                  float* norm, void* workspace, size_t workspace_bytes,
                                  ts_stream_t stream) {
  const Lists l{tensors, outs, numels, dtypes, out_dtypes, count};
  ts_status s = check_lists("grad_clip", l, true);
  if (s != TS_OK) return s;
  if (norm == nullptr) return ts_host::fail(TS_ERR_INVALID_ARGUMENT, "grad_clip: NULL norm");
  s = check_max_norm("grad_clip", max_norm);
  if (s != TS_OK) return s;
  s = check_workspace("grad_clip", workspace, workspace_bytes, count);
  if (s != TS_OK) return s;
  hipStream_t st = static_cast<hipStream_t>(stream);
  double* partial = static_cast<double*>(workspace);
  int nparts = 0;
  s = launch_squares(l, partial, (int64_t)(workspace_bytes / sizeof(double)), &nparts, st);
  if (s != TS_OK) return s;
  if (nparts == 0 || nparts > kOwnParts) {  // (no values at all: the norm is 0)
    s = launch_final(partial, nparts, norm, st);
    if (s != TS_OK) return s;
    return launch_scale(l, nullptr, 0, norm, nullptr, max_norm, st);
  }
  return launch_scale(l, partial, nparts, nullptr, norm, max_norm, st);
}
