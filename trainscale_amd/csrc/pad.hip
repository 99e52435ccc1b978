// Matrices of 16-bit elements copied into contiguous, zero-padded ones (or out of padded ones), up
// to 8 of them in a launch: what the MFMA products need of operands whose sizes, strides or
// addresses they do not take.
//   dst[r][c] = r < rows and c < cols ? src[r row_stride + c col_stride] : 0
//
// Bound by HBM where the matrices are large, by the launch where they are small, so all of a call's
// operands share one. A workgroup copies a 64 x 64 tile, 8 elements of the closer-strided dimension
// to a lane, 16 bytes at any element address where that dimension is dense; a matrix stored column
// by column is turned in LDS, so that both sides of it stay in 128-byte runs. Measured on MI355X,
// bf16: [8192, 4100] 36 us (3.8 TB/s; torch's fill and copy 35), [4096, 14336] stored by columns 39 us
// (6.1 TB/s; torch's copy 233); the gated block at 34 x 168 x 145 28 us a forward, 54 when each
// operand had a fill and a copy of its own.
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

constexpr int kPadJobs = 8;
constexpr int kPadTile = 64;

struct PadJob {
  const uint16_t* src;
  int64_t rs, cs, rows, cols;
  uint16_t* dst;
  int64_t drows, dcols;
};
struct PadArgs {
  PadJob job[kPadJobs];
  int64_t end[kPadJobs];  // workgroups up to and with this job
};

// v[i] = p[i * stride], i < n, the others 0.
__device__ inline void gather8(const uint16_t* p, int64_t stride, int n, uint16_t (&v)[8]) {
  if (n >= 8 && stride == 1) {
    const u32x4 q = ld16_any(p);
    __builtin_memcpy(v, &q, 16);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i * stride] : (uint16_t)0;
}
__device__ inline void put8(uint16_t* p, const uint16_t (&v)[8], int64_t n) {
  if (n >= 8) {
    u32x4 q;
    __builtin_memcpy(&q, v, 16);
    st16_any(p, q);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < n) p[i] = v[i];
}
__device__ inline int clip8(int64_t n) { return n >= 8 ? 8 : n > 0 ? (int)n : 0; }

__global__ __launch_bounds__(256) void pad_matrices(const PadArgs a) {
  __shared__ uint16_t tile[kPadTile][kPadTile + 2];
  const int64_t bid = blockIdx.x;
  int j = 0;
  while (j < kPadJobs - 1 && bid >= a.end[j]) ++j;
  const PadJob& p = a.job[j];
  const int64_t t = bid - (j ? a.end[j - 1] : 0), ct = (p.dcols + kPadTile - 1) / kPadTile;
  const int64_t r0 = t / ct * kPadTile, c0 = t % ct * kPadTile;
  const bool turn = p.cs > p.rs;
  const int k = threadIdx.x & 7, line = threadIdx.x >> 3;  // 8 groups of 8 of 32 lines
  if (turn) {
#pragma unroll
    for (int h = 0; h < kPadTile; h += 32) {
      const int64_t c = c0 + line + h, r = r0 + k * 8;
      uint16_t v[8];
      gather8(p.src + r * p.rs + c * p.cs, p.rs, c < p.cols ? clip8(p.rows - r) : 0, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) tile[k * 8 + i][line + h] = v[i];
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < kPadTile; h += 32) {
    const int64_t r = r0 + line + h, c = c0 + k * 8;
    uint16_t v[8];
    if (turn) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = tile[line + h][k * 8 + i];
    } else {
      gather8(p.src + r * p.rs + c * p.cs, p.cs, r < p.rows ? clip8(p.cols - c) : 0, v);
    }
    if (r < p.drows) put8(p.dst + r * p.dcols + c, v, p.dcols - c);
  }
}

}  // namespace

extern "C" ts_status ts_pad_matrices(const ts_pad_job* jobs, int32_t count, ts_dtype dtype,
                                     ts_stream_t stream) {
  using ts_host::fail;
  if (dtype != TS_BF16 && dtype != TS_F16)
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "pad_matrices: dtype must be bf16 or fp16");
  if (count < 0 || count > kPadJobs || (count > 0 && jobs == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "pad_matrices: 0 to %d jobs, got %d", kPadJobs,
                (int)count);
  PadArgs a{};
  int64_t blocks = 0;
  for (int i = 0; i < kPadJobs; ++i) {
    if (i < count) {
      const ts_pad_job& j = jobs[i];
      constexpr int64_t kMost = (int64_t)1 << 40;  // keeps every product below in 64 bits
      if (j.rows < 0 || j.cols < 0 || j.dst_rows < j.rows || j.dst_cols < j.cols ||
          j.dst_rows > kMost || j.dst_cols > kMost)
        return fail(TS_ERR_SHAPE, "pad_matrices: [%lld, %lld] into [%lld, %lld]",
                    (long long)j.rows, (long long)j.cols, (long long)j.dst_rows,
                    (long long)j.dst_cols);
      if (j.row_stride < 0 || j.col_stride < 0)
        return fail(TS_ERR_SHAPE, "pad_matrices: negative stride");
      const int64_t rt = (j.dst_rows + kPadTile - 1) / kPadTile;
      const int64_t ct = (j.dst_cols + kPadTile - 1) / kPadTile;
      if (rt > 0 && ct > 0) {
        if (j.dst == nullptr || (j.src == nullptr && j.rows > 0 && j.cols > 0))
          return fail(TS_ERR_INVALID_ARGUMENT, "pad_matrices: NULL pointer");
        if (((reinterpret_cast<uintptr_t>(j.src) | reinterpret_cast<uintptr_t>(j.dst)) & 1u) != 0)
          return fail(TS_ERR_INVALID_ARGUMENT, "pad_matrices: pointers must be 2-byte aligned");
        if (rt > ts_plan::max_blocks(256) / ct || rt * ct > ts_plan::max_blocks(256) - blocks)
          return fail(TS_ERR_SHAPE, "pad_matrices: too large");
        a.job[i] = PadJob{static_cast<const uint16_t*>(j.src), j.row_stride, j.col_stride, j.rows,
                          j.cols, static_cast<uint16_t*>(j.dst), j.dst_rows, j.dst_cols};
        blocks += rt * ct;
      }
    }
    a.end[i] = blocks;
  }
  if (blocks == 0) return TS_OK;
  hipLaunchKernelGGL(pad_matrices, dim3((unsigned)blocks), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  return ts_host::check_launch("pad_matrices");
}
