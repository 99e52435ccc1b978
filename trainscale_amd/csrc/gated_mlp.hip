// Gated feed-forward block for gfx950, forward and backward:
//   g = x Wg^T, u = x Wu^T, a = act(g) * u, y = a Wd^T          (x [N, H], Wg and Wu [F, H], Wd [O, F])
//   da = dy Wd, dg = da u act'(g), du = da act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T a
// act: silu g s(g); gelu g Phi(g); its tanh form g s(2 sqrt(2/pi) (g + 0.044715 g^3)); relu, with
// s(z) = 1 / (1 + e^-z). Without Wd, y = a.
//
// Products run on the MFMA core (gemm.hpp), 16-bit operands and fp32 sums. The backward's operands
// are transposes of what is in memory and are read in place, as MN-major operands: transposed copies
// of the weights for da and dx were slower than that at every size (N 8190, H 8192, F 4096: backward
// 2400 us in place, 2510 with copies). What is fused:
//   * Both projections are one product: a workgroup's 256 columns are the same 128 columns of g
//     and of u, so that a lane holds g and u of one element and forms a in registers; x is read
//     once for both. Where a backward will follow, the epilogue also writes what it multiplies da
//     by, u act'(g) and act(g), in fp32: kept in 16 bits, g and u would add their roundings to
//     those of dg and du (measured rms error of dx and the projections' gradients 1.76 of one bf16
//     rounding against 1.41).
//   * da never reaches memory: the epilogue of dy Wd reads the two factors and writes dg and du.
//   * dx sums both products in one accumulation (K is the concatenation of dg and du), and
//     dx, dWg, dWu and dWd, which are independent, share one grid.
// a is rounded to 16 bits between the products, as dg and du are: MFMA operands are 16-bit.
//
// Bound by the matrix cores (at the power limit) from a few hundred rows on, by reading the weights
// below. Measured on MI355X, N 8192, H = O = 4096, F 14336 bf16: projections 1585 us (1.21 PFLOP/s),
// down 705 (1.37), gradients of g and u 965 (1.00: their epilogue moves 1.4 GB that no product hides;
// starting workgroups apart changed nothing), dx and the weights' gradients 3634-3707 (1.30-1.32); the
// library's 8192^3 products reach 1.63 with k contiguous in both operands, as the first two, 1.39 in
// one, as da and dx, and 1.21 in neither. Without w_down its place is taken by mlp_gate_bwd, 317 us
// there (5.3 TB/s).
#include <math.h>

#include "common.hpp"
#include "gemm.hpp"
#include "plan.hpp"

namespace {

using namespace ts;
using ts_gemm::AccOf;
using ts_gemm::Cfg;
using ts_gemm::f32x4;
using ts_gemm::kKMajor;
using ts_gemm::kMNMajor;
using ts_gemm::wide_col;
using ts_gemm::widen;

// ---------------------------------------------------------------------------
// Activations. Each keeps NaN, and the relative accuracy of small values of either sign.
// ---------------------------------------------------------------------------
__device__ inline float sigmoid_f(float z) {
  return __builtin_amdgcn_rcpf(1.f + fast_exp2(-z * kLog2e));
}

constexpr float kGeluK = 0.7978845608028654f;   // sqrt(2 / pi)
constexpr float kGeluC = 0.044715f;
constexpr float kSqrtHalf = 0.7071067811865476f;
constexpr float kInvSqrt2Pi = 0.3989422804014327f;
// Beyond this the tanh form is g or 0 in fp32; its polynomial would overflow far out.
constexpr float kGeluFar = 30.f;

// act(g), and its derivative in d.
template <int kAct>
__device__ inline float act_d(float g, float& d) {
  if constexpr (kAct == TS_ACT_SILU) {
    const float s = sigmoid_f(g);
    d = s * (1.f + g * (1.f - s));
    return g * s;
  } else if constexpr (kAct == TS_ACT_GELU) {
    const float cdf = 0.5f * erfcf(-kSqrtHalf * g);
    d = cdf + g * kInvSqrt2Pi * fast_exp2(-0.5f * kLog2e * g * g);
    return g * cdf;
  } else if constexpr (kAct == TS_ACT_GELU_TANH) {
    const float c = fabsf(g) > kGeluFar ? copysignf(kGeluFar, g) : g;
    const float s = sigmoid_f(2.f * kGeluK * c * (1.f + kGeluC * c * c));
    d = s + c * s * (1.f - s) * 2.f * kGeluK * (1.f + 3.f * kGeluC * c * c);
    return g * s;
  } else {
    d = g > 0.f ? 1.f : g == g ? 0.f : g;
    return g < 0.f ? 0.f : g;
  }
}

// Calls f with the activation as a compile-time constant (a uniform branch).
template <typename F>
__device__ inline void with_act(int act, F&& f) {
  switch (act) {
    case TS_ACT_SILU: f(std::integral_constant<int, TS_ACT_SILU>()); break;
    case TS_ACT_GELU: f(std::integral_constant<int, TS_ACT_GELU>()); break;
    case TS_ACT_GELU_TANH: f(std::integral_constant<int, TS_ACT_GELU_TANH>()); break;
    default: f(std::integral_constant<int, TS_ACT_RELU>()); break;
  }
}

// Two 16-bit roundings in one register.
template <typename T>
__device__ inline uint32_t pack2(float lo, float hi) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  const t2 v = {(T)lo, (T)hi};
  return __builtin_bit_cast(uint32_t, v);
}

// ---------------------------------------------------------------------------
// Products on 256 x 256 (kW 8) or 128 x 128 (kW 4) tiles
// ---------------------------------------------------------------------------

// C [M, N] = sum over the segments s of A_s [M, K] B_s [N, K]^T. Row strides are those of a
// K-major operand's rows, or between consecutive k of an MN-major one.
struct Product {
  const __bf16* A[2];  // 16-bit elements of the kernel's type
  const __bf16* B[2];
  int64_t lda, ldb[2];
  int64_t M, N, K;
  int32_t segs;
  int32_t splits;  // slots the segments' joint K (segs * K) is cut into, 1: whole
  int64_t kper;    // k per slot
  void* C;         // [M, N], contiguous
  float* part;     // [splits][M][N] where splits > 1
};

struct Gated {  // what the gated epilogues read and write, [N, F] contiguous each
  float* p;     // u act'(g), or NULL: not kept
  float* q;     // act(g)
  void* a;
  void* dg;
  void* du;
  int32_t act;
};

enum Epi : int {
  kEpiStore = 0,     // C, or a slot's fp32 partial
  kEpiGatedFwd = 1,  // the columns are pairs of g and u: writes a, and p and q where given
  kEpiGatedBwd = 2   // the product is da: reads p and q, writes dg and du
};

// The lanes' 16-byte pieces of rows of a [M, N] matrix in the accumulators' order.
template <int kW, typename F>
__device__ inline void epi_store(const AccOf<kW>& acc, int64_t M, int64_t N, int64_t gm0,
                                 int64_t nb, F&& store) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int i = 0; i < Cfg<kW>::kTI; ++i) {
    const int64_t gm = gm0 + 16 * i;
#pragma unroll
    for (int p = 0; p < Cfg<kW>::kTJ / 2; ++p) {
      const int64_t gc = nb + wide_col(p, g);
      store(acc.t[i][2 * p], acc.t[i][2 * p + 1], gm, gc, gm < M && gc < N);
    }
  }
}

template <typename T, int kEpi, int kMA, int kMB, int kW, int kSegs>
__device__ inline void product_tile(const Product& a, const Gated& e, int64_t bid, uint8_t* smem) {
  using C = Cfg<kW>;
  constexpr bool kPair = kEpi == kEpiGatedFwd;
  constexpr int kBN = kPair ? C::kBM / 2 : C::kBM;  // columns of C that the tile covers
  const int64_t MT = (a.M + C::kBM - 1) / C::kBM;
  const int64_t NT = (a.N + kBN - 1) / kBN;
  int64_t slot, mt, nt;
  ts_plan::gemm_piece_of(bid, MT, NT, a.splits, slot, mt, nt);
  const int64_t m0 = mt * C::kBM, n0 = nt * kBN;
  const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wm = wid >> 1, wn = wid & 1;
  AccOf<kW> acc;
  ts_gemm::clear<kW>(acc);
  if constexpr (kPair) {
    const ts_gemm::OpLoader<kKMajor, kW> la(a.A[0], a.lda, a.M, m0);
    const ts_gemm::PairLoader<kW> lb(a.B[0], a.ldb[0], a.B[1], a.ldb[1], a.N, n0);
    ts_gemm::mainloop_acc<kKMajor, kKMajor, kW, T>(la, lb, a.K, wn * (C::CW / 2),
                                                   C::kBM / 2 + wn * (C::CW / 2), smem, acc);
  } else {
    // dx has two segments (dg and du, each its own weight)
    const int64_t lo = slot * a.kper;  // of the joint K
    int64_t left = kSegs * a.K - lo < a.kper ? kSegs * a.K - lo : a.kper;
    int64_t k0 = lo;
#pragma unroll 1
    for (int s = 0; s < kSegs; ++s) {
      const int64_t n = kSegs == 1 || a.K - k0 > left ? left : a.K - k0;
      if (kSegs == 1 || n > 0) {     // uniform
        const __bf16* A = a.A[s] + (kMA == kKMajor ? k0 : k0 * a.lda);
        const __bf16* B = a.B[s] + (kMB == kKMajor ? k0 : k0 * a.ldb[s]);
        ts_gemm::mainloop_more<kMA, kMB, kW, T>(A, a.lda, a.M, B, a.ldb[s], a.N, n, m0, n0, smem,
                                                acc);
        left -= n;
        k0 += n;
        if (kSegs > 1) __syncthreads();  // the operands' tiles in LDS are free again
      }
      k0 -= a.K;
    }
  }
  const int64_t gm0 = m0 + wm * C::RW + (lane & 15);  // this lane's row of row block i: gm0 + 16 i
  const int g4 = lane >> 4;
  if constexpr (kEpi == kEpiStore) {
    const int64_t nb = n0 + wn * C::CW;
    if (a.splits > 1) {
      float* P = a.part + slot * a.M * a.N;
#pragma unroll
      for (int i = 0; i < C::kTI; ++i)
#pragma unroll
        for (int j = 0; j < C::kTJ; ++j) {
          const int64_t gm = gm0 + 16 * i, gc = nb + j * 16 + g4 * 4;
          if (gm < a.M && gc < a.N) *reinterpret_cast<f32x4*>(P + gm * a.N + gc) = acc.t[i][j];
        }
    } else {
      T* out = static_cast<T*>(a.C);
      epi_store<kW>(acc, a.M, a.N, gm0, nb,
                    [&](const f32x4& x, const f32x4& y, int64_t gm, int64_t gc, bool in) {
                      const u32x4 v = widen(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]),
                                            pack2<T>(y[0], y[1]), pack2<T>(y[2], y[3]));
                      if (in) st16(out + gm * a.N + gc, v);
                    });
    }
  } else if constexpr (kEpi == kEpiGatedFwd) {
    // column tiles 0 .. kHJ - 1 are g, the others u of the same columns
    const int64_t nb = n0 + wn * (C::CW / 2);
    T* O = static_cast<T*>(e.a);
    with_act(e.act, [&](auto act) {
#pragma unroll
      for (int i = 0; i < C::kTI; ++i) {
        const int64_t gm = gm0 + 16 * i;
#pragma unroll
        for (int j = 0; j < C::kHJ; ++j) {
          f32x4 p, q;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const float u = acc.t[i][C::kHJ + j][b];
            float d;
            q[b] = act_d<decltype(act)::value>(acc.t[i][j][b], d);
            p[b] = u * d;
            acc.t[i][j][b] = q[b] * u;
          }
          const int64_t gc = nb + 16 * j + 4 * g4;
          if (e.p != nullptr && gm < a.M && gc < a.N) {
            *reinterpret_cast<f32x4*>(e.p + gm * a.N + gc) = p;
            *reinterpret_cast<f32x4*>(e.q + gm * a.N + gc) = q;
          }
        }
      }
    });
#pragma unroll
    for (int i = 0; i < C::kTI; ++i)
#pragma unroll
      for (int p = 0; p < C::kHJ / 2; ++p) {
        const int64_t gm = gm0 + 16 * i, gc = nb + wide_col(p, g4);
        const f32x4 x = acc.t[i][2 * p], y = acc.t[i][2 * p + 1];
        const u32x4 v = widen(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(y[0], y[1]),
                              pack2<T>(y[2], y[3]));
        if (gm < a.M && gc < a.N) st16(O + gm * a.N + gc, v);
      }
  } else {
    const int64_t nb = n0 + wn * C::CW;
    T* DG = static_cast<T*>(e.dg);
    T* DU = static_cast<T*>(e.du);
    // Half a row block at a time, its factors loaded while the half before it is worked on.
    constexpr int kSteps = 2 * C::kTI;
    f32x4 p[2][C::kHJ], q[2][C::kHJ];
    auto load = [&](int s) {
      const int64_t gm = gm0 + 16 * (s / 2);
#pragma unroll
      for (int j = 0; j < C::kHJ; ++j) {
        const int64_t gc = nb + 16 * (s % 2 * C::kHJ + j) + 4 * g4;
        const bool in = gm < a.M && gc < a.N;
        p[s % 2][j] = in ? *reinterpret_cast<const f32x4*>(e.p + gm * a.N + gc) : f32x4{0, 0, 0, 0};
        q[s % 2][j] = in ? *reinterpret_cast<const f32x4*>(e.q + gm * a.N + gc) : f32x4{0, 0, 0, 0};
      }
    };
    load(0);
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (s + 1 < kSteps) load(s + 1);
      const int64_t gm = gm0 + 16 * (s / 2);
#pragma unroll
      for (int j = 0; j < C::kHJ; ++j) {
        const f32x4 da = acc.t[s / 2][s % 2 * C::kHJ + j];
        p[s % 2][j] *= da;
        q[s % 2][j] *= da;
      }
#pragma unroll
      for (int j = 0; j < C::kHJ; j += 2) {
        const int64_t gc = nb + wide_col((s % 2 * C::kHJ + j) / 2, g4);
        const f32x4 p0 = p[s % 2][j], p1 = p[s % 2][j + 1], q0 = q[s % 2][j], q1 = q[s % 2][j + 1];
        const u32x4 vg = widen(pack2<T>(p0[0], p0[1]), pack2<T>(p0[2], p0[3]),
                               pack2<T>(p1[0], p1[1]), pack2<T>(p1[2], p1[3]));
        const u32x4 vu = widen(pack2<T>(q0[0], q0[1]), pack2<T>(q0[2], q0[3]),
                               pack2<T>(q1[0], q1[1]), pack2<T>(q1[2], q1[3]));
        if (gm < a.M && gc < a.N) {
          st16(DG + gm * a.N + gc, vg);
          st16(DU + gm * a.N + gc, vu);
        }
      }
    }
  }
}

template <typename T, int kEpi, int kMA, int kMB, int kW>
__global__ __launch_bounds__(64 * kW) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mlp_product(const Product a, const Gated e) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[Cfg<kW>::kLdsBytes];
  product_tile<T, kEpi, kMA, kMB, kW, 1>(a, e, blockIdx.x, smem);
}

// dx and the weights' gradients in one grid: they are independent, and the tiles of one fill the
// CUs that another leaves.
struct Grads {
  Product dx;     // pieces 0 .. end[0]
  Product dw[3];  // dWg, dWu, dWd: up to end[1], end[2], end[3]
  int64_t end[4];
};

template <typename T, int kW>
__global__ __launch_bounds__(64 * kW) __attribute__((amdgpu_waves_per_eu(2, 2)))
void mlp_grads(const Grads a) {
  __shared__ __attribute__((aligned(16))) uint8_t smem[Cfg<kW>::kLdsBytes];
  const int64_t bid = blockIdx.x;
  const Gated none{};
  if (bid < a.end[0]) {
    product_tile<T, kEpiStore, kKMajor, kMNMajor, kW, 2>(a.dx, none, bid, smem);
  } else {
    const int w = bid < a.end[1] ? 0 : bid < a.end[2] ? 1 : 2;
    product_tile<T, kEpiStore, kMNMajor, kMNMajor, kW, 1>(a.dw[w], none, bid - a.end[w], smem);
  }
}

// ---------------------------------------------------------------------------
// Few rows (decoding): bound by reading the weights once. A workgroup owns 16 or 32 output features
// and every row; its waves take k-blocks of 64 in turn. Each wave streams the 128-byte runs of its 16
// weight rows (of both projections) and of x into a ring of its own in LDS, kDepth k-blocks ahead,
// and never waits for another wave until their sums are added in LDS, in wave order, at the end.
// The weights are the MFMAs' first operand, so a lane ends with four features of one row.
// The eight lanes of a load into LDS that share a row read its 128 bytes whole, where a load into
// MFMA operands takes 16 bytes of 16 rows at a time. Measured on MI355X, 16 rows, [14336, 4096] pair
// and [4096, 14336] (352 MB, three sets in turn): registers 85 us, LDS 72 us, the weights past the
// caches 66 us (5.3 TB/s; one row 62 us). 64 rows: registers 157 us, LDS 107 us, with two
// feature tiles a workgroup for the pair 96 us, products on 128 x 128 tiles with K in 12 slots 103 us (and
// 20 against 13 us at [2048, 768]).
// ---------------------------------------------------------------------------
struct Few {
  const __bf16* x;
  int64_t ldx;
  const __bf16* w[2];
  int64_t ldw[2];
  int64_t N, F, K;
  float* p;
  float* q;
  void* out;
  int32_t act;
};

// 16 rows from row r0 of a [rows, ld] matrix, for k-blocks in tiles of 16 x 128 bytes.
struct FewTile {
  ts_gemm::i32x4 rsrc;
  uint32_t off[2];
  uint32_t tail[2];  // off, or out of range where the last, short k-block has no such k
};
__device__ inline FewTile few_tile(const __bf16* p, int64_t ld, int64_t rows, int64_t r0,
                                   int64_t K) {
  FewTile t;
  const int lane = threadIdx.x & 63;
  int64_t valid = rows - r0;
  if (valid > 16) valid = 16;
  if (valid < 0) valid = 0;
  t.rsrc = ts_gemm::make_rsrc(p + r0 * ld, (uint64_t)valid * (uint64_t)ld * 2);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int row = u * 8 + (lane >> 3);
    const int chunk = ts_gemm::swz(row, lane & 7);
    t.off[u] = (uint32_t)(row * ld * 2 + chunk * 16);
    t.tail[u] = K / ts_gemm::BK * ts_gemm::BK + chunk * 8 < K ? t.off[u] : ts_gemm::kOob;
  }
  return t;
}
template <int kAux>
__device__ inline void few_issue(const FewTile& t, int64_t kb, bool last, uint8_t* lds) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
    ts_gemm::buffer_load_lds(t.rsrc, (ts_gemm::lds_ptr_t)(lds + u * 1024), 16,
                             (int)(last ? t.tail[u] : t.off[u]), (int)(kb * 128), 0, kAux);
}

// kNT 16-row tiles of x, kFT 16-feature tiles. kStream: the weights are read past the caches.
template <typename T, int kNT, int kFT, bool kPair, bool kStream>
__global__ __launch_bounds__(64 * ts_plan::kMlpFewWaves) void mlp_few(const Few a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  constexpr int kP = (kPair ? 2 : 1) * kFT;  // weight tiles: kFT of the first product, then the other's
  constexpr int kDepth = ts_plan::mlp_few_depth(kNT);
  constexpr int kTiles = kP + kNT;
  constexpr int kStage = kTiles * 2048;
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int waves = blockDim.x >> 6;
  const int64_t f0 = (int64_t)blockIdx.x * (16 * kFT);
  uint8_t* ring = smem + wid * (kDepth * kStage);
  FewTile tile[kTiles];
#pragma unroll
  for (int p = 0; p < kP; ++p)
    tile[p] = few_tile(a.w[p / kFT], a.ldw[p / kFT], a.F, f0 + p % kFT * 16, a.K);
#pragma unroll
  for (int t = 0; t < kNT; ++t) tile[kP + t] = few_tile(a.x, a.ldx, a.N, t * 16, a.K);
  f32x4 acc[kP][kNT];
#pragma unroll
  for (int p = 0; p < kP; ++p)
#pragma unroll
    for (int t = 0; t < kNT; ++t) acc[p][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t blocks = (a.K + ts_gemm::BK - 1) / ts_gemm::BK;
  const int64_t part = a.K % ts_gemm::BK != 0 ? blocks - 1 : blocks;  // the short block's index
  auto issue = [&](int64_t kb, int slot) {
#pragma unroll
    for (int q = 0; q < kTiles; ++q) {
      uint8_t* to = ring + slot * kStage + q * 2048;
      if (q < kP && kStream) few_issue<kBufNt>(tile[q], kb, kb == part, to);
      else few_issue<0>(tile[q], kb, kb == part, to);
    }
  };
  const int64_t mine = wid < blocks ? (blocks - wid + waves - 1) / waves : 0;  // this wave's blocks
#pragma unroll
  for (int d = 0; d < kDepth; ++d)
    if (d < mine) issue(wid + (int64_t)d * waves, d);
  int slot = 0;
  for (int64_t n = 0; n < mine; ++n) {
    // loads return in order: all but those of the blocks behind this one
    const int64_t behind = mine - 1 - n;
    static_assert(kDepth == 2 || kDepth == 3, "waits");
    if (kDepth == 3 && behind >= 2) ts_gemm::wait_vmcnt<2 * 2 * kTiles>();
    else if (behind >= 1) ts_gemm::wait_vmcnt<2 * kTiles>();
    else ts_gemm::wait_vmcnt<0>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* s = ring + slot * kStage;
    ts_gemm::bf16x8 w[kP][2], x[kNT][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int p = 0; p < kP; ++p) ts_gemm::read_op_k<1>(s + p * 2048, 0, lane, ks, &w[p][ks]);
#pragma unroll
      for (int t = 0; t < kNT; ++t)
        ts_gemm::read_op_k<1>(s + (kP + t) * 2048, 0, lane, ks, &x[t][ks]);
    }
    // read before the slot is filled again
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    if (n + kDepth < mine) issue(wid + (n + kDepth) * waves, slot);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int p = 0; p < kP; ++p)
#pragma unroll
        for (int t = 0; t < kNT; ++t)
          acc[p][t] = ts_gemm::mfma<T>(w[p][ks], x[t][ks], acc[p][t]);
    slot = slot + 1 == kDepth ? 0 : slot + 1;
  }
  __syncthreads();  // every wave is done with its ring
  f32x4* sums = reinterpret_cast<f32x4*>(smem);  // [waves][kP][kNT][64]
#pragma unroll
  for (int p = 0; p < kP; ++p)
#pragma unroll
    for (int t = 0; t < kNT; ++t) sums[((wid * kP + p) * kNT + t) * 64 + lane] = acc[p][t];
  __syncthreads();
  for (int i = threadIdx.x; i < kFT * kNT * 64; i += blockDim.x) {
    constexpr int kQ = kPair ? 2 : 1;
    f32x4 s[kQ];
#pragma unroll
    for (int q = 0; q < kQ; ++q) {
      const f32x4* at = sums + q * kFT * kNT * 64 + i;
      s[q] = at[0];
      for (int v = 1; v < waves; ++v) s[q] += at[v * kP * kNT * 64];
    }
    const int t = i >> 6;
    const int64_t r = t % kNT * 16 + (i & 15), fo = f0 + t / kNT * 16 + ((i & 63) >> 4) * 4;
    if (r >= a.N || fo >= a.F) continue;
    const int64_t at = r * a.F + fo;
    if constexpr (kPair) {
      f32x4 p, q;
      with_act(a.act, [&](auto act) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float d;
          q[b] = act_d<decltype(act)::value>(s[0][b], d);
          p[b] = s[1][b] * d;
          s[0][b] = q[b] * s[1][b];
        }
      });
      if (a.p != nullptr) {
        *reinterpret_cast<f32x4*>(a.p + at) = p;
        *reinterpret_cast<f32x4*>(a.q + at) = q;
      }
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at) =
        make_uint2(pack2<T>(s[0][0], s[0][1]), pack2<T>(s[0][2], s[0][3]));
  }
}

// ---------------------------------------------------------------------------
// Partials of a split K, added in slot order and rounded once
// ---------------------------------------------------------------------------
struct SumJobs {
  const float* part[4];
  void* out[4];
  int64_t quads[4];  // elements / 4
  int32_t splits[4];
  int64_t end[4];    // workgroups up to and with this job
};
constexpr int kSumUnroll = 8;

template <typename T>
__global__ __launch_bounds__(256) void mlp_sum_slots(const SumJobs s) {
  const int64_t bid = blockIdx.x;
  int j = 0;
  while (j < 3 && bid >= s.end[j]) ++j;
  const int64_t i = (bid - (j ? s.end[j - 1] : 0)) * 256 + threadIdx.x;
  const int64_t n = s.quads[j];
  if (i >= n) return;
  const f32x4* p = reinterpret_cast<const f32x4*>(s.part[j]);
  f32x4 sum{0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < s.splits[j]; p0 += kSumUnroll) {
    f32x4 v[kSumUnroll];
#pragma unroll
    for (int q = 0; q < kSumUnroll; ++q)
      v[q] = p0 + q < s.splits[j] ? p[(p0 + q) * n + i] : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < kSumUnroll; ++q) sum += v[q];
  }
  static_cast<uint2*>(s.out[j])[i] = make_uint2(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]));
}

// ---------------------------------------------------------------------------
// Without the down projection: dg and du of da = dy, element by element
// ---------------------------------------------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void mlp_gate_bwd(const T* __restrict__ da, int64_t ldd,
                                                    const float* __restrict__ p,
                                                    const float* __restrict__ q,
                                                    T* __restrict__ dg, T* __restrict__ du,
                                                    int64_t nvec, int64_t F8) {
  const int64_t v = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (v >= nvec) return;
  const int64_t r = v / F8;
  const u32x4 qd = ld16_stream(da + r * ldd + (v - r * F8) * 8);
  const u32x4 p0 = ld16_stream(p + v * 8), p1 = ld16_stream(p + v * 8 + 4);
  const u32x4 q0 = ld16_stream(q + v * 8), q1 = ld16_stream(q + v * 8 + 4);
  float d[8], P[8], Q[8];
  Elt<T>::unpack(qd, d);
  Elt<float>::unpack(p0, P);
  Elt<float>::unpack(p1, P + 4);
  Elt<float>::unpack(q0, Q);
  Elt<float>::unpack(q1, Q + 4);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    P[i] *= d[i];
    Q[i] *= d[i];
  }
  st16(dg + v * 8, Elt<T>::pack(P));
  st16(du + v * 8, Elt<T>::pack(Q));
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
ts_plan::MlpShape shape_of(const ts_gated_mlp_args& a) {
  return ts_plan::MlpShape{a.N, a.H, a.F, a.w_down != nullptr ? a.O : 0};
}

static_assert(TS_MLP_DX == ts_plan::kMlpDx && TS_MLP_DW_GATE == ts_plan::kMlpDwGate &&
              TS_MLP_DW_UP == ts_plan::kMlpDwUp && TS_MLP_DW_DOWN == ts_plan::kMlpDwDown,
              "the plan's gradients");

constexpr int64_t kMaxDim = (int64_t)1 << 21;  // 32-bit offsets inside a tile

ts_status check_args(const char* who, const ts_gated_mlp_args* a) {
  using ts_host::fail;
  if (a == nullptr) return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL arguments", who);
  if (a->dtype != TS_BF16 && a->dtype != TS_F16)
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: dtype must be bf16 or fp16", who);
  if (a->activation < TS_ACT_SILU || a->activation > TS_ACT_RELU)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: unknown activation %d", who, (int)a->activation);
  const bool down = a->w_down != nullptr;
  if (a->N < 0 || a->H <= 0 || a->F <= 0 || (down && a->O <= 0))
    return fail(TS_ERR_SHAPE, "%s: bad shape N=%lld H=%lld F=%lld O=%lld", who, (long long)a->N,
                (long long)a->H, (long long)a->F, (long long)a->O);
  if (a->H % 8 || a->F % 8 || (down && a->O % 8))
    return fail(TS_ERR_SHAPE, "%s: H, F and O must be multiples of 8", who);
  if (a->H > kMaxDim || a->F > kMaxDim || (down && a->O > kMaxDim) ||
      a->N > ((int64_t)1 << 31))
    return fail(TS_ERR_SHAPE, "%s: more than 2^21 features or 2^31 rows", who);
  if (a->ldx < a->H || a->ld_gate < a->H || a->ld_up < a->H || (down && a->ld_down < a->F))
    return fail(TS_ERR_SHAPE, "%s: row stride shorter than a row", who);
  if (a->ldx % 8 || a->ld_gate % 8 || a->ld_up % 8 || (down && a->ld_down % 8))
    return fail(TS_ERR_SHAPE, "%s: row strides must be multiples of 8", who);
  if (a->ldx > kMaxDim || a->ld_gate > kMaxDim || a->ld_up > kMaxDim ||
      (down && a->ld_down > kMaxDim))
    return fail(TS_ERR_SHAPE, "%s: row strides above 2^21", who);
  if (a->N > 0 && (a->x == nullptr || a->w_gate == nullptr || a->w_up == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL operand", who);
  if (!ts_host::aligned16(a->x) || !ts_host::aligned16(a->w_gate) ||
      !ts_host::aligned16(a->w_up) || !ts_host::aligned16(a->w_down))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: operands must be 16-byte aligned", who);
  return TS_OK;
}

const __bf16* raw(const void* p) { return static_cast<const __bf16*>(p); }

Product product(const void* A, int64_t lda, const void* B, int64_t ldb, int64_t M, int64_t N,
                int64_t K, void* C) {
  Product p{};
  p.A[0] = p.A[1] = raw(A);
  p.B[0] = p.B[1] = raw(B);
  p.lda = lda;
  p.ldb[0] = p.ldb[1] = ldb;
  p.M = M;
  p.N = N;
  p.K = K;
  p.segs = 1;
  p.splits = 1;
  p.kper = K;
  p.C = C;
  return p;
}

void set_split(Product& p, const ts_plan::KSplit& k, float* part) {
  p.splits = (int32_t)k.splits;
  p.kper = k.splits > 1 ? k.kper : p.segs * p.K;
  p.part = part;
}

template <typename T, int kEpi, int kMA, int kMB>
ts_status launch_product(const Product& p, const Gated& e, int waves, hipStream_t st,
                         const char* name) {
  const int64_t tiles = ts_plan::mlp_tiles(p.M, p.N, waves, kEpi == kEpiGatedFwd) * p.splits;
  if (tiles <= 0) return TS_OK;
  if (tiles > ts_plan::max_blocks(64 * waves))
    return ts_host::fail(TS_ERR_SHAPE, "%s: too many tiles", name);
  if (waves == 8)
    hipLaunchKernelGGL((mlp_product<T, kEpi, kMA, kMB, 8>), dim3((unsigned)tiles), dim3(512), 0,
                       st, p, e);
  else
    hipLaunchKernelGGL((mlp_product<T, kEpi, kMA, kMB, 4>), dim3((unsigned)tiles), dim3(256), 0,
                       st, p, e);
  return ts_host::check_launch(name);
}

void add_job(SumJobs& s, int& n, const Product& p) {
  if (p.C == nullptr || p.splits <= 1) return;
  s.part[n] = p.part;
  s.out[n] = p.C;
  s.quads[n] = p.M * p.N / 4;
  s.splits[n] = p.splits;
  s.end[n] = (n ? s.end[n - 1] : 0) + (s.quads[n] + 255) / 256;
  ++n;
}

template <typename T>
ts_status launch_sums(SumJobs& s, int n, hipStream_t st) {
  if (n == 0) return TS_OK;
  const int64_t blocks = s.end[n - 1];
  for (int j = n; j < 4; ++j) s.end[j] = blocks;
  if (blocks > ts_plan::max_blocks(256)) return ts_host::fail(TS_ERR_SHAPE, "mlp_sum_slots: too large");
  hipLaunchKernelGGL(mlp_sum_slots<T>, dim3((unsigned)blocks), dim3(256), 0, st, s);
  return ts_host::check_launch("mlp_sum_slots");
}

#define TS_TRY(x)                  \
  do {                             \
    const ts_status s_ = (x);      \
    if (s_ != TS_OK) return s_;    \
  } while (0)

template <typename T, int kNT, int kFT, bool kPair>
ts_status launch_few_rows(const Few& f, hipStream_t st) {
  const int64_t blocks = (f.F + 16 * kFT - 1) / (16 * kFT);
  const int waves = ts_plan::mlp_few_waves(f.K);
  const size_t lds =
      (size_t)waves * ((kPair ? 2 : 1) * kFT + kNT) * ts_plan::mlp_few_depth(kNT) * 2048;
  if (ts_plan::mlp_few_stream(f.F, f.K, kPair))
    hipLaunchKernelGGL((mlp_few<T, kNT, kFT, kPair, true>), dim3((unsigned)blocks),
                       dim3(64 * waves), lds, st, f);
  else
    hipLaunchKernelGGL((mlp_few<T, kNT, kFT, kPair, false>), dim3((unsigned)blocks),
                       dim3(64 * waves), lds, st, f);
  return ts_host::check_launch("mlp_few");
}

template <typename T, bool kPair>
ts_status launch_few(const Few& f, hipStream_t st) {
  const bool two = ts_plan::mlp_few_two(f.N, f.F, kPair);
  if (f.N <= 16) return launch_few_rows<T, 1, 1, kPair>(f, st);
  if (f.N <= 32) {
    if constexpr (!kPair)
      if (two) return launch_few_rows<T, 2, 2, kPair>(f, st);
    return launch_few_rows<T, 2, 1, kPair>(f, st);
  }
  if (f.N <= 48)
    return two ? launch_few_rows<T, 3, 2, kPair>(f, st) : launch_few_rows<T, 3, 1, kPair>(f, st);
  return two ? launch_few_rows<T, 4, 2, kPair>(f, st) : launch_few_rows<T, 4, 1, kPair>(f, st);
}

template <typename T>
ts_status fwd_few(const ts_gated_mlp_args& a, float* p, float* q, void* act, void* out,
                  hipStream_t st) {
  TS_TRY((launch_few<T, true>(Few{raw(a.x), a.ldx, {raw(a.w_gate), raw(a.w_up)},
                                  {a.ld_gate, a.ld_up}, a.N, a.F, a.H, p, q, act,
                                  a.activation}, st)));
  if (out == nullptr) return TS_OK;
  return launch_few<T, false>(Few{raw(act), a.F, {raw(a.w_down), nullptr}, {a.ld_down, 0}, a.N,
                                  a.O, a.F, nullptr, nullptr, out, 0}, st);
}

template <typename T>
ts_status fwd_typed(const ts_gated_mlp_args& a, const ts_plan::MlpFwdPlan& pl, float* keep_p,
                    float* keep_q, void* act, void* out, void* ws, hipStream_t st) {
  if (a.N <= ts_plan::kMlpFewRows) return fwd_few<T>(a, keep_p, keep_q, act, out, st);
  Product p = product(a.x, a.ldx, a.w_gate, a.ld_gate, a.N, a.F, a.H, nullptr);
  p.B[1] = raw(a.w_up);
  p.ldb[1] = a.ld_up;
  const Gated e{keep_p, keep_q, act, nullptr, nullptr, a.activation};
  TS_TRY((launch_product<T, kEpiGatedFwd, kKMajor, kKMajor>(p, e, pl.up_waves, st, "mlp_gated")));
  if (out == nullptr) return TS_OK;
  Product d = product(act, a.F, a.w_down, a.ld_down, a.N, a.O, a.F, out);
  set_split(d, pl.down, static_cast<float*>(ws));
  TS_TRY((launch_product<T, kEpiStore, kKMajor, kKMajor>(d, e, pl.down_waves, st, "mlp_down")));
  SumJobs s{};
  int n = 0;
  add_job(s, n, d);
  return launch_sums<T>(s, n, st);
}

template <typename T, int kW>
ts_status launch_grads(const Grads& g, hipStream_t st) {
  if (g.end[3] <= 0) return TS_OK;
  if (g.end[3] > ts_plan::max_blocks(Cfg<kW>::kThreads))
    return ts_host::fail(TS_ERR_SHAPE, "mlp_grads: too many tiles");
  hipLaunchKernelGGL((mlp_grads<T, kW>), dim3((unsigned)g.end[3]),
                     dim3(Cfg<kW>::kThreads), 0, st, g);
  return ts_host::check_launch("mlp_grads");
}

template <typename T>
ts_status bwd_typed(const ts_gated_mlp_args& a, const ts_plan::MlpBwdPlan& pl,
                    const ts_plan::MlpBwdWorkspace& w, const float* keep_p, const float* keep_q,
                    const void* act, const void* dout, int64_t ldd, void* dx, void* dwg, void* dwu,
                    void* dwd, uint8_t* ws, hipStream_t st) {
  void* dg = ws + w.dg;
  void* du = ws + w.du;
  const bool inner = dx != nullptr || dwg != nullptr || dwu != nullptr;
  const bool down = a.w_down != nullptr;
  if (inner && down) {
    const Gated e{const_cast<float*>(keep_p), const_cast<float*>(keep_q), nullptr, dg, du,
                  a.activation};
    const Product p = product(dout, ldd, a.w_down, a.ld_down, a.N, a.F, a.O, nullptr);
    TS_TRY((launch_product<T, kEpiGatedBwd, kKMajor, kMNMajor>(p, e, pl.da_waves, st,
                                                               "mlp_gated_bwd")));
  } else if (inner) {
    const int64_t nvec = a.N * a.F / 8, blocks = (nvec + 255) / 256;
    if (blocks > ts_plan::max_blocks(256))
      return ts_host::fail(TS_ERR_SHAPE, "mlp_gate_bwd: too large");
    hipLaunchKernelGGL(mlp_gate_bwd<T>, dim3((unsigned)blocks), dim3(256), 0, st,
                       static_cast<const T*>(dout), ldd, keep_p, keep_q, static_cast<T*>(dg),
                       static_cast<T*>(du), nvec, a.F / 8);
    TS_TRY(ts_host::check_launch("mlp_gate_bwd"));
  }
  Grads g{};
  g.dx = product(dg, a.F, a.w_gate, a.ld_gate, a.N, a.H, a.F, dx);
  g.dx.A[1] = raw(du);
  g.dx.B[1] = raw(a.w_up);
  g.dx.ldb[1] = a.ld_up;
  g.dx.segs = 2;
  g.dw[0] = product(dg, a.F, a.x, a.ldx, a.F, a.H, a.N, dwg);
  g.dw[1] = product(du, a.F, a.x, a.ldx, a.F, a.H, a.N, dwu);
  g.dw[2] = product(dout, ldd, act, a.F, a.O, a.F, a.N, dwd);
  set_split(g.dx, pl.dx, reinterpret_cast<float*>(ws + w.dx));
  for (int i = 0; i < 3; ++i) set_split(g.dw[i], pl.dw, reinterpret_cast<float*>(ws + w.dw[i]));
  SumJobs s{};
  int n = 0;
  int64_t end = 0;
  for (int i = 0; i < 4; ++i) {
    const Product& p = i == 0 ? g.dx : g.dw[i - 1];
    if (p.C != nullptr) end += ts_plan::mlp_tiles(p.M, p.N, pl.grad_waves, false) * p.splits;
    g.end[i] = end;
    add_job(s, n, p);
  }
  TS_TRY((pl.grad_waves == 8 ? launch_grads<T, 8>(g, st) : launch_grads<T, 4>(g, st)));
  return launch_sums<T>(s, n, st);
}

}  // namespace

extern "C" size_t ts_gated_mlp_fwd_workspace_size(int64_t N, int64_t H, int64_t F, int64_t O) {
  if (N <= 0 || H <= 0 || F <= 0 || O < 0) return 0;
  const ts_plan::MlpShape s{N, H, F, O};
  return (size_t)ts_plan::mlp_fwd_workspace(s, ts_plan::mlp_fwd_plan(s));
}

extern "C" size_t ts_gated_mlp_bwd_grads_workspace_size(int64_t N, int64_t H, int64_t F, int64_t O,
                                                        int32_t grads) {
  grads &= ts_plan::kMlpGrads;
  if (N <= 0 || H <= 0 || F <= 0 || O < 0 || grads == 0) return 0;
  const ts_plan::MlpShape s{N, H, F, O};
  return (size_t)ts_plan::mlp_bwd_workspace(s, ts_plan::mlp_bwd_plan(s, grads), grads).total;
}

extern "C" size_t ts_gated_mlp_bwd_workspace_size(int64_t N, int64_t H, int64_t F, int64_t O) {
  size_t most = 0;
  for (int32_t grads = 1; grads <= ts_plan::kMlpGrads; ++grads) {
    const size_t n = ts_gated_mlp_bwd_grads_workspace_size(N, H, F, O, grads);
    if (n > most) most = n;
  }
  return most;
}

extern "C" ts_status ts_gated_mlp_fwd(const ts_gated_mlp_args* args, float* keep_p,
                                      float* keep_q, void* act, void* out, void* workspace,
                                      size_t workspace_bytes, ts_stream_t stream) {
  using ts_host::fail;
  TS_TRY(check_args("gated_mlp_fwd", args));
  if (args->N == 0) return TS_OK;
  if (act == nullptr || (out == nullptr) != (args->w_down == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_fwd: out goes with w_down, act is needed");
  if ((keep_p == nullptr) != (keep_q == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_fwd: keep_p and keep_q go together");
  if (!ts_host::aligned16(keep_p) || !ts_host::aligned16(keep_q) || !ts_host::aligned16(act) ||
      !ts_host::aligned16(out) || !ts_host::aligned16(workspace))
    return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_fwd: outputs must be 16-byte aligned");
  const ts_plan::MlpShape s = shape_of(*args);
  const ts_plan::MlpFwdPlan pl = ts_plan::mlp_fwd_plan(s);
  const size_t need = (size_t)ts_plan::mlp_fwd_workspace(s, pl);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TS_ERR_WORKSPACE, "gated_mlp_fwd: workspace of %zu bytes, need %zu",
                workspace_bytes, need);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return args->dtype == TS_BF16
             ? fwd_typed<__bf16>(*args, pl, keep_p, keep_q, act, out, workspace, st)
             : fwd_typed<_Float16>(*args, pl, keep_p, keep_q, act, out, workspace, st);
}

extern "C" ts_status ts_gated_mlp_bwd(const ts_gated_mlp_args* args, const float* keep_p,
                                      const float* keep_q, const void* act, const void* dout,
                                      int64_t ld_dout, void* dx, void* dw_gate, void* dw_up,
                                      void* dw_down, void* workspace, size_t workspace_bytes,
                                      ts_stream_t stream) {
  using ts_host::fail;
  TS_TRY(check_args("gated_mlp_bwd", args));
  if (args->N == 0) return fail(TS_ERR_SHAPE, "gated_mlp_bwd: no rows (the gradients are zeros)");
  const bool down = args->w_down != nullptr;
  const bool inner = dx != nullptr || dw_gate != nullptr || dw_up != nullptr;
  if ((inner && (keep_p == nullptr || keep_q == nullptr)) || dout == nullptr ||
      (dw_down != nullptr && act == nullptr))
    return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_bwd: NULL operand");
  if (!down && dw_down != nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_bwd: dw_down without w_down");
  const int64_t cols = down ? args->O : args->F;
  if (ld_dout < cols || ld_dout % 8 || ld_dout > kMaxDim)
    return fail(TS_ERR_SHAPE, "gated_mlp_bwd: bad row stride of dout");
  for (const void* p : {(const void*)keep_p, (const void*)keep_q, act, dout, (const void*)dx, (const void*)dw_gate,
                        (const void*)dw_up, (const void*)dw_down, (const void*)workspace})
    if (!ts_host::aligned16(p))
      return fail(TS_ERR_INVALID_ARGUMENT, "gated_mlp_bwd: buffers must be 16-byte aligned");
  const int grads = (dx != nullptr ? TS_MLP_DX : 0) | (dw_gate != nullptr ? TS_MLP_DW_GATE : 0) |
                    (dw_up != nullptr ? TS_MLP_DW_UP : 0) |
                    (dw_down != nullptr ? TS_MLP_DW_DOWN : 0);
  if (grads == 0) return TS_OK;
  const ts_plan::MlpShape s = shape_of(*args);
  const ts_plan::MlpBwdPlan pl = ts_plan::mlp_bwd_plan(s, grads);
  const ts_plan::MlpBwdWorkspace w = ts_plan::mlp_bwd_workspace(s, pl, grads);
  const size_t need = (size_t)w.total;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TS_ERR_WORKSPACE, "gated_mlp_bwd: workspace of %zu bytes, need %zu",
                workspace_bytes, need);
  hipStream_t st = static_cast<hipStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  return args->dtype == TS_BF16
             ? bwd_typed<__bf16>(*args, pl, w, keep_p, keep_q, act, dout, ld_dout, dx, dw_gate, dw_up,
                                 dw_down, ws, st)
             : bwd_typed<_Float16>(*args, pl, w, keep_p, keep_q, act, dout, ld_dout, dx, dw_gate, dw_up,
                                   dw_down, ws, st);
}
