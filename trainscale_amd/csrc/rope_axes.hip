// Rotary positions with several axes (time, height and width of images and video) for gfx950:
// pair i of a head's first R elements is turned by the angle pos[axis(i)] f(i); the elements behind
// them stay as they are. Backward is the transpose: sin negated.
//
// Angles. Positions are integers, so only the fraction of a turn that a frequency makes per
// position matters: f(i) / (2 pi) modulo 1 as a fixed-point fraction of 96 bits, turns[i] and 32
// signed bits in rest[i], formed on the host. Its product with the position modulo a turn, to 64 bits,
// is the angle's fraction of a turn, exact for every 64-bit position of either sign but for 2^-64 of
// a turn and the fraction's own rounding (2^-97 of a turn per position, 4e-10 rad at 2^63; without
// the rest 2^-65, more than fp32's rounding from 2^38 on), with no range reduction. Its nearest
// quarter turn comes off as integers; the rest, within an eighth of a turn, is rounded to fp32
// once, and sin and cos are Taylor polynomials there (terms past 2e-9 left out). An fp32 product of
// position and frequency would be off by up to 2^-24 of the angle, 0.06 rad at position 1 million.
//
// A workgroup handles tpb consecutive tokens and every head of both tensors at those tokens. Its
// threads issue their first task's loads, fill LDS with the tokens' cos and sin (once per token and
// frequency, shared by all heads), meet one barrier, rotate and store. A task is a vector from each
// half of a head's rotated part (or one of adjacent pairs), or a vector of what stays. Vectors are
// 16 bytes, 8 where the halves are not whole 16-byte vectors, single elements otherwise; any
// element address will do.
//
// Bound by HBM. Measured on MI355X, a direction: [1, 32768, 64 + 8, 128] bf16 196 us (6.2 TB/s),
// [8, 1369, 16 + 16, 80] fp16 28 us (4.4 TB/s; 2 tokens a workgroup 27, 8 of them 36), 16 tokens of 32 + 8
// heads 4 us; adjacent pairs of the first 272 us (4.5 TB/s).
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

constexpr int kMaxHalf = 256;
constexpr int kMaxThreads = 1024;
constexpr int kLdsAngles = 4096;  // tpb * half at most

struct AxesArgs {
  const void* q_in;
  void* q_out;
  int64_t q_in_sb, q_in_ss, q_in_sh, q_out_sb, q_out_ss, q_out_sh;
  const void* k_in;
  void* k_out;
  int64_t k_in_sb, k_in_ss, k_in_sh, k_out_sb, k_out_ss, k_out_sh;
  const int64_t* pos;
  int64_t pos_sa, pos_sb, pos_ss;
  int64_t S, ntok;
  uint64_t s_magic;                   // ts_plan::magic64_for(S)
  uint32_t tpt_magic, tph_magic;      // ts_plan::magic_for of the two below
  int32_t tasks_per_token, tasks_per_head;
  int32_t Hq, Hk, half, pairs, tpb;   // pairs: rotating tasks of a head
  int32_t backward;
  uint64_t turns[kMaxHalf];
  int32_t rest[kMaxHalf];
  uint8_t axis[kMaxHalf];
};

// cos and sin of the angle whose fraction of a turn is t / 2^64.
__device__ inline void turn_cos_sin(uint64_t t, float& c, float& s) {
  const uint64_t up = t + ((uint64_t)1 << 61);
  const int quarter = (int)(up >> 62);
  const int64_t rest = (int64_t)(t - ((uint64_t)quarter << 62));  // within an eighth of a turn
  constexpr float kHi = 6.2831855f * 0x1p-64f, kLo = -1.7484555e-7f * 0x1p-64f;  // 2 pi / 2^64
  const float r = (float)rest;
  const float x = __builtin_fmaf(r, kHi, r * kLo);  // rad
  const float z = x * x;
  const float sn = x + x * z * (-1.6666666667e-1f + z * (8.3333333333e-3f +
                   z * (-1.9841269841e-4f + z * 2.7557319224e-6f)));
  const float cs = 1.f + z * (-0.5f + z * (4.1666666667e-2f + z * (-1.3888888889e-3f +
                   z * (2.4801587302e-5f - z * 2.7557319224e-7f))));
  const float a = quarter & 1 ? sn : cs, b = quarter & 1 ? cs : sn;
  c = quarter == 1 || quarter == 2 ? -a : a;
  s = quarter & 2 ? -b : b;
}

// A vector of kBytes (16, 8, or one element) and its values in fp32.
template <typename T, int kBytes>
struct Vec;
template <typename T>
struct Vec<T, 16> {
  static constexpr int n = Elt<T>::kVec;
  u32x4 q;
  __device__ inline void load(const T* p) { q = ld16_any_stream(p); }
  __device__ inline void get(float* f) const { Elt<T>::unpack(q, f); }
  __device__ static inline void put(T* p, const float* f) { st16_any_stream(p, Elt<T>::pack(f)); }
};
template <typename T>
struct Vec<T, 8> {
  static constexpr int n = Elt<T>::kVec / 2;
  typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
  typedef u32x2_t any_t __attribute__((aligned(2)));
  u32x2_t q;
  __device__ inline void load(const T* p) {
    q = __builtin_nontemporal_load(reinterpret_cast<const any_t*>(p));
  }
  __device__ inline void get(float* f) const {
    float w[Elt<T>::kVec];
    Elt<T>::unpack(u32x4{q[0], q[1], 0u, 0u}, w);
#pragma unroll
    for (int i = 0; i < n; ++i) f[i] = w[i];
  }
  __device__ static inline void put(T* p, const float* f) {
    float w[Elt<T>::kVec] = {};
#pragma unroll
    for (int i = 0; i < n; ++i) w[i] = f[i];
    const u32x4 v = Elt<T>::pack(w);
    __builtin_nontemporal_store(u32x2_t{v[0], v[1]}, reinterpret_cast<any_t*>(p));
  }
};
template <typename T>
struct Vec<T, 0> {
  static constexpr int n = 1;
  float q;
  __device__ inline void load(const T* p) { q = Elt<T>::load1(p); }
  __device__ inline void get(float* f) const { f[0] = q; }
  __device__ static inline void put(T* p, const float* f) { Elt<T>::store1(p, f[0]); }
};

template <typename T>
struct Head {
  const T* src;
  T* dst;
  int i, j;  // token slot, task of the head
};

template <typename T, int kBytes, bool kInterleaved>
struct AxesTask {
  using V = Vec<T, kBytes>;
  V a, b;
  // First elements of the task's vectors; a task past the pairs copies one vector.
  __device__ static inline void where(const AxesArgs& p, int j, int& e1, int& e2) {
    if (j >= p.pairs) {
      e1 = 2 * p.half + (j - p.pairs) * V::n;
      e2 = -1;
    } else if constexpr (kInterleaved) {
      e1 = kBytes == 0 ? 2 * j : j * V::n;
      e2 = kBytes == 0 ? e1 + 1 : -1;
    } else {
      e1 = j * V::n;
      e2 = p.half + e1;
    }
  }
  __device__ inline void load(const AxesArgs& p, const Head<T>& h) {
    int e1, e2;
    where(p, h.j, e1, e2);
    a.load(h.src + e1);
    if (e2 >= 0) b.load(h.src + e2);
  }
  __device__ inline void finish(const AxesArgs& p, const Head<T>& h, const float* cs,
                                const float* sn) const {
    int e1, e2;
    where(p, h.j, e1, e2);
    float x[V::n], y[V::n];
    a.get(x);
    if (h.j < p.pairs) {
      const float* c = cs + h.i * p.half;
      const float* s = sn + h.i * p.half;
      if constexpr (kInterleaved && kBytes != 0) {
#pragma unroll
        for (int k = 0; k < V::n / 2; ++k) {
          const float cc = c[e1 / 2 + k], ss = s[e1 / 2 + k], u = x[2 * k], v = x[2 * k + 1];
          x[2 * k] = u * cc - v * ss;
          x[2 * k + 1] = v * cc + u * ss;
        }
      } else {
        b.get(y);
        const int f = kInterleaved ? e1 / 2 : e1;
#pragma unroll
        for (int k = 0; k < V::n; ++k) {
          const float cc = c[f + k], ss = s[f + k], u = x[k], v = y[k];
          x[k] = u * cc - v * ss;
          y[k] = v * cc + u * ss;
        }
        V::put(h.dst + e2, y);
      }
    }
    V::put(h.dst + e1, x);
  }
};

// kOne: one token a workgroup, whose addresses and positions are uniform.
template <typename T, int kBytes, bool kInterleaved, bool kOne>
__global__ __launch_bounds__(kMaxThreads) void rope_axes_kernel(const AxesArgs a) {
  extern __shared__ float lds[];
  const int tpb = kOne ? 1 : a.tpb;
  float* cs = lds;
  float* sn = lds + tpb * a.half;
  const int64_t tok0 = (int64_t)blockIdx.x * tpb;
  const int64_t left = a.ntok - tok0;
  const int here = left < tpb ? (int)left : tpb;
  const int total = here * a.tasks_per_token;
  auto batch_of = [&](int64_t t) {
    return a.s_magic == 0 ? t : (int64_t)__umul64hi((uint64_t)t, a.s_magic);
  };
  auto head = [&](int f) {
    Head<T> h;
    const ts_plan::RopeTask rt =
        kOne ? ts_plan::rope_head_task(f, a.tasks_per_head, a.tph_magic)
             : ts_plan::rope_task(f, a.tasks_per_token, a.tpt_magic, a.tasks_per_head,
                                  a.tph_magic);
    h.i = kOne ? 0 : rt.i;
    h.j = rt.j;
    const int64_t t = tok0 + h.i, b = batch_of(t), s = t - b * a.S;
    // both candidates, then a select: a branch would fetch the chosen strides per lane
    const bool is_q = rt.hh < a.Hq;
    const int kh = rt.hh - a.Hq;
    const T* qs = static_cast<const T*>(a.q_in) + b * a.q_in_sb + s * a.q_in_ss;
    T* qd = static_cast<T*>(a.q_out) + b * a.q_out_sb + s * a.q_out_ss;
    const T* ks = static_cast<const T*>(a.k_in) + b * a.k_in_sb + s * a.k_in_ss;
    T* kd = static_cast<T*>(a.k_out) + b * a.k_out_sb + s * a.k_out_ss;
    qs += rt.hh * a.q_in_sh;
    qd += rt.hh * a.q_out_sh;
    ks += kh * a.k_in_sh;
    kd += kh * a.k_out_sh;
    h.src = is_q ? qs : ks;
    h.dst = is_q ? qd : kd;
    return h;
  };
  int f = threadIdx.x;
  Head<T> h{};
  AxesTask<T, kBytes, kInterleaved> task;
  if (f < total) {
    h = head(f);
    task.load(a, h);
  }
  const int n = here * a.half;
  for (int idx = threadIdx.x; idx < n; idx += blockDim.x) {
    const int i = kOne ? 0 : idx / a.half;
    const int p = idx - i * a.half;
    const int64_t t = tok0 + i, b = batch_of(t), s = t - b * a.S;
    const int64_t pos = a.pos[a.axis[p] * a.pos_sa + b * a.pos_sb + s * a.pos_ss];
    const int64_t rest = __mul64hi(pos, (int64_t)a.rest[p] * ((int64_t)1 << 32));
    float c, w;
    turn_cos_sin((uint64_t)pos * a.turns[p] + (uint64_t)rest, c, w);
    cs[idx] = c;
    sn[idx] = a.backward ? -w : w;
  }
  __syncthreads();
  if (f < total) task.finish(a, h, cs, sn);
  for (f += blockDim.x; f < total; f += blockDim.x) {
    h = head(f);
    task.load(a, h);
    task.finish(a, h, cs, sn);
  }
}

template <typename T, int kBytes, bool kInterleaved>
ts_status launch_typed(AxesArgs& a, int D, bool in_place, hipStream_t st) {
  constexpr int n = Vec<T, kBytes>::n;
  a.pairs = kInterleaved && kBytes != 0 ? 2 * a.half / n : a.half / n;
  const int stay = in_place ? 0 : (D - 2 * a.half) / n;
  a.tasks_per_head = a.pairs + stay;
  a.tasks_per_token = a.tasks_per_head * (a.Hq + a.Hk);
  const ts_plan::RopeBlock blk =
      ts_plan::rope_block(a.tasks_per_token, a.half, kMaxThreads, kLdsAngles);
  a.tpb = blk.tpb;
  if ((a.tpb > 1 && !ts_plan::magic_exact((uint64_t)a.tpb * a.tasks_per_token,
                                          (uint64_t)a.tasks_per_token)) ||
      !ts_plan::magic_exact((uint64_t)a.tasks_per_token, (uint64_t)a.tasks_per_head) ||
      !ts_plan::magic64_exact((uint64_t)a.ntok, (uint64_t)a.S))
    return ts_host::fail(TS_ERR_SHAPE, "rope_axes: too many heads or tokens");
  a.tpt_magic = ts_plan::magic_for((uint32_t)a.tasks_per_token);
  a.tph_magic = ts_plan::magic_for((uint32_t)a.tasks_per_head);
  a.s_magic = ts_plan::magic64_for((uint64_t)a.S);
  const int64_t blocks = (a.ntok + a.tpb - 1) / a.tpb;
  if (blocks > ts_plan::max_blocks(blk.threads))
    return ts_host::fail(TS_ERR_SHAPE, "rope_axes: too many tokens");
  const size_t lds = 2 * sizeof(float) * (size_t)a.tpb * a.half;
  if (a.tpb == 1)
    hipLaunchKernelGGL((rope_axes_kernel<T, kBytes, kInterleaved, true>), dim3((unsigned)blocks),
                       dim3(blk.threads), lds, st, a);
  else
    hipLaunchKernelGGL((rope_axes_kernel<T, kBytes, kInterleaved, false>), dim3((unsigned)blocks),
                       dim3(blk.threads), lds, st, a);
  return ts_host::check_launch("rope_axes_kernel");
}

template <typename T, int kBytes>
ts_status launch_layout(AxesArgs& a, int D, bool interleaved, bool in_place, hipStream_t st) {
  return interleaved ? launch_typed<T, kBytes, true>(a, D, in_place, st)
                     : launch_typed<T, kBytes, false>(a, D, in_place, st);
}

template <typename T>
ts_status launch_rope(AxesArgs& a, int D, bool interleaved, bool in_place, hipStream_t st) {
  constexpr int V = Elt<T>::kVec;
  const int unit = interleaved ? 2 * a.half : a.half;  // what the vectors have to divide
  if (unit % V == 0 && (in_place || D % V == 0))
    return launch_layout<T, 16>(a, D, interleaved, in_place, st);
  if (unit % (V / 2) == 0 && (in_place || D % (V / 2) == 0))
    return launch_layout<T, 8>(a, D, interleaved, in_place, st);
  return launch_layout<T, 0>(a, D, interleaved, in_place, st);
}

}  // namespace

extern "C" ts_status ts_rope_axes(const ts_rope_axes_args* p, ts_stream_t stream) {
  using ts_host::fail;
  if (p == nullptr) return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: NULL arguments");
  if (!ts_host::valid_dtype(p->dtype))
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "rope_axes: bad dtype");
  if (p->B < 0 || p->S < 0 || p->Hq < 0 || p->Hk < 0 || p->D <= 0)
    return fail(TS_ERR_SHAPE, "rope_axes: bad shape B=%lld S=%lld Hq=%lld Hk=%lld D=%lld",
                (long long)p->B, (long long)p->S, (long long)p->Hq, (long long)p->Hk,
                (long long)p->D);
  if (p->R <= 0 || p->R % 2 != 0 || p->R > p->D || p->R / 2 > kMaxHalf)
    return fail(TS_ERR_SHAPE, "rope_axes: %lld rotated of %lld elements (even, at most %d)",
                (long long)p->R, (long long)p->D, 2 * kMaxHalf);
  if (p->D > 4096 || p->Hq + p->Hk > 4096)
    return fail(TS_ERR_SHAPE, "rope_axes: more than 4096 heads or elements of a head");
  if (p->axes < 1 || p->axes > 255)
    return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: 1 to 255 axes, got %d", (int)p->axes);
  if ((p->interleaved != 0 && p->interleaved != 1) || (p->backward != 0 && p->backward != 1))
    return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: interleaved and backward must be 0 or 1");
  if (p->turns == nullptr || p->axis == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: NULL frequencies");
  for (int64_t i = 0; i < p->R / 2; ++i)
    if (p->axis[i] < 0 || p->axis[i] >= p->axes)
      return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: axis %d of pair %lld", (int)p->axis[i],
                  (long long)i);
  if (p->B == 0 || p->S == 0 || p->Hq + p->Hk == 0) return TS_OK;
  if (p->B > ((int64_t)1 << 40) / p->S) return fail(TS_ERR_SHAPE, "rope_axes: too many tokens");
  if ((p->Hq > 0 && (p->q_in == nullptr || p->q_out == nullptr)) ||
      (p->Hk > 0 && (p->k_in == nullptr || p->k_out == nullptr)) || p->position_ids == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "rope_axes: NULL pointer");

  AxesArgs a{};
  a.q_in = p->q_in; a.q_out = p->q_out;
  a.q_in_sb = p->q_in_sb; a.q_in_ss = p->q_in_ss; a.q_in_sh = p->q_in_sh;
  a.q_out_sb = p->q_out_sb; a.q_out_ss = p->q_out_ss; a.q_out_sh = p->q_out_sh;
  a.k_in = p->k_in; a.k_out = p->k_out;
  a.k_in_sb = p->k_in_sb; a.k_in_ss = p->k_in_ss; a.k_in_sh = p->k_in_sh;
  a.k_out_sb = p->k_out_sb; a.k_out_ss = p->k_out_ss; a.k_out_sh = p->k_out_sh;
  a.pos = p->position_ids;
  a.pos_sa = p->pos_sa; a.pos_sb = p->pos_sb; a.pos_ss = p->pos_ss;
  a.S = p->S;
  a.ntok = p->B * p->S;
  a.Hq = (int32_t)p->Hq;
  a.Hk = (int32_t)p->Hk;
  a.half = (int32_t)(p->R / 2);
  a.backward = p->backward;
  for (int i = 0; i < a.half; ++i) {
    a.turns[i] = p->turns[i];
    a.rest[i] = p->turns_rest != nullptr ? p->turns_rest[i] : 0;
    a.axis[i] = (uint8_t)p->axis[i];
  }
  // in place, the elements that stay need no copy
  const bool in_place = (p->Hq == 0 || p->q_in == p->q_out) && (p->Hk == 0 || p->k_in == p->k_out);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool il = p->interleaved != 0;
  switch (p->dtype) {
    case TS_BF16: return launch_rope<__bf16>(a, (int)p->D, il, in_place, st);
    case TS_F16: return launch_rope<_Float16>(a, (int)p->D, il, in_place, st);
    case TS_F32: return launch_rope<float>(a, (int)p->D, il, in_place, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "rope_axes: bad dtype");
}
