// Clipped policy loss with a KL term over token log-probabilities, for gfx950:
//   d = logp - old, r = exp(d), x = ref - logp
//   policy = -min(r A, clip(r, 1 - low, 1 + high) A),  kl = exp(x) - x - 1
//   loss = sum of weight (policy + kl_coef kl) over the valid tokens
//   dloss/dlogp = weight ((clipped ? 0 : -r A) - kl_coef (exp(x) - 1))
// weight: 1 / valid tokens ("token"), 1 / (valid tokens of the sequence * sequences that have
// any) ("sequence"), or 1 ("sum").
//
// A token costs up to 17 bytes of reading in each direction and some 60 operations: bound by
// arithmetic and memory alike for large batches (512 x 8192 fp32 tokens: 24 us for the sums, 10
// to join them, 16 for the backward, where the bytes alone take 8 and 11), and by launches and
// host time for the usual ones (4 x 500 tokens: 10 and 5 us). So: one pass over
// the tokens and one workgroup that joins its partial sums (up to kSmallUnits units: both in one
// launch), one launch backward. A wave owns a unit of kUnit tokens of one row and reduces
// without LDS or barrier; rows of few tokens and few rows of many tokens both spread over the
// chip. The backward forms each token's terms again from the inputs: the weights are known only
// when all tokens have been counted, and reading the inputs twice costs less than writing,
// reading and scaling a gradient.
//
// Numerics: log ratios are differences in double (the inputs' difference is exact there), and a
// token is clipped where d lies beyond log(1 + high) or log(1 - low), compared in double: no
// rounding of exp decides it. The sums' terms are formed and added in double, in a fixed order;
// the gradient's in fp32, and in double where that leaves fp32's range: a far token's exp may
// overflow while its gradient, after the weight, does not. Without an advantage (A = 0) the policy's
// term is 0 for any finite d.
#include <math.h>

#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;

constexpr int kThreads = 256;
constexpr int kFinalThreads = 1024;
constexpr int kPer = 4;                              // neighbouring tokens of a lane in a step
constexpr int kUnit = ts_plan::kPolicyUnit;          // tokens of a wave
constexpr int kSteps = kUnit / (kWave * kPer);
constexpr int kSmallUnits = ts_plan::kPolicySmallUnits;
constexpr int64_t kMaxUnits = ts_plan::max_blocks(kThreads) * (kThreads / kWave);
static_assert(kSteps * kWave * kPer == kUnit, "a unit is whole steps");

struct Unit {
  double policy, kl;
  int clipped, count;
};

struct Rows {  // a [rows, tokens] tensor of log-probs: of the logits' type or fp32; p may be NULL
  const void* p;
  int64_t ld;
  int f32;
};

struct Args {
  Rows logp, old, ref;
  const float* adv;
  int64_t lda;
  int adv_per_token;
  const uint8_t* mask;  // may be NULL: every token is valid
  int64_t ldm;
  int64_t rows, tokens, units_per_row, units;
  double log_high, log_low;  // log(1 + high), log(1 - low)
  double high, low;          // 1 + high, 1 - low
  double kl_coef;
};

typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// kPer values from element i on, of which the first n are read (n == kPer: one load).
template <typename T>
__device__ inline void load_values(const T* p, int n, float (&f)[kPer]) {
  if (n == kPer) {
    if constexpr (sizeof(T) == 4) {
      Elt<float>::unpack(ld16_any(p), f);
    } else {
      const u32x2_any h = *reinterpret_cast<const u32x2_any*>(p);
      const u32x4 q = {h[0], h[1], 0u, 0u};
      float all[Elt<T>::kVec];
      Elt<T>::unpack(q, all);
#pragma unroll
      for (int j = 0; j < kPer; ++j) f[j] = all[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) f[j] = j < n ? Elt<T>::load1(p + j) : 0.f;
  }
}
template <typename T>
__device__ inline void load_rows(const Rows& a, int64_t row, int64_t i, int n, float (&f)[kPer]) {
  if (a.f32)
    load_values<float>(static_cast<const float*>(a.p) + row * a.ld + i, n, f);
  else
    load_values<T>(static_cast<const T*>(a.p) + row * a.ld + i, n, f);
}
// Which of the n tokens are valid, one bit each.
__device__ inline int load_mask(const Args& a, int64_t row, int64_t i, int n) {
  const int all = (1 << n) - 1;
  if (a.mask == nullptr) return all;
  const uint8_t* p = a.mask + row * a.ldm + i;
  int bits = 0;
  if (n == kPer) {
    const uint32_t w = *reinterpret_cast<const u32_any*>(p);
#pragma unroll
    for (int j = 0; j < kPer; ++j) bits |= ((w >> (8 * j)) & 255u) != 0u ? 1 << j : 0;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (j < n && p[j] != 0) bits |= 1 << j;
  }
  return bits;
}

struct Tokens {
  float lp[kPer], old[kPer], ref[kPer], adv[kPer];
  int valid;
};
template <typename T>
__device__ inline void load_tokens(const Args& a, int64_t row, int64_t i, int n, Tokens& t) {
  t.valid = load_mask(a, row, i, n);
  load_rows<T>(a.logp, row, i, n, t.lp);
  if (a.old.p != nullptr) load_rows<T>(a.old, row, i, n, t.old);
  if (a.ref.p != nullptr) load_rows<T>(a.ref, row, i, n, t.ref);
  if (a.adv_per_token) {
    load_values<float>(a.adv + row * a.lda + i, n, t.adv);
  } else {
    const float v = a.adv[row * a.lda];
#pragma unroll
    for (int j = 0; j < kPer; ++j) t.adv[j] = v;
  }
}

// A token's clip test, in double: beyond log(1 + high) or log(1 - low).
__device__ inline bool is_clipped(const Args& a, double d, float adv) {
  return (adv > 0.f && d > a.log_high) || (adv < 0.f && d < a.log_low);
}

// Whether the policy's term is 0 whatever exp(d), which overflows for large d.
__device__ inline bool is_zero(double d, float adv) { return adv == 0.f && fabs(d) < INFINITY; }

// Forward: the terms of the sums in double. The policy's terms have either sign and nearly cancel
// where the advantages are centred, so fp32's rounding of each would show in the loss (2e-6 of it
// at 512 x 8192 tokens).
//
// exp(x) = 2^k exp(r), r = x - k ln 2: exp(r) - 1 - r = r^2 (1/2! + r/3! + ... + r^8/10!) for
// |r| <= ln 2 / 2, whose next term is below 2^-41 of exp(r) - 1 - r. `rise2` is exp(x) - 1 - x,
// which near 0 (k = 0) is that series itself, without cancellation.
__device__ inline double exp_f64(double x, double& rise2) {
  const double c = x < -800. ? -800. : x > 800. ? 800. : x;  // a NaN stays one
  const double k = __builtin_rint(c * 1.4426950408889634);
  double r = __builtin_fma(-k, 0.6931471805599453, c);
  r = __builtin_fma(-k, 2.3190468138462996e-17, r);
  double s = 1. / 3628800.;
  s = __builtin_fma(s, r, 1. / 362880.);
  s = __builtin_fma(s, r, 1. / 40320.);
  s = __builtin_fma(s, r, 1. / 5040.);
  s = __builtin_fma(s, r, 1. / 720.);
  s = __builtin_fma(s, r, 1. / 120.);
  s = __builtin_fma(s, r, 1. / 24.);
  s = __builtin_fma(s, r, 1. / 6.);
  s = __builtin_fma(s, r, 0.5);
  s *= r * r;
  const double e = __builtin_ldexp(1. + (r + s), (int)k);
  rise2 = k == 0. ? s : (e - 1.) - x;
  return e;
}

struct Terms {
  double policy, kl;
  bool clipped;
};
__device__ inline Terms token_terms(const Args& a, float lp, float old, float ref, float adv) {
  Terms t;
  double rise2;
  const double d = a.old.p != nullptr ? (double)lp - (double)old : 0.;
  t.clipped = is_clipped(a, d, adv);
  const double r = t.clipped ? (adv > 0.f ? a.high : a.low) : exp_f64(d, rise2);
  t.policy = is_zero(d, adv) ? 0. : -(r * (double)adv);
  t.kl = 0.;
  if (a.ref.p != nullptr) exp_f64((double)ref - (double)lp, t.kl);
  return t;
}

// Backward, in fp32: exp(x) to about 1.5 units in the last place, 2^(x log2 e) with the product's
// rounding error put back (the hardware's 2^p is good to one). Results below 2^-126 are 0; where
// 2^p overflows the result is an infinity or a NaN (an infinity times the error), which the caller
// forms again in double.
constexpr float kLog2eLow = 1.925963033e-8f;  // log2 e - (float)log2 e
__device__ inline float exp_f32(float x) {
  const float p = x * kLog2e;
  float low = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -p));
  low = fabsf(p) < 1e4f ? low * kLn2 : 0.f;  // minus infinity's error is no number
  const float e = fast_exp2(p);
  return __builtin_fmaf(e, low, e);
}

// exp(x) - 1. Below 1/2 the series x + x^2/2! + ... + x^9/9!, whose next term is below 2^-29 of
// the sum; above, the difference loses at most two bits.
__device__ inline float expm1_f32(float x) {
  float s = 2.75573192e-6f;  // 1/9!
  s = __builtin_fmaf(s, x, 2.48015873e-5f);
  s = __builtin_fmaf(s, x, 1.98412698e-4f);
  s = __builtin_fmaf(s, x, 1.38888889e-3f);
  s = __builtin_fmaf(s, x, 8.33333333e-3f);
  s = __builtin_fmaf(s, x, 4.16666667e-2f);
  s = __builtin_fmaf(s, x, 1.66666667e-1f);
  s = __builtin_fmaf(s, x, 0.5f);
  return fabsf(x) < 0.5f ? __builtin_fmaf(x * x, s, x) : exp_f32(x) - 1.f;
}

// d(policy + kl_coef kl) / d logp of a token. Finite where every step stays in fp32's range.
__device__ inline float token_grad(const Args& a, float lp, float old, float ref, float adv) {
  const double d = a.old.p != nullptr ? (double)lp - (double)old : 0.;
  float g = is_clipped(a, d, adv) ? 0.f : -(exp_f32((float)d) * adv);
  if (a.kl_coef != 0.)
    g = __builtin_fmaf(-(float)a.kl_coef, expm1_f32((float)((double)ref - (double)lp)), g);
  return g;
}

// The same in double, times the weight, rounded once.
__device__ inline float token_grad_f64(const Args& a, float lp, float old, float ref, float adv,
                                       double w) {
  double rise2;
  const double d = a.old.p != nullptr ? (double)lp - (double)old : 0.;
  double g = 0.;
  if (!is_clipped(a, d, adv) && !is_zero(d, adv)) g = -(exp_f64(d, rise2) * (double)adv);
  if (a.kl_coef != 0.) {
    const double x = (double)ref - (double)lp, e = exp_f64(x, rise2);
    g -= a.kl_coef * (fabs(x) < 0.25 ? rise2 + x : e - 1.);
  }
  return (float)(g * w);
}

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}
__device__ inline int wave_sum_int(int v) {
#pragma unroll
  for (int m = kWave / 2; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// The sums of unit u, in every lane of the wave.
template <typename T>
__device__ inline Unit unit_sums(const Args& a, int64_t u) {
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = (uint32_t)u / (uint32_t)a.units_per_row;  // below 2^31
  const int64_t first = (u - row * a.units_per_row) * kUnit + lane * kPer;
  Tokens t[kSteps];
  int n[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int64_t i = first + s * kWave * kPer, left = a.tokens - i;
    n[s] = left >= kPer ? kPer : left > 0 ? (int)left : 0;
    t[s].valid = 0;
    if (n[s] > 0) load_tokens<T>(a, row, i, n[s], t[s]);
  }
  Unit sum = {0., 0., 0, 0};
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if ((t[s].valid >> j) & 1) {
        const Terms e = token_terms(a, t[s].lp[j], t[s].old[j], t[s].ref[j], t[s].adv[j]);
        sum.policy += e.policy;
        sum.kl += e.kl;
        sum.clipped += e.clipped ? 1 : 0;
        ++sum.count;
      }
    }
  }
  sum.policy = wave_sum_f64(sum.policy);
  if (a.ref.p != nullptr) sum.kl = wave_sum_f64(sum.kl);
  sum.clipped = wave_sum_int(sum.clipped);
  sum.count = wave_sum_int(sum.count);
  return sum;
}

struct Outs {
  float *loss, *policy, *kl, *clipped, *weights;
  int reduction;
};

// Joins the units of all rows, in a fixed order, with kFinalThreads threads; `units` is global
// memory or LDS. `lanes` (a power of two up to 64) lanes share a row.
__device__ inline void join_units(const Unit* units, const Args& a, const Outs& o, int lanes) {
  __shared__ double red[kFinalThreads / kWave][5];
  const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
  const int sub = threadIdx.x % lanes;
  const int64_t row0 = threadIdx.x / lanes, step = kFinalThreads / lanes;
  // over the rows: policy, kl, clipped, valid tokens, rows with any (each row's mean of the
  // first three with "sequence", its sum otherwise)
  double all[5] = {0., 0., 0., 0., 0.};
  const int64_t rounds = (a.rows + step - 1) / step;  // uniform: every lane shuffles
  for (int64_t k = 0; k < rounds; ++k) {
    const int64_t row = row0 + k * step;
    double v[3] = {0., 0., 0.};
    int count = 0;  // a row has fewer than 2^31 tokens
    if (row < a.rows) {
#pragma unroll 4
      for (int64_t u = sub; u < a.units_per_row; u += lanes) {
        const Unit x = units[row * a.units_per_row + u];
        v[0] += x.policy;
        v[1] += x.kl;
        v[2] += (double)x.clipped;
        count += x.count;
      }
    }
    for (int m = lanes / 2; m >= 1; m >>= 1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) v[i] += __shfl_xor(v[i], m, kWave);
      count += __shfl_xor(count, m, kWave);
    }
    if (sub == 0 && row < a.rows) {
      const double w =
          o.reduction == TS_POLICY_SEQUENCE ? (count > 0 ? 1. / (double)count : 0.) : 1.;
#pragma unroll
      for (int i = 0; i < 3; ++i) all[i] += v[i] * w;
      all[3] += (double)count;
      all[4] += count > 0 ? 1. : 0.;
      o.weights[row] = (float)w;
    }
  }
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const double s = wave_sum_f64(all[i]);
    if (lane == 0) red[wid][i] = s;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    double s = 0.;
    for (int w = 0; w < kFinalThreads / kWave; ++w) s += red[w][i];
    all[i] = s;
  }
  const double n = o.reduction == TS_POLICY_TOKEN ? all[3] : o.reduction == TS_POLICY_SEQUENCE ? all[4] : 1.;
  const double scale = 1. / (n > 1. ? n : 1.);
  if (threadIdx.x == 0) {
    *o.policy = (float)(all[0] * scale);
    *o.kl = (float)(all[1] * scale);
    *o.clipped = (float)(all[2] * scale);
    // (an infinite KL that is only watched stays out of the loss, as out of the gradient)
    const double kl = a.kl_coef != 0. ? a.kl_coef * all[1] : 0.;
    *o.loss = (float)((all[0] + kl) * scale);
  }
  if (sub == 0)
    for (int64_t row = row0; row < a.rows; row += step)  // the thread's own weights
      o.weights[row] = (float)((double)o.weights[row] * scale);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void policy_units(Args a, Unit* __restrict__ units) {
  const int64_t u = (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave;
  if (u >= a.units) return;  // whole waves
  const Unit s = unit_sums<T>(a, u);
  if ((threadIdx.x & (kWave - 1)) == 0) units[u] = s;
}

__global__ __launch_bounds__(kFinalThreads) void policy_join(const Unit* __restrict__ units, Args a,
                                                             Outs o, int lanes) {
  join_units(units, a, o, lanes);
}

// Few units: sums and join in one workgroup.
template <typename T>
__global__ __launch_bounds__(kFinalThreads) void policy_small(Args a, Outs o, int lanes) {
  __shared__ Unit units[kSmallUnits];
  for (int u = threadIdx.x / kWave; u < (int)a.units; u += kFinalThreads / kWave) {
    const Unit s = unit_sums<T>(a, u);
    if ((threadIdx.x & (kWave - 1)) == 0) units[u] = s;
  }
  __syncthreads();
  join_units(units, a, o, lanes);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void policy_bwd(Args a, const float* __restrict__ weights,
                                                       const float* __restrict__ dloss,
                                                       T* __restrict__ grad, int64_t ldg) {
  const int64_t u = (int64_t)blockIdx.x * (kThreads / kWave) + threadIdx.x / kWave;
  if (u >= a.units) return;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t row = (uint32_t)u / (uint32_t)a.units_per_row;  // below 2^31
  const int64_t first = (u - row * a.units_per_row) * kUnit + lane * kPer;
  const double w64 = (double)weights[row] * (double)*dloss;
  const float w = (float)w64;
  Tokens t[kSteps];
  int n[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const int64_t i = first + s * kWave * kPer, left = a.tokens - i;
    n[s] = left >= kPer ? kPer : left > 0 ? (int)left : 0;
    if (n[s] > 0) load_tokens<T>(a, row, i, n[s], t[s]);
  }
  float far = 0.f;  // a NaN once a gradient of this lane is none or infinite
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    if (n[s] == 0) continue;
    float g[Elt<T>::kVec] = {};
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      if ((t[s].valid >> j) & 1) {
        g[j] = token_grad(a, t[s].lp[j], t[s].old[j], t[s].ref[j], t[s].adv[j]) * w;
        far = __builtin_fmaf(g[j], 0.f, far);
      }
    }
    T* out = grad + row * ldg + first + s * kWave * kPer;
    if (n[s] == kPer) {
      const u32x4 q = Elt<T>::pack(g);
      if constexpr (sizeof(T) == 4)
        st16_any(out, q);
      else
        *reinterpret_cast<u32x2_any*>(out) = u32x2_any{q[0], q[1]};
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j)
        if (j < n[s]) Elt<T>::store1(out + j, g[j]);
    }
  }
  // Rare: those are formed again in double, from the operands read again, and written over.
  // (Behind the steps, where no operand is held any more: in them it took 8 registers more.)
  if (far == 0.f) return;
#pragma unroll 1
  for (int k = 0; k < kSteps * kPer; ++k) {
    const int64_t i = first + k / kPer * (kWave * kPer) + k % kPer;
    T* out = grad + row * ldg + i;
    if (i >= a.tokens || fabsf(Elt<T>::load1(out)) < INFINITY) continue;
    float lp[kPer], old[kPer], ref[kPer];
    load_rows<T>(a.logp, row, i, 1, lp);
    if (a.old.p != nullptr) load_rows<T>(a.old, row, i, 1, old);
    if (a.ref.p != nullptr) load_rows<T>(a.ref, row, i, 1, ref);
    const float adv = a.adv[row * a.lda + (a.adv_per_token ? i : 0)];
    Elt<T>::store1(out, token_grad_f64(a, lp[0], old[0], ref[0], adv, w64));
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

bool misaligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size != 0; }

ts_status check_rows(const char* what, const char* name, const void* p, int64_t ld, int32_t t,
                     int32_t own, int64_t tokens) {
  using ts_host::fail;
  if (p == nullptr) return TS_OK;
  if (!ts_host::valid_dtype(t) || (t != own && t != TS_F32))
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: %s is neither fp32 nor of the log-probs' dtype", what,
                name);
  if (ld < tokens) return fail(TS_ERR_SHAPE, "%s: %s has rows that overlap", what, name);
  if (misaligned(p, ts_host::dtype_size((ts_dtype)t)))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: %s is not aligned to its elements", what, name);
  return TS_OK;
}

ts_status make_args(const char* what, const ts_policy_inputs* in, Args* a) {
  using ts_host::fail;
  if (in == nullptr) return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL inputs", what);
  if (!ts_host::valid_dtype(in->dtype)) return fail(TS_ERR_UNSUPPORTED_DTYPE, "%s: bad dtype", what);
  if (in->rows < 0 || in->tokens < 0) return fail(TS_ERR_SHAPE, "%s: negative size", what);
  if (in->reduction < TS_POLICY_TOKEN || in->reduction > TS_POLICY_SUM)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: bad reduction", what);
  if (!(in->clip_low >= 0.) || !(in->clip_high >= 0.))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: clip bounds must be >= 0", what);
  if (!(in->kl_coef >= 0.) || isinf(in->kl_coef))
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: kl_coef must be finite and >= 0", what);
  if (in->kl_coef > 0. && in->ref == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "%s: kl_coef without reference log-probs", what);
  a->rows = in->rows;
  a->tokens = in->tokens;
  a->units_per_row = (in->tokens + kUnit - 1) / kUnit;
  if (in->tokens > 0x7fffffff || (in->rows > 0 && a->units_per_row > kMaxUnits / in->rows))
    return fail(TS_ERR_SHAPE, "%s: too many tokens", what);
  a->units = a->units_per_row * in->rows;
  if (a->units > 0) {
    if (in->logp == nullptr || in->adv == nullptr)
      return fail(TS_ERR_INVALID_ARGUMENT, "%s: NULL pointer", what);
    ts_status s = check_rows(what, "logp", in->logp, in->ld_logp, in->dtype, in->dtype, in->tokens);
    if (s == TS_OK)
      s = check_rows(what, "old", in->old, in->ld_old, in->old_dtype, in->dtype, in->tokens);
    if (s == TS_OK)
      s = check_rows(what, "ref", in->ref, in->ld_ref, in->ref_dtype, in->dtype, in->tokens);
    if (s == TS_OK)
      s = check_rows(what, "adv", in->adv, in->ld_adv, TS_F32, TS_F32,
                     in->adv_per_token ? in->tokens : 1);
    if (s != TS_OK) return s;
    if (in->mask != nullptr && in->ld_mask < in->tokens)
      return fail(TS_ERR_SHAPE, "%s: mask has rows that overlap", what);
  }
  a->logp = Rows{in->logp, in->ld_logp, in->dtype == TS_F32};
  a->old = Rows{in->old, in->ld_old, in->old_dtype == TS_F32};
  a->ref = Rows{in->ref, in->ld_ref, in->ref_dtype == TS_F32};
  a->adv = in->adv;
  a->lda = in->ld_adv;
  a->adv_per_token = in->adv_per_token != 0;
  a->mask = in->mask;
  a->ldm = in->ld_mask;
  a->log_high = log1p(in->clip_high);
  a->log_low = in->clip_low < 1. ? log1p(-in->clip_low) : -INFINITY;
  a->high = 1. + in->clip_high;
  a->low = 1. - in->clip_low;
  a->kl_coef = in->kl_coef;
  return TS_OK;
}

}  // namespace

extern "C" size_t ts_policy_loss_workspace_size(int64_t rows, int64_t tokens) {
  if (rows <= 0 || tokens <= 0) return 0;
  const int64_t per = (tokens + kUnit - 1) / kUnit;
  if (tokens > 0x7fffffff || per > kMaxUnits / rows || per * rows <= kSmallUnits) return 0;
  return (size_t)(per * rows) * sizeof(Unit);
}

extern "C" ts_status ts_policy_loss_fwd(const ts_policy_inputs* in, float* loss, float* policy_loss,
                                        float* kl, float* clip_fraction, float* weights,
                                        void* workspace, size_t workspace_bytes,
                                        ts_stream_t stream) {
  using ts_host::fail;
  Args a;
  ts_status s = make_args("policy_loss_fwd", in, &a);
  if (s != TS_OK) return s;
  if (loss == nullptr || policy_loss == nullptr || kl == nullptr || clip_fraction == nullptr ||
      (weights == nullptr && a.rows > 0))
    return fail(TS_ERR_INVALID_ARGUMENT, "policy_loss_fwd: NULL pointer");
  const size_t need = ts_policy_loss_workspace_size(a.rows, a.tokens);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need || misaligned(workspace, 8)))
    return fail(TS_ERR_WORKSPACE, "policy_loss_fwd: workspace missing, too small or unaligned");
  const Outs o{loss, policy_loss, kl, clip_fraction, weights, in->reduction};
  // lanes that share a row in the join: as many as leave all rows one round
  int lanes = 1;
  while (lanes < kWave && lanes < a.units_per_row && 2 * lanes * a.rows <= kFinalThreads) lanes *= 2;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (need == 0) {  // no tokens at all: zeros
    const dim3 grid(1), block(kFinalThreads);
    switch (in->dtype) {
      case TS_BF16: hipLaunchKernelGGL(policy_small<__bf16>, grid, block, 0, st, a, o, lanes); break;
      case TS_F16: hipLaunchKernelGGL(policy_small<_Float16>, grid, block, 0, st, a, o, lanes); break;
      default: hipLaunchKernelGGL(policy_small<float>, grid, block, 0, st, a, o, lanes);
    }
    return ts_host::check_launch("policy_small");
  }
  Unit* units = static_cast<Unit*>(workspace);
  constexpr int kWaves = kThreads / kWave;
  const dim3 grid((unsigned)((a.units + kWaves - 1) / kWaves)), block(kThreads);
  switch (in->dtype) {
    case TS_BF16: hipLaunchKernelGGL(policy_units<__bf16>, grid, block, 0, st, a, units); break;
    case TS_F16: hipLaunchKernelGGL(policy_units<_Float16>, grid, block, 0, st, a, units); break;
    default: hipLaunchKernelGGL(policy_units<float>, grid, block, 0, st, a, units);
  }
  s = ts_host::check_launch("policy_units");
  if (s != TS_OK) return s;
  hipLaunchKernelGGL(policy_join, dim3(1), dim3(kFinalThreads), 0, st, units, a, o, lanes);
  return ts_host::check_launch("policy_join");
}

extern "C" ts_status ts_policy_loss_bwd(const ts_policy_inputs* in, const float* weights,
                                        const float* dloss, void* dlogp, int64_t ld_dlogp,
                                        ts_stream_t stream) {
  using ts_host::fail;
  Args a;
  const ts_status s = make_args("policy_loss_bwd", in, &a);
  if (s != TS_OK || a.units == 0) return s;
  if (weights == nullptr || dloss == nullptr || dlogp == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "policy_loss_bwd: NULL pointer");
  if (ld_dlogp < a.tokens) return fail(TS_ERR_SHAPE, "policy_loss_bwd: rows that overlap");
  if (misaligned(dlogp, ts_host::dtype_size((ts_dtype)in->dtype)))
    return fail(TS_ERR_INVALID_ARGUMENT, "policy_loss_bwd: dlogp is not aligned to its elements");
  hipStream_t st = static_cast<hipStream_t>(stream);
  constexpr int kWaves = kThreads / kWave;
  const dim3 grid((unsigned)((a.units + kWaves - 1) / kWaves)), block(kThreads);
  switch (in->dtype) {
    case TS_BF16:
      hipLaunchKernelGGL(policy_bwd<__bf16>, grid, block, 0, st, a, weights, dloss,
                         static_cast<__bf16*>(dlogp), ld_dlogp);
      break;
    case TS_F16:
      hipLaunchKernelGGL(policy_bwd<_Float16>, grid, block, 0, st, a, weights, dloss,
                         static_cast<_Float16*>(dlogp), ld_dlogp);
      break;
    default:
      hipLaunchKernelGGL(policy_bwd<float>, grid, block, 0, st, a, weights, dloss,
                         static_cast<float*>(dlogp), ld_dlogp);
  }
  return ts_host::check_launch("policy_bwd");
}
