// Token embedding with scaling, and its gradient by sorted tokens, for gfx950:
//   out[n, :]  = round(scale * weight[id[n], :])
//   grad[v, :] = round(scale * sum over n with id[n] = v of dout[n, :])     (fp32 sums)
// An id outside [0, V) gives a row of NaN and no gradient; the padding id gives no gradient.
//
// Forward: a gather, HBM-bound (one row read and one written per token), one 16-byte vector a
// thread. The rows are read through the caches: frequent tokens' rows come from there (16384
// tokens of 4096 bf16: 33 us against 47 us with streaming loads).
//
// Backward: HBM-bound by the dense gradient (V rows written, N read). The tokens are sorted by
// id, stably, so the tokens of every gradient row are one run of the sorted list: its sum is
// formed and written once, without atomics on floats, in an order that depends on the ids alone.
// The sort is a radix sort of (id, position) pairs by digits of up to 10 bits: ids below 2^20
// take two passes (a histogram and a scatter each). Up to kEmbedSmallTokens tokens are placed by
// counting, in one launch. Padding and out-of-range ids get the key V, behind all rows.
//
// Most rows of a large vocabulary have no token. The whole gradient is cleared by a plain fill,
// which runs at the card's write rate, and the rows with tokens are written over it: 16384
// tokens of 128256 x 4096 bf16 took 249 us with one kernel over all rows (each looked up in the
// sorted list, then zeroed or summed: the few sums hold up the stores behind them). The fill
// waits for nothing and the sort occupies a few workgroups, so every launch of the sort carries
// a share of the fill as further workgroups: 161 us in all for that gradient (6.5 TB/s), the sort
// within it, then 33 to 48 us for the rows with tokens.
//
// Token frequencies are far from uniform (a frequent token, or one filler token in most places,
// would leave one workgroup with thousands of rows), so runs are cut: wherever kEmbedChunk
// neighbours in the sorted list, from a multiple of kEmbedChunk on, share one id, their sum is
// formed beforehand as one fp32 row, and the same again over kEmbedChunk such sums. A row's sum
// then reads at most 2 (kEmbedChunk - 1) token rows, twice as many rows of sums, and
// N / kEmbedChunk^2 rows of sums of sums. Which stretches those are follows from the sorted ids:
// no list is kept.
#include "common.hpp"
#include "plan.hpp"

namespace {

using namespace ts;
using ts_plan::kEmbedChunk;

constexpr int kThreads = 256;
constexpr int kWaveKeys = 256;                   // keys of a wave in one step: 4 a lane
constexpr int kKeysPerLane = kWaveKeys / kWave;
constexpr int kMaxBins = 1 << ts_plan::kEmbedMaxBits;

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------

// One 16-byte vector of a row, or the row's last elements (v == nvec, fewer than a vector).
template <typename T>
__device__ inline void load_part(const T* __restrict__ row, int v, int nvec, int tail,
                                 float (&f)[Elt<T>::kVec]) {
  constexpr int V = Elt<T>::kVec;
  if (v < nvec) {
    Elt<T>::unpack(ld16_any(row + (int64_t)v * V), f);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = i < tail ? Elt<T>::load1(row + (int64_t)v * V + i) : 0.f;
  }
}
template <typename T>
__device__ inline void store_part(T* __restrict__ row, int v, int nvec, int tail,
                                  const float (&f)[Elt<T>::kVec]) {
  constexpr int V = Elt<T>::kVec;
  if (v < nvec) {
    st16_any_stream(row + (int64_t)v * V, Elt<T>::pack(f));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < tail) Elt<T>::store1(row + (int64_t)v * V + i, f[i]);
  }
}

template <typename T, int TPR>
__global__ __launch_bounds__(kThreads) void embed_fwd(const int64_t* __restrict__ ids, int64_t N,
                                                      const T* __restrict__ w, int64_t ldw,
                                                      int64_t V, int nvec, int tail, int slices,
                                                      float scale, T* __restrict__ out,
                                                      int64_t ldo) {
  constexpr int VE = Elt<T>::kVec;
  const int64_t n = (int64_t)(blockIdx.x / slices) * (kThreads / TPR) + threadIdx.x / TPR;
  const int v = (int)(blockIdx.x % slices) * TPR + threadIdx.x % TPR;
  if (n >= N || v >= nvec + (tail > 0)) return;
  const int64_t id = ids[n];
  const bool in = id >= 0 && id < V;
  const T* row = w + (in ? id : 0) * ldw;
  T* o = out + n * ldo;
  float f[VE];
  load_part(row, v, nvec, tail, f);
#pragma unroll
  for (int i = 0; i < VE; ++i) f[i] = in ? f[i] * scale : __builtin_nanf("");
  store_part(o, v, nvec, tail, f);
}

// ---------------------------------------------------------------------------
// Fill with zeros: bytes [first, first + bytes) of the gradient, the share of one launch
// ---------------------------------------------------------------------------
struct Fill {
  uint8_t* p;
  int64_t bytes;
};
constexpr int kFillBytes = 16 * kThreads;  // of a workgroup

// Workgroup `block` of those that fill, a vector a thread: the fastest fill found (four vectors a
// thread 5.8 TB/s, one 6.5; workgroups of 1024 threads 6.1).
__device__ inline void fill_zero(const Fill& f, int64_t block) {
  const int64_t nvec = f.bytes / 16, v = block * kThreads + threadIdx.x;
  if (v < nvec) st16_any_stream(f.p + v * 16, u32x4{0u, 0u, 0u, 0u});
  // the last bytes, in elements of two
  const int64_t e = nvec * 16 + threadIdx.x * 2;
  if (block == 0 && e < f.bytes) *reinterpret_cast<uint16_t*>(f.p + e) = 0;
}

__global__ __launch_bounds__(kThreads) void embed_fill(Fill f) { fill_zero(f, blockIdx.x); }

// ---------------------------------------------------------------------------
// Sort of (key, position) by key
// ---------------------------------------------------------------------------

__device__ inline uint32_t key_of(int64_t id, int64_t V, int64_t padding) {
  return id >= 0 && id < V && id != padding ? (uint32_t)id : (uint32_t)V;
}

// Lanes of the wave whose key is valid and has this lane's digit.
__device__ inline uint64_t same_digit(uint32_t digit, int bits, bool valid) {
  uint64_t m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1u;
    const uint64_t bal = __ballot(one);
    m &= one ? bal : ~bal;
  }
  return m;
}

// Exclusive prefix sums over the workgroup's threads (kT of them); `lds` holds kT / 64 + 1.
template <int kT>
__device__ inline int block_exclusive(int v, int* lds) {
  const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
  int inc = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int u = __shfl_up(inc, d, kWave);
    if (lane >= d) inc += u;
  }
  if (lane == kWave - 1) lds[wid] = inc;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int i = 0; i < kT / kWave; ++i) before += i < wid ? lds[i] : 0;
  __syncthreads();
  return before + inc - v;
}

// Ranks the wave's keys among equal digits of the wave, in their order: rank[r] for key r * 64 +
// lane; cnt[digit] (the wave's own, cleared) ends as the digit's count.
__device__ inline void wave_ranks(const uint32_t (&digit)[kKeysPerLane],
                                  const bool (&valid)[kKeysPerLane], int bits, volatile int* cnt,
                                  int (&rank)[kKeysPerLane]) {
  const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
  for (int r = 0; r < kKeysPerLane; ++r) {
    const uint64_t m = same_digit(digit[r], bits, valid[r]);
    const int below = __popcll(m & ((1ull << lane) - 1));
    const int prev = valid[r] ? cnt[digit[r]] : 0;
    __builtin_amdgcn_wave_barrier();
    if (valid[r] && below == 0) cnt[digit[r]] = prev + __popcll(m);
    __builtin_amdgcn_wave_barrier();
    rank[r] = prev + below;
  }
}

// Up to kEmbedSmallTokens tokens, one launch: a key's place is the number of smaller keys and of
// equal ones before it. Workgroup b < blocks places the keys [b kRankKeys, (b + 1) kRankKeys): its
// lanes form groups of kRankKeys, a key a lane, and the groups share the list, which each
// workgroup holds in LDS, and add their counts up. 67 million comparisons for 8192 keys, two
// operations each, beside the whole of the gradient's fill, which the other workgroups do. 16
// keys a workgroup: with 32 the counting ends late (8192 tokens, 65 MB of gradient: 26 us with
// 16, 35 with 32), with 8 too many workgroups load the list (33).
constexpr int kRankKeys = 16;
constexpr int kRankGroups = kThreads / kRankKeys;

__global__ __launch_bounds__(kThreads) void sort_ranks(const int64_t* __restrict__ ids, int N,
                                                       int64_t V, int64_t padding,
                                                       uint32_t* __restrict__ keys,
                                                       uint32_t* __restrict__ vals, int blocks,
                                                       Fill fill) {
  extern __shared__ __attribute__((aligned(16))) uint32_t key[];  // the padded list
  __shared__ int counts[kRankGroups][kRankKeys];
  if ((int)blockIdx.x >= blocks) return fill_zero(fill, (int)blockIdx.x - blocks);
  const ts_plan::EmbedRanks p = ts_plan::embed_ranks(N, kRankGroups);
  // behind the list: no key is as large
  for (int i = threadIdx.x; i < p.padded; i += kThreads)
    key[i] = i < N ? key_of(ids[i], V, padding) : ~0u;
  __syncthreads();
  const int lane = threadIdx.x % kRankKeys, group = threadIdx.x / kRankKeys;
  const int own = (int)blockIdx.x * kRankKeys, i = own + lane;
  const uint32_t k = key[i];
  int count = 0;
  for (int j = group * p.len; j < (group + 1) * p.len; j += 8) {
    // before the workgroup's own keys equal ones count (own and len: multiples of 8)
    const uint32_t t = k + (j < own ? 1u : 0u);
    const uint4 q = *reinterpret_cast<const uint4*>(key + j);
    const uint4 r = *reinterpret_cast<const uint4*>(key + j + 4);
    count += (q.x < t) + (q.y < t) + (q.z < t) + (q.w < t);
    count += (r.x < t) + (r.y < t) + (r.z < t) + (r.w < t);
  }
  counts[group][lane] = count;
  __syncthreads();
  if (group != 0 || i >= N) return;
  int at = 0;
#pragma unroll 4
  for (int g = 0; g < kRankGroups; ++g) at += counts[g][lane];
#pragma unroll 4
  for (int j = 0; j < kRankKeys; ++j) at += j < lane && key[own + j] == k;
  keys[at] = k;
  vals[at] = (uint32_t)i;
}

// One pass over many workgroups: workgroup b < blocks owns keys [b * len, (b + 1) * len), those
// behind fill. First the digits' counts, table[b][digit], then the scatter, whose workgroups each
// form the digits' starts from the whole table (at most kEmbedMaxBlocks rows of it).
template <bool kFirst>
__global__ __launch_bounds__(kThreads) void sort_counts(const int64_t* __restrict__ ids,
                                                        const uint32_t* __restrict__ keys_in,
                                                        int64_t N, int64_t len, int64_t V,
                                                        int64_t padding, int shift, int bits,
                                                        int* __restrict__ table, int blocks,
                                                        Fill fill) {
  __shared__ int cnt[kMaxBins];
  if ((int)blockIdx.x >= blocks) return fill_zero(fill, (int)blockIdx.x - blocks);
  const int bins = 1 << bits;
  for (int d = threadIdx.x; d < bins; d += kThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * len;
  const int64_t end = first + len < N ? first + len : N;
  for (int64_t i = first + threadIdx.x; i < end; i += kThreads) {
    const uint32_t key = kFirst ? key_of(ids[i], V, padding) : keys_in[i];
    atomicAdd(&cnt[(key >> shift) & (uint32_t)(bins - 1)], 1);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kThreads) table[(int64_t)blockIdx.x * bins + d] = cnt[d];
}

template <bool kFirst>
__global__ __launch_bounds__(kThreads) void sort_scatter(
    const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys_in,
    const uint32_t* __restrict__ vals_in, int64_t N, int64_t len, int64_t V, int64_t padding,
    int shift, int bits, const int* __restrict__ table, uint32_t* __restrict__ keys_out,
    uint32_t* __restrict__ vals_out, int blocks, Fill fill) {
  constexpr int kWaves = kThreads / kWave;
  constexpr int kPer = kMaxBins / kThreads;  // most bins of a thread
  __shared__ int cnt[kWaves][kMaxBins];
  __shared__ int base[kMaxBins];
  __shared__ int scan[kWaves];
  if ((int)blockIdx.x >= blocks) return fill_zero(fill, (int)blockIdx.x - blocks);
  const int lane = threadIdx.x & (kWave - 1), wid = threadIdx.x / kWave;
  const int bins = 1 << bits;
  const int per = bins > kThreads ? bins / kThreads : 1;
  {
    int total[kPer], before[kPer], sum = 0;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      total[k] = before[k] = 0;
      const int d = threadIdx.x * per + k;
      if (k < per && d < bins) {
#pragma unroll 8
        for (int b = 0; b < blocks; ++b) {
          const int c = table[(int64_t)b * bins + d];
          total[k] += c;
          before[k] += b < (int)blockIdx.x ? c : 0;
        }
      }
      sum += total[k];
    }
    int at = block_exclusive<kThreads>(sum, scan);
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int d = threadIdx.x * per + k;
      if (k < per && d < bins) base[d] = at + before[k];
      at += total[k];
    }
  }
  const int64_t first = (int64_t)blockIdx.x * len;
  const int64_t end = first + len < N ? first + len : N;
  for (int64_t start = first; start < end; start += kWaves * kWaveKeys) {
    for (int i = threadIdx.x; i < kWaves * bins; i += kThreads) cnt[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();  // also orders base, and the last step's reads of cnt
    uint32_t key[kKeysPerLane], val[kKeysPerLane], digit[kKeysPerLane];
    bool valid[kKeysPerLane];
    int rank[kKeysPerLane];
#pragma unroll
    for (int r = 0; r < kKeysPerLane; ++r) {
      const int64_t i = start + wid * kWaveKeys + r * kWave + lane;
      valid[r] = i < end;
      if constexpr (kFirst) {
        key[r] = valid[r] ? key_of(ids[i], V, padding) : 0;
        val[r] = (uint32_t)i;
      } else {
        key[r] = valid[r] ? keys_in[i] : 0;
        val[r] = valid[r] ? vals_in[i] : 0;
      }
      digit[r] = (key[r] >> shift) & (uint32_t)(bins - 1);
    }
    wave_ranks(digit, valid, bits, cnt[wid], rank);
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kThreads) {
      int at = base[d];
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const int c = cnt[w][d];
        cnt[w][d] = at;
        at += c;
      }
      base[d] = at;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kKeysPerLane; ++r) {
      if (valid[r]) {
        const int pos = cnt[wid][digit[r]] + rank[r];
        keys_out[pos] = key[r];
        vals_out[pos] = val[r];
      }
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Sums
// ---------------------------------------------------------------------------

// Adds part v of token rows token(i), i in [i0, i1), to acc, kU rows in flight. The rows are read
// through the caches: what the layer above has just written is there in part (measured over all
// of the backward's reads, 50 -> 40 us for 16384 tokens of 4096 bf16).
template <int kU, typename T, typename F>
__device__ inline void add_tokens(const T* __restrict__ dout, int64_t ldd, F token, int64_t i0,
                                  int64_t i1, int v, int nvec, int tail,
                                  float (&acc)[Elt<T>::kVec]) {
  constexpr int V = Elt<T>::kVec;
  for (int64_t i = i0; i < i1; i += kU) {
    const T* row[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) row[u] = dout + (int64_t)token(i + u < i1 ? i + u : i) * ldd;
    if (v < nvec) {
      u32x4 q[kU];
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (i + u < i1) q[u] = ld16_any(row[u] + (int64_t)v * V);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (i + u < i1) {
          float f[V];
          Elt<T>::unpack(q[u], f);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += f[e];
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (i + u < i1) {
          float f[V];
          load_part(row[u], v, nvec, tail, f);
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] += f[e];
        }
      }
    }
  }
}

// Adds part v of rows c0 .. c1 - 1 of fp32 sums.
template <int V>
__device__ inline void add_sums(const float* __restrict__ sums, int64_t ld, int64_t c0, int64_t c1,
                                int v, float (&acc)[V]) {
  constexpr int kU = 4;
  for (int64_t c = c0; c < c1; c += kU) {
    float4 q[kU][V / 4];
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int h = 0; h < V / 4; ++h)
        if (c + u < c1)
          q[u][h] = *reinterpret_cast<const float4*>(sums + (c + u) * ld + (int64_t)v * V + 4 * h);
#pragma unroll
    for (int u = 0; u < kU; ++u)
#pragma unroll
      for (int h = 0; h < V / 4; ++h) {
        if (c + u < c1) {
          acc[4 * h] += q[u][h].x;
          acc[4 * h + 1] += q[u][h].y;
          acc[4 * h + 2] += q[u][h].z;
          acc[4 * h + 3] += q[u][h].w;
        }
      }
  }
}

// Sum of chunk c where all of it is one row's: from its kEmbedChunk tokens (kLevel 1), or from
// the sums of its kEmbedChunk chunks (kLevel 2). A row is cut into slices of TPR vectors.
template <typename T, int TPR, int kLevel>
__global__ __launch_bounds__(kThreads) void embed_chunk_sums(
    const T* __restrict__ dout, int64_t ldd, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ vals, int64_t chunks, uint32_t none, int nvec, int tail,
    int slices, const float* __restrict__ sums_in, float* __restrict__ sums_out, int64_t ld) {
  constexpr int V = Elt<T>::kVec;
  constexpr int64_t kSpan = kLevel == 1 ? kEmbedChunk : (int64_t)kEmbedChunk * kEmbedChunk;
  const int64_t c = (int64_t)(blockIdx.x / slices) * (kThreads / TPR) + threadIdx.x / TPR;
  const int v = (int)(blockIdx.x % slices) * TPR + threadIdx.x % TPR;
  if (c >= chunks || v >= nvec + (tail > 0)) return;
  const uint32_t key = keys[c * kSpan];
  if (key == none || key != keys[c * kSpan + kSpan - 1]) return;
  float acc[V] = {};
  if constexpr (kLevel == 1)
    add_tokens<8>(dout, ldd, [=](int64_t i) { return vals[i]; }, c * kSpan, c * kSpan + kSpan, v,
                  nvec, tail, acc);
  else
    add_sums<V>(sums_in, ld, c * kEmbedChunk, (c + 1) * kEmbedChunk, v, acc);
#pragma unroll
  for (int h = 0; h < V / 4; ++h)
    *reinterpret_cast<float4*>(sums_out + c * ld + (int64_t)v * V + 4 * h) =
        make_float4(acc[4 * h], acc[4 * h + 1], acc[4 * h + 2], acc[4 * h + 3]);
}

// First index in [lo, N) whose key is not `key`, which the keys before lo have.
__device__ inline int64_t run_end(const uint32_t* __restrict__ keys, int64_t N, int64_t lo,
                                  uint32_t key) {
  int64_t hi = N, step = 1;
  while (lo + step <= N && keys[lo + step - 1] == key) {
    lo += step;
    step *= 2;
  }
  if (lo + step - 1 < N) hi = lo + step - 1;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] == key) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// The rows that have tokens: the lanes of position i in the sorted list take the run that begins
// there, if one does. Where the lanes are whole waves, each wave reads the pairs of positions
// i - 1 .. i + 62 at once: whether a run begins, where it ends and which tokens it has follow
// without another load (16384 tokens of 4096 bf16: 60 -> 50 us). Two token rows in flight a lane:
// most runs are short, and fewer registers mean more runs at a time (8 rows 40 us, 2 rows 33).
template <typename T, int TPR>
__global__ __launch_bounds__(kThreads) void embed_runs(
    const T* __restrict__ dout, int64_t ldd, const uint32_t* __restrict__ keys,
    const uint32_t* __restrict__ vals, int64_t N, uint32_t none, int nvec, int tail, int slices,
    const float* __restrict__ sums1, const float* __restrict__ sums2, int64_t ld, float scale,
    T* __restrict__ grad) {
  constexpr int VE = Elt<T>::kVec;
  const int64_t i = (int64_t)(blockIdx.x / slices) * (kThreads / TPR) + threadIdx.x / TPR;
  if (i >= N) return;
  const int part = (int)(blockIdx.x % slices) * TPR + threadIdx.x % TPR;
  const bool mine = part < nvec + (tail > 0);
  // lanes behind the row's end read its first part for nothing: the wave stays whole where lanes
  // read one another's tokens
  const int v = mine ? part : 0;
  float acc[VE] = {};
  uint32_t key;
  int64_t e;
  bool done = false;
  if constexpr (TPR >= kWave) {
    const int64_t j = i - 1 + (threadIdx.x & (kWave - 1));
    const bool in = j >= 0 && j < N;
    const uint32_t k = in ? keys[j] : ~0u, t = in ? vals[j] : 0u;  // ~0: no key
    key = __builtin_amdgcn_readlane(k, 1);
    if (key == none || key == (uint32_t)__builtin_amdgcn_readlane(k, 0)) return;
    const uint64_t other = __ballot(k != key) & ~1ull;
    e = other != 0 ? i - 1 + __builtin_ctzll(other) : run_end(keys, N, i + kWave - 1, key);
    if (ts_plan::embed_run(i, e).t0 == e && other != 0) {  // no whole chunk: these tokens alone
      const int n = (int)(e - i);
      add_tokens<2>(dout, ldd,
                    [=](int64_t a) { return (uint32_t)__builtin_amdgcn_readlane(t, (int)a + 1); },
                    0, n, v, nvec, tail, acc);
      done = true;
    }
  } else {
    key = keys[i];
    if (key == none || (i > 0 && keys[i - 1] == key)) return;
    e = run_end(keys, N, i + 1, key);
  }
  if (!done) {
    const ts_plan::EmbedRun run = ts_plan::embed_run(i, e);
    const auto token = [=](int64_t a) { return vals[a]; };
    add_tokens<2>(dout, ldd, token, i, run.t0, v, nvec, tail, acc);
    add_sums<VE>(sums1, ld, run.a0, run.a1, v, acc);
    add_sums<VE>(sums2, ld, run.b0, run.b1, v, acc);
    add_sums<VE>(sums1, ld, run.c0, run.c1, v, acc);
    add_tokens<2>(dout, ldd, token, run.t1, e, v, nvec, tail, acc);
  }
#pragma unroll
  for (int k = 0; k < VE; ++k) acc[k] *= scale;
  if (mine) store_part(grad + (int64_t)key * ((int64_t)nvec * VE + tail), v, nvec, tail, acc);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

template <typename T>
ts_status fwd_typed(const int64_t* ids, int64_t N, const void* w, int64_t ldw, int64_t V, int64_t H,
                    float scale, void* out, int64_t ldo, hipStream_t st) {
  const int nvec = (int)(H / Elt<T>::kVec), tail = (int)(H % Elt<T>::kVec);
  const int parts = nvec + (tail > 0);
  const int tpr = ts_plan::embed_fwd_lanes(parts);
  const int slices = (parts + tpr - 1) / tpr;
  const int64_t per = kThreads / tpr, blocks = (N + per - 1) / per * slices;
  if (blocks > ts_plan::max_blocks(kThreads))
    return ts_host::fail(TS_ERR_SHAPE, "embedding_fwd: too many tokens");
#define TS_FWD(R)                                                                             \
  hipLaunchKernelGGL((embed_fwd<T, R>), dim3((unsigned)blocks), dim3(kThreads), 0, st, ids, N, \
                     static_cast<const T*>(w), ldw, V, nvec, tail, slices, scale, static_cast<T*>(out), \
                     ldo)
  switch (tpr) {
    case 8: TS_FWD(8); break;
    case 32: TS_FWD(32); break;
    case 128: TS_FWD(128); break;
    default: TS_FWD(256); break;
  }
#undef TS_FWD
  return ts_host::check_launch("embed_fwd");
}

struct BwdArgs {
  const int64_t* ids;
  int64_t N, V, H, padding, ldd;
  const void* dout;
  void* grad;
  float scale;
  uint8_t* ws;
};

// The next of `left` shares of the gradient's fill.
Fill next_fill(uint8_t** p, int64_t* bytes, int left) {
  const int64_t n = left > 1 ? *bytes / left / kFillBytes * kFillBytes : *bytes;
  const Fill f{*p, n};
  *p += n;
  *bytes -= n;
  return f;
}
int64_t fill_blocks(const Fill& f) { return (f.bytes + kFillBytes - 1) / kFillBytes; }

// Clears the gradient and sorts the tokens; *keys and *vals are where the sorted pairs end up.
ts_status launch_sort(const BwdArgs& a, const ts_plan::EmbedWorkspace& w, int64_t grad_bytes,
                      const uint32_t** keys, const uint32_t** vals, hipStream_t st) {
  const ts_plan::EmbedSort p = ts_plan::embed_sort(a.N, a.V);
  uint32_t* k[2] = {reinterpret_cast<uint32_t*>(a.ws + w.keys[0]),
                    reinterpret_cast<uint32_t*>(a.ws + w.keys[1])};
  uint32_t* v[2] = {reinterpret_cast<uint32_t*>(a.ws + w.vals[0]),
                    reinterpret_cast<uint32_t*>(a.ws + w.vals[1])};
  *keys = k[0];
  *vals = v[0];
  uint8_t* to_fill = static_cast<uint8_t*>(a.grad);
  if (a.N == 0) {
    const Fill f{to_fill, grad_bytes};
    hipLaunchKernelGGL(embed_fill, dim3((unsigned)fill_blocks(f)), dim3(kThreads), 0, st, f);
    return ts_host::check_launch("embed_fill");
  }
  if (p.blocks == 0) {
    const Fill f{to_fill, grad_bytes};
    const int list = ts_plan::embed_ranks((int)a.N, kRankGroups).padded;
    const int ranks = (int)((a.N + kRankKeys - 1) / kRankKeys);
    hipLaunchKernelGGL(sort_ranks, dim3((unsigned)(ranks + fill_blocks(f))),
                       dim3(kThreads), 4 * (size_t)list, st, a.ids, (int)a.N, a.V, a.padding,
                       k[0], v[0], ranks, f);
    return ts_host::check_launch("sort_ranks");
  }
  int* table = reinterpret_cast<int*>(a.ws + w.table);
  const int blocks = (int)p.blocks;
  int left = 2 * p.passes;
  const dim3 block(kThreads);
  for (int i = 0; i < p.passes; ++i) {
    const int shift = i * p.bits, to = i & 1, from = to ^ 1;
    const Fill f1 = next_fill(&to_fill, &grad_bytes, left--);
    const Fill f2 = next_fill(&to_fill, &grad_bytes, left--);
    const dim3 g1((unsigned)(blocks + fill_blocks(f1))), g2((unsigned)(blocks + fill_blocks(f2)));
    if (i == 0) {
      hipLaunchKernelGGL(sort_counts<true>, g1, block, 0, st, a.ids, k[from], a.N, p.len, a.V,
                         a.padding, shift, p.bits, table, blocks, f1);
      hipLaunchKernelGGL(sort_scatter<true>, g2, block, 0, st, a.ids, k[from], v[from], a.N,
                         p.len, a.V, a.padding, shift, p.bits, table, k[to], v[to], blocks, f2);
    } else {
      hipLaunchKernelGGL(sort_counts<false>, g1, block, 0, st, a.ids, k[from], a.N, p.len, a.V,
                         a.padding, shift, p.bits, table, blocks, f1);
      hipLaunchKernelGGL(sort_scatter<false>, g2, block, 0, st, a.ids, k[from], v[from], a.N,
                         p.len, a.V, a.padding, shift, p.bits, table, k[to], v[to], blocks, f2);
    }
    const ts_status s = ts_host::check_launch("sort_scatter");
    if (s != TS_OK) return s;
    *keys = k[to];
    *vals = v[to];
  }
  return TS_OK;
}

template <typename T, int TPR>
ts_status bwd_shaped(const BwdArgs& a, hipStream_t st) {
  constexpr int VE = Elt<T>::kVec;
  constexpr int kSlots = kThreads / TPR;
  const ts_plan::EmbedWorkspace w = ts_plan::embed_workspace(a.N, a.V, a.H);
  const int nvec = (int)(a.H / VE), tail = (int)(a.H % VE), parts = nvec + (tail > 0);
  const int slices = (parts + TPR - 1) / TPR;
  const int64_t c1 = a.N / kEmbedChunk, c2 = c1 / kEmbedChunk;
  const int64_t grad_bytes = a.V * a.H * (int64_t)sizeof(T);
  const int64_t runs = (a.N + kSlots - 1) / kSlots * slices;
  const int64_t b1 = (c1 + kSlots - 1) / kSlots * slices, b2 = (c2 + kSlots - 1) / kSlots * slices;
  if (runs > ts_plan::max_blocks(kThreads) ||
      grad_bytes / kFillBytes > ts_plan::max_blocks(kThreads) - 1024)
    return ts_host::fail(TS_ERR_SHAPE, "embedding_bwd: tensor too large");
  const uint32_t *keys, *vals;
  const ts_status s = launch_sort(a, w, grad_bytes, &keys, &vals, st);
  if (s != TS_OK || a.N == 0) return s;
  const T* dout = static_cast<const T*>(a.dout);
  float* sums1 = reinterpret_cast<float*>(a.ws + w.sums1);
  float* sums2 = reinterpret_cast<float*>(a.ws + w.sums2);
  const uint32_t none = (uint32_t)a.V;
  if (c1 > 0)
    hipLaunchKernelGGL((embed_chunk_sums<T, TPR, 1>), dim3((unsigned)b1), dim3(kThreads), 0, st,
                       dout, a.ldd, keys, vals, c1, none, nvec, tail, slices, sums2, sums1, w.ld);
  if (c2 > 0)
    hipLaunchKernelGGL((embed_chunk_sums<T, TPR, 2>), dim3((unsigned)b2), dim3(kThreads), 0, st,
                       dout, a.ldd, keys, vals, c2, none, nvec, tail, slices, sums1, sums2, w.ld);
  hipLaunchKernelGGL((embed_runs<T, TPR>), dim3((unsigned)runs), dim3(kThreads), 0, st, dout, a.ldd,
                     keys, vals, a.N, none, nvec, tail, slices, sums1, sums2, w.ld, a.scale,
                     static_cast<T*>(a.grad));
  return ts_host::check_launch("embed_runs");
}

template <typename T>
ts_status bwd_typed(const BwdArgs& a, hipStream_t st) {
  const int64_t parts = (a.H + Elt<T>::kVec - 1) / Elt<T>::kVec;
  if (parts <= 8) return bwd_shaped<T, 8>(a, st);
  if (parts <= 32) return bwd_shaped<T, 32>(a, st);
  if (parts <= 128) return bwd_shaped<T, 128>(a, st);
  return bwd_shaped<T, 256>(a, st);
}

bool bad_address(const void* p, ts_dtype t) {
  return reinterpret_cast<uintptr_t>(p) % ts_host::dtype_size(t) != 0;
}

}  // namespace

extern "C" ts_status ts_embedding_fwd(const int64_t* ids, int64_t N, const void* weight,
                                      int64_t ldw, ts_dtype dtype, int64_t V, int64_t H,
                                      float scale, void* out, int64_t ldo, ts_stream_t stream) {
  using ts_host::fail;
  if (!ts_host::valid_dtype(dtype))
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "embedding_fwd: bad dtype");
  if (N < 0 || V < 0 || H < 0 || H > 0x7fffffff)
    return fail(TS_ERR_SHAPE, "embedding_fwd: bad sizes");
  if (N == 0 || H == 0) return TS_OK;
  if (V == 0) return fail(TS_ERR_SHAPE, "embedding_fwd: no rows to look up");
  if (ldw < H || ldo < H) return fail(TS_ERR_SHAPE, "embedding_fwd: row stride below the width");
  if (ids == nullptr || weight == nullptr || out == nullptr)
    return fail(TS_ERR_INVALID_ARGUMENT, "embedding_fwd: NULL pointer");
  if (bad_address(weight, dtype) || bad_address(out, dtype) ||
      reinterpret_cast<uintptr_t>(ids) % 8 != 0)
    return fail(TS_ERR_INVALID_ARGUMENT, "embedding_fwd: a tensor is not aligned to its elements");
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_BF16: return fwd_typed<__bf16>(ids, N, weight, ldw, V, H, scale, out, ldo, st);
    case TS_F16: return fwd_typed<_Float16>(ids, N, weight, ldw, V, H, scale, out, ldo, st);
    case TS_F32: return fwd_typed<float>(ids, N, weight, ldw, V, H, scale, out, ldo, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "embedding_fwd: bad dtype");
}

extern "C" size_t ts_embedding_bwd_workspace_size(int64_t N, int64_t V, int64_t H) {
  if (N < 0 || V < 0 || H < 0 || N > ts_plan::kEmbedMaxIndex || V > ts_plan::kEmbedMaxIndex ||
      H > 0x7fffffff)
    return 0;
  return (size_t)ts_plan::embed_workspace(N, V, H).bytes;
}

extern "C" ts_status ts_embedding_bwd(const int64_t* ids, int64_t N, const void* dout, int64_t ldd,
                                      ts_dtype dtype, int64_t V, int64_t H, float scale,
                                      int64_t padding_idx, void* grad_weight, void* workspace,
                                      size_t workspace_bytes, ts_stream_t stream) {
  using ts_host::fail;
  if (!ts_host::valid_dtype(dtype))
    return fail(TS_ERR_UNSUPPORTED_DTYPE, "embedding_bwd: bad dtype");
  if (N < 0 || V < 0 || H < 0 || N > ts_plan::kEmbedMaxIndex || V > ts_plan::kEmbedMaxIndex ||
      H > 0x7fffffff)
    return fail(TS_ERR_SHAPE, "embedding_bwd: bad sizes");
  if (V == 0 || H == 0) return TS_OK;
  if (grad_weight == nullptr || (N > 0 && (ids == nullptr || dout == nullptr)))
    return fail(TS_ERR_INVALID_ARGUMENT, "embedding_bwd: NULL pointer");
  if (N > 0 && ldd < H) return fail(TS_ERR_SHAPE, "embedding_bwd: row stride below the width");
  if (bad_address(grad_weight, dtype) || bad_address(dout, dtype) ||
      reinterpret_cast<uintptr_t>(ids) % 8 != 0)
    return fail(TS_ERR_INVALID_ARGUMENT, "embedding_bwd: a tensor is not aligned to its elements");
  if (workspace_bytes < ts_embedding_bwd_workspace_size(N, V, H) || workspace == nullptr ||
      !ts_host::aligned16(workspace))
    return fail(TS_ERR_WORKSPACE, "embedding_bwd: workspace missing, too small or unaligned");
  const BwdArgs a{ids, N, V, H, padding_idx, ldd, dout, grad_weight, scale,
                  static_cast<uint8_t*>(workspace)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TS_BF16: return bwd_typed<__bf16>(a, st);
    case TS_F16: return bwd_typed<_Float16>(a, st);
    case TS_F32: return bwd_typed<float>(a, st);
  }
  return fail(TS_ERR_UNSUPPORTED_DTYPE, "embedding_bwd: bad dtype");
}
