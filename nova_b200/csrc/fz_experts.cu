// Mixture of experts: the router's gate, tokens sorted by expert and back, and their
// gradients. All are bound by memory (or, for a handful of tokens, by launch latency):
// every kernel reads its inputs once and writes its outputs once, with no atomics on
// floating-point values, so results do not depend on scheduling.
// Measured (B200, copy bandwidth 6.55 TB/s): router, 65536 tokens, 256 experts, 8 picks, all
// logits normalised: 32 us (0.34 of the copy bandwidth: instruction issue), backward 28 us
// (0.77). 16384 tokens of 4096 floats, 4 of 64 experts, capacity 1280: sort 12 us (latency of
// its three steps), dispatch 268 us (0.92), combine 178 us, its backward 416 us (0.98).
#include <cooperative_groups.h>

#include <climits>
#include <cstdint>

#include "fz_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;

bool aligned16(const void *a, const void *b = nullptr, const void *c = nullptr) {
  return (((uintptr_t)a | (uintptr_t)b | (uintptr_t)c) & 15) == 0;
}

// ---------------------------------------------------------------- router

// Logits as unsigned keys in the same order: NaN above all (an addition gives the canonical,
// positive NaN), -0 equal to +0, and 0 free to mark what has been taken.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(__fadd_rn(v, 0.0f));
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_key(uint32_t key) {
  return __uint_as_float(key ^ ((uint32_t)((int32_t)~key >> 31) | 0x80000000u));
}
constexpr uint32_t kKeyMinusInf = 0x007fffffu;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kFull, v, d));
  return v;
}

// e^(v - top), at most 1: the hardware's 2^x (2 ulp) of (v - top) log2(e). With d = top - v that
// argument's roundings make the relative error up to 2^-24 (4 + 2.2 d): small weights have fewer
// digits, in proportion to their logarithm. (expf would hold 2 ulp for all; its instructions would
// add to what the forward is bound by.)
__device__ __forceinline__ float exp_below(float v, float top) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(__fmul_rn(__fsub_rn(v, top), 1.4426950408889634f)));
  return y;
}

// Descending sort of a lane's N keys: Batcher's odd-even merge network.
template <int N>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q > 0; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t x = key[i + j], y = key[i + j + q];
            key[i + j] = max(x, y);
            key[i + j + q] = min(x, y);
          }
}

template <int NE>
__device__ __forceinline__ void load_row(float (&v)[NE], const float *row, int lane, int experts) {
#pragma unroll
  for (int i = 0; i < NE; ++i) v[i] = lane + 32 * i < experts ? row[lane + 32 * i] : -INFINITY;
}

// A warp's token, expert e = lane + 32 i in register i of lane `lane`. Experts are picked by
// their keys alone: every lane sorts its own keys once, a pick is the largest of the lanes'
// heads (one warp-wide reduction) and its lane moves its list up. Then the experts whose keys
// were picked are found in ascending order, each taking the first open pick of its key: ties
// go to the lowest experts, and those that are too many find none.
template <int NE>
__device__ __forceinline__ void route_token(float *weights, int32_t *ids, const float (&v)[NE], int64_t t,
                                            int experts, int k, int renormalize, int lane) {
  uint32_t own[NE], key[NE];
#pragma unroll
  for (int i = 0; i < NE; ++i) own[i] = key[i] = order_key(v[i]);
  sort_keys(key);
  uint32_t mine = 0;  // lane j: the j-th pick's key; 0: none
  for (int j = 0; j < k; ++j) {
    const uint32_t top = __reduce_max_sync(kFull, key[0]);
    if (top <= kKeyMinusInf) break;  // only -inf (or nothing) left
    const int owner = __ffs(__ballot_sync(kFull, key[0] == top)) - 1;
    if (lane == j) mine = top;
    if (lane == owner) {
#pragma unroll
      for (int i = 0; i + 1 < NE; ++i) key[i] = key[i + 1];
      key[NE - 1] = 0;
    }
  }
  const uint32_t last = __reduce_min_sync(kFull, mine ? mine : 0xffffffffu);  // the smallest picked
  const bool any = __any_sync(kFull, mine != 0);
  int id = -1;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    unsigned found = __ballot_sync(kFull, any && own[i] >= last);
    while (found) {
      const int from = __ffs(found) - 1;
      found &= found - 1;
      const uint32_t its = __shfl_sync(kFull, own[i], from);
      const unsigned open = __ballot_sync(kFull, mine == its && id < 0);
      if (lane == __ffs(open) - 1) id = from + 32 * i;
    }
  }
  const float logit = from_key(mine);
  const float top = __shfl_sync(kFull, logit, 0);
  const float num = id >= 0 ? exp_below(logit, top) : 0.0f;
  float den = num;
  if (!renormalize) {
    den = 0.0f;
#pragma unroll
    for (int i = 0; i < NE; ++i) den = __fadd_rn(den, lane + 32 * i < experts ? exp_below(v[i], top) : 0.0f);
  }
  den = warp_sum(den);
  if (lane < k) {
    weights[t * k + lane] = id >= 0 ? __fdiv_rn(num, den) : 0.0f;
    ids[t * k + lane] = id;
  }
}

// One warp per token, the next token's logits fetched ahead.
template <int NE>
__global__ void __launch_bounds__(256) route_kernel(float *__restrict__ weights, int32_t *__restrict__ ids,
                                                    const float *__restrict__ logits, int64_t tokens, int experts,
                                                    int k, int renormalize) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  float v[NE], next[NE];
  if (t < tokens) load_row(next, logits + t * experts, lane, experts);
  for (; t < tokens; t += warps) {
#pragma unroll
    for (int i = 0; i < NE; ++i) v[i] = next[i];
    if (t + warps < tokens) load_row(next, logits + (t + warps) * experts, lane, experts);
    route_token(weights, ids, v, t, experts, k, renormalize, lane);
  }
}

// The K largest of two descending lists of K, descending, in a.
template <int K>
__device__ __forceinline__ void merge_keys(uint32_t (&a)[K], const uint32_t (&b)[K]) {
#pragma unroll
  for (int i = 0; i < K; ++i) a[i] = max(a[i], b[K - 1 - i]);  // a bitonic sequence
#pragma unroll
  for (int d = K / 2; d > 0; d /= 2)
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (!(i & d)) {
        const uint32_t x = a[i], y = a[i + d];
        a[i] = max(x, y);
        a[i + d] = min(x, y);
      }
}

// L lanes per token, expert e = sub + L i in register i (at most L N experts, K <= L picks).
// Bound by instruction issue, which the 32 / L tokens of a warp share: a lane's K largest keys come
// from sorting networks, the token's from rounds of merging with another lane's, with
// no exchange per pick. A pick's place is the number of larger keys, so that each lane
// writes its own picks. Tokens with equal keys among their picks or at their end, or with
// a NaN, are left to route_token. (With a warp a token throughout: 65536 tokens, 256 experts, 8
// picks 49 us, 32 so; 16384 tokens, 1024 experts, 8 picks 110 us, 39 so.)
template <int L, int N, int K>
__global__ void __launch_bounds__(256) route_team_kernel(float *__restrict__ weights, int32_t *__restrict__ ids,
                                                         const float *__restrict__ logits, int64_t tokens,
                                                         int experts, int k, int renormalize) {
  pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane % L;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t w = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); w * (32 / L) < tokens; w += warps) {
    const int64_t t = w * (32 / L) + lane / L;
    const bool on = t < tokens;
    const float *row = logits + t * experts;
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = on && sub + L * i < experts ? row[sub + L * i] : -INFINITY;
    uint32_t top[K];
#pragma unroll
    for (int g = 0; g < N; g += K) {
      uint32_t key[K];
#pragma unroll
      for (int i = 0; i < K; ++i) key[i] = order_key(v[g + i]);
      sort_keys(key);
      if (g == 0) {
#pragma unroll
        for (int i = 0; i < K; ++i) top[i] = key[i];
      } else {
        merge_keys(top, key);
      }
    }
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
      uint32_t other[K];
#pragma unroll
      for (int i = 0; i < K; ++i) other[i] = __shfl_xor_sync(kFull, top[i], d);
      merge_keys(top, other);
    }
    int picks = 0;
    uint32_t last = 0, mine = 0;  // the smallest key picked; lane j's: the j-th
    bool odd = top[0] == 0xffffffffu;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      const bool picked = j < k && top[j] > kKeyMinusInf;
      picks += picked;
      if (picked) odd = odd || (j > 0 && top[j] == last);
      if (picked) last = top[j];
      if (picked && j == sub) mine = top[j];
    }
    const float end = from_key(last), most = from_key(top[0]);
    unsigned chosen = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) chosen |= (unsigned)(v[i] >= end) << i;
    if (picks == 0) chosen = 0;
    int count = __popc(chosen);
    float den = mine ? exp_below(from_key(mine), most) : 0.0f;
    if (!renormalize) {
      den = 0.0f;
#pragma unroll
      for (int i = 0; i < N; ++i) den = __fadd_rn(den, exp_below(v[i], most));  // -inf: 0
    }
#pragma unroll
    for (int d = 1; d < L; d *= 2) {
      count += __shfl_xor_sync(kFull, count, d);
      den = __fadd_rn(den, __shfl_xor_sync(kFull, den, d));
    }
    odd = odd || count != picks;
    if (odd) chosen = 0;
    while (__any_sync(kFull, chosen != 0)) {
      if (chosen) {
        const int e = sub + L * (__ffs(chosen) - 1);
        chosen &= chosen - 1;
        const float x = row[e];
        const uint32_t key = order_key(x);
        int place = 0;
#pragma unroll
        for (int j = 0; j < K; ++j) place += top[j] > key;
        weights[t * k + place] = __fdiv_rn(exp_below(x, most), den);
        ids[t * k + place] = e;
      }
    }
    if (on && !odd && sub >= picks && sub < k) {
      weights[t * k + sub] = 0.0f;
      ids[t * k + sub] = -1;
    }
    for (unsigned left = __ballot_sync(kFull, odd && sub == 0); left; left &= left - 1) {
      const int64_t its = w * (32 / L) + (__ffs(left) - 1) / L;
      float u[N * L / 32];
      load_row(u, logits + its * experts, lane, experts);
      route_token(weights, ids, u, its, experts, k, renormalize, lane);
    }
  }
}

// One warp per token; the chosen experts' upstream gradients are spread over a row in
// shared memory, which the warp then turns into the row of dlogits.
template <int NE>
__global__ void __launch_bounds__(256) route_backward_kernel(float *__restrict__ dlogits,
                                                             const float *__restrict__ dweights,
                                                             const float *__restrict__ weights,
                                                             const int32_t *__restrict__ ids,
                                                             const float *__restrict__ logits, int64_t tokens,
                                                             int experts, int k, int renormalize) {
  pdl_wait();
  __shared__ float rows[8][NE * 32];
  const int lane = threadIdx.x & 31;
  float *up = rows[threadIdx.x >> 5];
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  int64_t t = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  float v[NE], next[NE], next_w = 0.0f, next_dw = 0.0f;
  int next_id = -1;
  const auto fetch = [&](int64_t at) {
    if (at >= tokens) return;
    if (!renormalize) load_row(next, logits + at * experts, lane, experts);
    if (lane < k) {
      next_id = ids[at * k + lane];
      next_w = weights[at * k + lane];
      next_dw = dweights[at * k + lane];
    }
  };
  fetch(t);
#pragma unroll
  for (int i = 0; i < NE; ++i) up[lane + 32 * i] = 0.0f;
  for (; t < tokens; t += warps) {
    const bool held = next_id >= 0 && next_id < experts;
    const int id = held ? next_id : -1;
    const float w = held ? next_w : 0.0f, dw = held ? next_dw : 0.0f;
    if (!renormalize)
#pragma unroll
      for (int i = 0; i < NE; ++i) v[i] = next[i];
    fetch(t + warps);
    const float dot = warp_sum(__fmul_rn(w, dw));
    const bool any = __any_sync(kFull, held);
    __syncwarp();
    if (held) up[id] = renormalize ? __fmul_rn(w, __fsub_rn(dw, dot)) : dw;
    __syncwarp();
    float *out = dlogits + t * experts;
    if (renormalize || !any) {
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (lane + 32 * i < experts) out[lane + 32 * i] = up[lane + 32 * i];
    } else {
      float top = v[0];
#pragma unroll
      for (int i = 1; i < NE; ++i) top = fmaxf(top, v[i]);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, d));
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        v[i] = lane + 32 * i < experts ? exp_below(v[i], top) : 0.0f;
        s = __fadd_rn(s, v[i]);
      }
      const float inv = __fdiv_rn(1.0f, warp_sum(s));
#pragma unroll
      for (int i = 0; i < NE; ++i)
        if (lane + 32 * i < experts)
          out[lane + 32 * i] = __fmul_rn(__fmul_rn(v[i], inv), __fsub_rn(up[lane + 32 * i], dot));
    }
    __syncwarp();
    if (held) up[id] = 0.0f;  // the row is clean again for the next token
  }
}

// ---------------------------------------------------------------- sort by expert

// One cluster sorts everything (a counting sort): each warp owns a contiguous run of
// choices and counts them per expert in shared memory; the CTAs exchange their totals
// through distributed shared memory; then each warp places its run, in order, from its
// own first place per expert. Equal experts within a warp's 32 choices are ranked by
// ballots over the expert's bits, so the order is stable whatever the scheduling.
// The ids of the next kSortAhead groups of 32 are in flight.
constexpr int kSortAhead = 4, kMaxSortCtas = 16;
__global__ void __launch_bounds__(1024) sort_kernel(int32_t *__restrict__ slot, int32_t *__restrict__ src,
                                                    int32_t *__restrict__ counts, int32_t *__restrict__ offsets,
                                                    const int32_t *__restrict__ ids, int n, int experts,
                                                    int capacity, int rows, int per_warp, int bits) {
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nwarps = blockDim.x >> 5;
  extern __shared__ int32_t sh[];
  int32_t *hist = sh;                       // [nwarps][experts]: counts, then the next place among the CTA's choices
  int32_t *total = sh + nwarps * experts;   // [experts]: this CTA's counts
  int32_t *start = total + experts;         // [experts]: the expert's first row
  int32_t *all = start + experts;           // [experts]: counts over the cluster
  int32_t *ahead = all + experts;           // [experts]: counts of the CTAs before this one
  __shared__ int32_t scan[32];

  for (int i = tid; i < nwarps * experts; i += blockDim.x) hist[i] = 0;
  __syncthreads();
  const int64_t first = ((int64_t)rank * nwarps + warp) * per_warp;
  const int end = (int)(first + per_warp < n ? first + per_warp : n);
  int32_t *mine = hist + warp * experts;
  // an id; `experts` if it names none
  const auto read = [&](int64_t i) {
    const int e = i < end ? ids[i] : -1;
    return e >= 0 && e < experts ? e : experts;
  };
  for (int64_t i0 = first; i0 < end; i0 += 32 * kSortAhead) {
    int e[kSortAhead];
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) e[u] = read(i0 + u * 32 + lane);
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u)
      if (e[u] < experts) atomicAdd(&mine[e[u]], 1);
  }
  __syncthreads();
  // exclusive sums over this CTA's warps, eight loads in flight
  for (int e = tid; e < experts; e += blockDim.x) {
    int s = 0;
    for (int w0 = 0; w0 < nwarps; w0 += 8) {
      int c[8];
#pragma unroll
      for (int w = 0; w < 8; ++w) c[w] = hist[(w0 + w) * experts + e];
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        hist[(w0 + w) * experts + e] = s;
        s += c[w];
      }
    }
    total[e] = s;
  }
  if (ctas > 1) cluster.sync();
  else __syncthreads();
  // counts over the cluster, and those of the CTAs before this one
  for (int e = tid; e < experts; e += blockDim.x) {
    int c[kMaxSortCtas], s = 0, before = 0;
#pragma unroll
    for (int r = 0; r < kMaxSortCtas; ++r) c[r] = r < ctas ? cluster.map_shared_rank(total, r)[e] : 0;
#pragma unroll
    for (int r = 0; r < kMaxSortCtas; ++r) {
      before += r < rank ? c[r] : 0;
      s += c[r];
    }
    all[e] = s;
    ahead[e] = before;
  }
  // the experts' first rows: e * capacity, or the exclusive sum of the counts
  // (experts <= 1024 = one value a thread over up to 1024 threads; fewer threads loop)
  __syncthreads();
  int carry = 0;
  for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
    const int e = e0 + tid;
    const int c = e < experts ? all[e] : 0;
    int x = c;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(kFull, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) scan[warp] = x;
    __syncthreads();
    int before = 0, sum = 0;
    for (int w = 0; w < nwarps; ++w) {
      if (w < warp) before += scan[w];
      sum += scan[w];
    }
    if (e < experts) {
      const int begin = capacity ? e * capacity : carry + before + x - c;
      start[e] = begin;
      if (rank == 0) {
        counts[e] = c;
        offsets[e] = begin;
      }
    }
    carry += sum;
    __syncthreads();
  }
  if (rank == 0 && tid == 0) offsets[experts] = capacity ? experts * capacity : carry;
  // empty rows
  if (capacity) {
    for (int64_t r = rank * (int)blockDim.x + tid; r < rows; r += ctas * (int)blockDim.x)
      if ((int)r % capacity >= all[(int)r / capacity]) src[r] = -1;
  } else {
    for (int64_t r = (int64_t)carry + rank * (int)blockDim.x + tid; r < rows; r += ctas * (int)blockDim.x) src[r] = -1;
  }
  // places
  int next[kSortAhead];
#pragma unroll
  for (int u = 0; u < kSortAhead; ++u) next[u] = read(first + u * 32 + lane);
  for (int64_t i0 = first; i0 < end; i0 += 32 * kSortAhead) {
    int e[kSortAhead];
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      e[u] = next[u];
      next[u] = read(i0 + (kSortAhead + u) * 32 + lane);
    }
#pragma unroll
    for (int u = 0; u < kSortAhead; ++u) {
      const int64_t i = i0 + u * 32 + lane;
      unsigned peers = kFull;  // the lanes with this lane's expert
      for (int b = 0; b < bits; ++b) {
        const unsigned set = __ballot_sync(kFull, e[u] >> b & 1);
        peers &= e[u] >> b & 1 ? set : ~set;
      }
      const bool has = e[u] < experts;
      int at = -1;
      if (has) {
        at = ahead[e[u]] + mine[e[u]] + __popc(peers & ((1u << lane) - 1u));
        at = capacity && at >= capacity ? -1 : start[e[u]] + at;
      }
      __syncwarp();
      if (has && lane == __ffs(peers) - 1) mine[e[u]] += __popc(peers);
      __syncwarp();
      if (i < end) {
        slot[i] = at;
        if (at >= 0) src[at] = (int)i;
      }
    }
  }
  if (ctas > 1) cluster.sync();  // no CTA leaves while another may read its totals
}

// ---------------------------------------------------------------- rows to experts and back

// Work is cut into pieces of one token and kUnroll vectors a lane, taken by a team of P
// lanes: a warp (rows of many vectors: several pieces), or 8 or 2 lanes where a row has at
// most 32 or 8 vectors, so that narrow rows do not leave a warp's lanes idle (32768 tokens of
// 16 floats, 8 choices: combine 32 us with a warp a token, 11 us so). VEC = 4: rows of float4
// (width a multiple of 4, 16-byte aligned buffers), else 1. Every value is read or written
// once: the token's row once for its k copies, each expert's row once.
constexpr int kUnroll = 4;

template <int VEC>
struct Vec;
template <>
struct Vec<4> {
  using T = float4;
  static __device__ __forceinline__ T zero() { return make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  static __device__ __forceinline__ T fma(float w, T y, T a) {
    return make_float4(__fmaf_rn(w, y.x, a.x), __fmaf_rn(w, y.y, a.y), __fmaf_rn(w, y.z, a.z),
                       __fmaf_rn(w, y.w, a.w));
  }
  static __device__ __forceinline__ T scale(float w, T y) {
    return make_float4(__fmul_rn(w, y.x), __fmul_rn(w, y.y), __fmul_rn(w, y.z), __fmul_rn(w, y.w));
  }
  static __device__ __forceinline__ float dot(T a, T b, float s) {
    return __fmaf_rn(a.w, b.w, __fmaf_rn(a.z, b.z, __fmaf_rn(a.y, b.y, __fmaf_rn(a.x, b.x, s))));
  }
};
template <>
struct Vec<1> {
  using T = float;
  static __device__ __forceinline__ T zero() { return 0.0f; }
  static __device__ __forceinline__ T fma(float w, T y, T a) { return __fmaf_rn(w, y, a); }
  static __device__ __forceinline__ T scale(float w, T y) { return __fmul_rn(w, y); }
  static __device__ __forceinline__ float dot(T a, T b, float s) { return __fmaf_rn(a, b, s); }
};

// Zero the piece [c0, c0 + 32 * kUnroll) of the empty ones among 32 rows from r0.
template <int VEC>
__device__ __forceinline__ void zero_empty(typename Vec<VEC>::T *rows, const int32_t *src, int64_t r0,
                                           int64_t num_rows, int64_t nvec, int64_t c0, int lane) {
  const int64_t r = r0 + lane;
  unsigned empty = __ballot_sync(kFull, r < num_rows && src[r < num_rows ? r : 0] < 0);
  while (empty) {
    const int b = __ffs(empty) - 1;
    empty &= empty - 1;
    typename Vec<VEC>::T *row = rows + (r0 + b) * nvec;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t c = c0 + u * 32 + lane;
      if (c < nvec) row[c] = Vec<VEC>::zero();
    }
  }
}

template <int VEC, int P>
__global__ void __launch_bounds__(256) dispatch_kernel(typename Vec<VEC>::T *__restrict__ rows,
                                                       const typename Vec<VEC>::T *__restrict__ x,
                                                       const int32_t *__restrict__ slot,
                                                       const int32_t *__restrict__ src, int64_t tokens, int64_t k,
                                                       int64_t num_rows, int64_t nvec, int64_t chunks) {
  using V = Vec<VEC>;
  pdl_wait();
  constexpr int kTeams = 32 / P;
  const int lane = threadIdx.x & 31, sub = lane % P;
  // warps' pieces: of kTeams tokens each, then groups of 32 rows to look for empty ones in
  const int64_t work = (tokens * chunks + kTeams - 1) / kTeams;
  const int64_t zero_chunks = (nvec + 32 * kUnroll - 1) / (32 * kUnroll);
  const int64_t all = work + (num_rows + 31) / 32 * zero_chunks;
  const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t p = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); p < all; p += warps) {
    if (p >= work) {
      const int64_t q = p - work, g = q / zero_chunks;
      zero_empty<VEC>(rows, src, g * 32, num_rows, nvec, (q - g * zero_chunks) * 32 * kUnroll, lane);
      continue;
    }
    const int64_t piece = p * kTeams + lane / P, t = piece / chunks, c0 = (piece - t * chunks) * P * kUnroll + sub;
    if (t >= tokens) continue;
    typename V::T v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) v[u] = c0 + u * P < nvec ? x[t * nvec + c0 + u * P] : V::zero();
    for (int64_t j = 0; j < k; ++j) {
      const int64_t r = slot[t * k + j];
      if (r < 0 || r >= num_rows) continue;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (c0 + u * P < nvec) rows[r * nvec + c0 + u * P] = v[u];
    }
  }
}

template <int VEC, int P>
__global__ void __launch_bounds__(256) combine_kernel(typename Vec<VEC>::T *__restrict__ out,
                                                      const typename Vec<VEC>::T *__restrict__ rows,
                                                      const float *__restrict__ weights,
                                                      const int32_t *__restrict__ slot, int64_t tokens, int64_t k,
                                                      int64_t num_rows, int64_t nvec, int64_t chunks) {
  using V = Vec<VEC>;
  pdl_wait();
  constexpr int kTeams = 32 / P;
  const int lane = threadIdx.x & 31, sub = lane % P;
  const int64_t work = (tokens * chunks + kTeams - 1) / kTeams, warps = (int64_t)gridDim.x * (blockDim.x >> 5);
  for (int64_t p = (int64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); p < work; p += warps) {
    const int64_t piece = p * kTeams + lane / P, t = piece / chunks, c0 = (piece - t * chunks) * P * kUnroll + sub;
    if (t >= tokens) continue;
    typename V::T acc[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) acc[u] = V::zero();
    for (int64_t j = 0; j < k; ++j) {
      const int64_t r = slot[t * k + j];
      if (r < 0 || r >= num_rows) continue;
      const float w = weights ? weights[t * k + j] : 1.0f;
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (c0 + u * P < nvec) acc[u] = V::fma(w, rows[r * nvec + c0 + u * P], acc[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (c0 + u * P < nvec) out[t * nvec + c0 + u * P] = acc[u];
  }
}

// A team takes one choice: its row of drows and its dweight.
template <int VEC, int P>
__global__ void __launch_bounds__(256) combine_backward_kernel(
    typename Vec<VEC>::T *__restrict__ drows, float *__restrict__ dweights,
    const typename Vec<VEC>::T *__restrict__ dout, const typename Vec<VEC>::T *__restrict__ rows,
    const float *__restrict__ weights, const int32_t *__restrict__ slot, const int32_t *__restrict__ src,
    int64_t tokens, int64_t k, int64_t num_rows, int64_t nvec) {
  using V = Vec<VEC>;
  pdl_wait();
  // threads that go through the pieces together, a warp or a CTA, and their teams
  constexpr int kUnit = P > 32 ? P : 32, kTeams = kUnit / P, kWarps = kUnit / 32;
  const int lane = threadIdx.x & 31, sub = threadIdx.x % P, warp = threadIdx.x % kUnit / 32;
  const int64_t choices = tokens * k, work = (choices + kTeams - 1) / kTeams;
  const int64_t zero_chunks = (nvec + 32 * kUnroll - 1) / (32 * kUnroll);
  const int64_t zeros = (num_rows + 31) / 32 * zero_chunks, all = work + (zeros + kWarps - 1) / kWarps;
  const int64_t units = (int64_t)gridDim.x * (blockDim.x / kUnit);
  __shared__ float sums[2][kWarps];
  int parity = 0;
  for (int64_t p = (int64_t)blockIdx.x * (blockDim.x / kUnit) + threadIdx.x / kUnit; p < all; p += units) {
    if (p >= work) {
      const int64_t q = (p - work) * kWarps + warp, g = q / zero_chunks;
      if (q < zeros)
        zero_empty<VEC>(drows, src, g * 32, num_rows, nvec, (q - g * zero_chunks) * 32 * kUnroll, lane);
      continue;
    }
    const int64_t choice = p * kTeams + threadIdx.x % kUnit / P, r = choice < choices ? slot[choice] : -1;
    float s = 0.0f;
    if (r >= 0 && r < num_rows) {
      const float w = weights ? weights[choice] : 1.0f;
      const typename V::T *g = dout + choice / k * nvec;
      for (int64_t c0 = sub; c0 < nvec; c0 += P * kUnroll) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int64_t c = c0 + u * P;
          if (c < nvec) {
            const typename V::T d = g[c];
            if (dweights) s = V::dot(d, rows[r * nvec + c], s);
            drows[r * nvec + c] = V::scale(w, d);
          }
        }
      }
    }
    if (dweights) {
#pragma unroll
      for (int d = (P > 32 ? 32 : P) / 2; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(kFull, s, d));
      if constexpr (P > 32) {
        if (lane == 0) sums[parity][warp] = s;
        __syncthreads();  // one a choice: the next one's sums go to the other half
        s = sums[parity][0];
#pragma unroll
        for (int i = 1; i < kWarps; ++i) s = __fadd_rn(s, sums[parity][i]);
        parity ^= 1;
      }
      if (sub == 0 && choice < choices) dweights[choice] = s;
    }
  }
}

// Arguments that dispatch, combine and its backward share.
int check_rows(const char *who, int64_t tokens, int64_t k, int64_t num_rows, int64_t width) {
  const std::string name(who);
  FZ_REQUIRE(tokens >= 0 && k >= 1 && num_rows >= 0 && width >= 0, name + ": negative size or k < 1");
  FZ_REQUIRE(k <= INT_MAX && tokens <= INT_MAX / k && num_rows <= INT_MAX,
             name + ": tokens * k and the rows must be below 2^31");
  FZ_REQUIRE(width <= INT_MAX, name + ": width must be below 2^31");
  return FZ_OK;
}

// Lanes a row of nvec vectors, and f(Lanes<P>) for them.
template <int P>
struct Lanes {
  static constexpr int value = P;
};
template <class F>
int with_lanes(int64_t nvec, F f) {
  if (nvec <= 2 * kUnroll) return f(Lanes<2>{});
  if (nvec <= 8 * kUnroll) return f(Lanes<8>{});
  return f(Lanes<32>{});
}
// Whether a choice's gradients are a CTA's work, not a warp's: where a row is at least three
// passes of the CTA, or of two of a warp's and there are fewer choices than warps. Warps are slow
// on few rows (288 tokens of 6843 floats, 2 choices, 121 us against 11; 600 of 4096, 4 choices,
// 27 against 17) and a little on many (8192 of 4096, 2 choices, 108 against 103); CTAs on many
// shorter rows (16384 of 2400, 2 choices, 142 us against 131).
bool wide_choices(int64_t choices, int64_t nvec) {
  return nvec >= 768 || (nvec > 256 && choices < (int64_t)32 * fz::num_sms());
}
int64_t chunks_of(int64_t nvec, int lanes) { return (nvec + lanes * kUnroll - 1) / (lanes * kUnroll); }
// Pieces of `tokens` rows for warps, and of the rows that may be empty.
int64_t warp_pieces(int64_t tokens, int64_t chunks, int lanes) { return (tokens * chunks * lanes + 31) / 32; }
int64_t zero_pieces(int64_t num_rows, int64_t nvec) { return (num_rows + 31) / 32 * chunks_of(nvec, 32); }

unsigned warps_grid(int64_t pieces) { return fz::grid_for(pieces, 8, 8, 4); }

// Resident warps go through the tokens (their registers allow 6 or 3 CTAs an SM).
template <int NE>
unsigned route_grid(int64_t tokens) {
  return fz::grid_for(tokens, 8, NE <= 8 ? 6 : 3);
}

template <int NE>
int launch_route(float *w, int32_t *ids, const float *logits, int64_t tokens, int experts, int k, int renorm,
                 cudaStream_t s) {
  FZ_CUDA(fz::launch_pdl(route_kernel<NE>, dim3(route_grid<NE>(tokens)), dim3(256), 0, s, w, ids, logits, tokens,
                         experts, k, renorm));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}
template <int L, int N, int K>
int launch_route_team(float *w, int32_t *ids, const float *logits, int64_t tokens, int experts, int k, int renorm,
                      cudaStream_t s) {
  FZ_CUDA(fz::launch_pdl(route_team_kernel<L, N, K>, dim3(fz::grid_for((tokens * L + 31) / 32, 8, 4)), dim3(256), 0, s, w,
                         ids, logits, tokens, experts, k, renorm));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}
template <int NE>
int launch_route_backward(float *dl, const float *dw, const float *w, const int32_t *ids, const float *logits,
                          int64_t tokens, int experts, int k, int renorm, cudaStream_t s) {
  FZ_CUDA(fz::launch_pdl(route_backward_kernel<NE>, dim3(route_grid<NE>(tokens)), dim3(256), 0, s, dl, dw, w, ids,
                         logits, tokens, experts, k, renorm));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

int check_route(const char *who, int64_t tokens, int64_t experts, int64_t k) {
  const std::string name(who);
  FZ_REQUIRE(tokens >= 0 && experts >= 1 && k >= 1, name + ": negative or zero size");
  FZ_REQUIRE(experts <= FZ_MAX_EXPERTS, name + ": more than FZ_MAX_EXPERTS experts");
  FZ_REQUIRE(k <= experts && k <= FZ_MAX_CHOICES, name + ": k must be at most experts and FZ_MAX_CHOICES");
  FZ_REQUIRE(tokens <= INT_MAX / k, name + ": tokens * k must be below 2^31");
  return FZ_OK;
}

}  // namespace

extern "C" int fz_route(float *weights, int32_t *ids, const float *logits, int64_t tokens, int64_t experts,
                        int64_t k, int renormalize, void *stream) {
  if (int rc = check_route("fz_route", tokens, experts, k)) return rc;
  if (tokens == 0) return FZ_OK;
  FZ_REQUIRE(weights && ids && logits, "fz_route: null pointer");
  cudaStream_t s = fz::resolve(stream);
  const int e = (int)experts, kk = (int)k, rn = renormalize != 0;
  // Up to 8 picks, the fewest lanes a token whose registers hold the experts: 262144 tokens of 64
  // experts, 26 us with 4 lanes, 36 with 8; 65536 of 256, 32 with 8, 39 with 16; 16384 of 512, 17
  // with 16, 21 with 32.
  if (k <= 4) {
    if (e <= 64) return launch_route_team<4, 16, 4>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 128) return launch_route_team<4, 32, 4>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 256) return launch_route_team<8, 32, 4>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 512) return launch_route_team<16, 32, 4>(weights, ids, logits, tokens, e, kk, rn, s);
    return launch_route_team<32, 32, 4>(weights, ids, logits, tokens, e, kk, rn, s);
  }
  if (k <= 8) {
    if (e <= 64) return launch_route_team<8, 8, 8>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 128) return launch_route_team<8, 16, 8>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 256) return launch_route_team<8, 32, 8>(weights, ids, logits, tokens, e, kk, rn, s);
    if (e <= 512) return launch_route_team<16, 32, 8>(weights, ids, logits, tokens, e, kk, rn, s);
    return launch_route_team<32, 32, 8>(weights, ids, logits, tokens, e, kk, rn, s);
  }
  if (e <= 32) return launch_route<1>(weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 64) return launch_route<2>(weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 128) return launch_route<4>(weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 256) return launch_route<8>(weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 512) return launch_route<16>(weights, ids, logits, tokens, e, kk, rn, s);
  return launch_route<32>(weights, ids, logits, tokens, e, kk, rn, s);
}

extern "C" int fz_route_backward(float *dlogits, const float *dweights, const float *weights, const int32_t *ids,
                                 const float *logits, int64_t tokens, int64_t experts, int64_t k,
                                 int renormalize, void *stream) {
  if (int rc = check_route("fz_route_backward", tokens, experts, k)) return rc;
  if (tokens == 0) return FZ_OK;
  FZ_REQUIRE(dlogits && dweights && weights && ids && logits, "fz_route_backward: null pointer");
  cudaStream_t s = fz::resolve(stream);
  const int e = (int)experts, kk = (int)k, rn = renormalize != 0;
  if (e <= 32) return launch_route_backward<1>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 64) return launch_route_backward<2>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 128) return launch_route_backward<4>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 256) return launch_route_backward<8>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
  if (e <= 512) return launch_route_backward<16>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
  return launch_route_backward<32>(dlogits, dweights, weights, ids, logits, tokens, e, kk, rn, s);
}

extern "C" int fz_expert_sort(int32_t *slot, int32_t *src, int32_t *counts, int32_t *offsets, const int32_t *ids,
                              int64_t tokens, int64_t k, int64_t experts, int64_t capacity, void *stream) {
  FZ_REQUIRE(tokens >= 0 && k >= 1 && experts >= 1 && capacity >= 0, "fz_expert_sort: negative or zero size");
  FZ_REQUIRE(experts <= FZ_MAX_EXPERTS, "fz_expert_sort: more than FZ_MAX_EXPERTS experts");
  FZ_REQUIRE(k <= INT_MAX && tokens <= INT_MAX / k && capacity <= INT_MAX / experts,
             "fz_expert_sort: tokens * k and experts * capacity must be below 2^31");
  const int64_t n = tokens * k, rows = capacity ? experts * capacity : n;
  FZ_REQUIRE(counts && offsets, "fz_expert_sort: null pointer");
  FZ_REQUIRE((n == 0 || (slot && ids)) && (rows == 0 || src), "fz_expert_sort: null pointer");
  // Few choices: one CTA of few warps (fewer histograms to scan); many: a cluster of 8 or 16.
  const int ctas = n > 131072 ? 16 : n > 8192 || rows > 65536 ? 8 : 1;
  const int threads = n > 1024 || experts > 256 || ctas > 1 ? 1024 : 256;
  const int warps = ctas * threads / 32;
  const int per_warp = (int)((n + warps - 1) / warps);
  int bits = 1;  // of numbers up to `experts`
  while ((experts >> bits) != 0) ++bits;
  const size_t smem = sizeof(int32_t) * (size_t)experts * (threads / 32 + 4);
  FZ_CUDA(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(sizeof(int32_t) * FZ_MAX_EXPERTS * (1024 / 32 + 4))));
  if (ctas > 8) FZ_CUDA(cudaFuncSetAttribute(sort_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = fz::resolve(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FZ_CUDA(cudaLaunchKernelEx(&cfg, sort_kernel, slot, src, counts, offsets, ids, (int)n, (int)experts,
                             (int)capacity, (int)rows, per_warp, bits));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

extern "C" int fz_expert_dispatch(float *rows, const float *x, const int32_t *slot, const int32_t *src,
                                  int64_t tokens, int64_t k, int64_t num_rows, int64_t width, void *stream) {
  if (int rc = check_rows("fz_expert_dispatch", tokens, k, num_rows, width)) return rc;
  if (num_rows == 0 || width == 0) return FZ_OK;
  FZ_REQUIRE(rows && src && (tokens == 0 || (x && slot)), "fz_expert_dispatch: null pointer");
  cudaStream_t s = fz::resolve(stream);
  const auto launch = [&](auto vec, int64_t nvec) {
    constexpr int kVec = decltype(vec)::value;
    using T = typename Vec<kVec>::T;
    return with_lanes(nvec, [&](auto lanes) {
      constexpr int P = decltype(lanes)::value;
      const int64_t chunks = chunks_of(nvec, P);
      const unsigned grid = warps_grid(warp_pieces(tokens, chunks, P) + zero_pieces(num_rows, nvec));
      FZ_CUDA(fz::launch_pdl(dispatch_kernel<kVec, P>, dim3(grid), dim3(256), 0, s, (T *)rows, (const T *)x, slot,
                             src, tokens, k, num_rows, nvec, chunks));
      FZ_CHECK_LAUNCH();
      return (int)FZ_OK;
    });
  };
  return width % 4 == 0 && aligned16(rows, x) ? launch(Lanes<4>{}, width / 4) : launch(Lanes<1>{}, width);
}

extern "C" int fz_expert_combine(float *out, const float *rows, const float *weights, const int32_t *slot,
                                 int64_t tokens, int64_t k, int64_t num_rows, int64_t width, void *stream) {
  if (int rc = check_rows("fz_expert_combine", tokens, k, num_rows, width)) return rc;
  if (tokens == 0 || width == 0) return FZ_OK;
  FZ_REQUIRE(out && slot && (num_rows == 0 || rows), "fz_expert_combine: null pointer");
  cudaStream_t s = fz::resolve(stream);
  const auto launch = [&](auto vec, int64_t nvec) {
    constexpr int kVec = decltype(vec)::value;
    using T = typename Vec<kVec>::T;
    return with_lanes(nvec, [&](auto lanes) {
      constexpr int P = decltype(lanes)::value;
      const int64_t chunks = chunks_of(nvec, P);
      FZ_CUDA(fz::launch_pdl(combine_kernel<kVec, P>, dim3(warps_grid(warp_pieces(tokens, chunks, P))), dim3(256), 0,
                             s, (T *)out, (const T *)rows, weights, slot, tokens, k, num_rows, nvec, chunks));
      FZ_CHECK_LAUNCH();
      return (int)FZ_OK;
    });
  };
  return width % 4 == 0 && aligned16(out, rows) ? launch(Lanes<4>{}, width / 4) : launch(Lanes<1>{}, width);
}

extern "C" int fz_expert_combine_backward(float *drows, float *dweights, const float *dout, const float *rows,
                                          const float *weights, const int32_t *slot, const int32_t *src,
                                          int64_t tokens, int64_t k, int64_t num_rows, int64_t width,
                                          void *stream) {
  if (int rc = check_rows("fz_expert_combine_backward", tokens, k, num_rows, width)) return rc;
  if (tokens == 0 && (num_rows == 0 || width == 0)) return FZ_OK;
  const bool data = num_rows > 0 && width > 0;
  FZ_REQUIRE((!data || (drows && src && (tokens == 0 || dout))) && (tokens == 0 || slot) &&
                 (!dweights || !data || tokens == 0 || rows),
             "fz_expert_combine_backward: null pointer");
  cudaStream_t s = fz::resolve(stream);
  const auto launch = [&](auto vec, int64_t nvec) {
    constexpr int kVec = decltype(vec)::value;
    using T = typename Vec<kVec>::T;
    const auto with = [&](auto lanes) {
      constexpr int P = decltype(lanes)::value;
      const unsigned grid = warps_grid(warp_pieces(tokens * k, 1, P) + zero_pieces(num_rows, nvec));
      FZ_CUDA(fz::launch_pdl(combine_backward_kernel<kVec, P>, dim3(grid), dim3(256), 0, s, (T *)drows, dweights,
                             (const T *)dout, (const T *)rows, weights, slot, src, tokens, k, num_rows, nvec));
      FZ_CHECK_LAUNCH();
      return (int)FZ_OK;
    };
    return wide_choices(tokens * k, nvec) ? with(Lanes<256>{}) : with_lanes(nvec, with);
  };
  return width % 4 == 0 && aligned16(drows, dout, rows) ? launch(Lanes<4>{}, width / 4) : launch(Lanes<1>{}, width);
}
