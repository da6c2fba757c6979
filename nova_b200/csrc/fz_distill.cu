// Distillation from a teacher's top logits: the loss and its gradient.
//
// Bound by memory: the forward reads the student's logits once (4 bytes a value), the
// backward reads them once more and writes dz (8 bytes). Per row, a thread keeps a running
// maximum m and sum of exp((z - m) / tau), 16 values at a time; the sums are joined over
// the row's team: a warp for small vocabularies, a CTA of 128 or 512 threads for larger
// ones, a cluster of CTAs where few rows would leave SMs idle (team_of). With the tail
// bucket the row's entries are marked in a bitmap in shared memory and go to a sum of their
// own, so that the tail's mass qT is summed directly (1 - sum of q inside would cancel where
// the student is sure of itself), and an id named twice counts once. The maximum and the
// log of the sum are kept apart: a large common offset of the logits, or a row of the type's
// lowest value, costs no digits.
// The backward streams the row once more, writing dz from the saved statistics, and then
// overwrites the entries' columns.
// Measured (B200, copy bandwidth 6.55 TB/s), 64 entries a row: 4096 rows of 131072, forward
// 324 us (1.01 of the copy bandwidth), backward 662 us (0.99); 2048 rows of 50001 (no two
// alike aligned) 80 and 141 us (0.78, 0.89: the last wave of CTAs and their fixed cost); 8192
// rows of 2000, a warp each, 25 and 37 us.
#include <cooperative_groups.h>

#include <climits>
#include <cstdint>

#include "fz_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr float kLog2e = 1.4426950408889634f;

// 2^x to within 2 ulp (results below the normal range flush to 0, next to sums that are
// at least 1).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A running sum s of exp((z - m) / tau), a = log2(e) / tau. m = -inf: empty so far.
struct Lse {
  float m, s;
};
__device__ __forceinline__ float floor_of(float m) { return m == -INFINITY ? 0.0f : m; }
// 2^(a (z - m))
__device__ __forceinline__ float term(float z, float m, float a) { return ex2(__fmul_rn(__fsub_rn(z, m), a)); }
__device__ __forceinline__ Lse join(Lse p, Lse q, float a) {
  const float m = fmaxf(p.m, q.m), at = floor_of(m);
  return {m, __fmaf_rn(p.s, term(p.m, at, a), __fmul_rn(q.s, term(q.m, at, a)))};
}
__device__ __forceinline__ Lse warp_join(Lse p, float a) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
    const Lse q{__shfl_xor_sync(kFull, p.m, d), __shfl_xor_sync(kFull, p.s, d)};
    p = join(p, q, a);
  }
  return p;
}
// NaN and +inf logits make the sum NaN.
template <int N>
__device__ __forceinline__ void take(Lse &p, const float (&x)[N], float a) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > p.m) {
    p.s = __fmul_rn(p.s, term(p.m, top, a));
    p.m = top;
  }
  const float at = floor_of(p.m);
  float s = term(x[0], at, a);
#pragma unroll
  for (int i = 1; i < N; ++i) s = __fadd_rn(s, term(x[i], at, a));
  p.s = __fadd_rn(p.s, s);
}

// ---------------------------------------------------------------- teams
// T threads work on a row: 32 (eight rows a CTA) or a whole CTA.
__host__ __device__ constexpr int threads_of(int t) { return t == 32 ? 256 : t; }

template <int T>
__device__ __forceinline__ int team_thread() {
  return T == 32 ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
}
template <int T>
__device__ __forceinline__ void team_sync() {
  if constexpr (T == 32) __syncwarp();
  else __syncthreads();
}
template <int T>
__device__ __forceinline__ bool team_any(bool v) {
  if constexpr (T == 32) return __any_sync(kFull, v);
  else return __syncthreads_or(v);
}
template <int T, bool MAX>
__device__ __forceinline__ float team_fold(float v, float *sh) {
  const auto fold = [](float a, float b) { return MAX ? fmaxf(a, b) : __fadd_rn(a, b); };
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fold(v, __shfl_xor_sync(kFull, v, d));
  if constexpr (T > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < T / 32; ++w) v = fold(v, sh[w]);
  }
  return v;
}

// ---------------------------------------------------------------- the teacher's side of a row

struct Teacher {
  bool some;           // the row has entries
  float listed, tail;  // sum p, pT
  float slack;         // what rounding alone may leave in pT
  __device__ __forceinline__ float mass() const { return __fadd_rn(listed, tail); }
  // Where the student gives the columns outside the entries no mass that fp32 holds (there are
  // none, or all are masked), pT (log pT - log qT) would turn a rounding of pT into an infinite
  // loss: a pT that is no larger than its rounding is 0 there.
  __device__ __forceinline__ void settle(float log_q_tail) {
    if (log_q_tail < -87.336545f && tail <= slack) tail = 0.0f;  // log 2^-126
  }
};
// log qT from the maximum and log sum of all logits and of those outside the entries
__device__ __forceinline__ float log_tail_mass(float m, float log_sum, float tail_m, float log_tail, float tau) {
  return __fadd_rn(__fdiv_rn(__fsub_rn(tail_m, m), tau), __fsub_rn(log_tail, log_sum));
}

// Made by the whole team in shared memory: id[i] (-1: padding), p[i], the student's logit
// z[i] there and, when asked for, logp[i] = log p[i].
template <int T>
__device__ __forceinline__ Teacher read_teacher(int *id, float *p, float *z, float *logp, const float *row,
                                                const int32_t *ids, const float *teacher, const float *lse,
                                                int64_t r, int k, int vocab, float tau, float *sh) {
  const int tid = team_thread<T>();
  bool some = false;
  float top = -INFINITY;
  for (int i = tid; i < k; i += T) {
    const int v = ids[r * k + i];
    const bool ok = v >= 0 && v < vocab;
    const float t = ok ? teacher[r * k + i] : -INFINITY;
    id[i] = ok ? v : -1;
    p[i] = t;
    if (z) z[i] = ok ? row[v] : 0.0f;
    some = some || (ok && (lse || t != -INFINITY));
    top = fmaxf(top, t);
  }
  Teacher t{team_any<T>(some), 0.0f, 0.0f, 0.0f};
  if (!t.some) return t;
  float shift;
  if (!lse) {
    top = team_fold<T, true>(top, sh);
    float s = 0.0f;
    for (int i = tid; i < k; i += T)
      if (id[i] >= 0) s = __fadd_rn(s, expf(__fdiv_rn(__fsub_rn(p[i], top), tau)));
    shift = logf(team_fold<T, false>(s, sh));
  } else {
    top = 0.0f;
    shift = lse[r];
  }
  float s = 0.0f;
  for (int i = tid; i < k; i += T) {
    const float l = __fsub_rn(__fdiv_rn(__fsub_rn(p[i], top), tau), shift);
    const float q = id[i] >= 0 ? expf(l) : 0.0f;
    if (logp) logp[i] = l;
    p[i] = q;
    s = __fadd_rn(s, q);
  }
  t.listed = team_fold<T, false>(s, sh);
  if (lse) {
    const float rest = __fsub_rn(1.0f, t.listed);
    t.tail = rest < 0.0f ? 0.0f : rest;  // NaN stays
    // To first order, with u = 2^-24 and L = |lse|: the sum of p, at most 24 additions deep
    // (k <= 1024), 24 u; expf 4 u; p's argument, t / tau and the difference rounded, (L + 2 H) u
    // with the entries' entropy H <= log 1024; the caller's lse, 2 roundings of it and as much
    // again of its sum, (3 L + 6) u.
    t.slack = __fmul_rn(__fmaf_rn(fabsf(shift), 4.0f, 48.0f), 1.0f / (1 << 24));
  }
  return t;
}

// Columns of a row are counted from `shift` before its start, so that 16-byte accesses to an
// unaligned row begin at multiples of 4: column c of the row lies at c + shift.
struct Row {
  const float *aligned;  // 16-byte aligned; the row's first value is aligned[shift]
  int shift, end;        // end = vocab + shift
};
__device__ __forceinline__ Row row_at(const float *row, int vocab) {
  const int shift = (int)(((uintptr_t)row >> 2) & 3);
  return {row - shift, shift, vocab + shift};
}
__device__ __forceinline__ bool inside(const Row &r, int c) { return c >= r.shift && c + 4 <= r.end; }
__device__ __forceinline__ void load4(float *x, const Row &r, int c) {
  if (inside(r, c)) {
    const float4 q = *reinterpret_cast<const float4 *>(r.aligned + c);
    x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = c + i >= r.shift && c + i < r.end ? r.aligned[c + i] : -INFINITY;
  }
}
constexpr int kUnroll = 4;  // float4s a thread has in flight

template <bool TAIL, int T>
__global__ void __launch_bounds__(threads_of(T)) distill_kernel(float *__restrict__ loss, float *__restrict__ stats,
                                                                const float *__restrict__ logits, int64_t ld,
                                                                const int32_t *__restrict__ ids,
                                                                const float *__restrict__ teacher,
                                                                const float *__restrict__ teacher_lse, int64_t rows,
                                                                int vocab, int k, float tau, int slice) {
  pdl_wait();
  constexpr int kTeams = threads_of(T) / T, kWarps = T / 32;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = T == 512 ? (int)cluster.block_rank() : 0, ctas = T == 512 ? (int)cluster.num_blocks() : 1;
  const int team = T == 32 ? (int)threadIdx.x / 32 : 0, tid = team_thread<T>(), lane = tid & 31, warp = tid >> 5;
  const int64_t r = (int64_t)(blockIdx.x / ctas) * kTeams + team;
  extern __shared__ float dyn[];
  const int words = TAIL ? slice / 32 : 0;
  int *id = reinterpret_cast<int *>(dyn) + team * (4 * k + words);
  float *p = reinterpret_cast<float *>(id + k), *logp = p + k, *z = logp + k;
  uint32_t *marks = reinterpret_cast<uint32_t *>(z + k);
  __shared__ float sh[kWarps];
  __shared__ Lse part[2][kWarps];
  __shared__ Lse whole[2];  // outside the entries (without TAIL: all), inside
  if (T == 32 && r >= rows) return;

  const float a = __fdiv_rn(kLog2e, tau);
  const float *start = logits + r * ld;
  const Row row = row_at(start, vocab);
  const int from = rank * slice, to = min(from + slice, row.end);  // slice: a multiple of 128
  Teacher t = read_teacher<T>(id, p, rank == 0 ? z : nullptr, logp, start, ids, teacher, teacher_lse, r, k,
                                    vocab, tau, sh);
  if (!t.some) {  // the same in every CTA of the cluster
    if (rank == 0 && tid == 0) loss[r] = 0.0f;
    if (rank == 0 && tid < 4) stats[r * 4 + tid] = 0.0f;
    return;
  }
  if (TAIL) {
    for (int i = tid; i < words; i += T) marks[i] = 0u;
    team_sync<T>();
    for (int i = tid; i < k; i += T) {
      const int at = id[i] + row.shift;
      if (id[i] >= 0 && at >= from && at < to) atomicOr(&marks[(at - from) >> 5], 1u << (at & 31));
    }
    team_sync<T>();
  }

  Lse out{-INFINITY, 0.0f}, in{-INFINITY, 0.0f};
  for (int c = from + 4 * tid; c < to; c += kUnroll * 4 * T) {
    float x[kUnroll * 4];
    const int last = c + (kUnroll - 1) * 4 * T;
    if (inside(row, c) && last < to && inside(row, last)) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const float4 q = *reinterpret_cast<const float4 *>(row.aligned + c + u * 4 * T);
        x[u * 4] = q.x, x[u * 4 + 1] = q.y, x[u * 4 + 2] = q.z, x[u * 4 + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        if (c + u * 4 * T < to) {
          load4(x + u * 4, row, c + u * 4 * T);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[u * 4 + i] = -INFINITY;
        }
      }
    }
    if (TAIL) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int at = c + u * 4 * T;
        const uint32_t m = at < to ? marks[(at - from) >> 5] >> (at & 31) & 15u : 0u;
        if (m) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (m >> i & 1) {
              const float y[1] = {x[u * 4 + i]};
              take(in, y, a);
              x[u * 4 + i] = -INFINITY;
            }
        }
      }
    }
    take(out, x, a);
  }
  out = warp_join(out, a);
  if (TAIL) in = warp_join(in, a);
  if constexpr (T > 32) {
    if (lane == 0) {
      part[0][warp] = out;
      part[1][warp] = in;
    }
    __syncthreads();
    if (warp < (TAIL ? 2 : 1)) {
      const Lse mine = warp_join(lane < kWarps ? part[warp][lane] : Lse{-INFINITY, 0.0f}, a);
      if (lane == 0) whole[warp] = mine;
    }
    if (ctas > 1) cluster.sync();
    else __syncthreads();
  }
  if (rank == 0 && warp == 0) {
    Lse sum = out, tail = out;
    if constexpr (T > 32) {
      sum = tail = whole[0];
      if (TAIL) in = whole[1];
      for (int q = 1; q < ctas; ++q) {
        const Lse *theirs = cluster.map_shared_rank(whole, q);
        sum = tail = join(sum, theirs[0], a);
        if (TAIL) in = join(in, theirs[1], a);
      }
    }
    if (TAIL) sum = join(in, tail, a);
    const float log_sum = logf(sum.s);
    float l = 0.0f;
    for (int i = lane; i < k; i += 32) {
      const float w = p[i];
      if (id[i] < 0 || w == 0.0f) continue;
      const float logq = __fsub_rn(__fdiv_rn(__fsub_rn(z[i], sum.m), tau), log_sum);
      l = __fmaf_rn(w, __fsub_rn(logp[i], logq), l);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l = __fadd_rn(l, __shfl_xor_sync(kFull, l, d));
    if (lane == 0) {
      const float log_tail = logf(tail.s);
      if (TAIL) {
        const float logq = log_tail_mass(sum.m, log_sum, tail.m, log_tail, tau);
        t.settle(logq);
        if (t.tail != 0.0f) l = __fmaf_rn(t.tail, __fsub_rn(logf(t.tail), logq), l);
      }
      loss[r] = __fmul_rn(__fmul_rn(tau, tau), l);
      *reinterpret_cast<float4 *>(stats + r * 4) = make_float4(sum.m, log_sum, tail.m, log_tail);
    }
  }
  if (T > 32 && ctas > 1) cluster.sync();  // no CTA leaves while its sums may be read
}

// dz from z and the row's statistics, without its entries.
struct Slope {
  float a, m, l2, inside, tm, t2, outside;
  template <bool TAIL>
  __device__ __forceinline__ float at(float z) const {
    float d = __fmul_rn(inside, ex2(__fmaf_rn(__fsub_rn(z, m), a, -l2)));
    if (TAIL) d = __fmaf_rn(-outside, ex2(__fmaf_rn(__fsub_rn(z, tm), a, -t2)), d);
    return d;
  }
};

template <bool TAIL, bool VEC, int T>
__device__ __forceinline__ void stream_slope(float *out, const Row &row, const Slope &s, int from, int to, int tid) {
  if constexpr (VEC) {  // out and the row are equally far from 16-byte alignment
    float *aligned = out - row.shift;
    for (int c = from + 4 * tid; c < to; c += kUnroll * 4 * T) {
      float x[kUnroll * 4];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (c + u * 4 * T < to) load4(x + u * 4, row, c + u * 4 * T);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int at = c + u * 4 * T;
        if (at >= to) break;
        float d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) d[i] = s.at<TAIL>(x[u * 4 + i]);
        if (inside(row, at)) {
          *reinterpret_cast<float4 *>(aligned + at) = make_float4(d[0], d[1], d[2], d[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (at + i >= row.shift && at + i < row.end) aligned[at + i] = d[i];
        }
      }
    }
  } else {
    const int first = max(from, row.shift);
    for (int c = first + tid; c < to; c += T) out[c - row.shift] = s.at<TAIL>(row.aligned[c]);
  }
}

// The ids that are named, and which of them twice: a hash table of `size` (a power of two, at
// least 2 k) slots.
constexpr int kTwice = 1 << 30;  // ids are below 2^23
__device__ __forceinline__ int hash(int id, int size) { return (int)((uint32_t)id * 2654435761u >> 16) & (size - 1); }
template <int T>
__device__ __forceinline__ void name_ids(const int *id, int *table, int k, int size, int tid) {
  for (int i = tid; i < size; i += T) table[i] = -1;
  team_sync<T>();
  for (int i = tid; i < k; i += T) {
    const int v = id[i];
    if (v < 0) continue;
    for (int at = hash(v, size);; at = (at + 1) & (size - 1)) {
      const int was = atomicCAS(&table[at], -1, v);
      if (was == -1) break;
      if ((was & (kTwice - 1)) == v) {
        atomicOr(&table[at], kTwice);
        break;
      }
    }
  }
  team_sync<T>();
}
__device__ __forceinline__ bool named_twice(const int *table, int size, int id) {
  int at = hash(id, size);
  while ((table[at] & (kTwice - 1)) != id) at = (at + 1) & (size - 1);
  return table[at] & kTwice;
}

template <bool TAIL, int T>
__global__ void __launch_bounds__(threads_of(T)) distill_backward_kernel(
    float *__restrict__ dlogits, int64_t ldd, const float *__restrict__ dloss, const float *__restrict__ stats,
    const float *__restrict__ logits, int64_t ld, const int32_t *__restrict__ ids,
    const float *__restrict__ teacher, const float *__restrict__ teacher_lse, int64_t rows, int vocab, int k,
    float tau, int slice, int ctas, int table_size) {
  pdl_wait();
  constexpr int kTeams = threads_of(T) / T;
  const int team = T == 32 ? (int)threadIdx.x / 32 : 0, tid = team_thread<T>();
  const int64_t r = (int64_t)(blockIdx.x / ctas) * kTeams + team;
  const int rank = (int)(blockIdx.x % ctas);
  extern __shared__ float dyn[];
  int *id = reinterpret_cast<int *>(dyn) + team * (3 * k + table_size);
  float *p = reinterpret_cast<float *>(id + k), *z = p + k;
  int *table = reinterpret_cast<int *>(z + k);
  __shared__ float sh[T / 32];
  if (T == 32 && r >= rows) return;
  const float *start = logits + r * ld;
  float *out = dlogits + r * ldd;
  const Row row = row_at(start, vocab);
  const int from = rank * slice, to = min(from + slice, row.end);  // slice: a multiple of 128
  Teacher t =
      read_teacher<T>(id, p, z, nullptr, start, ids, teacher, teacher_lse, r, k, vocab, tau, sh);
  if (!t.some) {
    for (int c = max(from, row.shift) + tid; c < to; c += T) out[c - row.shift] = 0.0f;
    return;
  }
  const float scale = __fmul_rn(tau, dloss[r]);
  const float4 st = *reinterpret_cast<const float4 *>(stats + r * 4);
  if (TAIL) t.settle(log_tail_mass(st.x, st.y, st.z, st.w, tau));
  const Slope s{__fdiv_rn(kLog2e, tau),        st.x, __fmul_rn(st.y, kLog2e), __fmul_rn(scale, t.mass()), st.z,
                __fmul_rn(st.w, kLog2e), __fmul_rn(scale, t.tail)};
  const bool vec = (((uintptr_t)out >> 2) & 3) == (uintptr_t)row.shift;
  // (outside maximum -inf: every column outside is masked, and 0 - 0)
  const bool tail = TAIL && t.tail != 0.0f && st.z != -INFINITY;
  if (vec && tail) stream_slope<true, true, T>(out, row, s, from, to, tid);
  else if (vec) stream_slope<false, true, T>(out, row, s, from, to, tid);
  else if (tail) stream_slope<true, false, T>(out, row, s, from, to, tid);
  else stream_slope<false, false, T>(out, row, s, from, to, tid);
  name_ids<T>(id, table, k, table_size, tid);  // a barrier, too
  // the entries' columns, each by its first entry; the entries of an id that is named twice
  // are looked for by a warp (300 rows of 1000 entries, a few named twice: 450 us with a thread
  // for each and no account of which ids were, 38 so)
  const int lane = tid & 31;
  for (int i0 = tid - lane; i0 < k; i0 += T) {
    const int i = i0 + lane, c = i < k ? id[i] : -1, at = c + row.shift;
    bool mine = c >= 0 && at >= from && at < to;
    float sum = mine ? p[i] : 0.0f;
    for (unsigned todo = __ballot_sync(kFull, mine && named_twice(table, table_size, c)); todo; todo &= todo - 1) {
      const int who = __ffs(todo) - 1, v = __shfl_sync(kFull, c, who);
      bool before = false;
      float all = 0.0f;
      for (int j = lane; j < k; j += 32)
        if (id[j] == v) {
          before = before || j < i0 + who;
          all = __fadd_rn(all, p[j]);
        }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) all = __fadd_rn(all, __shfl_xor_sync(kFull, all, d));
      before = __any_sync(kFull, before);
      if (lane == who) {
        sum = all;
        mine = !before;
      }
    }
    if (mine) out[c] = __fsub_rn(s.at<false>(z[i]), __fmul_rn(scale, sum));
  }
}

int check_distill(const char *who, int64_t rows, int64_t vocab, int64_t k, int64_t ld, float temperature) {
  const std::string name(who);
  FZ_REQUIRE(rows >= 0 && vocab >= 1 && k >= 1, name + ": negative or zero size");
  FZ_REQUIRE(vocab <= (1 << 23), name + ": vocab above 2^23");
  FZ_REQUIRE(k <= FZ_MAX_TEACHER, name + ": more than FZ_MAX_TEACHER entries");
  FZ_REQUIRE(ld >= vocab, name + ": row pitch below vocab");
  FZ_REQUIRE(rows <= INT_MAX / 8, name + ": too many rows");
  // (its square, the loss's factor, has to be a normal number)
  FZ_REQUIRE(temperature >= 1e-18f && temperature <= 1e18f, name + ": temperature must be in [1e-18, 1e18]");
  return FZ_OK;
}

// Threads and CTAs a row (times with 64 entries).
// A warp a row where that gives every SM more than 8 CTAs' worth of rows: 4096 rows of 2000,
// 14 and 23 us forward and backward against 22 and 28 with 128 threads and 56 and 61 with 512;
// 100 rows of 4096, 9 and 13 against 5 and 7. 128 threads where rows are short, or of medium
// length and more than 3 an SM: 1024 of 16384, 18 and 29 us against 26 and 31 with 512; 148,
// 12 and 14 against 7 and 9. Else 512.
// More than one CTA (in the forward a cluster, whose barriers and repeated reading of the
// entries cost more than the last wave's idle SMs once there are two CTAs an SM): while no more
// than two an SM result; 8 rows of 131072, 7.9 us forward with 8 against 15.0 with one, 464
// rows, 101 against 55. The backward's CTAs know nothing of one another, so it also splits
// many rows into pieces of 40000 columns and more, which shortens the last wave. 4096 rows, alone
// and with the forward before it (of which L2 then holds the last rows), us with 1, 2, 4 and 8 CTAs:
// 50000 columns, 268 282 349 499 and 424 439 506 658; 80000, 421 403 462 622 and 636 620 680 853;
// 131072, 685 663 671 843 and 1016 992 1012 1177; 165000, 883 855 832 979 and 1297 1267 1254 1401;
// 1500 rows of 320000, 625 610 596 580 and 922 905 891 878. (Fewer rows in between differ by 2 %.)
struct Team {
  int threads, ctas, slice;
};
Team team_of(int64_t rows, int64_t vocab, int64_t k, bool backward) {
  const int64_t sms = fz::num_sms();
  Team t{512, 1, 0};
  if (vocab <= 4096) t.threads = k <= 256 && rows > 8 * sms ? 32 : 128;
  else if (vocab <= 16384 && rows > 3 * sms) t.threads = 128;
  if (t.threads == 512) {
    const int64_t least = backward ? 4096 : 8192;  // columns a CTA
    while (t.ctas < 8 && ((rows * t.ctas * 2 <= 2 * sms && vocab >= least * t.ctas * 2) ||
                          (backward && rows > 2 * sms && vocab >= 40000 * (int64_t)t.ctas * 2) ||
                          vocab > ((int64_t)t.ctas << 20)))  // a slice's marks have to fit in shared memory
      t.ctas *= 2;
  }
  t.slice = (int)(((vocab + 3 + t.ctas - 1) / t.ctas + 127) / 128 * 128);
  return t;
}

template <typename... KArgs, typename... Args>
int launch_team(void (*kernel)(KArgs...), int64_t rows, const Team &t, size_t smem, bool cluster, cudaStream_t s,
                Args... args) {
  if (smem > 32 * 1024)
    FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(t.threads == 32 ? (rows + 7) / 8 : rows * t.ctas));
  cfg.blockDim = dim3((unsigned)threads_of(t.threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster ? (unsigned)t.ctas : 1u;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FZ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

}  // namespace

extern "C" int fz_distill(float *loss, float *stats, const float *logits, int64_t ld, const int32_t *ids,
                          const float *teacher, const float *teacher_lse, int64_t rows, int64_t vocab, int64_t k,
                          float temperature, void *stream) {
  if (int rc = check_distill("fz_distill", rows, vocab, k, ld, temperature)) return rc;
  if (rows == 0) return FZ_OK;
  FZ_REQUIRE(loss && stats && logits && ids && teacher, "fz_distill: null pointer");
  FZ_REQUIRE(((uintptr_t)stats & 15) == 0, "fz_distill: stats must be 16-byte aligned");
  const Team t = team_of(rows, vocab, k, false);
  const size_t smem = ((size_t)k * 16 + (teacher_lse ? (size_t)t.slice / 8 : 0)) * (t.threads == 32 ? 8 : 1);
  const auto kernel = teacher_lse ? (t.threads == 32    ? distill_kernel<true, 32>
                                     : t.threads == 128 ? distill_kernel<true, 128>
                                                        : distill_kernel<true, 512>)
                                  : (t.threads == 32    ? distill_kernel<false, 32>
                                     : t.threads == 128 ? distill_kernel<false, 128>
                                                        : distill_kernel<false, 512>);
  return launch_team(kernel, rows, t, smem, true, fz::resolve(stream), loss, stats, logits, ld, ids, teacher,
                     teacher_lse, rows, (int)vocab, (int)k, temperature, t.slice);
}

extern "C" int fz_distill_backward(float *dlogits, int64_t ldd, const float *dloss, const float *stats,
                                   const float *logits, int64_t ld, const int32_t *ids, const float *teacher,
                                   const float *teacher_lse, int64_t rows, int64_t vocab, int64_t k,
                                   float temperature, void *stream) {
  if (int rc = check_distill("fz_distill_backward", rows, vocab, k, ld, temperature)) return rc;
  FZ_REQUIRE(ldd >= vocab, "fz_distill_backward: row pitch below vocab");
  if (rows == 0) return FZ_OK;
  FZ_REQUIRE(dlogits && dloss && stats && logits && ids && teacher, "fz_distill_backward: null pointer");
  FZ_REQUIRE(((uintptr_t)stats & 15) == 0, "fz_distill_backward: stats must be 16-byte aligned");
  FZ_REQUIRE(dlogits != logits, "fz_distill_backward: dlogits may not overlap logits");
  const Team t = team_of(rows, vocab, k, true);
  int table = 2;
  while (table < 2 * k) table *= 2;
  const size_t smem = ((size_t)k * 12 + (size_t)table * 4) * (t.threads == 32 ? 8 : 1);
  const auto kernel = teacher_lse ? (t.threads == 32    ? distill_backward_kernel<true, 32>
                                     : t.threads == 128 ? distill_backward_kernel<true, 128>
                                                        : distill_backward_kernel<true, 512>)
                                  : (t.threads == 32    ? distill_backward_kernel<false, 32>
                                     : t.threads == 128 ? distill_backward_kernel<false, 128>
                                                        : distill_backward_kernel<false, 512>);
  return launch_team(kernel, rows, t, smem, false, fz::resolve(stream), dlogits, ldd, dloss, stats, logits, ld, ids,
                     teacher, teacher_lse, rows, (int)vocab, (int)k, temperature, t.slice, t.ctas, table);
}
