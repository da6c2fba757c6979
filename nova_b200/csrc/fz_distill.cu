// Distillation from a teacher's top logits: the loss and its gradient.
//
// Per row, one pass over the student's logits keeps a running maximum m and sum of
// exp((z - m) / tau) per thread, joined over the CTA and, where few rows would leave SMs
// idle, over a cluster of CTAs that share the row. With the tail bucket the row's entries
// are marked in a bitmap in shared memory and go to a sum of their own, so that the tail's
// mass qT is summed directly (1 - sum of q inside would cancel where the student is sure
// of itself), and an id named twice counts once. The maximum and the log of the sum are
// kept apart: a large common offset of the logits, or a row of the type's lowest value,
// costs no digits.
// The backward streams the row once more, writing dz from the saved statistics, and then
// overwrites the entries' columns.
#include <cooperative_groups.h>

#include <climits>
#include <cstdint>

#include "fz_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512;
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
    const Lse q{__shfl_xor_sync(0xffffffffu, p.m, d), __shfl_xor_sync(0xffffffffu, p.s, d)};
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
#pragma unroll
  for (int i = 0; i < N; ++i) p.s = __fadd_rn(p.s, term(x[i], at, a));
}

// The teacher's side of one row.
struct Teacher {
  int count;         // nonzero if the row has entries
  float mass, tail;  // P = sum p + pT, pT
};

__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) s = __fadd_rn(s, sh[w]);
  return s;
}
__device__ __forceinline__ float block_max(float v, float *sh) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = -INFINITY;
  for (int w = 0; w < kThreads / 32; ++w) s = fmaxf(s, sh[w]);
  return s;
}

// Made by the whole CTA in shared memory: id[i] (-1: padding), p[i] and, when asked for,
// logp[i] = log p[i].
__device__ Teacher read_teacher(int *id, float *p, float *logp, const int32_t *ids, const float *teacher,
                                const float *lse, int64_t r, int k, int vocab, float tau, float *sh) {
  int n = 0;
  float top = -INFINITY;
  for (int i = threadIdx.x; i < k; i += kThreads) {
    const int v = ids[r * k + i];
    const bool ok = v >= 0 && v < vocab;
    const float t = ok ? teacher[r * k + i] : -INFINITY;
    id[i] = ok ? v : -1;
    p[i] = t;
    n += ok && (lse || t != -INFINITY);
    top = fmaxf(top, t);
  }
  Teacher T{__syncthreads_or(n), 0.0f, 0.0f};
  if (!T.count) return T;
  float shift = 0.0f;
  if (!lse) {
    top = block_max(top, sh);
    float s = 0.0f;
    for (int i = threadIdx.x; i < k; i += kThreads)
      if (id[i] >= 0) s = __fadd_rn(s, expf(__fdiv_rn(__fsub_rn(p[i], top), tau)));
    shift = logf(block_sum(s, sh));
  } else {
    top = 0.0f;
    shift = lse[r];
  }
  float s = 0.0f;
  for (int i = threadIdx.x; i < k; i += kThreads) {
    const float l = __fsub_rn(__fdiv_rn(__fsub_rn(p[i], top), tau), shift);
    const float q = id[i] >= 0 ? expf(l) : 0.0f;
    if (logp) logp[i] = l;
    p[i] = q;
    s = __fadd_rn(s, q);
  }
  s = block_sum(s, sh);
  if (lse) {
    const float rest = __fsub_rn(1.0f, s);
    T.tail = rest < 0.0f ? 0.0f : rest;  // NaN stays
  }
  T.mass = __fadd_rn(s, T.tail);
  return T;
}

// One cluster of CTAs per row; each takes a slice of the columns. Columns are counted
// from `shift` before the row's start, so that the float4s of an unaligned row begin at
// multiples of 4.
template <bool TAIL>
__global__ void __launch_bounds__(kThreads) distill_kernel(float *__restrict__ loss, float *__restrict__ stats,
                                                           const float *__restrict__ logits, int64_t ld,
                                                           const int32_t *__restrict__ ids,
                                                           const float *__restrict__ teacher,
                                                           const float *__restrict__ teacher_lse, int vocab, int k,
                                                           float tau, int slice) {
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  const int64_t r = blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  extern __shared__ float dyn[];
  int *id = reinterpret_cast<int *>(dyn);
  float *p = dyn + k, *logp = dyn + 2 * k;
  uint32_t *marks = reinterpret_cast<uint32_t *>(dyn + 3 * k);
  __shared__ float sh[kThreads / 32];
  __shared__ Lse part[2][kThreads / 32];
  __shared__ Lse whole[2];  // outside the entries (without TAIL: all), inside

  const float a = __fdiv_rn(kLog2e, tau);
  const float *row = logits + r * ld;
  const int shift = (int)(((uintptr_t)row >> 2) & 3);
  const int from = rank * slice, to = min(from + slice, vocab + shift);  // slice: a multiple of 128
  const Teacher T = read_teacher(id, p, logp, ids, teacher, teacher_lse, r, k, vocab, tau, sh);
  if (!T.count) {  // the same in every CTA of the cluster
    if (rank == 0 && tid == 0) loss[r] = 0.0f;
    if (rank == 0 && tid < 4) stats[r * 4 + tid] = 0.0f;
    return;
  }
  if (TAIL) {
    for (int i = tid; i < slice / 32; i += kThreads) marks[i] = 0u;
    __syncthreads();
    for (int i = tid; i < k; i += kThreads) {
      const int at = id[i] + shift;
      if (id[i] >= 0 && at >= from && at < to) atomicOr(&marks[(at - from) >> 5], 1u << (at & 31));
    }
    __syncthreads();
  }

  Lse out{-INFINITY, 0.0f}, in{-INFINITY, 0.0f};
  const float *aligned = row - shift;
  for (int c = from + 4 * tid; c < to; c += 4 * kThreads) {
    float x[4];
    if (c >= shift && c + 4 <= vocab + shift) {
      const float4 q = *reinterpret_cast<const float4 *>(aligned + c);
      x[0] = q.x, x[1] = q.y, x[2] = q.z, x[3] = q.w;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = c + i >= shift && c + i < vocab + shift ? aligned[c + i] : -INFINITY;
    }
    if (TAIL) {
      const uint32_t m = marks[(c - from) >> 5] >> (c & 31) & 15u;
      if (m) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (m >> i & 1) {
            const float y[1] = {x[i]};
            take(in, y, a);
            x[i] = -INFINITY;
          }
      }
    }
    take(out, x, a);
  }
  out = warp_join(out, a);
  if (TAIL) in = warp_join(in, a);
  if (lane == 0) {
    part[0][warp] = out;
    part[1][warp] = in;
  }
  __syncthreads();
  if (warp < (TAIL ? 2 : 1)) {
    const Lse mine = warp_join(lane < kThreads / 32 ? part[warp][lane] : Lse{-INFINITY, 0.0f}, a);
    if (lane == 0) whole[warp] = mine;
  }
  cluster.sync();
  if (rank == 0 && warp == 0) {
    Lse sum{-INFINITY, 0.0f}, tail{-INFINITY, 0.0f};
    for (int q = 0; q < ctas; ++q) {
      const Lse *theirs = cluster.map_shared_rank(whole, q);
      if (TAIL) {
        tail = join(tail, theirs[0], a);
        sum = join(sum, theirs[1], a);
      } else {
        sum = join(sum, theirs[0], a);
      }
    }
    if (TAIL) sum = join(sum, tail, a);
    const float log_sum = logf(sum.s);
    float l = 0.0f;
    for (int i = lane; i < k; i += 32) {
      const float w = p[i];
      if (id[i] < 0 || w == 0.0f) continue;
      const float logq = __fsub_rn(__fdiv_rn(__fsub_rn(row[id[i]], sum.m), tau), log_sum);
      l = __fmaf_rn(w, __fsub_rn(logp[i], logq), l);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l = __fadd_rn(l, __shfl_xor_sync(0xffffffffu, l, d));
    if (lane == 0) {
      const float log_tail = logf(tail.s);
      if (TAIL && T.tail != 0.0f) {
        const float logq =
            __fadd_rn(__fdiv_rn(__fsub_rn(tail.m, sum.m), tau), __fsub_rn(log_tail, log_sum));
        l = __fmaf_rn(T.tail, __fsub_rn(logf(T.tail), logq), l);
      }
      loss[r] = __fmul_rn(__fmul_rn(tau, tau), l);
      stats[r * 4] = sum.m;
      stats[r * 4 + 1] = log_sum;
      stats[r * 4 + 2] = tail.m;
      stats[r * 4 + 3] = log_tail;
    }
  }
  cluster.sync();  // no CTA leaves while its sums may be read
}

template <bool TAIL>
__global__ void __launch_bounds__(kThreads) distill_backward_kernel(
    float *__restrict__ dlogits, int64_t ldd, const float *__restrict__ dloss, const float *__restrict__ stats,
    const float *__restrict__ logits, int64_t ld, const int32_t *__restrict__ ids,
    const float *__restrict__ teacher, const float *__restrict__ teacher_lse, int vocab, int k, float tau, int slice, int ctas) {
  pdl_wait();
  const int64_t r = blockIdx.x / ctas;
  const int rank = (int)(blockIdx.x - r * ctas), tid = threadIdx.x;
  extern __shared__ float dyn[];
  int *id = reinterpret_cast<int *>(dyn);
  float *p = dyn + k;
  __shared__ float sh[kThreads / 32];
  const Teacher T = read_teacher(id, p, nullptr, ids, teacher, teacher_lse, r, k, vocab, tau, sh);
  const float *row = logits + r * ld;
  float *out = dlogits + r * ldd;
  const int from = rank * slice, to = min(from + slice, vocab);
  if (!T.count) {
    for (int c = from + tid; c < to; c += kThreads) out[c] = 0.0f;
    return;
  }
  const float a = __fdiv_rn(kLog2e, tau), scale = __fmul_rn(tau, dloss[r]);
  const float m = stats[r * 4], l2 = __fmul_rn(stats[r * 4 + 1], kLog2e), inside = __fmul_rn(scale, T.mass);
  const float tm = stats[r * 4 + 2], t2 = __fmul_rn(stats[r * 4 + 3], kLog2e), outside = __fmul_rn(scale, T.tail);
  for (int c = from + tid; c < to; c += kThreads) {
    const float x = row[c];
    float d = __fmul_rn(inside, ex2(__fmaf_rn(__fsub_rn(x, m), a, -l2)));
    if (TAIL && T.tail != 0.0f) d = __fmaf_rn(-outside, ex2(__fmaf_rn(__fsub_rn(x, tm), a, -t2)), d);
    out[c] = d;
  }
  __syncthreads();
  // the entries' columns, each by its first entry
  for (int i = tid; i < k; i += kThreads) {
    const int c = id[i];
    if (c < from || c >= to) continue;
    float s = 0.0f;
    bool again = false;
    for (int j = 0; j < k; ++j)
      if (id[j] == c) {
        again = again || j < i;
        s = __fadd_rn(s, p[j]);
      }
    if (again) continue;
    out[c] = __fmaf_rn(inside, ex2(__fmaf_rn(__fsub_rn(row[c], m), a, -l2)), -__fmul_rn(scale, s));
  }
}

int check_distill(const char *who, int64_t rows, int64_t vocab, int64_t k, int64_t ld, float temperature) {
  const std::string name(who);
  FZ_REQUIRE(rows >= 0 && vocab >= 1 && k >= 1, name + ": negative or zero size");
  FZ_REQUIRE(vocab <= (1 << 23), name + ": vocab above 2^23");
  FZ_REQUIRE(k <= FZ_MAX_TEACHER, name + ": more than FZ_MAX_TEACHER entries");
  FZ_REQUIRE(ld >= vocab, name + ": row pitch below vocab");
  FZ_REQUIRE(rows <= INT_MAX / 8, name + ": too many rows");
  FZ_REQUIRE(temperature > 0.0f && temperature < INFINITY, name + ": temperature must be positive and finite");
  return FZ_OK;
}

// CTAs per row: the fewest (1, 2, 4, 8) that give every SM two, while a slice keeps 4096
// columns, and enough that a slice's marks fit in shared memory.
int ctas_per_row(int64_t rows, int64_t vocab) {
  int n = 1;
  while (n < 8 && ((rows * n < 2 * (int64_t)fz::num_sms() && vocab / (2 * n) >= 4096) || vocab / n > (1 << 20)))
    n *= 2;
  return n;
}

}  // namespace

extern "C" int fz_distill(float *loss, float *stats, const float *logits, int64_t ld, const int32_t *ids,
                          const float *teacher, const float *teacher_lse, int64_t rows, int64_t vocab, int64_t k,
                          float temperature, void *stream) {
  if (int rc = check_distill("fz_distill", rows, vocab, k, ld, temperature)) return rc;
  if (rows == 0) return FZ_OK;
  FZ_REQUIRE(loss && stats && logits && ids && teacher, "fz_distill: null pointer");
  const int ctas = ctas_per_row(rows, vocab);
  const int slice = (int)(((vocab + 3 + ctas - 1) / ctas + 127) / 128 * 128);
  const size_t smem = (size_t)k * 12 + (teacher_lse ? (size_t)slice / 8 : 0);
  auto kernel = teacher_lse ? distill_kernel<true> : distill_kernel<false>;
  if (smem > 48 * 1024)
    FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kThreads);
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
  FZ_CUDA(cudaLaunchKernelEx(&cfg, kernel, loss, stats, logits, ld, ids, teacher, teacher_lse, (int)vocab,
                             (int)k, temperature, slice));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

extern "C" int fz_distill_backward(float *dlogits, int64_t ldd, const float *dloss, const float *stats,
                                   const float *logits, int64_t ld, const int32_t *ids, const float *teacher,
                                   const float *teacher_lse, int64_t rows, int64_t vocab, int64_t k,
                                   float temperature, void *stream) {
  if (int rc = check_distill("fz_distill_backward", rows, vocab, k, ld, temperature)) return rc;
  FZ_REQUIRE(ldd >= vocab, "fz_distill_backward: row pitch below vocab");
  if (rows == 0) return FZ_OK;
  FZ_REQUIRE(dlogits && dloss && stats && logits && ids && teacher, "fz_distill_backward: null pointer");
  FZ_REQUIRE(dlogits != logits, "fz_distill_backward: dlogits may not overlap logits");
  const int ctas = ctas_per_row(rows, vocab);
  const int slice = (int)((vocab + ctas - 1) / ctas);
  const size_t smem = (size_t)k * 8;
  auto kernel = teacher_lse ? distill_backward_kernel<true> : distill_backward_kernel<false>;
  FZ_CUDA(fz::launch_pdl(kernel, dim3((unsigned)(rows * ctas)), dim3(kThreads), smem, fz::resolve(stream), dlogits,
                         ldd, dloss, stats, logits, ld, ids, teacher, teacher_lse, (int)vocab, (int)k,
                         temperature, slice, ctas));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}
