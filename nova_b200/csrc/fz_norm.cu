// Group norm with an activation, channels last, and its gradients.
#include <climits>
#include <cstdint>

#include "fz_common.cuh"

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float sigmoid(float v) { return __fdiv_rn(1.0f, __fadd_rn(1.0f, expf(-v))); }
__device__ __forceinline__ float phi(float v) {
  return __fmul_rn(0.5f, __fadd_rn(1.0f, erff(__fmul_rn(v, 0.70710678118654752f))));
}

__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case FZ_ACT_RELU: return v > 0.0f ? v : 0.0f;
    case FZ_ACT_SILU: return __fmul_rn(v, sigmoid(v));
    case FZ_ACT_GELU: return __fmul_rn(v, phi(v));
    default: return v;
  }
}

__device__ __forceinline__ float act_slope(int act, float v) {
  switch (act) {
    case FZ_ACT_RELU: return v > 0.0f ? 1.0f : 0.0f;
    case FZ_ACT_SILU: {
      const float s = sigmoid(v);
      return __fmul_rn(s, __fmaf_rn(v, __fsub_rn(1.0f, s), 1.0f));
    }
    case FZ_ACT_GELU:
      return __fmaf_rn(__fmul_rn(v, 0.39894228040143268f), expf(__fmul_rn(-0.5f, __fmul_rn(v, v))), phi(v));
    default: return 1.0f;
  }
}

__device__ __forceinline__ float block_sum(float v, float *sh) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, d));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.0f;
  for (int w = 0; w < kThreads / 32; ++w) s = __fadd_rn(s, sh[w]);
  __syncthreads();
  return s;
}

// One CTA per (b, g).
__global__ void __launch_bounds__(kThreads) group_norm_kernel(float *__restrict__ y, float *__restrict__ mean_out,
                                                              float *__restrict__ rstd_out,
                                                              const float *__restrict__ x,
                                                              const float *__restrict__ gamma,
                                                              const float *__restrict__ beta, int64_t teams,
                                                              int64_t len, int64_t channels, int groups, int cg,
                                                              float eps, int act) {
  pdl_wait();
  __shared__ float sh[kThreads / 32];
  const int64_t m = len * cg;
  for (int64_t team = blockIdx.x; team < teams; team += gridDim.x) {
    const int64_t b = team / groups;
    const int g = (int)(team - b * groups);
    const int64_t base = b * len * channels + (int64_t)g * cg;
    float s = 0.0f;
    for (int64_t i = threadIdx.x; i < m; i += kThreads) s = __fadd_rn(s, x[base + i / cg * channels + i % cg]);
    const float mean = __fdiv_rn(block_sum(s, sh), (float)m);
    s = 0.0f;
    for (int64_t i = threadIdx.x; i < m; i += kThreads) {
      const float d = __fsub_rn(x[base + i / cg * channels + i % cg], mean);
      s = __fmaf_rn(d, d, s);
    }
    const float rstd = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(block_sum(s, sh), (float)m), eps)));
    if (mean_out && threadIdx.x == 0) {
      mean_out[team] = mean;
      rstd_out[team] = rstd;
    }
    for (int64_t i = threadIdx.x; i < m; i += kThreads) {
      const int c = (int)(i % cg);
      const int64_t at = base + i / cg * channels + c;
      const float xh = __fmul_rn(__fsub_rn(x[at], mean), rstd);
      y[at] = act_value(act, __fmaf_rn(xh, gamma ? gamma[g * cg + c] : 1.0f, beta ? beta[g * cg + c] : 0.0f));
    }
  }
}

__global__ void __launch_bounds__(kThreads) group_norm_dx_kernel(
    float *__restrict__ dx, const float *__restrict__ dy, const float *__restrict__ x,
    const float *__restrict__ mean_in, const float *__restrict__ rstd_in, const float *__restrict__ gamma,
    const float *__restrict__ beta, int64_t teams, int64_t len, int64_t channels, int groups, int cg, int act) {
  pdl_wait();
  __shared__ float sh[kThreads / 32];
  const int64_t m = len * cg;
  for (int64_t team = blockIdx.x; team < teams; team += gridDim.x) {
    const int64_t b = team / groups;
    const int g = (int)(team - b * groups);
    const int64_t base = b * len * channels + (int64_t)g * cg;
    const float mean = mean_in[team], rstd = rstd_in[team];
    float s1 = 0.0f, s2 = 0.0f;
    for (int pass = 0; pass < 2; ++pass) {
      float k1 = 0.0f, k2 = 0.0f;
      if (pass) {
        k1 = __fdiv_rn(block_sum(s1, sh), (float)m);
        k2 = __fdiv_rn(block_sum(s2, sh), (float)m);
      }
      for (int64_t i = threadIdx.x; i < m; i += kThreads) {
        const int c = (int)(i % cg);
        const int64_t at = base + i / cg * channels + c;
        const float ga = gamma ? gamma[g * cg + c] : 1.0f;
        const float xh = __fmul_rn(__fsub_rn(x[at], mean), rstd);
        const float v = __fmaf_rn(xh, ga, beta ? beta[g * cg + c] : 0.0f);
        const float a = __fmul_rn(__fmul_rn(dy[at], act_slope(act, v)), ga);
        if (pass) {
          dx[at] = __fmul_rn(rstd, __fsub_rn(__fsub_rn(a, k1), __fmul_rn(xh, k2)));
        } else {
          s1 = __fadd_rn(s1, a);
          s2 = __fmaf_rn(a, xh, s2);
        }
      }
    }
  }
}

// 32 channels a CTA, 8 rows at a time.
__global__ void __launch_bounds__(kThreads) group_norm_dparam_kernel(
    float *__restrict__ dgamma, float *__restrict__ dbeta, const float *__restrict__ dy,
    const float *__restrict__ x, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
    const float *__restrict__ gamma, const float *__restrict__ beta, int64_t rows, int64_t len, int64_t channels,
    int groups, int cg, int act) {
  pdl_wait();
  __shared__ float sh[2][8][32];
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  float s1 = 0.0f, s2 = 0.0f;
  if (c < channels) {
    const float ga = gamma ? gamma[c] : 1.0f, be = beta ? beta[c] : 0.0f;
    for (int64_t r = part; r < rows; r += 8) {
      const int64_t team = r / len * groups + c / cg;
      const float xh = __fmul_rn(__fsub_rn(x[r * channels + c], mean_in[team]), rstd_in[team]);
      const float dv = __fmul_rn(dy[r * channels + c], act_slope(act, __fmaf_rn(xh, ga, be)));
      s1 = __fadd_rn(s1, dv);
      s2 = __fmaf_rn(dv, xh, s2);
    }
  }
  sh[0][part][lane] = s1;
  sh[1][part][lane] = s2;
  __syncthreads();
  if (part == 0 && c < channels) {
    for (int p = 1; p < 8; ++p) {
      s1 = __fadd_rn(s1, sh[0][p][lane]);
      s2 = __fadd_rn(s2, sh[1][p][lane]);
    }
    if (dgamma) dgamma[c] = s2;
    if (dbeta) dbeta[c] = s1;
  }
}

int check_sizes(const char *who, int64_t batch, int64_t len, int64_t channels, int64_t groups) {
  const std::string name(who);
  FZ_REQUIRE(batch >= 0 && len >= 0 && channels >= 1 && groups >= 1, name + ": negative or zero size");
  FZ_REQUIRE(channels % groups == 0, name + ": channels must be a multiple of groups");
  FZ_REQUIRE(channels <= INT_MAX && len <= INT64_MAX / 16 / channels &&
                 (len == 0 || batch <= INT64_MAX / 16 / channels / len),
             name + ": too many elements");
  return FZ_OK;
}

}  // namespace

extern "C" int fz_group_norm_workspace(int64_t batch, int64_t len, int64_t channels, int64_t groups, int backward,
                                       size_t *bytes) {
  FZ_REQUIRE(bytes, "fz_group_norm_workspace: null pointer");
  *bytes = 0;
  if (int rc = check_sizes("fz_group_norm_workspace", batch, len, channels, groups)) return rc;
  (void)backward;
  return FZ_OK;
}

extern "C" int fz_group_norm(float *y, float *mean, float *rstd, const float *x, const float *gamma,
                             const float *beta, int64_t batch, int64_t len, int64_t channels, int64_t groups,
                             float eps, int act, void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check_sizes("fz_group_norm", batch, len, channels, groups)) return rc;
  FZ_REQUIRE(act >= FZ_ACT_NONE && act <= FZ_ACT_GELU, "fz_group_norm: unknown activation");
  FZ_REQUIRE(eps >= 0.0f, "fz_group_norm: eps must not be negative");
  FZ_REQUIRE(!mean == !rstd, "fz_group_norm: mean and rstd are written together");
  (void)workspace;
  (void)workspace_bytes;
  if (batch == 0 || len == 0) return FZ_OK;
  FZ_REQUIRE(x && y, "fz_group_norm: null pointer");
  FZ_REQUIRE(x != y, "fz_group_norm: y may not overlap x");
  const int64_t teams = batch * groups;
  FZ_CUDA(fz::launch_pdl(group_norm_kernel, dim3(fz::grid_for(teams, 1, 8, 4)), dim3(kThreads), 0,
                         fz::resolve(stream), y, mean, rstd, x, gamma, beta, teams, len, channels, (int)groups,
                         (int)(channels / groups), eps, act));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

extern "C" int fz_group_norm_backward(float *dx, float *dgamma, float *dbeta, const float *dy, const float *x,
                                      const float *mean, const float *rstd, const float *gamma, const float *beta,
                                      int64_t batch, int64_t len, int64_t channels, int64_t groups, int act,
                                      void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check_sizes("fz_group_norm_backward", batch, len, channels, groups)) return rc;
  FZ_REQUIRE(act >= FZ_ACT_NONE && act <= FZ_ACT_GELU, "fz_group_norm_backward: unknown activation");
  (void)workspace;
  (void)workspace_bytes;
  const bool data = batch > 0 && len > 0;
  FZ_REQUIRE(!data || (dx && dy && x && mean && rstd), "fz_group_norm_backward: null pointer");
  FZ_REQUIRE(!data || (dx != x && dx != dy), "fz_group_norm_backward: dx may not overlap x or dy");
  cudaStream_t s = fz::resolve(stream);
  const int64_t teams = batch * groups;
  const int cg = (int)(channels / groups);
  if (data) {
    FZ_CUDA(fz::launch_pdl(group_norm_dx_kernel, dim3(fz::grid_for(teams, 1, 8, 4)), dim3(kThreads), 0, s, dx, dy,
                           x, mean, rstd, gamma, beta, teams, len, channels, (int)groups, cg, act));
    FZ_CHECK_LAUNCH();
  }
  if (dgamma || dbeta) {
    FZ_CUDA(fz::launch_pdl(group_norm_dparam_kernel, dim3((unsigned)((channels + 31) / 32)), dim3(kThreads), 0, s,
                           dgamma, dbeta, dy, x, mean, rstd, gamma, beta, batch * len, len > 0 ? len : 1, channels,
                           (int)groups, cg, act));
    FZ_CHECK_LAUNCH();
  }
  return FZ_OK;
}
