// Group norm with an activation, channels last, and its gradients.
//
// x is [batch, len, channels]; the team (b, g) is the len x c block of sample b's group g
// of c = channels / groups channels, m = len * c values. All kernels are bound by HBM:
// forward 8 bytes a value (read x, write y), backward 12 (read x and dy, write dx), if a
// team's values are read once. So they stay in registers between the statistics and the
// result, in the smallest set of threads that holds a team:
//   * row kernels: a team of at most 256 vectors (of 4, 2 or 1 floats, as alignment
//     allows) is held by 4 to 32 lanes of a warp, of at most 2048 vectors by a CTA;
//   * tile kernels: a tile of rows x columns (several whole groups wide, or a part of
//     one) a CTA; the tiles of a team exchange their statistics through distributed
//     shared memory in one cluster, of up to 16 CTAs;
//   * larger teams: the tile kernels in two launches that leave the statistics in the
//     workspace and read x (and dy) twice; the second launch takes the tiles in reverse,
//     so it finds the last of what the first read in L2.
// Statistics: the mean, then the sum of squares about it, so that a common offset of x
// does not cancel; parts are joined by (n, mean, M2) <- the union's (Chan, Golub and
// LeVeque). Everything is summed in a fixed order.
//
// Backward: with xh and v recomputed from x, dv = dy act'(v) and, per channel,
// sum dv and sum dv xh: these give dbeta and dgamma, and weighted by gamma and summed over
// the group's channels the two sums that dx needs. A thread sees only few channels, whose
// sums it keeps in registers; per-CTA (or, in the row kernels, per-team) partial sums go to
// the workspace and a last launch adds them up.
#include <cooperative_groups.h>

#include <climits>
#include <cstdint>

#include "fz_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRowThreads = 256;
constexpr int kTileForward = 512, kTileBackward = 256;  // threads
// Vectors of x a tile kernel's thread holds: what the registers of two CTAs an SM leave.
__host__ __device__ constexpr int held(int v) { return v == 4 ? 8 : v == 2 ? 12 : 16; }
constexpr int kMaxCluster = 16;

// ---------------------------------------------------------------- activations

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float sigmoid(float v) {
  return rcp(__fadd_rn(1.0f, ex2(__fmul_rn(v, -1.4426950408889634f))));
}

// Phi(v) and, through e, exp(-v^2 / 2). With h = Phi(-|v|) = exp(-v^2 / 2) R(t), t = 1 /
// (1 + 0.3 |v|): R is a polynomial of degree 8 without constant term, fitted to the least
// largest relative error on |v| <= 14 (Remez; 1.5e-7). erff would take the forward from
// memory- to issue-bound.
__device__ __forceinline__ float phi(float v, float *e) {
  const float t = rcp(__fmaf_rn(fabsf(v), 0.3f, 1.0f));
  *e = ex2(__fmul_rn(__fmul_rn(v, v), -0.72134752044448170f));
  float r = __fmaf_rn(0.035674769431352615f, t, -0.1572030633687973f);
  r = __fmaf_rn(r, t, 0.20635347068309784f);
  r = __fmaf_rn(r, t, -0.05368361622095108f);
  r = __fmaf_rn(r, t, 0.1285616159439087f);
  r = __fmaf_rn(r, t, 0.09991349279880524f);
  r = __fmaf_rn(r, t, 0.12075395882129669f);
  r = __fmaf_rn(r, t, 0.11962930113077164f);
  const float h = __fmul_rn(__fmul_rn(r, t), *e);
  return v < 0.0f ? h : __fsub_rn(1.0f, h);  // NaN: h is NaN
}

template <int V>
__device__ __forceinline__ void activate(int act, float (&v)[V]) {
  if (act == FZ_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __fmul_rn(v[j], sigmoid(v[j]));
  } else if (act == FZ_ACT_GELU) {
    float e;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __fmul_rn(v[j], phi(v[j], &e));
  } else if (act == FZ_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = v[j] > 0.0f ? v[j] : 0.0f;
  }
}

// d *= act'(v)
template <int V>
__device__ __forceinline__ void times_slope(int act, float (&d)[V], const float (&v)[V]) {
  if (act == FZ_ACT_SILU) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const float s = sigmoid(v[j]);
      d[j] = __fmul_rn(d[j], __fmul_rn(s, __fmaf_rn(v[j], __fsub_rn(1.0f, s), 1.0f)));
    }
  } else if (act == FZ_ACT_GELU) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      float e;
      const float p = phi(v[j], &e);
      d[j] = __fmul_rn(d[j], __fmaf_rn(__fmul_rn(v[j], 0.39894228040143268f), e, p));
    }
  } else if (act == FZ_ACT_RELU) {
#pragma unroll
    for (int j = 0; j < V; ++j) d[j] = v[j] > 0.0f ? d[j] : 0.0f;
  }
}

// ---------------------------------------------------------------- vectors

template <int V>
__device__ __forceinline__ void load(float (&r)[V], const float *p) {
  if constexpr (V == 4) {
    const float4 q = *reinterpret_cast<const float4 *>(p);
    r[0] = q.x, r[1] = q.y, r[2] = q.z, r[3] = q.w;
  } else if constexpr (V == 2) {
    const float2 q = *reinterpret_cast<const float2 *>(p);
    r[0] = q.x, r[1] = q.y;
  } else {
    r[0] = *p;
  }
}
template <int V>
__device__ __forceinline__ void store(float *p, const float (&r)[V]) {
  if constexpr (V == 4) *reinterpret_cast<float4 *>(p) = make_float4(r[0], r[1], r[2], r[3]);
  else if constexpr (V == 2) *reinterpret_cast<float2 *>(p) = make_float2(r[0], r[1]);
  else *p = r[0];
}
template <int V>
__device__ __forceinline__ void load_or(float (&r)[V], const float *p, float otherwise) {
  if (p) {
    load(r, p);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = otherwise;
  }
}

// (n, mean, M2) of a union.
struct Moments {
  float n, mean, m2;
};
__device__ __forceinline__ Moments join(Moments a, Moments b) {
  if (b.n == 0.0f) return a;
  if (a.n == 0.0f) return b;
  const float n = __fadd_rn(a.n, b.n), d = __fsub_rn(b.mean, a.mean), f = __fdiv_rn(b.n, n);
  return {n, __fmaf_rn(d, f, a.mean), __fmaf_rn(__fmul_rn(d, d), __fmul_rn(a.n, f), __fadd_rn(a.m2, b.m2))};
}
__device__ __forceinline__ float rstd_of(float m2, float m, float eps) {
  return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(m2, m), eps)));
}

struct Norm {
  const float *x, *gamma, *beta;
  float *y, *mean, *rstd;
  const float *dy, *mean_in, *rstd_in;
  float *dx;
  float *part;  // per-channel partial sums, or null: [part][2][...]
  float *stat;  // two-launch tiles: statistics of a group's tiles
  int64_t batch, len, channels;
  int groups, c;  // c: channels a group
  float m, eps;
  int act;
};

// ---------------------------------------------------------------- row kernels

// Sum over the P lanes (or, P = kRowThreads, threads) of a team.
template <int P>
__device__ __forceinline__ float team_sum(float v, float *sh) {
#pragma unroll
  for (int d = (P < 32 ? P : 32) / 2; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kFull, v, d));
  if constexpr (P > 32) {
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[0];
#pragma unroll
    for (int w = 1; w < P / 32; ++w) v = __fadd_rn(v, sh[w]);
  }
  return v;
}

// Teams id, id + stride, ... belong to P lanes each, stride a multiple of groups, so a
// set of lanes keeps its group and a lane its channels. U teams are in flight at a time.
// Lane vector i covers the team's vectors i * P + lane.
template <int V, int P, int NV>
struct RowTeam {
  int g, part;
  bool on;
  int at[NV];  // offset of each vector in the sample's group, -1 behind the end
  int channel[NV];
  __device__ RowTeam(const Norm &a, int stride) {
    const int id = P > 32 ? (int)blockIdx.x : (int)((blockIdx.x * kRowThreads + threadIdx.x) / P);
    on = id < stride;
    part = id / a.groups;
    g = id - part * a.groups;
    const int cv = a.c / V, nv = (int)a.len * cv;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int q = i * P + (int)(threadIdx.x % P), l = q / cv;
      const int ch = (q - l * cv) * V;
      at[i] = q < nv ? l * (int)a.channels + ch : -1;
      channel[i] = g * a.c + (q < nv ? ch : 0);
    }
  }
};

template <int V, int P, int NV, int U>
__global__ void __launch_bounds__(kRowThreads) norm_rows_kernel(const Norm a, int stride) {
  pdl_wait();
  __shared__ float sh[kRowThreads / 32];
  const RowTeam<V, P, NV> t(a, stride);
  const int parts = stride / a.groups;
  const int64_t sample = a.len * a.channels;
  for (int64_t b0 = 0; b0 < a.batch; b0 += (int64_t)parts * U) {
    float x[U][NV][V], mean[U], rstd[U];
    bool on[U];
    int64_t base[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t b = b0 + (int64_t)u * parts + t.part;
      on[u] = t.on && b < a.batch;
      base[u] = b * sample + (int64_t)t.g * a.c;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (on[u] && t.at[i] >= 0) {
          load(x[u][i], a.x + base[u] + t.at[i]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) x[u][i][j] = 0.0f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s = __fadd_rn(s, x[u][i][j]);
      mean[u] = s;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) mean[u] = __fdiv_rn(team_sum<P>(mean[u], sh), a.m);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t.at[i] >= 0)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float d = __fsub_rn(x[u][i][j], mean[u]);
            s = __fmaf_rn(d, d, s);
          }
      rstd[u] = s;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) rstd[u] = rstd_of(team_sum<P>(rstd[u], sh), a.m, a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (t.at[i] < 0) continue;
      float ga[V], be[V];
      load_or(ga, a.gamma ? a.gamma + t.channel[i] : nullptr, 1.0f);
      load_or(be, a.beta ? a.beta + t.channel[i] : nullptr, 0.0f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!on[u]) continue;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[j] = __fmaf_rn(__fmul_rn(__fsub_rn(x[u][i][j], mean[u]), rstd[u]), ga[j], be[j]);
        activate(a.act, v);
        store(a.y + base[u] + t.at[i], v);
      }
    }
    if (a.mean && threadIdx.x % P == 0)
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (on[u]) {
          const int64_t team = (b0 + (int64_t)u * parts + t.part) * a.groups + t.g;
          a.mean[team] = mean[u];
          a.rstd[team] = rstd[u];
        }
  }
}

template <int V, int P, int NV, int U>
__global__ void __launch_bounds__(kRowThreads) norm_rows_backward_kernel(const Norm a, int stride) {
  pdl_wait();
  __shared__ float sh[kRowThreads / 32];
  const RowTeam<V, P, NV> t(a, stride);
  const int parts = stride / a.groups;
  const int64_t sample = a.len * a.channels;
  float db[NV][V], dg[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) db[i][j] = dg[i][j] = 0.0f;
  for (int64_t b0 = 0; b0 < a.batch; b0 += (int64_t)parts * U) {
    float x[U][NV][V], d[U][NV][V], mean[U], rstd[U], s1[U], s2[U];
    bool on[U];
    int64_t base[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t b = b0 + (int64_t)u * parts + t.part;
      on[u] = t.on && b < a.batch;
      base[u] = b * sample + (int64_t)t.g * a.c;
      mean[u] = on[u] ? a.mean_in[b * a.groups + t.g] : 0.0f;
      rstd[u] = on[u] ? a.rstd_in[b * a.groups + t.g] : 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (on[u] && t.at[i] >= 0) {
          load(x[u][i], a.x + base[u] + t.at[i]);
          load(d[u][i], a.dy + base[u] + t.at[i]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) x[u][i][j] = d[u][i][j] = 0.0f;
        }
      }
    }
    // x <- xh, d <- dv gamma
#pragma unroll
    for (int u = 0; u < U; ++u) s1[u] = s2[u] = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float ga[V], be[V];
      load_or(ga, a.gamma ? a.gamma + t.channel[i] : nullptr, 1.0f);
      load_or(be, a.beta ? a.beta + t.channel[i] : nullptr, 0.0f);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!on[u] || t.at[i] < 0) continue;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          x[u][i][j] = __fmul_rn(__fsub_rn(x[u][i][j], mean[u]), rstd[u]);
          v[j] = __fmaf_rn(x[u][i][j], ga[j], be[j]);
        }
        times_slope(a.act, d[u][i], v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          db[i][j] = __fadd_rn(db[i][j], d[u][i][j]);
          dg[i][j] = __fmaf_rn(d[u][i][j], x[u][i][j], dg[i][j]);
          d[u][i][j] = __fmul_rn(d[u][i][j], ga[j]);
          s1[u] = __fadd_rn(s1[u], d[u][i][j]);
          s2[u] = __fmaf_rn(d[u][i][j], x[u][i][j], s2[u]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      s1[u] = __fdiv_rn(team_sum<P>(s1[u], sh), a.m);
      s2[u] = __fdiv_rn(team_sum<P>(s2[u], sh), a.m);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (!on[u] || t.at[i] < 0) continue;
        float v[V];
#pragma unroll
        for (int j = 0; j < V; ++j)
          v[j] = __fmul_rn(rstd[u], __fsub_rn(__fsub_rn(d[u][i][j], s1[u]), __fmul_rn(x[u][i][j], s2[u])));
        store(a.dx + base[u] + t.at[i], v);
      }
  }
  if (a.part && t.on) {
    // [part][2][groups][len * c]: every vector of the team a column of its own
    const int64_t row = (int64_t)a.groups * a.len * a.c;
    float *p = a.part + (int64_t)t.part * 2 * row + (int64_t)t.g * a.len * a.c;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t.at[i] >= 0) {
        float *q = p + (i * P + (int64_t)(threadIdx.x % P)) * V;
        store(q, db[i]);
        store(q + row, dg[i]);
      }
  }
}

// ---------------------------------------------------------------- tile kernels

// How a launch cuts samples into tiles (see norm_plan).
struct Tiling {
  int cols;      // vectors a tile is wide
  int q;         // whole groups a tile holds (1 where a group is split)
  int split;     // tiles a group's columns are split into
  int bundles;   // tiles side by side over a sample's groups (without the split)
  int ty;        // thread rows of a tile
  int rows;      // rows a tile
  int chunks;    // tiles one below the other
  int k;         // tiles that share statistics: split * chunks
};

template <int V, int THREADS>
struct Tile {
  int64_t b;
  int k, chunk;
  int q;             // groups in this tile
  int g0;            // its first group
  int cols;          // its vectors a row
  int tx, ty;
  bool on;           // this thread holds a column
  int channel;       // its first channel
  int group;         // its group, counted from g0
  int row0, rows;    // its rows
  int64_t base;
  // share: which of the k tiles that share statistics; team: which set of them
  __device__ Tile(const Norm &a, const Tiling &t, int64_t team, int share) {
    b = team / t.bundles;
    k = share;
    const int bundle = (int)(team - b * t.bundles);
    chunk = share / t.split;
    const int piece = share - chunk * t.split, cv = a.c / V;
    g0 = bundle * t.q;
    q = min(t.q, a.groups - g0);
    cols = t.split > 1 ? min(t.cols, cv - piece * t.cols) : q * cv;
    tx = threadIdx.x % t.cols;
    ty = threadIdx.x / t.cols;
    on = ty < t.ty && tx < cols;
    channel = g0 * a.c + (piece * t.cols + tx) * V;
    group = t.split > 1 ? 0 : tx / cv;
    row0 = chunk * t.rows;
    rows = (int)min((int64_t)t.rows, a.len - row0);
    base = (b * a.len + row0) * a.channels + channel;
  }
  // values of one group in the tile
  __device__ float count(const Norm &a, const Tiling &t) const {
    return (float)rows * (float)(t.split > 1 ? cols * V : a.c);
  }
  // the same of another tile that shares the statistics
  static __device__ float count_of(const Norm &a, const Tiling &t, int share) {
    const int chunk = share / t.split, piece = share - chunk * t.split;
    const float r = (float)min((int64_t)t.rows, a.len - (int64_t)chunk * t.rows);
    return r * (float)(t.split > 1 ? min(t.cols, a.c / V - piece * t.cols) * V : a.c);
  }
};

// sums[g] of the threads' v over the tile's groups; sh holds a float a thread. A warp takes
// a group at a time.
template <int V, int THREADS>
__device__ __forceinline__ void group_sums(float v, float *sh, float *sums, const Tile<V, THREADS> &me,
                                           const Tiling &t, int cv) {
  sh[threadIdx.x] = me.on ? v : 0.0f;
  __syncthreads();
  const int lane = threadIdx.x & 31, width = t.split > 1 ? me.cols : cv;
  for (int g = threadIdx.x >> 5; g < me.q; g += THREADS / 32) {
    float s = 0.0f;
    for (int i = lane; i < width * t.ty; i += 32) {
      const int y = i / width;
      s = __fadd_rn(s, sh[y * t.cols + g * cv + (i - y * width)]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s = __fadd_rn(s, __shfl_xor_sync(kFull, s, d));
    if (lane == 0) sums[g] = s;
  }
  __syncthreads();
}

template <int V, int THREADS>
__device__ __forceinline__ void load_tile(float (&x)[held(V)][V], const float *p, const Tile<V, THREADS> &me,
                                          const Tiling &t, int64_t channels) {
#pragma unroll
  for (int i = 0; i < held(V); ++i) {
    const int r = me.ty + i * t.ty;
    if (me.on && r < me.rows) {
      load(x[i], p + me.base + r * channels);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) x[i][j] = 0.0f;
    }
  }
}

// The tile's own mean and M2 per group, in shared memory.
template <int V, int THREADS>
__device__ __forceinline__ void tile_moments(const float (&x)[held(V)][V], float *sh, float *mean, float *m2,
                                             const Norm &a, const Tile<V, THREADS> &me, const Tiling &t) {
  const int cv = a.c / V;
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < held(V); ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) s = __fadd_rn(s, x[i][j]);
  group_sums(s, sh, m2, me, t, cv);
  const float n = me.count(a, t);
  for (int g = threadIdx.x; g < me.q; g += THREADS) mean[g] = __fdiv_rn(m2[g], n);
  __syncthreads();
  const float mu = me.on ? mean[me.group] : 0.0f;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < held(V); ++i)
    if (me.ty + i * t.ty < me.rows)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = __fsub_rn(x[i][j], mu);
        s = __fmaf_rn(d, d, s);
      }
  group_sums(s, sh, m2, me, t, cv);
}

template <int V, int THREADS>
__device__ __forceinline__ void write_tile(const float (&x)[held(V)][V], float mean, float rstd, const Norm &a,
                                           const Tile<V, THREADS> &me, const Tiling &t) {
  if (!me.on) return;
  float ga[V], be[V];
  load_or(ga, a.gamma ? a.gamma + me.channel : nullptr, 1.0f);
  load_or(be, a.beta ? a.beta + me.channel : nullptr, 0.0f);
#pragma unroll
  for (int i = 0; i < held(V); ++i) {
    const int r = me.ty + i * t.ty;
    if (r >= me.rows) break;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = __fmaf_rn(__fmul_rn(__fsub_rn(x[i][j], mean), rstd), ga[j], be[j]);
    activate(a.act, v);
    store(a.y + me.base + r * a.channels, v);
  }
}

// One cluster per set of tiles that share statistics.
template <int V>
__global__ void __launch_bounds__(kTileForward, 2) norm_tile_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileForward;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ float sh[T], mean[T], m2[T], mean_all[T], rstd_all[T];
  const Tile<V, T> me(a, t, blockIdx.x / t.k, (int)(blockIdx.x % t.k));
  float x[held(V)][V];
  load_tile(x, a.x, me, t, a.channels);
  tile_moments(x, sh, mean, m2, a, me, t);
  if (t.k > 1) cluster.sync();
  for (int g = threadIdx.x; g < me.q; g += T) {
    Moments s{0.0f, 0.0f, 0.0f};
    if (t.k > 1) {
      for (int r = 0; r < t.k; ++r)
        s = join(s, {Tile<V, T>::count_of(a, t, r), cluster.map_shared_rank(mean, r)[g],
                     cluster.map_shared_rank(m2, r)[g]});
    } else {
      s = {a.m, mean[g], m2[g]};
    }
    mean_all[g] = s.mean;
    rstd_all[g] = rstd_of(s.m2, a.m, a.eps);
    if (a.mean && me.k == 0) {
      a.mean[me.b * a.groups + me.g0 + g] = s.mean;
      a.rstd[me.b * a.groups + me.g0 + g] = rstd_all[g];
    }
  }
  __syncthreads();
  if (t.k > 1) cluster.barrier_arrive();
  if (me.on) write_tile(x, mean_all[me.group], rstd_all[me.group], a, me, t);
  if (t.k > 1) cluster.barrier_wait();  // no CTA leaves while its statistics may be read
}

// The two-launch form: statistics to stat[(b * groups + g) * k + tile] = (mean, M2) ...
template <int V>
__global__ void __launch_bounds__(kTileForward, 2) norm_tile_stats_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileForward;
  __shared__ float sh[T], mean[T], m2[T];
  const Tile<V, T> me(a, t, blockIdx.x / t.k, (int)(blockIdx.x % t.k));
  float x[held(V)][V];
  load_tile(x, a.x, me, t, a.channels);
  tile_moments(x, sh, mean, m2, a, me, t);
  for (int g = threadIdx.x; g < me.q; g += T) {
    float *s = a.stat + ((me.b * a.groups + me.g0 + g) * t.k + me.k) * 2;
    s[0] = mean[g];
    s[1] = m2[g];
  }
}
// ... and the result from them: a warp joins a group's tiles.
template <int V>
__global__ void __launch_bounds__(kTileForward, 2) norm_tile_apply_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileForward;
  __shared__ float mean_all[T], rstd_all[T];
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const Tile<V, T> me(a, t, block / t.k, (int)(block % t.k));
  float x[held(V)][V];
  load_tile(x, a.x, me, t, a.channels);
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < me.q; g += T / 32) {
    const int64_t team = me.b * a.groups + me.g0 + g;
    Moments s{0.0f, 0.0f, 0.0f};
    for (int r = lane; r < t.k; r += 32) {
      const float2 p = *reinterpret_cast<const float2 *>(a.stat + (team * t.k + r) * 2);
      s = join(s, {Tile<V, T>::count_of(a, t, r), p.x, p.y});
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const Moments o{__shfl_down_sync(kFull, s.n, d), __shfl_down_sync(kFull, s.mean, d),
                      __shfl_down_sync(kFull, s.m2, d)};
      s = join(s, o);
    }
    if (lane == 0) {
      mean_all[g] = s.mean;
      rstd_all[g] = rstd_of(s.m2, a.m, a.eps);
      if (a.mean && me.k == 0) {
        a.mean[team] = s.mean;
        a.rstd[team] = rstd_all[g];
      }
    }
  }
  __syncthreads();
  if (me.on) write_tile(x, mean_all[me.group], rstd_all[me.group], a, me, t);
}

// x <- xh, d <- dv gamma, and the column sums of dv and dv xh of this thread's rows.
template <int V, int THREADS>
__device__ __forceinline__ void tile_gradient(float (&x)[held(V)][V], float (&d)[held(V)][V], float (&db)[V],
                                              float (&dg)[V], const Norm &a, const Tile<V, THREADS> &me,
                                              const Tiling &t) {
#pragma unroll
  for (int j = 0; j < V; ++j) db[j] = dg[j] = 0.0f;
  if (!me.on) return;
  float ga[V], be[V];
  load_or(ga, a.gamma ? a.gamma + me.channel : nullptr, 1.0f);
  load_or(be, a.beta ? a.beta + me.channel : nullptr, 0.0f);
  const int64_t team = me.b * a.groups + me.g0 + me.group;
  const float mean = a.mean_in[team], rstd = a.rstd_in[team];
#pragma unroll
  for (int i = 0; i < held(V); ++i) {
    if (me.ty + i * t.ty >= me.rows) break;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      x[i][j] = __fmul_rn(__fsub_rn(x[i][j], mean), rstd);
      v[j] = __fmaf_rn(x[i][j], ga[j], be[j]);
    }
    times_slope(a.act, d[i], v);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      db[j] = __fadd_rn(db[j], d[i][j]);
      dg[j] = __fmaf_rn(d[i][j], x[i][j], dg[j]);
      d[i][j] = __fmul_rn(d[i][j], ga[j]);
    }
  }
}

// The tile's sums: per channel into `part`, and gamma-weighted per group into s1, s2
// (shared memory). sh: 2 V floats a thread.
template <int V, int THREADS>
__device__ __forceinline__ void tile_gradient_sums(const float (&db)[V], const float (&dg)[V], float *sh, float *s1,
                                                   float *s2, const Norm &a, const Tile<V, THREADS> &me,
                                                   const Tiling &t) {
  const int wide = t.cols * V;  // channels of a full tile
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (me.ty < t.ty) {
      sh[me.ty * wide + me.tx * V + j] = db[j];
      sh[(t.ty + me.ty) * wide + me.tx * V + j] = dg[j];
    }
  }
  __syncthreads();
  const int n = me.cols * V, first = me.channel - me.tx * V;
  for (int i = threadIdx.x; i < 2 * n; i += THREADS) {
    const int which = i >= n, ch = i - which * n;
    float *col = sh + which * t.ty * wide + ch;
    float s = col[0];
    for (int y = 1; y < t.ty; ++y) s = __fadd_rn(s, col[y * wide]);
    col[0] = s;
    if (a.part) a.part[((me.b * t.chunks + me.chunk) * 2 + which) * a.channels + first + ch] = s;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, width = t.split > 1 ? n : a.c;
  for (int g = threadIdx.x >> 5; g < me.q; g += THREADS / 32) {
    float u = 0.0f, w = 0.0f;
    for (int i = lane; i < width; i += 32) {
      const float ga = a.gamma ? a.gamma[first + g * a.c + i] : 1.0f;
      u = __fmaf_rn(ga, sh[g * a.c + i], u);
      w = __fmaf_rn(ga, sh[t.ty * wide + g * a.c + i], w);
    }
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) {
      u = __fadd_rn(u, __shfl_xor_sync(kFull, u, e));
      w = __fadd_rn(w, __shfl_xor_sync(kFull, w, e));
    }
    if (lane == 0) {
      s1[g] = u;
      s2[g] = w;
    }
  }
  __syncthreads();
}

template <int V, int THREADS>
__device__ __forceinline__ void write_gradient(const float (&x)[held(V)][V], const float (&d)[held(V)][V],
                                               float k1, float k2, const Norm &a, const Tile<V, THREADS> &me,
                                               const Tiling &t) {
  const float rstd = a.rstd_in[me.b * a.groups + me.g0 + me.group];
#pragma unroll
  for (int i = 0; i < held(V); ++i) {
    const int r = me.ty + i * t.ty;
    if (r >= me.rows) break;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j)
      v[j] = __fmul_rn(rstd, __fsub_rn(__fsub_rn(d[i][j], k1), __fmul_rn(x[i][j], k2)));
    store(a.dx + me.base + r * a.channels, v);
  }
}

template <int V>
__global__ void __launch_bounds__(kTileBackward, 2) norm_tile_backward_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileBackward;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ float sh[2 * V * T], s1[T], s2[T], k1[T], k2[T];
  const Tile<V, T> me(a, t, blockIdx.x / t.k, (int)(blockIdx.x % t.k));
  float x[held(V)][V], d[held(V)][V], db[V], dg[V];
  load_tile(x, a.x, me, t, a.channels);
  load_tile(d, a.dy, me, t, a.channels);
  tile_gradient(x, d, db, dg, a, me, t);
  tile_gradient_sums(db, dg, sh, s1, s2, a, me, t);
  if (t.k > 1) cluster.sync();
  for (int g = threadIdx.x; g < me.q; g += T) {
    float u = s1[g], w = s2[g];
    if (t.k > 1) {
      u = w = 0.0f;
      for (int r = 0; r < t.k; ++r) {
        u = __fadd_rn(u, cluster.map_shared_rank(s1, r)[g]);
        w = __fadd_rn(w, cluster.map_shared_rank(s2, r)[g]);
      }
    }
    k1[g] = __fdiv_rn(u, a.m);
    k2[g] = __fdiv_rn(w, a.m);
  }
  __syncthreads();
  if (t.k > 1) cluster.barrier_arrive();
  if (me.on) write_gradient(x, d, k1[me.group], k2[me.group], a, me, t);
  if (t.k > 1) cluster.barrier_wait();
}

template <int V>
__global__ void __launch_bounds__(kTileBackward, 2) norm_tile_sums_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileBackward;
  __shared__ float sh[2 * V * T], s1[T], s2[T];
  const Tile<V, T> me(a, t, blockIdx.x / t.k, (int)(blockIdx.x % t.k));
  float x[held(V)][V], d[held(V)][V], db[V], dg[V];
  load_tile(x, a.x, me, t, a.channels);
  load_tile(d, a.dy, me, t, a.channels);
  tile_gradient(x, d, db, dg, a, me, t);
  tile_gradient_sums(db, dg, sh, s1, s2, a, me, t);
  for (int g = threadIdx.x; g < me.q; g += T) {
    float *s = a.stat + ((me.b * a.groups + me.g0 + g) * t.k + me.k) * 2;
    s[0] = s1[g];
    s[1] = s2[g];
  }
}

template <int V>
__global__ void __launch_bounds__(kTileBackward, 2) norm_tile_dx_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int T = kTileBackward;
  __shared__ float k1[T], k2[T];
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const Tile<V, T> me(a, t, block / t.k, (int)(block % t.k));
  float x[held(V)][V], d[held(V)][V], db[V], dg[V];
  load_tile(x, a.x, me, t, a.channels);
  load_tile(d, a.dy, me, t, a.channels);
  const int lane = threadIdx.x & 31;
  for (int g = threadIdx.x >> 5; g < me.q; g += T / 32) {
    const int64_t team = me.b * a.groups + me.g0 + g;
    float u = 0.0f, w = 0.0f;
    for (int r = lane; r < t.k; r += 32) {
      const float2 p = *reinterpret_cast<const float2 *>(a.stat + (team * t.k + r) * 2);
      u = __fadd_rn(u, p.x);
      w = __fadd_rn(w, p.y);
    }
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) {
      u = __fadd_rn(u, __shfl_xor_sync(kFull, u, e));
      w = __fadd_rn(w, __shfl_xor_sync(kFull, w, e));
    }
    if (lane == 0) {
      k1[g] = __fdiv_rn(u, a.m);
      k2[g] = __fdiv_rn(w, a.m);
    }
  }
  tile_gradient(x, d, db, dg, a, me, t);
  __syncthreads();
  if (me.on) write_gradient(x, d, k1[me.group], k2[me.group], a, me, t);
}

// ---------------------------------------------------------------- the parameters' gradients

// dbeta[c] and dgamma[c] from part[p][2][groups][len][c] (len = 1 for the tile kernels'
// per-channel rows): 32 channels a CTA, the p x len rows over its warps and over the CTAs of
// a cluster, which fold their sums through distributed shared memory in order.
constexpr int kFoldWarps = 16;
__global__ void __launch_bounds__(kFoldWarps * 32) norm_fold_kernel(float *__restrict__ dgamma,
                                                                    float *__restrict__ dbeta,
                                                                    const float *__restrict__ part, int64_t parts,
                                                                    int64_t len, int64_t channels, int groups, int c) {
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  __shared__ float sh[2][kFoldWarps][32];
  __shared__ float sum[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t ch = (int64_t)(blockIdx.x / ctas) * 32 + lane;
  float s[2] = {0.0f, 0.0f};
  if (ch < channels) {
    const int64_t row = channels * len, g = ch / c, col = g * len * c + (ch - g * c);
    const uint32_t n = (uint32_t)(parts * len), per = (uint32_t)len;
#pragma unroll 4
    for (uint32_t r = rank * kFoldWarps + warp; r < n; r += ctas * kFoldWarps) {
      const uint32_t p = r / per, l = r - p * per;
      const float *at = part + p * 2 * row + col + (int64_t)l * c;
      s[0] = __fadd_rn(s[0], at[0]);
      s[1] = __fadd_rn(s[1], at[row]);
    }
  }
  sh[0][warp][lane] = s[0];
  sh[1][warp][lane] = s[1];
  __syncthreads();
  if (warp < 2) {
    float u = sh[warp][0][lane];
#pragma unroll
    for (int w = 1; w < kFoldWarps; ++w) u = __fadd_rn(u, sh[warp][w][lane]);
    sum[warp][lane] = u;
  }
  cluster.sync();
  if (rank == 0 && warp < 2 && ch < channels) {
    float u = 0.0f;
    for (int r = 0; r < ctas; ++r) u = __fadd_rn(u, cluster.map_shared_rank(&sum[0][0], r)[warp * 32 + lane]);
    float *out = warp ? dgamma : dbeta;
    if (out) out[ch] = u;
  }
  cluster.sync();
}

// ---------------------------------------------------------------- choosing a kernel

// How a call runs, from its sizes alone (and the buffers' alignment, through v).
struct Plan {
  int v;                 // floats a vector
  int lanes, nv;         // row kernels: lanes a team (0: tile kernels), vectors a lane
  int stride;            // row kernels: teams in flight
  unsigned grid;
  Tiling t;
  bool cluster;          // tile kernels: statistics within a cluster
  int64_t parts, part_len;  // rows of the per-channel partial sums (backward)
  size_t part_floats, stat_floats;
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan norm_plan(int64_t batch, int64_t len, int64_t channels, int64_t groups, int v, bool backward) {
  Plan p{};
  const int64_t c = channels / groups;
  while (c % v) v /= 2;
  p.v = v;
  const int64_t cv = c / v, vectors = len * cv, teams = batch * groups;
  // Row kernels up to 2048 vectors; above 256 (a CTA's worth) only where a row's piece of
  // a group is at least 512 bytes, else the tile kernels, which take several groups' pieces
  // of a row together.
  if (len * channels <= INT_MAX && (vectors <= 256 || (vectors <= 2048 && c >= 128))) {
    p.lanes = vectors <= 4 ? 4 : vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 256 ? 32 : kRowThreads;
    p.nv = 1;
    while ((int64_t)p.nv * p.lanes < vectors) p.nv *= 2;
    const int64_t per_cta = kRowThreads / p.lanes;
    // enough teams in flight to fill the SMs a few times over; a multiple of groups
    int64_t want = (int64_t)fz::num_sms() * 16 * per_cta / (p.lanes > 32 ? 2 : 1);
    if (want > teams) want = teams;
    want = want / groups * groups;
    if (want < groups) want = groups;
    p.stride = (int)want;
    p.grid = (unsigned)up(want, per_cta);
    if (backward) {
      p.parts = want / groups;
      p.part_len = len;
      p.part_floats = (size_t)(p.parts * 2 * channels * len);
    }
    return p;
  }
  // Tiles: whole groups side by side until a row's piece has 128 bytes, or a part of one
  // group where it has more vectors than a CTA has threads.
  const int threads = backward ? kTileBackward : kTileForward;
  Tiling &t = p.t;
  t.q = 1;
  t.split = (int)up(cv, threads);
  if (t.split == 1) {
    const int64_t want = up(32, c);
    t.q = (int)(want < groups ? want : groups);
    while (t.q > 1 && t.q * cv > threads) --t.q;
    t.cols = (int)(t.q * cv);
  } else {
    t.cols = (int)up(cv, t.split);
  }
  t.bundles = (int)up(groups, t.q);
  t.ty = threads / t.cols;
  t.rows = t.ty * held(v);
  if (t.rows > len) t.rows = (int)len;
  t.chunks = (int)up(len, t.rows);
  const int64_t k = (int64_t)t.split * t.chunks;
  t.k = (int)k;
  p.cluster = k <= kMaxCluster;
  p.grid = (unsigned)(batch * t.bundles * k);
  if (backward) {
    p.parts = batch * t.chunks;
    p.part_len = 1;
    p.part_floats = (size_t)(p.parts * 2 * channels);
  }
  if (!p.cluster) p.stat_floats = (size_t)(teams * k * 2);
  return p;
}

int vector_of(std::initializer_list<const void *> ptrs) {
  uintptr_t all = 0;
  for (const void *p : ptrs) all |= (uintptr_t)p;
  return (all & 15) == 0 ? 4 : (all & 7) == 0 ? 2 : 1;
}

// Launch `kernel` over clusters of `k` CTAs (k = 1: none).
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kernel)(KArgs...), unsigned grid, int threads, int k, cudaStream_t s, Args... args) {
  if (k > 8) FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)k;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  FZ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

using RowKernel = void (*)(const Norm, int);
template <int V>
RowKernel row_kernel(int lanes, int nv) {
  if (lanes == 4) return norm_rows_kernel<V, 4, 1, 4>;
  if (lanes == 8) return norm_rows_kernel<V, 8, 1, 4>;
  if (lanes == 16) return norm_rows_kernel<V, 16, 1, 4>;
  if (lanes == 32)
    return nv == 1 ? norm_rows_kernel<V, 32, 1, 4> : nv == 2 ? norm_rows_kernel<V, 32, 2, 4>
         : nv == 4 ? norm_rows_kernel<V, 32, 4, 2> : norm_rows_kernel<V, 32, 8, 1>;
  return nv == 2 ? norm_rows_kernel<V, kRowThreads, 2, 1> : nv == 4 ? norm_rows_kernel<V, kRowThreads, 4, 1>
       : norm_rows_kernel<V, kRowThreads, 8, 1>;
}
template <int V>
RowKernel row_backward_kernel(int lanes, int nv) {
  if (lanes == 4) return norm_rows_backward_kernel<V, 4, 1, 4>;
  if (lanes == 8) return norm_rows_backward_kernel<V, 8, 1, 4>;
  if (lanes == 16) return norm_rows_backward_kernel<V, 16, 1, 4>;
  if (lanes == 32)
    return nv == 1 ? norm_rows_backward_kernel<V, 32, 1, 4> : nv == 2 ? norm_rows_backward_kernel<V, 32, 2, 2>
         : nv == 4 ? norm_rows_backward_kernel<V, 32, 4, 1> : norm_rows_backward_kernel<V, 32, 8, 1>;
  return nv == 2 ? norm_rows_backward_kernel<V, kRowThreads, 2, 1>
       : nv == 4 ? norm_rows_backward_kernel<V, kRowThreads, 4, 1> : norm_rows_backward_kernel<V, kRowThreads, 8, 1>;
}

template <int V>
int run_forward(const Norm &a, const Plan &p, cudaStream_t s) {
  if (p.lanes) {
    FZ_CUDA(fz::launch_pdl(row_kernel<V>(p.lanes, p.nv), dim3(p.grid), dim3(kRowThreads), 0, s, a, p.stride));
    FZ_CHECK_LAUNCH();
    return FZ_OK;
  }
  if (p.cluster) return launch_cluster(norm_tile_kernel<V>, p.grid, kTileForward, p.t.k, s, a, p.t);
  if (int rc = launch_cluster(norm_tile_stats_kernel<V>, p.grid, kTileForward, 1, s, a, p.t)) return rc;
  return launch_cluster(norm_tile_apply_kernel<V>, p.grid, kTileForward, 1, s, a, p.t);
}

template <int V>
int run_backward(const Norm &a, const Plan &p, cudaStream_t s) {
  if (p.lanes) {
    FZ_CUDA(fz::launch_pdl(row_backward_kernel<V>(p.lanes, p.nv), dim3(p.grid), dim3(kRowThreads), 0, s, a,
                           p.stride));
    FZ_CHECK_LAUNCH();
    return FZ_OK;
  }
  if (p.cluster) return launch_cluster(norm_tile_backward_kernel<V>, p.grid, kTileBackward, p.t.k, s, a, p.t);
  if (int rc = launch_cluster(norm_tile_sums_kernel<V>, p.grid, kTileBackward, 1, s, a, p.t)) return rc;
  return launch_cluster(norm_tile_dx_kernel<V>, p.grid, kTileBackward, 1, s, a, p.t);
}

int check_sizes(const char *who, int64_t batch, int64_t len, int64_t channels, int64_t groups) {
  const std::string name(who);
  FZ_REQUIRE(batch >= 0 && len >= 0 && channels >= 1 && groups >= 1, name + ": negative or zero size");
  FZ_REQUIRE(channels % groups == 0, name + ": channels must be a multiple of groups");
  FZ_REQUIRE(channels <= INT_MAX && len <= INT_MAX && batch <= INT_MAX, name + ": too many elements");
  FZ_REQUIRE(len == 0 || batch == 0 || (batch <= INT_MAX / len && batch * len <= ((int64_t)1 << 36) / channels),
             name + ": too many elements");
  return FZ_OK;
}

size_t bytes_of(const Plan &p) { return (p.part_floats + p.stat_floats) * sizeof(float); }

}  // namespace

extern "C" int fz_group_norm_workspace(int64_t batch, int64_t len, int64_t channels, int64_t groups, int backward,
                                       size_t *bytes) {
  FZ_REQUIRE(bytes, "fz_group_norm_workspace: null pointer");
  *bytes = 0;
  if (int rc = check_sizes("fz_group_norm_workspace", batch, len, channels, groups)) return rc;
  if (batch == 0 || len == 0) return FZ_OK;
  // whatever the buffers' alignment, and for a forward before the backward on one workspace
  for (int v = 4; v > 0; v /= 2)
    for (int dir = 0; dir <= (backward != 0); ++dir) {
      const size_t n = bytes_of(norm_plan(batch, len, channels, groups, v, dir != 0));
      if (n > *bytes) *bytes = n;
    }
  return FZ_OK;
}

extern "C" int fz_group_norm(float *y, float *mean, float *rstd, const float *x, const float *gamma,
                             const float *beta, int64_t batch, int64_t len, int64_t channels, int64_t groups,
                             float eps, int act, void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check_sizes("fz_group_norm", batch, len, channels, groups)) return rc;
  FZ_REQUIRE(act >= FZ_ACT_NONE && act <= FZ_ACT_GELU, "fz_group_norm: unknown activation");
  FZ_REQUIRE(eps >= 0.0f, "fz_group_norm: eps must not be negative");
  FZ_REQUIRE(!mean == !rstd, "fz_group_norm: mean and rstd are written together");
  if (batch == 0 || len == 0) return FZ_OK;
  FZ_REQUIRE(x && y, "fz_group_norm: null pointer");
  FZ_REQUIRE(x != y, "fz_group_norm: y may not overlap x");
  const Plan p = norm_plan(batch, len, channels, groups, vector_of({x, y, gamma, beta}), false);
  FZ_REQUIRE(bytes_of(p) == 0 || (workspace && workspace_bytes >= bytes_of(p) && (uintptr_t)workspace % 16 == 0),
             "fz_group_norm: workspace too small or not 16-byte aligned");
  Norm a{};
  a.x = x, a.gamma = gamma, a.beta = beta, a.y = y, a.mean = mean, a.rstd = rstd;
  a.stat = (float *)workspace;
  a.batch = batch, a.len = len, a.channels = channels, a.groups = (int)groups, a.c = (int)(channels / groups);
  a.m = (float)(len * a.c), a.eps = eps, a.act = act;
  cudaStream_t s = fz::resolve(stream);
  return p.v == 4 ? run_forward<4>(a, p, s) : p.v == 2 ? run_forward<2>(a, p, s) : run_forward<1>(a, p, s);
}

extern "C" int fz_group_norm_backward(float *dx, float *dgamma, float *dbeta, const float *dy, const float *x,
                                      const float *mean, const float *rstd, const float *gamma, const float *beta,
                                      int64_t batch, int64_t len, int64_t channels, int64_t groups, int act,
                                      void *workspace, size_t workspace_bytes, void *stream) {
  if (int rc = check_sizes("fz_group_norm_backward", batch, len, channels, groups)) return rc;
  FZ_REQUIRE(act >= FZ_ACT_NONE && act <= FZ_ACT_GELU, "fz_group_norm_backward: unknown activation");
  cudaStream_t s = fz::resolve(stream);
  if (batch == 0 || len == 0) {
    for (float *g : {dgamma, dbeta})
      if (g)
        if (int rc = fz_fill_f32(g, 0.0f, channels, stream)) return rc;
    return FZ_OK;
  }
  FZ_REQUIRE(dx && dy && x && mean && rstd, "fz_group_norm_backward: null pointer");
  FZ_REQUIRE(dx != x && dx != dy, "fz_group_norm_backward: dx may not overlap x or dy");
  const Plan p = norm_plan(batch, len, channels, groups, vector_of({x, dy, dx, gamma, beta}), true);
  FZ_REQUIRE(bytes_of(p) == 0 || (workspace && workspace_bytes >= bytes_of(p) && (uintptr_t)workspace % 16 == 0),
             "fz_group_norm_backward: workspace too small or not 16-byte aligned");
  Norm a{};
  a.x = x, a.gamma = gamma, a.beta = beta, a.dy = dy, a.mean_in = mean, a.rstd_in = rstd, a.dx = dx;
  a.stat = (float *)workspace;
  a.part = dgamma || dbeta ? (float *)workspace + p.stat_floats : nullptr;
  a.batch = batch, a.len = len, a.channels = channels, a.groups = (int)groups, a.c = (int)(channels / groups);
  a.m = (float)(len * a.c), a.act = act;
  if (int rc = p.v == 4 ? run_backward<4>(a, p, s) : p.v == 2 ? run_backward<2>(a, p, s) : run_backward<1>(a, p, s))
    return rc;
  if (!a.part) return FZ_OK;
  // CTAs a block of 32 channels: as many as have 4 rows a warp, until the SMs are filled
  const int64_t blocks = up(channels, 32);
  int ctas = 1;
  while (ctas < 8 && blocks * ctas < fz::num_sms() && p.parts * p.part_len > (int64_t)ctas * 2 * kFoldWarps * 4)
    ctas *= 2;
  return launch_cluster(norm_fold_kernel, (unsigned)(blocks * ctas), kFoldWarps * 32, ctas, s, dgamma, dbeta,
                        (const float *)a.part, p.parts, p.part_len, channels, (int)groups, a.c);
}
