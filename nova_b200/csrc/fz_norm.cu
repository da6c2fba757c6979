// Group norm with an activation, channels last, and its gradients.
//
// x is [batch, len, channels]; the team (b, g) is the len x c block of sample b's group g
// of c = channels / groups channels, m = len * c values. Bound by HBM: forward 8 bytes a
// value (read x, write y), backward 12 (read x and dy, write dx), if a team's values are
// read once. So they stay in registers between the statistics and the result, in the
// smallest set of threads that holds a team:
//   * row kernels: a team of at most 256 vectors (of 4, 2 or 1 floats, as alignment
//     allows) is held by 4 to 32 lanes of a warp, of at most 2048 vectors by a CTA;
//   * tile kernels: a tile of rows x columns (several whole groups wide, or a part of
//     one) a CTA; the tiles of a team exchange their statistics through distributed
//     shared memory in one cluster, of up to 16 CTAs. Where c is no multiple of 4 but a row
//     of channels is whole vectors of 4, they may lie across two groups ("mixed":
//     statistics per vector and group, two groups' values spread over a vector). Against
//     vectors that stay in a group, SiLU, forward and backward: [64, 1024, 264] / 8 104 -> 37
//     and 214 -> 88 us, [64, 1024, 120] / 8 32 -> 21 and 55 -> 34 us, [16, 1369, 320] / 32
//     21.5 -> 19 and 37 -> 32 us, [64, 4096, 256] / 128 140 -> 123 and 263 -> 208 us;
//   * larger teams: the tile kernels in two launches that leave the statistics in the
//     workspace (of very many tiles, joined by a launch between them) and read x (and dy)
//     twice; the second launch takes the tiles in reverse, so it finds the last of what the
//     first read in L2. (Taking the batch a few samples at a time instead, so that all of it
//     is found there, cost more in launches than it saved: [8, 16384, 512] 205 against 161 us.)
// Measured (B200, copy bandwidth 6.55 TB/s): rows, [65536, 4096] in 32 groups, GELU: forward
// 378 us, backward 563 us (0.87 of the copy bandwidth both). Clusters, [64, 4096, 256] in 32
// groups, SiLU: forward 98 us (0.84), backward 198 us (0.62: the tiles of x and dy fill the
// registers, and a cluster's CTAs wait for one another). Two launches, [8, 16384, 512]: 152
// and 257 us. A first version with one CTA a team, reading x three times: 566 us for the
// maps' forward, 16.6 ms for the rows' two passes.
// Far from that: short samples, whose tiles are small ([1990, 7, 2368] / 32: 264 and 252 us, 6.6
// and 4.2 times what their bytes take), above all one row of a group of more than 2048 vectors
// ([8192, 16384] in one group 1.23 and 3.22 ms, 7.5 and 13 times; [20000, 4097] 5.05 ms both ways,
// 50 and 34 times), and widths that no vector divides (2.5 to 4 times).
// Statistics: the mean, then the sum of squares about it, so that a common offset of x
// does not cancel; parts are joined as (n, mean, M2) (Chan, Golub and LeVeque). Everything
// is summed in a fixed order.
//
// Backward: with xh and v recomputed from x, dv = dy act'(v) and, per channel,
// sum dv and sum dv xh: these give dbeta and dgamma, and weighted by gamma and summed over
// the group's channels the two sums that dx needs. A thread sees only few channels, whose
// sums it keeps in registers; partial sums (in the row kernels a row a CTA's teams, in the tile
// kernels a row a run of samples and row of tiles) go to the workspace and a last launch adds
// them up: 16 more bytes a value, divided by the rows that a row of sums stands for (three or
// more, and at least 16 for wide groups, once there are many samples).
#include <cooperative_groups.h>

#include <climits>
#include <cstdint>
#include <mutex>
#include <type_traits>

#include "fz_common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRowThreads = 256, kTileThreads = 256;
constexpr int kTileCtas = 2;  // resident an SM
constexpr int kMaxTileGroups = 16;  // groups side by side in a tile
// Vectors of x (backward: of x and of dy) a tile kernel's thread holds: what the registers of
// two CTAs an SM leave.
__host__ __device__ constexpr int held(int v, bool backward) { return (v == 4 ? 16 : 32) / (backward ? 2 : 1); }
// Tiles of at most a half or a quarter of that run in kernels made for it, SHORT = 1 and 2, with 3
// and 4 CTAs an SM: what a tile costs beside its rows is then spread over more of them.
// [1024, 64, 640] / 32, SiLU, 3 rows a thread: forward 222 us with the kernels for 16 rows, 163
// with those for 8, 134 with those for 4; backward 178 with those for 8, 145 with those for 4.
constexpr int kShortest = 2;
constexpr int kMaxCluster = 16;
// Tiles of a group whose statistics every tile of the second launch joins for itself; those of more
// are joined once, by a launch between the two (one group of 32 channels: 131072 rows, 256 tiles,
// 14.8 us without and 15.8 with it; 262144 rows, 24.5 and 23.9; 2^22 rows, 683 and 275; 2^24 rows,
// 14.4 and 1.05 ms).
constexpr int kMostTiles = 256;

// ---------------------------------------------------------------- activations

// They use the hardware's 2^x and reciprocal (2 and 1 ulp) without correcting the argument's
// rounding, and for Phi a polynomial (1.5e-7), because the row kernels issue instructions on 60 % of
// cycles with these alone. Measured against 64 bits, for standard normal v, norm-wise (and with CUDA's
// expf, erfcf and IEEE division in their place): SiLU 4.8e-8 (4.0e-8), its slope 4.9e-8 (4.9e-8), GELU
// 4.4e-8 (3.5e-8), its slope 7.3e-8 (4.6e-8). Far out on the negative side, where the results vanish,
// the exponent's rounding shows: SiLU is off by 9e-7 of itself at -12 (1.9e-7), GELU by 1.5e-6 at -5
// (1.5e-6).
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

// Paired fp32 arithmetic: one instruction for two values, each rounded as the scalar
// instruction rounds. The row kernels would otherwise be bound by instruction issue.
using Pair = unsigned long long;
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(Pair p, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

__device__ __forceinline__ Pair from_lane(Pair a, int mask) { return __shfl_xor_sync(kFull, a, mask); }
template <class F>
__device__ __forceinline__ Pair each(F f, Pair v) {
  float a, b;
  unpair(v, a, b);
  return pair(f(a), f(b));
}
template <class F>
__device__ __forceinline__ Pair each(F f, Pair v, Pair w, Pair x) {
  float a, b, c, d, g, h;
  unpair(v, a, b);
  unpair(w, c, d);
  unpair(x, g, h);
  return pair(f(a, c, g), f(b, d, h));
}
// The same for a value of its own, where no vector of two is possible.
struct One {
  float f;
};
__device__ __forceinline__ One add2(One a, One b) { return {__fadd_rn(a.f, b.f)}; }
__device__ __forceinline__ One mul2(One a, One b) { return {__fmul_rn(a.f, b.f)}; }
__device__ __forceinline__ One fma2(One a, One b, One c) { return {__fmaf_rn(a.f, b.f, c.f)}; }
__device__ __forceinline__ One from_lane(One a, int mask) { return {__shfl_xor_sync(kFull, a.f, mask)}; }
template <class F>
__device__ __forceinline__ One each(F f, One v) {
  return {f(v.f)};
}
template <class F>
__device__ __forceinline__ One each(F f, One v, One w, One x) {
  return {f(v.f, w.f, x.f)};
}
template <class E>
__device__ __forceinline__ E both(float a) {
  if constexpr (std::is_same_v<E, One>) return {a};
  else return pair(a, a);
}

template <class E>
__device__ __forceinline__ E sigmoid2(E v) {
  const E e = each([](float a) { return ex2(a); }, mul2(v, both<E>(-1.4426950408889634f)));
  return each([](float a) { return rcp(a); }, add2(e, both<E>(1.0f)));
}

// Phi(v) and exp(-v^2 / 2). With h = Phi(-|v|) = exp(-v^2 / 2) R(t), t = 1 / (1 + 0.3 |v|):
// R is a polynomial of degree 8 without constant term, fitted to the least largest relative
// error on |v| <= 14 (Remez; 1.5e-7).
template <class E>
__device__ __forceinline__ E phi2(E v, E *e) {
  const E c = fma2(each([](float a) { return fabsf(a); }, v), both<E>(0.3f), both<E>(1.0f));
  const E t = each([](float a) { return rcp(a); }, c);
  *e = each([](float a) { return ex2(a); }, mul2(mul2(v, v), both<E>(-0.72134752044448170f)));
  E r = fma2(both<E>(0.035674769431352615f), t, both<E>(-0.1572030633687973f));
  r = fma2(r, t, both<E>(0.20635347068309784f));
  r = fma2(r, t, both<E>(-0.05368361622095108f));
  r = fma2(r, t, both<E>(0.1285616159439087f));
  r = fma2(r, t, both<E>(0.09991349279880524f));
  r = fma2(r, t, both<E>(0.12075395882129669f));
  r = fma2(r, t, both<E>(0.11962930113077164f));
  const E h = mul2(mul2(r, t), *e);
  // NaN: both are
  return each([](float a, float low, float high) { return a < 0.0f ? low : high; }, v, h,
              fma2(h, both<E>(-1.0f), both<E>(1.0f)));
}

template <int ACT, class E>
__device__ __forceinline__ E activate2(E v) {
  if constexpr (ACT == FZ_ACT_SILU) return mul2(v, sigmoid2(v));
  if constexpr (ACT == FZ_ACT_GELU) {
    E e;
    return mul2(v, phi2(v, &e));
  }
  if constexpr (ACT == FZ_ACT_RELU) return each([](float a) { return a > 0.0f ? a : 0.0f; }, v);
  return v;
}

// d act'(v)
template <int ACT, class E>
__device__ __forceinline__ E times_slope2(E d, E v) {
  if constexpr (ACT == FZ_ACT_SILU) {
    const E s = sigmoid2(v), rest = fma2(s, both<E>(-1.0f), both<E>(1.0f));
    return mul2(d, mul2(s, fma2(v, rest, both<E>(1.0f))));
  }
  if constexpr (ACT == FZ_ACT_GELU) {
    E e;
    const E p = phi2(v, &e);
    return mul2(d, fma2(mul2(v, both<E>(0.39894228040143268f)), e, p));
  }
  if constexpr (ACT == FZ_ACT_RELU) return each([](float a, float x, float) { return a > 0.0f ? x : 0.0f; }, v, d, d);
  return d;
}

// f(Act<ACT>) for the activation of the call: chosen once around a loop, not in it.
template <int ACT>
struct Act {
  static constexpr int value = ACT;
};
template <class F>
__device__ __forceinline__ void with_activation(int act, F f) {
  switch (act) {
    case FZ_ACT_RELU: f(Act<FZ_ACT_RELU>{}); break;
    case FZ_ACT_SILU: f(Act<FZ_ACT_SILU>{}); break;
    case FZ_ACT_GELU: f(Act<FZ_ACT_GELU>{}); break;
    default: f(Act<FZ_ACT_NONE>{}); break;
  }
}

// ---------------------------------------------------------------- vectors

// V floats in registers as pairs, or a float. ([2922, 1082, 31] in one group, SiLU: 374 and 751 us
// with a float as a pair with an idle half, 322 and 464 so.)
template <int V>
struct Vec {
  using E = std::conditional_t<V == 1, One, Pair>;
  static constexpr int N = V == 4 ? 2 : 1;
  E p[N];
};
template <int V>
__device__ __forceinline__ Vec<V> splat(float a) {
  Vec<V> r;
  const auto p = both<typename Vec<V>::E>(a);
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i) r.p[i] = p;
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> load(const float *q) {
  Vec<V> r;
  if constexpr (V == 4) {
    const float4 f = *reinterpret_cast<const float4 *>(q);
    r.p[0] = pair(f.x, f.y);
    r.p[1] = pair(f.z, f.w);
  } else if constexpr (V == 2) {
    const float2 f = *reinterpret_cast<const float2 *>(q);
    r.p[0] = pair(f.x, f.y);
  } else {
    r.p[0] = {*q};
  }
  return r;
}
template <int V>
__device__ __forceinline__ void store(float *q, const Vec<V> &r) {
  if constexpr (V == 1) {
    *q = r.p[0].f;
  } else {
    float a, b, c, d;
    unpair(r.p[0], a, b);
    if constexpr (V == 4) {
      unpair(r.p[1], c, d);
      *reinterpret_cast<float4 *>(q) = make_float4(a, b, c, d);
    } else {
      *reinterpret_cast<float2 *>(q) = make_float2(a, b);
    }
  }
}
template <int V>
__device__ __forceinline__ Vec<V> load_or(const float *q, float otherwise) {
  return q ? load<V>(q) : splat<V>(otherwise);
}
// Tiles are fetched ahead through shared memory that each thread has to itself: it copies
// the vectors that it will process a few tiles later, asynchronously, waits for its own
// copies and reads them back, so no barrier is needed and no registers are held meanwhile.
template <int V>
__device__ __forceinline__ void copy_async(float *to, const float *from) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (V == 4) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  else if constexpr (V == 2) asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The sum of a vector's values.
template <int V>
__device__ __forceinline__ float total(const Vec<V> &r) {
  if constexpr (V == 1) {
    return r.p[0].f;
  } else {
    float a, b;
    unpair(V == 4 ? add2(r.p[0], r.p[Vec<V>::N - 1]) : r.p[0], a, b);
    return __fadd_rn(a, b);
  }
}
// s += x; s += (x - mean)^2
template <int V>
__device__ __forceinline__ void sum_into(Vec<V> &s, const Vec<V> &x) {
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i) s.p[i] = add2(s.p[i], x.p[i]);
}
template <int V>
__device__ __forceinline__ void square_into(Vec<V> &s, const Vec<V> &x, const Vec<V> &minus_mean) {
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i) {
    const auto d = add2(x.p[i], minus_mean.p[i]);
    s.p[i] = fma2(d, d, s.p[i]);
  }
}
// act(gamma (x - mean) rstd + beta)
template <int ACT, int V>
__device__ __forceinline__ Vec<V> normalize(const Vec<V> &x, const Vec<V> &minus_mean, const Vec<V> &rstd,
                                            const Vec<V> &gamma, const Vec<V> &beta) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i)
    r.p[i] = activate2<ACT>(fma2(mul2(add2(x.p[i], minus_mean.p[i]), rstd.p[i]), gamma.p[i], beta.p[i]));
  return r;
}
// x <- xh, d <- dv gamma; dv and dv xh are added to db and dg
template <int ACT, int V>
__device__ __forceinline__ void gradient(Vec<V> &x, Vec<V> &d, Vec<V> &db, Vec<V> &dg, const Vec<V> &minus_mean,
                                         const Vec<V> &rstd, const Vec<V> &gamma, const Vec<V> &beta) {
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i) {
    x.p[i] = mul2(add2(x.p[i], minus_mean.p[i]), rstd.p[i]);
    const auto dv = times_slope2<ACT>(d.p[i], fma2(x.p[i], gamma.p[i], beta.p[i]));
    db.p[i] = add2(db.p[i], dv);
    dg.p[i] = fma2(dv, x.p[i], dg.p[i]);
    d.p[i] = mul2(dv, gamma.p[i]);
  }
}
// rstd (d - k1 - xh k2)
template <int V>
__device__ __forceinline__ Vec<V> finish(const Vec<V> &xh, const Vec<V> &d, const Vec<V> &minus_k1,
                                         const Vec<V> &minus_k2, const Vec<V> &rstd) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < Vec<V>::N; ++i)
    r.p[i] = mul2(rstd.p[i], fma2(xh.p[i], minus_k2.p[i], add2(d.p[i], minus_k1.p[i])));
  return r;
}

__device__ __forceinline__ float rstd_of(float m2, float inv_m, float eps) {
  return rsqrtf(__fmaf_rn(m2, inv_m, eps));
}

struct Norm {
  const float *x, *gamma, *beta;
  float *y, *mean, *rstd;
  const float *dy, *mean_in, *rstd_in;
  float *dx;
  float *part;  // per-channel partial sums, or null: [part][2][...]
  float *stat;  // two-launch tiles: statistics of a group's tiles
  float2 *whole;  // and, of many tiles, those of the group, or null
  int64_t batch, len, channels;
  int groups, c;  // c: channels a group
  float m, inv_m, eps;  // inv_m = 1 / m
  int act;
  int *err;  // tiles in a cluster: where a wait that gave up is recorded
};

// ---------------------------------------------------------------- row kernels

// The sums of U values each over the P lanes (or, P = kRowThreads and U = 1, threads) of a
// team. Four values go through one butterfly: after the two steps that halve how many
// values a lane carries, lane l holds (a part of) value which(l), and `done` of its whole
// sum is computed once for it; every lane then fetches all U.
template <int P, int U, class Done>
__device__ __forceinline__ void team_sums(float (&v)[U], float *sh, Done done) {
  const int lane = threadIdx.x & 31;
  if constexpr (U == 4 && P <= 32) {
    const bool hi = lane & (P / 2), lo = lane & (P / 4);
    float a = __fadd_rn(hi ? v[2] : v[0], __shfl_xor_sync(kFull, hi ? v[0] : v[2], P / 2));
    float b = __fadd_rn(hi ? v[3] : v[1], __shfl_xor_sync(kFull, hi ? v[1] : v[3], P / 2));
    a = __fadd_rn(lo ? b : a, __shfl_xor_sync(kFull, lo ? a : b, P / 4));
#pragma unroll
    for (int d = P / 8; d > 0; d >>= 1) a = __fadd_rn(a, __shfl_xor_sync(kFull, a, d));
    a = done(a);
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = __shfl_sync(kFull, a, (u >> 1) * (P / 2) + (u & 1) * (P / 4), P);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int d = (P < 32 ? P : 32) / 2; d > 0; d >>= 1) v[u] = __fadd_rn(v[u], __shfl_xor_sync(kFull, v[u], d));
      if constexpr (P > 32) {
        __syncthreads();
        if (lane == 0) sh[threadIdx.x >> 5] = v[u];
        __syncthreads();
        v[u] = sh[0];
#pragma unroll
        for (int w = 1; w < P / 32; ++w) v[u] = __fadd_rn(v[u], sh[w]);
      }
      v[u] = done(v[u]);
    }
  }
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
// gamma and beta of a lane's vectors: in registers where there are few, else from L1
template <int V, int NV>
struct Affine {
  static constexpr bool kKeep = NV <= 2;
  Vec<V> gamma[kKeep ? NV : 1], beta[kKeep ? NV : 1];
  __device__ Affine(const Norm &a, const int (&channel)[NV]) {
    if constexpr (kKeep)
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        gamma[i] = load_or<V>(a.gamma ? a.gamma + channel[i] : nullptr, 1.0f);
        beta[i] = load_or<V>(a.beta ? a.beta + channel[i] : nullptr, 0.0f);
      }
  }
  __device__ __forceinline__ void get(const Norm &a, const int (&channel)[NV], int i, Vec<V> &ga, Vec<V> &be) const {
    if constexpr (kKeep) {
      ga = gamma[i];
      be = beta[i];
    } else {
      ga = load_or<V>(a.gamma ? a.gamma + channel[i] : nullptr, 1.0f);
      be = load_or<V>(a.beta ? a.beta + channel[i] : nullptr, 0.0f);
    }
  }
};

// The row kernels' shape by vectors a lane: teams in flight U, resident CTAs an SM, and
// stages fetched ahead (about 190 KB an SM in all).
__host__ __device__ constexpr int row_u(int p, int nv) { return p > 32 ? 1 : nv == 1 ? 4 : nv == 2 ? 2 : 1; }
__host__ __device__ constexpr int row_ctas(bool backward, int nv) {
  return backward ? (nv == 8 ? 1 : 2) : 3;
}
__host__ __device__ constexpr int row_stages(bool backward, int nv) { return backward ? 3 : nv == 8 ? 2 : 4; }
__host__ __device__ constexpr int row_smem(bool backward, int p, int nv, int v) {
  return row_stages(backward, nv) * (backward ? 2 : 1) * kRowThreads * row_u(p, nv) * nv * v * 4;
}

template <int V, int P, int NV>
__global__ void __launch_bounds__(kRowThreads, row_ctas(false, NV)) norm_rows_kernel(const Norm a, int stride) {
  pdl_wait();
  constexpr int U = row_u(P, NV), S = row_stages(false, NV);
  extern __shared__ __align__(16) float fifo[];  // [S][U][NV][threads] vectors
  __shared__ float sh[kRowThreads / 32];
  const RowTeam<V, P, NV> t(a, stride);
  const Affine<V, NV> affine(a, t.channel);
  const int parts = stride / a.groups, step = parts * U, batch = t.on ? (int)a.batch : 0;
  const int64_t hop = (int64_t)parts * a.len * a.channels;  // floats from one team in flight to the next
  const int64_t first = (int64_t)t.part * a.len * a.channels + (int64_t)t.g * a.c;
  const float *from = a.x + first;
  float *to = a.y + first;
  int64_t team = (int64_t)t.part * a.groups + t.g;
  float *mine = fifo + (int)threadIdx.x * V;
  const auto fetch = [&](int s, int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u * parts < batch)
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (t.at[i] >= 0) copy_async<V>(mine + ((s * U + u) * NV + i) * kRowThreads * V, from + t.at[i]);
      from += hop;
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, t.part + s * step);
  int s = 0;
  for (int b0 = 0; b0 < (int)a.batch; b0 += step, s = s + 1 < S ? s + 1 : 0) {
    const int b = b0 + t.part;
    Vec<V> x[U][NV];
    float mean[U], rstd[U];
    copy_wait<S - 1>();
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NV; ++i)
        x[u][i] = b + u * parts < batch && t.at[i] >= 0
                      ? load<V>(mine + ((s * U + u) * NV + i) * kRowThreads * V)
                      : splat<V>(0.0f);
    fetch(s, b + S * step);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<V> q = x[u][0];
#pragma unroll
      for (int i = 1; i < NV; ++i) sum_into(q, x[u][i]);
      mean[u] = total(q);
    }
    team_sums<P, U>(mean, sh, [&](float v) { return __fdiv_rn(v, a.m); });  // exact for a constant
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<V> q = splat<V>(0.0f);
      const Vec<V> minus = splat<V>(-mean[u]);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t.at[i] >= 0) square_into(q, x[u][i], minus);
      rstd[u] = total(q);
    }
    team_sums<P, U>(rstd, sh, [&](float v) { return rstd_of(v, a.inv_m, a.eps); });
    with_activation(a.act, [&](auto act) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (b + u * parts < batch) {
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (t.at[i] >= 0) {
              Vec<V> ga, be;
              affine.get(a, t.channel, i, ga, be);
              store(to + u * hop + t.at[i],
                    normalize<decltype(act)::value>(x[u][i], splat<V>(-mean[u]), splat<V>(rstd[u]), ga, be));
            }
        }
      }
    });
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (a.mean && threadIdx.x % P == 0 && b + u * parts < batch) {
        a.mean[team + (int64_t)u * stride] = mean[u];
        a.rstd[team + (int64_t)u * stride] = rstd[u];
      }
    to += U * hop;
    team += (int64_t)U * stride;
  }
  copy_wait<0>();
}

// Sums of many terms are taken in two levels, so that their rounding errors grow with the number of
// blocks of kNear terms and not with that of the terms.
constexpr int kNear = 16;

// fold: teams of a CTA that share a group and whose channel sums are added up in the CTA.
template <int V, int P, int NV>
__global__ void __launch_bounds__(kRowThreads, row_ctas(true, NV))
    norm_rows_backward_kernel(const Norm a, int stride, int fold) {
  pdl_wait();
  constexpr int U = row_u(P, NV), S = row_stages(true, NV);
  extern __shared__ __align__(16) float fifo[];  // [S][2][U][NV][threads] vectors, then the CTA's channel sums
  __shared__ float sh[kRowThreads / 32];
  const RowTeam<V, P, NV> t(a, stride);
  const Affine<V, NV> affine(a, t.channel);
  const int parts = stride / a.groups, step = parts * U, batch = t.on ? (int)a.batch : 0;
  const int64_t hop = (int64_t)parts * a.len * a.channels;
  const int64_t first = (int64_t)t.part * a.len * a.channels + (int64_t)t.g * a.c;
  const float *from_x = a.x + first, *from_d = a.dy + first;
  float *to = a.dx + first;
  int64_t team = (int64_t)t.part * a.groups + t.g;
  float *mine = fifo + (int)threadIdx.x * V;
  const auto fetch = [&](int s, int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (b + u * parts < batch)
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (t.at[i] >= 0) {
            copy_async<V>(mine + ((s * 2 * U + u) * NV + i) * kRowThreads * V, from_x + t.at[i]);
            copy_async<V>(mine + (((s * 2 + 1) * U + u) * NV + i) * kRowThreads * V, from_d + t.at[i]);
          }
      from_x += hop;
      from_d += hop;
    }
    copy_commit();
  };
  float next_mean[U], next_rstd[U];
  const auto fetch_stats = [&](int b) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      next_mean[u] = b + u * parts < batch ? a.mean_in[team] : 0.0f;
      next_rstd[u] = b + u * parts < batch ? a.rstd_in[team] : 0.0f;
      team += stride;
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(s, t.part + s * step);
  fetch_stats(t.part);
  Vec<V> db[NV], dg[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) db[i] = dg[i] = splat<V>(0.0f);
  // The sums of earlier blocks of steps. Four and eight vectors of 4 a lane leave no registers for
  // them: there they stay in memory (the asm hides where `sums` points), and a block has 64 steps,
  // for a block's end stops the stream of loads for 5 us ([16384, 8192] in one group: 463 us with
  // one block, 507 with blocks of 16).
  constexpr bool kInMemory = V == 4 && NV > 2;
  constexpr int kBlock = kInMemory ? 64 : kNear;
  Vec<V> blocks[2 * NV], *sums = blocks;
  if constexpr (kInMemory) asm volatile("" : "+l"(sums)::"memory");
  bool carried = false;
  const auto carry = [&](bool last) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (carried) {
        sum_into(db[i], sums[2 * i]);
        sum_into(dg[i], sums[2 * i + 1]);
      }
      if (!last) {
        sums[2 * i] = db[i];
        sums[2 * i + 1] = dg[i];
        db[i] = dg[i] = splat<V>(0.0f);
      }
    }
    carried = true;
  };
  int s = 0;
  for (int b0 = 0; b0 < (int)a.batch;) {
    if (b0) carry(false);
    const int end = (int)min((int64_t)a.batch, b0 + (int64_t)kBlock * step);
#pragma unroll 1
    for (; b0 < end; b0 += step, s = s + 1 < S ? s + 1 : 0) {
      const int b = b0 + t.part;
      Vec<V> x[U][NV], d[U][NV];
      float rstd[U], s1[U], s2[U];
      float minus[U];
      copy_wait<S - 1>();
#pragma unroll
      for (int u = 0; u < U; ++u) {
        minus[u] = -next_mean[u];
        rstd[u] = next_rstd[u];
        s1[u] = s2[u] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const bool in = b + u * parts < batch && t.at[i] >= 0;
          x[u][i] = in ? load<V>(mine + ((s * 2 * U + u) * NV + i) * kRowThreads * V) : splat<V>(0.0f);
          d[u][i] = in ? load<V>(mine + (((s * 2 + 1) * U + u) * NV + i) * kRowThreads * V) : splat<V>(0.0f);
        }
      }
      fetch(s, b + S * step);
      fetch_stats(b + step);
      with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (t.at[i] < 0) continue;
          Vec<V> ga, be, b_sum = splat<V>(0.0f), g_sum = b_sum;  // of U teams, then of all
          affine.get(a, t.channel, i, ga, be);
#pragma unroll
          for (int u = 0; u < U; ++u) {
            // behind the batch x, d, mean and rstd are 0, and so is all that they give
            gradient<decltype(act)::value>(x[u][i], d[u][i], b_sum, g_sum, splat<V>(minus[u]), splat<V>(rstd[u]), ga, be);
            Vec<V> w;
#pragma unroll
            for (int j = 0; j < Vec<V>::N; ++j) w.p[j] = mul2(d[u][i].p[j], x[u][i].p[j]);
            s1[u] = __fadd_rn(s1[u], total(d[u][i]));
            s2[u] = __fadd_rn(s2[u], total(w));
          }
          sum_into(db[i], b_sum);
          sum_into(dg[i], g_sum);
        }
      });
      const auto over_m = [&](float v) { return __fmul_rn(v, -a.inv_m); };
      team_sums<P, U>(s1, sh, over_m);
      team_sums<P, U>(s2, sh, over_m);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (b + u * parts < batch)
#pragma unroll
          for (int i = 0; i < NV; ++i)
            if (t.at[i] >= 0)
              store(to + t.at[i], finish(x[u][i], d[u][i], splat<V>(s1[u]), splat<V>(s2[u]), splat<V>(rstd[u])));
        to += hop;
      }
    }
  }
  copy_wait<0>();
  if (!a.part) return;
  carry(true);
  // Per channel, over the rows of the sample and the CTA's `fold` teams of the group, in
  // order: part[row][2][channels]. The teams' sums (at most 8192 floats) take the place of
  // the first stage.
  constexpr int kTeams = kRowThreads / P;
  const int id0 = (int)blockIdx.x * kTeams, wide = (int)a.len * a.c;
  float *own = fifo + (int)(threadIdx.x / P) * wide;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t.at[i] >= 0) store(own + (i * P + (int)(threadIdx.x % P)) * V, which ? dg[i] : db[i]);
    __syncthreads();
    const int first = kTeams / fold;  // teams with channels of their own
    for (int i = threadIdx.x; i < first * a.c; i += kRowThreads) {
      const int team = i / a.c, ch = i - team * a.c, id = id0 + team;
      if (id >= stride) break;
      float sum = 0.0f;
      for (int f = 0; f < fold; ++f)
        for (int l = 0; l < (int)a.len; ++l) sum = __fadd_rn(sum, fifo[(team + f * first) * wide + l * a.c + ch]);
      const int row = id / (a.groups * fold), g = id % a.groups;
      a.part[((int64_t)row * 2 + which) * a.channels + (int64_t)g * a.c + ch] = sum;
    }
  }
}

// ---------------------------------------------------------------- tile kernels

// How a launch cuts samples into tiles (see norm_plan).
struct Tiling {
  int cols;      // vectors a tile is wide
  int wide;      // thread columns: cols, or the next power of two
  int tall;      // thread rows: as many as fit
  int slices;    // of the thread rows: those of a warp where it holds whole ones (wide
  int each;      // divides 32), else one thread row each; the thread rows of a slice
  int q;         // whole groups a tile holds (1 where a group is split)
  int split;     // tiles a group's columns are split into
  int bundles;   // tiles side by side over a sample's groups (without the split)
  int rows;      // rows a tile
  int chunks;    // tiles one below the other
  int k;         // tiles that share statistics: split * chunks
  int run;       // samples whose tiles at one place a CTA takes one after the other
  int units;     // the pieces of work that leaves: runs of a set's tiles (in a cluster) or of one
};

// How a tile kernel gets the statistics of a set of tiles: kInCluster, one cluster a set
// (k <= 16 tiles), each CTA pushing its share to all of them; or in two launches, kParts
// leaving each tile's in the workspace and kWhole joining them. CTAs (clusters) are
// resident and go through the tiles (sets) in turn, the next tile fetched ahead, so its
// loads run while a set waits for its statistics.
enum : int { kInCluster = 0, kParts = 1, kWhole = 2 };

// One tile, as a thread sees it.
template <int V>
struct Tile {
  int b, chunk, k;
  int g0, q, cols;  // its first group, its groups, its vectors a row
  int rows, mine;   // its rows, and those of this thread (0: none)
  int most;         // rows of the thread that has most
  int full, rest;   // rows = full * thread rows + rest
  int channel;      // this thread's first channel
  int64_t at;       // offset of this thread's first vector
  int row;          // where the run's parameter sums go
  bool begins, ends;  // the run
};

// The groups (counted from the tile's first) of a thread's vector: values before `from` belong
// to lo, the others to hi. Only mixed vectors (V = 4, c >= 2) have two.
template <int V, bool MIXED>
struct Place {
  int lo, hi, from;
  __device__ Place(const Norm &a, const Tiling &t, int tx) {
    if (MIXED) {
      lo = tx * V / a.c;
      hi = (tx * V + V - 1) / a.c;
      from = hi * a.c - tx * V;  // 0 or less: the whole vector is hi's
    } else {
      lo = hi = t.split > 1 ? 0 : tx / (a.c / V);
      from = V;
    }
  }
  // the sums over a vector's values of each group
  __device__ __forceinline__ void gather(const Vec<V> &x, float &l, float &h) const {
    float f[4];
    unpair(x.p[0], f[0], f[1]);
    unpair(x.p[Vec<V>::N - 1], f[2], f[3]);
    l = h = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      l = __fadd_rn(l, j < from ? f[j] : 0.0f);
      h = __fadd_rn(h, j < from ? 0.0f : f[j]);
    }
  }
  __device__ __forceinline__ Vec<V> spread(float l, float h) const {
    if constexpr (MIXED) {
      Vec<V> r;
      r.p[0] = pair(0 < from ? l : h, 1 < from ? l : h);
      r.p[Vec<V>::N - 1] = pair(2 < from ? l : h, 3 < from ? l : h);
      return r;
    } else {
      return splat<V>(l);
    }
  }
};

// A CTA's walk over the tiles: (run of samples, bundle, share) counted in mixed radix, since a
// division a tile costs as much as a good part of its arithmetic, and the samples of each run.
// kWhole walks from the last tile. RUNS: runs may be of more than one sample; kernels for those are
// apart ([1024, 64, 640] / 32, backward: 149 us with their walk and sums and runs of one, 140 so).
template <int V, int MODE, bool MIXED, bool RUNS = false>
struct Walk {
  int block, in_run, bundle, share, dblock, dbundle, dshare, left;  // left: units, this one included
  int tx, ty;       // thread column and row; past the last row: a row that no tile has
  int slice;        // its thread row's
  bool leaves;      // this thread leaves its column's share of its slice
  unsigned invert;  // by which to multiply instead of dividing by the thread rows
  __device__ Walk(const Tiling &t, int rank) {
    const int k = MODE == kInCluster ? 1 : t.k;
    const int first = MODE == kInCluster ? (int)blockIdx.x / t.k : (int)blockIdx.x;
    const int step = MODE == kInCluster ? (int)gridDim.x / t.k : (int)gridDim.x;
    left = first < t.units ? (t.units - 1 - first) / step + 1 : 0;
    share = MODE == kInCluster ? rank : first % k;
    bundle = first / k % t.bundles;
    block = first / k / t.bundles;
    in_run = 0;
    dshare = MODE == kInCluster ? 0 : step % k;
    dbundle = step / k % t.bundles;
    dblock = step / k / t.bundles;
    ty = (int)threadIdx.x / t.wide;
    tx = (int)threadIdx.x - ty * t.wide;
    slice = ty / t.each;
    leaves = ty < t.tall && ty == slice * t.each;
    if (ty >= t.tall) ty = INT_MAX;
    invert = (1u << 22) / t.tall + 1;
  }
  // x / tall: exact, since x <= 32 tall and 32 tall^2 <= 2^21
  __device__ int over_tall(int x) const { return (int)((unsigned)x * invert >> 22); }
  __device__ void advance(const Norm &a, const Tiling &t) {
    if (RUNS) {
      if (++in_run < t.run && block * t.run + in_run < (int)a.batch) return;
      in_run = 0;
    }
    --left;
    int carry = 0;
    if (MODE != kInCluster) {
      share += dshare;
      carry = share >= t.k;
      share -= carry ? t.k : 0;
    }
    bundle += dbundle + carry;
    carry = bundle >= t.bundles;
    bundle -= carry ? t.bundles : 0;
    block += dblock + carry;
  }
  __device__ Tile<V> get(const Norm &a, const Tiling &t) const {
    Tile<V> r;
    const bool back = MODE == kWhole;
    const int at = back ? t.bundles - 1 - bundle : bundle, b = RUNS ? block * t.run + in_run : block;
    r.b = back ? (int)a.batch - 1 - b : b;
    r.begins = !RUNS || in_run == 0;
    r.ends = !RUNS || in_run + 1 == t.run || b + 1 == (int)a.batch;
    r.k = back ? t.k - 1 - share : share;
    r.chunk = t.split > 1 ? r.k / t.split : r.k;
    r.row = block * t.chunks + r.chunk;
    const int piece = r.k - r.chunk * t.split;
    r.g0 = at * t.q;
    r.q = min(t.q, a.groups - r.g0);
    r.cols = t.split > 1 ? min(t.cols, a.c / V - piece * t.cols) : MIXED ? r.q * a.c / V : r.q * (a.c / V);
    const int64_t row0 = (int64_t)r.chunk * t.rows;
    r.rows = (int)min((int64_t)t.rows, a.len - row0);
    r.channel = r.g0 * a.c + (piece * t.cols + tx) * V;
    r.mine = tx < r.cols && ty < r.rows ? over_tall(r.rows - 1 - ty) + 1 : 0;
    r.full = over_tall(r.rows);
    r.rest = r.rows - r.full * t.tall;
    r.most = r.full + (r.rest > 0);
    r.at = (r.b * a.len + row0 + ty) * a.channels + r.channel;
    return r;
  }
};

// Values of one group in tile `k` of a set.
__device__ __forceinline__ float count_of(const Norm &a, const Tiling &t, int k, int v) {
  const int chunk = t.split > 1 ? k / t.split : k, piece = k - chunk * t.split;
  const float rows = (float)min((int64_t)t.rows, a.len - (int64_t)chunk * t.rows);
  return rows * (float)(t.split > 1 ? min(t.cols, a.c / v - piece * t.cols) * v : a.c);
}

// The loops over a thread's rows end, four rows at a time, behind the tile's last, so that a
// short tile costs what it has: [2048, 64, 40] / 4 in vectors of 2, forward 57 -> 40 us, backward
// 69 -> 44 us; [16, 1369, 320] / 32, backward 38 -> 35 us. A forward of vectors of 4
// runs all of its rows: with the branches between its loads and sums, [64, 1024, 264] / 8 took
// 43 us instead of 37, [4096, 40, 52] / 4 49 instead of 57.
template <int V, int N>
__device__ __forceinline__ bool behind(int i, const Tile<V> &me) {
  return (V < 4 || N < held(4, false)) && i % 4 == 0 && i >= me.most;
}

// A tile's vectors to a thread's place in shared memory ([held][threads] vectors), and back.
// Behind a thread's rows they are 0, or what is given (apart from one another: with a 0 that is
// given, [114, 53, 2720] / 16 in vectors of 2 took 53 us forward instead of 46).
template <int V, int N>
__device__ __forceinline__ void fetch_tile(float *fifo, const float *p, const Tile<V> &me, int64_t step) {
  const float *q = p + me.at;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (behind<V, N>(i, me)) break;
    if (i < me.mine) copy_async<V>(fifo + (i * kTileThreads + (int)threadIdx.x) * V, q);
    q += step;
  }
}
template <int V, int N>
__device__ __forceinline__ void take_tile(Vec<V> (&x)[N], const float *fifo, const Tile<V> &me) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (behind<V, N>(i, me)) break;
    x[i] = i < me.mine ? load<V>(fifo + (i * kTileThreads + (int)threadIdx.x) * V) : splat<V>(0.0f);
  }
}
template <int V, int N>
__device__ __forceinline__ void take_tile(Vec<V> (&x)[N], const float *fifo, const Tile<V> &me,
                                          const Vec<V> &none) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (behind<V, N>(i, me)) break;
    x[i] = i < me.mine ? load<V>(fifo + (i * kTileThreads + (int)threadIdx.x) * V) : none;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kFull, v, d));
  return v;
}

// The sum of v over the thread rows of a slice that is a warp's.
__device__ __forceinline__ float over_rows(float v, int each) {
  for (int d = 16; d * each > 16; d >>= 1) v = __fadd_rn(v, __shfl_xor_sync(kFull, v, d));
  return v;
}
// Rows of the tile that slice y holds.
template <int V>
__device__ __forceinline__ int rows_of_slice(int y, const Tile<V> &me, const Tiling &t) {
  return me.full * t.each + min(max(me.rest - y * t.each, 0), t.each);
}

// The tile's own moments. column_moments: each slice reduces a column (mixed: its values of
// each group) to its mean and the sum of squares about it, with a barrier at the end.
// group_moments: (mean, M2) of group g in every lane of the warp that asks, M2 = sum of theirs
// + n_column (mean_column - mean)^2. sh: [slices][wide], mixed [slices][wide][2].
template <int V, int MODE, bool MIXED, int N>
__device__ __forceinline__ void column_moments(const Vec<V> (&x)[N], float2 *sh, const Tile<V> &me, const Tiling &t,
                                               const Walk<V, MODE, MIXED> &walk, const Place<V, MIXED> &place) {
  Vec<V> s = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) {
    if (behind<V, N>(i, me)) break;
    sum_into(s, x[i]);
  }
  const int rows = rows_of_slice(walk.slice, me, t);  // 0: nothing of this slice is read
  const int at = walk.slice * t.wide + walk.tx;
  if constexpr (MIXED) {
    float lo, hi;
    place.gather(s, lo, hi);
    const float mean_lo = __fdiv_rn(over_rows(lo, t.each), (float)(rows * max(place.from, 1)));
    const float mean_hi = __fdiv_rn(over_rows(hi, t.each), (float)(rows * (V - max(place.from, 0))));
    const Vec<V> minus = place.spread(-mean_lo, -mean_hi);
    s = splat<V>(0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (behind<V, N>(i, me)) break;
      if (i < me.mine) square_into(s, x[i], minus);
    }
    place.gather(s, lo, hi);
    lo = over_rows(lo, t.each);
    hi = over_rows(hi, t.each);
    if (walk.leaves) *reinterpret_cast<float4 *>(sh + at * 2) = make_float4(mean_lo, lo, mean_hi, hi);
  } else {
    const float mean = __fdiv_rn(over_rows(total(s), t.each), (float)(rows * V));
    const Vec<V> minus = splat<V>(-mean);
    s = splat<V>(0.0f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (behind<V, N>(i, me)) break;
      if (i < me.mine) square_into(s, x[i], minus);
    }
    const float m2 = over_rows(total(s), t.each);
    if (walk.leaves) sh[at] = make_float2(mean, m2);
  }
  __syncthreads();
}
template <int V, bool MIXED>
__device__ __forceinline__ float2 group_moments(const float2 *sh, int g, const Norm &a, const Tile<V> &me,
                                                const Tiling &t) {
  const int lane = threadIdx.x & 31, begin = g * a.c, end = begin + a.c;  // channels
  const int first = begin / V, width = t.split > 1 ? me.cols : MIXED ? (end - 1) / V - first + 1 : a.c / V;
  const int total = t.slices * width, dy = 32 / width, dc = 32 - dy * width;
  const int y0 = lane / width, c0 = lane - y0 * width;
  const auto each = [&](auto f) {  // f(values, their mean and M2) for this lane's entries
    for (int i = lane, y = y0, c = c0; i < total; i += 32) {
      const int col = first + c;
      const int values = MIXED ? min(col * V + V, end) - max(col * V, begin) : V;
      const int n = rows_of_slice(y, me, t) * values;
      // a mixed column's values of the group that ends in it stand first
      if (n) f((float)n, sh[MIXED ? (y * t.wide + col) * 2 + (end >= col * V + V) : y * t.wide + col]);
      y += dy, c += dc;
      if (c >= width) c -= width, ++y;
    }
  };
  float u = 0.0f, w = 0.0f;
  each([&](float n, float2 p) { u = __fmaf_rn(n, p.x, u); });
  const float mean = __fdiv_rn(warp_sum(u), (float)me.rows * (float)(t.split > 1 ? me.cols * V : a.c));
  each([&](float n, float2 p) {
    const float d = __fsub_rn(p.x, mean);
    w = __fadd_rn(w, __fmaf_rn(__fmul_rn(d, d), n, p.y));
  });
  return make_float2(mean, warp_sum(w));
}

// mean and rstd of the union of lanes' (n, mean, M2); every lane gets them.
__device__ __forceinline__ float2 join_lanes(float n, float2 p, const Norm &a) {
  const float mean = __fdiv_rn(warp_sum(__fmul_rn(n, p.x)), a.m), d = __fsub_rn(p.x, mean);
  const float m2 = warp_sum(n == 0.0f ? 0.0f : __fmaf_rn(__fmul_rn(d, d), n, p.y));
  return make_float2(mean, rstd_of(m2, a.inv_m, a.eps));
}

// The statistics that a cluster's CTAs push to one another: all[parity][CTA][group]. Each
// push is an asynchronous store that counts its bytes on the receiving CTA's mbarrier of that
// parity, so a tile costs neither a cluster barrier nor the fence that comes with one (which
// would wait for the tile's own stores to memory). Parities suffice: a CTA pushes tile n + 2
// only after it got all of tile n + 1, which the others push after they have read tile n.
constexpr unsigned long long kWaitNs = 4000000000ull;  // 4 s
constexpr int kErrNormExchange = 16;
struct Exchange {
  float2 all[2][kMaxCluster][kMaxTileGroups];
  uint64_t bar[2];
  int gave_up;
};
__device__ __forceinline__ uint32_t shared_address(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void exchange_init(Exchange &x) {
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&x.bar[i])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    x.gave_up = 0;
  }
}
// One thread: this tile's bytes are to come.
__device__ __forceinline__ void exchange_expect(Exchange &x, int parity, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(&x.bar[parity])),
               "r"(bytes)
               : "memory");
}
// Lane r < k: group g's pair to CTA r.
__device__ __forceinline__ void exchange_push(Exchange &x, int parity, int from, int g, int to, float2 v) {
  uint32_t slot, bar;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(slot) : "r"(shared_address(&x.all[parity][from][g])), "r"(to));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(shared_address(&x.bar[parity])), "r"(to));
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(slot),
               "l"(pair(v.x, v.y)), "r"(bar)
               : "memory");
}
// Until this tile's pairs are there. A wait that takes 4 s is given up and recorded; the CTA
// then waits no more and runs to its end.
__device__ __forceinline__ void exchange_wait(Exchange &x, int parity, int phase, int *err) {
  const auto ready = [&]() {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(shared_address(&x.bar[parity])), "r"(phase)
        : "memory");
    return ok != 0;
  };
  if (ready()) return;
  volatile int *gave_up = &x.gave_up;
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  while (!ready() && !*gave_up) {
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > kWaitNs) {
      *gave_up = 1;
      atomicCAS(err, 0, kErrNormExchange);
    }
  }
}

template <int V, int MODE, bool MIXED, int SHORT>
__global__ void __launch_bounds__(kTileThreads, kTileCtas + SHORT) norm_tile_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int N = held(V, false) >> SHORT;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) float fifo[];
  __shared__ __align__(16) float2 sh[kTileThreads * (MIXED ? 2 : 1)];
  // by parity of the tile: a warp may be a tile ahead of one that still reads
  __shared__ float2 stats_by[2][kMaxTileGroups];
  __shared__ Exchange exchange;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool joined = MODE == kInCluster && t.k > 1;
  Walk<V, MODE, MIXED> walk(t, MODE == kInCluster ? (int)cluster.block_rank() : 0);
  if (joined) {
    exchange_init(exchange);
    __syncthreads();
    cluster.barrier_arrive();
  }
  const int64_t step = (int64_t)t.tall * a.channels;
  const Place<V, MIXED> place(a, t, walk.tx);
  const float share = joined && lane < t.k ? count_of(a, t, lane, V) : 0.0f;
  Tile<V> me, next;
  if (walk.left) {
    next = walk.get(a, t);
    fetch_tile<V, N>(fifo, a.x, next, step);
  }
  copy_commit();
  if (joined) cluster.barrier_wait();  // all of the cluster's CTAs run
  for (int i = 0; walk.left; ++i) {
    const int n = i & 1;
    me = next;
    walk.advance(a, t);
    Vec<V> x[N];
    copy_wait<0>();
    take_tile(x, fifo, me);
    if (walk.left) {
      next = walk.get(a, t);
      fetch_tile<V, N>(fifo, a.x, next, step);
    }
    copy_commit();
    if (MODE != kWhole) column_moments(x, sh, me, t, walk, place);
    if (joined) {
      if (threadIdx.x == kTileThreads - 1) exchange_expect(exchange, n, t.k * me.q * (int)sizeof(float2));
      for (int g = warp; g < me.q; g += kTileThreads / 32) {
        const float2 m = group_moments<V, MIXED>(sh, g, a, me, t);
        if (lane < t.k) exchange_push(exchange, n, me.k, g, lane, m);
      }
      if (warp < me.q) exchange_wait(exchange, n, i >> 1 & 1, a.err);
    }
    float2 *stats = stats_by[n];
    for (int g = warp; g < me.q; g += kTileThreads / 32) {
      const int64_t team = (int64_t)me.b * a.groups + me.g0 + g;
      if (MODE == kParts) {
        const float2 m = group_moments<V, MIXED>(sh, g, a, me, t);
        if (lane == 0) reinterpret_cast<float2 *>(a.stat)[team * t.k + me.k] = m;
        continue;
      }
      float2 r;
      if (joined) {
        r = join_lanes(share, lane < t.k ? exchange.all[n][lane][g] : make_float2(0.0f, 0.0f), a);
      } else if (MODE == kInCluster) {
        r = group_moments<V, MIXED>(sh, g, a, me, t);
        r.y = rstd_of(r.y, a.inv_m, a.eps);
      } else if (a.whole) {
        r = a.whole[team];
      } else {
        const float2 *q = reinterpret_cast<const float2 *>(a.stat) + team * t.k;
        float u = 0.0f, w = 0.0f;
        for (int i = lane; i < t.k; i += 32) u = __fmaf_rn(count_of(a, t, i, V), q[i].x, u);
        const float mean = __fdiv_rn(warp_sum(u), a.m);
        for (int i = lane; i < t.k; i += 32) {
          const float d = __fsub_rn(q[i].x, mean);
          w = __fadd_rn(w, __fmaf_rn(__fmul_rn(d, d), count_of(a, t, i, V), q[i].y));
        }
        r = make_float2(mean, rstd_of(warp_sum(w), a.inv_m, a.eps));
      }
      if (lane == 0) {
        stats[g] = r;
        if (a.mean && me.k == 0) {
          a.mean[team] = r.x;
          a.rstd[team] = r.y;
        }
      }
    }
    __syncthreads();
    if (MODE != kParts) {
      const float2 lo = stats[me.mine ? place.lo : 0], hi = stats[me.mine ? place.hi : 0];
      const Vec<V> ga = load_or<V>(a.gamma && me.mine ? a.gamma + me.channel : nullptr, 1.0f);
      const Vec<V> be = load_or<V>(a.beta && me.mine ? a.beta + me.channel : nullptr, 0.0f);
      const Vec<V> minus = place.spread(-lo.x, -hi.x), rstd = place.spread(lo.y, hi.y);
      float *q = a.y + me.at;
      with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (i >= me.most) break;
          const Vec<V> r = normalize<decltype(act)::value>(x[i], minus, rstd, ga, be);
          if (i < me.mine) store(q, r);
          q += step;
        }
      });
    }
  }
  copy_wait<0>();
  if (joined) cluster.sync();  // after a wait that was given up, too, no CTA leaves while another may push to it
}

// The tile's sums of dv and dv xh. column_sums: per slice and channel to sh[slices][2][wide * V],
// with a barrier at the end. Then, a warp a group, group_sums adds up the slices, leaves the
// channels' sums in `part` and gives the gamma-weighted sums over the group to every lane.
// Many channels a group, or many slices, are added up over the slices by all threads first.
__device__ __forceinline__ bool together(const Norm &a, const Tiling &t) { return a.c > 32 || t.slices > 8; }
// A channel's sum over a tile of a run: added up in `run_sums` ([2][wide * V], each value the same
// thread's in all of the run's tiles), it leaves for `part` at the run's end.
template <int V>
__device__ __forceinline__ void run_sum(float s, int which, int ch, float *run_sums, const Norm &a,
                                        const Tile<V> &me, const Tiling &t, int tx) {
  if (!a.part) return;
  float *sum = run_sums + which * t.wide * V + ch;
  if (!me.begins) s = __fadd_rn(*sum, s);
  if (me.ends) a.part[((int64_t)me.row * 2 + which) * a.channels + (me.channel - tx * V + ch)] = s;
  else *sum = s;
}
template <int V, int MODE, bool MIXED, bool RUNS>
__device__ __forceinline__ void column_sums(Vec<V> db, Vec<V> dg, float *sh, float *run_sums, const Norm &a,
                                            const Tile<V> &me, const Tiling &t, const Walk<V, MODE, MIXED, RUNS> &walk) {
  const int row = t.wide * V;
  for (int d = 16; d * t.each > 16; d >>= 1) {
#pragma unroll
    for (int i = 0; i < Vec<V>::N; ++i) {
      db.p[i] = add2(db.p[i], from_lane(db.p[i], d));
      dg.p[i] = add2(dg.p[i], from_lane(dg.p[i], d));
    }
  }
  if (walk.leaves) {
    float *q = sh + walk.slice * 2 * row + walk.tx * V;
    store(q, db);
    store(q + row, dg);
  }
  __syncthreads();
  if (together(a, t)) {
    const int n = me.cols * V, slices = t.slices;
    for (int i = threadIdx.x; i < 2 * n; i += kTileThreads) {
      const int which = i >= n, ch = i - (which ? n : 0);
      float *q = sh + which * row + ch;
      float s = q[0];
      for (int y = 1; y < slices; ++y) s = __fadd_rn(s, q[y * 2 * row]);
      q[0] = s;
      if (RUNS) run_sum(s, which, ch, run_sums, a, me, t, walk.tx);
    }
    __syncthreads();
  }
}
template <int V, bool RUNS>
__device__ __forceinline__ float2 group_sums(const float *sh, float *run_sums, int g, const Norm &a,
                                             const Tile<V> &me, const Tiling &t, int tx) {
  const bool whole = together(a, t);
  const int lane = threadIdx.x & 31, row = t.wide * V, slices = whole ? 1 : t.slices;
  const int width = t.split > 1 ? me.cols * V : a.c, first = me.channel - tx * V + g * a.c;
  float *part = !RUNS && a.part ? a.part + (int64_t)me.row * 2 * a.channels + first : nullptr;
  float u = 0.0f, w = 0.0f;
  for (int i = lane; i < 2 * width; i += 32) {
    const int which = i >= width, ch = i - (which ? width : 0);
    const float *q = sh + which * row + g * a.c + ch;
    float s = q[0];
    for (int y = 1; y < slices; ++y) s = __fadd_rn(s, q[y * 2 * row]);
    if (RUNS && !whole) run_sum(s, which, g * a.c + ch, run_sums, a, me, t, tx);
    if (!RUNS && part) part[which * a.channels + ch] = s;
    s = __fmul_rn(a.gamma ? a.gamma[first + ch] : 1.0f, s);
    if (which) w = __fadd_rn(w, s);
    else u = __fadd_rn(u, s);
  }
  return make_float2(warp_sum(u), warp_sum(w));
}

template <int V, int MODE, bool MIXED, int SHORT, bool RUNS>
__global__ void __launch_bounds__(kTileThreads, kTileCtas + SHORT) norm_tile_backward_kernel(const Norm a, const Tiling t) {
  pdl_wait();
  constexpr int N = held(V, true) >> SHORT, kStage = N * kTileThreads * V;
  cg::cluster_group cluster = cg::this_cluster();
  extern __shared__ __align__(16) float fifo[];  // x and dy of one tile
  __shared__ __align__(16) float sh[2 * V * kTileThreads];
  __shared__ float run_sums[RUNS ? 2 * V * kTileThreads : 1];
  __shared__ float2 means_by[2][kMaxTileGroups];
  __shared__ Exchange exchange;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool joined = MODE == kInCluster && t.k > 1;
  Walk<V, MODE, MIXED, RUNS> walk(t, MODE == kInCluster ? (int)cluster.block_rank() : 0);
  if (joined) {
    exchange_init(exchange);
    __syncthreads();
    cluster.barrier_arrive();
  }
  const int64_t step = (int64_t)t.tall * a.channels;
  const Place<V, MIXED> place(a, t, walk.tx);
  Tile<V> me, next;
  float2 lo, hi, next_lo = make_float2(0.0f, 0.0f), next_hi = next_lo;  // mean and rstd of the vector's groups
  const auto fetch = [&]() {
    if (walk.left) {
      next = walk.get(a, t);
      fetch_tile<V, N>(fifo, a.x, next, step);
      fetch_tile<V, N>(fifo + kStage, a.dy, next, step);
      const int64_t team = (int64_t)next.b * a.groups + next.g0;
      const int l = next.mine ? place.lo : 0, h = next.mine ? place.hi : 0;
      next_lo = make_float2(a.mean_in[team + l], a.rstd_in[team + l]);
      if (MIXED) next_hi = make_float2(a.mean_in[team + h], a.rstd_in[team + h]);
    }
    copy_commit();
  };
  fetch();
  if (joined) cluster.barrier_wait();
  for (int i = 0; walk.left; ++i) {
    const int n = i & 1;
    me = next;
    lo = next_lo;
    hi = next_hi;
    walk.advance(a, t);
    Vec<V> x[N], d[N], db = splat<V>(0.0f), dg = db;
    copy_wait<0>();
    // behind a thread's rows x is the mean and dy 0: xh is 0 there (a mean without x, times rstd,
    // may be infinite), and so is what they add to their column's sums
    take_tile(x, fifo, me, place.spread(lo.x, hi.x));
    take_tile(d, fifo + kStage, me);
    fetch();
    const Vec<V> rstd = place.spread(lo.y, hi.y);
    {
      const Vec<V> ga = load_or<V>(a.gamma && me.mine ? a.gamma + me.channel : nullptr, 1.0f);
      const Vec<V> be = load_or<V>(a.beta && me.mine ? a.beta + me.channel : nullptr, 0.0f);
      const Vec<V> minus = place.spread(-lo.x, -hi.x);
      // (a thread without rows has another group's statistics: it adds nothing to its column)
      if (me.mine) with_activation(a.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          if (behind<V, N>(i, me)) break;
          gradient<decltype(act)::value>(x[i], d[i], db, dg, minus, rstd, ga, be);
        }
      });
    }
    if (MODE != kWhole) column_sums(db, dg, sh, run_sums, a, me, t, walk);
    if (joined) {
      if (threadIdx.x == kTileThreads - 1) exchange_expect(exchange, n, t.k * me.q * (int)sizeof(float2));
      for (int g = warp; g < me.q; g += kTileThreads / 32) {
        const float2 m = group_sums<V, RUNS>(sh, run_sums, g, a, me, t, walk.tx);
        if (lane < t.k) exchange_push(exchange, n, me.k, g, lane, m);
      }
      if (warp < me.q) exchange_wait(exchange, n, i >> 1 & 1, a.err);
    }
    float2 *means = means_by[n];
    for (int g = warp; g < me.q; g += kTileThreads / 32) {
      const int64_t team = (int64_t)me.b * a.groups + me.g0 + g;
      float2 m = make_float2(0.0f, 0.0f);
      if (MODE == kParts || (MODE == kInCluster && !joined)) m = group_sums<V, RUNS>(sh, run_sums, g, a, me, t, walk.tx);
      if (MODE == kParts) {
        if (lane == 0) reinterpret_cast<float2 *>(a.stat)[team * t.k + me.k] = m;
        continue;
      }
      float u = m.x, w = m.y;
      if (MODE == kWhole && a.whole) {
        if (lane == 0) u = a.whole[team].x, w = a.whole[team].y;
      } else if (MODE == kWhole) {
        const float2 *q = reinterpret_cast<const float2 *>(a.stat) + team * t.k;
        for (int i = lane; i < t.k; i += 32) u = __fadd_rn(u, q[i].x), w = __fadd_rn(w, q[i].y);
      } else if (joined && lane < t.k) {
        u = exchange.all[n][lane][g].x, w = exchange.all[n][lane][g].y;
      }
      if (MODE == kWhole || joined) u = warp_sum(u), w = warp_sum(w);
      u = __fmul_rn(u, -a.inv_m);
      w = __fmul_rn(w, -a.inv_m);
      if (lane == 0) means[g] = make_float2(u, w);
    }
    __syncthreads();
    if (MODE != kParts) {
      const float2 l = means[me.mine ? place.lo : 0], h = means[me.mine ? place.hi : 0];
      const Vec<V> k1 = place.spread(l.x, h.x), k2 = place.spread(l.y, h.y);
      float *q = a.dx + me.at;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (behind<V, N>(i, me)) break;
        const Vec<V> r = finish(x[i], d[i], k1, k2, rstd);
        if (i < me.mine) store(q, r);
        q += step;
      }
    }
  }
  copy_wait<0>();
  if (joined) cluster.sync();
}

// ---------------------------------------------------------------- many tiles a group

// Between the two launches: a group's k pairs, by a CTA, in place of every tile's joining all of
// them, which is quadratic in k. (mean, rstd), or of the backward's sums their totals; in 64 bits,
// since a thread may have thousands.
constexpr int kJoinThreads = 512;
__device__ __forceinline__ double join_sum(double v, double *sh) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < kJoinThreads / 32; ++w) v += sh[w];
  return v;
}
template <bool BACKWARD>
__global__ void __launch_bounds__(kJoinThreads) norm_join_kernel(const Norm a, const Tiling t, int v) {
  pdl_wait();
  __shared__ double sh[kJoinThreads / 32];
  const int64_t team = blockIdx.x;
  const float2 *q = reinterpret_cast<const float2 *>(a.stat) + team * t.k;
  double u = 0.0, w = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < t.k; i += kJoinThreads) {
    u += BACKWARD ? (double)q[i].x : (double)count_of(a, t, i, v) * q[i].x;
    if (BACKWARD) w += q[i].y;
  }
  u = join_sum(u, sh);
  if (BACKWARD) {
    w = join_sum(w, sh);
    if (threadIdx.x == 0) a.whole[team] = make_float2((float)u, (float)w);
    return;
  }
  const double m = (double)a.len * a.c, mean = u / m;
#pragma unroll 4
  for (int i = threadIdx.x; i < t.k; i += kJoinThreads) {
    const double d = q[i].x - mean;
    w += d * d * count_of(a, t, i, v) + q[i].y;
  }
  w = join_sum(w, sh);
  if (threadIdx.x == 0) a.whole[team] = make_float2((float)mean, (float)(1.0 / sqrt(w / m + a.eps)));
}

// ---------------------------------------------------------------- the parameters' gradients

// dbeta[c] and dgamma[c] from part[rows][2][channels]: 32 channels a CTA, the rows over its
// warps and over the CTAs of a cluster, which fold their sums through distributed shared
// memory in order; a warp's rows in blocks of kNear.
constexpr int kFoldWarps = 16;
__global__ void __launch_bounds__(kFoldWarps * 32) norm_fold_kernel(float *__restrict__ dgamma,
                                                                    float *__restrict__ dbeta,
                                                                    const float *__restrict__ part, int rows,
                                                                    int64_t channels) {
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ctas = (int)cluster.num_blocks();
  __shared__ float sh[2][kFoldWarps][32];
  __shared__ float sum[2][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t ch = (int64_t)(blockIdx.x / ctas) * 32 + lane;
  float u = 0.0f, w = 0.0f;
  if (ch < channels) {
    const int step = ctas * kFoldWarps;
    const int64_t hop = (int64_t)step * 2 * channels;
    int r = rank * kFoldWarps + warp;
    const float *at = part + (int64_t)r * 2 * channels + ch;
    for (; r < rows - (kNear - 1) * step; r += kNear * step) {
      float us = 0.0f, ws = 0.0f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float x[kNear / 2], y[kNear / 2];  // in flight together
#pragma unroll
        for (int i = 0; i < kNear / 2; ++i, at += hop) x[i] = at[0], y[i] = at[channels];
#pragma unroll
        for (int i = 0; i < kNear / 2; ++i) us = __fadd_rn(us, x[i]), ws = __fadd_rn(ws, y[i]);
      }
      u = __fadd_rn(u, us);
      w = __fadd_rn(w, ws);
    }
    float us = 0.0f, ws = 0.0f;
#pragma unroll 8
    for (; r < rows; r += step, at += hop) us = __fadd_rn(us, at[0]), ws = __fadd_rn(ws, at[channels]);
    u = __fadd_rn(u, us);
    w = __fadd_rn(w, ws);
  }
  sh[0][warp][lane] = u;
  sh[1][warp][lane] = w;
  __syncthreads();
  if (warp < 2) {
    u = sh[warp][0][lane];
#pragma unroll
    for (int i = 1; i < kFoldWarps; ++i) u = __fadd_rn(u, sh[warp][i][lane]);
    sum[warp][lane] = u;
  }
  if (ctas > 1) cluster.sync();
  if (rank == 0 && warp < 2 && ch < channels) {
    for (int r = 1; r < ctas; ++r) u = __fadd_rn(u, cluster.map_shared_rank(&sum[0][0], r)[warp * 32 + lane]);
    float *out = warp ? dgamma : dbeta;
    if (out) out[ch] = u;
  }
  if (ctas > 1) cluster.sync();
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
  bool join;             // two-launch tiles: statistics joined by a launch between them
  bool mixed;            // tile kernels: vectors of 4 across groups
  int shorter;           // tile kernels in a cluster: those for short tiles
  int parts;             // rows of the per-channel partial sums (backward)
  int fold;              // row kernels: teams a CTA adds up
  size_t part_floats, stat_floats;
};

int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t power_of_two(int64_t a) {
  int64_t p = 1;
  while (p < a) p *= 2;
  return p;
}

// Thread columns for tiles of `cols` vectors: the next power of two where a warp then holds whole
// rows and more columns cost at most a ninth of the thread rows, else just as many
// ([16, 1024, 640] in 32 groups, 10 vectors: 25 and 44 us against 28 and 52 with 16 columns;
// [8, 4096, 1920], 15 vectors: 133 us with 16 columns, 146 with 15).
int64_t columns_for(int64_t cols) {
  const int64_t wide = power_of_two(cols);
  return wide <= 32 && kTileThreads / wide * 9 >= kTileThreads / cols * 8 ? wide : cols;
}

// tiles: not the row kernels.
Plan norm_plan(int64_t batch, int64_t len, int64_t channels, int64_t groups, int v, bool backward, bool tiles = false) {
  Plan p{};
  const int64_t c = channels / groups;
  int whole = v;  // floats a vector that stays in a group
  while (c % whole) whole /= 2;
  int64_t cv = c / whole, vectors = len * cv;
  const int64_t teams = batch * groups;
  // Row kernels up to 2048 vectors; above 256 (a CTA's worth) only where a row's piece of
  // a group is at least 512 bytes, else the tile kernels, which take several groups' pieces
  // of a row together.
  const bool rows = !tiles && len * channels <= INT_MAX && (vectors <= 256 || (vectors <= 2048 && c >= 128));
  // Else tiles, of mixed vectors where others would be floats or pairs of them. (Tiles where row
  // kernels would do: [8192, 3, 680] / 4 forward 135 us against 31, [2048, 48, 40] / 4 20 against 12.)
  const int64_t unit = c % 2 ? 4 : 2;  // groups that make whole vectors
  const bool can_mix = v == 4 && c % 4 && c >= 2 && channels % 4 == 0 && unit * c <= 4 * kTileThreads;
  // But a backward whose row kernel holds 8 vectors of 1 or 2 floats a thread (one CTA an SM) takes
  // mixed tiles that hold a sample's rows whole and enough values: of odd c, 1200 ([2941, 8, 1020]
  // / 4, 138 us by rows, 95 so; [4096, 8, 1048] / 8, 275 and 171; of 960 values [25000, 48, 20] / 4, 132
  // and 187); of even c, with 10 rows, 2400 ([1470, 24, 680] / 4, 105 and 83; of 1200 [20000, 30, 40] / 4,
  // 107 and 147), or 1900 where a warp gets few groups ([2048, 48, 40] / 4, 26 and 21; [12500, 48, 40] / 4,
  // 91 and 98).
  if (rows && backward && can_mix && (vectors > 1024 || (vectors > 128 && vectors <= 256))) {
    const Plan m = norm_plan(batch, len, channels, groups, v, true, true);
    const int64_t values = m.t.q * c * len, few = (int64_t)fz::num_sms() * 8 * 16;
    if (m.t.k == 1 && (c % 2 ? values >= 1200 : len >= 10 && values >= (teams <= few ? 1900 : 2400))) return m;
  }
  p.mixed = !rows && can_mix;
  if (!p.mixed) v = whole;
  cv = c / v, vectors = len * cv;
  p.v = v;
  if (rows) {
    p.lanes = vectors <= 4 ? 4 : vectors <= 8 ? 8 : vectors <= 16 ? 16 : vectors <= 256 ? 32 : kRowThreads;
    p.nv = 1;
    while ((int64_t)p.nv * p.lanes < vectors) p.nv *= 2;
    const int64_t per_cta = kRowThreads / p.lanes;
    // Teams in flight: what is resident, a multiple of groups.
    int64_t want = (int64_t)fz::num_sms() * per_cta * row_ctas(backward, p.nv);
    if (want > teams) want = teams;
    want = want / groups * groups;
    if (want < groups) want = groups;
    p.stride = (int)want;
    p.grid = (unsigned)up(want, per_cta);
    if (backward) {
      p.fold = per_cta % groups == 0 ? (int)(per_cta / groups) : 1;
      p.parts = (int)up(want, groups * p.fold);
      p.part_floats = (size_t)p.parts * 2 * channels;
    }
    return p;
  }
  // Tiles: whole groups side by side, or a part of one group where it has more vectors than a
  // CTA has threads.
  Tiling &t = p.t;
  t.q = 1;
  t.split = p.mixed ? 1 : (int)up(cv, kTileThreads);
  if (t.split == 1) {
    // Of the numbers of groups that give 48 to 192 bytes a row, the one that wastes the fewest
    // thread columns (their number is a power of two), the larger of equals; tiles of less
    // than 96 bytes only where they bring the cluster to 8 CTAs.
    double best = 0.0;
    const int64_t some = p.mixed ? unit : 1;
    for (int64_t q = some; q <= groups && q <= kMaxTileGroups && q * c <= kTileThreads * v; q += some) {
      if (q > some && q * c > (p.mixed ? 64 : 48)) break;
      const int64_t cols = q * c / v, thread_rows = kTileThreads / columns_for(cols);
      const int64_t tall = thread_rows * held(v, backward);
      double use = (double)(cols * thread_rows) / kTileThreads * groups / (double)(up(groups, q) * q);
      if (q * c < 24) use *= q * c / 24.0;
      if (up(len, tall) > 8 && up(len, tall) <= 2 * kMaxCluster) use *= 0.6;
      if (use >= best) best = use, t.q = (int)q;
    }
    t.cols = (int)(t.q * c / v);
  } else {
    // Of the numbers of pieces that a cluster holds, the one whose tiles take the least, each four
    // rows of a thread beside its own; two launches cost as much again.
    double best = 0.0;
    for (int64_t n = t.split; n <= kMaxCluster || n == up(cv, kTileThreads); ++n) {
      const int64_t rows = kTileThreads / columns_for(up(cv, n)), chunks = up(len, rows * held(v, backward));
      const double cost = (double)(n * chunks) * (up(up(len, chunks), rows) + 4) * (n * chunks > kMaxCluster ? 1.6 : 1.0);
      if (best == 0.0 || cost < best) best = cost, t.split = (int)n;
    }
    t.cols = (int)up(cv, t.split);
  }
  t.wide = (int)columns_for(t.cols);
  t.tall = kTileThreads / t.wide;
  t.each = 32 % t.wide == 0 ? 32 / t.wide : 1;
  t.slices = t.tall / t.each;
  t.bundles = (int)up(groups, t.q);
  // Rows: as few tiles one below the other as hold the sample, or, where those would leave
  // SMs idle, as many as a cluster takes and that keep four rows a thread.
  const int64_t ty = t.tall, most = ty * held(v, backward);
  int64_t chunks = up(len, most);
  const int64_t idle = up((int64_t)fz::num_sms() * kTileCtas, batch * t.bundles * t.split);
  int64_t room = kMaxCluster / t.split;
  if (room > up(len, ty * 4)) room = up(len, ty * 4);
  if (room > idle) room = idle;
  if (chunks < room) chunks = room;
  t.rows = (int)up(len, chunks);
  t.chunks = (int)up(len, t.rows);
  const int64_t k = (int64_t)t.split * t.chunks;
  t.k = (int)k;
  p.cluster = k <= kMaxCluster;
  while (p.shorter < kShortest && up(t.rows, t.tall) <= held(v, backward) >> (p.shorter + 1)) ++p.shorter;
  // The backward leaves 2 floats a channel, row of tiles and run of samples: with runs of one, as
  // much as x for tiles of two rows, and twice that for one. So a CTA takes the tiles of up to 16
  // samples at one place in turn, until the sums are an eighth of x, as long as every CTA still has
  // 16 such runs (a run more or less than the others' then costs little). [65536, 16384] in one
  // group: 25.4 ms and 0.5 GB of sums with runs of 16, 36.6 ms and 8.6 GB with runs of one;
  // [4000, 9, 4096] / 4, 954 and 1545 us. Narrow groups' tiles have three rows and more, and runs
  // cost them more than they save: [20000, 11, 400] / 4, 576 and 544 us, [1990, 7, 2368] / 32 (mixed)
  // 295 and 248.
  const int64_t ctas = (int64_t)fz::num_sms() * (kTileCtas + (p.cluster ? p.shorter : 0));
  const auto units = [&](int64_t run) { return up(batch, run) * t.bundles * k; };  // in tiles
  int64_t run = 1;
  while (backward && !p.mixed && c >= 128 && t.rows * run < 16 && units(2 * run) >= 16 * ctas) run *= 2;
  t.run = (int)run;
  t.units = (int)(p.cluster ? units(run) / k : units(run));
  if (backward) {
    p.parts = (int)(up(batch, run) * t.chunks);
    p.part_floats = (size_t)p.parts * 2 * channels;
  }
  p.join = !p.cluster && k > kMostTiles;
  if (!p.cluster) p.stat_floats = (size_t)(teams * (k + p.join) * 2);
  return p;
}

int vector_of(std::initializer_list<const void *> ptrs) {
  uintptr_t all = 0;
  for (const void *p : ptrs) all |= (uintptr_t)p;
  return (all & 15) == 0 ? 4 : (all & 7) == 0 ? 2 : 1;
}

cudaLaunchConfig_t config(unsigned grid, int threads, int smem, int k, cudaStream_t s, cudaLaunchAttribute *attr) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)k;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// Launch a kernel over clusters of `k` CTAs (k = 1: none).
template <typename... KArgs, typename... Args>
int launch_cluster(void (*kernel)(KArgs...), unsigned grid, int threads, int smem, int k, cudaStream_t s,
                   Args... args) {
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config(grid, threads, smem, k, s, attr);
  FZ_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

// Shared memory and cluster sizes that a kernel asks for, and (tile kernels in clusters)
// how many clusters of k CTAs are resident at once, asked for once a device, kernel and k.
int resident_clusters(const void *kernel, int threads, int smem, int k, int *count) {
  struct Entry {
    const void *kernel;
    int device, k, count;
  };
  static std::mutex mu;
  static Entry known[512];
  static int entries = 0;
  int device = 0;
  FZ_CUDA(cudaGetDevice(&device));
  std::lock_guard<std::mutex> lock(mu);
  for (int i = 0; i < entries; ++i)
    if (known[i].kernel == kernel && known[i].device == device && known[i].k == k) {
      *count = known[i].count;
      return FZ_OK;
    }
  FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (k > 8) FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = config((unsigned)k, threads, smem, k, nullptr, attr);
  int n = 0;
  FZ_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
  FZ_REQUIRE(n > 0, "group norm: a cluster does not fit the device");
  if (entries < 512) known[entries++] = {kernel, device, k, n};
  *count = n;
  return FZ_OK;
}

template <typename... KArgs, typename... Args>
int launch_rows(void (*kernel)(KArgs...), unsigned grid, int smem, cudaStream_t s, Args... args) {
  FZ_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  FZ_CUDA(fz::launch_pdl(kernel, dim3(grid), dim3(kRowThreads), (size_t)smem, s, args...));
  FZ_CHECK_LAUNCH();
  return FZ_OK;
}

template <int V, int P, int NV>
int run_row(const Norm &a, const Plan &p, bool backward, cudaStream_t s) {
  if (backward)
    return launch_rows(norm_rows_backward_kernel<V, P, NV>, p.grid, row_smem(true, P, NV, V), s, a, p.stride, p.fold);
  return launch_rows(norm_rows_kernel<V, P, NV>, p.grid, row_smem(false, P, NV, V), s, a, p.stride);
}

template <int V>
int run_rows(const Norm &a, const Plan &p, bool backward, cudaStream_t s) {
  switch (p.lanes) {
    case 4: return run_row<V, 4, 1>(a, p, backward, s);
    case 8: return run_row<V, 8, 1>(a, p, backward, s);
    case 16: return run_row<V, 16, 1>(a, p, backward, s);
    case 32:
      return p.nv == 1   ? run_row<V, 32, 1>(a, p, backward, s)
             : p.nv == 2 ? run_row<V, 32, 2>(a, p, backward, s)
             : p.nv == 4 ? run_row<V, 32, 4>(a, p, backward, s)
                         : run_row<V, 32, 8>(a, p, backward, s);
    default:
      return p.nv == 2   ? run_row<V, kRowThreads, 2>(a, p, backward, s)
             : p.nv == 4 ? run_row<V, kRowThreads, 4>(a, p, backward, s)
                         : run_row<V, kRowThreads, 8>(a, p, backward, s);
  }
}

template <int V, int MODE, bool MIXED, int SHORT = 0>
int run_tile(Norm a, const Plan &p, bool backward, cudaStream_t s) {
  if (MODE == kInCluster)
    if (int rc = fz::device_error_word(&a.err)) return rc;
  constexpr bool kRuns = MODE != kWhole && !MIXED;
  const auto kernel = !backward                ? norm_tile_kernel<V, MODE, MIXED, SHORT>
                      : kRuns && p.t.run > 1 ? norm_tile_backward_kernel<V, MODE, MIXED, SHORT, kRuns>
                                             : norm_tile_backward_kernel<V, MODE, MIXED, SHORT, false>;
  const int smem = (held(V, backward) >> SHORT) * kTileThreads * V * 4 * (backward ? 2 : 1);
  const int k = MODE == kInCluster ? p.t.k : 1;
  int resident = 0;
  if (int rc = resident_clusters((const void *)kernel, kTileThreads, smem, k, &resident)) return rc;
  Tiling t = p.t;
  if (MODE == kWhole) t.run = 1, t.units = (int)(a.batch * t.bundles * t.k);
  const int64_t grid = (int64_t)(t.units < resident ? t.units : resident) * k;
  return launch_cluster(kernel, (unsigned)grid, kTileThreads, smem, k, s, a, t);
}

template <int V, bool MIXED>
int run_tiles(Norm a, const Plan &p, bool backward, cudaStream_t s) {
  if (p.cluster)
    return p.shorter == 2   ? run_tile<V, kInCluster, MIXED, 2>(a, p, backward, s)
           : p.shorter == 1 ? run_tile<V, kInCluster, MIXED, 1>(a, p, backward, s)
                            : run_tile<V, kInCluster, MIXED>(a, p, backward, s);
  if (int rc = run_tile<V, kParts, MIXED>(a, p, backward, s)) return rc;
  if (p.join) {
    const int64_t teams = a.batch * a.groups;
    a.whole = reinterpret_cast<float2 *>(a.stat) + teams * p.t.k;
    if (int rc = launch_cluster(backward ? norm_join_kernel<true> : norm_join_kernel<false>, (unsigned)teams, kJoinThreads,
                                0, 1, s, a, p.t, V))
      return rc;
  }
  return run_tile<V, kWhole, MIXED>(a, p, backward, s);
}

int run(const Norm &a, const Plan &p, bool backward, cudaStream_t s) {
  if (p.mixed) return run_tiles<4, true>(a, p, backward, s);
  if (p.lanes)
    return p.v == 4   ? run_rows<4>(a, p, backward, s)
           : p.v == 2 ? run_rows<2>(a, p, backward, s)
                      : run_rows<1>(a, p, backward, s);
  return p.v == 4   ? run_tiles<4, false>(a, p, backward, s)
         : p.v == 2 ? run_tiles<2, false>(a, p, backward, s)
                    : run_tiles<1, false>(a, p, backward, s);
}

int check_sizes(const char *who, int64_t batch, int64_t len, int64_t channels, int64_t groups) {
  const std::string name(who);
  FZ_REQUIRE(batch >= 0 && len >= 0 && channels >= 1 && groups >= 1, name + ": negative or zero size");
  FZ_REQUIRE(channels % groups == 0, name + ": channels must be a multiple of groups");
  // 2^36 values in at most 2^30 rows of channels (batch numbers are 32-bit in the kernels)
  const int64_t rows = (int64_t)1 << 30, values = (int64_t)1 << 36;
  FZ_REQUIRE(channels <= rows && len <= rows && batch <= rows, name + ": too many elements");
  FZ_REQUIRE(len == 0 || batch == 0 || (batch <= rows / len && batch * len <= values / channels),
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
  a.m = (float)(len * a.c), a.inv_m = (float)(1.0 / (double)(len * a.c)), a.eps = eps, a.act = act;
  cudaStream_t s = fz::resolve(stream);
  return run(a, p, false, s);
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
  a.m = (float)(len * a.c), a.inv_m = (float)(1.0 / (double)(len * a.c)), a.act = act;
  if (int rc = run(a, p, true, s)) return rc;
  if (!a.part) return FZ_OK;
  // CTAs a block of 32 channels: as many as have 4 rows a warp, until the SMs are filled
  const int64_t blocks = up(channels, 32);
  int ctas = 1;
  while (ctas < 8 && blocks * ctas < fz::num_sms() && p.parts > ctas * 2 * kFoldWarps * 4) ctas *= 2;
  return launch_cluster(norm_fold_kernel, (unsigned)(blocks * ctas), kFoldWarps * 32, 0, ctas, s, dgamma, dbeta,
                        (const float *)a.part, p.parts, channels);
}
