// Host-memory test double of the C ABI in include/fusion_b200.h.
//
// TEST INFRASTRUCTURE ONLY. It lets the CPU test suite run the C++ host layer
// (nova_b200/host: the fusion-IR lowering, the autodiff engine, Fusion's op
// semantics and quirks) without a GPU: tests/hostfake/build_fake.py links a copy
// of the pybind module against this library in tests/hostfake/_build/. The
// product library nova_b200/libfusion_b200.so never contains or loads it, and it
// is never a fallback: it exists so host-logic bugs surface on CPU before a GPU
// run. "Device" pointers here are host pointers; every op is a scalar loop with
// the IEEE fp32 semantics the sm_100a kernels implement.
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <string>
#include <vector>

#include "fusion_b200.h"

namespace {
thread_local std::string g_err;
int64_t g_launches = 0;
std::set<std::string> g_programs;

int fail(int code, const std::string &m) {
  g_err = m;
  return code;
}

float binop(int op, float a, float b) {
  switch (op) {
    case FZ_ADD: return a + b;
    case FZ_SUB: return a - b;
    case FZ_MUL: return a * b;
    case FZ_DIV: return a / b;
    case FZ_POW: return b == 2.0f ? a * a : std::pow(a, b);
    case FZ_MAXIMUM: return a > b ? a : b;
    case FZ_GT: return a > b ? 1.0f : 0.0f;
    case FZ_GE: return a >= b ? 1.0f : 0.0f;
  }
  return 0.0f;
}

static float tf32_lo1(float x) {
  uint32_t u;
  std::memcpy(&u, &x, 4);
  u &= 0xffffe000u;
  float h;
  std::memcpy(&h, &u, 4);
  float r = x - h;
  std::memcpy(&u, &r, 4);
  if ((u & 0x7f800000u) != 0x7f800000u) u = (u + 0xfffu + ((u >> 13) & 1u)) & 0xffffe000u;
  std::memcpy(&r, &u, 4);
  return r;
}

float unop(int op, float a) {
  switch (op) {
    case FZ_EXP: return std::exp(a);
    case FZ_LOG: return std::log(a);
    case FZ_SQRT: return std::sqrt(a);
    case FZ_TF32_LO: return tf32_lo1(a);
    default: return a;
  }
}

// Visit every index of a plan; fn(offsets in elements of each operand).
template <class Fn>
void walk(const fz_ewise_plan &p, Fn fn) {
  int64_t total = 1;
  for (int d = 0; d < p.ndim; ++d) total *= p.size[d];
  std::vector<int64_t> idx(p.ndim > 0 ? p.ndim : 1, 0);
  std::vector<int64_t> off(p.num_operands);
  for (int64_t i = 0; i < total; ++i) {
    for (int k = 0; k < p.num_operands; ++k) {
      int64_t o = 0;
      for (int d = 0; d < p.ndim; ++d) o += idx[d] * p.stride_bytes[k][d] / 4;
      off[k] = o;
    }
    fn(off.data());
    for (int d = p.ndim - 1; d >= 0; --d) {
      if (++idx[d] < p.size[d]) break;
      idx[d] = 0;
    }
  }
}
}  // namespace

extern "C" {

const char *fz_last_error(void) { return g_err.c_str(); }
int fz_version(void) { return 1; }
int fz_device_count(int *c) { *c = 1; return FZ_OK; }
int fz_set_device(int d) { return d == 0 ? FZ_OK : fail(FZ_ERR_INVALID, "Invalid device index"); }
int fz_get_device(int *d) { *d = 0; return FZ_OK; }
void *fz_default_stream(void) { static int s; return &s; }
int fz_stream_sync(void *) { return FZ_OK; }
int fz_device_sync(void) { return FZ_OK; }
// live allocations, so pool_used_bytes reports what the host keeps
std::map<void *, size_t> g_live;
size_t g_live_bytes = 0;
int fz_malloc(void **p, size_t bytes, void *) {
  *p = nullptr;
  if (!bytes) return FZ_OK;
  *p = std::aligned_alloc(256, (bytes + 255) & ~(size_t)255);
  if (!*p) return fail(FZ_ERR_OOM, "host allocation failed");
  g_live[*p] = bytes;
  g_live_bytes += bytes;
  return FZ_OK;
}
int fz_free(void *p, void *) {
  auto it = g_live.find(p);
  if (it != g_live.end()) {
    g_live_bytes -= it->second;
    g_live.erase(it);
  }
  std::free(p);
  return FZ_OK;
}
int fz_pool_release(void) { return FZ_OK; }
int fz_pool_stats(size_t *r, size_t *u) { if (r) *r = g_live_bytes; if (u) *u = g_live_bytes; return FZ_OK; }
int fz_memcpy_h2d(void *d, const void *s, size_t n, void *) { if (n) std::memcpy(d, s, n); return FZ_OK; }
int fz_memcpy_d2h(void *d, const void *s, size_t n, void *) { if (n) std::memcpy(d, s, n); return FZ_OK; }
int fz_memcpy_d2d(void *d, const void *s, size_t n, void *) { if (n) std::memmove(d, s, n); return FZ_OK; }
int fz_fill_f32(float *d, float v, int64_t n, void *) { for (int64_t i = 0; i < n; ++i) d[i] = v; ++g_launches; return FZ_OK; }
int fz_host_alloc(void **p, size_t b) { return fz_malloc(p, b ? b : 1, nullptr); }
int fz_host_free(void *p) { std::free(p); return FZ_OK; }
int fz_timer_create(void **t) { *t = std::malloc(1); return FZ_OK; }
int fz_timer_start(void *, void *) { return FZ_OK; }
int fz_timer_stop(void *, void *) { return FZ_OK; }
int fz_timer_elapsed_ms(void *, float *ms) { *ms = 0.0f; return FZ_OK; }
int fz_timer_destroy(void *t) { std::free(t); return FZ_OK; }
int64_t fz_launch_count(void) { return g_launches; }
int fz_kernel_status(void) { return FZ_OK; }

int fz_ewise_binary(int op, const fz_ewise_plan *p, float *out, const float *a, const float *b, void *) {
  if (p->num_operands != 3) return fail(FZ_ERR_INVALID, "elementwise plan: wrong operand count");
  walk(*p, [&](const int64_t *o) { out[o[0]] = binop(op, a[o[1]], b[o[2]]); });
  ++g_launches;
  return FZ_OK;
}
int fz_ewise_binary_contig(int op, int64_t n, float *out, const float *a, const float *b, void *) {
  for (int64_t i = 0; i < n; ++i) out[i] = binop(op, a[i], b[i]);
  ++g_launches;
  return FZ_OK;
}
int fz_ewise_unary(int op, const fz_ewise_plan *p, float *out, const float *a, void *) {
  walk(*p, [&](const int64_t *o) { out[o[0]] = unop(op, a[o[1]]); });
  ++g_launches;
  return FZ_OK;
}
int fz_sub_inplace(float *x, const float *y, int64_t n, void *) {
  for (int64_t i = 0; i < n; ++i) x[i] = x[i] - y[i];
  ++g_launches;
  return FZ_OK;
}

int fz_fused_launch(const fz_program *pg, const fz_ewise_plan *p, float *const *outs,
                    const float *const *leaves, void *) {
  if (p->num_operands != pg->num_outputs + pg->num_leaves)
    return fail(FZ_ERR_INVALID, "fz_fused_launch: plan operand count != outputs + leaves");
  g_programs.insert(std::string(reinterpret_cast<const char *>(pg->nodes),
                                sizeof(fz_node) * pg->num_nodes));
  std::vector<float> t(pg->num_nodes);
  walk(*p, [&](const int64_t *o) {
    auto val = [&](int s) { return s >= 0 ? t[s] : leaves[-1 - s][o[pg->num_outputs + (-1 - s)]]; };
    for (int i = 0; i < pg->num_nodes; ++i) {
      const fz_node &n = pg->nodes[i];
      t[i] = n.kind == FZ_NODE_BINARY ? binop(n.op, val(n.src0), val(n.src1))
             : n.kind == FZ_NODE_UNARY ? unop(n.op, val(n.src0)) : n.imm;
    }
    for (int k = 0; k < pg->num_outputs; ++k) outs[k][o[k]] = t[pg->out_node[k]];
  });
  ++g_launches;
  return FZ_OK;
}
int fz_fused_cache_size(void) { return (int)g_programs.size(); }

int fz_reduce(int op, float *out, const float *in, int64_t outer, int64_t len, int64_t inner, void *) {
  for (int64_t o = 0; o < outer; ++o)
    for (int64_t j = 0; j < inner; ++j) {
      const float *q = in + o * len * inner + j;
      float acc = op == FZ_RMAX ? -INFINITY : 0.0f;
      for (int64_t r = 0; r < len; ++r) {
        float v = q[r * inner];
        if (op == FZ_RMAX) {
          if (acc != acc) continue;
          if (v != v || v > acc || (v == 0.0f && acc == 0.0f && !std::signbit(v))) acc = v;
        } else {
          acc += v;
        }
      }
      if (op == FZ_RMEAN) acc = acc / (float)len;
      out[o * inner + j] = acc;
    }
  ++g_launches;
  return FZ_OK;
}

int fz_swapaxes(float *out, const float *in, const int64_t *shape, int nd, int a1, int a2, void *) {
  if (a1 < 0) a1 += nd;
  if (a2 < 0) a2 += nd;
  std::vector<int64_t> os(shape, shape + nd), ist(nd), ost(nd), idx(nd, 0);
  std::swap(os[a1], os[a2]);
  int64_t r = 1, q = 1, total = 1;
  for (int d = nd - 1; d >= 0; --d) {
    ist[d] = r; r *= shape[d];
    ost[d] = q; q *= os[d];
    total *= shape[d];
  }
  for (int64_t i = 0; i < total; ++i) {
    int64_t o = 0;
    for (int d = 0; d < nd; ++d) o += idx[d] * ost[d == a1 ? a2 : d == a2 ? a1 : d];
    out[o] = in[i];
    for (int d = nd - 1; d >= 0; --d) {
      if (++idx[d] < shape[d]) break;
      idx[d] = 0;
    }
  }
  ++g_launches;
  return FZ_OK;
}

int fz_gemm_f32(int64_t batch, int64_t M, int64_t N, int64_t K, const float *A, int64_t lda,
                int64_t sA, int tA, const float *B, int64_t ldb, int64_t sB, int tB, float *C,
                int64_t ldc, int64_t sC, void *) {
  for (int64_t b = 0; b < batch; ++b)
    for (int64_t i = 0; i < M; ++i)
      for (int64_t j = 0; j < N; ++j) {
        double s = 0;
        for (int64_t k = 0; k < K; ++k) {
          float x = tA ? A[b * sA + k * lda + i] : A[b * sA + i * lda + k];
          float y = tB ? B[b * sB + j * ldb + k] : B[b * sB + k * ldb + j];
          s += (double)x * (double)y;
        }
        C[b * sC + i * ldc + j] = (float)s;
      }
  ++g_launches;
  return FZ_OK;
}


int64_t g_epilogue_launches = 0;
int fz_gemm_f32_epilogue(int64_t batch, int64_t M, int64_t N, int64_t K, const float *A,
                         const float *A_lo, int64_t lda, int64_t sA, int tA, const float *B,
                         const float *B_lo, int64_t ldb, int64_t sB, int tB,
                         const struct fz_program *pg, const fz_epi_input *inputs,
                         float *const *outs, int64_t ldc, int64_t sC, void *st) {
  if (!pg || pg->num_leaves < 1 || pg->num_leaves > FZ_MAX_LEAVES || pg->num_outputs > FZ_MAX_OUTPUTS)
    return fail(FZ_ERR_INVALID, "fz_gemm_f32_epilogue: bad program");
  std::vector<float> P((size_t)(batch * M * N));
  int64_t before = g_launches;
  int rc = fz_gemm_f32_split(batch, M, N, K, A, A_lo, lda, sA, tA, B, B_lo, ldb, sB, tB, P.data(), N,
                             M * N, st);
  if (rc) return rc;
  fz_ewise_plan plan{};
  plan.ndim = 3;
  plan.num_operands = pg->num_outputs + pg->num_leaves;
  plan.size[0] = batch;
  plan.size[1] = M;
  plan.size[2] = N;
  auto set = [&](int k, int64_t b, int64_t m, int64_t n) {
    plan.stride_bytes[k][0] = b * 4;
    plan.stride_bytes[k][1] = m * 4;
    plan.stride_bytes[k][2] = n * 4;
  };
  for (int k = 0; k < pg->num_outputs; ++k) set(k, sC, ldc, 1);
  std::vector<const float *> leaves(pg->num_leaves);
  leaves[0] = P.data();
  set(pg->num_outputs, M * N, N, 1);
  for (int k = 1; k < pg->num_leaves; ++k) {
    const fz_epi_input &in = inputs[k - 1];
    if (in.col_stride != 0 && in.col_stride != 1)
      return fail(FZ_ERR_INVALID, "fz_gemm_f32_epilogue: input column stride must be 0 or 1");
    leaves[k] = in.ptr;
    set(pg->num_outputs + k, in.batch_stride, in.row_stride, in.col_stride);
  }
  rc = fz_fused_launch(pg, &plan, outs, leaves.data(), st);
  g_launches = before + 1;  // one kernel on the device
  ++g_epilogue_launches;
  return rc;
}
int fz_gemm_epilogue_compile(const struct fz_program *, const fz_epi_input *, int, int, int, int) {
  return FZ_OK;
}

int fz_stream_create(void **s) { static int token; *s = &token; return FZ_OK; }
void *fz_upload_stream(void) { static int token; return &token; }
int fz_event_record(void **e, void *) { static int token; *e = &token; return FZ_OK; }
int fz_stream_wait_event(void *, void *) { return FZ_OK; }
int fz_event_destroy(void *) { return FZ_OK; }
int fz_stream_destroy(void *) { return FZ_OK; }
int fz_stream_wait(void *, void *) { return FZ_OK; }
int fz_gemm_set_tma_stores(int) { return FZ_OK; }
int fz_gemm_set_tiles(int mode) { return mode >= 0 && mode <= 2 ? FZ_OK : fail(FZ_ERR_INVALID, "fz_gemm_set_tiles: unknown mode"); }

int fz_tf32_lo(float *lo, const float *x, int64_t n, void *) {
  for (int64_t i = 0; i < n; ++i) lo[i] = tf32_lo1(x[i]);
  ++g_launches;
  return FZ_OK;
}

// A supplied lo plane must hold the remainders of the operand's current values:
// a stale plane (the host reusing one after the operand changed) is an error here.
static int check_lo(const float *X, const float *X_lo, int64_t rows, int64_t cols, int64_t ld,
                    int64_t sb, int64_t batch, const char *name) {
  if (!X_lo) return FZ_OK;
  for (int64_t b = 0; b < batch; ++b)
    for (int64_t r = 0; r < rows; ++r)
      for (int64_t c = 0; c < cols; ++c) {
        const int64_t o = b * sb + r * ld + c;
        const float want = tf32_lo1(X[o]);
        if (std::memcmp(&want, &X_lo[o], 4) != 0)
          return fail(FZ_ERR_INVALID, std::string("fz_gemm_f32_split: stale lo plane for ") + name);
      }
  return FZ_OK;
}

int fz_gemm_f32_split(int64_t batch, int64_t M, int64_t N, int64_t K, const float *A,
                      const float *A_lo, int64_t lda, int64_t sA, int tA, const float *B,
                      const float *B_lo, int64_t ldb, int64_t sB, int tB, float *C, int64_t ldc,
                      int64_t sC, void *st) {
  int rc = check_lo(A, A_lo, tA ? K : M, tA ? M : K, lda, sA, sA ? batch : 1, "A");
  if (!rc) rc = check_lo(B, B_lo, tB ? N : K, tB ? K : N, ldb, sB, sB ? batch : 1, "B");
  if (rc) return rc;
  return fz_gemm_f32(batch, M, N, K, A, lda, sA, tA, B, ldb, sB, tB, C, ldc, sC, st);
}

// Collectives. With a transport set (fake_comm_set_transport: a host callback that sums
// a buffer over the ranks of a host process group, e.g. gloo), communicators of more
// than one rank work and fz_comm_allreduce sums through it; otherwise world must be 1.
// Stream time is emulated for the watchdog: fz_stream_delay marks the streams busy for
// that long, and fz_comm_wait with a shorter timeout then aborts the communicator and
// fails as the real one does.
typedef int (*fake_allreduce_fn)(float *buf, int64_t n);
static fake_allreduce_fn g_transport = nullptr;
static double g_busy_s = 0.0;
struct FakeComm {
  int world;
  bool aborted;
};
void fake_comm_set_transport(fake_allreduce_fn fn) { g_transport = fn; }

int fz_stream_delay(void *, double seconds) {
  if (!(seconds >= 0.0 && seconds <= 60.0)) return fail(FZ_ERR_INVALID, "fz_stream_delay: seconds must be in [0, 60]");
  g_busy_s += seconds;
  return FZ_OK;
}
// Philox-4x32-10 (Salmon et al., SC'11), the device generator's stream layout.
static void philox(uint64_t ctr, uint64_t key, uint32_t c[4]) {
  c[0] = (uint32_t)ctr; c[1] = (uint32_t)(ctr >> 32); c[2] = 0; c[3] = 0;
  uint32_t k0 = (uint32_t)key, k1 = (uint32_t)(key >> 32);
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c[0], p1 = (uint64_t)0xCD9E8D57u * c[2];
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c[1] ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c[3] ^ k1;
    c[1] = (uint32_t)p1; c[3] = (uint32_t)p0; c[0] = n0; c[2] = n2;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
}
static float philox_unit(uint64_t seed, uint64_t i) {
  uint32_t c[4];
  philox(i / 4, seed, c);
  return (float)(c[i % 4] >> 8) * 5.9604644775390625e-08f;
}
int fz_philox_uniform(float *out, int64_t n, uint64_t seed, uint64_t offset, float lo, float hi, void *) {
  if (offset % 4 || !(lo < hi)) return fail(FZ_ERR_INVALID, "fz_philox_uniform: bad arguments");
  for (int64_t i = 0; i < n; ++i) {
    float v = std::fmaf(hi - lo, philox_unit(seed, offset + (uint64_t)i), lo);
    out[i] = v >= hi ? std::nextafterf(hi, lo) : v;
  }
  ++g_launches;
  return FZ_OK;
}
int fz_philox_dropout(float *out, const float *x, int64_t n, float rate, float keep, uint64_t seed,
                      uint64_t offset, void *) {
  if (offset % 4 || !(rate >= 0.0f && rate < 1.0f)) return fail(FZ_ERR_INVALID, "fz_philox_dropout: bad arguments");
  for (int64_t i = 0; i < n; ++i) {
    const float m = philox_unit(seed, offset + (uint64_t)i) > rate ? 1.0f : 0.0f;
    out[i] = (x[i] * m) / keep;
  }
  ++g_launches;
  return FZ_OK;
}

// Operators for training language models: plain loops in double, rounded once.
static double act_of(int a, double v) {
  if (a == FZ_ACT_RELU) return v > 0 ? v : 0.0;
  if (a == FZ_ACT_SILU) return v / (1 + std::exp(-v));
  if (a == FZ_ACT_GELU) return 0.5 * v * (1 + std::erf(v / std::sqrt(2.0)));
  return v;
}
static double slope_of(int a, double v) {
  if (a == FZ_ACT_RELU) return v > 0 ? 1.0 : 0.0;
  if (a == FZ_ACT_SILU) {
    const double s = 1 / (1 + std::exp(-v));
    return s * (1 + v * (1 - s));
  }
  if (a == FZ_ACT_GELU)
    return 0.5 * (1 + std::erf(v / std::sqrt(2.0))) + v * std::exp(-0.5 * v * v) * 0.3989422804014327;
  return 1.0;
}
int fz_group_norm_workspace(int64_t, int64_t, int64_t channels, int64_t groups, int, size_t *bytes) {
  *bytes = 64;
  return groups >= 1 && channels % groups == 0 ? FZ_OK : fail(FZ_ERR_INVALID, "fz_group_norm_workspace: bad sizes");
}
int fz_group_norm(float *y, float *mean, float *rstd, const float *x, const float *gamma, const float *beta,
                  int64_t batch, int64_t len, int64_t channels, int64_t groups, float eps, int act, void *work,
                  size_t bytes, void *) {
  if (!work || bytes < 64) return fail(FZ_ERR_INVALID, "fz_group_norm: workspace too small");
  const int64_t c = channels / groups;
  for (int64_t b = 0; b < batch; ++b)
    for (int64_t g = 0; g < groups; ++g) {
      double m = 0, v = 0;
      auto at = [&](int64_t l, int64_t i) { return (b * len + l) * channels + g * c + i; };
      for (int64_t l = 0; l < len; ++l)
        for (int64_t i = 0; i < c; ++i) m += x[at(l, i)];
      m /= (double)(len * c);
      for (int64_t l = 0; l < len; ++l)
        for (int64_t i = 0; i < c; ++i) v += (x[at(l, i)] - m) * (x[at(l, i)] - m);
      const double r = 1 / std::sqrt(v / (double)(len * c) + eps);
      if (mean) mean[b * groups + g] = (float)m, rstd[b * groups + g] = (float)r;
      for (int64_t l = 0; l < len; ++l)
        for (int64_t i = 0; i < c; ++i) {
          const double ga = gamma ? gamma[g * c + i] : 1.0, be = beta ? beta[g * c + i] : 0.0;
          y[at(l, i)] = (float)act_of(act, (x[at(l, i)] - m) * r * ga + be);
        }
    }
  ++g_launches;
  return FZ_OK;
}
int fz_group_norm_backward(float *dx, float *dgamma, float *dbeta, const float *dy, const float *x,
                           const float *mean, const float *rstd, const float *gamma, const float *beta,
                           int64_t batch, int64_t len, int64_t channels, int64_t groups, int act, void *work,
                           size_t bytes, void *) {
  if (!work || bytes < 64) return fail(FZ_ERR_INVALID, "fz_group_norm_backward: workspace too small");
  const int64_t c = channels / groups;
  std::vector<double> dg(channels, 0.0), db(channels, 0.0);
  for (int64_t b = 0; b < batch; ++b)
    for (int64_t g = 0; g < groups; ++g) {
      const double m = mean[b * groups + g], r = rstd[b * groups + g];
      double s1 = 0, s2 = 0;
      for (int pass = 0; pass < 2; ++pass)
        for (int64_t l = 0; l < len; ++l)
          for (int64_t i = 0; i < c; ++i) {
            const int64_t at = (b * len + l) * channels + g * c + i, ch = g * c + i;
            const double ga = gamma ? gamma[ch] : 1.0, xh = (x[at] - m) * r;
            const double dv = dy[at] * slope_of(act, xh * ga + (beta ? beta[ch] : 0.0)), a = dv * ga;
            if (!pass) {
              s1 += a;
              s2 += a * xh;
              dg[ch] += dv * xh;
              db[ch] += dv;
            } else {
              dx[at] = (float)(r * (a - (s1 + xh * s2) / (double)(len * c)));
            }
          }
    }
  for (int64_t ch = 0; ch < channels; ++ch) {
    if (dgamma) dgamma[ch] = (float)dg[ch];
    if (dbeta) dbeta[ch] = (float)db[ch];
  }
  ++g_launches;
  return FZ_OK;
}
int fz_route(float *w, int32_t *ids, const float *logits, int64_t tokens, int64_t experts, int64_t k, int renorm,
             void *) {
  for (int64_t t = 0; t < tokens; ++t) {
    const float *z = logits + t * experts;
    std::vector<bool> taken(experts, false);
    double den = 0;
    float top = -INFINITY;
    for (int64_t j = 0; j < k; ++j) {
      int64_t best = -1;
      for (int64_t e = 0; e < experts; ++e) {
        if (taken[e] || z[e] == -INFINITY) continue;
        if (best < 0 || (z[e] != z[e] && z[best] == z[best]) || z[e] > z[best]) best = e;
      }
      if (j == 0 && best >= 0) {
        top = z[best];
        if (!renorm)
          for (int64_t e = 0; e < experts; ++e) den += std::exp((double)z[e] - top);
      }
      ids[t * k + j] = (int32_t)best;
      const double num = best >= 0 ? std::exp((double)z[best] - top) : 0.0;
      if (best >= 0) taken[best] = true;
      if (renorm) den += num;
    }
    for (int64_t j = 0; j < k; ++j) {
      const int32_t e = ids[t * k + j];
      w[t * k + j] = e < 0 ? 0.0f : (float)(std::exp((double)z[e] - top) / den);
    }
  }
  ++g_launches;
  return FZ_OK;
}
int fz_route_backward(float *dl, const float *dw, const float *w, const int32_t *ids, const float *logits,
                      int64_t tokens, int64_t experts, int64_t k, int renorm, void *) {
  for (int64_t t = 0; t < tokens; ++t) {
    double dot = 0, den = 0, top = -INFINITY;
    bool any = false;
    for (int64_t j = 0; j < k; ++j)
      if (ids[t * k + j] >= 0) {
        dot += (double)w[t * k + j] * dw[t * k + j];
        any = true;
      }
    const float *z = logits + t * experts;
    for (int64_t e = 0; e < experts; ++e) top = z[e] > top ? z[e] : top;
    for (int64_t e = 0; e < experts; ++e) den += std::exp(z[e] - top);
    for (int64_t e = 0; e < experts; ++e) {
      double up = 0;
      for (int64_t j = 0; j < k; ++j)
        if (ids[t * k + j] == e) up = renorm ? w[t * k + j] * (dw[t * k + j] - dot) : dw[t * k + j];
      dl[t * experts + e] = (float)(renorm || !any ? up : std::exp(z[e] - top) / den * (up - dot));
    }
  }
  ++g_launches;
  return FZ_OK;
}
int fz_expert_sort(int32_t *slot, int32_t *src, int32_t *counts, int32_t *offsets, const int32_t *ids,
                   int64_t tokens, int64_t k, int64_t experts, int64_t capacity, void *) {
  const int64_t n = tokens * k, rows = capacity ? experts * capacity : n;
  for (int64_t e = 0; e < experts; ++e) counts[e] = 0;
  for (int64_t i = 0; i < n; ++i)
    if (ids[i] >= 0 && ids[i] < experts) ++counts[ids[i]];
  offsets[0] = 0;
  for (int64_t e = 0; e < experts; ++e) offsets[e + 1] = offsets[e] + (int32_t)(capacity ? capacity : counts[e]);
  std::vector<int32_t> used(experts, 0);
  for (int64_t r = 0; r < rows; ++r) src[r] = -1;
  for (int64_t i = 0; i < n; ++i) {
    slot[i] = -1;
    const int32_t e = ids[i];
    if (e < 0 || e >= experts) continue;
    const int32_t place = used[e]++;
    if (capacity && place >= capacity) continue;
    slot[i] = offsets[e] + place;
    src[slot[i]] = (int32_t)i;
  }
  ++g_launches;
  return FZ_OK;
}
int fz_expert_dispatch(float *rows, const float *x, const int32_t *, const int32_t *src, int64_t, int64_t k,
                       int64_t num_rows, int64_t width, void *) {
  for (int64_t r = 0; r < num_rows; ++r)
    for (int64_t c = 0; c < width; ++c) rows[r * width + c] = src[r] < 0 ? 0.0f : x[src[r] / k * width + c];
  ++g_launches;
  return FZ_OK;
}
int fz_expert_combine(float *out, const float *rows, const float *w, const int32_t *slot, int64_t tokens, int64_t k,
                      int64_t, int64_t width, void *) {
  for (int64_t t = 0; t < tokens; ++t)
    for (int64_t c = 0; c < width; ++c) {
      double s = 0;
      for (int64_t j = 0; j < k; ++j) {
        const int64_t r = slot[t * k + j];
        if (r >= 0) s += (w ? (double)w[t * k + j] : 1.0) * rows[r * width + c];
      }
      out[t * width + c] = (float)s;
    }
  ++g_launches;
  return FZ_OK;
}
int fz_expert_combine_backward(float *drows, float *dw, const float *dout, const float *rows, const float *w,
                               const int32_t *slot, const int32_t *src, int64_t tokens, int64_t k, int64_t num_rows,
                               int64_t width, void *) {
  for (int64_t r = 0; r < num_rows; ++r)
    for (int64_t c = 0; c < width; ++c)
      drows[r * width + c] = src[r] < 0 ? 0.0f : (w ? w[src[r]] : 1.0f) * dout[src[r] / k * width + c];
  for (int64_t i = 0; dw && i < tokens * k; ++i) {
    double s = 0;
    for (int64_t c = 0; slot[i] >= 0 && c < width; ++c) s += (double)dout[i / k * width + c] * rows[slot[i] * width + c];
    dw[i] = (float)s;
  }
  ++g_launches;
  return FZ_OK;
}
// p (per entry, 0 for padding), the teacher's mass and tail; false if the row has no entries.
static bool teacher_of(const int32_t *ids, const float *t, const float *lse, int64_t vocab, int64_t k, double tau,
                       std::vector<double> &p, std::vector<double> &logp, double &mass, double &tail) {
  double top = -INFINITY, sum = 0;
  bool any = false;
  for (int64_t i = 0; i < k; ++i)
    if (ids[i] >= 0 && ids[i] < vocab && (lse || t[i] != -INFINITY)) {
      any = true;
      top = t[i] > top ? t[i] : top;
    }
  mass = tail = 0;
  if (!any) return false;
  for (int64_t i = 0; i < k; ++i)
    if (ids[i] >= 0 && ids[i] < vocab) sum += std::exp((t[i] - top) / tau);
  for (int64_t i = 0; i < k; ++i) {
    const bool ok = ids[i] >= 0 && ids[i] < vocab;
    logp[i] = lse ? t[i] / tau - *lse : (t[i] - top) / tau - std::log(sum);
    p[i] = ok ? std::exp(logp[i]) : 0.0;
    mass += p[i];
  }
  if (lse && mass < 1) tail = 1 - mass;
  mass += tail;
  return true;
}
int fz_distill(float *loss, float *stats, const float *logits, int64_t ld, const int32_t *ids, const float *teacher,
               const float *lse, int64_t rows, int64_t vocab, int64_t k, float tau, void *) {
  std::vector<double> p(k), logp(k);
  for (int64_t r = 0; r < rows; ++r) {
    double mass, tail, l = 0;
    const float *z = logits + r * ld;
    float *st = stats + r * 4;
    loss[r] = st[0] = st[1] = st[2] = st[3] = 0.0f;
    if (!teacher_of(ids + r * k, teacher + r * k, lse ? lse + r : nullptr, vocab, k, tau, p, logp, mass, tail)) continue;
    std::set<int64_t> inside;
    for (int64_t i = 0; i < k; ++i) inside.insert(ids[r * k + i]);
    double m = -INFINITY, tm = -INFINITY, s = 0, ts = 0;
    for (int64_t v = 0; v < vocab; ++v) {
      m = z[v] > m ? z[v] : m;
      if (!inside.count(v)) tm = z[v] > tm ? z[v] : tm;
    }
    for (int64_t v = 0; v < vocab; ++v) {
      s += std::exp((z[v] - m) / tau);
      if (!inside.count(v)) ts += std::exp((z[v] - tm) / tau);
    }
    for (int64_t i = 0; i < k; ++i)
      if (p[i] != 0) l += p[i] * (logp[i] - ((z[ids[r * k + i]] - m) / tau - std::log(s)));
    if (tail != 0) l += tail * (std::log(tail) - ((tm - m) / tau + std::log(ts) - std::log(s)));
    loss[r] = (float)(tau * tau * l);
    st[0] = (float)m, st[1] = (float)std::log(s), st[2] = (float)tm, st[3] = (float)std::log(ts);
  }
  ++g_launches;
  return FZ_OK;
}
int fz_distill_backward(float *dz, int64_t ldd, const float *dloss, const float *stats, const float *logits,
                        int64_t ld, const int32_t *ids, const float *teacher, const float *lse, int64_t rows,
                        int64_t vocab, int64_t k, float tau, void *) {
  std::vector<double> p(k), logp(k);
  for (int64_t r = 0; r < rows; ++r) {
    double mass, tail;
    const float *z = logits + r * ld, *st = stats + r * 4;
    const bool any = teacher_of(ids + r * k, teacher + r * k, lse ? lse + r : nullptr, vocab, k, tau, p, logp, mass, tail);
    std::map<int64_t, double> inside;
    for (int64_t i = 0; any && i < k; ++i)
      if (ids[r * k + i] >= 0) inside[ids[r * k + i]] += p[i];
    for (int64_t v = 0; v < vocab; ++v) {
      double g = any ? mass * std::exp((z[v] - (double)st[0]) / tau - st[1]) : 0.0;
      if (inside.count(v)) g -= inside[v];
      else if (tail != 0) g -= tail * std::exp((z[v] - (double)st[2]) / tau - st[3]);
      dz[r * ldd + v] = any ? (float)(tau * dloss[r] * g) : 0.0f;
    }
  }
  ++g_launches;
  return FZ_OK;
}

int fz_comm_unique_id(unsigned char id[FZ_UNIQUE_ID_BYTES]) { std::memset(id, 0, FZ_UNIQUE_ID_BYTES); return FZ_OK; }
int fz_comm_init(void **c, int world, int, const unsigned char *) {
  if (world != 1 && !g_transport) return fail(FZ_ERR_UNSUPPORTED, "host test double: world must be 1");
  *c = new FakeComm{world, false};
  return FZ_OK;
}
int fz_comm_allreduce(void *comm, const float *s, float *r, int64_t n, float scale, void *) {
  FakeComm *c = static_cast<FakeComm *>(comm);
  if (c->aborted) return fail(FZ_ERR_INVALID, "fz_comm_allreduce: communicator was aborted");
  if (r != s) std::memmove(r, s, sizeof(float) * (size_t)n);
  if (c->world > 1 && g_transport(r, n) != 0) return fail(FZ_ERR_NCCL, "host transport failed");
  for (int64_t i = 0; i < n; ++i) r[i] = r[i] * scale;
  return FZ_OK;
}
int fz_comm_group_start(void) { return FZ_OK; }
int fz_comm_group_end(void) { return FZ_OK; }
int fz_comm_broadcast(void *, float *, int64_t, int, void *) { return FZ_OK; }
int fz_comm_wait(void *comm, void *, double timeout_s) {
  FakeComm *c = static_cast<FakeComm *>(comm);
  const bool late = g_busy_s > timeout_s;
  g_busy_s = 0.0;
  if (late) {
    c->aborted = true;
    return fail(FZ_ERR_TIMEOUT, "collective did not complete within " + std::to_string(timeout_s) +
                                    " s; communicator aborted");
  }
  return FZ_OK;
}
int fz_comm_destroy(void *c) { delete static_cast<FakeComm *>(c); return FZ_OK; }

}  // extern "C"
