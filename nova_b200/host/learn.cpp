// The language-model training operators on values (see learn.hpp).
#include "learn.hpp"

#include <limits>
#include <numeric>

namespace fusion_b200 {

namespace {

size_t product(const std::vector<size_t> &s, size_t from, size_t to) {
  return std::accumulate(s.begin() + from, s.begin() + to, (size_t)1, std::multiplies<size_t>());
}

// The device pointer of an operand, materialised; every operand of a call has to live on
// the device that is current (bind_device of the first).
const float *operand(const RawTensor &t, const char *what) {
  FB_CHECK(t.is_initialised(), std::string(what) + ": uninitialised tensor");
  FB_CHECK(t.dtype() == DType::FLOAT32, std::string(what) + ": tensors must be FLOAT32");
  const float *p = t.data();
  int cur = 0;
  fz_check(fz_get_device(&cur), "fz_get_device");
  FB_CHECK(t.size() == 0 || t.expr()->buf->device == cur, std::string(what) + ": operands on different devices");
  return p;
}

const int32_t *operand(const Indices &t, const char *what) {
  FB_CHECK(t.is_initialised(), std::string(what) + ": uninitialised indices");
  int cur = 0;
  fz_check(fz_get_device(&cur), "fz_get_device");
  FB_CHECK(t.size() == 0 || t.cuda_device() == cur, std::string(what) + ": operands on different devices");
  return t.data();
}

RawTensor result(std::shared_ptr<DeviceBuffer> buf, std::vector<size_t> shape, Device device) {
  return RawTensor::from_buffer(std::move(buf), std::move(shape), DType::FLOAT32, device);
}

std::shared_ptr<DeviceBuffer> buffer(size_t n) { return std::make_shared<DeviceBuffer>(n); }

void check_norm(const RawTensor &x, const RawTensor &gamma, const RawTensor &beta, int64_t groups) {
  FB_CHECK(x.is_initialised() && x.rank() >= 2, "group_norm: x must be [batch, ..., channels]");
  const size_t c = x.shape().back();
  FB_CHECK(groups >= 1 && c >= 1 && c % (size_t)groups == 0, "group_norm: channels must be a multiple of groups");
  FB_CHECK(gamma.is_initialised() == beta.is_initialised(), "group_norm: gamma and beta go together");
  FB_CHECK(!gamma.is_initialised() || (gamma.size() == c && beta.size() == c),
           "group_norm: gamma and beta must hold one value a channel");
}

}  // namespace

int activation_code(const std::string &name) {
  if (name == "none") return FZ_ACT_NONE;
  if (name == "relu") return FZ_ACT_RELU;
  if (name == "silu") return FZ_ACT_SILU;
  if (name == "gelu") return FZ_ACT_GELU;
  throw std::invalid_argument("unknown activation '" + name + "': none, relu, silu or gelu");
}

// ---------------------------------------------------------------- indices
Indices::Indices(std::vector<size_t> shape, Device device) : shape_(std::move(shape)), device_(device) {
  FB_CHECK(!shape_.empty(), "Indices: empty shape");
  bind_device(device_);
  buf_ = buffer(size());
}

Indices::Indices(std::vector<size_t> shape, const std::vector<int32_t> &values, Device device)
    : Indices(std::move(shape), device) {
  FB_CHECK(values.size() == size(), "Indices: data size != product(shape)");
  if (values.empty()) return;
  fz_check(fz_memcpy_h2d(buf_->ptr, values.data(), values.size() * sizeof(int32_t), nullptr), "fz_memcpy_h2d");
  fz_check(fz_stream_sync(nullptr), "fz_stream_sync");  // `values` may go away on return
}

size_t Indices::size() const { return shape_.empty() ? 0 : product(shape_, 0, shape_.size()); }

void Indices::to_host(int32_t *dst) const {
  if (!size()) return;
  bind_device(device_);
  fz_check(fz_memcpy_d2h(dst, buf_->ptr, size() * sizeof(int32_t), nullptr), "fz_memcpy_d2h");
}

// ---------------------------------------------------------------- experts
ExpertPlan::ExpertPlan(const Indices &i, int64_t e, int64_t cap) : ids(i), experts(e), capacity(cap) {
  FB_CHECK(ids.is_initialised() && ids.shape().size() >= 1, "ExpertPlan: uninitialised ids");
  bind_device(ids.device());
  k = (int64_t)ids.shape().back();
  FB_CHECK(k >= 1, "ExpertPlan: ids must be [..., k] with k >= 1");
  FB_CHECK(experts >= 1 && experts <= FZ_MAX_EXPERTS, "ExpertPlan: experts must be in [1, 1024]");
  FB_CHECK(capacity >= 0 && capacity <= std::numeric_limits<int32_t>::max() / experts,
           "ExpertPlan: capacity must not be negative, and experts * capacity below 2^31");
  tokens = (int64_t)ids.size() / k;
  FB_CHECK(tokens <= std::numeric_limits<int32_t>::max() / k, "ExpertPlan: tokens * k must be below 2^31");
  rows = capacity ? experts * capacity : tokens * k;
  const int32_t *p = operand(ids, "ExpertPlan");
  slot = Indices(ids.shape(), ids.device());
  src = Indices({(size_t)rows}, ids.device());
  counts = Indices({(size_t)experts}, ids.device());
  offsets = Indices({(size_t)experts + 1}, ids.device());
  fz_check(fz_expert_sort(slot.data(), src.data(), counts.data(), offsets.data(), p, tokens, k, experts, capacity,
                          nullptr),
           "fz_expert_sort");
}

std::vector<size_t> ExpertPlan::token_shape() const {
  return std::vector<size_t>(ids.shape().begin(), ids.shape().end() - 1);
}

namespace math {

// ---------------------------------------------------------------- group norm
GroupNormStats group_norm(const RawTensor &x, const RawTensor &gamma, const RawTensor &beta, int64_t groups,
                          float eps, int act) {
  check_norm(x, gamma, beta, groups);
  FB_CHECK(eps >= 0.0f, "group_norm: eps must not be negative");
  bind_device(x.device());
  const float *px = operand(x, "group_norm");
  const float *pg = gamma.is_initialised() ? operand(gamma, "group_norm") : nullptr;
  const float *pb = beta.is_initialised() ? operand(beta, "group_norm") : nullptr;
  const auto &s = x.shape();
  const int64_t batch = (int64_t)s[0], c = (int64_t)s.back(), len = (int64_t)product(s, 1, s.size() - 1);
  size_t bytes = 0;
  fz_check(fz_group_norm_workspace(batch, len, c, groups, 0, &bytes), "fz_group_norm_workspace");
  DeviceBuffer work((bytes + 3) / 4);
  auto y = buffer(x.size()), mean = buffer((size_t)(batch * groups)), rstd = buffer((size_t)(batch * groups));
  fz_check(fz_group_norm(y->ptr, mean->ptr, rstd->ptr, px, pg, pb, batch, len, c, groups, eps, act, work.ptr, bytes,
                         nullptr),
           "fz_group_norm");
  const std::vector<size_t> stat{(size_t)batch, (size_t)groups};
  return {result(y, s, x.device()), result(mean, stat, x.device()), result(rstd, stat, x.device())};
}

std::vector<RawTensor> group_norm_backward(const RawTensor &dy, const RawTensor &x, const GroupNormStats &st,
                                           const RawTensor &gamma, const RawTensor &beta, int64_t groups, int act,
                                           bool params) {
  FB_CHECK(dy.size() == x.size(), "group_norm: gradient size mismatch");
  bind_device(x.device());
  const float *px = operand(x, "group_norm"), *pd = operand(dy, "group_norm");
  const float *pg = gamma.is_initialised() ? operand(gamma, "group_norm") : nullptr;
  const float *pb = beta.is_initialised() ? operand(beta, "group_norm") : nullptr;
  const auto &s = x.shape();
  const int64_t batch = (int64_t)s[0], c = (int64_t)s.back(), len = (int64_t)product(s, 1, s.size() - 1);
  size_t bytes = 0;
  fz_check(fz_group_norm_workspace(batch, len, c, groups, 1, &bytes), "fz_group_norm_workspace");
  DeviceBuffer work((bytes + 3) / 4);
  auto dx = buffer(x.size());
  std::shared_ptr<DeviceBuffer> dg, db;
  if (params) dg = buffer((size_t)c), db = buffer((size_t)c);
  fz_check(fz_group_norm_backward(dx->ptr, dg ? dg->ptr : nullptr, db ? db->ptr : nullptr, pd, px, st.mean.data(),
                                  st.rstd.data(), pg, pb, batch, len, c, groups, act, work.ptr, bytes, nullptr),
           "fz_group_norm_backward");
  return {result(dx, s, x.device()), dg ? result(dg, gamma.shape(), x.device()) : RawTensor(),
          db ? result(db, beta.shape(), x.device()) : RawTensor()};
}

// ---------------------------------------------------------------- router
std::pair<RawTensor, Indices> route(const RawTensor &logits, int64_t k, bool renormalize) {
  FB_CHECK(logits.is_initialised() && logits.rank() >= 1, "route: logits must be [..., experts]");
  bind_device(logits.device());
  const auto &s = logits.shape();
  const int64_t experts = (int64_t)s.back(), tokens = (int64_t)product(s, 0, s.size() - 1);
  FB_CHECK(experts >= 1 && experts <= FZ_MAX_EXPERTS, "route: experts must be in [1, 1024]");
  FB_CHECK(k >= 1 && k <= experts && k <= FZ_MAX_CHOICES, "route: k must be in [1, min(experts, 32)]");
  const float *p = operand(logits, "route");
  std::vector<size_t> out(s.begin(), s.end() - 1);
  out.push_back((size_t)k);
  auto w = buffer((size_t)(tokens * k));
  Indices ids(out, logits.device());
  fz_check(fz_route(w->ptr, ids.data(), p, tokens, experts, k, renormalize, nullptr), "fz_route");
  return {result(w, out, logits.device()), ids};
}

RawTensor route_backward(const RawTensor &dweights, const RawTensor &weights, const Indices &ids,
                         const RawTensor &logits, bool renormalize) {
  FB_CHECK(dweights.size() == weights.size(), "route: gradient size mismatch");
  bind_device(logits.device());
  const auto &s = logits.shape();
  const int64_t experts = (int64_t)s.back(), tokens = (int64_t)product(s, 0, s.size() - 1);
  const float *pd = operand(dweights, "route"), *pw = operand(weights, "route"), *pl = operand(logits, "route");
  auto dl = buffer(logits.size());
  fz_check(fz_route_backward(dl->ptr, pd, pw, operand(ids, "route"), pl, tokens, experts,
                             (int64_t)weights.shape().back(), renormalize, nullptr),
           "fz_route_backward");
  return result(dl, s, logits.device());
}

// ---------------------------------------------------------------- dispatch and combine
RawTensor expert_dispatch(const RawTensor &x, const ExpertPlan &plan) {
  FB_CHECK(x.is_initialised() && x.rank() >= 1, "expert_dispatch: x must be [..., width]");
  const size_t width = x.shape().back();
  FB_CHECK(product(x.shape(), 0, x.rank() - 1) == (size_t)plan.tokens,
           "expert_dispatch: x and the plan have different numbers of tokens");
  bind_device(x.device());
  const float *p = operand(x, "expert_dispatch");
  std::vector<size_t> shape = plan.capacity
                                  ? std::vector<size_t>{(size_t)plan.experts, (size_t)plan.capacity, width}
                                  : std::vector<size_t>{(size_t)plan.rows, width};
  auto rows = buffer((size_t)plan.rows * width);
  fz_check(fz_expert_dispatch(rows->ptr, p, operand(plan.slot, "expert_dispatch"),
                              operand(plan.src, "expert_dispatch"), plan.tokens, plan.k, plan.rows, (int64_t)width,
                              nullptr),
           "fz_expert_dispatch");
  return result(rows, shape, x.device());
}

static void check_combine(const RawTensor &rows, const RawTensor &weights, const ExpertPlan &plan) {
  FB_CHECK(rows.is_initialised() && rows.rank() >= 2, "expert_combine: rows must be [..., width]");
  FB_CHECK(product(rows.shape(), 0, rows.rank() - 1) == (size_t)plan.rows,
           "expert_combine: rows and the plan have different numbers of rows");
  FB_CHECK(!weights.is_initialised() || weights.size() == (size_t)(plan.tokens * plan.k),
           "expert_combine: weights must hold one value a choice");
}

RawTensor expert_combine(const RawTensor &rows, const RawTensor &weights, const ExpertPlan &plan,
                         const std::vector<size_t> &out_shape) {
  check_combine(rows, weights, plan);
  const size_t width = rows.shape().back();
  FB_CHECK(product(out_shape, 0, out_shape.size()) == (size_t)plan.tokens * width,
           "expert_combine: result shape mismatch");
  bind_device(rows.device());
  const float *p = operand(rows, "expert_combine");
  const float *w = weights.is_initialised() ? operand(weights, "expert_combine") : nullptr;
  auto out = buffer((size_t)plan.tokens * width);
  fz_check(fz_expert_combine(out->ptr, p, w, operand(plan.slot, "expert_combine"), plan.tokens, plan.k, plan.rows,
                             (int64_t)width, nullptr),
           "fz_expert_combine");
  return result(out, out_shape, rows.device());
}

std::vector<RawTensor> expert_combine_backward(const RawTensor &dout, const RawTensor &rows,
                                               const RawTensor &weights, const ExpertPlan &plan,
                                               bool want_weights) {
  check_combine(rows, weights, plan);
  const size_t width = rows.shape().back();
  FB_CHECK(dout.size() == (size_t)plan.tokens * width, "expert_combine: gradient size mismatch");
  bind_device(rows.device());
  const float *pd = operand(dout, "expert_combine"), *p = operand(rows, "expert_combine");
  const float *w = weights.is_initialised() ? operand(weights, "expert_combine") : nullptr;
  auto drows = buffer(rows.size());
  std::shared_ptr<DeviceBuffer> dw;
  if (want_weights && weights.is_initialised()) dw = buffer(weights.size());
  fz_check(fz_expert_combine_backward(drows->ptr, dw ? dw->ptr : nullptr, pd, p, w,
                                      operand(plan.slot, "expert_combine"), operand(plan.src, "expert_combine"),
                                      plan.tokens, plan.k, plan.rows, (int64_t)width, nullptr),
           "fz_expert_combine_backward");
  return {result(drows, rows.shape(), rows.device()),
          dw ? result(dw, weights.shape(), rows.device()) : RawTensor()};
}

// ---------------------------------------------------------------- distillation
DistillStats distill(const RawTensor &logits, const Indices &ids, const RawTensor &teacher,
                     const RawTensor &teacher_lse, float temperature) {
  FB_CHECK(logits.is_initialised() && logits.rank() >= 1, "distill: logits must be [..., vocab]");
  const auto &s = logits.shape();
  const size_t vocab = s.back(), rows = product(s, 0, s.size() - 1);
  FB_CHECK(ids.is_initialised() && teacher.is_initialised() && ids.shape() == teacher.shape(),
           "distill: ids and teacher must have the same shape [..., k]");
  const size_t k = ids.shape().back();
  FB_CHECK(k >= 1 && k <= FZ_MAX_TEACHER, "distill: a list must have 1 to 1024 entries");
  FB_CHECK(product(ids.shape(), 0, ids.shape().size() - 1) == rows,
           "distill: logits and ids have different numbers of rows");
  FB_CHECK(!teacher_lse.is_initialised() || teacher_lse.size() == rows,
           "distill: teacher_lse must hold one value a row");
  FB_CHECK(vocab >= 1 && vocab <= ((size_t)1 << 23), "distill: vocab must be in [1, 2^23]");
  bind_device(logits.device());
  const float *pz = operand(logits, "distill"), *pt = operand(teacher, "distill");
  const float *pl = teacher_lse.is_initialised() ? operand(teacher_lse, "distill") : nullptr;
  auto loss = buffer(rows), stats = buffer(rows * 4);
  fz_check(fz_distill(loss->ptr, stats->ptr, pz, (int64_t)vocab, operand(ids, "distill"), pt, pl, (int64_t)rows,
                      (int64_t)vocab, (int64_t)k, temperature, nullptr),
           "fz_distill");
  std::vector<size_t> shape(s.begin(), s.end() - 1);
  if (shape.empty()) shape.push_back(1);
  return {result(loss, shape, logits.device()), result(stats, {rows, 4}, logits.device())};
}

RawTensor distill_backward(const RawTensor &dloss, const RawTensor &stats, const RawTensor &logits,
                           const Indices &ids, const RawTensor &teacher, const RawTensor &teacher_lse,
                           float temperature) {
  const size_t vocab = logits.shape().back(), rows = product(logits.shape(), 0, logits.rank() - 1);
  FB_CHECK(dloss.size() == rows, "distill: gradient size mismatch");
  bind_device(logits.device());
  const float *pd = operand(dloss, "distill"), *pz = operand(logits, "distill"), *pt = operand(teacher, "distill");
  const float *pl = teacher_lse.is_initialised() ? operand(teacher_lse, "distill") : nullptr;
  auto dz = buffer(logits.size());
  fz_check(fz_distill_backward(dz->ptr, (int64_t)vocab, pd, operand(stats, "distill"), pz, (int64_t)vocab,
                               operand(ids, "distill"), pt, pl, (int64_t)rows, (int64_t)vocab,
                               (int64_t)ids.shape().back(), temperature, nullptr),
           "fz_distill_backward");
  return result(dz, logits.shape(), logits.device());
}

}  // namespace math
}  // namespace fusion_b200
