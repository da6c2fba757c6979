// Operators for training language models over the B200 tensor: group norm with an
// activation (channels last), the router's gate, tokens sorted by expert and back, and
// distillation from a teacher's top logits. No reference counterpart. The functions here
// run on values; autodiff.cpp traces them (OpKind::GroupNorm .. OpKind::Distill).
// They run when called, on the thread's stream, and lower their pending inputs first.
#pragma once

#include <memory>
#include <string>
#include <vector>

#include "tensor.hpp"

namespace fusion_b200 {

// An immutable int32 array on the device: expert choices, rows, token ids. Fusion's
// tensors are fp32 throughout, so whole numbers have a type of their own.
class Indices {
 public:
  Indices() = default;
  // From host values (copied to the device).
  Indices(std::vector<size_t> shape, const std::vector<int32_t> &values, Device device);
  // Of the given shape on the current device, to be written by a kernel.
  Indices(std::vector<size_t> shape, Device device);
  const std::vector<size_t> &shape() const { return shape_; }
  size_t size() const;
  Device device() const { return device_; }
  bool is_initialised() const { return buf_ != nullptr; }
  int32_t *data() const { return buf_ ? reinterpret_cast<int32_t *>(buf_->ptr) : nullptr; }
  int cuda_device() const { return buf_ ? buf_->device : 0; }
  void to_host(int32_t *dst) const;

 private:
  std::vector<size_t> shape_;
  std::shared_ptr<DeviceBuffer> buf_;
  Device device_{};
};

// Where each choice of a batch of tokens goes when sorted by expert (fz_expert_sort).
struct ExpertPlan {
  Indices ids, slot, src, counts, offsets;
  int64_t tokens = 0, k = 0, experts = 0, capacity = 0, rows = 0;
  // ids [..., k]; capacity 0 packs the experts' rows, else gives each that many.
  ExpertPlan(const Indices &ids, int64_t experts, int64_t capacity);
  std::vector<size_t> token_shape() const;  // ids' shape without its last axis
};

struct GroupNormStats {
  RawTensor y, mean, rstd;
};
struct DistillStats {
  RawTensor loss, stats;
};

int activation_code(const std::string &name);  // "none", "relu", "silu", "gelu"

namespace math {
// x [batch, ..., channels]; gamma and beta [channels], or both uninitialised.
GroupNormStats group_norm(const RawTensor &x, const RawTensor &gamma, const RawTensor &beta, int64_t groups,
                          float eps, int act);
// dx, dgamma, dbeta (the last two uninitialised unless `params`).
std::vector<RawTensor> group_norm_backward(const RawTensor &dy, const RawTensor &x, const GroupNormStats &s,
                                           const RawTensor &gamma, const RawTensor &beta, int64_t groups, int act,
                                           bool params);
// logits [..., experts] -> weights [..., k], ids [..., k].
std::pair<RawTensor, Indices> route(const RawTensor &logits, int64_t k, bool renormalize);
RawTensor route_backward(const RawTensor &dweights, const RawTensor &weights, const Indices &ids,
                         const RawTensor &logits, bool renormalize);
// x [..., width] -> rows [experts, capacity, width], or [rows, width] packed.
RawTensor expert_dispatch(const RawTensor &x, const ExpertPlan &plan);
// rows [..., width] -> [token shape..., width]; weights [..., k] or uninitialised (ones).
RawTensor expert_combine(const RawTensor &rows, const RawTensor &weights, const ExpertPlan &plan,
                         const std::vector<size_t> &out_shape);
// drows in rows' shape, dweights (uninitialised unless wanted) in weights' shape.
std::vector<RawTensor> expert_combine_backward(const RawTensor &dout, const RawTensor &rows,
                                               const RawTensor &weights, const ExpertPlan &plan, bool want_weights);
// logits [..., vocab], ids and teacher [..., k], teacher_lse [...] or uninitialised.
DistillStats distill(const RawTensor &logits, const Indices &ids, const RawTensor &teacher,
                     const RawTensor &teacher_lse, float temperature);
RawTensor distill_backward(const RawTensor &dloss, const RawTensor &stats, const RawTensor &logits,
                           const Indices &ids, const RawTensor &teacher, const RawTensor &teacher_lse,
                           float temperature);
}  // namespace math

// What the traced operators take besides their differentiable inputs.
struct LearnParam {
  int64_t groups = 1, k = 1;
  float eps = 0.0f, temperature = 1.0f;
  int act = 0;
  bool renormalize = true;
  std::shared_ptr<const ExpertPlan> plan;
  Indices ids;  // Distill: the teacher's; Route: written by the forward
  RawTensor teacher, teacher_lse;
  std::vector<size_t> shape;  // Combine: the result's
};

}  // namespace fusion_b200
