// The `hip` dialect's OpEnvs of the operators at the vocabulary: raf.op.embedding and
// raf.op.embedding_dx (in the reference EmbeddingImpl and EmbeddingDxImpl,
// src/op/dialect/cuda/embedding.cc), and the extension ops raf.op.topk_distill, _dx and _step.  They
// call the gfx950 kernels through the C ABI of rafhip_vocab.h only.
//
// As in hip_dialect.cc the stream is looked up at Execute time, arguments that the kernels do not
// take are reported through error_msgs, and an OpEnv requests one workspace.
#include <algorithm>
#include <sstream>

#include "raf_iface.h"
#include "rafhip_vocab.h"

namespace raf {
namespace op {
namespace hip {

using device_api::DeviceAPI;
using value::AsTensor;
using value::AsTuple;
using value::Value;

namespace {

void Check(const char* what, int status) {
  if (status == RAFHIP_OK) return;
  std::ostringstream ss;
  ss << what << " failed with status " << status << ": " << rafhip_last_error();
  throw Error(ss.str());
}

int32_t KernelDType(const DType& t) {
  if (t.code == kDLFloat) return t.bits == 32 ? RAFHIP_F32 : t.bits == 16 ? RAFHIP_F16 : -1;
  return t.code == kDLBfloat && t.bits == 16 ? RAFHIP_BF16 : -1;
}

void* Stream() { return DeviceAPI::Get(DevType::kROCM())->GetStream(); }

}  // namespace

// What the OpEnvs below share: the op's name, the checks every one of them makes, the workspace.
class VocabHipEnv : public OpEnv {
 public:
  explicit VocabHipEnv(const char* op) : op_(op), name_(TruncateName(GetUniqueName(op))) {}
  std::string name() const override { return name_; }

 protected:
  void RequireDevice(const CallValues& cv) {
    if (cv->device.device_type() != DevType::kROCM()) error_msgs.push_back(op_ + ": device is not rocm");
    if (error_msgs.empty() && rafhip_device_count() <= 0) error_msgs.push_back(op_ + ": no HIP device is visible");
  }
  void RequireDType(int32_t dtype, const char* what) {
    if (dtype < 0) error_msgs.push_back(op_ + ": unsupported dtype of " + what);
  }
  void RequireWorkspace(const CallValues& cv, int64_t bytes) {
    if (!error_msgs.empty()) return;
    if (bytes < 0) {
      const std::string why = rafhip_last_error();
      error_msgs.push_back(op_ + ": unsupported sizes" + (why.empty() ? "" : ": " + why));
      return;
    }
    workspace_bytes_ = bytes;
    if (bytes > 0) RequestWorkspace(&workspace_, cv->device, bytes);
  }
  // The inputs and outputs of an Execute have the shapes, dtypes and devices that the OpEnv was made
  // for: the kernels take them from there.
  const TensorView& Same(const Value& v, const TensorView& made_for, const char* what) const {
    const TensorView& t = AsTensor(v)->tensor;
    RAF_CHECK(t.shape == made_for.shape, op_ + ": the shape of " + what + " changed since the OpEnv was made");
    RAF_CHECK(t.dtype.code == made_for.dtype.code && t.dtype.bits == made_for.dtype.bits,
              op_ + ": the dtype of " + what + " changed since the OpEnv was made");
    RAF_CHECK(t.device.device_type() == made_for.device.device_type() && t.device.device_id() == made_for.device.device_id(),
              op_ + ": the device of " + what + " changed since the OpEnv was made");
    return t;
  }

  std::string op_, name_;
  void* workspace_ = nullptr;
  int64_t workspace_bytes_ = 0;
};

class EmbeddingHipEnv : public VocabHipEnv {
 public:
  explicit EmbeddingHipEnv(const CallValues& cv) : VocabHipEnv("raf.op.hip.embedding") {
    const auto* args = cv->args_as<schema::EmbeddingArgs>();
    if (!args) {
      error_msgs.push_back(op_ + ": call does not carry EmbeddingArgs");
      return;
    }
    arg_indices = {args->FieldIndex("x"), args->FieldIndex("indices")};
    x_ = args->x->tensor;
    ids_ = args->indices->tensor;
    out_ = AsTensor(cv->out)->tensor;
    x_dtype_ = KernelDType(x_.dtype);
    out_dtype_ = KernelDType(args->out_dtype);
    scale_ = (float)args->scale;
    first_row_ = args->first_row;
    RequireDType(x_dtype_, "x");
    RequireDType(out_dtype_, "the output");
    RequireDevice(cv);
  }

  void Execute(const CallValues& cv) override {
    const auto* args = cv->args_as<schema::EmbeddingArgs>();
    RAF_CHECK(args != nullptr, op_ + " expects EmbeddingArgs");
    Execute(std::vector<Value>{args->x, args->indices}, cv->out);
  }

  void Execute(const std::vector<Value>& inputs, Value output) override {
    RAF_CHECK(inputs.size() == 2, op_ + " takes x and indices");
    const TensorView& x = Same(inputs[0], x_, "x");
    const TensorView& ids = Same(inputs[1], ids_, "indices");
    const TensorView& out = Same(output, out_, "the output");
    Check("rafhip_embedding",
          rafhip_embedding(x.data, x_dtype_, x.shape[0], x.shape[1], ids.data, ids.dtype.bits, ids.numel(), first_row_,
                           scale_, out.data, out_dtype_, Stream()));
  }

  static OpEnv* make(const CallValues& cv) { return new EmbeddingHipEnv(cv); }

 private:
  TensorView x_, ids_, out_;
  int32_t x_dtype_ = -1, out_dtype_ = -1;
  float scale_ = 1.f;
  int64_t first_row_ = 0;
};

class EmbeddingDxHipEnv : public VocabHipEnv {
 public:
  explicit EmbeddingDxHipEnv(const CallValues& cv) : VocabHipEnv("raf.op.hip.embedding_dx") {
    const auto* args = cv->args_as<schema::EmbeddingDxArgs>();
    if (!args) {
      error_msgs.push_back(op_ + ": call does not carry EmbeddingDxArgs");
      return;
    }
    arg_indices = {args->FieldIndex("dy"), args->FieldIndex("indices"), args->FieldIndex("grad")};
    args_ = *args;
    dy_ = args->dy->tensor;
    ids_ = args->indices->tensor;
    out_ = AsTensor(cv->out)->tensor;
    dy_dtype_ = KernelDType(args->dy->tensor.dtype);
    out_dtype_ = KernelDType(args->out_dtype);
    RequireDType(dy_dtype_, "dy");
    RequireDType(out_dtype_, "the output");
    RequireDevice(cv);
    RequireWorkspace(cv, rafhip_embedding_dx_workspace_bytes(args->indices->tensor.numel(), out_.shape[0], out_.shape[1]));
  }

  void Execute(const CallValues& cv) override {
    const auto* args = cv->args_as<schema::EmbeddingDxArgs>();
    RAF_CHECK(args != nullptr, op_ + " expects EmbeddingDxArgs");
    Execute(std::vector<Value>{args->dy, args->indices, args->grad}, cv->out);
  }

  void Execute(const std::vector<Value>& inputs, Value output) override {
    RAF_CHECK(inputs.size() == 3, op_ + " takes dy, indices and grad");
    const TensorView& dy = Same(inputs[0], dy_, "dy");
    const TensorView& ids = Same(inputs[1], ids_, "indices");
    const TensorView& out = Same(output, out_, "the output");
    RAF_CHECK((inputs[2] != nullptr) == (args_.grad != nullptr), op_ + ": grad came or went since the OpEnv was made");
    if (inputs[2]) RAF_CHECK(Same(inputs[2], out_, "grad").data == out.data, op_ + ": the output of a call with grad is grad");
    Check("rafhip_embedding_dx",
          rafhip_embedding_dx(dy.data, dy_dtype_, ids.data, ids.dtype.bits, ids.numel(), out.shape[0], out.shape[1],
                              args_.first_row, args_.has_padding ? 1 : 0, args_.padding_index, (float)args_.scale, out.data,
                              out_dtype_, args_.grad ? 1 : 0, workspace_, workspace_bytes_, Stream()));
  }

  static OpEnv* make(const CallValues& cv) { return new EmbeddingDxHipEnv(cv); }

 private:
  schema::EmbeddingDxArgs args_;
  TensorView dy_, ids_, out_;
  int32_t dy_dtype_ = -1, out_dtype_ = -1;
};

class TopkDistillHipEnv : public VocabHipEnv {
 public:
  enum Kind { kLoss, kGradient, kBoth };

  TopkDistillHipEnv(const CallValues& cv, const char* op, Kind kind) : VocabHipEnv(op), kind_(kind) {
    const auto* args = cv->args_as<schema::TopkDistillArgs>();
    if (!args) {
      error_msgs.push_back(op_ + ": call does not carry TopkDistillArgs");
      return;
    }
    for (const char* field : {"logits", "topk_indices", "topk_logits", "labels", "dloss", "stats"})
      arg_indices.push_back(args->FieldIndex(field));
    for (const auto& t : {args->logits, args->topk_indices, args->topk_logits, args->labels, args->dloss, args->stats})
      ins_.push_back(t ? t->tensor : TensorView());
    has_labels_ = args->labels != nullptr;
    if (kind == kGradient) {
      outs_ = {AsTensor(cv->out)->tensor};
    } else {
      for (const Value& field : AsTuple(cv->out)->fields) outs_.push_back(AsTensor(field)->tensor);
    }
    const TensorView& z = args->logits->tensor;
    const TensorView& index = args->topk_indices->tensor;
    width_ = z.shape.back();
    call_.rows = 1;
    for (int i = 0; i + 1 < z.ndim(); ++i) call_.rows *= z.shape[i];
    call_.vocab = args->vocab_size;
    call_.row_stride = width_;
    call_.logits_dtype = KernelDType(z.dtype);
    call_.topk_dtype = KernelDType(args->topk_logits->tensor.dtype);
    call_.index_bits = index.dtype.bits;
    call_.temperature = (float)args->temperature;
    call_.soft_weight = (float)args->soft_weight;
    call_.hard_weight = (float)args->hard_weight;
    RequireDType(call_.logits_dtype, "logits");
    RequireDType(call_.topk_dtype, "topk_logits");
    RequireDevice(cv);
    if (!error_msgs.empty()) return;
    if (index.shape.back() > RAFHIP_MAX_TOPK) {
      error_msgs.push_back(op_ + ": more than " + std::to_string(RAFHIP_MAX_TOPK) + " teacher entries in a row");
      return;
    }
    call_.topk = (int32_t)index.shape.back();
    // Also checks the numbers, for the gradient too, which needs no workspace.
    const int64_t bytes = rafhip_topk_distill_workspace_bytes(&call_);
    RequireWorkspace(cv, kind == kGradient && bytes > 0 ? 0 : bytes);
  }

  void Execute(const CallValues& cv) override {
    const auto* args = cv->args_as<schema::TopkDistillArgs>();
    RAF_CHECK(args != nullptr, op_ + " expects TopkDistillArgs");
    Execute(std::vector<Value>{args->logits, args->topk_indices, args->topk_logits, args->labels, args->dloss, args->stats},
            cv->out);
  }

  void Execute(const std::vector<Value>& inputs, Value output) override {
    RAF_CHECK(inputs.size() == 6, op_ + " takes logits, topk_indices, topk_logits, labels, dloss and stats");
    rafhip_topk_distill_args call = call_;
    call.logits = Same(inputs[0], ins_[0], "logits").data;
    call.topk_indices = Same(inputs[1], ins_[1], "topk_indices").data;
    call.topk_logits = Same(inputs[2], ins_[2], "topk_logits").data;
    RAF_CHECK((inputs[3] != nullptr) == has_labels_, op_ + ": labels came or went since the OpEnv was made");
    call.labels = inputs[3] ? Same(inputs[3], ins_[3], "labels").data : nullptr;
    const float* dloss = nullptr;
    int64_t dloss_count = 0;
    if (kind_ != kLoss) {
      const TensorView& d = Same(inputs[4], ins_[4], "dloss");
      dloss = static_cast<const float*>(d.data);
      dloss_count = d.numel();
    }
    if (kind_ == kGradient) {
      const TensorView& stats = Same(inputs[5], ins_[5], "stats");
      Check("rafhip_topk_distill_dx",
            rafhip_topk_distill_dx(&call, dloss, dloss_count, static_cast<const float*>(stats.data),
                                   Same(output, outs_[0], "dlogits").data, width_, Stream()));
      return;
    }
    const auto outs = AsTuple(output);
    RAF_CHECK(outs->fields.size() == 2, op_ + " has two outputs");
    float* loss = static_cast<float*>(Same(outs->fields[0], outs_[0], "loss").data);
    if (kind_ == kLoss) {
      float* stats = static_cast<float*>(Same(outs->fields[1], outs_[1], "stats").data);
      Check("rafhip_topk_distill", rafhip_topk_distill(&call, loss, stats, workspace_, workspace_bytes_, Stream()));
      return;
    }
    Check("rafhip_topk_distill_step",
          rafhip_topk_distill_step(&call, dloss, dloss_count, loss, Same(outs->fields[1], outs_[1], "dlogits").data, width_,
                                   workspace_, workspace_bytes_, Stream()));
  }

  static OpEnv* make(const CallValues& cv) { return new TopkDistillHipEnv(cv, "raf.op.hip.topk_distill", kLoss); }
  static OpEnv* make_dx(const CallValues& cv) { return new TopkDistillHipEnv(cv, "raf.op.hip.topk_distill_dx", kGradient); }
  static OpEnv* make_step(const CallValues& cv) { return new TopkDistillHipEnv(cv, "raf.op.hip.topk_distill_step", kBoth); }

 private:
  Kind kind_;
  std::vector<TensorView> ins_, outs_;  // in the schema's order
  bool has_labels_ = false;
  rafhip_topk_distill_args call_ = {};
  int64_t width_ = 0;
};

// The reference's embedding backends are cuda's, plevel 10.
RAF_REGISTER_DIALECT_OP(hip, embedding, 30);
RAF_OP_ENV_MAKER("raf.op.hip.embedding", EmbeddingHipEnv::make);
RAF_REGISTER_DIALECT_OP(hip, embedding_dx, 30);
RAF_OP_ENV_MAKER("raf.op.hip.embedding_dx", EmbeddingDxHipEnv::make);
RAF_REGISTER_DIALECT_OP(hip, topk_distill, 30);
RAF_OP_ENV_MAKER("raf.op.hip.topk_distill", TopkDistillHipEnv::make);
RAF_REGISTER_DIALECT_OP(hip, topk_distill_dx, 30);
RAF_OP_ENV_MAKER("raf.op.hip.topk_distill_dx", TopkDistillHipEnv::make_dx);
RAF_REGISTER_DIALECT_OP(hip, topk_distill_step, 30);
RAF_OP_ENV_MAKER("raf.op.hip.topk_distill_step", TopkDistillHipEnv::make_step);

}  // namespace hip
}  // namespace op
}  // namespace raf
