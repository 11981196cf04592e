// functs::rotary: rotary positions (fx_rotary of include/fxhip.h), with their gradient.
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include <cmath>
#include <unordered_set>
#include <vector>

#include "rotary_ops.h"

namespace functs {
fx_rotary_desc rotaryDesc(const char* op, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved, int64_t depth, c10::Device dev) {
  onGpu(op, positions, "positions", dev);
  onGpu(op, frequencies, "frequencies", dev);
  noGrad(op, frequencies, "frequencies");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong, op, ": positions must be int32 or int64, got ", positions.scalar_type());
  TORCH_CHECK((frequencies.scalar_type() == at::kDouble || frequencies.scalar_type() == at::kFloat) && frequencies.dim() == 1, op,
              ": frequencies must be float64 or float32 [pairs], got ", frequencies.scalar_type(), " ", frequencies.sizes());
  const int64_t pairs = frequencies.numel();
  TORCH_CHECK(pairs >= 1 && 2 * pairs <= depth, op, ": ", depth, " columns hold 1 to ", depth / 2, " pairs, got frequencies of ", pairs);
  TORCH_CHECK(std::isfinite((float)magnitude), op, ": magnitude must be finite, got ", magnitude);
  fx_rotary_desc d;
  memset(&d, 0, sizeof d);
  d.positions = positions.data_ptr();
  d.frequencies = frequencies.data_ptr();
  d.depth = sized(op, depth, "the depth");
  d.pairs = (int32_t)pairs;
  d.positions_64 = positions.scalar_type() == at::kLong;
  d.frequencies_32 = frequencies.scalar_type() == at::kFloat;
  d.interleaved = interleaved;
  d.magnitude = (float)magnitude;
  return d;
}

namespace {
constexpr char kOp[] = "functs::rotary";

// x [tokens, heads, depth] or [batch, tokens, heads, depth]
Tensor turned(const Tensor& x_, const Tensor& positions_, const Tensor& frequencies_, double magnitude, bool interleaved, bool back) {
  TORCH_CHECK(x_.is_cuda(), kOp, " runs on the GPU only; x is a ", x_.device(), " tensor");
  TORCH_CHECK((x_.dim() == 3 || x_.dim() == 4) && x_.size(-2) >= 1, kOp, ": x must be [tokens, heads, depth] or [batch, tokens, heads, depth], got ", x_.sizes());
  const int dtype = dtypeOf(kOp, x_.scalar_type(), "x");
  const bool batched = x_.dim() == 4;
  const int64_t B = batched ? x_.size(0) : 1, T = x_.size(-3);
  TORCH_CHECK((positions_.dim() == 1 && positions_.size(0) == T) || (batched && positions_.dim() == 2 && positions_.size(0) == B && positions_.size(1) == T), kOp,
              ": positions must be [", T, "]", batched ? " or [" : "", batched ? std::to_string(B) + ", " + std::to_string(T) + "]" : "", ", got ", positions_.sizes());
  const auto dev = x_.device();
  c10::DeviceGuard guard(dev);
  // (what the checks of rotaryDesc refuse is refused before anything is copied: contiguous() keeps device, type and sizes)
  const Tensor positions = positions_.dim() == 2 && positions_.stride(1) == 1 ? positions_ : positions_.contiguous(), frequencies = frequencies_.resolve_neg().contiguous();
  fx_rotary_desc d = rotaryDesc(kOp, positions, frequencies, magnitude, interleaved, x_.size(-1), dev);
  Tensor x = x_.resolve_neg();
  if (x.stride(-1) != 1) x = x.contiguous();
  // (an x whose numbers fill its memory keeps its order of dimensions)
  Tensor y = x.is_non_overlapping_and_dense() ? at::empty_strided(x.sizes(), x.strides(), x.options()) : at::empty(x.sizes(), x.options());
  d.x = x.data_ptr();
  d.y = y.data_ptr();
  d.x_batch_stride = batched ? x.stride(0) : 0;
  d.x_token_stride = x.stride(-3);
  d.x_head_stride = x.stride(-2);
  d.y_batch_stride = batched ? y.stride(0) : 0;
  d.y_token_stride = y.stride(-3);
  d.y_head_stride = y.stride(-2);
  d.position_batch_stride = positions.dim() == 2 ? positions.stride(0) : 0;
  d.batch = sized(kOp, B, "the batch");
  d.tokens = sized(kOp, T, "the number of tokens");
  d.heads = sized(kOp, x.size(-2), "the number of heads");
  d.dtype = dtype;
  d.back = back;
  FX_OK_OR_THROW(fx_rotary(&d, streamOf(dev)));
  return y;
}

Tensor rotaryOf(const Tensor& x, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved, bool back);

// A leaf's gradient is added up on the stream on which its first graph was made.  While that graph lives, a backward pass captured on another
// stream would wait for this one in the middle of the capture; the default stream cannot be waited for there, and the engine ends the process.
bool capturing(c10::Device dev) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream() != nullptr && c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None;
}
// Of a captured backward pass that is at this operator: whether anything that it runs behind, the gradients of leaves among it, is the default stream's
bool defaultStreamBehind(c10::Device dev) {
  const c10::Stream none = c10::hip::getDefaultHIPStreamMasqueradingAsCUDA(dev.index()).unwrap();
  const auto* const runs = torch::autograd::get_current_graph_task_exec_info();   // (empty: all nodes run)
  const auto here = torch::autograd::get_current_node();
  std::vector<torch::autograd::Node*> ahead{here.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!ahead.empty()) {
    auto* const node = ahead.back();
    ahead.pop_back();
    if (!node) continue;
    for (const auto& edge : node->next_edges()) {
      auto* const next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (runs && !runs->empty()) {
        const auto it = runs->find(next);
        if (it == runs->end() || !it->second.should_execute()) continue;
      }
      const auto made = next->stream();
      if (made && *made == none) return true;
      ahead.push_back(next);
    }
  }
  return false;
}

// The gradient of a rotation is the rotation back, which has a gradient of its own
struct Rotary : public torch::autograd::Function<Rotary> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved,
                        bool back) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({positions, frequencies});
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["back"] = back;
    return turned(x, positions, frequencies, magnitude, interleaved, back);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    Tensor x;
    if (grads[0].defined()) {
      if (grads[0].is_cuda()) {
        c10::DeviceGuard guard(grads[0].device());
        TORCH_CHECK(!capturing(grads[0].device()) || !defaultStreamBehind(grads[0].device()), kOp,
                    ": this captured backward pass comes to a tensor that is in a living graph of the default stream; drop its results before the capture");
      }
      const auto saved = ctx->get_saved_variables();
      x = rotaryOf(grads[0], saved[0], saved[1], ctx->saved_data["magnitude"].toDouble(), ctx->saved_data["interleaved"].toBool(), !ctx->saved_data["back"].toBool());
    }
    return {x, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor rotaryOf(const Tensor& x, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved, bool back) {
  TORCH_CHECK(!x._fw_grad(0).defined(), kOp, " has no forward-mode derivative: x carries a tangent");
  if (!at::GradMode::is_enabled() || !x.requires_grad()) return turned(x, positions, frequencies, magnitude, interleaved, back);
  // (the same for a leaf that is turned itself, as soon as the call is captured and on whichever stream its graph was made)
  if (x.is_cuda() && x.is_leaf()) {
    c10::DeviceGuard guard(x.device());
    if (capturing(x.device())) {
      const auto node = torch::autograd::impl::try_get_grad_accumulator(x);
      const auto made = node ? node->stream() : std::nullopt;
      const c10::Stream now = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).unwrap();
      TORCH_CHECK(!made || *made == now, kOp, ": x is in a graph of another stream that is alive; drop its results before this capture");
    }
  }
  return Rotary::apply(x, positions, frequencies, magnitude, interleaved, back);
}

Tensor rotary(const Tensor& x, const Tensor& positions, const Tensor& frequencies, double magnitude, bool interleaved) {
  return rotaryOf(x, positions, frequencies, magnitude, interleaved, false);
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(functs, m) {
  m.def("rotary(Tensor x, Tensor positions, Tensor frequencies, float magnitude=1.0, bool interleaved=False) -> Tensor", rotary);
}
}  // namespace functs
