// functs::beam_select: the best continuations of a beam search (fx_beam_select of include/fxhip.h).
#include <torch/library.h>

#include <tuple>

#include "op_checks.h"

namespace functs {
namespace {
std::tuple<Tensor, Tensor, Tensor> beamSelect(const Tensor& logits_, const Tensor& scores_, int64_t count, const std::optional<Tensor>& ended_, int64_t end_word) {
  static const char op[] = "functs::beam_select";
  TORCH_CHECK(logits_.is_cuda(), op, " runs on the GPU only; logits is a ", logits_.device(), " tensor");
  const auto dev = logits_.device();
  TORCH_CHECK(logits_.dim() == 3, op, ": logits must be [requests, beams, words], got ", logits_.sizes());
  const int dtype = dtypeOf(op, logits_.scalar_type(), "logits");
  const int64_t B = logits_.size(0), K = logits_.size(1), V = logits_.size(2);
  onGpu(op, scores_, "scores", dev);
  TORCH_CHECK(scores_.scalar_type() == at::kFloat && scores_.dim() == 2 && scores_.size(0) == B && scores_.size(1) == K, op, ": scores must be float32 [", B, ", ", K, "], got ",
              scores_.scalar_type(), " ", scores_.sizes());
  noGrad(op, logits_, "logits");
  noGrad(op, scores_, "scores");
  TORCH_CHECK(count >= 0, op, ": count must not be negative, got ", count);
  if (count == 0) count = K;
  c10::DeviceGuard guard(dev);
  Tensor ended;
  if (ended_ && ended_->defined()) {
    onGpu(op, *ended_, "ended", dev);
    TORCH_CHECK((ended_->scalar_type() == at::kBool || ended_->scalar_type() == at::kByte) && ended_->dim() == 2 && ended_->size(0) == B && ended_->size(1) == K, op,
                ": ended must be bool or uint8 [", B, ", ", K, "], got ", ended_->scalar_type(), " ", ended_->sizes());
    ended = ended_->contiguous();
  }
  Tensor logits = logits_.resolve_neg();
  if (logits.stride(2) != 1 && V > 1) logits = logits.contiguous();
  const Tensor scores = scores_.resolve_neg().contiguous();
  fx_beam_select_desc d;
  memset(&d, 0, sizeof d);
  d.requests = sized(op, B, "the number of requests");
  d.beams = sized(op, K, "the number of beams");
  d.words = sized(op, V, "the number of words");
  d.count = sized(op, count, "count");
  d.dtype = dtype;
  // (scratch memory of this call alone, from the allocator of the current stream: calls on other streams and captured graphs have their own)
  const size_t bytes = fx_beam_select_workspace_bytes(&d);
  TORCH_CHECK(bytes > 0, "fxhip: ", fx_last_error(), " (", op, ")");
  const auto on = at::TensorOptions().device(dev);
  const Tensor ws = at::empty({(int64_t)bytes}, on.dtype(at::kByte));
  Tensor out_scores = at::empty({B, count}, on.dtype(at::kFloat)), beams = at::empty({B, count}, on.dtype(at::kInt)), words = at::empty({B, count}, on.dtype(at::kLong));
  d.logits = logits.data_ptr();
  d.request_stride = logits.stride(0);
  d.beam_stride = logits.stride(1);
  d.scores = scores.data_ptr<float>();
  d.ended = ended.defined() ? (const uint8_t*)ended.data_ptr() : nullptr;
  d.end_word = end_word;
  d.out_scores = out_scores.data_ptr<float>();
  d.out_beams = beams.data_ptr<int32_t>();
  d.out_words = words.data_ptr<int64_t>();
  d.workspace = ws.data_ptr();
  d.workspace_bytes = bytes;
  FX_OK_OR_THROW(fx_beam_select(&d, streamOf(dev)));
  return {out_scores, beams, words};
}
}  // namespace

TORCH_LIBRARY_FRAGMENT(functs, m) {
  m.def("beam_select(Tensor logits, Tensor scores, int count=0, Tensor? ended=None, int end_word=-1) -> (Tensor, Tensor, Tensor)", beamSelect);
}
}  // namespace functs
