// torch operators of the dense block, over the C-ABI of libcuda_mace_b200.so:
//
//   cmace_b200::gated_feed_forward(x, w_gate, w_up, w_down, activation, status)
//
// This file owns what the C-ABI leaves to its caller: checks of the arguments, outputs and workspaces through the caching allocator, the
// current stream, and the autograd node.  The node is here and not in Python because a training step of a small block is as long as
// its host side: forward and backward of 105 rows of 32 took 137 us with a node in Python, 97 us with this one.
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/script.h>

#include "../../include/cuda_mace_b200.h"

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

void check(int rc, const char *what) { TORCH_CHECK(rc == 0, what, " failed (", rc, "): ", cmace_last_error()); }

cmace_stream_t current_stream() { return (cmace_stream_t)c10::cuda::getCurrentCUDAStream().stream(); }

Tensor workspace(const Tensor &like, bool f32, int64_t rows, int64_t width, int64_t hidden, bool backward) {
  const int64_t bytes = cmace_gated_ff_workspace_bytes(f32, rows, (int)width, (int)hidden, backward);
  TORCH_CHECK(bytes >= 0, cmace_last_error());
  return at::empty({bytes}, like.options().dtype(torch::kUInt8));
}

Tensor forward_rows(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation, const Tensor &status) {
  const bool f32 = x.scalar_type() == torch::kFloat32;
  const int64_t width = wg.size(0), hidden = wg.size(1), rows = x.numel() / width;
  Tensor y = at::empty_like(x);
  const Tensor ws = workspace(x, f32, rows, width, hidden, false);
  if (f32)
    check(cmace_gated_ff_fwd_f32(x.data_ptr<float>(), wg.data_ptr<float>(), wu.data_ptr<float>(), wd.data_ptr<float>(), rows, (int)width, (int)hidden,
                                 (int)activation, y.data_ptr<float>(), ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), current_stream()),
          "gated_feed_forward");
  else
    check(cmace_gated_ff_fwd_bf16(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), rows, (int)width, (int)hidden, (int)activation, y.data_ptr(),
                                  ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), current_stream()),
          "gated_feed_forward");
  return y;
}

class GatedFeedForward : public torch::autograd::Function<GatedFeedForward> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation,
                        const Tensor &status) {
    ctx->save_for_backward({x, wg, wu, wd});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["status"] = status;
    return forward_rows(x, wg, wu, wd, activation, status);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &wg = saved[1];
    const bool f32 = x.scalar_type() == torch::kFloat32;
    const int64_t width = wg.size(0), hidden = wg.size(1), rows = x.numel() / width, activation = ctx->saved_data["activation"].toInt();
    const Tensor status = ctx->saved_data["status"].toTensor();
    variable_list out(6);
    if (!grad[0].defined()) return out;
    {
      const at::AutoGradMode off(false);
      const Tensor gy = grad[0].contiguous();
      void *to[4];
      for (int i = 0; i < 4; i++) {
        if (ctx->needs_input_grad(i)) out[i] = at::empty_like(saved[i]);
        to[i] = out[i].defined() ? out[i].data_ptr() : nullptr;
      }
      const Tensor ws = workspace(x, f32, rows, width, hidden, true);
      const auto run = f32 ? (int (*)(const void *, const void *, const void *, const void *, const void *, int64_t, int, int, int, void *, void *, void *, void *,
                                      void *, int64_t, int32_t *, cmace_stream_t))cmace_gated_ff_bwd_f32
                           : cmace_gated_ff_bwd_bf16;
      check(run(x.data_ptr(), wg.data_ptr(), saved[2].data_ptr(), saved[3].data_ptr(), gy.data_ptr(), rows, (int)width, (int)hidden, (int)activation, to[0],
                to[1], to[2], to[3], ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), current_stream()),
            "gated_feed_forward backward");
    }
    if (at::GradMode::is_enabled()) {   // create_graph: differentiating these once more is an error, not a zero
      variable_list found, marked;
      for (const Tensor &t : out)
        if (t.defined()) found.push_back(t);
      auto error = std::make_shared<torch::autograd::DelayedError>("gated_feed_forward is differentiable once", (int64_t)found.size());
      for (Tensor &t : found) t.requires_grad_(true);
      marked = (*error)(std::move(found));
      int at = 0;
      for (Tensor &t : out)
        if (t.defined()) t = marked[at++];
    }
    return out;
  }
};

Tensor gated_feed_forward(const Tensor &x_, const Tensor &wg_, const Tensor &wu_, const Tensor &wd_, int64_t activation, const Tensor &status) {
  const int device = c10::cuda::current_device();
  for (const Tensor *t : {&x_, &wg_, &wu_, &wd_}) {
    TORCH_CHECK(t->is_cuda(), "cuda_mace_b200 operators need CUDA tensors (there is no CPU path)");
    TORCH_CHECK(t->get_device() == device, "operand on cuda:", t->get_device(), " while cuda:", device, " is the current device");
    TORCH_CHECK_TYPE(t->scalar_type() == x_.scalar_type() && (x_.scalar_type() == torch::kFloat32 || x_.scalar_type() == torch::kBFloat16),
                     "gated_feed_forward needs float32 or bfloat16 operands of one type");
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "gated_feed_forward has no forward-mode derivative");
  }
  TORCH_CHECK(x_.dim() >= 1 && wg_.dim() == 2 && wu_.dim() == 2 && wd_.dim() == 2, "gated_feed_forward needs rows and weight matrices");
  const int64_t width = wg_.size(0), hidden = wg_.size(1);
  TORCH_CHECK(width >= 1 && hidden >= 1 && x_.size(-1) == width && wu_.size(0) == width && wu_.size(1) == hidden && wd_.size(0) == hidden && wd_.size(1) == width,
              "shape mismatch: x ", x_.sizes(), ", w_gate ", wg_.sizes(), ", w_up ", wu_.sizes(), ", w_down ", wd_.sizes());
  TORCH_CHECK(width <= 1 << 20 && hidden <= 1 << 20, "gated_feed_forward: widths up to 2^20");
  TORCH_CHECK(status.is_cuda() && status.get_device() == device && status.scalar_type() == torch::kInt32 && status.numel() >= 1,
              "gated_feed_forward: status has to be an int32 of the current device");
  const Tensor x = x_.contiguous(), wg = wg_.contiguous(), wu = wu_.contiguous(), wd = wd_.contiguous();
  if (at::GradMode::is_enabled() && (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
    return GatedFeedForward::apply(x, wg, wu, wd, activation, status);
  return forward_rows(x, wg, wu, wd, activation, status);
}

}  // namespace

TORCH_LIBRARY(cmace_b200, m) {
  m.def("gated_feed_forward(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int activation, Tensor status) -> Tensor", &gated_feed_forward);
}
