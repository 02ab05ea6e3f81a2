// torch operators of the dense block, over the C-ABI of libcuda_mace_b200.so:
//
//   cmace_b200::gated_feed_forward(x, w_gate, w_up, w_down, activation, status)
//   cmace_b200::gated_feed_forward_backward(grad, x, w_gate, w_up, w_down, activation, wanted, status)
//
// This file owns what the C-ABI leaves to its caller: checks of the arguments, outputs and workspaces through the caching allocator, the
// current stream, and the autograd node.  The node is here and not in Python because a training step of a small block is as long as
// its host side: forward and backward of 105 rows of 32 took 137 us with a node in Python, 97 us with this one.
// Kernels are registered by dispatch key (CUDA, Autograd, Meta), and one calls the next through the dispatcher, so that a tracer records the operator
// itself: recorded through its insides it would be an output that nobody writes.
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

// what needs no values: types, dimensions
void check_operands(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd) {
  for (const Tensor *t : {&x, &wg, &wu, &wd})
    TORCH_CHECK_TYPE(t->scalar_type() == x.scalar_type() && (x.scalar_type() == torch::kFloat32 || x.scalar_type() == torch::kBFloat16),
                     "gated_feed_forward needs float32 or bfloat16 operands of one type");
  TORCH_CHECK(x.dim() >= 1 && wg.dim() == 2 && wu.dim() == 2 && wd.dim() == 2, "gated_feed_forward needs rows and weight matrices");
  const auto width = wg.sym_size(0), hidden = wg.sym_size(1);
  TORCH_CHECK(width >= 1 && hidden >= 1 && x.sym_size(-1) == width && wu.sym_size(0) == width && wu.sym_size(1) == hidden && wd.sym_size(0) == hidden &&
                  wd.sym_size(1) == width,
              "shape mismatch: x ", x.sym_sizes(), ", w_gate ", wg.sym_sizes(), ", w_up ", wu.sym_sizes(), ", w_down ", wd.sym_sizes());
  TORCH_CHECK(width <= 1 << 20 && hidden <= 1 << 20, "gated_feed_forward: widths up to 2^20");
}
void check_device(std::initializer_list<const Tensor *> all, const Tensor &status) {
  const int device = c10::cuda::current_device();
  for (const Tensor *t : all) {
    TORCH_CHECK(t->is_cuda(), "cuda_mace_b200 operators need CUDA tensors (there is no CPU path)");
    TORCH_CHECK(t->get_device() == device, "operand on cuda:", t->get_device(), " while cuda:", device, " is the current device");
  }
  TORCH_CHECK(status.is_cuda() && status.get_device() == device && status.scalar_type() == torch::kInt32 && status.numel() >= 1,
              "gated_feed_forward: status has to be an int32 of the current device");
}

Tensor forward_cuda(const Tensor &x_, const Tensor &wg_, const Tensor &wu_, const Tensor &wd_, int64_t activation, const Tensor &status) {
  check_device({&x_, &wg_, &wu_, &wd_}, status);
  check_operands(x_, wg_, wu_, wd_);
  const Tensor x = x_.contiguous(), wg = wg_.contiguous(), wu = wu_.contiguous(), wd = wd_.contiguous();
  const bool f32 = x.scalar_type() == torch::kFloat32;
  const int64_t width = wg.size(0), hidden = wg.size(1), rows = x.numel() / width;
  Tensor y = at::empty_like(x);
  const Tensor ws = workspace(x, f32, rows, width, hidden, false);
  const auto run = f32 ? (int (*)(const void *, const void *, const void *, const void *, int64_t, int, int, int, void *, void *, int64_t, int32_t *,
                                  cmace_stream_t))cmace_gated_ff_fwd_f32
                       : cmace_gated_ff_fwd_bf16;
  check(run(x.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), rows, (int)width, (int)hidden, (int)activation, y.data_ptr(), ws.data_ptr(),
            ws.numel(), status.data_ptr<int32_t>(), current_stream()),
        "gated_feed_forward");
  return y;
}

using Gradients = std::tuple<Tensor, Tensor, Tensor, Tensor>;   // undefined: not wanted

Gradients backward_cuda(const Tensor &gy_, const Tensor &x_, const Tensor &wg_, const Tensor &wu_, const Tensor &wd_, int64_t activation,
                        std::array<bool, 4> wanted, const Tensor &status) {
  check_device({&gy_, &x_, &wg_, &wu_, &wd_}, status);
  check_operands(x_, wg_, wu_, wd_);
  TORCH_CHECK(gy_.sizes() == x_.sizes() && gy_.scalar_type() == x_.scalar_type(), "gated_feed_forward: a gradient ", gy_.sizes(), " of type ",
              gy_.scalar_type(), " for rows ", x_.sizes());
  const Tensor gy = gy_.contiguous(), saved[4] = {x_.contiguous(), wg_.contiguous(), wu_.contiguous(), wd_.contiguous()};
  const bool f32 = gy.scalar_type() == torch::kFloat32;
  const int64_t width = wg_.size(0), hidden = wg_.size(1), rows = gy.numel() / width;
  Tensor out[4];
  void *to[4] = {};
  for (int i = 0; i < 4; i++)
    if (wanted[i]) {
      out[i] = at::empty_like(saved[i]);
      to[i] = out[i].data_ptr();
    }
  const Tensor ws = workspace(gy, f32, rows, width, hidden, true);
  const auto run = f32 ? (int (*)(const void *, const void *, const void *, const void *, const void *, int64_t, int, int, int, void *, void *, void *, void *,
                                  void *, int64_t, int32_t *, cmace_stream_t))cmace_gated_ff_bwd_f32
                       : cmace_gated_ff_bwd_bf16;
  check(run(saved[0].data_ptr(), saved[1].data_ptr(), saved[2].data_ptr(), saved[3].data_ptr(), gy.data_ptr(), rows, (int)width, (int)hidden,
            (int)activation, to[0], to[1], to[2], to[3], ws.data_ptr(), ws.numel(), status.data_ptr<int32_t>(), current_stream()),
        "gated_feed_forward backward");
  return {out[0], out[1], out[2], out[3]};
}

// Shapes alone, for tracers
Tensor like(const Tensor &t) { return at::empty_symint(t.sym_sizes(), t.options()); }
Tensor forward_meta(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t, const Tensor &) {
  check_operands(x, wg, wu, wd);
  return like(x);
}
Gradients backward_meta(const Tensor &, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t, std::array<bool, 4> wanted,
                        const Tensor &) {
  return {wanted[0] ? like(x) : Tensor(), wanted[1] ? like(wg) : Tensor(), wanted[2] ? like(wu) : Tensor(), wanted[3] ? like(wd) : Tensor()};
}

Tensor call_forward(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation, const Tensor &status) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("cmace_b200::gated_feed_forward", "").typed<decltype(forward_cuda)>();
  const at::AutoDispatchBelowADInplaceOrView below;
  return op.call(x, wg, wu, wd, activation, status);
}

class GatedFeedForward : public torch::autograd::Function<GatedFeedForward> {
 public:
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation,
                        const Tensor &status) {
    ctx->save_for_backward({x, wg, wu, wd});
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["status"] = status;
    return call_forward(x, wg, wu, wd, activation, status);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grad) {
    static const auto op =
        c10::Dispatcher::singleton().findSchemaOrThrow("cmace_b200::gated_feed_forward_backward", "").typed<decltype(backward_cuda)>();
    const variable_list saved = ctx->get_saved_variables();
    variable_list out(6);
    if (!grad[0].defined()) return out;
    std::array<bool, 4> wanted;
    for (int i = 0; i < 4; i++) wanted[i] = ctx->needs_input_grad(i);
    {
      const at::AutoGradMode off(false);
      const at::AutoDispatchBelowADInplaceOrView below;
      std::tie(out[0], out[1], out[2], out[3]) =
          op.call(grad[0], saved[0], saved[1], saved[2], saved[3], ctx->saved_data["activation"].toInt(), wanted, ctx->saved_data["status"].toTensor());
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

Tensor forward_autograd(const Tensor &x, const Tensor &wg, const Tensor &wu, const Tensor &wd, int64_t activation, const Tensor &status) {
  bool wanted = false;
  for (const Tensor *t : {&x, &wg, &wu, &wd}) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t->_fw_grad(0).defined(), "gated_feed_forward has no forward-mode derivative");
    wanted = wanted || t->requires_grad();
  }
  if (!wanted || !at::GradMode::is_enabled()) return call_forward(x, wg, wu, wd, activation, status);
  return GatedFeedForward::apply(x.contiguous(), wg.contiguous(), wu.contiguous(), wd.contiguous(), activation, status);
}

}  // namespace

TORCH_LIBRARY(cmace_b200, m) {
  m.def("gated_feed_forward(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int activation, Tensor status) -> Tensor");
  m.def("gated_feed_forward_backward(Tensor grad, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int activation, bool[4] wanted, Tensor status) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(cmace_b200, CUDA, m) {
  m.impl("gated_feed_forward", &forward_cuda);
  m.impl("gated_feed_forward_backward", &backward_cuda);
}
TORCH_LIBRARY_IMPL(cmace_b200, Autograd, m) { m.impl("gated_feed_forward", &forward_autograd); }
TORCH_LIBRARY_IMPL(cmace_b200, Meta, m) {
  m.impl("gated_feed_forward", &forward_meta);
  m.impl("gated_feed_forward_backward", &backward_meta);
}
