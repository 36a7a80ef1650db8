// Operators of the experts of one GPU: tokens sorted by expert and back, with gradients, rows
// quantised to 8-bit integers, and their grouped GEMM.  No counterpart in the reference.
#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "../core/utils.h"
#include "../kernels/expert_rows.h"
#include "../kernels/grouped_gemm.h"
#include "registration.h"

namespace pplx {
namespace {

constexpr int64_t kMaxRows = int64_t{1} << 30;

// Launches on the device and the current stream of `on`.
template <typename F>
void launch_on(const at::Tensor& on, F&& launch) {
  if (on.is_meta()) return;
  const c10::cuda::OptionalCUDAGuard guard(on.device());
  try {
    launch(at::cuda::getCurrentCUDAStream());
  } catch (const Error& e) {
    TORCH_CHECK(false, e.what());
  }
}

// The operators check Meta tensors as they check others and then return, so that torch.compile, and
// tests without a GPU, meet the same refusals.
void check_device(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda() || t.is_meta(), op, ": ", name, " must be a CUDA tensor");
}

void check_device(const at::Tensor& t, const at::Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " must be on ", like.device(), ", not on ",
              t.device());
}

// (For CUDA tensors the allocation itself, without another pass through the dispatcher.)
at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
  if (like.is_cuda()) return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
  return at::empty(sizes, like.options().dtype(type));
}

template <typename T>
T* data(const at::Tensor& t) {
  return t.is_meta() ? nullptr : static_cast<T*>(t.data_ptr());
}

FloatType float_type(const at::Tensor& t, const char* op, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return FloatType::kBFloat16;
    case at::kHalf: return FloatType::kHalf;
    case at::kFloat: return FloatType::kFloat;
    default: TORCH_CHECK(false, op, ": ", name, " must be bfloat16, float16 or float32");
  }
}

// Tokens and rows are read in an order of their own: a result in the memory of the input would be read
// back as input.
void check_apart(const at::Tensor& written, const at::Tensor& read, const char* op, const char* name,
                 const char* from) {
  const at::MemOverlapStatus s = at::get_overlap_status(written, read);
  TORCH_CHECK(s != at::MemOverlapStatus::Full && s != at::MemOverlapStatus::Partial, op, ": ", name,
              " must not share memory with ", from);
}

// [tokens, hidden] with contiguous columns; the distance of two rows in elements.
int64_t token_stride(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.dim() == 2, op, ": ", name, " must be [tokens, hidden]");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, op, ": the columns of ", name,
              " must be contiguous");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), op, ": the rows of ", name,
              " must not overlap");
  return t.size(0) <= 1 ? t.size(1) : t.stride(0);
}

void check_hidden(int64_t hidden, const char* op) {
  TORCH_CHECK(hidden < (int64_t{1} << 30), op, ": rows of 2^30 elements or more");
}

// Rows as the capacity says: [rows, hidden] or [experts, capacity, hidden], contiguous.
void check_rows(const at::Tensor& t, const ExpertRowsView& v, int64_t hidden, const at::Tensor& like,
                const char* op, const char* name) {
  check_device(t, like, op, name);
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " must be contiguous");
  if (v.capacity > 0) {
    TORCH_CHECK(t.dim() == 3 && t.size(0) == v.num_experts && t.size(1) == v.capacity &&
                    t.size(2) == hidden,
                op, ": ", name, " must be [", v.num_experts, ", ", v.capacity, ", ", hidden, "]");
  } else {
    TORCH_CHECK(t.dim() == 2 && t.size(0) == v.num_rows && t.size(1) == hidden, op, ": ", name,
                " must be [", v.num_rows, ", ", hidden, "]");
  }
}

ExpertRowsView make_view(const at::Tensor& counts, const at::Tensor& offsets,
                         const at::Tensor& row_of, int64_t capacity, const at::Tensor& like,
                         const char* op) {
  check_device(counts, like, op, "counts");
  check_device(offsets, like, op, "offsets");
  check_device(row_of, like, op, "row_of");
  TORCH_CHECK(counts.scalar_type() == at::kInt && offsets.scalar_type() == at::kInt &&
                  row_of.scalar_type() == at::kInt,
              op, ": counts, offsets and row_of must be int32");
  TORCH_CHECK(counts.dim() == 1 && counts.size(0) > 0 && counts.is_contiguous() &&
                  offsets.dim() == 1 && offsets.size(0) == counts.size(0) + 1 &&
                  offsets.is_contiguous() && row_of.dim() == 2 && row_of.size(1) > 0 &&
                  row_of.is_contiguous(),
              op, ": counts, offsets and row_of must be contiguous, [experts], [experts + 1] and "
              "[tokens, topk]");
  TORCH_CHECK(capacity >= 0, op, ": capacity must not be negative");
  ExpertRowsView v;
  const int64_t experts = counts.size(0);
  const int64_t rows = capacity > 0 ? experts * capacity : row_of.numel();
  TORCH_CHECK(capacity <= kMaxRows && rows <= kMaxRows && row_of.numel() <= kMaxRows, op,
              ": more than 2^30 rows");
  v.counts = data<int32_t>(counts);
  v.offsets = data<int32_t>(offsets);
  v.row_of = data<int32_t>(row_of);
  v.num_tokens = static_cast<int>(row_of.size(0));
  v.topk = static_cast<int>(row_of.size(1));
  v.num_experts = static_cast<int>(experts);
  v.capacity = static_cast<int>(capacity);
  v.num_rows = rows;
  return v;
}

const uint32_t* bound_ptr(const std::optional<at::Tensor>& bound_m, const at::Tensor& like,
                          const char* op) {
  if (!bound_m.has_value()) return nullptr;
  check_device(*bound_m, like, op, "bound_m");
  TORCH_CHECK(bound_m->numel() == 1 && bound_m->element_size() == 4 &&
                  !bound_m->is_floating_point(),
              op, ": bound_m must be a 32-bit integer scalar tensor");
  return data<const uint32_t>(*bound_m);
}

const float* weights_ptr(const at::Tensor& weights, const ExpertRowsView& v, const at::Tensor& like,
                         const char* op) {
  check_device(weights, like, op, "weights");
  TORCH_CHECK(weights.scalar_type() == at::kFloat && weights.dim() == 2 &&
                  weights.size(0) == v.num_tokens && weights.size(1) == v.topk &&
                  weights.is_contiguous(),
              op, ": weights must be a contiguous float32 tensor of [", v.num_tokens, ", ", v.topk,
              "]");
  return data<float>(weights);
}

// ------------------------------------------------------------------------ sort ----

std::tuple<at::Tensor, at::Tensor, at::Tensor> sort_by_expert_op(
    const at::Tensor& indices, int64_t num_experts, int64_t capacity,
    const std::optional<at::Tensor>& bound_m) {
  const char* op = "sort_by_expert";
  check_device(indices, op, "indices");
  TORCH_CHECK(indices.scalar_type() == at::kInt || indices.scalar_type() == at::kUInt32 ||
                  indices.scalar_type() == at::kLong,
              op, ": indices must be int32, uint32 or int64");
  TORCH_CHECK(indices.dim() == 2 && indices.size(1) > 0 && indices.is_contiguous(), op,
              ": indices must be contiguous, [tokens, topk]");
  TORCH_CHECK(num_experts > 0 && num_experts <= 1024, op, ": num_experts must be in [1, 1024]");
  TORCH_CHECK(capacity >= 0, op, ": capacity must not be negative");
  TORCH_CHECK(indices.numel() <= kMaxRows && capacity <= kMaxRows &&
                  num_experts * capacity <= kMaxRows,
              op, ": more than 2^30 rows");
  const uint32_t* bound = bound_ptr(bound_m, indices, op);
  at::Tensor counts = empty({num_experts}, indices, at::kInt);
  at::Tensor offsets = empty({num_experts + 1}, indices, at::kInt);
  at::Tensor row_of = empty(indices.sizes(), indices, at::kInt);
  SortByExpertCall c;
  c.indices = data<void>(indices);
  c.wide_indices = indices.scalar_type() == at::kLong;
  c.bound_m = bound;
  c.num_tokens = static_cast<int>(indices.size(0));
  c.topk = static_cast<int>(indices.size(1));
  c.num_experts = static_cast<int>(num_experts);
  c.capacity = static_cast<int>(capacity);
  c.counts = data<int32_t>(counts);
  c.offsets = data<int32_t>(offsets);
  c.row_of = data<int32_t>(row_of);
  launch_on(indices, [&](cudaStream_t stream) { launch_sort_by_expert(c, stream); });
  return {counts, offsets, row_of};
}

// --------------------------------------------------------------------- permute ----

at::Tensor empty_rows(const at::Tensor& x, const at::Tensor& counts, const at::Tensor& row_of,
                      int64_t capacity, at::ScalarType type) {
  TORCH_CHECK(x.dim() == 2 && counts.dim() == 1 && capacity >= 0 && capacity <= kMaxRows,
              "tokens must be [tokens, hidden], counts [experts] and capacity not negative");
  if (capacity > 0) return empty({counts.size(0), capacity, x.size(1)}, x, type);
  return empty({row_of.numel(), x.size(1)}, x, type);
}

void permute_tokens_out_op(const at::Tensor& x, const at::Tensor& counts, const at::Tensor& offsets,
                       const at::Tensor& row_of, int64_t capacity, at::Tensor& out,
                       bool zero_rest) {
  const char* op = "permute_tokens";
  check_device(x, op, "x");
  PermuteCall c;
  c.rows = make_view(counts, offsets, row_of, capacity, x, op);
  c.x_stride = token_stride(x, op, "x") * x.element_size();
  TORCH_CHECK(x.size(0) == c.rows.num_tokens, op, ": x and row_of disagree on the token count");
  check_hidden(x.size(1), op);
  check_rows(out, c.rows, x.size(1), x, op, "out");
  TORCH_CHECK(out.scalar_type() == x.scalar_type(), op, ": out must have the type of x");
  check_apart(out, x, op, "out", "x");
  c.x = data<void>(x);
  c.out = data<void>(out);
  c.row_bytes = x.size(1) * x.element_size();
  c.zero_rest = zero_rest;
  launch_on(x, [&](cudaStream_t stream) { launch_permute_tokens(c, stream); });
}

at::Tensor permute_tokens_op(const at::Tensor& x, const at::Tensor& counts, const at::Tensor& offsets,
                             const at::Tensor& row_of, int64_t capacity, bool zero_rest) {
  at::Tensor out = empty_rows(x, counts, row_of, capacity, x.scalar_type());
  permute_tokens_out_op(x, counts, offsets, row_of, capacity, out, zero_rest);
  return out;
}

void permute_tokens_int8_out_op(const at::Tensor& x, const at::Tensor& counts, const at::Tensor& offsets,
                            const at::Tensor& row_of, int64_t capacity, at::Tensor& out,
                            at::Tensor& out_scale, bool zero_rest) {
  const char* op = "permute_tokens_int8";
  check_device(x, op, "x");
  const ExpertRowsView v = make_view(counts, offsets, row_of, capacity, x, op);
  QuantizeRowsCall c;
  c.rows = &v;
  c.x_stride = token_stride(x, op, "x");
  c.type = float_type(x, op, "x");
  TORCH_CHECK(x.size(0) == v.num_tokens, op, ": x and row_of disagree on the token count");
  check_hidden(x.size(1), op);
  check_rows(out, v, x.size(1), x, op, "out");
  check_device(out_scale, x, op, "out_scale");
  TORCH_CHECK(out.scalar_type() == at::kChar, op, ": out must be int8");
  TORCH_CHECK(out_scale.scalar_type() == at::kFloat && out_scale.is_contiguous() &&
                  out_scale.sizes() == out.sizes().slice(0, out.dim() - 1),
              op, ": out_scale must be contiguous float32, one per row of out");
  check_apart(out, x, op, "out", "x");
  check_apart(out_scale, x, op, "out_scale", "x");
  c.zero_rest = zero_rest;
  c.x = data<void>(x);
  c.q = data<int8_t>(out);
  c.scale = data<float>(out_scale);
  c.hidden = static_cast<int>(x.size(1));
  launch_on(x, [&](cudaStream_t stream) { launch_quantize_rows(c, stream); });
}

std::tuple<at::Tensor, at::Tensor> permute_tokens_int8_op(
    const at::Tensor& x, const at::Tensor& counts, const at::Tensor& offsets,
    const at::Tensor& row_of, int64_t capacity, bool zero_rest) {
  at::Tensor out = empty_rows(x, counts, row_of, capacity, at::kChar);
  at::Tensor scale = empty(out.sizes().slice(0, out.dim() - 1), x, at::kFloat);
  permute_tokens_int8_out_op(x, counts, offsets, row_of, capacity, out, scale, zero_rest);
  return {out, scale};
}

// ------------------------------------------------------------------- unpermute ----

void unpermute_tokens_out_op(const at::Tensor& y, const at::Tensor& counts, const at::Tensor& offsets,
                         const at::Tensor& row_of, int64_t capacity,
                         const std::optional<at::Tensor>& weights, at::Tensor& out,
                         const std::optional<at::Tensor>& bound_m) {
  const char* op = "unpermute_tokens";
  check_device(y, op, "y");
  UnpermuteCall c;
  c.rows = make_view(counts, offsets, row_of, capacity, y, op);
  c.type = float_type(y, op, "y");
  c.out_stride = token_stride(out, op, "out");
  check_device(out, y, op, "out");
  TORCH_CHECK(out.scalar_type() == y.scalar_type(), op, ": out must have the type of y");
  TORCH_CHECK(out.size(0) >= c.rows.num_tokens, op, ": out has fewer rows than row_of");
  check_hidden(out.size(1), op);
  check_rows(y, c.rows, out.size(1), y, op, "y");
  check_apart(out, y, op, "out", "y");
  if (weights.has_value()) c.weights = weights_ptr(*weights, c.rows, y, op);
  c.bound_m = bound_ptr(bound_m, y, op);
  c.y = data<void>(y);
  c.out = data<void>(out);
  c.hidden = static_cast<int>(out.size(1));
  launch_on(y, [&](cudaStream_t stream) { launch_unpermute_tokens(c, stream); });
}

at::Tensor unpermute_tokens_op(const at::Tensor& y, const at::Tensor& counts,
                               const at::Tensor& offsets, const at::Tensor& row_of,
                               int64_t capacity, const std::optional<at::Tensor>& weights) {
  TORCH_CHECK(y.dim() >= 1 && row_of.dim() == 2, "unpermute_tokens: y must be rows, row_of [tokens, topk]");
  at::Tensor out = empty({row_of.size(0), y.size(-1)}, y, y.scalar_type());
  unpermute_tokens_out_op(y, counts, offsets, row_of, capacity, weights, out, std::nullopt);
  return out;
}

void unpermute_tokens_backward_op(const at::Tensor& grad, const std::optional<at::Tensor>& y,
                                  const at::Tensor& counts, const at::Tensor& offsets,
                                  const at::Tensor& row_of, int64_t capacity,
                                  const at::Tensor& weights,
                                  const std::optional<at::Tensor>& grad_y,
                                  const std::optional<at::Tensor>& grad_weights) {
  const char* op = "unpermute_tokens_backward";
  check_device(grad, op, "grad");
  UnpermuteBackwardCall c;
  c.rows = make_view(counts, offsets, row_of, capacity, grad, op);
  c.type = float_type(grad, op, "grad");
  c.grad_stride = token_stride(grad, op, "grad");
  const int64_t hidden = grad.size(1);
  check_hidden(hidden, op);
  TORCH_CHECK(grad.size(0) == c.rows.num_tokens, op, ": grad and row_of disagree on the token count");
  if (y.has_value()) {
    check_rows(*y, c.rows, hidden, grad, op, "y");
    TORCH_CHECK(y->scalar_type() == grad.scalar_type(), op, ": grad must have the type of y");
    c.y = data<void>(*y);
  }
  TORCH_CHECK(y.has_value() || !grad_weights.has_value(), op, ": grad_weights needs y");
  c.weights = weights_ptr(weights, c.rows, grad, op);
  c.grad = data<void>(grad);
  c.hidden = static_cast<int>(hidden);
  if (grad_y.has_value()) {
    check_rows(*grad_y, c.rows, hidden, grad, op, "grad_y");
    TORCH_CHECK(grad_y->scalar_type() == grad.scalar_type(), op, ": grad_y must have the type of grad");
    c.grad_y = data<void>(*grad_y);
  }
  if (grad_weights.has_value()) {
    check_device(*grad_weights, grad, op, "grad_weights");
    TORCH_CHECK(grad_weights->scalar_type() == at::kFloat && grad_weights->is_contiguous() &&
                    grad_weights->sizes() == row_of.sizes(),
                op, ": grad_weights must be a contiguous float32 tensor like row_of");
    c.grad_weights = data<float>(*grad_weights);
  }
  launch_on(grad, [&](cudaStream_t stream) { launch_unpermute_backward(c, stream); });
}

// ------------------------------------------------------------------- gradients ----

using Variables = torch::autograd::variable_list;
using torch::autograd::AutogradContext;

at::Tensor call_permute(const at::Tensor& x, const at::Tensor& counts, const at::Tensor& offsets,
                        const at::Tensor& row_of, int64_t capacity, bool zero_rest) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pplx_kernels_b200::permute_tokens", "")
                       .typed<decltype(permute_tokens_op)>();
  return op.call(x, counts, offsets, row_of, capacity, zero_rest);
}

at::Tensor call_unpermute(const at::Tensor& y, const at::Tensor& counts, const at::Tensor& offsets,
                          const at::Tensor& row_of, int64_t capacity,
                          const std::optional<at::Tensor>& weights) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pplx_kernels_b200::unpermute_tokens", "")
                       .typed<decltype(unpermute_tokens_op)>();
  return op.call(y, counts, offsets, row_of, capacity, weights);
}

void call_unpermute_backward(const at::Tensor& grad, const std::optional<at::Tensor>& y,
                             const at::Tensor& counts, const at::Tensor& offsets,
                             const at::Tensor& row_of, int64_t capacity, const at::Tensor& weights,
                             const std::optional<at::Tensor>& grad_y,
                             const std::optional<at::Tensor>& grad_weights) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("pplx_kernels_b200::unpermute_tokens_backward", "")
                       .typed<decltype(unpermute_tokens_backward_op)>();
  op.call(grad, y, counts, offsets, row_of, capacity, weights, grad_y, grad_weights);
}

// Rows without a token are zero where a gradient is recorded: what is computed with them may enter
// the gradients of weights, multiplied by zeros.
class Permute : public torch::autograd::Function<Permute> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& counts,
                            const at::Tensor& offsets, const at::Tensor& row_of, int64_t capacity) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({counts, offsets, row_of});
    ctx->saved_data["capacity"] = capacity;
    return call_permute(x, counts, offsets, row_of, capacity, true);
  }
  static Variables backward(AutogradContext* ctx, const Variables& grads) {
    const Variables rows = ctx->get_saved_variables();
    return {call_unpermute(grads[0].contiguous(), rows[0], rows[1], rows[2],
                           ctx->saved_data["capacity"].toInt(), std::nullopt),
            {}, {}, {}, {}};
  }
};

class Unpermute : public torch::autograd::Function<Unpermute> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& weights,
                            const at::Tensor& counts, const at::Tensor& offsets,
                            const at::Tensor& row_of, int64_t capacity) {
    at::AutoDispatchBelowADInplaceOrView below;
    // (Only the gradient of the weights reads the rows: without it they need not be kept.)
    ctx->save_for_backward({weights.requires_grad() ? y : at::Tensor(), weights, counts, offsets, row_of});
    ctx->saved_data["capacity"] = capacity;
    return call_unpermute(y, counts, offsets, row_of, capacity, weights);
  }
  static Variables backward(AutogradContext* ctx, const Variables& grads) {
    const Variables saved = ctx->get_saved_variables();
    const at::Tensor &y = saved[0], &weights = saved[1], grad = grads[0].contiguous();
    const int64_t capacity = ctx->saved_data["capacity"].toInt();
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "unpermute_tokens: its gradient has no derivative of its own (create_graph)");
    at::Tensor grad_y, grad_weights;
    if (ctx->needs_input_grad(0))
      grad_y = empty_rows(grad, saved[2], saved[4], capacity, grad.scalar_type());
    if (ctx->needs_input_grad(1)) grad_weights = at::empty_like(weights);
    auto given = [](const at::Tensor& t) {
      return t.defined() ? std::optional<at::Tensor>(t) : std::nullopt;
    };
    call_unpermute_backward(grad, given(y), saved[2], saved[3], saved[4], capacity, weights,
                            given(grad_y), given(grad_weights));
    return {grad_y, grad_weights, {}, {}, {}, {}};
  }
};

class Sum : public torch::autograd::Function<Sum> {  // unpermute without weights
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& counts,
                            const at::Tensor& offsets, const at::Tensor& row_of, int64_t capacity) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({counts, offsets, row_of});
    ctx->saved_data["capacity"] = capacity;
    return call_unpermute(y, counts, offsets, row_of, capacity, std::nullopt);
  }
  static Variables backward(AutogradContext* ctx, const Variables& grads) {
    const Variables rows = ctx->get_saved_variables();
    return {call_permute(grads[0].contiguous(), rows[0], rows[1], rows[2],
                         ctx->saved_data["capacity"].toInt(), true),
            {}, {}, {}, {}};
  }
};

// No operator has a forward-mode derivative: a tangent would be dropped without a word and count as
// zero in what follows, so a tensor that carries one is refused.
void check_no_tangent(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), op, ": ", name,
              " carries a tangent; forward-mode derivatives are not implemented");
}

// fn(tensor, argument) for the tensors on the stack that `schema` describes.
template <typename F>
void for_tensors(const c10::FunctionSchema& schema, const torch::jit::Stack& stack, F&& fn) {
  const size_t n = schema.arguments().size(), first = stack.size() - n;
  for (size_t i = 0; i < n; ++i)
    if (stack[first + i].isTensor() && stack[first + i].toTensor().defined())
      fn(stack[first + i].toTensor(), schema.arguments()[i]);
}

bool is_written(const c10::Argument& argument) {
  return argument.alias_info() != nullptr && argument.alias_info()->isWrite();
}

// What operators without a gradient of their own do in place of recording one.  A written tensor that a
// gradient is recorded for is refused, as by torch's own `out=`.
void not_differentiable(const c10::OperatorHandle& op, c10::DispatchKeySet keys,
                        torch::jit::Stack* stack) {
  const char* name = op.schema().name().c_str() + op.schema().name().rfind(':') + 1;
  for_tensors(op.schema(), *stack, [&](const at::Tensor& t, const c10::Argument& argument) {
    check_no_tangent(t, name, argument.name().c_str());
    TORCH_CHECK(!(is_written(argument) && t.requires_grad() && at::GradMode::is_enabled()), name, ": ",
                argument.name(),
                " is written and requires a gradient, which is not recorded; use torch.no_grad() or detach()");
  });
  op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
}

// Written tensors count as changed, so that a backward pass that saved them notices (in inference mode as
// well, where only tensors made there have no version).
void count_changes(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  c10::SmallVector<at::Tensor, 4> written;
  for_tensors(op.schema(), *stack, [&](const at::Tensor& t, const c10::Argument& argument) {
    if (is_written(argument) && !t.is_inference()) written.push_back(t);
  });
  op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
  for (const at::Tensor& t : written) torch::autograd::impl::bump_version(t);
}

at::Tensor permute_tokens_autograd(const at::Tensor& x, const at::Tensor& counts,
                                   const at::Tensor& offsets, const at::Tensor& row_of,
                                   int64_t capacity, bool zero_rest) {
  check_no_tangent(x, "permute_tokens", "x");
  if (at::GradMode::is_enabled() && x.requires_grad()) {
    // (Any type is copied, but the gradient is a sum of rows: refused here, not in the backward pass.)
    float_type(x, "permute_tokens", "x, which requires a gradient,");
    return Permute::apply(x, counts, offsets, row_of, capacity);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_permute(x, counts, offsets, row_of, capacity, zero_rest);
}

at::Tensor unpermute_tokens_autograd(const at::Tensor& y, const at::Tensor& counts,
                                     const at::Tensor& offsets, const at::Tensor& row_of,
                                     int64_t capacity, const std::optional<at::Tensor>& weights) {
  check_no_tangent(y, "unpermute_tokens", "y");
  if (weights.has_value()) check_no_tangent(*weights, "unpermute_tokens", "weights");
  if (at::GradMode::is_enabled()) {
    if (weights.has_value() && (y.requires_grad() || weights->requires_grad()))
      return Unpermute::apply(y, *weights, counts, offsets, row_of, capacity);
    if (y.requires_grad()) return Sum::apply(y, counts, offsets, row_of, capacity);
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return call_unpermute(y, counts, offsets, row_of, capacity, weights);
}

// -------------------------------------------------------------------- int8 ----

void quantize_rows_int8_out_op(const at::Tensor& x, const std::optional<at::Tensor>& counts,
                           at::Tensor& out, at::Tensor& out_scale) {
  const char* op = "quantize_rows_int8";
  check_device(x, op, "x");
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3, op, ": x must be [rows, k] or [experts, rows, k]");
  const int64_t planes = x.dim() == 3 ? x.size(0) : 1;
  const int64_t rows = x.size(-2), k = x.size(-1);
  QuantizeRowsCall c;
  c.type = float_type(x, op, "x");
  TORCH_CHECK(k <= 1 || x.stride(-1) == 1, op, ": the columns of x must be contiguous");
  c.x_stride = rows > 1 ? x.stride(-2) : planes > 1 ? x.stride(0) : k;
  TORCH_CHECK(planes <= 1 || x.stride(0) == rows * c.x_stride, op,
              ": the experts' rows of x must follow each other evenly");
  TORCH_CHECK(planes * rows <= 1 || c.x_stride >= k, op, ": the rows of x must not overlap");
  check_hidden(k, op);
  check_device(out, x, op, "out");
  check_device(out_scale, x, op, "out_scale");
  TORCH_CHECK(out.scalar_type() == at::kChar && out.sizes() == x.sizes() && out.is_contiguous(), op,
              ": out must be a contiguous int8 tensor like x");
  TORCH_CHECK(out_scale.scalar_type() == at::kFloat && out_scale.is_contiguous() &&
                  out_scale.sizes() == x.sizes().slice(0, x.dim() - 1),
              op, ": out_scale must be contiguous float32, one per row of x");
  check_apart(out, x, op, "out", "x");
  check_apart(out_scale, x, op, "out_scale", "x");
  if (counts.has_value()) {
    check_device(*counts, x, op, "counts");
    TORCH_CHECK(x.dim() == 3 && counts->scalar_type() == at::kInt && counts->is_contiguous() &&
                    counts->dim() == 1 && counts->size(0) == planes,
                op, ": counts must be a contiguous int32 tensor of [experts], for x of [experts, "
                "rows, k]");
    c.counts = data<int32_t>(*counts);
  }
  TORCH_CHECK(rows <= kMaxRows, op, ": more than 2^30 rows");
  c.plane_rows = static_cast<int>(rows);
  c.num_rows = planes * rows;
  c.x = data<void>(x);
  c.q = data<int8_t>(out);
  c.scale = data<float>(out_scale);
  c.hidden = static_cast<int>(k);
  launch_on(x, [&](cudaStream_t stream) { launch_quantize_rows(c, stream); });
}

std::tuple<at::Tensor, at::Tensor> quantize_rows_int8_op(const at::Tensor& x,
                                                         const std::optional<at::Tensor>& counts) {
  TORCH_CHECK(x.dim() == 2 || x.dim() == 3,
              "quantize_rows_int8: x must be [rows, k] or [experts, rows, k]");
  at::Tensor out = empty(x.sizes(), x, at::kChar);
  at::Tensor scale = empty(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  quantize_rows_int8_out_op(x, counts, out, scale);
  return {out, scale};
}

// Stride of a dimension; one that is never used counts as `packed`.
int64_t used_stride(const at::Tensor& t, int64_t dim, int64_t packed) {
  return t.size(dim) > 1 ? t.stride(dim) : packed;
}

void grouped_gemm_int8_op(const at::Tensor& xq, const at::Tensor& x_scale, const at::Tensor& wq,
                          const at::Tensor& w_scale, const std::optional<at::Tensor>& counts,
                          const std::optional<at::Tensor>& offsets, at::Tensor& out, bool swiglu,
                          const std::optional<at::Tensor>& status, int64_t expected_rows) {
  const char* op = "grouped_gemm_int8";
  check_device(xq, op, "xq");
  check_device(x_scale, xq, op, "x_scale");
  check_device(wq, xq, op, "wq");
  check_device(w_scale, xq, op, "w_scale");
  check_device(out, xq, op, "out");
  const bool one_plane = offsets.has_value();
  const int64_t d = one_plane ? 2 : 3;
  TORCH_CHECK(xq.scalar_type() == at::kChar && wq.scalar_type() == at::kChar, op,
              ": xq and wq must be int8");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kHalf, op,
              ": out must be bfloat16 or float16");
  TORCH_CHECK(xq.dim() == d && out.dim() == d && wq.dim() == 3, op, ": xq and out must be ",
              one_plane ? "[rows, k] and [rows, n_out] where offsets are given"
                        : "[experts, rows, k] and [experts, rows, n_out] where no offsets are given",
              ", wq [experts, n, k]");
  const int64_t E = wq.size(0), rows = xq.size(-2), k = xq.size(-1), n_out = out.size(-1);
  const int64_t w_rows = swiglu ? 2 * n_out : n_out;
  TORCH_CHECK(wq.size(1) == w_rows && wq.size(2) == k, op, ": wq must be [experts, ",
              swiglu ? "2 * " : "", "n_out, k]");
  TORCH_CHECK(out.size(-2) == rows && (one_plane || (xq.size(0) == E && out.size(0) == E)), op,
              ": xq, wq and out disagree on the experts or rows");
  TORCH_CHECK(xq.stride(-1) == 1 && wq.stride(2) == 1 && out.stride(-1) == 1, op,
              ": the last dimension must be contiguous");
  TORCH_CHECK(x_scale.scalar_type() == at::kFloat && w_scale.scalar_type() == at::kFloat, op,
              ": scales must be float32");
  TORCH_CHECK(x_scale.sizes() == xq.sizes().slice(0, d - 1) && x_scale.is_contiguous(), op,
              ": x_scale must be contiguous, one per row of xq");
  TORCH_CHECK(w_scale.dim() == 2 && w_scale.size(0) == E && w_scale.size(1) == w_rows &&
                  w_scale.is_contiguous(),
              op, ": w_scale must be contiguous, [experts, rows of wq]");
  TORCH_CHECK(rows <= kMaxRows && n_out <= kMaxRows, op, ": more than 2^30 rows or columns");
  Int8GemmCall c;
  if (counts.has_value()) {
    check_device(*counts, xq, op, "counts");
    TORCH_CHECK(counts->scalar_type() == at::kInt && counts->dim() == 1 && counts->size(0) == E &&
                    counts->is_contiguous(),
                op, ": counts must be a contiguous int32 tensor of [experts]");
    c.counts = data<int32_t>(*counts);
  }
  if (one_plane) {
    check_device(*offsets, xq, op, "offsets");
    TORCH_CHECK(counts.has_value(), op, ": offsets need counts");
    TORCH_CHECK(offsets->scalar_type() == at::kInt && offsets->dim() == 1 &&
                    (offsets->size(0) == E || offsets->size(0) == E + 1) && offsets->is_contiguous(),
                op, ": offsets must be a contiguous int32 tensor of [experts] or [experts + 1]");
    c.offsets = data<int32_t>(*offsets);
  }
  if (status.has_value()) {
    check_device(*status, xq, op, "status");
    TORCH_CHECK(status->element_size() == 4 && status->numel() >= 1, op,
                ": status must be a 32-bit CUDA tensor");
    c.status = data<uint32_t>(*status);
  }
  TORCH_CHECK(expected_rows >= 0, op, ": expected_rows must not be negative");
  c.x = data<void>(xq);
  c.x_stride_row = used_stride(xq, d - 2, k);
  c.x_stride_e = one_plane ? 0 : used_stride(xq, 0, rows * c.x_stride_row);
  c.sx = data<float>(x_scale);
  c.sx_stride_e = one_plane ? 0 : rows;
  c.w = data<void>(wq);
  c.w_stride_row = used_stride(wq, 1, k);
  c.w_stride_e = used_stride(wq, 0, w_rows * c.w_stride_row);
  c.sw = data<float>(w_scale);
  c.sw_stride_e = w_rows;
  c.out = data<void>(out);
  c.out_stride_row = used_stride(out, d - 2, n_out);
  c.out_stride_e = one_plane ? 0 : used_stride(out, 0, rows * c.out_stride_row);
  TORCH_CHECK(c.x_stride_row >= k && c.w_stride_row >= k && c.out_stride_row >= n_out, op,
              ": rows must not overlap");
  // (Planes behind each other, or rows of all experts in turn.)
  TORCH_CHECK(one_plane || E <= 1 || c.out_stride_e >= (rows - 1) * c.out_stride_row + n_out ||
                  (c.out_stride_e >= n_out && c.out_stride_row >= (E - 1) * c.out_stride_e + n_out),
              op, ": the experts' rows of out must not overlap");
  check_apart(out, xq, op, "out", "xq");
  c.num_experts = static_cast<int>(E);
  c.rows_per_expert = static_cast<int>(rows);
  c.n_out = static_cast<int>(n_out);
  TORCH_CHECK(k <= kMaxRows, op, ": k is too large");
  c.k = static_cast<int>(k);
  c.swiglu = swiglu;
  c.fp16 = out.scalar_type() == at::kHalf;
  c.expected_total_rows = expected_rows;
  try {
    check_grouped_gemm_int8(c);
  } catch (const Error& e) {
    TORCH_CHECK(false, e.what());
  }
  launch_on(xq, [&](cudaStream_t stream) { launch_grouped_gemm_int8(c, stream); });
}

}  // namespace

void register_expert_ops(torch::Library& m) {
  m.def("sort_by_expert(Tensor indices, int num_experts, int capacity, Tensor? bound_m) -> "
        "(Tensor counts, Tensor offsets, Tensor row_of)");
  m.impl("sort_by_expert", c10::kCUDA, &sort_by_expert_op);
  m.impl("sort_by_expert", c10::kMeta, &sort_by_expert_op);
  m.def("permute_tokens(Tensor x, Tensor counts, Tensor offsets, Tensor row_of, int capacity, "
        "bool zero_rest) -> Tensor");
  m.impl("permute_tokens", c10::kCUDA, &permute_tokens_op);
  m.impl("permute_tokens", c10::kMeta, &permute_tokens_op);
  m.impl("permute_tokens", torch::dispatch(c10::DispatchKey::Autograd, &permute_tokens_autograd));
  m.def("permute_tokens_out(Tensor x, Tensor counts, Tensor offsets, Tensor row_of, int capacity, "
        "Tensor! out, bool zero_rest) -> ()");
  m.impl("permute_tokens_out", c10::kCUDA, &permute_tokens_out_op);
  m.impl("permute_tokens_out", c10::kMeta, &permute_tokens_out_op);
  m.def("permute_tokens_int8(Tensor x, Tensor counts, Tensor offsets, Tensor row_of, int capacity, "
        "bool zero_rest) -> (Tensor out, Tensor out_scale)");
  m.impl("permute_tokens_int8", c10::kCUDA, &permute_tokens_int8_op);
  m.impl("permute_tokens_int8", c10::kMeta, &permute_tokens_int8_op);
  m.def("permute_tokens_int8_out(Tensor x, Tensor counts, Tensor offsets, Tensor row_of, "
        "int capacity, Tensor! out, Tensor! out_scale, bool zero_rest) -> ()");
  m.impl("permute_tokens_int8_out", c10::kCUDA, &permute_tokens_int8_out_op);
  m.impl("permute_tokens_int8_out", c10::kMeta, &permute_tokens_int8_out_op);
  m.def("unpermute_tokens(Tensor y, Tensor counts, Tensor offsets, Tensor row_of, int capacity, "
        "Tensor? weights) -> Tensor");
  m.impl("unpermute_tokens", c10::kCUDA, &unpermute_tokens_op);
  m.impl("unpermute_tokens", c10::kMeta, &unpermute_tokens_op);
  m.impl("unpermute_tokens", torch::dispatch(c10::DispatchKey::Autograd, &unpermute_tokens_autograd));
  m.def("unpermute_tokens_out(Tensor y, Tensor counts, Tensor offsets, Tensor row_of, int capacity, "
        "Tensor? weights, Tensor! out, Tensor? bound_m) -> ()");
  m.impl("unpermute_tokens_out", c10::kCUDA, &unpermute_tokens_out_op);
  m.impl("unpermute_tokens_out", c10::kMeta, &unpermute_tokens_out_op);
  m.def("unpermute_tokens_backward(Tensor grad, Tensor? y, Tensor counts, Tensor offsets, "
        "Tensor row_of, int capacity, Tensor weights, Tensor!? grad_y, Tensor!? grad_weights) -> ()");
  m.impl("unpermute_tokens_backward", c10::kCUDA, &unpermute_tokens_backward_op);
  m.impl("unpermute_tokens_backward", c10::kMeta, &unpermute_tokens_backward_op);
  m.def("quantize_rows_int8(Tensor x, Tensor? counts) -> (Tensor out, Tensor out_scale)");
  m.impl("quantize_rows_int8", c10::kCUDA, &quantize_rows_int8_op);
  m.impl("quantize_rows_int8", c10::kMeta, &quantize_rows_int8_op);
  m.def("quantize_rows_int8_out(Tensor x, Tensor? counts, Tensor! out, Tensor! out_scale) -> ()");
  m.impl("quantize_rows_int8_out", c10::kCUDA, &quantize_rows_int8_out_op);
  m.impl("quantize_rows_int8_out", c10::kMeta, &quantize_rows_int8_out_op);
  m.def("grouped_gemm_int8(Tensor xq, Tensor x_scale, Tensor wq, Tensor w_scale, Tensor? counts, "
        "Tensor? offsets, Tensor! out, bool swiglu, Tensor!? status, int expected_rows=0) -> ()");
  m.impl("grouped_gemm_int8", c10::kCUDA, &grouped_gemm_int8_op);
  m.impl("grouped_gemm_int8", c10::kMeta, &grouped_gemm_int8_op);
  for (const char* op : {"permute_tokens_out", "permute_tokens_int8", "permute_tokens_int8_out",
                         "unpermute_tokens_out", "unpermute_tokens_backward", "quantize_rows_int8",
                         "quantize_rows_int8_out", "grouped_gemm_int8"})
    m.impl(op, c10::DispatchKey::Autograd,
           torch::CppFunction::makeFromBoxedFunction<&not_differentiable>());
  for (const char* op : {"permute_tokens_out", "permute_tokens_int8_out", "unpermute_tokens_out",
                         "unpermute_tokens_backward", "quantize_rows_int8_out", "grouped_gemm_int8"})
    m.impl(op, c10::DispatchKey::ADInplaceOrView,
           torch::CppFunction::makeFromBoxedFunction<&count_changes>());
}

}  // namespace pplx
