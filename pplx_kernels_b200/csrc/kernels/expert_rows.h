// Tokens sorted by expert and back on one GPU, and the quantisation of rows to 8-bit integers --
// host interface.  No counterpart in the reference, whose tokens always pass through its all-to-all.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace pplx {

enum class FloatType { kBFloat16, kHalf, kFloat };

// Where the rows of the experts are.  Rows of expert e: offsets[e] .. offsets[e] + counts[e].
// capacity 0: one expert's rows after the other's, offsets[num_experts] in all; otherwise
// offsets[e] = e * capacity.  Kernels that take a view skip rows outside [0, num_rows).
struct ExpertRowsView {
  const int32_t* counts = nullptr;   // [num_experts]
  const int32_t* offsets = nullptr;  // [num_experts + 1]
  const int32_t* row_of = nullptr;   // [num_tokens][topk], -1 for an entry without a row
  int num_tokens = 0, topk = 0, num_experts = 0, capacity = 0;
  int64_t num_rows = 0;              // rows of the tensor of rows
};

// Stable counting sort of the routing: entries of one expert keep the order of (token, k).
// Entries that name no expert of [0, num_experts), that belong to tokens at or beyond *bound_m or
// that come after `capacity` others of their expert get no row.
struct SortByExpertCall {
  const void* indices = nullptr;  // [num_tokens][topk]
  bool wide_indices = false;      // 64-bit integers, otherwise 32-bit
  const uint32_t* bound_m = nullptr;
  int num_tokens = 0, topk = 0, num_experts = 0, capacity = 0;
  int32_t* counts = nullptr;
  int32_t* offsets = nullptr;
  int32_t* row_of = nullptr;
};
void launch_sort_by_expert(const SortByExpertCall& call, cudaStream_t stream);

// rows[row_of[t, k]] = x[t].  zero_rest: rows that no entry has are set to zero, otherwise they are
// untouched.
struct PermuteCall {
  ExpertRowsView rows;
  const void* x = nullptr;
  int64_t x_stride = 0;   // bytes
  void* out = nullptr;    // [num_rows] packed rows
  int64_t row_bytes = 0;
  bool zero_rest = false;
  bool streaming = false;  // set by the launcher
};
void launch_permute_tokens(const PermuteCall& call, cudaStream_t stream);

// out[t] = sum over k of weights[t, k] * y[row_of[t, k]] (weights null: 1), in fp32, rounded once.
// Tokens without a row are set to zero; tokens at or beyond *bound_m are untouched.
struct UnpermuteCall {
  ExpertRowsView rows;
  FloatType type = FloatType::kBFloat16;
  const void* y = nullptr;             // [num_rows] packed rows
  const float* weights = nullptr;      // [num_tokens][topk]
  const uint32_t* bound_m = nullptr;
  void* out = nullptr;
  int64_t out_stride = 0;              // elements
  int hidden = 0;
  bool streaming = false;              // set by the launcher
};
void launch_unpermute_tokens(const UnpermuteCall& call, cudaStream_t stream);

// Gradients of the above for that of out: grad_y[row_of[t, k]] = weights[t, k] * grad[t], rows that
// no entry has zero; grad_weights[t, k] = <y[row_of[t, k]], grad[t]>, 0 for an entry without a row.
struct UnpermuteBackwardCall {
  ExpertRowsView rows;
  FloatType type = FloatType::kBFloat16;
  const void* grad = nullptr;
  int64_t grad_stride = 0;             // elements
  const void* y = nullptr;             // read for grad_weights only
  const float* weights = nullptr;
  void* grad_y = nullptr;              // optional
  float* grad_weights = nullptr;       // optional
  int hidden = 0;
};
void launch_unpermute_backward(const UnpermuteBackwardCall& call, cudaStream_t stream);

// Rows to 8-bit integers: a = max(max |x|, 1e-30), scale = a * (1 / 127), q = rint(x * (127 * (1 / a))), each
// step rounded to fp32.
// `rows` given: the row of token t goes to every row_of[t, k] (zero_rest as above).  Otherwise row
// r of `num_rows` goes to row r; with `counts`, rows r % plane_rows >= counts[r / plane_rows] are
// skipped.
struct QuantizeRowsCall {
  const ExpertRowsView* rows = nullptr;
  bool zero_rest = false;
  const int32_t* counts = nullptr;
  int plane_rows = 0;
  int64_t num_rows = 0;
  FloatType type = FloatType::kBFloat16;
  const void* x = nullptr;
  int64_t x_stride = 0;   // elements
  int8_t* q = nullptr;    // packed rows
  float* scale = nullptr;
  int hidden = 0;
  bool streaming = false;  // set by the launcher
};
void launch_quantize_rows(const QuantizeRowsCall& call, cudaStream_t stream);

}  // namespace pplx
