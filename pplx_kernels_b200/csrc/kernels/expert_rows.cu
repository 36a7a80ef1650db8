// Tokens sorted by expert and back on one GPU, with the gradients, and rows quantised to 8-bit
// integers.  All of it is bound by memory: the sort reads and writes a few bytes per entry of the
// routing, the others read each token (or row) once and write each row (or token) once.
//
// Every kernel goes token by token: the rows of a token are found through row_of, so a token is
// read once for all its rows, and the order in which a token's rows are summed is that of its
// entries, whatever the experts are.  No atomics: the same call gives the same bits.
#include "expert_rows.h"

#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../core/device_utils.cuh"
#include "../core/ptx.cuh"
#include "../core/utils.h"

namespace pplx {
namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kMaxSortExperts = 1024;

// ------------------------------------------------------------------------ sort ----

constexpr int kSortThreads = 1024;

// Warps take runs of entries.  A warp counts its entries per expert and remembers for each entry
// how many of its expert came before it in the run; the runs' counts are then summed over the warps
// and the experts.
template <typename Index>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortByExpertCall c) {
  extern __shared__ uint32_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int E = c.num_experts;
  uint32_t* seen = smem;               // [warps][E]
  uint32_t* first = smem + warps * E;  // [E + 1]
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const Index* indices = static_cast<const Index*>(c.indices);
  const int n = c.num_tokens * c.topk;
  int live = n;
  if (c.bound_m != nullptr)
    live = static_cast<int>(min(*c.bound_m, static_cast<uint32_t>(c.num_tokens))) * c.topk;
  for (int i = tid; i < warps * E; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  const int per = (ceil_div(n, warps) + 31) & ~31;
  const int begin = min(warp * per, n), end = min(begin + per, n);
  uint32_t* mine = seen + warp * E;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const int i = i0 + lane;
    int e = E;  // none
    if (i < min(end, live)) {
      const Index v = indices[i];
      if (v < static_cast<Index>(E)) e = static_cast<int>(v);
    }
    const uint32_t same = __match_any_sync(kAll, e);
    const uint32_t before = __popc(same & ((1u << lane) - 1u));
    const uint32_t base = e < E ? mine[e] : 0u;
    __syncwarp();
    if (e < E && before == 0) mine[e] = base + __popc(same);
    __syncwarp();
    if (i < end) c.row_of[i] = e < E ? static_cast<int32_t>(base + before) : -1;
  }
  __syncthreads();
  for (int e = tid; e < E; e += blockDim.x) {
    uint32_t run = 0;
    for (int w = 0; w < warps; ++w) {
      const uint32_t v = seen[w * E + e];
      seen[w * E + e] = run;
      run += v;
    }
    first[e] = run;
    c.counts[e] = c.capacity > 0 ? min(static_cast<int>(run), c.capacity) : static_cast<int>(run);
  }
  __syncthreads();
  if (warp == 0) warp_exclusive_scan_smem(first, E, lane, true);
  __syncthreads();
  for (int e = tid; e <= E; e += blockDim.x)
    c.offsets[e] = c.capacity > 0 ? e * c.capacity : static_cast<int>(first[e]);
  for (int i = begin + lane; i < end; i += 32) {
    const int32_t local = c.row_of[i];  // (of this thread)
    if (local < 0) continue;
    const int e = static_cast<int>(indices[i]);
    const int pos = static_cast<int>(mine[e]) + local;
    if (c.capacity > 0) c.row_of[i] = pos < c.capacity ? e * c.capacity + pos : -1;
    else c.row_of[i] = static_cast<int>(first[e]) + pos;
  }
}

// --------------------------------------------------------------------- helpers ----

// A row that no entry of the routing has.
__device__ __forceinline__ bool is_rest(const ExpertRowsView& v, int64_t row) {
  if (v.capacity == 0) return row >= v.offsets[v.num_experts];
  const int64_t e = row / v.capacity;
  return e >= v.num_experts || row - e * v.capacity >= v.counts[e];
}

// Row of entry (t, k), or -1.
__device__ __forceinline__ int row_at(const ExpertRowsView& v, int64_t t, int k) {
  const int32_t r = v.row_of[t * v.topk + k];
  return static_cast<uint32_t>(r) < static_cast<uint64_t>(v.num_rows) ? r : -1;
}

template <typename T, int kVec>
struct alignas(sizeof(T) * kVec) Pack {
  T v[kVec];
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// --------------------------------------------------------------------- permute ----

// A warp per (token, piece of its columns); behind the tokens, a warp per (row, piece) of the rows
// to be cleared.
template <typename V>
__global__ void __launch_bounds__(kThreads) permute_kernel(const PermuteCall c) {
  constexpr int kBatch = 4;  // vectors of a lane in flight
  const ExpertRowsView& r = c.rows;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int lane = threadIdx.x & 31;
  const int vecs = static_cast<int>(c.row_bytes / static_cast<int64_t>(sizeof(V)));
  const int pieces = ceil_div(vecs, 32 * kBatch);
  const int64_t units = (r.num_tokens + (c.zero_rest ? r.num_rows : 0)) * static_cast<int64_t>(pieces);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); u < units;
       u += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t t = u / pieces;
    const int col = static_cast<int>(u - t * pieces) * 32 * kBatch + lane;
    V v[kBatch] = {};
    auto store = [&](int64_t row) {
      V* dst = reinterpret_cast<V*>(static_cast<uint8_t*>(c.out) + row * c.row_bytes);
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (col + 32 * b < vecs) dst[col + 32 * b] = v[b];
    };
    if (t >= r.num_tokens) {
      if (is_rest(r, t - r.num_tokens)) store(t - r.num_tokens);
      continue;
    }
    const V* src = reinterpret_cast<const V*>(static_cast<const uint8_t*>(c.x) + t * c.x_stride);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (col + 32 * b < vecs) v[b] = src[col + 32 * b];
    for (int k = 0; k < r.topk; ++k) {
      const int row = row_at(r, t, k);
      if (row >= 0) store(row);
    }
  }
}

// ------------------------------------------------------------------- unpermute ----

// A warp per (token, piece of 32 vectors).
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) unpermute_kernel(const UnpermuteCall c) {
  constexpr int kBatch = 4;  // rows whose vectors a lane has in flight
  using P = Pack<T, kVec>;
  const ExpertRowsView& r = c.rows;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int lane = threadIdx.x & 31;
  const int vecs = c.hidden / kVec;
  const int pieces = ceil_div(vecs, 32);
  int64_t tokens = r.num_tokens;
  if (c.bound_m != nullptr) tokens = min(tokens, static_cast<int64_t>(*c.bound_m));
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
       u < tokens * pieces; u += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t t = u / pieces;
    const int col = static_cast<int>(u - t * pieces) * 32 + lane;
    if (col >= vecs) continue;
    float sum[kVec] = {};
    for (int k0 = 0; k0 < r.topk; k0 += kBatch) {
      P v[kBatch];
      float w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int row = k0 + b < r.topk ? row_at(r, t, k0 + b) : -1;
        w[b] = row < 0 ? 0.0f : c.weights != nullptr ? c.weights[t * r.topk + k0 + b] : 1.0f;
        v[b] = P{};
        if (row >= 0)
          v[b] = reinterpret_cast<const P*>(static_cast<const T*>(c.y) +
                                            static_cast<int64_t>(row) * c.hidden)[col];
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum[j] = fmaf(w[b], to_float(v[b].v[j]), sum[j]);
    }
    P o;
#pragma unroll
    for (int j = 0; j < kVec; ++j) o.v[j] = from_float<T>(sum[j]);
    reinterpret_cast<P*>(static_cast<T*>(c.out) + t * c.out_stride)[col] = o;
  }
}

// A block per token; behind the tokens, a block per row to be cleared.
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) unpermute_backward_kernel(const UnpermuteBackwardCall c) {
  constexpr int kBatch = 4;
  using P = Pack<T, kVec>;
  __shared__ float part[kBatch][kWarps];
  const ExpertRowsView& r = c.rows;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vecs = c.hidden / kVec;
  auto row_ptr = [&](auto* base, int64_t row) { return base + row * c.hidden; };
  const int64_t blocks = r.num_tokens + (c.grad_y != nullptr ? r.num_rows : 0);
  for (int64_t t = blockIdx.x; t < blocks; t += gridDim.x) {
    if (t >= r.num_tokens) {
      const int64_t row = t - r.num_tokens;
      if (is_rest(r, row))
        for (int col = tid; col < vecs; col += kThreads)
          reinterpret_cast<P*>(row_ptr(static_cast<T*>(c.grad_y), row))[col] = P{};
      continue;
    }
    const P* grad = reinterpret_cast<const P*>(static_cast<const T*>(c.grad) + t * c.grad_stride);
    for (int k0 = 0; k0 < r.topk; k0 += kBatch) {
      int row[kBatch];
      float w[kBatch], dot[kBatch] = {};
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        row[b] = k0 + b < r.topk ? row_at(r, t, k0 + b) : -1;
        w[b] = k0 + b < r.topk ? c.weights[t * r.topk + k0 + b] : 0.0f;
      }
      for (int col = tid; col < vecs; col += kThreads) {
        const P g = grad[col];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          if (row[b] < 0) continue;
          if (c.grad_weights != nullptr) {
            const P y = reinterpret_cast<const P*>(row_ptr(static_cast<const T*>(c.y), row[b]))[col];
#pragma unroll
            for (int j = 0; j < kVec; ++j) dot[b] = fmaf(to_float(y.v[j]), to_float(g.v[j]), dot[b]);
          }
          if (c.grad_y != nullptr) {
            P o;
#pragma unroll
            for (int j = 0; j < kVec; ++j) o.v[j] = from_float<T>(w[b] * to_float(g.v[j]));
            reinterpret_cast<P*>(row_ptr(static_cast<T*>(c.grad_y), row[b]))[col] = o;
          }
        }
      }
      if (c.grad_weights == nullptr) continue;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        float s = dot[b];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        if (lane == 0) part[b][warp] = s;
      }
      __syncthreads();
      if (tid < kBatch && k0 + tid < r.topk) {
        float s = 0.0f;
        for (int w2 = 0; w2 < kWarps; ++w2) s += part[tid][w2];
        c.grad_weights[t * r.topk + k0 + tid] = s;
      }
      __syncthreads();
    }
  }
}

// -------------------------------------------------------------------- quantise ----

// Bits of |v| as an integer: ordered like |v|, infinities above all numbers and NaN above those.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// The largest magnitude of a row as the scale's numerator; a row of smaller values than 1e-30 keeps
// a scale whose inverse is finite.  An infinity or a NaN in the row makes the scale one, and what
// is computed with the row non-finite.
__device__ __forceinline__ float row_amax(uint32_t bits) {
  return __uint_as_float(max(bits, __float_as_uint(1e-30f)));
}

__device__ __forceinline__ int8_t quantize(float v, float inv) {
  return static_cast<int8_t>(max(min(__float2int_rn(v * inv), 127), -127));
}

// A block per token (or row of x); behind them, a block per row to be cleared.
template <typename T, int kVec>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeRowsCall c,
                                                            const ExpertRowsView r) {
  using P = Pack<T, kVec>;
  using Q = Pack<int8_t, kVec>;
  __shared__ uint32_t part[kWarps];
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int vecs = c.hidden / kVec;
  const bool permuted = r.row_of != nullptr;
  const int64_t sources = permuted ? r.num_tokens : c.num_rows;
  const int64_t blocks = sources + (c.zero_rest ? r.num_rows : 0);
  for (int64_t t = blockIdx.x; t < blocks; t += gridDim.x) {
    if (t >= sources) {
      const int64_t row = t - sources;
      if (!is_rest(r, row)) continue;
      for (int col = tid; col < vecs; col += kThreads)
        reinterpret_cast<Q*>(c.q + row * c.hidden)[col] = Q{};
      if (tid == 0) c.scale[row] = 0.0f;
      continue;
    }
    if (c.counts != nullptr) {
      const int64_t plane = t / c.plane_rows;
      if (t - plane * c.plane_rows >= c.counts[plane]) continue;
    }
    const P* x = reinterpret_cast<const P*>(static_cast<const T*>(c.x) + t * c.x_stride);
    uint32_t bits = 0;
    for (int col = tid; col < vecs; col += kThreads) {
      const P v = x[col];
#pragma unroll
      for (int j = 0; j < kVec; ++j) bits = max(bits, magnitude(to_float(v.v[j])));
    }
    bits = __reduce_max_sync(kAll, bits);
    if (lane == 0) part[warp] = bits;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) bits = max(bits, part[w]);
    __syncthreads();
    const float amax = row_amax(bits);
    const float inv = 127.0f / amax, scale = amax / 127.0f;
    const int targets = permuted ? r.topk : 1;
    for (int col = tid; col < vecs; col += kThreads) {
      const P v = x[col];
      Q o;
#pragma unroll
      for (int j = 0; j < kVec; ++j) o.v[j] = quantize(to_float(v.v[j]), inv);
      for (int k = 0; k < targets; ++k) {
        const int64_t row = permuted ? row_at(r, t, k) : t;
        if (row >= 0) reinterpret_cast<Q*>(c.q + row * c.hidden)[col] = o;
      }
    }
    for (int k = tid; k < targets; k += kThreads) {
      const int64_t row = permuted ? row_at(r, t, k) : t;
      if (row >= 0) c.scale[row] = scale;
    }
  }
}

// ---------------------------------------------------------------------- launch ----

// Largest power of two, at most `most`, that divides every address and length given.
int alignment(int most, std::initializer_list<uint64_t> values) {
  uint64_t all = static_cast<uint64_t>(most);
  for (uint64_t v : values) all |= v;
  return static_cast<int>(all & (~all + 1));
}

uint64_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Enough blocks to fill every SM with 2048 threads; they loop over the rest.
unsigned blocks_for(int64_t wanted) {
  return static_cast<unsigned>(
      std::max<int64_t>(1, std::min<int64_t>(wanted, static_cast<int64_t>(get_sm_count()) * 8)));
}

template <typename Call>
void launch(void (*kernel)(const Call), const Call& c, int64_t blocks, cudaStream_t stream) {
  void* params[] = {const_cast<Call*>(&c)};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(blocks_for(blocks)),
                                   dim3(kThreads), params, 0, stream));
}

// Calls fn(T{}, integral_constant<kVec>) for the type and for vectors of `bytes` bytes.
template <typename T, typename Fn>
void with_vector(int bytes, Fn&& fn) {
  constexpr int kFull = 16 / static_cast<int>(sizeof(T));
  if (bytes == 16) return fn(T{}, std::integral_constant<int, kFull>{});
  if (bytes == 8) return fn(T{}, std::integral_constant<int, kFull / 2>{});
  if (bytes == 4) return fn(T{}, std::integral_constant<int, kFull / 4>{});
  if constexpr (sizeof(T) == 2) return fn(T{}, std::integral_constant<int, 1>{});
}

template <typename Fn>
void with_type(FloatType type, int bytes, Fn&& fn) {
  if (type == FloatType::kBFloat16) with_vector<__nv_bfloat16>(bytes, fn);
  else if (type == FloatType::kHalf) with_vector<__half>(bytes, fn);
  else with_vector<float>(bytes, fn);
}

int size_of(FloatType t) { return t == FloatType::kFloat ? 4 : 2; }

}  // namespace

void launch_sort_by_expert(const SortByExpertCall& c, cudaStream_t stream) {
  PPLX_CHECK(c.num_experts > 0 && c.num_experts <= kMaxSortExperts, "num_experts out of range");
  auto* kernel = c.wide_indices ? sort_kernel<uint64_t> : sort_kernel<uint32_t>;
  const int warps = kSortThreads / 32;
  const size_t smem = sizeof(uint32_t) * (static_cast<size_t>(warps + 1) * c.num_experts + 1);
  CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(smem)));
  void* params[] = {const_cast<SortByExpertCall*>(&c)};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(1),
                                   dim3(kSortThreads), params, smem, stream));
}

void launch_permute_tokens(const PermuteCall& c, cudaStream_t stream) {
  const int64_t items = c.rows.num_tokens + (c.zero_rest ? c.rows.num_rows : 0);
  if (items == 0 || c.row_bytes == 0) return;
  const int vec = alignment(16, {address(c.x), address(c.out), static_cast<uint64_t>(c.row_bytes),
                                 static_cast<uint64_t>(c.x_stride)});
  const int64_t pieces = ceil_div<int64_t>(c.row_bytes / vec, 128);
  const int64_t blocks = ceil_div<int64_t>(items * pieces, kWarps);
  switch (vec) {
    case 16: return launch(permute_kernel<int4>, c, blocks, stream);
    case 8: return launch(permute_kernel<int2>, c, blocks, stream);
    case 4: return launch(permute_kernel<int>, c, blocks, stream);
    case 2: return launch(permute_kernel<short>, c, blocks, stream);
    default: return launch(permute_kernel<char>, c, blocks, stream);
  }
}

void launch_unpermute_tokens(const UnpermuteCall& c, cudaStream_t stream) {
  if (c.rows.num_tokens == 0 || c.hidden == 0) return;
  const uint64_t size = size_of(c.type);
  const int vec = alignment(16, {address(c.y), address(c.out), c.hidden * size, c.out_stride * size});
  with_type(c.type, vec, [&](auto t, auto v) {
    const int64_t pieces = ceil_div<int64_t>(c.hidden / v.value, 32);
    launch(unpermute_kernel<decltype(t), v.value>, c,
           ceil_div<int64_t>(c.rows.num_tokens * pieces, kWarps), stream);
  });
}

void launch_unpermute_backward(const UnpermuteBackwardCall& c, cudaStream_t stream) {
  const int64_t blocks = c.rows.num_tokens + (c.grad_y != nullptr ? c.rows.num_rows : 0);
  if (blocks == 0) return;
  const uint64_t size = size_of(c.type);
  const int vec = alignment(16, {address(c.y), address(c.grad), address(c.grad_y), c.hidden * size,
                                 c.grad_stride * size});
  with_type(c.type, vec, [&](auto t, auto v) {
    launch(unpermute_backward_kernel<decltype(t), v.value>, c, blocks, stream);
  });
}

void launch_quantize_rows(const QuantizeRowsCall& c, cudaStream_t stream) {
  ExpertRowsView r{};
  if (c.rows != nullptr) r = *c.rows;
  const int64_t blocks = (c.rows != nullptr ? r.num_tokens : c.num_rows) +
                         (c.zero_rest ? r.num_rows : 0);
  if (blocks == 0) return;
  const uint64_t size = size_of(c.type);
  // A vector of x of `vec` bytes becomes one of vec / size bytes of q.
  const int vec = std::min<int>(
      alignment(16, {address(c.x), c.hidden * size, c.x_stride * size}),
      alignment(16, {address(c.q), static_cast<uint64_t>(c.hidden)}) * static_cast<int>(size));
  with_type(c.type, vec, [&](auto t, auto v) {
    auto* kernel = quantize_kernel<decltype(t), v.value>;
    void* params[] = {const_cast<QuantizeRowsCall*>(&c), &r};
    CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(blocks_for(blocks)),
                                     dim3(kThreads), params, 0, stream));
  });
}

}  // namespace pplx
