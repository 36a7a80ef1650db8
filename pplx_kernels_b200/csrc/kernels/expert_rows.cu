// Tokens sorted by expert and back on one GPU, with the gradients, and rows quantised to 8-bit
// integers.  All of it is bound by memory: the sort reads and writes a few bytes per entry of the
// routing, the others read each token (or row) once and write each row (or token) once.
//
// Every kernel goes token by token: the rows of a token are found through row_of, so a token is
// read once for all its rows, and the order in which a token's rows are summed is that of its
// entries, whatever the experts are.  No atomics: the same call gives the same bits.
#include "expert_rows.h"

#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../core/device_utils.cuh"
#include "../core/ptx.cuh"
#include "../core/tcgen05.cuh"
#include "../core/utils.h"

namespace pplx {
namespace {

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kMaxSortExperts = 1024;  // (their numbers and one more take 11 bits)

// ------------------------------------------------------------------------ sort ----

constexpr int kSortThreads = 512;

__device__ __forceinline__ uint32_t ld_cluster(const uint32_t* p, uint32_t cta) {
  uint32_t addr, v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(tc::smem_u32(p)), "r"(cta));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

// Warps take runs of entries.  A warp counts its entries per expert and remembers for each entry
// how many of its expert came before it in the run; the runs' counts are then summed over the warps,
// the blocks (one, or a cluster whose blocks read each other's sums) and the experts.  Bound by
// latency: of the entries' loads (up to eight of a lane at once), of the votes that find a warp's entries
// of one expert, of the barriers.
template <typename Index>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const SortByExpertCall c) {
  constexpr int kHeld = 8;
  extern __shared__ uint32_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  const int blocks = gridDim.x;
  const int E = c.num_experts;
  uint32_t* seen = smem;               // [warps][E]
  uint32_t* mine_all = smem + warps * E;  // [E] entries of this block
  uint32_t* before_of = mine_all + E;  // [E] entries of the blocks before this one
  uint32_t* first = before_of + E;     // [E + 1]
  for (int i = tid; i < warps * E; i += blockDim.x) seen[i] = 0;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const Index* indices = static_cast<const Index*>(c.indices);
  const int n = c.num_tokens * c.topk;
  int live = n;
  if (c.bound_m != nullptr)
    live = static_cast<int>(min(*c.bound_m, static_cast<uint32_t>(c.num_tokens))) * c.topk;
  __syncthreads();
  const int runs = warps * blocks;
  const int per = (ceil_div(n, runs) + 31) & ~31;
  const int run = blockIdx.x * warps + warp;
  const int begin = static_cast<int>(min(static_cast<int64_t>(run) * per, static_cast<int64_t>(n)));
  const int end = min(begin + per, n);
  uint32_t* mine = seen + warp * E;
  const int bits = 32 - __clz(E);  // of the numbers 0 .. E
  auto load_index = [&](int i) { return i < min(end, live) ? indices[i] : static_cast<Index>(E); };
  auto expert_of = [&](Index v) { return v < static_cast<Index>(E) ? static_cast<int>(v) : E; };  // E: none
  // How many entries of the run came before this lane's of the same expert.
  auto count = [&](int e) {
    // (A vote per bit of the expert's number: 32768 entries 7.0 us, with match.any 7.6.)
    uint32_t same = kAll;
#pragma unroll
    for (int b = 0; b < 11; ++b) {
      if (b >= bits) break;
      const uint32_t set = __ballot_sync(kAll, (e >> b) & 1);
      same &= (e >> b) & 1 ? set : ~set;
    }
    const uint32_t before = __popc(same & ((1u << lane) - 1u));
    const uint32_t base = e < E ? mine[e] : 0u;
    __syncwarp();
    if (e < E && before == 0) mine[e] = base + __popc(same);
    __syncwarp();
    return static_cast<int32_t>(base + before);
  };
  // Up to kHeld entries of a lane stay in registers; longer runs keep the numbers in row_of.
  const bool held = per <= 32 * kHeld;
  int expert[kHeld], local[kHeld];
  if (held) {
    Index v[kHeld];
#pragma unroll
    for (int s = 0; s < kHeld; ++s) v[s] = load_index(begin + 32 * s + lane);  // (all on their way)
#pragma unroll
    for (int s = 0; s < kHeld; ++s) {
      if (32 * s >= per) break;
      expert[s] = expert_of(v[s]);
      local[s] = count(expert[s]);
    }
  } else {
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int e = expert_of(load_index(i0 + lane));
      const int32_t n_before = count(e);
      if (i0 + lane < end) c.row_of[i0 + lane] = e < E ? n_before : -1;
    }
  }
  __syncthreads();
  for (int e = tid; e < E; e += blockDim.x) {
    uint32_t sum = 0;
    for (int w = 0; w < warps; ++w) {
      const uint32_t v = seen[w * E + e];
      seen[w * E + e] = sum;
      sum += v;
    }
    mine_all[e] = sum;
    first[e] = sum;
  }
  if (blocks == 1)
    for (int e = tid; e < E; e += blockDim.x) before_of[e] = 0;
  if (blocks > 1) {
    tc::cluster_sync();
    for (int e = tid; e < E; e += blockDim.x) {
      uint32_t sum = 0, before = 0;
      for (int b0 = 0; b0 < blocks; b0 += 8) {  // (8 or 16 blocks)
        uint32_t v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = ld_cluster(&mine_all[e], b0 + j);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (b0 + j == static_cast<int>(blockIdx.x)) before = sum;
          sum += v[j];
        }
      }
      first[e] = sum;
      before_of[e] = before;
    }
    tc::cluster_sync();  // (no block leaves while others read its sums)
  } else {
    __syncthreads();
  }
  if (blockIdx.x == 0)
    for (int e = tid; e < E; e += blockDim.x)
      c.counts[e] = c.capacity > 0 ? min(static_cast<int>(first[e]), c.capacity) : static_cast<int>(first[e]);
  __syncthreads();
  if (warp == 0) warp_exclusive_scan_smem(first, E, lane, true);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= E; e += blockDim.x)
      c.offsets[e] = c.capacity > 0 ? e * c.capacity : static_cast<int>(first[e]);
  auto row_of = [&](int e, int32_t n_before) -> int32_t {
    const int pos = static_cast<int>(mine[e] + before_of[e]) + n_before;
    if (c.capacity > 0) return pos < c.capacity ? e * c.capacity + pos : -1;
    return static_cast<int>(first[e]) + pos;
  };
  if (held) {
#pragma unroll
    for (int s = 0; s < kHeld; ++s) {
      const int i = begin + 32 * s + lane;
      if (i < end) c.row_of[i] = expert[s] < E ? row_of(expert[s], local[s]) : -1;
    }
  } else {
    for (int i = begin + lane; i < end; i += 32) {
      const int32_t n_before = c.row_of[i];  // (written by this thread)
      if (n_before >= 0) c.row_of[i] = row_of(static_cast<int>(indices[i]), n_before);
    }
  }
}

// --------------------------------------------------------------------- helpers ----

// Rows that no entry of the routing has: candidates (all rows where there is a capacity, otherwise
// those behind the last expert's), and the row of candidate i, or -1 if an entry has it.
__device__ __forceinline__ int64_t rest_candidates(const ExpertRowsView& v) {
  if (v.capacity > 0) return v.num_rows;
  return v.num_rows - min(max(static_cast<int64_t>(v.offsets[v.num_experts]), int64_t{0}), v.num_rows);
}
__device__ __forceinline__ int64_t rest_row(const ExpertRowsView& v, int64_t candidates, int64_t i) {
  if (v.capacity == 0) return v.num_rows - candidates + i;
  const int64_t e = i / v.capacity;
  return i - e * v.capacity >= v.counts[e] ? i : -1;
}

// Row of entry (t, k), or -1.
__device__ __forceinline__ int row_at(const ExpertRowsView& v, int64_t t, int k) {
  const int32_t r = v.row_of[t * v.topk + k];
  return static_cast<uint32_t>(r) < static_cast<uint64_t>(v.num_rows) ? r : -1;
}

// kVec elements of a row as the words that memory moves: registers hold 16-bit values in pairs.
template <int kBytes>
struct Words {
  using type = uint32_t;
};
template <>
struct Words<16> {
  using type = uint4;
};
template <>
struct Words<8> {
  using type = uint2;
};
template <>
struct Words<2> {
  using type = uint16_t;
};
template <>
struct Words<1> {
  using type = uint8_t;
};

template <typename T, int kVec>
struct Vec {
  static constexpr int kBytes = kVec * static_cast<int>(sizeof(T));
  static constexpr int kWords = (kBytes + 3) / 4;
  using Memory = typename Words<kBytes>::type;
  uint32_t w[kWords];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void set(const Memory& m) {
    if constexpr (kBytes == 16) w[0] = m.x, w[1] = m.y, w[2] = m.z, w[3] = m.w;
    else if constexpr (kBytes == 8) w[0] = m.x, w[1] = m.y;
    else w[0] = m;
  }
  __device__ __forceinline__ void load(const void* row, int col) {
    set(reinterpret_cast<const Memory*>(row)[col]);
  }
  // What is read once leaves no copy in L1.
  __device__ __forceinline__ void load_once(const void* row, int col) {
    const Memory* p = reinterpret_cast<const Memory*>(row) + col;
    if constexpr (kBytes == 16) {
      const int4 v = ptx::ld_nc_v4(p);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
      set(*p);
    }
  }
  __device__ __forceinline__ void store(void* row, int col, bool streaming = false) const {
    Memory m;
    if constexpr (kBytes == 16) m = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (kBytes == 8) m = make_uint2(w[0], w[1]);
    else m = static_cast<Memory>(w[0]);
    Memory* p = reinterpret_cast<Memory*>(row) + col;
    if (streaming) __stcs(p, m);
    else *p = m;
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
    else if constexpr (std::is_same_v<T, __half>)
      return __half2float(__ushort_as_half(static_cast<uint16_t>(j & 1 ? w[j >> 1] >> 16 : w[j >> 1])));
    else return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
  }
  __device__ __forceinline__ void put(const float (&v)[kVec]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) w[j] = __float_as_uint(v[j]);
    } else if constexpr (kVec == 1) {
      if constexpr (std::is_same_v<T, __half>) w[0] = __half_as_ushort(__float2half_rn(v[0]));
      else w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
    } else {
#pragma unroll
      for (int j = 0; j < kVec; j += 2) {
        if constexpr (std::is_same_v<T, __half>) {
          const __half2 h = __floats2half2_rn(v[j], v[j + 1]);
          w[j >> 1] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(v[j], v[j + 1]);
          w[j >> 1] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
  }
};

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
  const int64_t rest = c.zero_rest ? rest_candidates(r) : 0;
  const int64_t units = (r.num_tokens + rest) * static_cast<int64_t>(pieces);
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); u < units;
       u += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t t = u / pieces;
    const int col = static_cast<int>(u - t * pieces) * 32 * kBatch + lane;
    V v[kBatch] = {};
    auto store = [&](int64_t row) {
      V* dst = reinterpret_cast<V*>(static_cast<uint8_t*>(c.out) + row * c.row_bytes);
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (col + 32 * b < vecs) {
          if (c.streaming) __stcs(dst + col + 32 * b, v[b]);
          else dst[col + 32 * b] = v[b];
        }
    };
    if (t >= r.num_tokens) {
      const int64_t row = rest_row(r, rest, t - r.num_tokens);
      if (row >= 0) store(row);
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

// A warp per (token, piece of its columns); a lane has kCols columns of kRows rows in flight.  4095
// tokens of 8 rows of 7168 bf16: 81 us, 6.5 TB/s.
template <typename T, int kVec, int kRows, int kCols>
__global__ void __launch_bounds__(kThreads) unpermute_kernel(const UnpermuteCall c) {
  using V = Vec<T, kVec>;
  const ExpertRowsView& r = c.rows;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int lane = threadIdx.x & 31;
  const int vecs = c.hidden / kVec;
  const int pieces = ceil_div(vecs, 32 * kCols);
  int64_t tokens = r.num_tokens;
  if (c.bound_m != nullptr) tokens = min(tokens, static_cast<int64_t>(*c.bound_m));
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
       u < tokens * pieces; u += static_cast<int64_t>(gridDim.x) * kWarps) {
    const int64_t t = u / pieces;
    const int col = static_cast<int>(u - t * pieces) * 32 * kCols + lane;
    float sum[kCols][kVec] = {};
    for (int k0 = 0; k0 < r.topk; k0 += kRows) {
      // Lane k holds entry k0 + k.
      int my_row = -1;
      float my_w = 0.0f;
      if (lane < kRows && k0 + lane < r.topk) {
        my_row = row_at(r, t, k0 + lane);
        my_w = my_row < 0 ? 0.0f : c.weights != nullptr ? c.weights[t * r.topk + k0 + lane] : 1.0f;
      }
      V v[kRows][kCols];
#pragma unroll
      for (int b = 0; b < kRows; ++b) {
        const int row = __shfl_sync(kAll, my_row, b);
        const T* y = static_cast<const T*>(c.y) + static_cast<int64_t>(row) * c.hidden;
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
          v[b][i].clear();
          if (row >= 0 && col + 32 * i < vecs) v[b][i].load_once(y, col + 32 * i);
        }
      }
#pragma unroll
      for (int b = 0; b < kRows; ++b) {
        const float w = __shfl_sync(kAll, my_w, b);
#pragma unroll
        for (int i = 0; i < kCols; ++i)
#pragma unroll
          for (int j = 0; j < kVec; ++j) sum[i][j] = fmaf(w, v[b][i].get(j), sum[i][j]);
      }
    }
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      V o;
      o.put(sum[i]);
      if (col + 32 * i < vecs)
        o.store(static_cast<T*>(c.out) + t * c.out_stride, col + 32 * i, c.streaming);
    }
  }
}

// A block per token; behind the tokens, a block per row to be cleared.  The gradient of a weight is a
// sum over thousands of products that largely cancel: those of a vector are summed in 32 bits, the
// vectors in 64.
template <typename T, int kVec, int kRows, int kCols>
__global__ void __launch_bounds__(kThreads) unpermute_backward_kernel(const UnpermuteBackwardCall c) {
  using V = Vec<T, kVec>;
  __shared__ double part[kRows][kWarps];
  const ExpertRowsView& r = c.rows;
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int tid = threadIdx.x, threads = blockDim.x, warp = tid >> 5, lane = tid & 31;
  const int vecs = c.hidden / kVec;
  auto row_ptr = [&](auto* base, int64_t row) { return base + row * c.hidden; };
  const int64_t rest = c.grad_y != nullptr ? rest_candidates(r) : 0;
  const int64_t blocks = r.num_tokens + rest;
  for (int64_t t = blockIdx.x; t < blocks; t += gridDim.x) {
    if (t >= r.num_tokens) {
      const int64_t row = rest_row(r, rest, t - r.num_tokens);
      V zero;
      zero.clear();
      if (row >= 0)
        for (int col = tid; col < vecs; col += threads)
          zero.store(row_ptr(static_cast<T*>(c.grad_y), row), col);
      continue;
    }
    const T* grad = static_cast<const T*>(c.grad) + t * c.grad_stride;
    for (int k0 = 0; k0 < r.topk; k0 += kRows) {
      // Lane k holds entry k0 + k.
      int my_row = -1;
      float my_w = 0.0f;
      if (lane < kRows && k0 + lane < r.topk) {
        my_row = row_at(r, t, k0 + lane);
        my_w = c.weights[t * r.topk + k0 + lane];
      }
      double dot[kRows] = {};
      for (int first = 0; first < vecs; first += threads * kCols) {  // (the same for all threads)
        const int col0 = first + tid;
        V g[kCols], y[kRows][kCols];
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
          g[i].clear();
          if (col0 + i * threads < vecs) g[i].load(grad, col0 + i * threads);
        }
        if (c.grad_weights != nullptr) {
#pragma unroll
          for (int b = 0; b < kRows; ++b) {
            const int row = __shfl_sync(kAll, my_row, b);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              const int col = col0 + i * threads;
              y[b][i].clear();
              if (row >= 0 && col < vecs) y[b][i].load_once(row_ptr(static_cast<const T*>(c.y), row), col);
            }
          }
        }
        if (c.grad_y != nullptr) {
#pragma unroll
          for (int b = 0; b < kRows; ++b) {
            const int row = __shfl_sync(kAll, my_row, b);
            const float w = __shfl_sync(kAll, my_w, b);
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              const int col = col0 + i * threads;
              float v[kVec];
#pragma unroll
              for (int j = 0; j < kVec; ++j) v[j] = w * g[i].get(j);
              V o;
              o.put(v);
              if (row >= 0 && col < vecs) o.store(row_ptr(static_cast<T*>(c.grad_y), row), col);
            }
          }
        }
        if (c.grad_weights != nullptr) {
#pragma unroll
          for (int b = 0; b < kRows; ++b)
#pragma unroll
            for (int i = 0; i < kCols; ++i) {
              float sum = 0.0f;
#pragma unroll
              for (int j = 0; j < kVec; ++j) sum = fmaf(y[b][i].get(j), g[i].get(j), sum);
              dot[b] += static_cast<double>(sum);
            }
        }
      }
      if (c.grad_weights == nullptr) continue;
#pragma unroll
      for (int b = 0; b < kRows; ++b) {
        double s = dot[b];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kAll, s, o);
        if (lane == 0) part[b][warp] = s;
      }
      __syncthreads();
      if (tid < kRows && k0 + tid < r.topk) {
        double s = 0.0;
        for (int w2 = 0; w2 < threads / 32; ++w2) s += part[tid][w2];
        // (Without a row it is zero whatever the gradient is: zeros times infinity are not.  Lane tid of the
        // first warp holds the row.)
        c.grad_weights[t * r.topk + k0 + tid] = my_row >= 0 ? static_cast<float>(s) : 0.0f;
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

// The row's factor by its rounded reciprocal and its scale by the rounded 1/127: products take the place
// of quotients, as in torch's `127.0 / a` and `a / 127.0`.  Each is within 2 roundings of the quotient
// (the reciprocal of a > 8.5e37 is subnormal: 2^-22 of it at most), and decides only values that lie next to
// the border of two integers.
__device__ __forceinline__ float row_factor(float amax) { return __fmul_rn(127.0f, __frcp_rn(amax)); }
__device__ __forceinline__ float row_scale(float amax) { return __fmul_rn(amax, 1.0f / 127.0f); }

// rint(v * inv) of four values, |v * inv| <= 127.0001, as bytes: adding 1.5 * 2^23 rounds to whole
// numbers, which are then the low bits.  (The product is rounded before: no fused add.)
__device__ __forceinline__ uint32_t quantize(float a, float b, float c, float d, float inv) {
  auto whole = [&](float v) { return __float_as_uint(__fadd_rn(__fmul_rn(v, inv), 12582912.0f)); };
  return __byte_perm(__byte_perm(whole(a), whole(b), 0x0040), __byte_perm(whole(c), whole(d), 0x0040),
                     0x5410);
}

// A team of threads per token (or row of x): a warp (kWarpTeam), or the block; behind them, a team
// per row to be cleared.  The first kHeld vectors of a thread stay in registers between the search
// for the largest value and the rounding; longer rows are read again for the rest.
template <typename T, int kVec, int kHeld, bool kWarpTeam, bool kPermuted>
__global__ void __launch_bounds__(kThreads, kHeld == 4 ? 6 : 3)
    quantize_kernel(const QuantizeRowsCall c, const ExpertRowsView r) {
  using V = Vec<T, kVec>;
  using Q = Vec<int8_t, kVec>;
  __shared__ uint32_t part[2][kWarps];
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tid = kWarpTeam ? lane : threadIdx.x, threads = kWarpTeam ? 32 : blockDim.x;
  const int teams = kWarpTeam ? blockDim.x >> 5 : 1;
  const int vecs = c.hidden / kVec;
  const int64_t sources = kPermuted ? r.num_tokens : c.num_rows;
  const int64_t rest = c.zero_rest ? rest_candidates(r) : 0;
  const int64_t items = sources + rest;
  int turn = 0;
  for (int64_t t = static_cast<int64_t>(blockIdx.x) * teams + (kWarpTeam ? warp : 0); t < items;
       t += static_cast<int64_t>(gridDim.x) * teams) {
    if (t >= sources) {
      const int64_t row = rest_row(r, rest, t - sources);
      if (row < 0) continue;
      Q zero;
      zero.clear();
      for (int col = tid; col < vecs; col += threads) zero.store(c.q + row * c.hidden, col);
      if (tid == 0) c.scale[row] = 0.0f;
      continue;
    }
    if (!kPermuted && c.counts != nullptr) {
      const int64_t plane = t / c.plane_rows;
      if (t - plane * c.plane_rows >= c.counts[plane]) continue;
    }
    const T* x = static_cast<const T*>(c.x) + t * c.x_stride;
    V held[kHeld];
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int col = tid + h * threads;
      held[h].clear();
      if (col < vecs) held[h].load_once(x, col);
    }
    int my_row = -1;  // lane k holds that of entry k
    if (kPermuted && lane < r.topk) my_row = row_at(r, t, lane);
    uint32_t bits = 0;
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
#pragma unroll
      for (int j = 0; j < kVec; ++j) bits = max(bits, magnitude(held[h].get(j)));
#pragma unroll 1
    for (int col = tid + kHeld * threads; col < vecs; col += threads) {
      V v;
      v.load(x, col);
#pragma unroll
      for (int j = 0; j < kVec; ++j) bits = max(bits, magnitude(v.get(j)));
    }
    bits = __reduce_max_sync(kAll, bits);
    if constexpr (!kWarpTeam) {
      if (lane == 0) part[turn][warp] = bits;
      __syncthreads();
      bits = __reduce_max_sync(kAll, lane < threads / 32 ? part[turn][lane] : 0u);
      turn ^= 1;  // (the next row's maxima go elsewhere, so one barrier is enough)
    }
    const float amax = row_amax(bits);
    const float inv = row_factor(amax), scale = row_scale(amax);
    // A row with an infinity or a NaN is zero throughout.
    const uint32_t keep = amax < __uint_as_float(0x7f800000u) ? 0xffffffffu : 0u;
    auto rounded = [&](const V& v) {
      Q o;
#pragma unroll
      for (int j = 0; j < kVec; j += 4)
        o.w[j >> 2] = keep & quantize(v.get(j), v.get(j + 1), kVec > 2 ? v.get(min(j + 2, kVec - 1)) : 0.0f,
                                      kVec > 2 ? v.get(min(j + 3, kVec - 1)) : 0.0f, inv);
      return o;
    };
    const int targets = kPermuted ? r.topk : 1;
    auto row_to = [&](int k) -> int64_t {
      if constexpr (!kPermuted) return t;
      return k < 32 ? __shfl_sync(kAll, my_row, k) : row_at(r, t, k);
    };
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const int col = tid + h * threads;
      const Q q = rounded(held[h]);
#pragma unroll 1
      for (int k = 0; k < targets; ++k) {
        const int64_t row = row_to(k);
        if (row >= 0 && col < vecs) q.store(c.q + row * c.hidden, col, c.streaming);
      }
    }
#pragma unroll 1
    for (int col0 = kHeld * threads; col0 < vecs; col0 += threads) {
      const int col = col0 + tid;
      V v;
      v.clear();
      if (col < vecs) v.load(x, col);
      const Q q = rounded(v);
#pragma unroll 1
      for (int k = 0; k < targets; ++k) {
        const int64_t row = row_to(k);
        if (row >= 0 && col < vecs) q.store(c.q + row * c.hidden, col, c.streaming);
      }
    }
    for (int k = 0; k < targets; ++k) {
      const int64_t row = row_to(k);
      if (row >= 0 && tid == 0) c.scale[row] = scale;
    }
  }
}

// The same for rows that are not vectors of four: a block per token (or row of x), four values per
// thread and turn, read one by one and (after the search for the largest) from the caches.  A row of q
// may begin at any byte: a thread stores the aligned word that its values and those of the lane below
// make up, and the ends of the row one byte at a time.
template <typename T, bool kPermuted, int kBlock>
__global__ void __launch_bounds__(kBlock) quantize_ragged_kernel(const QuantizeRowsCall c,
                                                                 const ExpertRowsView r) {
  using V = Vec<T, 1>;
  __shared__ uint32_t part[2][kBlock / 32];
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int64_t sources = kPermuted ? r.num_tokens : c.num_rows;
  const int64_t rest = c.zero_rest ? rest_candidates(r) : 0;
  int turn = 0;
  for (int64_t t = blockIdx.x; t < sources + rest; t += gridDim.x) {
    if (t >= sources) {
      const int64_t row = rest_row(r, rest, t - sources);
      if (row < 0) continue;
      for (int col = tid; col < c.hidden; col += kBlock) c.q[row * c.hidden + col] = 0;
      if (tid == 0) c.scale[row] = 0.0f;
      continue;
    }
    if (!kPermuted && c.counts != nullptr) {
      const int64_t plane = t / c.plane_rows;
      if (t - plane * c.plane_rows >= c.counts[plane]) continue;
    }
    const T* x = static_cast<const T*>(c.x) + t * c.x_stride;
    auto value = [&](int col) {
      V v;
      v.clear();
      if (col < c.hidden) v.load(x, col);
      return v.get(0);
    };
    uint32_t bits = 0;
    for (int col = tid; col < c.hidden; col += 4 * kBlock)
#pragma unroll
      for (int i = 0; i < 4; ++i) bits = max(bits, magnitude(value(col + i * kBlock)));
    bits = __reduce_max_sync(kAll, bits);
    if (lane == 0) part[turn][warp] = bits;
    __syncthreads();
    bits = __reduce_max_sync(kAll, lane < kBlock / 32 ? part[turn][lane] : 0u);
    turn ^= 1;  // (the next row's maxima go elsewhere, so one barrier is enough)
    const float amax = row_amax(bits);
    const float inv = row_factor(amax), scale = row_scale(amax);
    const uint32_t keep = amax < __uint_as_float(0x7f800000u) ? 0xffffffffu : 0u;
    const int targets = kPermuted ? r.topk : 1;
    int my_row = -1;  // lane k holds that of entry k
    if (kPermuted && lane < r.topk) my_row = row_at(r, t, lane);
    // A warp makes 32 words and stores 31: the lowest lane only hands its values up.  (The last word of
    // a row that begins inside one is behind the row's last values.)
    for (int turn_of = warp; turn_of * 31 * 4 < c.hidden + 4; turn_of += kBlock / 32) {
      const int col = (turn_of * 31 + lane - 1) * 4;
      uint32_t word = 0;
      if (col >= 0) word = keep & quantize(value(col), value(col + 1), value(col + 2), value(col + 3), inv);
      const uint32_t below = __shfl_up_sync(kAll, word, 1);
      for (int k = 0; k < targets; ++k) {
        int64_t row = t;
        if constexpr (kPermuted) row = k < 32 ? __shfl_sync(kAll, my_row, k) : row_at(r, t, k);
        if (row < 0 || lane == 0) continue;
        int8_t* q = c.q + row * c.hidden;
        const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(q) & 3u);
        const uint32_t out = __funnelshift_l(below, word, 8 * shift);
        const int at = col - shift;  // of the first byte of `out`
        if (at >= 0 && at + 4 <= c.hidden) {
          *reinterpret_cast<uint32_t*>(q + at) = out;
        } else {
#pragma unroll 1
          for (int j = max(0, -at); j < min(4, c.hidden - at); ++j)
            q[at + j] = static_cast<int8_t>(out >> (8 * j));
        }
      }
    }
    for (int k = tid; k < targets; k += kBlock) {
      const int64_t row = kPermuted ? row_at(r, t, k) : t;
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

// Twice the blocks that fill every SM with 2048 threads; they loop over the rest.  (Once or four
// times as many: 4096 x 28672 floats quantised in 103, 90, 90 us for once, twice, four times; copies of
// 4096 tokens of 2048 25.0, 23.2, 24.5 us; the gradients of 4095 x 8 rows of 7168 170, 165, 164 us; their
// sum 90, 91, 92 us.  Once for the smallest blocks, whose launches show.)
unsigned blocks_for(int64_t wanted, int threads) {
  const int64_t most = static_cast<int64_t>(get_sm_count()) * std::min(32, 2048 / threads) *
                       (threads < 64 ? 1 : 2);
  return static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(wanted, most)));
}

template <typename Call>
void launch(void (*kernel)(const Call), const Call& c, int64_t blocks, cudaStream_t stream,
            int threads = kThreads) {
  void* params[] = {const_cast<Call*>(&c)};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel),
                                   dim3(blocks_for(blocks, threads)), dim3(threads), params, 0, stream));
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

// Whether results are stored past L2's ordinary order (126 MB): where a call reads and writes more than
// that, its results would only drive each other out.  (4096 tokens of 2048 bf16 copied, 168 MB in all,
// 23.2 -> 20.8 us; 28672 x 4096 floats quantised 90 -> 87 us; 4095 x 8 rows of 7168 summed 84 -> 80 us.
// Not below: 1021 tokens of 7168 copied in 8 bits, 73 MB, 12.9 -> 15.5 us; 8168 x 2048 quantised 8.6 -> 11
// us, and the next kernel finds them in L2.)
bool stream_past_l2(int64_t bytes) { return bytes > (int64_t{126} << 20); }

// Rows that a call writes (or reads) at most: of a table with a capacity only those that entries of the
// routing have, unless the others are cleared.  (1024 tokens of 7168 bf16, top-6, to 64 x 512 rows, 470 MB
// of which 88 are written, and back: 32.2 us past L2, 29.4 through it; in 8 bits 12.0, 11.5.)
int64_t touched_rows(const ExpertRowsView& r, bool zero_rest) {
  return zero_rest ? r.num_rows : std::min(r.num_rows, static_cast<int64_t>(r.num_tokens) * r.topk);
}

int size_of(FloatType t) { return t == FloatType::kFloat ? 4 : 2; }

}  // namespace

void launch_sort_by_expert(const SortByExpertCall& c, cudaStream_t stream) {
  PPLX_CHECK(c.num_experts > 0 && c.num_experts <= kMaxSortExperts, "num_experts out of range");
  auto* kernel = c.wide_indices ? sort_kernel<uint64_t> : sort_kernel<uint32_t>;
  const int64_t n = static_cast<int64_t>(c.num_tokens) * c.topk;
  // us with 256 experts, one block of 256 / 512 threads, clusters of 8 / 16 blocks of 512: 8 entries
  // 3.0 / 3.3 / 4.3 / 4.9, 512 entries 3.7 / 3.6 / 4.3 / 4.9, 1024 entries 4.3 / 4.0 / 4.3 / 4.9, 2048
  // entries 5.6 / 4.9 / 4.2 / 4.9, 8192 entries 20.3 / 13.5 / 4.9 / 5.0, 32768 entries 92.7 / 51.9 / 7.5 /
  // 6.2.  (More than 65536 entries no longer fit the registers: 65536 11 us, 262144 42, 1048576 110.)
  const int blocks = n <= 1024 ? 1 : n <= 8192 ? 8 : 16;
  const int threads = n <= 256 ? 256 : kSortThreads;
  const int warps = threads / 32;
  const size_t smem = sizeof(uint32_t) * (static_cast<size_t>(warps + 3) * c.num_experts + 1);
  // (The most that any call takes, not this one's: threads that launch with other sizes set it too.)
  if (smem > 48 * 1024)
    CUDA_CHECK(cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        static_cast<int>(sizeof(uint32_t)) * ((kSortThreads / 32 + 3) * kMaxSortExperts + 1)));
  if (blocks > 8)
    CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  void* params[] = {const_cast<SortByExpertCall*>(&c)};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(blocks), dim3(threads),
                                   params, smem, stream, static_cast<unsigned>(blocks)));
}

void launch_permute_tokens(const PermuteCall& call, cudaStream_t stream) {
  PermuteCall c = call;
  c.streaming = stream_past_l2((c.rows.num_tokens + touched_rows(c.rows, c.zero_rest)) * c.row_bytes);
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

void launch_unpermute_tokens(const UnpermuteCall& call, cudaStream_t stream) {
  UnpermuteCall c = call;
  c.streaming =
      stream_past_l2((c.rows.num_tokens + touched_rows(c.rows, false)) * c.hidden * size_of(c.type));
  if (c.rows.num_tokens == 0 || c.hidden == 0) return;
  const uint64_t size = size_of(c.type);
  const int vec = alignment(16, {address(c.y), address(c.out), c.hidden * size, c.out_stride * size});
  with_type(c.type, vec, [&](auto t, auto v) {
    using T = decltype(t);
    auto pieces = [&](int cols) {
      return static_cast<int64_t>(c.rows.num_tokens) * ceil_div(c.hidden / v.value, 32 * cols);
    };
    // Where every warp has one piece at most the rows of a token come in fewer turns, otherwise two rows
    // and columns at a time keep most bytes in flight.  us for 4 x 1 and 2 x 2 (and 4 x 2, 8 x 1), bf16: 16
    // tokens of 2048, top-8 2.3, 3.1; 128 of 7168, top-8 3.7, 4.0; 512 of 7168 9.1, 8.4; 4095 of 7168 81.4,
    // 81.4 (84.2, 96.5); 4096 of 4096, top-2 23.2, 14.6 (19.1, 41.9); of 2048, top-6 21.2, 18.2 (20.7, 25.3).
    // Rows of odd width, whose vectors are single values, take four columns: 4095 of 3971, top-8 141 us with
    // two, 116 with four, 127 with eight; 300 of 1001, top-6 4.0, 3.8, 5.1.
    constexpr int kCols = v.value * sizeof(T) == 2 ? 4 : 2;
    if (pieces(1) <= static_cast<int64_t>(get_sm_count()) * 32)
      launch(unpermute_kernel<T, v.value, 4, 1>, c, ceil_div<int64_t>(pieces(1), kWarps), stream);
    else
      launch(unpermute_kernel<T, v.value, 2, kCols>, c, ceil_div<int64_t>(pieces(kCols), kWarps), stream);
  });
}

void launch_unpermute_backward(const UnpermuteBackwardCall& c, cudaStream_t stream) {
  const int64_t blocks = c.rows.num_tokens + (c.grad_y != nullptr ? c.rows.num_rows : 0);
  if (blocks == 0) return;
  const uint64_t size = size_of(c.type);
  const int vec = alignment(16, {address(c.y), address(c.grad), address(c.grad_y), c.hidden * size,
                                 c.grad_stride * size});
  with_type(c.type, vec, [&](auto t, auto v) {
    using T = decltype(t);
    // us for 2 rows x 2 columns, 2 x 4, 4 x 1, 8 x 1: 4096 tokens of 4096 bf16, top-2 28.3, 30.0, 34.1, 50.3;
    // top-4 50.8, 51.4, 50.2, 60.5; of 2048, top-6 38.2, 38.2, 42.9, 42.5; 4095 of 7168, top-8 159, 172,
    // 161, 160; 16 of 2048, top-8 4.9, 5.0, 3.7, 3.4.  Single values (odd widths) with four columns: 4095 of
    // 3971, top-8 194 -> 175 us, 16 of 999 7.0 -> 6.0.
    constexpr int kRows = 2, kCols = v.value * sizeof(T) == 2 ? 4 : 2;
    // As few threads as cover a token's vectors in whole turns of the block.
    const int vecs = c.hidden / v.value;
    const int turns = std::max(1, ceil_div(vecs, kThreads * kCols));
    const int threads = std::min(kThreads, std::max(32, round_up(ceil_div(vecs, turns * kCols), 32)));
    launch(unpermute_backward_kernel<T, v.value, kRows, kCols>, c, blocks, stream, threads);
  });
}

void launch_quantize_rows(const QuantizeRowsCall& call, cudaStream_t stream) {
  QuantizeRowsCall c = call;
  ExpertRowsView r{};
  if (c.rows != nullptr) r = *c.rows;
  // (Only the device knows how many counted rows there are.  32 x 1024 rows of 2048, us past L2 and not, all
  // live 30.9, 31.8, quantised twice and read back 105.5, 103.3; 32 live each 7.8, 7.8.)
  if (c.rows != nullptr)
    c.streaming = stream_past_l2(
        (touched_rows(r, c.zero_rest) + r.num_tokens * static_cast<int64_t>(size_of(c.type))) * c.hidden);
  else
    c.streaming = c.counts == nullptr && stream_past_l2(c.num_rows * (1 + size_of(c.type)) * c.hidden);
  const int64_t items = (c.rows != nullptr ? r.num_tokens : c.num_rows) +
                        (c.zero_rest ? r.num_rows : 0);
  if (items == 0) return;
  const uint64_t size = size_of(c.type);
  // A vector of x of `vec` bytes becomes one of vec / size bytes of q.
  const int vec = std::min<int>(
      alignment(16, {address(c.x), c.hidden * size, c.x_stride * size}),
      alignment(16, {address(c.q), static_cast<uint64_t>(c.hidden)}) * static_cast<int>(size));
  with_type(c.type, vec, [&](auto t, auto v) {
    using T = decltype(t);
    const int vecs = c.hidden / v.value;
    auto run = [&](auto* kernel, int threads, int64_t teams_wanted) {
      void* params[] = {&c, &r};
      CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel),
                                       dim3(blocks_for(teams_wanted, threads)), dim3(threads), params,
                                       0, stream));
    };
    auto pick = [&](auto permuted) {
      constexpr bool kPermuted = decltype(permuted)::value;
      if constexpr (v.value == 1) {
        // us with 256 and 64 threads: 30000 rows of 33 bf16 35.9, 16.4; 4095 of 401 7.2, 4.9; of 1001 9.5, 7.4;
        // 8168 of 2047 23.0, 18.9; 4095 of 3971 18.4, 19.3; 200 of 7001 4.8, 10.5; 4095 tokens copied to 8
        // rows, of 401 19.1, 11.9, of 1001 31.6, 24.0, of 3971 70.6, 78.4; 1 of 2047 6.6, 13.8.
        if (c.hidden <= 512 || (c.hidden <= 2048 && items > 8 * get_sm_count()))
          run(quantize_ragged_kernel<T, kPermuted, 64>, 64, items);
        else run(quantize_ragged_kernel<T, kPermuted, kThreads>, kThreads, items);
      } else {
        // A warp per row up to 256 vectors, a block above; copies of many tokens, whose rounded values are
        // stored several times, a block with eight vectors per thread above 128.  us for a block with four vectors per
        // thread, a warp with eight, a block with eight: 8168 rows of 2048 bf16 8.3, 7.3, 8.4; of 1408 7.8,
        // 6.8, 7.7; of 4096 15.9, -, 16.0; 4096 of 7168 14.7, -, 15.1; 4096 tokens of 2048 copied to 6 rows
        // 12.5, 13.3, 11.8; 1021 of 7168 to 8 rows 14.0, -, 13.4; 77 of 7168 5.1, -, 7.2.
        const int64_t by_warps = ceil_div<int64_t>(items, kWarps);
        if (vecs <= 32 * 4)
          return run(quantize_kernel<T, v.value, 4, true, kPermuted>, kThreads, by_warps);
        if constexpr (!kPermuted) {
          if (vecs <= 32 * 8)
            return run(quantize_kernel<T, v.value, 8, true, kPermuted>, kThreads, by_warps);
        }
        if (vecs <= kThreads * 4 && (!kPermuted || r.num_tokens <= 4 * get_sm_count()))
          return run(quantize_kernel<T, v.value, 4, false, kPermuted>, round_up(ceil_div(vecs, 4), 32),
                     items);
        const int threads = std::min(kThreads, round_up(ceil_div(vecs, 8), 32));
        run(quantize_kernel<T, v.value, 8, false, kPermuted>, threads, items);
      }
    };
    if (c.rows != nullptr) pick(std::true_type{});
    else pick(std::false_type{});
  });
}

}  // namespace pplx
