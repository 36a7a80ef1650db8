// Expert GEMM of 8-bit integers for sm_100a, one fp32 scale per token row and per weight row:
//   out[r, n] = sx[r] * sw[e][n] * sum_k x[r, k] * w[e][n, k]
// for the rows r of expert e, or SwiGLU of two such products when w[e] stacks a gate and an up
// projection.  The sums are exact in the 32-bit integers of tensor memory (kind::i8): K is at most
// 131071, so that K * 128 * 128 stays below 2^31.  Only the scaled result is rounded: the integer
// to fp32, two products, and once to bf16 or fp16.
//
// The rows of the experts lie in planes of their own ([experts][capacity], as the all-to-all
// delivers them), or one expert's after the other's with the first row of each in `offsets`.
//
// As in the bf16 kernel the WEIGHTS are the M operand of the MMAs and the tokens the N operand, so
// the work follows the rows there are; a stage of 128 bytes of K holds 128 integers, twice what a
// stage of the bf16 kernel holds.  A CTA owns a tile of 128 weight rows times a token tile of 16
// to 256 rows of one expert.
//
// Roles (persistent over tiles): warp 0 TMA producer, warp 1 MMA issuer, warp 2 tensor-memory
// allocation, warps 4-11 epilogue.  Two accumulators of 256 columns let the epilogue of a tile run
// under the MMAs of the next.  Every mbarrier wait is bounded: when one runs out the CTA raises a
// shared abort flag, all roles leave their loops, in-flight TMA loads are drained, tensor memory is
// freed and the kernel returns with *status = 1.
#include <algorithm>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../core/device_utils.cuh"
#include "../core/ptx.cuh"
#include "../core/tcgen05.cuh"
#include "../core/tensor_map.h"
#include "../core/utils.h"
#include "grouped_gemm.h"
#include "token_cut.cuh"
#include "token_tile.cuh"

namespace pplx {
namespace {

using namespace tok;
using namespace cut;

constexpr int kBlockM = 128;      // weight rows per CTA and tile
constexpr int kBlockK = 128;      // integers = bytes: one 128-byte swizzle row
constexpr int kUmmaK = 32;
constexpr int kMaxStages = 12;
constexpr int kThreads = 384;
constexpr int kTmemCols = 512;    // two accumulators of 256 columns
constexpr uint32_t kRowBytes = kBlockK;
constexpr uint32_t kWBytes = kBlockM * kRowBytes;
constexpr uint32_t kWaitLimitNs = 2000000000u;  // 2 s per wait
constexpr int kMaxExperts = 1024;
constexpr int kMaxK = 131071;
constexpr int kSegBytes = 256 + 16;  // 128 columns of 16 bits of one token, padded

struct Int8GemmArgs {
  const int32_t* counts;   // [num_experts] valid rows per expert; null: rows_per_expert
  const int32_t* offsets;  // [num_experts] first row per expert; null: planes of rows_per_expert
  const float* sx;
  int64_t sx_stride_e;
  const float* sw;
  int64_t sw_stride_e;
  uint16_t* out;           // bf16 or fp16
  int64_t out_stride_e, out_stride_row;
  uint32_t* status;
  int num_experts;
  int rows_per_expert;     // rows of a plane, or of all experts
  int n_out, k;
  uint32_t ring_bytes;
  bool fp16;
};

struct Control {
  uint64_t full[kMaxStages];
  uint64_t empty[kMaxStages];
  uint64_t tmem_full[2];
  uint64_t tmem_empty[2];
  uint32_t tmem_base;
  uint32_t abort_flag;
  uint32_t max_rows;
  uint32_t max_width;
  unsigned long long best_limit;
  alignas(16) float sx[2][kMaxTokens];  // scales of a tile's tokens, of two tiles in turn
  alignas(16) uint8_t seg[2][2][16][kSegBytes];  // [warp group][alternating][token][column]
};

struct TokenMaps {
  CUtensorMap x64, x16;
};

__device__ __forceinline__ float scaled(uint32_t sum, float sx, float sw) {
  return static_cast<float>(static_cast<int32_t>(sum)) * sx * sw;
}

__device__ __forceinline__ uint32_t pack(float a, float b, bool fp16) {
  if (!fp16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool SWIGLU>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_gemm_int8_kernel(const __grid_constant__ CUtensorMap tmap_w,
                             const __grid_constant__ TokenMaps tmap_x,
                             const __grid_constant__ Int8GemmArgs g) {
  constexpr int kUnit = 16;
  constexpr int kCols = SWIGLU ? kBlockM / 2 : kBlockM;  // output columns per CTA and tile
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control* ctl = reinterpret_cast<Control*>(ring + g.ring_bytes);
  uint32_t* tile_start = reinterpret_cast<uint32_t*>(ctl + 1);  // [E + 1]
  uint32_t* rows_of = tile_start + g.num_experts + 1;           // [E] valid rows
  uint32_t* row0_of = rows_of + g.num_experts;                  // [E] first row in the token plane

  const uint32_t worker = blockIdx.x, workers = gridDim.x;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  const int w_blocks = ceil_div<int>(g.n_out, kCols);
  const int num_kb = ceil_div<int>(g.k, kBlockK);

  // ---- set-up ---------------------------------------------------------------
  if (tid == 0) {
    ctl->abort_flag = 0;
    ctl->max_rows = 0;
    ctl->max_width = kUnit;
    for (int s = 0; s < kMaxStages; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&ctl->tmem_full[b], 1);
      tc::mbar_init(&ctl->tmem_empty[b], 8);  // epilogue warps
    }
    tc::fence_mbar_init();
    tc::tma_prefetch_desc(&tmap_w);
    tc::tma_prefetch_desc(&tmap_x.x64);
    tc::tma_prefetch_desc(&tmap_x.x16);
  }
  if (warp == 2) {
    tc::tmem_alloc(&ctl->tmem_base, kTmemCols);
    tc::tmem_relinquish();
  }
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  __syncthreads();
  constexpr int limit = kMmaTokens;
  for (int e = tid; e < g.num_experts; e += blockDim.x) {
    // (Counts and offsets that do not fit the tensors are cut to them.)
    int first = 0, most = g.rows_per_expert;
    if (g.offsets != nullptr) {
      first = min(max(g.offsets[e], 0), g.rows_per_expert);
      most -= first;
    }
    const int rows = g.counts != nullptr ? min(max(g.counts[e], 0), most) : most;
    rows_of[e] = static_cast<uint32_t>(rows);
    row0_of[e] = static_cast<uint32_t>(first);
    const Cut<kUnit> cut(rows, limit);
    tile_start[e] = static_cast<uint32_t>(cut.tiles * w_blocks);
    if (cut.tiles > 0) atomicMax(&ctl->max_width, static_cast<uint32_t>(cut.widest()));
  }
  __syncthreads();
  if (warp == 0) warp_exclusive_scan_smem(tile_start, g.num_experts, lane, true);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  const uint32_t total_tiles = tile_start[g.num_experts];
  // As many stages as the launch's widest token tile leaves room for.
  const uint32_t stage_bytes = kWBytes + ctl->max_width * kRowBytes;
  const uint32_t stages = min(g.ring_bytes / stage_bytes, static_cast<uint32_t>(kMaxStages));

  // ---- roles ----------------------------------------------------------------
  if (warp == 0) {
    if (tc::elect_one()) {
      uint32_t stage = 0, phase = 0;
      uint32_t pending = 0;        // stages that have been filled at least once
      uint32_t pending_phase = 0;  // parity of the phase each stage was last filled in
      bool ok = *abort_flag == 0u;
      for (uint32_t t = worker; t < total_tiles && ok; t += workers) {
        const Tile c = locate<kUnit>(tile_start, rows_of, g.num_experts, limit, t);
        const int row0 = static_cast<int>(row0_of[c.expert]) + c.first;
        const int x_plane = g.offsets != nullptr ? 0 : c.expert;
        const int w_row = c.w_blk * kCols;
        const uint32_t tx = kWBytes + static_cast<uint32_t>(c.width) * kRowBytes;
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = tc::mbar_wait(&ctl->empty[stage], phase ^ 1u, abort_flag, kWaitLimitNs);
          if (!ok) break;
          uint8_t* w_dst = ring + stage * stage_bytes;
          uint8_t* x_dst = w_dst + kWBytes;
          uint64_t* full = &ctl->full[stage];
          pending |= 1u << stage;
          pending_phase = (pending_phase & ~(1u << stage)) | (phase << stage);
          tc::mbar_arrive_expect_tx(full, tx);
          if constexpr (SWIGLU)
            tc::tma_load_5d(w_dst, &tmap_w, full, kb * kBlockK, 0, 0, w_row / 8, c.expert);
          else
            load_rows<false>(w_dst, &tmap_w, full, kb * kBlockK, w_row, c.expert);
          int r = 0;
          for (; r + 64 <= c.width; r += 64, x_dst += 64 * kRowBytes)
            load_rows<false>(x_dst, &tmap_x.x64, full, kb * kBlockK, row0 + r, x_plane);
          for (; r < c.width; r += 16, x_dst += 16 * kRowBytes)
            load_rows<false>(x_dst, &tmap_x.x16, full, kb * kBlockK, row0 + r, x_plane);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok || *abort_flag != 0u) {
        // Give the loads already issued a bounded time to land before the CTA
        // leaves: their destination is this CTA's shared memory.
        const uint64_t t0 = ptx::globaltimer_ns();
        for (uint32_t s = 0; s < stages; ++s) {
          if (!((pending >> s) & 1u)) continue;
          while (!tc::mbar_try_wait(&ctl->full[s], (pending_phase >> s) & 1u)) {
            if (ptx::globaltimer_ns() - t0 > 100000000ull) break;  // 100 ms in total
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (tc::elect_one()) {
      uint32_t stage = 0, phase = 0, local = 0;
      bool ok = *abort_flag == 0u;
      for (uint32_t t = worker; t < total_tiles && ok; t += workers, ++local) {
        const Tile c = locate<kUnit>(tile_start, rows_of, g.num_experts, limit, t);
        const uint32_t idesc = tc::make_instr_desc_i8(kBlockM, c.width);
        const uint32_t buf = local & 1u;
        const uint32_t use = local >> 1;  // how often this accumulator was used before
        ok = tc::mbar_wait(&ctl->tmem_empty[buf], (use & 1u) ^ 1u, abort_flag, kWaitLimitNs);
        if (!ok) break;
        tc::tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + buf * kMmaTokens;
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = tc::mbar_wait(&ctl->full[stage], phase, abort_flag, kWaitLimitNs);
          if (!ok) break;
          tc::tc_fence_after_sync();
          const uint8_t* w_src = ring + stage * stage_bytes;
          const uint64_t w_desc = tc::make_smem_desc_sw128(w_src);
          const uint64_t x_desc = tc::make_smem_desc_sw128(w_src + kWBytes);
#pragma unroll
          for (int k = 0; k < kBlockK / kUmmaK; ++k)
            tc::mma_i8_ss(tmem_d, tc::advance_smem_desc(w_desc, k * kUmmaK),
                          tc::advance_smem_desc(x_desc, k * kUmmaK), idesc, (kb | k) != 0);
          tc::mma_commit(&ctl->empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) tc::mma_commit(&ctl->tmem_full[buf]);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int ew = (warp - 4) & 3;   // tensor-memory lanes [32 * ew, +32)
    const int wg = (warp - 4) >> 2;  // 16-token groups wg, wg + 2, wg + 4, ...
    const int n_tid = tid - 128;     // 0..255 over the eight warps
    const int lt = n_tid & 127;      // thread of the warp group
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
    uint32_t local = 0;
    bool ok = *abort_flag == 0u;
    for (uint32_t t = worker; t < total_tiles && ok; t += workers, ++local) {
      const Tile c = locate<kUnit>(tile_start, rows_of, g.num_experts, limit, t);
      const int live = min(c.width, c.rows - c.first);  // tokens of the tile that exist
      const int col0 = c.w_blk * kCols;
      const int64_t row0 = static_cast<int64_t>(row0_of[c.expert]) + c.first;
      // The tile's scales, while its MMAs run.  (The table of the tile before is still read: the
      // barrier below is what ends that.)
      float* sx = ctl->sx[local & 1u];
      for (int n = n_tid; n < c.width; n += 256)
        sx[n] = n < live ? g.sx[c.expert * g.sx_stride_e + row0 + n] : 0.0f;
      float sw[4];  // plain: weight rows lane / 4 + 0, 8, 16, 24; SwiGLU: gate, up of two columns
      {
        const float* s = g.sw + c.expert * g.sw_stride_e;
        const int col = col0 + (SWIGLU ? ew * 16 : ew * 32) + (lane >> 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = SWIGLU ? col + (i >> 1) * 8 : col + i * 8;
          sw[i] = at < g.n_out ? s[SWIGLU && (i & 1) ? g.n_out + at : at] : 0.0f;
        }
      }
      const uint32_t buf = local & 1u;
      ok = tc::mbar_wait(&ctl->tmem_full[buf], (local >> 1) & 1u, abort_flag, kWaitLimitNs);
      // All eight warps leave together or not at all: the barriers below must never be
      // entered by only some of them.
      {
        uint32_t all_ok;
        asm volatile(
            "{\n\t"
            ".reg .pred p, q;\n\t"
            "setp.ne.u32 q, %1, 0;\n\t"
            "bar.red.and.pred p, 1, 256, q;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "}\n"
            : "=r"(all_ok)
            : "r"(ok ? 1u : 0u)
            : "memory");
        ok = all_ok != 0u;
      }
      if (!ok) break;
      tc::tc_fence_after_sync();
      const int groups = c.width >> 4;
      const uint32_t t_acc = t_lane + buf * kMmaTokens;
      // A thread's values lie across token rows; each group of 16 tokens passes through shared
      // memory so that rows leave in 16-byte pieces.
#pragma unroll 1
      for (int grp = wg, alt = 0; grp < groups; grp += 2, alt ^= 1) {
        uint32_t lo[8], hi[8];
        load_group(t_acc + grp * 16, lo, hi);
        const float2 s0 = *reinterpret_cast<const float2*>(&sx[grp * 16 + 2 * (lane & 3)]);
        const float2 s1 = *reinterpret_cast<const float2*>(&sx[grp * 16 + 8 + 2 * (lane & 3)]);
        tc::tmem_ld_wait();
        uint8_t(*seg)[kSegBytes] = ctl->seg[wg][alt];
        if constexpr (SWIGLU) {
          // Lanes 0-7 of every 16 are gate rows, 8-15 the up rows of the same columns.
          auto pair = [&](const uint32_t* v, float2 s, float gate, float up) {
            return pack(silu(scaled(v[0], s.x, gate)) * scaled(v[2], s.x, up),
                        silu(scaled(v[1], s.y, gate)) * scaled(v[3], s.y, up), g.fp16);
          };
          stmatrix_x4_trans(&seg[8 * (lane >> 4) + (lane & 7)][(ew * 16 + ((lane >> 3) & 1) * 8) * 2],
                            pair(lo, s0, sw[0], sw[1]), pair(hi, s0, sw[2], sw[3]),
                            pair(lo + 4, s1, sw[0], sw[1]), pair(hi + 4, s1, sw[2], sw[3]));
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const float2 s = b == 0 ? s0 : s1;
            auto pair = [&](uint32_t v0, uint32_t v1, float w) {
              return pack(scaled(v0, s.x, w), scaled(v1, s.y, w), g.fp16);
            };
            stmatrix_x4_trans(&seg[8 * b + (lane & 7)][(ew * 32 + (lane >> 3) * 8) * 2],
                              pair(lo[4 * b], lo[4 * b + 1], sw[0]),
                              pair(lo[4 * b + 2], lo[4 * b + 3], sw[1]),
                              pair(hi[4 * b], hi[4 * b + 1], sw[2]),
                              pair(hi[4 * b + 2], hi[4 * b + 3], sw[3]));
          }
        }
        sync_group(wg);
        constexpr int kPieces = kCols / 8;  // 16-byte pieces of a token's row segment
        const int piece = lt % kPieces;
        const int col = col0 + piece * 8;
#pragma unroll
        for (int tok16 = lt / kPieces; tok16 < 16; tok16 += 128 / kPieces) {
          const int n = grp * 16 + tok16;
          const int4 v = *reinterpret_cast<const int4*>(&seg[tok16][piece * 16]);
          if (n < live && col + 8 <= g.n_out)
            *reinterpret_cast<int4*>(g.out + c.expert * g.out_stride_e +
                                     (row0 + n) * g.out_stride_row + col) = v;
        }
      }
      tc::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&ctl->tmem_empty[buf]);
    }
  }

  // ---- teardown -------------------------------------------------------------
  tc::tc_fence_before_sync();
  __syncthreads();
  if (warp == 2) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tmem_base, kTmemCols);
  }
  if (tid == 0 && ctl->abort_flag != 0u && g.status != nullptr) *g.status = 1u;
}

// [planes][rows][k] bytes with k contiguous; boxes of 128 bytes x box_rows.
CUtensorMap make_operand_map(const void* base, int64_t planes, int64_t rows, int64_t k,
                             int64_t stride_row, int64_t stride_plane, int box_rows) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride_row),
                                 static_cast<cuuint64_t>(stride_plane)};
  const cuuint32_t box[3] = {kBlockK, static_cast<cuuint32_t>(box_rows), 1};
  return encode_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box);
}

// 128 weight rows per tile.  Plain: consecutive ones.  SwiGLU: [experts][2 * n_out][k] seen as
// [experts][n_out / 8][gate, up][8][k], so that a box of 8 x 2 x 8 rows is eight gate rows, the
// eight up rows of the same columns, the next eight gate rows, ...
CUtensorMap make_weight_map(const Int8GemmCall& c) {
  if (!c.swiglu)
    return make_operand_map(c.w, c.num_experts, c.n_out, c.k, c.w_stride_row, c.w_stride_e, kBlockM);
  const cuuint64_t row = static_cast<cuuint64_t>(c.w_stride_row);
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(c.k), 8, 2,
                              static_cast<cuuint64_t>(c.n_out / 8),
                              static_cast<cuuint64_t>(c.num_experts)};
  const cuuint64_t strides[4] = {row, row * static_cast<cuuint64_t>(c.n_out), row * 8,
                                 static_cast<cuuint64_t>(c.w_stride_e)};
  const cuuint32_t box[5] = {kBlockK, 8, 2, 8, 1};
  return encode_map(CU_TENSOR_MAP_DATA_TYPE_UINT8, 5, c.w, dims, strides, box);
}

template <bool SWIGLU>
void launch_one(const CUtensorMap& tmap_w, const TokenMaps& tmap_x, Int8GemmArgs g, int grid,
                cudaStream_t stream) {
  auto* kernel = grouped_gemm_int8_kernel<SWIGLU>;
  const size_t fixed =
      1024 + sizeof(Control) + sizeof(uint32_t) * (3 * static_cast<size_t>(g.num_experts) + 1);
  // The stages take what the tables leave, at least three of the widest.
  constexpr size_t kSmem = 227 * 1024;
  static_assert(kSmem - (1024 + sizeof(Control) + sizeof(uint32_t) * (3 * kMaxExperts + 1)) >=
                    3 * (kWBytes + kMmaTokens * kRowBytes) + 1024,
                "too little shared memory for the stages");
  g.ring_bytes = static_cast<uint32_t>((kSmem - fixed) & ~static_cast<size_t>(1023));
  const size_t smem = fixed + g.ring_bytes;
  CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(smem)));
  void* params[] = {const_cast<CUtensorMap*>(&tmap_w), const_cast<TokenMaps*>(&tmap_x), &g};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(grid),
                                   dim3(kThreads), params, smem, stream, 1));
}

}  // namespace

void check_grouped_gemm_int8(const Int8GemmCall& c) {
  PPLX_CHECK(c.num_experts > 0 && c.num_experts <= kMaxExperts, "num_experts out of range");
  PPLX_CHECK(c.k > 0 && c.k % 16 == 0 && c.k <= kMaxK,
             "K must be a positive multiple of 16, at most " << kMaxK
                                                             << " (the 32-bit sums are exact)");
  PPLX_CHECK(c.n_out > 0 && c.n_out % 8 == 0, "the output width must be a positive multiple of 8");
  PPLX_CHECK(c.x_stride_row % 16 == 0 && c.x_stride_e % 16 == 0 && c.w_stride_row % 16 == 0 &&
                 c.w_stride_e % 16 == 0,
             "operand strides must be multiples of 16 bytes");
  PPLX_CHECK(reinterpret_cast<uintptr_t>(c.out) % 16 == 0 && c.out_stride_row % 8 == 0 &&
                 c.out_stride_e % 8 == 0,
             "the output must be 16-byte aligned");
  PPLX_CHECK(reinterpret_cast<uintptr_t>(c.x) % 16 == 0 && reinterpret_cast<uintptr_t>(c.w) % 16 == 0,
             "the operands must be 16-byte aligned");
}

void launch_grouped_gemm_int8(const Int8GemmCall& c, cudaStream_t stream) {
  check_grouped_gemm_int8(c);
  if (c.rows_per_expert == 0) return;
  const int64_t planes = c.offsets != nullptr ? 1 : c.num_experts;
  auto tokens = [&](int box) {
    return make_operand_map(c.x, planes, c.rows_per_expert, c.k, c.x_stride_row,
                            planes == 1 ? c.rows_per_expert * c.x_stride_row : c.x_stride_e, box);
  };
  const TokenMaps tmap_x{tokens(64), tokens(16)};
  const CUtensorMap tmap_w = make_weight_map(c);
  Int8GemmArgs g{};
  g.counts = c.counts;
  g.offsets = c.offsets;
  g.sx = c.sx;
  g.sx_stride_e = c.sx_stride_e;
  g.sw = c.sw;
  g.sw_stride_e = c.sw_stride_e;
  g.out = static_cast<uint16_t*>(c.out);
  g.out_stride_e = c.out_stride_e;
  g.out_stride_row = c.out_stride_row;
  g.status = c.status;
  g.num_experts = c.num_experts;
  g.rows_per_expert = c.rows_per_expert;
  g.n_out = c.n_out;
  g.k = c.k;
  g.fp16 = c.fp16;
  const int grid = get_sm_count();
  if (c.swiglu) launch_one<true>(tmap_w, tmap_x, g, grid, stream);
  else launch_one<false>(tmap_w, tmap_x, g, grid, stream);
}

}  // namespace pplx
