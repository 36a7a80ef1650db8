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
// to 256 rows of one expert; or a CTA pair (cta_group::2) 256 weight rows, 128 in each CTA, times 32
// to 512, of which each CTA loads half (wide tiles as two halves that share the weights).  No TMA
// multicast is involved.
//
// What bounds it (cards differ by their power limit, 5 to 10 % from 256 rows per expert on): the weights'
// bytes up to some 128 rows per expert (32 experts of 2048 x 7168, up projection, 64 rows each: 142 to 150 us, 6.4
// to 6.8 TB/s with the rows); L2 around 256 rows (255 rows: 185 us alone, 158 by the bytes, 142 by the
// operations at twice the bf16 rate, 3.36 POPS); the tensor cores and the power limit above (1024 rows: 600
// to 700 us, 2.8 to 3.2 POPS; 8 experts of 4096 x 14336, down, 1024 rows: 295 to 350 us).  An epilogue that divided by the IEEE quotient and
// met two barriers per 16 tokens bound the tiles with short K: 128 experts of 768 x 2048, up, 256 rows 191
// us, now 93; down 77 -> 62.
//
// Roles (persistent over tiles): warp 0 TMA producer, warp 1 MMA issuer (leader CTA only), warp 2
// tensor-memory allocation, warps 4-11 epilogue.  Two accumulators of 256 columns let the epilogue
// of a tile run under the MMAs of the next; for wider tiles see below.  Every mbarrier wait is bounded:
// when one runs out the CTA raises a shared abort flag, all roles leave their loops, in-flight TMA loads
// are drained, tensor memory is freed and the kernel returns with *status = 1.
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
constexpr int kTmemCols = 512;
constexpr uint32_t kRowBytes = kBlockK;
constexpr uint32_t kWBytes = kBlockM * kRowBytes;
constexpr uint32_t kWaitLimitNs = 2000000000u;  // 2 s per wait
constexpr int kMaxExperts = 1024;
constexpr int kMaxK = 131071;
constexpr int kMaxSlots = 3;       // accumulators in tensor memory
constexpr int kThirdCols = 160;    // columns of each where there are three
constexpr int kTable = 32;        // tiles of a worker that are looked up in advance

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
  uint64_t tmem_full[kMaxSlots];
  uint64_t tmem_empty[kMaxSlots];
  uint32_t tmem_base;
  uint32_t abort_flag;
  uint32_t max_rows;
  uint32_t max_width;
  unsigned long long best_limit;
  Tile tiles[kTable];
  uint32_t warp_tiles[kThreads / 32];
  alignas(128) uint8_t seg[8][32 * 64];  // of each epilogue warp: 32 tokens' columns
  alignas(16) float sx[2][kMaxTokens];  // scales of a tile's tokens, of two tiles in turn
};

struct TokenMaps {
  CUtensorMap x64, x16;
};

__device__ __forceinline__ float scaled(uint32_t sum, float sx, float sw) {
  return static_cast<float>(static_cast<int32_t>(sum)) * sx * sw;
}

// silu(gate) * up by t = exp(-|gate|), which is at most 1: gate / (1 + t), and gate * t / (1 + t) for
// negative gates.  The reciprocal is the hardware's (one step of fp32 off); its argument lies in (1, 2], so
// no gate leaves its range (1 + exp(-gate) would, for gates below -87.33).
__device__ __forceinline__ float swiglu(float gate, float up) {
  const float t = __expf(-fabsf(gate));
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(1.0f + t));
  return (gate < 0.0f ? gate * t : gate) * inv * up;
}

__device__ __forceinline__ uint32_t pack(float a, float b, bool fp16) {
  if (!fp16) return pack_bf16(a, b);
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool SWIGLU, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_gemm_int8_kernel(const __grid_constant__ CUtensorMap tmap_w,
                             const __grid_constant__ TokenMaps tmap_x,
                             const __grid_constant__ Int8GemmArgs g) {
  constexpr int kCtas = kPair ? 2 : 1;
  constexpr int kUnit = 16 * kCtas;  // steps of an MMA's N: 16, or 32 for M = 256 over a pair
  constexpr int kCols = SWIGLU ? kBlockM / 2 : kBlockM;  // output columns per CTA and tile
  constexpr int kWarpCols = kCols / 4;       // of an epilogue warp
  constexpr int kPieces = kWarpCols / 8;     // 16-byte pieces of a token's row in them
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Control* ctl = reinterpret_cast<Control*>(ring + g.ring_bytes);
  uint32_t* tile_start = reinterpret_cast<uint32_t*>(ctl + 1);  // [E + 1]
  uint32_t* rows_of = tile_start + g.num_experts + 1;           // [E] valid rows
  uint32_t* row0_of = rows_of + g.num_experts;                  // [E] first row in the token plane

  const uint32_t cta_rank = kPair ? tc::cluster_ctarank() : 0u;
  const bool leader = cta_rank == 0u;
  const uint32_t worker = blockIdx.x / kCtas;   // tile-loop index
  const uint32_t workers = gridDim.x / kCtas;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  const int w_blocks = ceil_div<int>(g.n_out, kCols * kCtas);
  const int num_kb = ceil_div<int>(g.k, kBlockK);

  // ---- set-up ---------------------------------------------------------------
  if (tid == 0) {
    ctl->abort_flag = 0;
    ctl->max_rows = 0;
    ctl->max_width = kUnit;
    ctl->best_limit = ~0ull;
    for (int s = 0; s < kMaxStages; ++s) {
      tc::mbar_init(&ctl->full[s], 1);
      tc::mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < kMaxSlots; ++b) {
      tc::mbar_init(&ctl->tmem_full[b], 1);
      tc::mbar_init(&ctl->tmem_empty[b], 8 * kCtas);  // epilogue warps of the tile
    }
    tc::fence_mbar_init();
    tc::tma_prefetch_desc(&tmap_w);
    tc::tma_prefetch_desc(&tmap_x.x64);
    tc::tma_prefetch_desc(&tmap_x.x16);
  }
  if (warp == 2) {
    if constexpr (kPair) {
      tc::tmem_alloc_2cta(&ctl->tmem_base, kTmemCols);
      tc::tmem_relinquish_2cta();
    } else {
      tc::tmem_alloc(&ctl->tmem_base, kTmemCols);
      tc::tmem_relinquish();
    }
  }
  ptx::wait_for_previous_kernels();
  ptx::let_next_kernel_start();
  __syncthreads();
  // (Counts and offsets that do not fit the tensors are cut to them.)
  auto read_rows = [&](int e) {
    int first = 0, most = g.rows_per_expert;
    if (g.offsets != nullptr) {
      first = min(max(g.offsets[e], 0), g.rows_per_expert);
      most -= first;
    }
    const int rows = g.counts != nullptr ? min(max(g.counts[e], 0), most) : most;
    rows_of[e] = static_cast<uint32_t>(rows);
    row0_of[e] = static_cast<uint32_t>(first);
    return rows;
  };
  int limit = kPair ? kMaxTokens : kMmaTokens;
  uint32_t total_tiles, max_width;
  // One expert per thread, and none with more than one token tile: everything by two block barriers
  // (24 rows through 128 experts of 2048 x 768: 8.6 us, 9.3 the long way).
  const int my_rows = tid < g.num_experts ? read_rows(tid) : 0;
  for (int e = tid + kThreads; e < g.num_experts; e += kThreads) atomicMax(&ctl->max_rows, read_rows(e));
  {
    const uint32_t mine = my_rows > 0 ? w_blocks : 0;
    const uint32_t upto = warp_inclusive_scan(mine, lane);
    const uint32_t most = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(my_rows));
    if (lane == 31) {
      ctl->warp_tiles[warp] = upto;
      if (most > 0) atomicMax(&ctl->max_rows, most);
    }
    __syncthreads();
    const uint32_t max_rows = ctl->max_rows;
    if (max_rows <= kMmaTokens && g.num_experts <= kThreads) {
      uint32_t before = 0;
      total_tiles = 0;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        if (w == warp) before = total_tiles;
        total_tiles += ctl->warp_tiles[w];
      }
      max_width = max(round_up<uint32_t>(max_rows, kUnit), static_cast<uint32_t>(kUnit));
      const uint32_t start = before + upto - mine;
      if (tid < g.num_experts) tile_start[tid] = start;
      if (tid == 0) tile_start[g.num_experts] = total_tiles;
      // This worker's tiles of the thread's expert, as far as they are among its first.
      if (mine > 0)
        for (uint32_t i = start > worker ? (start - worker + workers - 1) / workers : 0;
             i < kTable && worker + i * workers < start + mine; ++i)
          ctl->tiles[i] = {tid, static_cast<int>(worker + i * workers - start), 0,
                           round_up(my_rows, kUnit), my_rows};
    } else {
      // The most token rows a tile may have.  One tile per expert up to 256 rows: there an expert is
      // bound by its weights, which more tiles would only read again.  Above, the limit that
      // minimises (waves of tiles) x (time of a tile).  Measured, in cycles per K block of 128 bytes
      // of a tile of w rows: 330 + 5/3 w up to 256 rows, 220 + 11/5 w up to 384 and 18/5 w - 340 above
      // (there are fewer stages); more than the 2 w cycles of its MMAs, because L2 delivers some 42
      // bytes per cycle and SM, of 16 KB of weights and 64 w bytes of tokens.  And the epilogue of more
      // than 256 rows is not hidden as a whole: 6 cycles per row with three accumulators, 10 with two.
      // Every CTA computes the same.  (us for one tile of all rows and two of half of them: 32 experts
      // of 2048 x 7168, up, 320 rows each 206, 255; 384: 241, 283; 512: 308, 310; down 320 rows 130,
      // 141; 512: 199, 171.)
      if (max_rows > kMmaTokens) {
        for (int cand = limit - kUnit * warp; 4 * cand >= limit; cand -= kUnit * (kThreads / 32)) {
          uint32_t tiles = 0, width = 0;
          for (int e = lane; e < g.num_experts; e += 32) {
            const Cut<kUnit> cut(static_cast<int>(rows_of[e]), cand);
            tiles += cut.tiles;
            width += cut.units * kUnit;
          }
          tiles = __reduce_add_sync(0xffffffffu, tiles);
          width = __reduce_add_sync(0xffffffffu, width);
          if (lane == 0) {
            const uint64_t waves =
                ceil_div<uint64_t>(static_cast<uint64_t>(tiles) * w_blocks, workers);
            const uint32_t w = width / tiles;
            const uint64_t each =
                max(max(330u + 5u * w / 3u, 220u + 11u * w / 5u), 18u * max(w, 100u) / 5u - 340u);
            const uint32_t drain = cand <= kMmaTokens ? 0u : cand <= 2 * kThirdCols ? 6u : 10u;
            const uint64_t cost = waves * (num_kb * each + drain * w);
            atomicMin(&ctl->best_limit, (cost << 16) | static_cast<uint64_t>(kMaxTokens - cand));
          }
        }
        __syncthreads();
        limit = kMaxTokens - static_cast<int>(ctl->best_limit & 0xffffu);
      }
      for (int e = tid; e < g.num_experts; e += kThreads) {
        const Cut<kUnit> cut(static_cast<int>(rows_of[e]), limit);
        tile_start[e] = static_cast<uint32_t>(cut.tiles * w_blocks);
        if (cut.tiles > 0) atomicMax(&ctl->max_width, static_cast<uint32_t>(cut.widest()));
      }
      __syncthreads();
      if (warp == 0) warp_exclusive_scan_smem(tile_start, g.num_experts, lane, true);
      __syncthreads();
      // The search for a tile takes one thread some 500 cycles: those of this worker's first tiles
      // are made side by side.
      total_tiles = tile_start[g.num_experts];
      max_width = ctl->max_width;
      if (tid < kTable && worker + tid * workers < total_tiles)
        ctl->tiles[tid] =
            locate<kUnit>(tile_start, rows_of, g.num_experts, limit, worker + tid * workers);
    }
  }
  auto tile = [&](uint32_t local) {
    return local < kTable ? ctl->tiles[local]
                          : locate<kUnit>(tile_start, rows_of, g.num_experts, limit,
                                          worker + local * workers);
  };
  tc::tc_fence_before_sync();
  __syncthreads();
  // The peer must see initialised barriers before anything arrives on them remotely.
  if constexpr (kPair) tc::cluster_sync();
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = ctl->tmem_base;
  // As many stages as the launch's widest token tile leaves room for.
  const uint32_t stage_bytes = kWBytes + max_width / kCtas * kRowBytes;
  const uint32_t stages = min(g.ring_bytes / stage_bytes, static_cast<uint32_t>(kMaxStages));
  // Accumulators are slots of tensor memory that the MMAs take in turn: two of 256 columns, or three
  // of 160 where a tile is wider than 256 rows, but none than 320.  A tile that is wider than a slot is
  // two halves, each with its MMAs and a slot of its own, so that the MMAs of a tile can begin while
  // the second half (with three: both) of the tile before is read out.
  const bool thirds = kPair && max_width > kMmaTokens && max_width <= 2 * kThirdCols;
  const int slot_cols = thirds ? kThirdCols : kMmaTokens;
  const uint32_t slots = thirds ? 3u : 2u;
  auto first_half = [&](int width) {
    return !kPair || width <= slot_cols ? width : ((width >> 1) + 31) & ~31;
  };

  // ---- roles ----------------------------------------------------------------
  if (warp == 0) {
    if (tc::elect_one()) {
      uint32_t stage = 0, phase = 0;
      uint32_t pending = 0;        // stages that have been filled at least once
      uint32_t pending_phase = 0;  // parity of the phase each stage was last filled in
      uint32_t local = 0;
      bool ok = *abort_flag == 0u;
      for (uint32_t t = worker; t < total_tiles && ok; t += workers, ++local) {
        const Tile c = tile(local);
        // This CTA's share of the tokens of each MMA.
        const int n0 = first_half(c.width);
        const int own0 = n0 / kCtas, own1 = (c.width - n0) / kCtas;
        const int tile_row = static_cast<int>(row0_of[c.expert]) + c.first;
        const int row0 = tile_row + static_cast<int>(cta_rank) * own0;
        const int row1 = tile_row + n0 + static_cast<int>(cta_rank) * own1;
        const int x_plane = g.offsets != nullptr ? 0 : c.expert;
        const int w_row = (c.w_blk * kCtas + static_cast<int>(cta_rank)) * kCols;
        const uint32_t tx = kCtas * kWBytes + static_cast<uint32_t>(c.width) * kRowBytes;
        for (int kb = 0; kb < num_kb; ++kb) {
          ok = tc::mbar_wait(&ctl->empty[stage], phase ^ 1u, abort_flag, kWaitLimitNs);
          if (!ok) break;
          uint8_t* w_dst = ring + stage * stage_bytes;
          uint8_t* x_dst = w_dst + kWBytes;
          uint64_t* full = &ctl->full[stage];
          pending |= 1u << stage;
          pending_phase = (pending_phase & ~(1u << stage)) | (phase << stage);
          // The bytes of both CTAs are counted on the leader's barrier, which only the leader
          // arms.
          if (leader) tc::mbar_arrive_expect_tx(full, tx);
          if constexpr (SWIGLU) {
            if constexpr (kPair)
              tc::tma_load_5d_2cta(w_dst, &tmap_w, full, kb * kBlockK, 0, 0, w_row / 8, c.expert);
            else
              tc::tma_load_5d(w_dst, &tmap_w, full, kb * kBlockK, 0, 0, w_row / 8, c.expert);
          } else {
            load_rows<kPair>(w_dst, &tmap_w, full, kb * kBlockK, w_row, c.expert);
          }
          auto load_tokens = [&](int row, int n) {
            int r = 0;
            for (; r + 64 <= n; r += 64, x_dst += 64 * kRowBytes)
              load_rows<kPair>(x_dst, &tmap_x.x64, full, kb * kBlockK, row + r, x_plane);
            for (; r < n; r += 16, x_dst += 16 * kRowBytes)
              load_rows<kPair>(x_dst, &tmap_x.x16, full, kb * kBlockK, row + r, x_plane);
          };
          load_tokens(row0, own0);
          if constexpr (kPair) load_tokens(row1, own1);
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
          // (The non-leader of a pair has no barrier of its own to watch; it just sits
          // out the time limit, which is far longer than any load takes.)
          while (!leader || !tc::mbar_try_wait(&ctl->full[s], (pending_phase >> s) & 1u)) {
            if (ptx::globaltimer_ns() - t0 > 100000000ull) break;  // 100 ms in total
          }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (leader && tc::elect_one()) {
      uint32_t stage = 0, phase = 0, local = 0;
      uint32_t slot = 0, lap = 0;  // the next accumulator, and the parity of its use
      auto next_slot = [&] {
        if (++slot == slots) slot = 0, lap ^= 1u;
      };
      auto next_stage = [&](uint32_t& at, uint32_t& parity) {
        if (++at == stages) at = 0, parity ^= 1u;
      };
      bool ok = *abort_flag == 0u;
      for (uint32_t t = worker; t < total_tiles && ok; t += workers, ++local) {
        const Tile c = tile(local);
        const int n0 = first_half(c.width), n1 = c.width - n0;
        const uint32_t idesc = tc::make_instr_desc_i8(kBlockM * kCtas, n0);
        const uint32_t idesc1 = tc::make_instr_desc_i8(kBlockM * kCtas, n1);
        const uint32_t slot0 = slot, lap0 = lap;
        next_slot();
        ok = tc::mbar_wait<kPair>(&ctl->tmem_empty[slot0], lap0 ^ 1u, abort_flag, kWaitLimitNs);
        if (!ok) break;
        tc::tc_fence_after_sync();
        // One half's MMAs of a K block.
        auto multiply = [&](uint32_t stage_at, uint32_t x_off, uint32_t tmem_d, uint32_t desc, int kb) {
          const uint8_t* w_src = ring + stage_at * stage_bytes;
          const uint64_t w_desc = tc::make_smem_desc_sw128(w_src);
          const uint64_t x_desc = tc::make_smem_desc_sw128(w_src + kWBytes + x_off);
#pragma unroll
          for (int k = 0; k < kBlockK / kUmmaK; ++k) {
            const uint64_t wd = tc::advance_smem_desc(w_desc, k * kUmmaK);
            const uint64_t xd = tc::advance_smem_desc(x_desc, k * kUmmaK);
            if constexpr (kPair) tc::mma_i8_ss_2cta(tmem_d, wd, xd, desc, (kb | k) != 0);
            else tc::mma_i8_ss(tmem_d, wd, xd, desc, (kb | k) != 0);
          }
        };
        auto commit = [&](uint64_t* bar) {  // in both CTAs of a pair
          if constexpr (kPair) tc::mma_commit_2cta(bar, 0x3);
          else tc::mma_commit(bar);
        };
        const uint32_t tmem0 = tmem_base + slot0 * slot_cols;
        if (!kPair || n1 == 0) {
          for (int kb = 0; kb < num_kb; ++kb) {
            ok = tc::mbar_wait(&ctl->full[stage], phase, abort_flag, kWaitLimitNs);
            if (!ok) break;
            tc::tc_fence_after_sync();
            multiply(stage, 0, tmem0, idesc, kb);
            commit(&ctl->empty[stage]);  // reusable once these MMAs have read it
            next_stage(stage, phase);
          }
          if (ok) commit(&ctl->tmem_full[slot0]);
          continue;
        }
        // Two halves: the first goes ahead, up to all stages, until the second's slot is free.
        const uint32_t slot1 = slot, lap1 = lap;
        next_slot();
        const uint32_t tmem1 = tmem_base + slot1 * slot_cols;
        uint32_t stage1 = stage, phase1 = phase;
        bool free1 = false;
        for (int kb0 = 0, kb1 = 0; kb1 < num_kb;) {
          if (!free1 && tc::mbar_try_wait<kPair>(&ctl->tmem_empty[slot1], lap1 ^ 1u)) {
            free1 = true;
            tc::tc_fence_after_sync();
          }
          if (free1 && kb1 < kb0) {
            multiply(stage1, n0 / kCtas * kRowBytes, tmem1, idesc1, kb1);
            commit(&ctl->empty[stage1]);
            next_stage(stage1, phase1);
            ++kb1;
          } else if (kb0 < num_kb && kb0 - kb1 < static_cast<int>(stages)) {
            ok = tc::mbar_wait(&ctl->full[stage], phase, abort_flag, kWaitLimitNs);
            if (!ok) break;
            tc::tc_fence_after_sync();
            multiply(stage, 0, tmem0, idesc, kb0);
            next_stage(stage, phase);
            if (++kb0 == num_kb) commit(&ctl->tmem_full[slot0]);
          } else {
            ok = tc::mbar_wait<kPair>(&ctl->tmem_empty[slot1], lap1 ^ 1u, abort_flag, kWaitLimitNs);
            if (!ok) break;
          }
        }
        if (ok) commit(&ctl->tmem_full[slot1]);
      }
    }
    __syncwarp();
  } else if (warp >= 4) {
    const int ew = (warp - 4) & 3;   // tensor-memory lanes [32 * ew, +32)
    const int wg = (warp - 4) >> 2;  // 32-token groups wg, wg + 2, wg + 4, ...
    const int n_tid = tid - 128;     // over the epilogue warps
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(ew * 32) << 16);
    uint32_t local = 0;
    uint32_t slot = 0, lap = 0;  // the next accumulator, and the parity of its use
    bool ok = *abort_flag == 0u;
    // A tile's scales are on their way while the tile before is finished.  sw, plain: weight rows
    // lane / 4 + 0, 8, 16, 24 of the warp; SwiGLU: gate and up of two columns.
    float next_sx[2], next_sw[4];
    auto fetch_scales = [&](const Tile& c) {
      const int live = min(c.width, c.rows - c.first);
      const float* sx = g.sx + c.expert * g.sx_stride_e + row0_of[c.expert] + c.first;
#pragma unroll
      for (int i = 0; i < 2; ++i) next_sx[i] = n_tid + 256 * i < live ? sx[n_tid + 256 * i] : 0.0f;
      const float* sw = g.sw + c.expert * g.sw_stride_e;
      const int col = (c.w_blk * kCtas + static_cast<int>(cta_rank)) * kCols + kWarpCols * ew + (lane >> 2);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = SWIGLU ? col + (i >> 1) * 8 : col + i * 8;
        next_sw[i] = at < g.n_out ? sw[SWIGLU && (i & 1) ? g.n_out + at : at] : 0.0f;
      }
    };
    if (worker < total_tiles) fetch_scales(tile(0));
    for (uint32_t t = worker; t < total_tiles && ok; t += workers, ++local) {
      const Tile c = tile(local);
      const int live = min(c.width, c.rows - c.first);  // tokens of the tile that exist
      const int col0 = (c.w_blk * kCtas + static_cast<int>(cta_rank)) * kCols;
      const int64_t row0 = static_cast<int64_t>(row0_of[c.expert]) + c.first;
      // (The table of the tile before is still read: the barriers below are what ends that.)
      float* sx = ctl->sx[local & 1u];
      sx[n_tid] = next_sx[0];
      sx[n_tid + 256] = next_sx[1];
      float sw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sw[i] = next_sw[i];
      // Where this thread stores: token lane / kPieces of every 32 / kPieces, 16 bytes.
      const int store_token = lane / kPieces, store_piece = lane % kPieces;
      const int store_col = col0 + kWarpCols * ew + store_piece * 8;
      uint16_t* out = g.out + c.expert * g.out_stride_e + row0 * g.out_stride_row + store_col;
      const int stored = store_col + 8 <= g.n_out ? live : 0;
      // 32 tokens at a time, the next ones on their way while these are finished.  A thread's values
      // lie across token rows; they pass through shared memory of the warp's own, so that rows leave
      // in 16-byte pieces.  (The pieces of a row of shared memory are in an order that keeps both
      // sides free of bank conflicts.)
      uint8_t* seg = ctl->seg[warp - 4];
      auto at = [&](int token, int piece) {
        return seg + token * (kPieces * 16) + ((piece ^ (token / (8 / kPieces) % kPieces)) * 16);
      };
      auto finish = [&](int n, const uint32_t (&lo)[16], const uint32_t (&hi)[16]) {
        __syncwarp();  // (the tokens before have been read)
#pragma unroll
        for (int b = 0; b < 4; b += SWIGLU ? 2 : 1) {
          const float2 s = *reinterpret_cast<const float2*>(&sx[n + 8 * b + 2 * (lane & 3)]);
          if constexpr (SWIGLU) {
            // Lanes 0-7 of every 16 are gate rows, 8-15 the up rows of the same columns.
            const float2 s1 = *reinterpret_cast<const float2*>(&sx[n + 8 * b + 8 + 2 * (lane & 3)]);
            auto pair = [&](const uint32_t* v, float2 t, float gate, float up) {
              return pack(swiglu(scaled(v[0], t.x, gate), scaled(v[2], t.x, up)),
                          swiglu(scaled(v[1], t.y, gate), scaled(v[3], t.y, up)), g.fp16);
            };
            stmatrix_x4_trans(at(8 * b + 8 * (lane >> 4) + (lane & 7), (lane >> 3) & 1),
                              pair(lo + 4 * b, s, sw[0], sw[1]), pair(hi + 4 * b, s, sw[2], sw[3]),
                              pair(lo + 4 * b + 4, s1, sw[0], sw[1]),
                              pair(hi + 4 * b + 4, s1, sw[2], sw[3]));
          } else {
            auto pair = [&](uint32_t v0, uint32_t v1, float w) {
              return pack(scaled(v0, s.x, w), scaled(v1, s.y, w), g.fp16);
            };
            stmatrix_x4_trans(at(8 * b + (lane & 7), lane >> 3), pair(lo[4 * b], lo[4 * b + 1], sw[0]),
                              pair(lo[4 * b + 2], lo[4 * b + 3], sw[1]),
                              pair(hi[4 * b], hi[4 * b + 1], sw[2]),
                              pair(hi[4 * b + 2], hi[4 * b + 3], sw[3]));
          }
        }
        __syncwarp();
#pragma unroll
        for (int t0 = 0; t0 < 32; t0 += 32 / kPieces) {
          const int token = n + t0 + store_token;
          const int4 v = *reinterpret_cast<const int4*>(at(t0 + store_token, store_piece));
          if (token < stored) *reinterpret_cast<int4*>(out + token * g.out_stride_row) = v;
        }
      };
      const int n0 = first_half(c.width);
      for (int from = 0; from < c.width && ok; from += n0) {
        uint64_t *full = &ctl->tmem_full[slot], *empty = &ctl->tmem_empty[slot];
        const uint32_t t_acc = t_lane + slot * slot_cols;
        ok = tc::mbar_wait(full, lap, abort_flag, kWaitLimitNs);
        if (++slot == slots) slot = 0, lap ^= 1u;
        // All eight warps leave together or not at all: this barrier must never be entered by only
        // some of them.
        {
          uint32_t all_ok;
          asm volatile(
              "{\n\t"
              ".reg .pred p, q;\n\t"
              "setp.ne.u32 q, %1, 0;\n\t"
              "bar.red.and.pred p, 1, %2, q;\n\t"
              "selp.u32 %0, 1, 0, p;\n\t"
              "}\n"
              : "=r"(all_ok)
              : "r"(ok ? 1u : 0u), "n"(256)
              : "memory");
          ok = all_ok != 0u;
        }
        if (!ok) break;
        tc::tc_fence_after_sync();
        if (from == 0 && t + workers < total_tiles) fetch_scales(tile(local + 1));
        // The accumulator is handed back when the warp has its last columns in registers.
        auto hand_back = [&] {
          tc::tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            if constexpr (kPair) tc::mbar_arrive_on_leader_relaxed(empty);
            else tc::mbar_arrive(empty);
          }
        };
        const int groups = (min(n0, c.width - from) + 31) >> 5;
        uint32_t lo[2][16], hi[2][16];
        int grp = wg;
        auto load = [&](int which, int at_grp) {
          tc::tmem_ld_16x256b_x4(t_acc + at_grp * 32, lo[which]);
          tc::tmem_ld_16x256b_x4(t_acc + (16u << 16) + at_grp * 32, hi[which]);
        };
        if (grp < groups) load(0, grp);
        else hand_back();
        auto step = [&](int now) {
          tc::tmem_ld_wait(lo[now]);
          tc::tmem_ld_wait(hi[now]);
          if (grp + 2 < groups) load(now ^ 1, grp + 2);
          else hand_back();
          finish(from + grp * 32, lo[now], hi[now]);
          grp += 2;
        };
#pragma unroll 1
        while (grp < groups) {
          step(0);
          if (grp < groups) step(1);
        }
      }
    }
  }

  // ---- teardown -------------------------------------------------------------
  tc::tc_fence_before_sync();
  __syncthreads();
  // Neither CTA of a pair may leave while the other can still touch its shared or
  // tensor memory.
  if constexpr (kPair) tc::cluster_sync();
  if (warp == 2) {
    tc::tc_fence_after_sync();
    if constexpr (kPair) tc::tmem_dealloc_2cta(tmem_base, kTmemCols);
    else tc::tmem_dealloc(tmem_base, kTmemCols);
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

template <bool SWIGLU, bool kPair>
void launch_one(const CUtensorMap& tmap_w, const TokenMaps& tmap_x, Int8GemmArgs g, int grid,
                cudaStream_t stream) {
  auto* kernel = grouped_gemm_int8_kernel<SWIGLU, kPair>;
  const size_t fixed =
      1024 + sizeof(Control) + sizeof(uint32_t) * (3 * static_cast<size_t>(g.num_experts) + 1);
  // The stages take what the tables leave, at least three of the widest.
  constexpr size_t kSmem = 227 * 1024;
  static_assert(kSmem - (1024 + sizeof(Control) + sizeof(uint32_t) * (3 * kMaxExperts + 1)) >=
                    3 * (kWBytes + kMmaTokens * kRowBytes) + 1024,
                "too little shared memory for the stages");
  g.ring_bytes = static_cast<uint32_t>((kSmem - fixed) & ~static_cast<size_t>(1023));
  const size_t smem = fixed + g.ring_bytes;
  // (The most that any call takes, not this one's: threads that launch with other sizes set it too.)
  CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(kSmem)));
  void* params[] = {const_cast<CUtensorMap*>(&tmap_w), const_cast<TokenMaps*>(&tmap_x), &g};
  CUDA_CHECK(launch_after_previous(reinterpret_cast<const void*>(kernel), dim3(kPair ? (grid & ~1) : grid),
                                   dim3(kThreads), params, smem, stream, kPair ? 2 : 1));
}

// Single CTAs, whose tiles of 128 weight rows divide a launch more finely, up to an expected mean of
// 64 rows per expert; pairs, which read the tokens half as often, from there on.  us, single and pairs,
// up projection: 128 experts of 768 x 2048, 8000 rows evenly 71.3 / 75.4, with a popularity of exponent
// 0.6 76.7 / 74.1, 1.2 81.3 / 80.1, 16000 rows 80.1 / 78.6, 90.3 / 85.7, 95.8 / 90.1; 64 experts of 1408
// x 2048, 1800 rows 62.6 / 64.9, 64.6 / 63.2, 68.2 / 65.0, 6000 rows 69.7 / 69.2, 75.9 / 71.8, 81.1 /
// 76.8; 32 experts of 2048 x 7168, 8000 rows 232 / 195, 232 / 211, 244 / 231.
bool want_pairs(const Int8GemmCall& c) {
  const int64_t rows = c.expected_total_rows > 0 ? c.expected_total_rows
                       : c.offsets != nullptr
                           ? c.rows_per_expert
                           : static_cast<int64_t>(c.num_experts) * c.rows_per_expert;
  return rows > 64 * static_cast<int64_t>(c.num_experts);
}

template <bool SWIGLU>
void launch_variant(const CUtensorMap& tmap_w, const TokenMaps& tmap_x, const Int8GemmArgs& g,
                    const Int8GemmCall& c, cudaStream_t stream) {
  const int grid = get_sm_count();
  if (want_pairs(c) && grid >= 2) launch_one<SWIGLU, true>(tmap_w, tmap_x, g, grid, stream);
  else launch_one<SWIGLU, false>(tmap_w, tmap_x, g, grid, stream);
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
  if (c.swiglu) launch_variant<true>(tmap_w, tmap_x, g, c, stream);
  else launch_variant<false>(tmap_w, tmap_x, g, c, stream);
}

}  // namespace pplx
