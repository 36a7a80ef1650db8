// Pieces shared by the expert GEMMs whose operands are 128-byte swizzle rows of K on both sides (bf16
// and 8-bit integers): the cut of the experts' rows into token tiles, the loads of a tile, the
// SwiGLU epilogue's arithmetic.
#pragma once

#include <cstdint>

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "../core/device_utils.cuh"
#include "../core/tcgen05.cuh"

namespace pplx {
namespace cut {

constexpr int kMmaTokens = 256;   // token rows per MMA
constexpr int kMaxTokens = 512;   // token rows per tile

struct Tile {
  int expert;
  int w_blk;    // block of weight rows (of the pair or the single CTA)
  int first;    // first token row of the tile inside its expert
  int width;    // token rows of the tile, a multiple of kUnit
  int rows;     // valid rows of the expert
};

// Token tiles of an expert: as few as `limit` rows per tile allow, as equal as whole units allow.
template <int kUnit>
struct Cut {
  int units, tiles;
  __device__ __forceinline__ Cut(int rows, int limit)
      : units((rows + kUnit - 1) / kUnit),
        // (Divisions by numbers that only the device knows take hundreds of cycles; most experts have
        // one tile.)
        tiles(units * kUnit <= limit ? min(units, 1) : (units * kUnit + limit - 1) / limit) {}
  __device__ __forceinline__ int widest() const {
    return (tiles == 1 ? units : (units + tiles - 1) / tiles) * kUnit;
  }
};

template <int kUnit>
__device__ __forceinline__ Tile locate(const uint32_t* tile_start, const uint32_t* rows_of,
                                       int num_experts, int limit, uint32_t t) {
  Tile c;
  c.expert = find_group(tile_start, num_experts, t);
  c.rows = static_cast<int>(rows_of[c.expert]);
  const Cut<kUnit> cut(c.rows, limit);
  const uint32_t rem = t - tile_start[c.expert];
  if (cut.tiles == 1) {
    c.w_blk = static_cast<int>(rem);
    c.first = 0;
    c.width = cut.units * kUnit;
    return c;
  }
  c.w_blk = static_cast<int>(rem / cut.tiles);
  const int i = static_cast<int>(rem) - c.w_blk * cut.tiles;
  const int each = cut.units / cut.tiles, wider = cut.units - each * cut.tiles;
  c.width = (each + (i < wider ? 1 : 0)) * kUnit;
  c.first = (i * each + min(i, wider)) * kUnit;
  return c;
}

__device__ __forceinline__ float silu(float v) { return v / (1.0f + __expf(-v)); }

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t pack_bits(uint32_t a, uint32_t b) {
  return pack_bf16(__uint_as_float(a), __uint_as_float(b));
}

// Token rows of a tile that its first MMA takes; the second takes the rest.
__device__ __forceinline__ int first_mma(int width) {
  return width <= kMmaTokens ? width : ((width >> 1) + 31) & ~31;
}

template <bool kPair>
__device__ __forceinline__ void load_rows(void* dst, const CUtensorMap* map, uint64_t* full, int k,
                                          int row, int plane) {
  if constexpr (kPair) tc::tma_load_3d_2cta(dst, map, full, k, row, plane);
  else tc::tma_load_3d(dst, map, full, k, row, plane);
}

}  // namespace cut
}  // namespace pplx
