// out16_epi.cuh -- epilogue of the CTA-pair core for row-major outputs in bf16 or f16.
#pragma once
#include <cstdint>
#include <cuda.h>

#include "gicc/device/gemm_core2.cuh"

namespace gicc {
namespace gemm {

struct Out16Epi {
  static constexpr bool kNeedsTileDone = false;
  static constexpr bool kPairHalves = false;
  static constexpr bool kStagedStore = true;
  static constexpr bool kSwizzledBox = true;
  uint16_t* C = nullptr;
  long long ldc = 0;
  int M = 0, N = 0;
  int fmt = 1;                       // 0 = f16, 1 = bf16
  int vec = 0;                       // C's base and row pitch are multiples of 16 bytes
  const CUtensorMap* tmC = nullptr;  // 32 x 32 boxes of C, 64-byte swizzle, valid when vec (set by the kernel)
  __device__ bool staged() const { return vec != 0; }
  __device__ const CUtensorMap* tmap() const { return tmC; }
  __device__ bool chunk_in_bounds(const TileInfo& ti, int row0, int c) const {
    return ti.m0 + row0 < M && ti.n0 + c < N;
  }
  __device__ int rows_left(const TileInfo& ti, int row0) const { return M - ti.m0 - row0; }
  __device__ __forceinline__ void pack(const uint32_t* r, uint4* v) const {
    uint32_t* w = reinterpret_cast<uint32_t*>(v);
    if (fmt) {
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = ptx::pack_bf16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) w[j] = ptx::pack_f16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
    }
  }
  __device__ static void fence_before_done() {}
  __device__ void tile_done(const TileInfo&) {}
  __device__ void begin_tile(const TileInfo&, int) {}
  __device__ void end_tile(const TileInfo&, int) {}
  // C whose base or pitch rules TMA out (an odd number of columns): one row of the box at a
  // time, 32 consecutive columns per warp store.
  static constexpr bool kRowStores = true;
  __device__ __forceinline__ void store_rows(const TileInfo& ti, int row0, int c, const uint16_t* box, int lane) const {
    const int gm = ti.m0 + row0, gn = ti.n0 + c + lane;
    const int rows = min(32, M - gm);
    if (gn >= N) return;
    uint16_t* p = C + (size_t)gm * ldc + gn;
#pragma unroll 8
    for (int i = 0; i < rows; ++i) p[(size_t)i * ldc] = box[i * 32 + (((lane >> 3) ^ ((i >> 1) & 3)) * 8) + (lane & 7)];
  }
  __device__ __forceinline__ void store(const TileInfo&, int, int, const uint32_t*) const {}  // never reached
};

}  // namespace gemm
}  // namespace gicc
