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
  uint16_t* C = nullptr;
  long long ldc = 0;
  int M = 0, N = 0;
  int fmt = 1;                       // 0 = f16, 1 = bf16
  int vec = 0;                       // C's base and row pitch are multiples of 16 bytes
  const CUtensorMap* tmC = nullptr;  // 32 x 32 boxes of C, valid when vec (set by the kernel)
  __device__ bool staged() const { return vec != 0; }
  __device__ const CUtensorMap* tmap() const { return tmC; }
  __device__ bool chunk_in_bounds(const TileInfo& ti, int row0, int c) const {
    return ti.m0 + row0 < M && ti.n0 + c < N;
  }
  __device__ __forceinline__ void pack(const uint32_t* r, uint4* v) const {
    uint32_t* w = reinterpret_cast<uint32_t*>(v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      w[j] = ptx::pack_16x2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]), fmt);
  }
  __device__ static void fence_before_done() {}
  __device__ void tile_done(const TileInfo&) {}
  __device__ void begin_tile(const TileInfo&, int) {}
  __device__ void end_tile(const TileInfo&, int) {}
  // Element stores: C whose base or pitch rules TMA out (an odd number of columns).
  __device__ __forceinline__ void store(const TileInfo& ti, int row, int c, const uint32_t* r) const {
    const int gm = ti.m0 + row, gn = ti.n0 + c;
    if (gm >= M) return;
    uint16_t* p = C + (size_t)gm * ldc + gn;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (gn + j < N) p[j] = (uint16_t)ptx::pack_16x2(__uint_as_float(r[j]), 0.f, fmt);
  }
};

}  // namespace gemm
}  // namespace gicc
