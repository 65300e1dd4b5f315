// ffn.cu -- the gated half of a feed-forward block, forward and backward.
//
//   forward   g = x Wg^T, u = x Wu^T, h = act(g) * u
//   backward  du = dh * act(g), dg = dh * u * act'(g),
//             dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// x [T, H], Wg and Wu [I, H], h and dh [T, I], all row-major, bf16 or f16, f32 accumulation.
//
// Forward, many rows (k_gated_pair): the CTA-pair core's 256 x 512 tile with its two column
// halves given to the two weights, so one tile holds g and u of the same 256 x 256 block of h
// and the activation and product run in the epilogue; x is read once for both.  Few rows
// (k_gated_split): the same on the split-K cluster core, which spreads the weights' stream
// over all SMs.
//
// For the backward pass the forward keeps g and u in f32 (`saved`): they enter dg and du as
// factors, and rounding them to 16 bits would add two roundings to the one that dg and du take
// themselves on their way to the tensor cores.  Their layout is private: float4 groups of four
// columns, the 32 rows of a TMEM lane quarter side by side, so every warp store and load is
// 512 contiguous bytes.
//
// Backward: k_gate_grad writes dg and du (16 bits, as MMA operands must be), then one launch
// (k_gated_bwd) runs the tiles of all three products: dx over the 2I deep concatenation of
// [dg | du] and [Wg ; Wu], and the two weight gradients over T.  The MMA reads operands of
// either major, so nothing is transposed in memory; putting the products into one launch
// leaves one partly filled last wave instead of two.  Products with few tiles for that (dx of few
// rows, small weight gradients over many) go to the split-K cluster core instead.
//
// Host entry points: gicc::ops::gated_linear, gated_linear_backward (C++, throw) and
// gicc_gated_linear, gicc_gated_linear_backward (C ABI, gicc/projections.h).
#include <algorithm>
#include <cuda.h>
#include <cuda_runtime.h>

#include "gicc/config.hpp"
#include "gicc/device/activation.cuh"
#include "gicc/device/gemm_core2.cuh"
#include "gicc/device/out16_epi.cuh"
#include "gicc/device/split_host.cuh"
#include "gicc/host_util.hpp"
#include "gicc/ops.hpp"
#include "gicc/projections.h"

namespace gicc {
namespace ffn {

using namespace gemm;

// ---- layout of the saved g and u -----------------------------------------------------------
__host__ __device__ inline int saved_cols(int I) { return (I + 15) / 16 * 16; }
__host__ __device__ inline size_t saved_plane(int T, int I) { return (size_t)((T + 31) / 32) * 32 * saved_cols(I); }
// float index of columns i .. i+3 (i % 4 == 0) of row t
__device__ __forceinline__ size_t saved_at(int t, int i, int I) {
  return (((size_t)(t >> 5) * (saved_cols(I) / 4) + (i >> 2)) * 32 + (t & 31)) * 4;
}

// ---- forward on CTA pairs ------------------------------------------------------------------
// Bound by the tensor pipe: 8192 x 8192 -> 8192 in 1410 us (1560 TFLOP/s), 4096 x 7168 -> 2048 in
// 165 us (1457: 128 tiles of 256 x 256 columns of h on 74 pairs).  NH = 1 halves the tile where that
// fills the pairs better (1001 x 2056 -> 5461: 60 us against 66).
struct GatedMaps {
  CUtensorMap x, g, u, h;
};

template <int NH>
struct GatedSched {
  static constexpr int kCols = NH * pair::BN2 / 2;  // columns of h per tile
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  int I, H;
  int num_m, num_n, group_m;
  int fmt;
  const GatedMaps* maps;  // set by the kernel
  __device__ int num_tiles() const { return num_m * num_n; }
  __device__ TileInfo tile(int t) const {
    int mb, nb;
    raster(t, num_m, num_n, group_m, mb, nb);
    TileInfo ti;
    ti.m0 = mb * 2 * BM;
    ti.n0 = nb * kCols;
    ti.a_row = ti.m0;
    ti.b_row = ti.n0;
    ti.kb0 = 0;
    ti.kb1 = (H + BK - 1) / BK;
    ti.aux = 0;
    ti.aux2 = 0;
    return ti;
  }
  __device__ bool producer_wait(const TileInfo&, int, uint64_t, volatile int*, ErrorRecord*) const { return true; }
  __device__ void issue_loads_pair(const TileInfo& ti, int kb, int crank, uint8_t* sA, uint8_t* sB, uint32_t bar) const {
    pair::tma_load_2d_pair(sA, &maps->x, bar, kb * BK, ti.a_row + crank * BM);
    if constexpr (NH == 2) {
      const int n = ti.b_row + crank * half_n(ti, 0) / 2;
      pair::tma_load_2d_pair(sB, &maps->g, bar, kb * BK, n);
      pair::tma_load_2d_pair(sB + pair::kBBytes, &maps->u, bar, kb * BK, n);
    } else {
      pair::tma_load_2d_pair(sB, crank == 0 ? &maps->g : &maps->u, bar, kb * BK, ti.b_row);
    }
  }
  // NH = 2: the tile's columns of each weight; NH = 1: of both
  __device__ int half_n(const TileInfo& ti, int) const {
    const int left = I - ti.n0;
    return NH == 2 ? min(pair::BN2, (left + 31) / 32 * 32) : 2 * min(pair::BN2 / 2, (left + 31) / 32 * 32);
  }
  __device__ uint32_t idesc(const TileInfo&, int n) const { return ptx::idesc_f16_f32(2 * BM, n, fmt, 0, 0); }
  __device__ uint64_t a_desc(const TileInfo&, uint32_t a, int k) const { return ptx::sdesc_kmajor_sw128(a + k * 32); }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const { return ptx::sdesc_kmajor_sw128(b + k * 32); }
};

struct GatedEpi : Out16Epi {
  static constexpr bool kGated = true;
  int kind = 0;
  float* saved = nullptr;  // g plane, then u plane; null: not kept
  template <int KIND>
  __device__ __forceinline__ void combine(const uint32_t* lo, uint32_t* hi) const {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      hi[j] = __float_as_uint(act::value(__uint_as_float(lo[j]), KIND) * __uint_as_float(hi[j]));
  }
  __device__ __forceinline__ void gate(const TileInfo& ti, int row, int c, const uint32_t* lo, uint32_t* hi) const {
    const int t = ti.m0 + row, i = ti.n0 + c;
    if (ti.m0 + (row & ~31) >= M) return;  // none of the warp's rows exists
    if (saved != nullptr && t < M) {
      float* g = saved + saved_at(t, i, N);
      float* u = g + saved_plane(M, N);
      const int left = saved_cols(N) - i;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (4 * j < left) {
          ptx::st_v4(g + 128 * j, make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]));
          ptx::st_v4(u + 128 * j, make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]));
        }
    }
    if (kind == ops::ACT_GELU) combine<ops::ACT_GELU>(lo, hi);
    else if (kind == ops::ACT_GELU_TANH) combine<ops::ACT_GELU_TANH>(lo, hi);
    else combine<ops::ACT_SILU>(lo, hi);
  }
};

template <int NH>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<NH>::kThreads, 1)
    k_gated_pair(const __grid_constant__ GatedMaps maps, GatedSched<NH> sched, GatedEpi epi, ErrorRecord* err,
                 uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.tmC = &maps.h;
  pair::gemm_core_pair<NH>(&maps.x, &maps.g, sched, epi, err, timeout_ns, -1);
}

// ---- forward for few rows ------------------------------------------------------------------
// Bound by the weights' stream from HBM behind 6 us of launch, first loads and the cluster's sum: 1 x
// 7168 -> 2048 (58.7 MB) in 18.5 us a call of a CUDA graph, against 76 and 46 us on the pairs; 37 x 4096
// -> 8200 (134 MB) in 28.5.  Both weights' columns go through one MMA: with few columns an MMA costs its
// issue (0.45 us a k-block with two, 0.22 with one).
struct GatedSplitOp : split::PlainOp {
  static constexpr int kAccs = 2;
  const CUtensorMap* tmU;  // set by the kernel
  uint16_t* h;
  long long ldh;
  int T, H, I, kind, vec, bn;
  float* saved;
  __device__ int depth() const { return (H + BK - 1) / BK; }
  __device__ void loads(int kb, int t0, int n0, uint8_t* x, uint8_t* w, uint64_t* bar) const {
    PlainOp::loads(kb, t0, n0, x, w, bar);
    ptx::tma_load_2d(w + bn * BK * 2, tmU, bar, kb * BK, n0);
  }
  __device__ __forceinline__ void emit(int t, int i, const float (*v)[4]) const {
    if (saved != nullptr && i < saved_cols(I)) {
      float* g = saved + saved_at(t, i, I);
      *reinterpret_cast<float4*>(g) = make_float4(v[0][0], v[0][1], v[0][2], v[0][3]);
      *reinterpret_cast<float4*>(g + saved_plane(T, I)) = make_float4(v[1][0], v[1][1], v[1][2], v[1][3]);
    }
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = act::value(v[0][j], kind) * v[1][j];
    split::store4_16(h + (size_t)t * ldh, i, I, o, type, vec);
  }
};

__global__ void __launch_bounds__(split::kThreads, 1)
    k_gated_split(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmG,
                  const __grid_constant__ CUtensorMap tmU, split::Shape sh, GatedSplitOp op, ErrorRecord* err,
                  uint64_t timeout_ns) {
  op.tmX = &tmX;
  op.tmW = &tmG;
  op.tmU = &tmU;
  split::split_core(sh, op, err, timeout_ns);
}

// ---- backward ------------------------------------------------------------------------------
// Tiles of 32 rows x 128 columns, two persistent blocks per SM.  In the saved layout a lane is a
// row and a tile's g and u are 16 KB each in one piece: they come by bulk copies into a ring of
// two, ahead of the arithmetic, and dh one tile ahead into registers; dh, dg and du pass through
// shared memory so that their global accesses are whole 256-byte row pieces.  Bound by its 14
// bytes per element (saved 8, dh 2, dg and du 4).  The first block also sets the tile counter of
// k_gated_bwd.  8192 x 8192: 132 us (without the ring 197; the 671 MB read alone take 103 at 6.54 TB/s,
// the last of the 268 MB written stay in L2); 4096 x 2048: 18 us.
constexpr int kGradCols = 128;
constexpr int kGradPitch = kGradCols + 8;  // 16-bit words: 16-byte accesses of 8 rows on 32 banks
constexpr uint32_t kGradPlane = 32 * kGradCols * 4;
constexpr uint32_t kGradBox = 32 * kGradPitch * 2;
constexpr uint32_t kGradSmem = 2 * 2 * kGradPlane + 3 * kGradBox + 32;

__global__ void __launch_bounds__(256, 2)
    k_gate_grad(const uint16_t* __restrict__ dh, long long lddh, const float* __restrict__ saved,
                uint16_t* __restrict__ dgu, int T, int I, int Ip, int kind, int fmt, int vec, unsigned int* counter,
                unsigned int first_tile, ErrorRecord* err, uint64_t timeout_ns) {
  extern __shared__ __align__(128) uint8_t grad_smem[];
  uint16_t* sd = reinterpret_cast<uint16_t*>(grad_smem + 4 * kGradPlane);
  uint16_t* so = sd + kGradBox / 2;  // dg, then du
  uint64_t* full = reinterpret_cast<uint64_t*>(grad_smem + 4 * kGradPlane + 3 * kGradBox);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(full + 2);
  ptx::griddep_launch();
  if (blockIdx.x == 0 && threadIdx.x == 0) *counter = first_tile;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int cols = saved_cols(I);
  const int tiles_x = (cols + kGradCols - 1) / kGradCols;
  const long long tiles = (long long)tiles_x * ((T + 31) / 32);
  const size_t plane = saved_plane(T, I), out_plane = (size_t)T * Ip;
  if (tid == 0) {
    ptx::mbar_init(&full[0], 1);
    ptx::mbar_init(&full[1], 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
  }
  __syncthreads();
  auto load_saved = [&](long long tile, int stage) {  // by one thread
    const int i0 = (int)(tile % tiles_x) * kGradCols;
    const float* g = saved + saved_at((int)(tile / tiles_x) * 32, i0, I);
    const uint32_t bytes = min(kGradCols, cols - i0) * 128;
    ptx::mbar_arrive_expect_tx(&full[stage], 2 * bytes);
    ptx::bulk_load(grad_smem + stage * 2 * kGradPlane, g, bytes, &full[stage]);
    ptx::bulk_load(grad_smem + (stage * 2 + 1) * kGradPlane, g + plane, bytes, &full[stage]);
  };
  alignas(16) uint16_t pre[16];  // stored in 16-byte pieces
  auto load_dh = [&](long long tile) {
    const int t0 = (int)(tile / tiles_x) * 32, i0 = (int)(tile % tiles_x) * kGradCols;
    const int rows = min(32, T - t0);
    if (vec) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int q = tid + k * 256, r = q / (kGradCols / 8), i = i0 + q % (kGradCols / 8) * 8;
        const uint16_t* p = dh + (size_t)(t0 + r) * lddh + i;
        if (r < rows && i + 8 <= I) {
          *reinterpret_cast<uint4*>(pre + 8 * k) = ptx::ld_v4_nc(p);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) pre[8 * k + e] = r < rows && i + e < I ? p[e] : (uint16_t)0;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int q = tid + k * 256, r = q / kGradCols, i = i0 + q % kGradCols;
        pre[k] = r < rows && i < I ? dh[(size_t)(t0 + r) * lddh + i] : (uint16_t)0;
      }
    }
  };
  long long tile = blockIdx.x;
  if (tile < tiles) {
    if (tid == 0) {
      load_saved(tile, 0);
      if (tile + gridDim.x < tiles) load_saved(tile + gridDim.x, 1);
    }
    load_dh(tile);
  }
  for (int it = 0; tile < tiles; tile += gridDim.x, ++it) {
    const int stage = it & 1;
    const int t0 = (int)(tile / tiles_x) * 32, i0 = (int)(tile % tiles_x) * kGradCols;
    const int rows = min(32, T - t0);
    if (vec) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int q = tid + k * 256;
        *reinterpret_cast<uint4*>(sd + q / (kGradCols / 8) * kGradPitch + q % (kGradCols / 8) * 8) =
            *reinterpret_cast<const uint4*>(pre + 8 * k);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int q = tid + k * 256;
        sd[q / kGradCols * kGradPitch + q % kGradCols] = pre[k];
      }
    }
    if (tile + gridDim.x < tiles) load_dh(tile + gridDim.x);
    if (!ptx::mbar_wait(&full[stage], (it >> 1) & 1, timeout_ns, abort_flag)) {
      if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 0, 0);
      *abort_flag = 1;
    }
    __syncthreads();
    if (*abort_flag) break;
    const int i = i0 + warp * 16;
    if (lane < rows && i < cols) {
      const uint4* gp = reinterpret_cast<const uint4*>(grad_smem + stage * 2 * kGradPlane) + warp * 128 + lane;
      const uint4* dp = reinterpret_cast<const uint4*>(sd + lane * kGradPitch + warp * 16);
      alignas(16) uint16_t d[16];
      *reinterpret_cast<uint4*>(d) = dp[0];
      *reinterpret_cast<uint4*>(d + 8) = dp[1];
      uint32_t og[8], ou[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 gv = gp[32 * j], uv = gp[32 * j + kGradPlane / 16];
        const float g[4] = {__uint_as_float(gv.x), __uint_as_float(gv.y), __uint_as_float(gv.z), __uint_as_float(gv.w)};
        const float u[4] = {__uint_as_float(uv.x), __uint_as_float(uv.y), __uint_as_float(uv.z), __uint_as_float(uv.w)};
        float a[4], e[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float dv = ptx::from_16(d[4 * j + k], fmt);
          float slope;
          a[k] = dv * act::value_grad(g[k], kind, &slope);
          e[k] = dv * u[k] * slope;
        }
        og[2 * j] = ptx::pack_16x2(e[0], e[1], fmt);
        og[2 * j + 1] = ptx::pack_16x2(e[2], e[3], fmt);
        ou[2 * j] = ptx::pack_16x2(a[0], a[1], fmt);
        ou[2 * j + 1] = ptx::pack_16x2(a[2], a[3], fmt);
      }
      uint4* pg = reinterpret_cast<uint4*>(so + lane * kGradPitch + warp * 16);
      uint4* pu = reinterpret_cast<uint4*>(so + kGradBox / 2 + lane * kGradPitch + warp * 16);
      pg[0] = make_uint4(og[0], og[1], og[2], og[3]);
      pg[1] = make_uint4(og[4], og[5], og[6], og[7]);
      pu[0] = make_uint4(ou[0], ou[1], ou[2], ou[3]);
      pu[1] = make_uint4(ou[4], ou[5], ou[6], ou[7]);
    }
    __syncthreads();
    if (tid == 0 && tile + 2 * (long long)gridDim.x < tiles) load_saved(tile + 2 * (long long)gridDim.x, stage);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int q = tid + k * 256, z = q / 512, r = q / (kGradCols / 8) % 32, col = q % (kGradCols / 8) * 8;
      if (r < rows && i0 + col < cols)  // cols <= Ip
        ptx::st_v4(dgu + z * out_plane + (size_t)(t0 + r) * Ip + i0 + col,
                   *reinterpret_cast<const uint4*>(so + z * (kGradBox / 2) + r * kGradPitch + col));
    }
  }
  // An aborted block lets the copies it has issued land before its shared memory goes.
  if (*abort_flag && tid == 0)
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_wait(&full[s], 0, 20000000ull, nullptr);
      ptx::mbar_wait(&full[s], 1, 20000000ull, nullptr);
    }
}

struct BwdMaps {
  CUtensorMap d_rows;  // [2][T][I] dg, du: boxes of 128 rows x 64 columns (A of dx, K-major)
  CUtensorMap d_split; // the same: boxes of as many rows as a split-K tile has
  CUtensorMap d_cols;  // the same: boxes of 64 rows x 64 columns (A of the weight gradients, M-major)
  CUtensorMap w[2];    // Wg, Wu [I][H]: boxes of 64 x 64 (B of dx, N-major)
  CUtensorMap x;       // [T][H]: boxes of 64 x 64 (B of the weight gradients, N-major)
  CUtensorMap dx, dwg, dwu;  // output boxes of 32 x 32
};

// The backward products' tiles on CTA pairs.  TileInfo::aux: 0 dx, 1 dWg, 2 dWu.  Tiles are taken
// in order from a counter: the products' depths differ, and the deeper comes first.  Bound by the
// tensor pipe: 8192 rows, 8192 x 8192 in 2694 us (1632 TFLOP/s), 4096 rows, 7168 x 2048 in 326 us
// (1476); 1001 rows, 2056 x 5461 on 256 x 512 tiles in 121 us, 158 in a fixed order.
template <int NH>
struct BwdSched {
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  static constexpr bool kDynamic = true;
  static constexpr bool kTileAhead = true;
  static constexpr bool kDependent = true;
  unsigned int* counter;
  __device__ int next_tile() const { return (int)atomicAdd(counter, 1u); }
  int T, H, I;
  int nx, nw;              // tiles of dx (0: not wanted here) and of each weight gradient (the same)
  int mx, mw, nn;          // 256-row m-blocks of dx and of a weight gradient; column blocks
  int x_first;             // dx's tiles first
  int group_m;
  int fmt;
  const BwdMaps* maps;
  __host__ __device__ int num_tiles() const { return nx + 2 * nw; }
  __device__ TileInfo tile(int t) const {
    TileInfo ti;
    int mb, nb;
    const bool is_x = x_first ? t < nx : t >= 2 * nw;
    if (is_x) {
      raster(x_first ? t : t - 2 * nw, mx, nn, group_m, mb, nb);
      ti.aux = 0;
      ti.kb1 = 2 * ((I + BK - 1) / BK);
    } else {
      const int w = x_first ? t - nx : t;
      raster(w % nw, mw, nn, group_m, mb, nb);
      ti.aux = 1 + w / nw;
      ti.kb1 = (T + BK - 1) / BK;
    }
    ti.kb0 = 0;
    ti.m0 = mb * 2 * BM;
    ti.n0 = nb * NH * pair::BN2;
    ti.a_row = ti.m0;
    ti.b_row = ti.n0;
    ti.aux2 = 0;
    return ti;
  }
  __device__ bool producer_wait(const TileInfo&, int, uint64_t, volatile int*, ErrorRecord*) const { return true; }
  __device__ void issue_loads_pair(const TileInfo& ti, int kb, int crank, uint8_t* sA, uint8_t* sB, uint32_t bar) const {
    constexpr uint32_t kBox = 64 * BK * 2;
    const int m = ti.a_row + crank * BM;
    const CUtensorMap* b = &maps->x;
    int k = kb * BK;
    if (ti.aux == 0) {
      const int nk = (I + BK - 1) / BK, z = kb >= nk ? 1 : 0;
      k = (kb - z * nk) * BK;
      b = &maps->w[z];
      pair::tma_load_3d_pair(sA, &maps->d_rows, bar, k, m, z);
    } else {
      pair::tma_load_3d_pair(sA, &maps->d_cols, bar, m, k, ti.aux - 1);
      pair::tma_load_3d_pair(sA + kBox, &maps->d_cols, bar, m + 64, k, ti.aux - 1);
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const int n = ti.b_row + h * pair::BN2 + crank * half_n(ti, h) / 2;
      pair::tma_load_2d_pair(sB + 2 * h * kBox, b, bar, n, k);
      pair::tma_load_2d_pair(sB + (2 * h + 1) * kBox, b, bar, n + 64, k);
    }
  }
  __device__ int half_n(const TileInfo& ti, int h) const {
    return max(0, min(pair::BN2, (H - ti.n0 - h * pair::BN2 + 31) / 32 * 32));
  }
  __device__ uint32_t idesc(const TileInfo& ti, int n) const {
    return ptx::idesc_f16_f32(2 * BM, n, fmt, ti.aux != 0, 1);
  }
  __device__ uint64_t a_desc(const TileInfo& ti, uint32_t a, int k) const {
    return ti.aux == 0 ? ptx::sdesc_kmajor_sw128(a + k * 32) : ptx::sdesc_mnmajor_sw128(a + k * 2048, 8192);
  }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const {
    return ptx::sdesc_mnmajor_sw128(b + k * 2048, 8192);
  }
};

struct BwdEpi : Out16Epi {
  static constexpr bool kRowStores = false;  // gradients have 16-byte aligned rows
  int T, I;
  const BwdMaps* maps;
  __device__ void begin_tile(const TileInfo& ti, int) {
    M = ti.aux == 0 ? T : I;
    tmC = ti.aux == 0 ? &maps->dx : ti.aux == 1 ? &maps->dwg : &maps->dwu;
  }
  __device__ bool staged() const { return true; }
};

template <int NH>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<NH>::kThreads, 1)
    k_gated_bwd(const __grid_constant__ BwdMaps maps, BwdSched<NH> sched, BwdEpi epi, ErrorRecord* err,
                uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.maps = &maps;
  pair::gemm_core_pair<NH>(&maps.d_rows, &maps.x, sched, epi, err, timeout_ns, -1);
}

// The same products on the split-K clusters: dx of few rows (over both weights' rows), or small
// weight gradients over many rows.  Bound by the weights' stream: dx of 16 rows, 7168 x 2048 in 15 us
// (pairs 31); by one round of few deep tiles: dW of 8192 rows, 512 x 512 in 22 us (pairs 54).
struct DxSplitOp : split::PlainOp {
  static constexpr int kAccs = 1;
  uint16_t* dx;
  long long lddx;
  int H, I, bn;
  __device__ int depth() const { return 2 * ((I + BK - 1) / BK); }
  // k_gate_grad's results, from here on
  __device__ void start(uint8_t*) { ptx::griddep_wait(); }
  __device__ uint32_t idesc(int n) const { return ptx::idesc_f16_f32(split::kRows, n, type, 0, 1); }
  __device__ uint64_t w_desc(uint32_t w, int k) const { return ptx::sdesc_mnmajor_sw128(w + k * 2048, 8192); }
  __device__ void loads(int kb, int t0, int n0, uint8_t* x, uint8_t* w, uint64_t* bar) const {
    const int nk = (I + BK - 1) / BK, z = kb >= nk ? 1 : 0, k = (kb - z * nk) * BK;
    for (int j = 0; j < bn; j += 64) ptx::tma_load_2d(w + j * BK * 2, tmW + z, bar, n0 + j, k);
    ptx::tma_load_3d(x, tmX, bar, k, t0, z);
  }
  __device__ __forceinline__ void emit(int t, int col, const float (*v)[4]) const {
    split::store4_16(dx + (size_t)t * lddx, col, H, v[0], type, 1);
  }
};
struct DwSplitOp : split::PlainOp {
  static constexpr int kAccs = 1;
  uint16_t *dwg, *dwu;
  long long lddw;
  int T, H, bn, mblocks;
  __device__ int z() const { return (int)blockIdx.y / mblocks; }  // 0 dWg, 1 dWu
  __device__ int depth() const { return (T + BK - 1) / BK; }
  __device__ void start(uint8_t*) { ptx::griddep_wait(); }
  __device__ uint32_t idesc(int n) const { return ptx::idesc_f16_f32(split::kRows, n, type, 1, 1); }
  __device__ uint64_t x_desc(uint32_t x, int k) const { return ptx::sdesc_mnmajor_sw128(x + k * 2048, 8192); }
  __device__ uint64_t w_desc(uint32_t w, int k) const { return ptx::sdesc_mnmajor_sw128(w + k * 2048, 8192); }
  __device__ void loads(int kb, int t0, int n0, uint8_t* x, uint8_t* w, uint64_t* bar) const {
    for (int j = 0; j < bn; j += 64) ptx::tma_load_2d(w + j * BK * 2, tmW, bar, n0 + j, kb * BK);
    ptx::tma_load_3d(x, tmX, bar, t0, kb * BK, z());
    ptx::tma_load_3d(x + 64 * BK * 2, tmX, bar, t0 + 64, kb * BK, z());
  }
  __device__ __forceinline__ void emit(int i, int col, const float (*v)[4]) const {
    split::store4_16((z() ? dwu : dwg) + (size_t)i * lddw, col, H, v[0], type, 1);
  }
};

__global__ void __launch_bounds__(split::kThreads, 1)
    k_gated_dx_split(const __grid_constant__ BwdMaps maps, split::Shape sh, DxSplitOp op, ErrorRecord* err,
                     uint64_t timeout_ns) {
  op.tmX = &maps.d_split;
  op.tmW = maps.w;
  split::split_core(sh, op, err, timeout_ns);
}
__global__ void __launch_bounds__(split::kThreads, 1)
    k_gated_dw_split(const __grid_constant__ BwdMaps maps, split::Shape sh, DwSplitOp op, ErrorRecord* err,
                     uint64_t timeout_ns) {
  op.tmX = &maps.d_cols;
  op.tmW = &maps.x;
  split::split_core(sh, op, err, timeout_ns);
}

namespace {
using split::check_rows;
using split::k16;

CUtensorMap map_128b(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  return make_tmap_2d(p, k16, 2, rows, cols, ld, box_rows, BK, CU_TENSOR_MAP_SWIZZLE_128B);
}
bool vec16(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * 2 & 15) == 0; }
CUtensorMap out_map(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, const CUtensorMap& unused) {
  return vec16(p, (long long)ld) ? make_tmap_2d(p, k16, 2, rows, cols, ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B) : unused;
}
constexpr uint32_t kSmemMax = 227 * 1024;
constexpr int kRingKb = 200;  // the split kernel's ring

template <int NH>
void launch_gated_pair(const GatedMaps& m, const GatedEpi& e, int T, int I, int H, cudaStream_t stream) {
  using Cf = pair::PairCfg<NH>;
  GatedSched<NH> s;
  s.I = I;
  s.H = H;
  s.num_m = (T + 2 * BM - 1) / (2 * BM);
  s.num_n = (I + s.kCols - 1) / s.kCols;
  s.group_m = ops::gemm_tuning().pair_group_m;
  s.fmt = e.fmt;
  s.maps = nullptr;
  static std::atomic<bool> done[64] = {};
  split::allow_smem(k_gated_pair<NH>, Cf::kSmemBytesSwizzled, done);
  const int grid = 2 * std::min(s.num_m * s.num_n, num_sms() / 2);
  k_gated_pair<NH><<<grid, Cf::kThreads, Cf::kSmemBytesSwizzled, stream>>>(m, s, e, device_error_record(),
                                                                         default_timeout_ns());
  GICC_CUDA(cudaGetLastError());
}

template <int NH>
void launch_gated_bwd(const BwdMaps& m, int T, int H, int I, bool need_x, bool need_w, int fmt, unsigned int* counter,
                      uint64_t timeout_ns, cudaStream_t stream) {
  using Cf = pair::PairCfg<NH>;
  BwdSched<NH> s;
  s.counter = counter;
  s.T = T;
  s.H = H;
  s.I = I;
  s.mx = (T + 2 * BM - 1) / (2 * BM);
  s.mw = (I + 2 * BM - 1) / (2 * BM);
  s.nn = (H + NH * pair::BN2 - 1) / (NH * pair::BN2);
  s.nx = need_x ? s.mx * s.nn : 0;
  s.nw = need_w ? s.mw * s.nn : 0;
  s.x_first = 2LL * I >= T;
  s.group_m = ops::gemm_tuning().pair_group_m;
  s.fmt = fmt;
  s.maps = nullptr;
  BwdEpi e;
  e.fmt = fmt;
  e.N = H;
  e.T = T;
  e.I = I;
  e.vec = 1;
  e.maps = nullptr;
  static std::atomic<bool> done[64] = {};
  split::allow_smem(k_gated_bwd<NH>, Cf::kSmemBytesSwizzled, done);
  const int grid = 2 * std::min(s.num_tiles(), num_sms() / 2);
  split::launch_dependent(k_gated_bwd<NH>, dim3(grid), Cf::kThreads, Cf::kSmemBytesSwizzled, stream, m, s, e,
                          device_error_record(), timeout_ns);
}

// Where the backward products run: dx and the weight gradients each on CTA pairs (together, in
// one launch) or on the split-K clusters, by expected time.
struct BwdPlan {
  bool x_split = false, w_split = false;
  int nh = 2;
  split::Plan px, pw;
};
BwdPlan plan_bwd(int T, int H, int I, bool need_x, bool need_w, int tile) {
  const int pairs = num_sms() / 2;
  const int kx = 2 * ((I + BK - 1) / BK), kw = (T + BK - 1) / BK;
  BwdPlan best;
  if (need_x && (tile == 0 || tile == 1))
    best.px = split::plan(T, H, I, 1, kRingKb, reinterpret_cast<const void*>(k_gated_dx_split), 64, 1, kx);
  if (need_w && (tile == 0 || tile == 1))
    best.pw = split::plan(I, H, T, 1, kRingKb, reinterpret_cast<const void*>(k_gated_dw_split), 64, 2, kw,
                          true);
  if (tile) {
    best.x_split = tile == 1 && need_x;
    best.w_split = tile == 1 && need_w;
    best.nh = tile == 3 ? 1 : 2;
    return best;
  }
  // us of the pairs' launch: a tile's k-blocks and what its epilogue costs beside them, shared by
  // the pairs; at the end the last tiles, or the deepest alone
  auto pair_us = [&](int nh, bool x, bool w) {
    if (!x && !w) return 0.0;
    const double nn = std::ceil(H / 32.0) * 32 / (nh * pair::BN2);  // the last column block costs its columns
    const double nx = x ? std::ceil(T / 256.0) * nn : 0, nw = w ? 2 * std::ceil(I / 256.0) * nn : 0;
    const double busy = std::min(1.0, (nx + nw) / pairs), step = nh == 2 ? 0.60 + 0.14 * busy : 0.33 + 0.07 * busy;
    const double cx = step * kx + 2.5 * nh, cw = step * kw + 2.5 * nh;
    const double longest = std::max(nx ? cx : 0.0, nw ? cw : 0.0), last = nx && nw ? std::min(cx, cw) : longest;
    const double even = nx + nw <= pairs ? longest : (nx * cx + nw * cw) / pairs + 0.5 * last;
    return std::max(even, longest) + 8.0;
  };
  double cost = -1;
  for (int nh = 2; nh >= 1; --nh)
    for (int xs = 0; xs <= (need_x && best.px.fits ? 1 : 0); ++xs)
      for (int ws = 0; ws <= (need_w && best.pw.fits ? 1 : 0); ++ws) {
        const double c = pair_us(nh, need_x && !xs, need_w && !ws) + (xs ? 1.25 * best.px.us : 0) +
                         (ws ? 1.25 * best.pw.us : 0);  // measured to estimated, with the launch: 1.1 to 1.4
        if (cost < 0 || c < cost) {
          cost = c;
          best.x_split = xs;
          best.w_split = ws;
          best.nh = nh;
        }
      }
  return best;
}

void check_16(const char* who, int fmt, int kind) {
  if (fmt < 0 || fmt > 1) throw std::runtime_error(std::string(who) + ": fmt must be 0 (f16) or 1 (bf16)");
  if (kind < 0 || kind >= ops::ACT_COUNT) throw std::runtime_error(std::string(who) + ": unknown activation");
}
// saved is written with 16-byte stores and read by bulk copies.
void check_saved(const char* who, const float* saved) {
  if (reinterpret_cast<uintptr_t>(saved) & 15) throw std::runtime_error(std::string(who) + ": saved must be 16-byte aligned");
}
}  // namespace
}  // namespace ffn

namespace ops {

// dg and du, rows of 128-byte multiples; then the tile counter
static int grad_pitch(int I) { return (I + 63) / 64 * 64; }
static size_t grad_counter_at(int T, int I) { return (size_t)2 * T * grad_pitch(I) * 2; }
size_t gated_saved_floats(int T, int I) { return 2 * ffn::saved_plane(T, I); }
size_t gated_grad_bytes(int T, int I) { return grad_counter_at(T, I) + 16; }

int gated_linear_tile(int T, int H, int I) {
  using namespace ffn;
  split::check_dims("gicc::gated_linear_tile", {T, H, I});
  return split::pick_tile(T, I, H, 2, kRingKb, reinterpret_cast<const void*>(k_gated_split));
}

void gated_linear(const void* x, const void* w_gate, const void* w_up, void* h, int T, int H, int I, long long ldx,
                  long long ldg, long long ldu, long long ldh, int kind, int fmt, float* saved, int tile,
                  cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::gated_linear");
  using namespace ffn;
  const char* who = "gicc::gated_linear";
  check_16(who, fmt, kind);
  if (T <= 0 || H <= 0 || I <= 0) throw std::runtime_error("gicc::gated_linear: empty shape");
  split::check_dims(who, {T, H, I});
  if (H % 8) throw std::runtime_error("gicc::gated_linear: H must be a multiple of 8 (16-byte TMA rows)");
  check_rows(who, "x", x, ldx, H);
  check_rows(who, "w_gate", w_gate, ldg, H);
  check_rows(who, "w_up", w_up, ldu, H);
  if (h == nullptr || ldh < I) throw std::runtime_error("gicc::gated_linear: h needs rows of at least I elements");
  check_saved(who, saved);
  if (tile < 0 || tile > 3)
    throw std::runtime_error("gicc::gated_linear: tile must be 0 (by shape), 1 (split), 2 (pairs, 256 x 512) or 3 (pairs, 256 x 256)");
  if (tile == 0) tile = gated_linear_tile(T, H, I);
  if (tile == 1) {
    const split::Plan p = split::plan(T, I, H, 2, kRingKb, reinterpret_cast<const void*>(k_gated_split));
    split::check_fits(who, p);
    GatedSplitOp op;
    op.h = static_cast<uint16_t*>(h);
    op.ldh = ldh;
    op.T = T;
    op.H = H;
    op.I = I;
    op.kind = kind;
    op.type = fmt;
    op.bn = p.sh.bn;
    op.tmX = op.tmW = op.tmU = nullptr;
    op.vec = (reinterpret_cast<uintptr_t>(h) & 7) == 0 && ldh % 4 == 0;
    op.saved = saved;
    static std::atomic<bool> done[64] = {};
    split::allow_smem(k_gated_split, kSmemMax, done);
    split::launch_clusters(k_gated_split, p.grid, p.splits, split::kThreads, p.smem, false, stream,
                           map_128b(x, T, H, ldx, p.sh.xrows), map_128b(w_gate, I, H, ldg, p.sh.bn),
                           map_128b(w_up, I, H, ldu, p.sh.bn), p.sh, op, device_error_record(), default_timeout_ns());
    return;
  }
  GatedMaps m;
  m.x = map_128b(x, T, H, ldx, BM);
  m.g = map_128b(w_gate, I, H, ldg, BM);
  m.u = map_128b(w_up, I, H, ldu, BM);
  m.h = out_map(h, T, I, ldh, m.x);
  GatedEpi e;
  e.C = static_cast<uint16_t*>(h);
  e.ldc = ldh;
  e.M = T;
  e.N = I;
  e.fmt = fmt;
  e.vec = vec16(h, ldh);
  e.kind = kind;
  e.saved = saved;
  if (tile == 2) launch_gated_pair<2>(m, e, T, I, H, stream);
  else launch_gated_pair<1>(m, e, T, I, H, stream);
}

void gated_linear_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const float* saved,
                           void* work, void* dx, void* dw_gate, void* dw_up, int T, int H, int I, long long lddh,
                           long long ldx, long long ldg, long long ldu, long long lddx, long long lddw, int kind, int fmt,
                           int tile, cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::gated_linear_backward");
  using namespace ffn;
  const char* who = "gicc::gated_linear_backward";
  check_16(who, fmt, kind);
  if (T <= 0 || H <= 0 || I <= 0) throw std::runtime_error("gicc::gated_linear_backward: empty shape");
  split::check_dims(who, {T, H, I});
  if (H % 8) throw std::runtime_error("gicc::gated_linear_backward: H must be a multiple of 8 (16-byte TMA rows)");
  check_rows(who, "x", x, ldx, H);
  check_rows(who, "w_gate", w_gate, ldg, H);
  check_rows(who, "w_up", w_up, ldu, H);
  if (dh == nullptr || lddh < I || saved == nullptr || work == nullptr || (reinterpret_cast<uintptr_t>(work) & 15))
    throw std::runtime_error("gicc::gated_linear_backward: dh, saved and a 16-byte aligned work area are needed");
  check_saved(who, saved);
  if ((dw_gate == nullptr) != (dw_up == nullptr))
    throw std::runtime_error("gicc::gated_linear_backward: both weight gradients or none");
  if (tile < 0 || tile > 3)
    throw std::runtime_error("gicc::gated_linear_backward: tile must be 0 (by shape), 1 (split), 2 (pairs, 256 x 512) or 3 (pairs, 256 x 256)");
  if (dx == nullptr && dw_gate == nullptr) return;
  if (dx != nullptr) check_rows(who, "dx", dx, lddx, H);
  if (dw_gate != nullptr) {
    check_rows(who, "dw_gate", dw_gate, lddw, H);
    check_rows(who, "dw_up", dw_up, lddw, H);
  }
  const int Ip = grad_pitch(I);
  const uint64_t timeout_ns = default_timeout_ns();  // reads the environment: once a call
  const BwdPlan plan = plan_bwd(T, H, I, dx != nullptr, dw_gate != nullptr, tile);
  if (plan.x_split) split::check_fits(who, plan.px);
  if (plan.w_split) split::check_fits(who, plan.pw);
  uint16_t* dgu = static_cast<uint16_t*>(work);
  unsigned int* counter = reinterpret_cast<unsigned int*>(static_cast<uint8_t*>(work) + grad_counter_at(T, I));
  const long long gtiles = (long long)((saved_cols(I) + kGradCols - 1) / kGradCols) * ((T + 31) / 32);
  const int ggrid = (int)std::min<long long>(gtiles, 2LL * num_sms());
  static std::atomic<bool> grad_done[64] = {};
  split::allow_smem(k_gate_grad, kGradSmem, grad_done);
  k_gate_grad<<<ggrid, 256, kGradSmem, stream>>>(static_cast<const uint16_t*>(dh), lddh, saved, dgu, T, I, Ip, kind, fmt,
                                                 vec16(dh, lddh) ? 1 : 0, counter, (unsigned)(num_sms() / 2),
                                                 device_error_record(), timeout_ns);
  GICC_CUDA(cudaGetLastError());

  BwdMaps m;
  m.d_rows = make_tmap_3d(dgu, k16, 2, 2, T, I, Ip, (uint64_t)T * Ip, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.d_cols = make_tmap_3d(dgu, k16, 2, 2, T, I, Ip, (uint64_t)T * Ip, 64, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.w[0] = map_128b(w_gate, I, H, ldg, 64);
  m.w[1] = map_128b(w_up, I, H, ldu, 64);
  m.x = map_128b(x, T, H, ldx, 64);
  m.dx = dx ? out_map(dx, T, H, lddx, m.x) : m.x;
  m.dwg = dw_gate ? out_map(dw_gate, I, H, lddw, m.x) : m.x;
  m.dwu = dw_up ? out_map(dw_up, I, H, lddw, m.x) : m.x;
  m.d_split = plan.x_split ? make_tmap_3d(dgu, k16, 2, 2, T, I, Ip, (uint64_t)T * Ip, plan.px.sh.xrows, BK,
                                          CU_TENSOR_MAP_SWIZZLE_128B)
                           : m.d_rows;
  const bool pair_x = dx != nullptr && !plan.x_split, pair_w = dw_gate != nullptr && !plan.w_split;
  if (pair_x || pair_w) {
    if (plan.nh == 2) launch_gated_bwd<2>(m, T, H, I, pair_x, pair_w, fmt, counter, timeout_ns, stream);
    else launch_gated_bwd<1>(m, T, H, I, pair_x, pair_w, fmt, counter, timeout_ns, stream);
  }
  if (plan.x_split) {
    DxSplitOp op;
    op.type = fmt;
    op.tmX = op.tmW = nullptr;
    op.dx = static_cast<uint16_t*>(dx);
    op.lddx = lddx;
    op.H = H;
    op.I = I;
    op.bn = plan.px.sh.bn;
    static std::atomic<bool> done[64] = {};
    split::allow_smem(k_gated_dx_split, kSmemMax, done);
    split::launch_clusters(k_gated_dx_split, plan.px.grid, plan.px.splits, split::kThreads, plan.px.smem, true, stream, m,
                           plan.px.sh, op, device_error_record(), timeout_ns);
  }
  if (plan.w_split) {
    DwSplitOp op;
    op.type = fmt;
    op.tmX = op.tmW = nullptr;
    op.dwg = static_cast<uint16_t*>(dw_gate);
    op.dwu = static_cast<uint16_t*>(dw_up);
    op.lddw = lddw;
    op.T = T;
    op.H = H;
    op.bn = plan.pw.sh.bn;
    op.mblocks = plan.pw.sh.mblocks;
    static std::atomic<bool> done[64] = {};
    split::allow_smem(k_gated_dw_split, kSmemMax, done);
    split::launch_clusters(k_gated_dw_split, plan.pw.grid, plan.pw.splits, split::kThreads, plan.pw.smem, true, stream, m,
                           plan.pw.sh, op, device_error_record(), timeout_ns);
  }
}

}  // namespace ops
}  // namespace gicc

static_assert(GICC_ACT_SILU == gicc::ops::ACT_SILU && GICC_ACT_GELU == gicc::ops::ACT_GELU &&
                  GICC_ACT_GELU_TANH == gicc::ops::ACT_GELU_TANH,
              "activations");
GICC_API size_t gicc_gated_saved_floats(int T, int I) {
  return T > 0 && I > 0 && std::max(T, I) <= gicc::gemm::split::kMaxDim ? gicc::ops::gated_saved_floats(T, I) : 0;
}
GICC_API size_t gicc_gated_grad_bytes(int T, int I) {
  return T > 0 && I > 0 && std::max(T, I) <= gicc::gemm::split::kMaxDim ? gicc::ops::gated_grad_bytes(T, I) : 0;
}
GICC_API int gicc_gated_linear(const void* x, const void* w_gate, const void* w_up, void* h, int T, int H, int I,
                               long long ldx, long long ldg, long long ldu, long long ldh, int kind, int fmt, float* saved,
                               cudaStream_t stream) {
  return gicc::guarded([&] {
    gicc::ops::gated_linear(x, w_gate, w_up, h, T, H, I, ldx, ldg, ldu, ldh, kind, fmt, saved, 0, stream);
  });
}
GICC_API int gicc_gated_linear_backward(const void* dh, const void* x, const void* w_gate, const void* w_up,
                                        const float* saved, void* work, void* dx, void* dw_gate, void* dw_up, int T, int H,
                                        int I, long long lddh, long long ldx, long long ldg, long long ldu, long long lddx,
                                        long long lddw, int kind, int fmt, cudaStream_t stream) {
  return gicc::guarded([&] {
    gicc::ops::gated_linear_backward(dh, x, w_gate, w_up, saved, work, dx, dw_gate, dw_up, T, H, I, lddh, ldx, ldg, ldu,
                                     lddx, lddw, kind, fmt, 0, stream);
  });
}
