// lora.cu -- a shared projection with the low-rank adapters of many requests.
//
//   y[t] = W x[t] + s[a] B[a] (A[a] x[t]),  a = adapter[t], -1: none
//
// x [T, K], W [N, K], A [L, r, K], B [L, N, r], y [T, N], bf16 or f16, f32 accumulation.
//
// Two kernels.  k_lora_down computes v[t] = s[a] A[a] x[t] ([T, r]); the projection then treats
// each adapter that a tile's rows use as further k-blocks behind the weight's: A operand v,
// B operand B[a], accumulated into the same TMEM accumulator, with the MMA's lane mask keeping
// every adapter to its own rows (adapter_lanes.cuh).  So rows keep their order, the product
// with B[a] costs no pass of its own over y, and a row without an adapter gets W x alone.
// v is rounded to 16 bits, as an MMA operand must be; it enters y only through the adapter's
// term.  A k-block holds 64 / w pieces of w = 16, 32 or 64 columns (the largest that divides r),
// each a piece of one adapter of the tile, with the swizzle of its width: pieces as wide as r,
// because TMA fills the missing columns of a wider box slowly (1.7 us a block at r = 16 in boxes
// of 64 columns, against 0.7 us at r = 64).
//
// Few rows: the split-K cluster core (k_lora_split); it starts while k_lora_down still runs and
// waits for v only before its adapter blocks.  Many rows: the CTA-pair core (k_lora_pair), whose
// lists of adapters per 256-row tile k_lora_down writes to the work area.
//
// Host entry points: gicc::ops::lora_linear (C++, throws) and gicc_lora_linear (C ABI,
// gicc/projections.h).
#include <algorithm>
#include <cstddef>
#include <cuda.h>
#include <cuda_runtime.h>

#include "gicc/config.hpp"
#include "gicc/device/adapter_lanes.cuh"
#include "gicc/device/gemm_core2.cuh"
#include "gicc/device/out16_epi.cuh"
#include "gicc/device/split_host.cuh"
#include "gicc/host_util.hpp"
#include "gicc/ops.hpp"
#include "gicc/projections.h"

namespace gicc {
namespace lora {

using namespace gemm;

constexpr int kMaxRank = 128;
constexpr int kMaxRows = 65535 * split::kRows;  // grid.z of k_lora_down
constexpr int kPairRows = 2 * BM;  // rows of a pair tile

// Per 256-row tile: how many adapters, which, and the lanes that each leaves alone.
struct TileLists {
  int* count = nullptr;      // [tiles]
  int* list = nullptr;       // [tiles][cap]
  uint32_t* skip = nullptr;  // [tiles][cap][8]
  int cap = 0;               // min(L, 256)
};

// How an adapter's r columns are cut into pieces of one width, and those into k-blocks.
struct Pieces {
  int w;      // columns of a piece: 64, 32 or 16
  int each;   // pieces of an adapter
  int block;  // pieces in a k-block
  __host__ __device__ int blocks(int adapters) const { return (adapters * each + block - 1) / block; }
};
inline Pieces pieces(int r) {
  Pieces p;
  p.w = r % 64 == 0 ? 64 : r % 32 == 0 ? 32 : 16;
  p.each = (r + p.w - 1) / p.w;
  p.block = BK / p.w;
  return p;
}
inline CUtensorMapSwizzle piece_swizzle(const Pieces& p) {
  return p.w == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : p.w == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B;
}

// ---- v = s A x ---------------------------------------------------------------------------------
// Grid (S, G, ceil(T / 128)): a cluster of S CTAs splits K for one 128-row tile and the adapters
// i with i % G == blockIdx.y of the tile's list (one group when there are many tiles).  The
// group's adapters go through the MMA side by side, `cap` at a time (128 columns: one MMA per
// k-step for all of them, and x is loaded once for all), into two TMEM accumulators in turn; a
// TMEM reader thread owns a row and keeps the columns of that row's adapter in registers.
// Bound by reading x and the used A[a]; the MMAs are small beside that.  8192 x 8192, r 64, 11
// adapters in 40 us (x alone 20 at 6.5 TB/s); one row, K 4096 in 9.5 us, most of it latency.
struct DownArgs {
  const int* adapter;
  const float* scale;
  uint16_t* v;
  int T, K, L, r;
  int rp;      // r rounded up to 16: columns of one adapter
  int cap;     // adapters side by side
  int xrows;   // rows of an x box
  int groups;
  int stages;
  int fmt;
  TileLists lists;  // count null: not wanted
};

constexpr int kDownCols = 128;  // columns of an accumulator
// Beside a k_lora_split CTA's ring both fit an SM.
constexpr uint32_t kDownRing = 92 * 1024;
constexpr uint32_t kDownMin = 227 * 512;  // with 1 KB of the system's each, two do not fit
__host__ __device__ constexpr uint32_t down_stage(int xrows, int cols) { return split::x_bytes(xrows) + cols * BK * 2; }
// as split::ring_bytes: the MMA reads 128 rows from the last x box on
__host__ __device__ constexpr uint32_t down_ring(int rp, int cols, int xrows, int stages) {
  uint32_t ring = stages * down_stage(xrows, cols);
  const uint32_t reach = (stages - 1) * split::x_bytes(xrows) + split::kRows * BK * 2;
  const uint32_t part = split::kRows * split::pitch(1, rp) * 4;
  if (reach > ring) ring = reach;
  return ((ring > part ? ring : part) + 127) / 128 * 128;
}
constexpr uint32_t kDownBar = (2 * split::kMaxStages + 5) * 8 + 8;
struct DownLists {
  LaneLists<split::kRows, false> tile;
  float row_scale[split::kRows];     // of the row's adapter
  signed char mine[split::kRows];    // the row's adapter is of this CTA's group
  alignas(16) LaneLists<kPairRows> pair;  // shared memory only where the pair lists are wanted
};

__global__ void __launch_bounds__(split::kThreads)
    k_lora_down(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, DownArgs p,
                ErrorRecord* err, uint64_t timeout_ns) {
  extern __shared__ uint8_t down_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(down_smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.stages, cap = p.cap;
  const uint32_t xb = split::x_bytes(p.xrows), ab = p.rp * BK * 2;  // one x box, one adapter's box
  uint8_t* sX = smem;
  uint8_t* sA = smem + stages * xb;
  uint8_t* after = smem + down_ring(p.rp, cap * p.rp, p.xrows, stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(after);
  uint64_t* empty = full + split::kMaxStages;
  uint64_t* tfull = empty + split::kMaxStages;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  DownLists& lists = *reinterpret_cast<DownLists*>(after + (kDownBar + 15) / 16 * 16);
  float* part = reinterpret_cast<float*>(smem);

  const uint32_t warp = ptx::warp_id();
  const uint32_t lane = ptx::lane_id();
  const int S = (int)split::cluster_size();
  const int c = (int)pair::cta_rank();
  const int g = blockIdx.y;
  const int t0 = (int)blockIdx.z * split::kRows;
  const int rows = min(split::kRows, p.T - t0);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(&tfull[a], 1);
      ptx::mbar_init(&tempty[a], 4);
    }
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmX);
    ptx::prefetch_tmap(&tmA);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 2 * kDownCols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // The projection may start now: every CTA of this grid that runs holds its TMEM already.
  ptx::griddep_launch();
  const uint32_t tmem = *tmem_slot;
  // One CTA per tile reports indexes out of range.
  lists.tile.build(p.adapter, t0, p.T, p.L, g == 0 && c == 0 ? err : nullptr, (int)threadIdx.x, split::kThreads);
  const int nkb = (p.K + BK - 1) / BK;
  const int kb0 = (int)((long long)nkb * c / S), nk = (int)((long long)nkb * (c + 1) / S) - kb0;
  const int n = lists.tile.n;
  const int mine = n > g ? (n - g + p.groups - 1) / p.groups : 0;  // adapters of this group
  const int passes = (mine + cap - 1) / cap;  // 0: no row of this tile is this cluster's

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int ps = 0; ps < passes && !*abort_flag; ++ps) {
        const int na = min(cap, mine - ps * cap);
        for (int k = 0; k < nk; ++k) {
          if (!ptx::mbar_wait(&empty[stage], phase ^ 1, timeout_ns, abort_flag)) {
            if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 0, 0);
            *abort_flag = 1;
            break;
          }
          ptx::mbar_arrive_expect_tx(&full[stage], xb + na * ab);
          ptx::tma_load_2d(sX + stage * xb, &tmX, &full[stage], (kb0 + k) * BK, t0);
          for (int j = 0; j < na; ++j)
            ptx::tma_load_3d(sA + (stage * cap + j) * ab, &tmA, &full[stage], (kb0 + k) * BK, 0,
                             lists.tile.list[g + (ps * cap + j) * p.groups]);
          ++issued;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (*abort_flag) {
        for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
          ptx::mbar_wait(&full[i % stages], (i / stages) & 1, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool issued = false;
      for (int ps = 0; ps < passes && !*abort_flag; ++ps) {
        const int acc = ps & 1, na = min(cap, mine - ps * cap);
        const uint32_t idesc = ptx::idesc_f16_f32(split::kRows, na * p.rp, p.fmt, 0, 0);
        bool ok = ptx::mbar_wait(&tempty[acc], ((ps >> 1) & 1) ^ 1, timeout_ns, abort_flag);
        for (int k = 0; ok && k < nk; ++k) {
          ok = ptx::mbar_wait(&full[stage], phase, timeout_ns, abort_flag);
          if (!ok) break;
          ptx::tc_fence_after();
          const uint32_t x = ptx::smem_u32(sX + stage * xb), a = ptx::smem_u32(sA + stage * cap * ab);
#pragma unroll
          for (int q = 0; q < BK / 16; ++q)
            ptx::mma_f16_ss(tmem + acc * kDownCols, ptx::sdesc_kmajor_sw128(x + q * 32),
                            ptx::sdesc_kmajor_sw128(a + q * 32), idesc, (k > 0 || q > 0) ? 1u : 0u);
          issued = true;
          ptx::mma_commit(&empty[stage]);
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 2, 0);
          *abort_flag = 1;
          break;
        }
        ptx::mma_commit(&tfull[acc]);
      }
      if (*abort_flag && issued) {
        ptx::mma_commit(drain);
        ptx::mbar_wait(drain, 0, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int row = q * 32 + (int)lane;
    // this row's adapter: which pass computes it, and where among the pass's columns
    int my = -1;
    if (row < rows) {
      const int a = p.adapter[t0 + row];
      if (a >= 0 && a < p.L) {
        const int s = lists.tile.slot(a);
        if (s % p.groups == g) {
          my = s / p.groups;
          lists.row_scale[row] = p.scale != nullptr ? p.scale[a] : 1.0f;
        }
      }
    }
    lists.mine[row] = my >= 0;
    float v[kMaxRank];
#pragma unroll
    for (int i = 0; i < kMaxRank; ++i) v[i] = 0.f;
    for (int ps = 0; ps < passes; ++ps) {
      const int acc = ps & 1, na = min(cap, mine - ps * cap);
      if (!ptx::mbar_wait_long(&tfull[acc], (ps >> 1) & 1, timeout_ns, abort_flag)) {
        if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 3, 0);
        *abort_flag = 1;
        break;
      }
      ptx::tc_fence_after();
      const uint32_t tbase = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * kDownCols;
      for (int j = 0; j < na; ++j) {
        const bool is_mine = my == ps * cap + j;
        if (!__any_sync(0xffffffffu, is_mine)) continue;
#pragma unroll
        for (int ch = 0; ch < kMaxRank / 16; ++ch) {
          if (ch * 16 >= p.rp) break;
          uint32_t r[16];
          ptx::tmem_ld16(tbase + j * p.rp + ch * 16, r);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (is_mine) v[ch * 16 + i] = __uint_as_float(r[i]);
        }
      }
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(&tempty[acc]);
    }
    // Every MMA has read its operands (the last pass's barrier), so the ring takes the partial.
    if (my >= 0 && !*abort_flag) {
      float* dst = part + row * split::pitch(1, p.rp);
#pragma unroll
      for (int ch = 0; ch < kMaxRank / 4; ++ch) {
        if (ch * 4 >= p.rp) break;
        *reinterpret_cast<float4*>(dst + ch * 4) = make_float4(v[ch * 4], v[ch * 4 + 1], v[ch * 4 + 2], v[ch * 4 + 3]);
      }
    }
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (p.lists.count != nullptr && g == 0 && c == 0 && (blockIdx.z & 1) == 0) {
    // the list of the 256-row tile that starts here, for the CTA-pair projection
    const int tile = blockIdx.z >> 1;
    lists.pair.build(p.adapter, t0, p.T, p.L, nullptr, (int)threadIdx.x, split::kThreads);
    const int m = lists.pair.n;  // <= min(L, 256) = cap
    for (int i = threadIdx.x; i < m; i += blockDim.x) p.lists.list[(size_t)tile * p.lists.cap + i] = lists.pair.list[i];
    for (int i = threadIdx.x; i < m * 8; i += blockDim.x)
      p.lists.skip[(size_t)tile * p.lists.cap * 8 + i] = lists.pair.skip[0][i];
    if (threadIdx.x == 0) p.lists.count[tile] = m;
  }
  pair::cluster_sync();
  if (passes > 0 && !*abort_flag) {
    const int g4 = p.r / 4;
    const int items = rows * g4;
    const uint32_t base = ptx::smem_u32(part);
    const int j1 = (int)((long long)items * (c + 1) / S);
    for (int j = (int)((long long)items * c / S) + (int)threadIdx.x; j < j1; j += split::kThreads) {
      const int row = j / g4, col = (j - row * g4) * 4;
      if (!lists.mine[row]) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t off = base + (row * split::pitch(1, p.rp) + col) * 4;
      for (int s = 0; s < S; ++s) {
        const float4 q = split::ld_cluster_f4(pair::map_to(off, s));
        sum.x += q.x;
        sum.y += q.y;
        sum.z += q.z;
        sum.w += q.w;
      }
      const float sc = lists.row_scale[row];
      const float o[4] = {sc * sum.x, sc * sum.y, sc * sum.z, sc * sum.w};
      split::store4_16(p.v + (size_t)(t0 + row) * p.r, col, p.r, o, p.fmt, 1);
    }
  }
  pair::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, 2 * kDownCols);
  }
}

// ---- the projection for few rows ---------------------------------------------------------------
// Bound by W's stream, then by the latency from v to y.  One row, K = N = 4096: 16.4 us a call with
// k_lora_down (the pairs 41); 64 rows with 64 adapters of rank 16, K 7168: 28.7 us (the pairs 86),
// 21 of them W alone.
struct LoraSplitOp : split::PlainOp {
  static constexpr int kAccs = 1;
  const int* adapter;
  uint16_t* y;
  long long ldy;
  int T, N, K, L;
  Pieces pc;
  int vec;
  uint32_t xpiece, wpiece;  // bytes of a piece of v and of B
  const CUtensorMap* tmV;  // set by the kernel
  const CUtensorMap* tmB;
  LaneLists<split::kRows>* lists;
  __device__ int depth() const { return (K + BK - 1) / BK; }
  uint8_t* sV;  // the tile's rows of v, piece by piece, loaded once: every CTA of the grid reads them
  static constexpr bool kExtra = true;
  __device__ void start(uint8_t* smem) {
    sV = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) & ~uintptr_t(1023));
    lists = reinterpret_cast<LaneLists<split::kRows>*>(sV + v_bytes());
  }
  __device__ void prepare(int t0, int tid) {
    lists->build(adapter, t0, T, L, nullptr, tid, 128);  // k_lora_down reports indexes out of range
  }
  // The MMA reads 128 rows of the last piece too; its rows behind the box are the lists.
  __host__ __device__ uint32_t v_bytes() const { return pc.each * xpiece; }
  __host__ static uint32_t extra_smem(const Pieces& pc, int xrows) {
    return 1024 + std::max<uint32_t>(pc.each * xrows * pc.w * 2 + sizeof(LaneLists<split::kRows>),
                                     (pc.each - 1) * xrows * pc.w * 2 + split::kRows * pc.w * 2);
  }
  __device__ void extra_blocks(int c, int S, int& e0, int& e1) const {
    const int n = pc.blocks(lists->n);
    e0 = n * c / S;
    e1 = n * (c + 1) / S;
  }
  __device__ void extra_shared(int t0, uint64_t* bar) const {
    ptx::griddep_wait();
    ptx::mbar_arrive_expect_tx(bar, v_bytes());
    for (int i = 0; i < pc.each; ++i) ptx::tma_load_2d(sV + i * xpiece, tmV, bar, i * pc.w, t0);
  }
  __device__ void extra_loads(int e, int n0, uint8_t* sW, uint64_t* bar) const {
    for (int j = 0; j < pc.block; ++j) {
      // behind the last piece the last once more: every k-block has the same bytes
      const int s = min(e * pc.block + j, lists->n * pc.each - 1), i = s / pc.each, k = (s - i * pc.each) * pc.w;
      ptx::tma_load_3d(sW + j * wpiece, tmB, bar, k, n0, lists->list[i]);
    }
  }
  // Unrolled for each width: the issuing thread is what bounds these short MMAs.
  template <int W>
  __device__ __forceinline__ void piece_mma(int e, uint32_t d, uint32_t w, uint32_t idesc) const {
    const int left = lists->n * pc.each - e * (BK / W);
    const uint64_t v0 = ptx::sdesc_kmajor(ptx::smem_u32(sV), W * 2), w0 = ptx::sdesc_kmajor(w, W * 2);
#pragma unroll
    for (int j = 0; j < BK / W; ++j) {
      if (j >= left) break;
      const int s = e * (BK / W) + j, i = pc.each == 1 ? s : s / pc.each, part = s - i * pc.each;
      const uint4 m = *reinterpret_cast<const uint4*>(lists->skip[i]);
      const uint32_t skip[4] = {m.x, m.y, m.z, m.w};
      const uint64_t vd = v0 + ((part * xpiece) >> 4), wd = w0 + ((j * wpiece) >> 4);  // start addresses, 16 bytes
#pragma unroll
      for (int k = 0; k < W / 16; ++k) ptx::mma_f16_ss_lanes(d, vd + 2 * k, wd + 2 * k, idesc, 1u, skip);
    }
  }
  __device__ void extra_mma(int e, uint32_t d, uint32_t w, uint32_t idesc) const {
    if (pc.w == 16) piece_mma<16>(e, d, w, idesc);
    else if (pc.w == 32) piece_mma<32>(e, d, w, idesc);
    else piece_mma<64>(e, d, w, idesc);
  }
  __device__ __forceinline__ void emit(int t, int col, const float (*v)[4]) const {
    split::store4_16(y + (size_t)t * ldy, col, N, v[0], type, vec);
  }
  // The next kernel of the stream may reuse what k_lora_down writes: end after it.
  __device__ void finish() const { ptx::griddep_wait(); }
};

__global__ void __launch_bounds__(split::kThreads, 1)
    k_lora_split(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                 const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmB, split::Shape sh,
                 LoraSplitOp op, ErrorRecord* err, uint64_t timeout_ns) {
  op.tmX = &tmX;
  op.tmW = &tmW;
  op.tmV = &tmV;
  op.tmB = &tmB;
  split::split_core(sh, op, err, timeout_ns);
}

// ---- the projection on CTA pairs ---------------------------------------------------------------
// Bound by the tensor pipe: 8192^3 in 678 us without adapters (the plain GEMM 680), 4096 rows of 256
// requests, K 7168, r 16 in 197 us against 164 without (five adapter k-blocks a tile, the wait for
// k_lora_down).
struct LoraMaps {
  CUtensorMap x, w, v, b, y;
};

template <int NH>
struct LoraSched {
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  static constexpr bool kLanes = true;
  static constexpr bool kDependent = true;
  int N, K;
  Pieces pc;
  int num_m, num_n, group_m;
  int fmt;
  TileLists lists;
  const LoraMaps* maps;
  __device__ int num_tiles() const { return num_m * num_n; }
  __device__ int weight_blocks() const { return (K + BK - 1) / BK; }
  __device__ TileInfo tile(int t) const {
    int mb, nb;
    raster(t, num_m, num_n, group_m, mb, nb);
    TileInfo ti;
    ti.m0 = mb * kPairRows;
    ti.n0 = nb * NH * pair::BN2;
    ti.a_row = ti.m0;
    ti.b_row = ti.n0;
    ti.kb0 = 0;
    const int n = (int)ptx::ld_cg(lists.count + mb);
    ti.kb1 = weight_blocks() + pc.blocks(n);
    ti.aux = mb * lists.cap;
    ti.aux2 = n * pc.each;  // pieces
    return ti;
  }
  __device__ bool producer_wait(const TileInfo&, int, uint64_t, volatile int*, ErrorRecord*) const { return true; }
  __device__ void issue_loads_pair(const TileInfo& ti, int kb, int crank, uint8_t* sA, uint8_t* sB, uint32_t bar) const {
    const int m = ti.a_row + crank * BM;
    const int n = ti.b_row + crank * half_n(ti, 0) / 2, n1 = ti.b_row + pair::BN2 + crank * half_n(ti, 1) / 2;
    const int e = kb - weight_blocks();
    if (e < 0) {
      pair::tma_load_2d_pair(sA, &maps->x, bar, kb * BK, m);
      pair::tma_load_2d_pair(sB, &maps->w, bar, kb * BK, n);
      if constexpr (NH == 2) pair::tma_load_2d_pair(sB + pair::kBBytes, &maps->w, bar, kb * BK, n1);
    } else {
      const uint32_t bytes = BM * pc.w * 2;
      for (int j = 0; j < pc.block; ++j) {
        const int s = min(e * pc.block + j, ti.aux2 - 1), i = s / pc.each, k = (s - i * pc.each) * pc.w;
        const int a = (int)ptx::ld_cg(lists.list + ti.aux + i);
        pair::tma_load_2d_pair(sA + j * bytes, &maps->v, bar, k, m);
        pair::tma_load_3d_pair(sB + j * bytes, &maps->b, bar, k, n, a);
        if constexpr (NH == 2) pair::tma_load_3d_pair(sB + pair::kBBytes + j * bytes, &maps->b, bar, k, n1, a);
      }
    }
  }
  __device__ int half_n(const TileInfo& ti, int h) const {
    return max(0, min(pair::BN2, (N - ti.n0 - h * pair::BN2 + 31) / 32 * 32));
  }
  __device__ uint32_t idesc(const TileInfo&, int n) const { return ptx::idesc_f16_f32(2 * BM, n, fmt, 0, 0); }
  __device__ uint64_t a_desc(const TileInfo&, uint32_t a, int k) const { return ptx::sdesc_kmajor_sw128(a + k * 32); }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const { return ptx::sdesc_kmajor_sw128(b + k * 32); }
  __device__ int lane_skip(const TileInfo& ti, int kb, uint32_t (*skip)[8]) const {
    const int e = kb - weight_blocks();
    if (e < 0) return -1;
    const int steps = pc.w / 16;  // k-steps of a piece
    const int n = min(pc.block, ti.aux2 - e * pc.block) * steps;
#pragma unroll
    for (int k = 0; k < BK / 16; ++k) {
      const int s = min(e * pc.block + k / steps, ti.aux2 - 1);
      const uint4* p = reinterpret_cast<const uint4*>(lists.skip + (size_t)(ti.aux + s / pc.each) * 8);
      const uint4 a = ptx::ld_v4_cg(p), b = ptx::ld_v4_cg(p + 1);
      skip[k][0] = a.x;
      skip[k][1] = a.y;
      skip[k][2] = a.z;
      skip[k][3] = a.w;
      skip[k][4] = b.x;
      skip[k][5] = b.y;
      skip[k][6] = b.z;
      skip[k][7] = b.w;
    }
    return n;
  }
  __device__ uint64_t piece_desc(uint32_t addr, int k) const {
    const int steps = pc.w / 16, j = k / steps;
    return ptx::sdesc_kmajor(addr + j * BM * pc.w * 2 + (k - j * steps) * 32, pc.w * 2);
  }
  __device__ uint64_t lane_a_desc(uint32_t a, int k) const { return piece_desc(a, k); }
  __device__ uint64_t lane_b_desc(uint32_t b, int k) const { return piece_desc(b, k); }
};

template <int NH>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<NH>::kThreads, 1)
    k_lora_pair(const __grid_constant__ LoraMaps maps, LoraSched<NH> sched, Out16Epi epi, ErrorRecord* err,
                uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.tmC = &maps.y;
  pair::gemm_core_pair<NH>(&maps.x, &maps.w, sched, epi, err, timeout_ns, -1);
}

namespace {
using split::k16;

struct Work {
  size_t v, count, list, skip, bytes;
  int cap;
};
Work work_layout(int T, int L, int r) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  const size_t tiles = (size_t)(T + kPairRows - 1) / kPairRows;
  Work w;
  w.cap = std::min(L, kPairRows);
  w.v = 0;
  w.count = up((size_t)T * r * 2);
  w.list = w.count + up(tiles * 4);
  w.skip = w.list + up(tiles * w.cap * 4);
  w.bytes = w.skip + up(tiles * w.cap * 32);
  return w;
}
// k_lora_split's ring: with v and the lists it leaves room for a k_lora_down CTA on the same SM.
int ring_kb(int T, int r) { return 104 - (std::min(split::kRows, (T + 7) / 8 * 8) * ((r + 15) / 16 * 16) * 2 + 1023) / 1024; }

template <int NH>
void launch_pair(const LoraMaps& m, const Out16Epi& e, int T, int N, int K, const Pieces& pc, const TileLists& lists,
                 uint64_t timeout_ns, cudaStream_t stream) {
  using Cf = pair::PairCfg<NH>;
  LoraSched<NH> s;
  s.N = N;
  s.K = K;
  s.pc = pc;
  s.num_m = (T + kPairRows - 1) / kPairRows;
  s.num_n = (N + Cf::kCols - 1) / Cf::kCols;
  s.group_m = ops::gemm_tuning().pair_group_m;
  s.fmt = e.fmt;
  s.lists = lists;
  s.maps = nullptr;
  static std::atomic<bool> done[64] = {};
  split::allow_smem(k_lora_pair<NH>, Cf::kSmemBytesSwizzled, done);
  const int grid = 2 * std::min(s.num_m * s.num_n, num_sms() / 2);
  split::launch_dependent(k_lora_pair<NH>, dim3(grid), Cf::kThreads, Cf::kSmemBytesSwizzled, stream, m, s, e,
                          device_error_record(), timeout_ns);
}
}  // namespace
}  // namespace lora

namespace ops {

size_t lora_work_bytes(int T, int L, int r) { return lora::work_layout(T, L, r).bytes; }

int lora_linear_tile(int T, int K, int N, int r) {
  using namespace lora;  // the pairs have k_lora_down in front of them
  split::check_dims("gicc::lora_linear_tile", {T, K, N, r});
  return split::pick_tile(T, N, K, 1, ring_kb(T, r), reinterpret_cast<const void*>(k_lora_split),
                          6.0 + 0.15 * ((K + BK - 1) / BK) + (double)T * K * 2 / 9.0e6);
}

void lora_linear(const void* x, const void* w, const void* lora_a, const void* lora_b, const int* adapter,
                 const float* scale, void* y, void* work, int T, int K, int N, int L, int r, long long ldx, long long ldw,
                 long long ldy, int fmt, int tile, cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::lora_linear");
  using namespace lora;
  const char* who = "gicc::lora_linear";
  if (fmt < 0 || fmt > 1) throw std::runtime_error("gicc::lora_linear: fmt must be 0 (f16) or 1 (bf16)");
  if (T <= 0 || K <= 0 || N <= 0 || L <= 0 || r <= 0) throw std::runtime_error("gicc::lora_linear: empty shape");
  split::check_dims(who, {T, K, N});
  if (K % 8 || r % 8) throw std::runtime_error("gicc::lora_linear: K and r must be multiples of 8 (16-byte TMA rows)");
  if (r > kMaxRank || L > kMaxAdapters) throw std::runtime_error("gicc::lora_linear: r <= 128 and L <= 8192");
  split::check_rows(who, "x", x, ldx, K);
  split::check_rows(who, "w", w, ldw, K);
  split::check_rows(who, "lora_a", lora_a, K, K);
  split::check_rows(who, "lora_b", lora_b, r, r);
  split::check_rows(who, "work", work, 8, 8);
  if (y == nullptr || ldy < N || adapter == nullptr)
    throw std::runtime_error("gicc::lora_linear: y needs rows of at least N elements, and adapter is needed");
  if (T > kMaxRows) throw std::runtime_error("gicc::lora_linear: at most " + std::to_string(kMaxRows) + " rows");
  if (tile < 0 || tile > 3)
    throw std::runtime_error("gicc::lora_linear: tile must be 0 (by shape), 1 (split), 2 (pairs, 256 x 512) or 3 (pairs, 256 x 256)");
  const int nkb = (K + BK - 1) / BK;
  if (tile == 0) tile = lora_linear_tile(T, K, N, r);

  const Work lay = work_layout(T, L, r);
  const uint64_t timeout_ns = default_timeout_ns();  // reads the environment: once a call
  uint8_t* base = static_cast<uint8_t*>(work);
  const int sms = num_sms();
  const int tiles = (T + split::kRows - 1) / split::kRows;
  DownArgs d;
  d.adapter = adapter;
  d.scale = scale;
  d.v = reinterpret_cast<uint16_t*>(base + lay.v);
  d.T = T;
  d.K = K;
  d.L = L;
  d.r = r;
  d.rp = (r + 15) / 16 * 16;
  d.xrows = std::min(split::kRows, (T + 7) / 8 * 8);
  d.fmt = fmt;
  if (tile != 1) {
    d.lists.count = reinterpret_cast<int*>(base + lay.count);
    d.lists.list = reinterpret_cast<int*>(base + lay.list);
    d.lists.skip = reinterpret_cast<uint32_t*>(base + lay.skip);
    d.lists.cap = lay.cap;
  }
  // Many tiles: one CTA per SM with a deep ring (k_lora_pair starts afterwards).  Few: smaller
  // CTAs, so that k_lora_split's fit beside them, the tiles' adapters (as many as there may be)
  // spread over further clusters.
  const int most = std::min(L, std::min(T, split::kRows));
  const uint32_t ring = tile == 1 ? kDownRing : 2 * kDownRing;
  int S = 1;
  while (S < 4 && S + 1 <= nkb && tiles * (S + 1) <= sms) ++S;
  if (tiles == 1 && nkb >= 2 * split::kMaxSplit) S = split::kMaxSplit;
  d.groups = std::max(1, std::min(most, split::clusters_at_once(reinterpret_cast<const void*>(k_lora_down), S) / tiles));
  d.cap = std::max(1, std::min(kDownCols / d.rp, (most + d.groups - 1) / d.groups));
  d.stages = std::max(2, std::min<int>(split::kMaxStages, ring / down_stage(d.xrows, d.cap * d.rp)));
  // More than half of an SM's at least: two of these CTAs on one SM would keep k_lora_split's off it.
  const uint32_t dsmem = std::max<uint32_t>(kDownMin, 1024 + down_ring(d.rp, d.cap * d.rp, d.xrows, d.stages) +
                                                          (kDownBar + 15) / 16 * 16 +
                                                          (tile != 1 ? sizeof(DownLists) : offsetof(DownLists, pair)));
  static std::atomic<bool> done_down[64] = {};
  split::allow_smem(k_lora_down, 227 * 1024, done_down, true);
  const CUtensorMap tA = make_tmap_3d(lora_a, k16, 2, L, r, K, K, (uint64_t)r * K, d.rp, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  split::launch_clusters(k_lora_down, dim3(S, d.groups, tiles), S, split::kThreads, dsmem, false, stream,
                         make_tmap_2d(x, k16, 2, T, K, ldx, d.xrows, BK, CU_TENSOR_MAP_SWIZZLE_128B), tA, d,
                         device_error_record(), timeout_ns);

  const Pieces pc = pieces(r);
  if (tile == 1) {
    split::Plan p = split::plan(T, N, K, 1, ring_kb(T, r), reinterpret_cast<const void*>(k_lora_split));
    p.smem += LoraSplitOp::extra_smem(pc, p.sh.xrows);
    LoraSplitOp op;
    op.adapter = adapter;
    op.y = static_cast<uint16_t*>(y);
    op.ldy = ldy;
    op.T = T;
    op.N = N;
    op.K = K;
    op.L = L;
    op.pc = pc;
    op.xpiece = p.sh.xrows * pc.w * 2;
    op.wpiece = p.sh.bn * pc.w * 2;
    op.type = fmt;
    op.vec = (reinterpret_cast<uintptr_t>(y) & 7) == 0 && ldy % 4 == 0;
    op.tmX = op.tmW = op.tmV = op.tmB = nullptr;
    op.lists = nullptr;
    op.sV = nullptr;
    static std::atomic<bool> done[64] = {};
    split::allow_smem(k_lora_split, 227 * 1024, done, true);
    split::launch_clusters(
        k_lora_split, p.grid, p.splits, split::kThreads, p.smem, true, stream,
        make_tmap_2d(x, k16, 2, T, K, ldx, p.sh.xrows, BK, CU_TENSOR_MAP_SWIZZLE_128B),
        make_tmap_2d(w, k16, 2, N, K, ldw, p.sh.bn, BK, CU_TENSOR_MAP_SWIZZLE_128B),
        make_tmap_2d(d.v, k16, 2, T, r, r, p.sh.xrows, pc.w, piece_swizzle(pc)),
        make_tmap_3d(lora_b, k16, 2, L, N, r, r, (uint64_t)N * r, p.sh.bn, pc.w, piece_swizzle(pc)), p.sh, op,
        device_error_record(), timeout_ns);
    return;
  }
  LoraMaps m;
  m.x = make_tmap_2d(x, k16, 2, T, K, ldx, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.w = make_tmap_2d(w, k16, 2, N, K, ldw, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.v = make_tmap_2d(d.v, k16, 2, T, r, r, BM, pc.w, piece_swizzle(pc));
  m.b = make_tmap_3d(lora_b, k16, 2, L, N, r, r, (uint64_t)N * r, BM, pc.w, piece_swizzle(pc));
  Out16Epi e;
  e.C = static_cast<uint16_t*>(y);
  e.ldc = ldy;
  e.M = T;
  e.N = N;
  e.fmt = fmt;
  e.vec = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && ldy % 8 == 0;
  m.y = e.vec ? make_tmap_2d(y, k16, 2, T, N, ldy, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B) : m.x;
  if (tile == 2) launch_pair<2>(m, e, T, N, K, pc, d.lists, timeout_ns, stream);
  else launch_pair<1>(m, e, T, N, K, pc, d.lists, timeout_ns, stream);
}

}  // namespace ops
}  // namespace gicc

GICC_API size_t gicc_lora_work_bytes(int T, int L, int r) {
  const bool ok = T > 0 && T <= gicc::lora::kMaxRows && L > 0 && L <= gicc::lora::kMaxAdapters && r > 0 &&
                  r <= gicc::lora::kMaxRank;
  return ok ? gicc::ops::lora_work_bytes(T, L, r) : 0;
}
GICC_API int gicc_lora_linear(const void* x, const void* w, const void* lora_a, const void* lora_b, const int* adapter,
                              const float* scale, void* y, void* work, int T, int K, int N, int L, int r, long long ldx,
                              long long ldw, long long ldy, int fmt, cudaStream_t stream) {
  return gicc::guarded([&] {
    gicc::ops::lora_linear(x, w, lora_a, lora_b, adapter, scale, y, work, T, K, N, L, r, ldx, ldw, ldy, fmt, 0, stream);
  });
}
