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
// term.  A tile pays one k-block (64 deep) per adapter it meets, r <= 64.
//
// Few rows: the split-K cluster core (k_lora_split); it starts while k_lora_down still runs and
// waits for v only before its adapter blocks.  Many rows: the CTA-pair core (k_lora_pair), whose
// lists of adapters per 256-row tile k_lora_down writes to the work area.
#include <algorithm>
#include <cuda.h>
#include <cuda_runtime.h>

#include "gicc/config.hpp"
#include "gicc/device/adapter_lanes.cuh"
#include "gicc/device/gemm_core2.cuh"
#include "gicc/device/out16_epi.cuh"
#include "gicc/device/split_host.cuh"
#include "gicc/host_util.hpp"
#include "gicc/ops.hpp"

namespace gicc {
namespace lora {

using namespace gemm;

constexpr int kMaxRank = 128;
constexpr int kPairRows = 2 * BM;  // rows of a pair tile

// Per 256-row tile: how many adapters, which, and the lanes that each leaves alone.
struct TileLists {
  int* count = nullptr;      // [tiles]
  int* list = nullptr;       // [tiles][cap]
  uint32_t* skip = nullptr;  // [tiles][cap][8]
  int cap = 0;               // min(L, 256)
};

// ---- v = s A x ---------------------------------------------------------------------------------
// Grid (S, G, ceil(T / 128)): a cluster of S CTAs splits K for one 128-row tile and the adapters
// i with i % G == blockIdx.y of the tile's list (one group when there are many tiles).  Bound by
// reading x and the used A[a] once; the MMAs (128 x r per k-block) are small beside that.
struct DownArgs {
  const int* adapter;
  const float* scale;
  uint16_t* v;
  int T, K, L, r;
  int rp;      // r rounded up to 16: columns of the MMA
  int xrows;   // rows of an x box
  int groups;
  int stages;
  int fmt;
  TileLists lists;  // count null: not wanted
};

// With its lists this leaves room for a k_lora_split CTA on the same SM.
constexpr uint32_t kDownRing = 80 * 1024;
__host__ __device__ constexpr uint32_t down_stage(int rp) { return split::kXBytes + rp * BK * 2; }
__host__ __device__ constexpr uint32_t down_ring(int rp, int stages) {
  const uint32_t ring = stages * down_stage(rp), part = split::kRows * split::pitch(1, rp) * 4;
  return ((ring > part ? ring : part) + 127) / 128 * 128;
}
struct DownLists {
  LaneLists<split::kRows> tile;
  LaneLists<kPairRows> pair;  // shared memory only where the pair lists are wanted
};

__global__ void __launch_bounds__(split::kThreads)
    k_lora_down(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, DownArgs p,
                ErrorRecord* err, uint64_t timeout_ns) {
  extern __shared__ uint8_t down_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(down_smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = p.stages;
  const uint32_t abytes = p.rp * BK * 2;
  uint8_t* sX = smem;
  uint8_t* sA = smem + stages * split::kXBytes;
  uint8_t* after = smem + down_ring(p.rp, stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(after);
  uint64_t* empty = full + split::kMaxStages;
  uint64_t* tfull = empty + split::kMaxStages;
  uint64_t* drain = tfull + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  DownLists& lists = *reinterpret_cast<DownLists*>(after + split::kBarBytes);
  float* part = reinterpret_cast<float*>(smem);

  const uint32_t warp = ptx::warp_id();
  const uint32_t lane = ptx::lane_id();
  const int S = (int)split::cluster_size();
  const int c = (int)pair::cta_rank();
  const int g = blockIdx.y;
  const int t0 = (int)blockIdx.z * split::kRows;
  const int rows = min(split::kRows, p.T - t0);
  const uint32_t ncols = split::tmem_cols(p.rp);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    ptx::mbar_init(tfull, 1);
    ptx::mbar_init(drain, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tmap(&tmX);
    ptx::prefetch_tmap(&tmA);
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, ncols);
    ptx::tmem_relinquish();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  // The projection may start now: every CTA of this grid that runs holds its TMEM already.
  ptx::griddep_launch();
  const uint32_t tmem = *tmem_slot;
  // One CTA per tile reports indexes out of range.
  lists.tile.build(p.adapter, t0, p.T, p.L, g == 0 && c == 0 ? err : nullptr);
  const int n = lists.tile.n;
  if (p.lists.count != nullptr && g == 0 && c == 0 && (blockIdx.z & 1) == 0) {
    // the list of the 256-row tile that starts here, for the CTA-pair projection
    const int tile = blockIdx.z >> 1;
    lists.pair.build(p.adapter, t0, p.T, p.L, nullptr);
    const int m = lists.pair.n;  // <= min(L, 256) = cap
    for (int i = threadIdx.x; i < m; i += blockDim.x) p.lists.list[(size_t)tile * p.lists.cap + i] = lists.pair.list[i];
    for (int i = threadIdx.x; i < m * 8; i += blockDim.x)
      p.lists.skip[(size_t)tile * p.lists.cap * 8 + i] = lists.pair.skip[0][i];
    if (threadIdx.x == 0) p.lists.count[tile] = m;
  }
  const int nkb = (p.K + BK - 1) / BK;
  const int kb0 = (int)((long long)nkb * c / S), nk = (int)((long long)nkb * (c + 1) / S) - kb0;
  const int mine = n > g ? (n - g + p.groups - 1) / p.groups : 0;
  const int steps = mine * nk;  // adapter-major; 0: no row of this tile is this cluster's

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t tx = p.xrows * BK * 2 + abytes;
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      for (int i = 0; i < steps; ++i) {
        if (!ptx::mbar_wait(&empty[stage], phase ^ 1, timeout_ns, abort_flag)) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 0, 0);
          *abort_flag = 1;
          break;
        }
        const int j = i / nk, kx = (kb0 + i - j * nk) * BK;
        ptx::mbar_arrive_expect_tx(&full[stage], tx);
        ptx::tma_load_2d(sX + stage * split::kXBytes, &tmX, &full[stage], kx, t0);
        ptx::tma_load_3d(sA + stage * abytes, &tmA, &full[stage], kx, 0, lists.tile.list[g + j * p.groups]);
        issued = i + 1;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (*abort_flag) {
        for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
          ptx::mbar_wait(&full[i % stages], (i / stages) & 1, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && steps > 0) {
      const uint32_t idesc = ptx::idesc_f16_f32(split::kRows, p.rp, p.fmt, 0, 0);
      int stage = 0;
      uint32_t phase = 0;
      int i = 0;
      for (; i < steps; ++i) {
        if (!ptx::mbar_wait(&full[stage], phase, timeout_ns, abort_flag)) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 2, 0);
          *abort_flag = 1;
          break;
        }
        ptx::tc_fence_after();
        const int j = i / nk;
        const uint32_t* skip = lists.tile.skip[g + j * p.groups];
        const uint32_t x = ptx::smem_u32(sX + stage * split::kXBytes), a = ptx::smem_u32(sA + stage * abytes);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k)
          ptx::mma_f16_ss_lanes(tmem, ptx::sdesc_kmajor_sw128(x + k * 32), ptx::sdesc_kmajor_sw128(a + k * 32), idesc,
                                (i - j * nk > 0 || k > 0) ? 1u : 0u, skip);
        ptx::mma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (i == steps) {
        ptx::mma_commit(tfull);
      } else if (i > 0) {
        ptx::mma_commit(drain);
        ptx::mbar_wait(drain, 0, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else if (steps > 0) {
    const int q = warp & 3;
    const int row = q * 32 + (int)lane;
    if (!ptx::mbar_wait_long(tfull, 0, timeout_ns, abort_flag)) {
      if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 3, 0);
      *abort_flag = 1;
    } else if (q * 32 < rows) {
      ptx::tc_fence_after();
      const uint32_t tbase = tmem + (static_cast<uint32_t>(q * 32) << 16);
      float* dst = part + row * split::pitch(1, p.rp);
      for (int col = 0; col < p.rp; col += 16) {
        uint32_t r[16];
        ptx::tmem_ld16(tbase + col, r);
        ptx::tmem_ld_wait();
        if (row < rows) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4*>(dst + col + 4 * j) = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
      }
    }
    __syncwarp();
  }
  ptx::tc_fence_before();
  __syncthreads();
  pair::cluster_sync();
  if (steps > 0 && !*abort_flag) {
    const int g4 = p.r / 4;
    const int items = rows * g4;
    const uint32_t base = ptx::smem_u32(part);
    const int j1 = (int)((long long)items * (c + 1) / S);
    for (int j = (int)((long long)items * c / S) + (int)threadIdx.x; j < j1; j += split::kThreads) {
      const int row = j / g4, col = (j - row * g4) * 4;
      const int a = LaneLists<split::kRows>::at(p.adapter, t0 + row, p.T, p.L);
      if (a < 0 || lists.tile.slot(a) % p.groups != g) continue;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      const uint32_t off = base + (row * split::pitch(1, p.rp) + col) * 4;
      for (int s = 0; s < S; ++s) {
        const float4 q = split::ld_cluster_f4(pair::map_to(off, s));
        sum.x += q.x;
        sum.y += q.y;
        sum.z += q.z;
        sum.w += q.w;
      }
      const float sc = p.scale[a];
      const float o[4] = {sc * sum.x, sc * sum.y, sc * sum.z, sc * sum.w};
      split::store4_16(p.v + (size_t)(t0 + row) * p.r, col, p.r, o, p.fmt, 1);
    }
  }
  pair::cluster_sync();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, ncols);
  }
}

// ---- the projection for few rows ---------------------------------------------------------------
struct LoraSplitOp {
  static constexpr int kAccs = 1;
  const int* adapter;
  uint16_t* y;
  long long ldy;
  int T, N, L, r, rc;  // rc: k-blocks of 64 per adapter
  int type, vec, bn;
  const CUtensorMap* tmV;  // set by the kernel
  const CUtensorMap* tmB;
  const LaneLists<split::kRows>* lists;
  __device__ int fmt() const { return type; }
  __device__ void prepare(uint8_t* smem, int t0, ErrorRecord*) {
    auto* l = reinterpret_cast<LaneLists<split::kRows>*>(smem);
    l->build(adapter, t0, T, L, nullptr);  // k_lora_down reports indexes out of range
    lists = l;
  }
  __device__ void extra_blocks(int c, int S, int& e0, int& e1) const {
    const int n = lists->n * rc;
    e0 = n * c / S;
    e1 = n * (c + 1) / S;
  }
  __device__ void extra_wait() const { ptx::griddep_wait(); }
  __device__ void extra_loads(int e, int t0, int n0, void* sX, void* sW, uint64_t* bar) const {
    const int s = e / rc, k = (e - s * rc) * BK;
    ptx::tma_load_2d(sX, tmV, bar, k, t0);
    ptx::tma_load_3d(sW, tmB, bar, k, n0, lists->list[s]);
  }
  __device__ void extra_mma(int e, uint32_t d, uint32_t x, uint32_t w, uint32_t idesc) const {
    const int s = e / rc, left = r - (e - s * rc) * BK;
    for (int k = 0; k < BK / 16 && k * 16 < left; ++k)
      ptx::mma_f16_ss_lanes(d, ptx::sdesc_kmajor_sw128(x + k * 32), ptx::sdesc_kmajor_sw128(w + k * 32), idesc, 1u,
                            lists->skip[s]);
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
  op.tmV = &tmV;
  op.tmB = &tmB;
  split::split_core(&tmX, &tmW, &tmW, sh, op, err, timeout_ns);
}

// ---- the projection on CTA pairs ---------------------------------------------------------------
struct LoraMaps {
  CUtensorMap x, w, v, b, y;
};

struct LoraSched {
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  int T, N, K, rc;
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
    ti.n0 = nb * 2 * pair::BN2;
    ti.a_row = ti.m0;
    ti.b_row = ti.n0;
    ti.kb0 = 0;
    ti.kb1 = weight_blocks() + __ldg(lists.count + mb) * rc;
    ti.aux = mb * lists.cap;
    ti.aux2 = 0;
    return ti;
  }
  __device__ bool producer_wait(const TileInfo&, int, uint64_t, volatile int*, ErrorRecord*) const { return true; }
  __device__ void issue_loads_pair(const TileInfo& ti, int kb, int crank, uint8_t* sA, uint8_t* sB, uint32_t bar) const {
    const int m = ti.a_row + crank * BM, n = ti.b_row + crank * BM;
    const int e = kb - weight_blocks();
    if (e < 0) {
      pair::tma_load_2d_pair(sA, &maps->x, bar, kb * BK, m);
      pair::tma_load_2d_pair(sB, &maps->w, bar, kb * BK, n);
      pair::tma_load_2d_pair(sB + pair::kBBytes, &maps->w, bar, kb * BK, n + pair::BN2);
    } else {
      const int s = e / rc, k = (e - s * rc) * BK;
      const int a = __ldg(lists.list + ti.aux + s);
      pair::tma_load_2d_pair(sA, &maps->v, bar, k, m);
      pair::tma_load_3d_pair(sB, &maps->b, bar, k, n, a);
      pair::tma_load_3d_pair(sB + pair::kBBytes, &maps->b, bar, k, n + pair::BN2, a);
    }
  }
  __device__ uint32_t idesc(const TileInfo&) const { return ptx::idesc_f16_f32(2 * BM, pair::BN2, fmt, 0, 0); }
  __device__ uint64_t a_desc(const TileInfo&, uint32_t a, int k) const { return ptx::sdesc_kmajor_sw128(a + k * 32); }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const { return ptx::sdesc_kmajor_sw128(b + k * 32); }
  __device__ bool lane_skip(const TileInfo& ti, int kb, uint32_t* skip) const {
    const int e = kb - weight_blocks();
    if (e < 0) return false;
    const uint4* p = reinterpret_cast<const uint4*>(lists.skip + (size_t)(ti.aux + e / rc) * 8);
    const uint4 a = __ldg(p), b = __ldg(p + 1);
    skip[0] = a.x;
    skip[1] = a.y;
    skip[2] = a.z;
    skip[3] = a.w;
    skip[4] = b.x;
    skip[5] = b.y;
    skip[6] = b.z;
    skip[7] = b.w;
    return true;
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<2>::kThreads, 1)
    k_lora_pair(const __grid_constant__ LoraMaps maps, LoraSched sched, Out16Epi epi, ErrorRecord* err,
                uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.tmC = &maps.y;
  pair::gemm_core_pair<2>(&maps.x, &maps.w, sched, epi, err, timeout_ns, -1);
}

namespace {
constexpr CUtensorMapDataType k16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;  // 16-bit words (f16 too: TMA moves bits)

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
void check_rows(const char* name, const void* p, long long ld, int cols) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15) || ld % 8 || ld < cols)
    throw std::runtime_error(std::string("gicc::lora_linear: ") + name +
                             " needs 16-byte aligned rows (base and pitch) of at least " + std::to_string(cols) + " elements");
}
template <class K>
void allow_smem(K kernel, uint32_t bytes, bool* done) {
  int dev = 0;
  GICC_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && done[dev]) return;
  GICC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done[dev] = true;
}
}  // namespace
}  // namespace lora

namespace ops {

size_t lora_work_bytes(int T, int L, int r) { return lora::work_layout(T, L, r).bytes; }

void lora_linear(const void* x, const void* w, const void* lora_a, const void* lora_b, const int* adapter,
                 const float* scale, void* y, void* work, int T, int K, int N, int L, int r, long long ldx, long long ldw,
                 long long ldy, int fmt, int tile, cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::lora_linear");
  using namespace lora;
  if (fmt < 0 || fmt > 1) throw std::runtime_error("gicc::lora_linear: fmt must be 0 (f16) or 1 (bf16)");
  if (T <= 0 || K <= 0 || N <= 0 || L <= 0 || r <= 0) throw std::runtime_error("gicc::lora_linear: empty shape");
  if (K % 8 || r % 8) throw std::runtime_error("gicc::lora_linear: K and r must be multiples of 8 (16-byte TMA rows)");
  if (r > kMaxRank || L > kMaxAdapters) throw std::runtime_error("gicc::lora_linear: r <= 128 and L <= 8192");
  check_rows("x", x, ldx, K);
  check_rows("w", w, ldw, K);
  check_rows("lora_a", lora_a, K, K);
  check_rows("lora_b", lora_b, r, r);
  check_rows("work", work, 8, 8);
  if (y == nullptr || ldy < N || adapter == nullptr || scale == nullptr)
    throw std::runtime_error("gicc::lora_linear: y needs rows of at least N elements; adapter and scale are needed");
  if (tile < 0 || tile > 2) throw std::runtime_error("gicc::lora_linear: tile must be 0 (by shape), 1 (split) or 2 (pairs)");
  if (tile == 0) tile = T <= 256 ? 1 : 2;

  const Work lay = work_layout(T, L, r);
  uint8_t* base = static_cast<uint8_t*>(work);
  const int sms = num_sms();
  const int tiles = (T + split::kRows - 1) / split::kRows;
  const int nkb = (K + BK - 1) / BK;
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
  if (tile == 2) {
    d.lists.count = reinterpret_cast<int*>(base + lay.count);
    d.lists.list = reinterpret_cast<int*>(base + lay.list);
    d.lists.skip = reinterpret_cast<uint32_t*>(base + lay.skip);
    d.lists.cap = lay.cap;
  }
  // Split K over clusters until about two CTAs per SM work; with few tiles, spread the tiles'
  // adapters (as many as there may be) over further clusters too.
  int S = 1;
  while (S < split::kMaxSplit && S * 2 <= nkb && tiles * S < 2 * sms) S *= 2;
  d.groups = std::max(1, std::min(std::min(L, std::min(T, split::kRows)), sms / (tiles * S)));
  d.stages = std::max(2, std::min<int>(split::kMaxStages, kDownRing / down_stage(d.rp)));
  const uint32_t dsmem = 1024 + down_ring(d.rp, d.stages) + split::kBarBytes +
                         (tile == 2 ? sizeof(DownLists) : sizeof(LaneLists<split::kRows>));
  static bool done_down[64] = {false};
  allow_smem(k_lora_down, 227 * 1024, done_down);
  const CUtensorMap tA = make_tmap_3d(lora_a, k16, 2, L, r, K, K, (uint64_t)r * K, d.rp, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  split::launch_clusters(k_lora_down, dim3(S, d.groups, tiles), S, split::kThreads, dsmem, false, stream,
                         make_tmap_2d(x, k16, 2, T, K, ldx, d.xrows, BK, CU_TENSOR_MAP_SWIZZLE_128B), tA, d,
                         device_error_record(), default_timeout_ns());

  const int rc = (r + BK - 1) / BK;
  if (tile == 1) {
    const split::Plan p = split::plan(T, N, K, 1, sizeof(LaneLists<split::kRows>));
    LoraSplitOp op;
    op.adapter = adapter;
    op.y = static_cast<uint16_t*>(y);
    op.ldy = ldy;
    op.T = T;
    op.N = N;
    op.L = L;
    op.r = r;
    op.rc = rc;
    op.type = fmt;
    op.vec = (reinterpret_cast<uintptr_t>(y) & 7) == 0 && ldy % 4 == 0;
    op.bn = p.sh.bn;
    op.tmV = op.tmB = nullptr;
    op.lists = nullptr;
    static bool done[64] = {false};
    allow_smem(k_lora_split, 227 * 1024, done);
    split::launch_clusters(
        k_lora_split, p.grid, p.splits, split::kThreads, p.smem, true, stream,
        make_tmap_2d(x, k16, 2, T, K, ldx, p.sh.xrows, BK, CU_TENSOR_MAP_SWIZZLE_128B),
        make_tmap_2d(w, k16, 2, N, K, ldw, p.sh.bn, BK, CU_TENSOR_MAP_SWIZZLE_128B),
        make_tmap_2d(d.v, k16, 2, T, r, r, p.sh.xrows, BK, CU_TENSOR_MAP_SWIZZLE_128B),
        make_tmap_3d(lora_b, k16, 2, L, N, r, r, (uint64_t)N * r, p.sh.bn, BK, CU_TENSOR_MAP_SWIZZLE_128B), p.sh, op,
        device_error_record(), default_timeout_ns());
    return;
  }
  using Cf = pair::PairCfg<2>;
  LoraMaps m;
  m.x = make_tmap_2d(x, k16, 2, T, K, ldx, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.w = make_tmap_2d(w, k16, 2, N, K, ldw, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.v = make_tmap_2d(d.v, k16, 2, T, r, r, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.b = make_tmap_3d(lora_b, k16, 2, L, N, r, r, (uint64_t)N * r, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  Out16Epi e;
  e.C = static_cast<uint16_t*>(y);
  e.ldc = ldy;
  e.M = T;
  e.N = N;
  e.fmt = fmt;
  e.vec = (reinterpret_cast<uintptr_t>(y) & 15) == 0 && ldy % 8 == 0;
  m.y = e.vec ? make_tmap_2d(y, k16, 2, T, N, ldy, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE) : m.x;
  LoraSched s;
  s.T = T;
  s.N = N;
  s.K = K;
  s.rc = rc;
  s.num_m = (T + kPairRows - 1) / kPairRows;
  s.num_n = (N + Cf::kCols - 1) / Cf::kCols;
  s.group_m = gemm_tuning().pair_group_m;
  s.fmt = fmt;
  s.lists = d.lists;
  s.maps = nullptr;
  static bool done[64] = {false};
  allow_smem(k_lora_pair, Cf::kSmemBytesStaged, done);
  const int grid = 2 * std::min(s.num_m * s.num_n, sms / 2);
  k_lora_pair<<<grid, Cf::kThreads, Cf::kSmemBytesStaged, stream>>>(m, s, e, device_error_record(), default_timeout_ns());
  GICC_CUDA(cudaGetLastError());
}

}  // namespace ops
}  // namespace gicc
