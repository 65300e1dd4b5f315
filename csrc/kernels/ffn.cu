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
// leaves one partly filled last wave instead of two.
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
struct GatedMaps {
  CUtensorMap x, g, u, h;
};

struct GatedSched {
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  int T, I, H;
  int num_m, num_n, group_m;
  int fmt;
  const GatedMaps* maps;  // set by the kernel
  __device__ int num_tiles() const { return num_m * num_n; }
  __device__ TileInfo tile(int t) const {
    int mb, nb;
    raster(t, num_m, num_n, group_m, mb, nb);
    TileInfo ti;
    ti.m0 = mb * 2 * BM;
    ti.n0 = nb * pair::BN2;
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
    pair::tma_load_2d_pair(sB, &maps->g, bar, kb * BK, ti.b_row + crank * BM);
    pair::tma_load_2d_pair(sB + pair::kBBytes, &maps->u, bar, kb * BK, ti.b_row + crank * BM);
  }
  __device__ uint32_t idesc(const TileInfo&) const { return ptx::idesc_f16_f32(2 * BM, pair::BN2, fmt, 0, 0); }
  __device__ uint64_t a_desc(const TileInfo&, uint32_t a, int k) const { return ptx::sdesc_kmajor_sw128(a + k * 32); }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const { return ptx::sdesc_kmajor_sw128(b + k * 32); }
  __device__ bool lane_skip(const TileInfo&, int, uint32_t*) const { return false; }
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
    if (kind == ops::ACT_SILU) combine<ops::ACT_SILU>(lo, hi);
    else if (kind == ops::ACT_GELU) combine<ops::ACT_GELU>(lo, hi);
    else combine<ops::ACT_GELU_TANH>(lo, hi);
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<2>::kThreads, 1)
    k_gated_pair(const __grid_constant__ GatedMaps maps, GatedSched sched, GatedEpi epi, ErrorRecord* err,
                 uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.tmC = &maps.h;
  pair::gemm_core_pair<2>(&maps.x, &maps.g, sched, epi, err, timeout_ns, -1);
}

// ---- forward for few rows ------------------------------------------------------------------
struct GatedSplitOp {
  static constexpr int kAccs = 2;
  uint16_t* h;
  long long ldh;
  int T, I, kind, type, vec;
  float* saved;
  __device__ int fmt() const { return type; }
  __device__ void prepare(uint8_t*, int, ErrorRecord*) {}
  __device__ void extra_blocks(int, int, int& e0, int& e1) const { e0 = e1 = 0; }
  __device__ void extra_wait() const {}
  __device__ void extra_loads(int, int, int, void*, void*, uint64_t*) const {}
  __device__ void extra_mma(int, uint32_t, uint32_t, uint32_t, uint32_t) const {}
  __device__ void finish() const {}
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
  split::split_core(&tmX, &tmG, &tmU, sh, op, err, timeout_ns);
}

// ---- backward ------------------------------------------------------------------------------
// One warp per 32 rows x 16 columns: a lane is a row (as in the saved layout), so g and u come
// as 512-byte warp loads and dh, dg and du as whole 32-byte sectors of a row.
__global__ void __launch_bounds__(256)
    k_gate_grad(const uint16_t* __restrict__ dh, long long lddh, const float* __restrict__ saved,
                uint16_t* __restrict__ dgu, int T, int I, int Ip, int kind, int fmt, int vec) {
  const int cb = saved_cols(I) / 16;
  const long long blocks = (long long)((T + 31) / 32) * cb;
  const int lane = threadIdx.x & 31;
  const size_t plane = saved_plane(T, I), out_plane = (size_t)T * Ip;
  for (long long b = (long long)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; b < blocks;
       b += (long long)gridDim.x * (blockDim.x / 32)) {
    const int t = (int)(b / cb) * 32 + lane, i = (int)(b % cb) * 16;
    if (t >= T) continue;
    const uint16_t* dp = dh + (size_t)t * lddh + i;
    uint16_t d[16];
    if (vec && i + 16 <= I) {
      *reinterpret_cast<uint4*>(d) = ptx::ld_v4_nc(dp);
      *reinterpret_cast<uint4*>(d + 8) = ptx::ld_v4_nc(dp + 8);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) d[j] = i + j < I ? dp[j] : (uint16_t)0;
    }
    const float* gp = saved + saved_at(t, i, I);
    uint32_t og[8], ou[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 gv = ptx::ld_v4_nc(gp + 128 * j), uv = ptx::ld_v4_nc(gp + plane + 128 * j);
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
    uint16_t* p = dgu + (size_t)t * Ip + i;  // Ip % 64 == 0: the row holds all 16 columns
    ptx::st_v4(p, make_uint4(og[0], og[1], og[2], og[3]));
    ptx::st_v4(p + 8, make_uint4(og[4], og[5], og[6], og[7]));
    ptx::st_v4(p + out_plane, make_uint4(ou[0], ou[1], ou[2], ou[3]));
    ptx::st_v4(p + out_plane + 8, make_uint4(ou[4], ou[5], ou[6], ou[7]));
  }
}

struct BwdMaps {
  CUtensorMap d_rows;  // [2][T][I] dg, du: boxes of 128 rows x 64 columns (A of dx, K-major)
  CUtensorMap d_cols;  // the same: boxes of 64 rows x 64 columns (A of the weight gradients, M-major)
  CUtensorMap wg, wu;  // [I][H]: boxes of 64 x 64 (B of dx, N-major)
  CUtensorMap x;       // [T][H]: boxes of 64 x 64 (B of the weight gradients, N-major)
  CUtensorMap dx, dwg, dwu;  // output boxes of 32 x 32
};

// TileInfo::aux: 0 dx, 1 dWg, 2 dWu.
struct BwdSched {
  static constexpr int kCommWarps = 0;
  static constexpr bool kOwnOperands = true;
  int T, H, I;
  int nx, nw;              // tiles of dx (0: not wanted) and of each weight gradient (0: not wanted)
  int mx, mw, nn;          // 256-row m-blocks of dx and of a weight gradient; 512-column n-blocks
  int x_first;             // dx's tiles first (the deeper product first, for a short last wave)
  int group_m;
  int fmt;
  const BwdMaps* maps;
  __device__ int num_tiles() const { return nx + 2 * nw; }
  __device__ TileInfo tile(int t) const {
    TileInfo ti;
    int mb, nb;
    const bool is_x = x_first ? t < nx : t >= 2 * nw;
    ti.kb0 = 0;
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
    ti.m0 = mb * 2 * BM;
    ti.n0 = nb * 2 * pair::BN2;
    ti.a_row = ti.m0;
    ti.b_row = ti.n0;
    ti.aux2 = 0;
    return ti;
  }
  __device__ bool producer_wait(const TileInfo&, int, uint64_t, volatile int*, ErrorRecord*) const { return true; }
  __device__ void issue_loads_pair(const TileInfo& ti, int kb, int crank, uint8_t* sA, uint8_t* sB, uint32_t bar) const {
    constexpr uint32_t kBox = 64 * BK * 2;
    const int m = ti.a_row + crank * BM, n = ti.b_row + crank * BM;
    const CUtensorMap* b = &maps->x;
    int k = kb * BK;
    if (ti.aux == 0) {
      const int nk = (I + BK - 1) / BK, z = kb >= nk ? 1 : 0;
      k = (kb - z * nk) * BK;
      b = z ? &maps->wu : &maps->wg;
      pair::tma_load_3d_pair(sA, &maps->d_rows, bar, k, m, z);
    } else {
      pair::tma_load_3d_pair(sA, &maps->d_cols, bar, m, k, ti.aux - 1);
      pair::tma_load_3d_pair(sA + kBox, &maps->d_cols, bar, m + 64, k, ti.aux - 1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      pair::tma_load_2d_pair(sB + j * kBox, b, bar, n + (j >> 1) * pair::BN2 + (j & 1) * 64, k);
  }
  __device__ uint32_t idesc(const TileInfo& ti) const {
    return ptx::idesc_f16_f32(2 * BM, pair::BN2, fmt, ti.aux != 0, 1);
  }
  __device__ uint64_t a_desc(const TileInfo& ti, uint32_t a, int k) const {
    return ti.aux == 0 ? ptx::sdesc_kmajor_sw128(a + k * 32) : ptx::sdesc_mnmajor_sw128(a + k * 2048, 8192);
  }
  __device__ uint64_t b_desc(const TileInfo&, uint32_t b, int k) const {
    return ptx::sdesc_mnmajor_sw128(b + k * 2048, 8192);
  }
  __device__ bool lane_skip(const TileInfo&, int, uint32_t*) const { return false; }
};

struct BwdEpi : Out16Epi {
  uint16_t *dx, *dwg, *dwu;
  long long lddx, lddw;
  int T, H, I;
  int vec_x, vec_w;
  const BwdMaps* maps;
  __device__ void begin_tile(const TileInfo& ti, int) {
    const bool is_x = ti.aux == 0;
    C = is_x ? dx : ti.aux == 1 ? dwg : dwu;
    ldc = is_x ? lddx : lddw;
    M = is_x ? T : I;
    N = H;
    vec = is_x ? vec_x : vec_w;
    tmC = is_x ? &maps->dx : ti.aux == 1 ? &maps->dwg : &maps->dwu;
  }
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::PairCfg<2>::kThreads, 1)
    k_gated_bwd(const __grid_constant__ BwdMaps maps, BwdSched sched, BwdEpi epi, ErrorRecord* err, uint64_t timeout_ns) {
  sched.maps = &maps;
  epi.maps = &maps;
  pair::gemm_core_pair<2>(&maps.d_rows, &maps.x, sched, epi, err, timeout_ns, -1);
}

namespace {
constexpr CUtensorMapDataType k16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;  // 16-bit words (f16 too: TMA moves bits)

CUtensorMap map_128b(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows) {
  return make_tmap_2d(p, k16, 2, rows, cols, ld, box_rows, BK, CU_TENSOR_MAP_SWIZZLE_128B);
}
bool vec16(const void* p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * 2 & 15) == 0; }
CUtensorMap out_map(const void* p, uint64_t rows, uint64_t cols, uint64_t ld, const CUtensorMap& unused) {
  return vec16(p, (long long)ld) ? make_tmap_2d(p, k16, 2, rows, cols, ld, 32, 32, CU_TENSOR_MAP_SWIZZLE_NONE) : unused;
}
template <class K>
void allow_smem(K kernel, uint32_t bytes, bool* done) {
  int dev = 0;
  GICC_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && done[dev]) return;
  GICC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (dev < 64) done[dev] = true;
}
constexpr uint32_t kSmemMax = 227 * 1024;

void check_16(const char* who, int fmt, int kind) {
  if (fmt < 0 || fmt > 1) throw std::runtime_error(std::string(who) + ": fmt must be 0 (f16) or 1 (bf16)");
  if (kind < 0 || kind >= ops::ACT_COUNT) throw std::runtime_error(std::string(who) + ": unknown activation");
}
void check_rows(const char* who, const char* name, const void* p, long long ld, int cols) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15) || ld % 8 || ld < cols)
    throw std::runtime_error(std::string(who) + ": " + name + " needs 16-byte aligned rows (base and pitch) of at least " +
                             std::to_string(cols) + " elements");
}
}  // namespace
}  // namespace ffn

namespace ops {

size_t gated_saved_floats(int T, int I) { return 2 * ffn::saved_plane(T, I); }
int gated_grad_pitch(int I) { return (I + 63) / 64 * 64; }

void gated_linear(const void* x, const void* w_gate, const void* w_up, void* h, int T, int H, int I, long long ldx,
                  long long ldg, long long ldu, long long ldh, int kind, int fmt, float* saved, int tile,
                  cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::gated_linear");
  using namespace ffn;
  const char* who = "gicc::gated_linear";
  check_16(who, fmt, kind);
  if (T <= 0 || H <= 0 || I <= 0) throw std::runtime_error("gicc::gated_linear: empty shape");
  if (H % 8) throw std::runtime_error("gicc::gated_linear: H must be a multiple of 8 (16-byte TMA rows)");
  check_rows(who, "x", x, ldx, H);
  check_rows(who, "w_gate", w_gate, ldg, H);
  check_rows(who, "w_up", w_up, ldu, H);
  if (h == nullptr || ldh < I) throw std::runtime_error("gicc::gated_linear: h needs rows of at least I elements");
  if (tile < 0 || tile > 2) throw std::runtime_error("gicc::gated_linear: tile must be 0 (by shape), 1 (split) or 2 (pairs)");
  if (tile == 0) tile = T <= 256 ? 1 : 2;
  if (tile == 1) {
    const split::Plan p = split::plan(T, I, H, 2, 0);
    GatedSplitOp op;
    op.h = static_cast<uint16_t*>(h);
    op.ldh = ldh;
    op.T = T;
    op.I = I;
    op.kind = kind;
    op.type = fmt;
    op.vec = (reinterpret_cast<uintptr_t>(h) & 7) == 0 && ldh % 4 == 0;
    op.saved = saved;
    static bool done[64] = {false};
    allow_smem(k_gated_split, kSmemMax, done);
    split::launch_clusters(k_gated_split, p.grid, p.splits, split::kThreads, p.smem, false, stream,
                           map_128b(x, T, H, ldx, p.sh.xrows), map_128b(w_gate, I, H, ldg, p.sh.bn),
                           map_128b(w_up, I, H, ldu, p.sh.bn), p.sh, op, device_error_record(), default_timeout_ns());
    return;
  }
  using Cf = pair::PairCfg<2>;
  GatedMaps m;
  m.x = map_128b(x, T, H, ldx, BM);
  m.g = map_128b(w_gate, I, H, ldg, BM);
  m.u = map_128b(w_up, I, H, ldu, BM);
  m.h = out_map(h, T, I, ldh, m.x);
  GatedSched s;
  s.T = T;
  s.I = I;
  s.H = H;
  s.num_m = (T + 2 * BM - 1) / (2 * BM);
  s.num_n = (I + pair::BN2 - 1) / pair::BN2;
  s.group_m = gemm_tuning().pair_group_m;
  s.fmt = fmt;
  s.maps = nullptr;
  GatedEpi e;
  e.C = static_cast<uint16_t*>(h);
  e.ldc = ldh;
  e.M = T;
  e.N = I;
  e.fmt = fmt;
  e.vec = vec16(h, ldh);
  e.kind = kind;
  e.saved = saved;
  static bool done[64] = {false};
  allow_smem(k_gated_pair, Cf::kSmemBytesStaged, done);
  const int grid = 2 * std::min(s.num_m * s.num_n, num_sms() / 2);
  k_gated_pair<<<grid, Cf::kThreads, Cf::kSmemBytesStaged, stream>>>(m, s, e, device_error_record(), default_timeout_ns());
  GICC_CUDA(cudaGetLastError());
}

void gated_linear_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const float* saved,
                           void* work, void* dx, void* dw_gate, void* dw_up, int T, int H, int I, long long lddh,
                           long long ldx, long long ldg, long long ldu, long long lddx, long long lddw, int kind, int fmt,
                           cudaStream_t stream) {
  NvtxRange nvtx("gicc::ops::gated_linear_backward");
  using namespace ffn;
  const char* who = "gicc::gated_linear_backward";
  check_16(who, fmt, kind);
  if (T <= 0 || H <= 0 || I <= 0) throw std::runtime_error("gicc::gated_linear_backward: empty shape");
  if (H % 8) throw std::runtime_error("gicc::gated_linear_backward: H must be a multiple of 8 (16-byte TMA rows)");
  check_rows(who, "x", x, ldx, H);
  check_rows(who, "w_gate", w_gate, ldg, H);
  check_rows(who, "w_up", w_up, ldu, H);
  if (dh == nullptr || lddh < I || saved == nullptr || work == nullptr || (reinterpret_cast<uintptr_t>(work) & 15))
    throw std::runtime_error("gicc::gated_linear_backward: dh, saved and a 16-byte aligned work area are needed");
  if ((dw_gate == nullptr) != (dw_up == nullptr))
    throw std::runtime_error("gicc::gated_linear_backward: both weight gradients or none");
  if ((dx != nullptr && lddx < H) || (dw_gate != nullptr && lddw < H))
    throw std::runtime_error("gicc::gated_linear_backward: gradients need rows of at least H elements");
  if (dx == nullptr && dw_gate == nullptr) return;
  const int Ip = gated_grad_pitch(I);
  uint16_t* dgu = static_cast<uint16_t*>(work);
  const long long blocks = (long long)((T + 31) / 32) * (saved_cols(I) / 16);
  const int ggrid = (int)std::min<long long>((blocks + 7) / 8, (long long)num_sms() * 8);
  k_gate_grad<<<ggrid, 256, 0, stream>>>(static_cast<const uint16_t*>(dh), lddh, saved, dgu, T, I, Ip, kind, fmt,
                                         vec16(dh, lddh) ? 1 : 0);
  GICC_CUDA(cudaGetLastError());

  using Cf = pair::PairCfg<2>;
  BwdMaps m;
  m.d_rows = make_tmap_3d(dgu, k16, 2, 2, T, I, Ip, (uint64_t)T * Ip, BM, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.d_cols = make_tmap_3d(dgu, k16, 2, 2, T, I, Ip, (uint64_t)T * Ip, 64, BK, CU_TENSOR_MAP_SWIZZLE_128B);
  m.wg = map_128b(w_gate, I, H, ldg, 64);
  m.wu = map_128b(w_up, I, H, ldu, 64);
  m.x = map_128b(x, T, H, ldx, 64);
  m.dx = dx ? out_map(dx, T, H, lddx, m.x) : m.x;
  m.dwg = dw_gate ? out_map(dw_gate, I, H, lddw, m.x) : m.x;
  m.dwu = dw_up ? out_map(dw_up, I, H, lddw, m.x) : m.x;
  BwdSched s;
  s.T = T;
  s.H = H;
  s.I = I;
  s.mx = (T + 2 * BM - 1) / (2 * BM);
  s.mw = (I + 2 * BM - 1) / (2 * BM);
  s.nn = (H + Cf::kCols - 1) / Cf::kCols;
  s.nx = dx ? s.mx * s.nn : 0;
  s.nw = dw_gate ? s.mw * s.nn : 0;
  s.x_first = 2LL * I >= T;
  s.group_m = gemm_tuning().pair_group_m;
  s.fmt = fmt;
  s.maps = nullptr;
  BwdEpi e;
  e.fmt = fmt;
  e.dx = static_cast<uint16_t*>(dx);
  e.dwg = static_cast<uint16_t*>(dw_gate);
  e.dwu = static_cast<uint16_t*>(dw_up);
  e.lddx = lddx;
  e.lddw = lddw;
  e.T = T;
  e.H = H;
  e.I = I;
  e.vec_x = dx && vec16(dx, lddx);
  e.vec_w = dw_gate && vec16(dw_gate, lddw) && vec16(dw_up, lddw);
  e.maps = nullptr;
  static bool done[64] = {false};
  allow_smem(k_gated_bwd, Cf::kSmemBytesStaged, done);
  const int tiles = s.nx + 2 * s.nw;
  const int grid = 2 * std::min(tiles, num_sms() / 2);
  k_gated_bwd<<<grid, Cf::kThreads, Cf::kSmemBytesStaged, stream>>>(m, s, e, device_error_record(), default_timeout_ns());
  GICC_CUDA(cudaGetLastError());
}

}  // namespace ops
}  // namespace gicc
