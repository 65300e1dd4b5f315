// split_host.cuh -- host side of the split-K cluster core: tile and split by shape, launch.
#pragma once
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "gicc/device/split_core.cuh"
#include "gicc/host_util.hpp"

namespace gicc {
namespace gemm {
namespace split {

constexpr int kMaxRowBlocks = 65535;      // grid.y
constexpr int kMaxDim = INT32_MAX - 1023;  // rounding a size up to a tile must not overflow

inline void check_dims(const char* who, std::initializer_list<int> dims) {
  for (int d : dims)
    if (d <= 0 || d > kMaxDim) throw std::runtime_error(std::string(who) + ": sizes from 1 to " + std::to_string(kMaxDim));
}

constexpr CUtensorMapDataType k16 = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;  // 16-bit words (f16 too: TMA moves bits)

inline void check_rows(const char* who, const char* name, const void* p, long long ld, int cols) {
  if (p == nullptr || (reinterpret_cast<uintptr_t>(p) & 15) || ld % 8 || ld < cols)
    throw std::runtime_error(std::string(who) + ": " + name + " needs 16-byte aligned rows (base and pitch) of at least " +
                             std::to_string(cols) + " elements");
}

struct Plan {
  Shape sh;
  bool fits = true;  // the launch takes so many row blocks
  int splits = 1;
  dim3 grid;
  uint32_t smem = 0;
  double us = 0;  // expected time
};

// Once per device: kernel may use `bytes` of dynamic shared memory.  Host threads may get here at once.
template <class K>
void allow_smem(K kernel, uint32_t bytes, std::atomic<bool>* done, bool shared_sm = false) {
  int dev = 0;
  GICC_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && done[dev]) return;
  GICC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  // Kernels meant to run beside another's CTAs: without this the SM keeps just one CTA's shared
  // memory configured, and the other kernel waits until the SM is idle.
  if (shared_sm)
    GICC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared));
  if (dev < 64) done[dev] = true;
}

// Clusters of S CTAs of a one-per-SM kernel that the current device runs at a time (fewer than
// SMs / S: a cluster stays within one GPC).  Every kernel that asks has kThreads threads and takes
// more than half of an SM's shared memory, so the first one's answer (at 200 KB) holds for all.
inline int clusters_at_once(const void* kernel, int S) {
  static std::atomic<int> cache[64][kMaxSplit + 1] = {};
  int dev = 0;
  GICC_CUDA(cudaGetDevice(&dev));
  if (dev < 64) {
    const int known = cache[dev][S];
    if (known) return known;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(S * 256);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = 200 * 1024;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = S;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  int n = 0;
  GICC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
  GICC_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
  n = std::max(n, 1);
  if (dev < 64) cache[dev][S] = n;
  return n;
}

// The split S and the column count bn with the shortest expected time.  A CTA streams its share
// of the depth: accs * bn weight rows from HBM and the tile's rows of X, which come from L2
// mostly.  All CTAs together get about 6 TB/s; one gets at most about 75 KB/us, computes
// 128 x 256 x 64 in 0.38 us, and takes 0.22 us for the smallest k-block.  Clusters beyond those
// that run at once wait for a further turn, which costs about 4 us to start and drain.
// col_step: what bn is a multiple of (64 for an N-major W); copies: products of this shape in the
// launch (grid.y = copies * row blocks); depth: k-blocks, where it is not K / 64; full_rows: every X
// box holds 128 rows (an M-major X).
inline Plan plan(int T, int N, int K, int accs, uint32_t ring_kb, const void* kernel,
                 int col_step = 16, int copies = 1, int depth = 0, bool full_rows = false) {
  Plan p;
  p.sh.T = T;
  p.sh.mblocks = (T + kRows - 1) / kRows;
  p.sh.xrows = full_rows ? kRows : std::min(kRows, (T + 7) / 8 * 8);
  const int tt = p.sh.mblocks * copies;
  p.fits = tt <= kMaxRowBlocks;
  const int nkb = depth ? depth : (K + BK - 1) / BK;
  p.us = -1;
  for (int S = 1; S <= kMaxSplit && S <= nkb; ++S) {
    const long long at_once = clusters_at_once(kernel, S);
    for (int bn = col_step; accs * bn <= kMaxCols; bn += col_step) {
      if ((uint32_t)p.sh.xrows * pitch(accs, bn) * 4 > ring_kb * 1024) break;  // the partial takes the ring's place
      const long long clusters = (long long)((N + bn - 1) / bn) * tt;
      const long long turns = (clusters + at_once - 1) / at_once;
      const int steps = (nkb + S - 1) / S;
      const double bytes = (double)steps * (accs * bn + 0.3 * p.sh.xrows) * (BK * 2);
      const double alone = std::max(bytes / 75.0e3, steps * std::max(0.22, 0.38 * accs * bn / 256));
      const double us = (turns - 1) * std::max(bytes * at_once * S / 6.0e6, alone) +
                        std::max(bytes * (clusters - (turns - 1) * at_once) * S / 6.0e6, alone) + 4.0 * turns + 0.3 * S +
                        0.5e-3 * std::min(T, kRows) * accs * bn / S;
      if (p.us < 0 || us < p.us) {
        p.us = us;
        p.sh.bn = bn;
        p.splits = S;
      }
    }
  }
  p.sh.group = 6 * (x_bytes(p.sh.xrows) + w_bytes(accs, p.sh.bn)) <= ring_kb * 1024 ? 2 : 1;
  const uint32_t per = p.sh.group * (x_bytes(p.sh.xrows) + w_bytes(accs, p.sh.bn));
  p.sh.stages = std::max(2, std::min<int>(kMaxStages, ring_kb * 1024 / per));
  p.grid = dim3((N + p.sh.bn - 1) / p.sh.bn * p.splits, tt, 1);
  p.smem = 1024 + ring_bytes(accs, p.sh.bn, p.sh.xrows, p.sh.group, p.sh.stages) + kBarBytes;
  return p;
}

// 1: the split-K clusters, 2 / 3: CTA pairs with 256 x 512 / 256 x 256 tiles (N counts one
// weight's columns; a pair tile holds accs of them side by side), by expected time.  pair_extra:
// us that the pairs' way costs besides.
inline int pick_tile(int T, int N, int K, int accs, uint32_t ring_kb, const void* kernel, double pair_extra = 0) {
  const int pairs = num_sms() / 2;
  const int nkb = (K + BK - 1) / BK;
  // A k-block of a pair's tile takes 0.74 / 0.40 us with all pairs at work (L2, power), 0.6 /
  // 0.33 us with few; the rest is set-up, first loads and the last tile's epilogue.
  auto pair_us = [&](int nh) {
    const int cols = nh * pair::BN2 / accs;
    const double tiles = (double)((T + 2 * BM - 1) / (2 * BM)) * ((N + cols - 1) / cols);
    const double turns = std::ceil(tiles / pairs), busy = std::min(1.0, tiles / pairs);
    return turns * nkb * (nh == 2 ? 0.60 + 0.14 * busy : 0.33 + 0.07 * busy) + (nh == 2 ? 12.0 : 10.0) + turns + pair_extra;
  };
  const double wide = pair_us(2), narrow = pair_us(1);
  const Plan split = plan(T, N, K, accs, ring_kb, kernel);
  if (split.fits && split.us <= wide && split.us <= narrow) return 1;
  return wide <= narrow ? 2 : 3;
}

inline void check_fits(const char* who, const Plan& p) {
  if (!p.fits)
    throw std::runtime_error(std::string(who) + ": too many rows for the split clusters (" + std::to_string(kMaxRowBlocks) +
                             " blocks of 128)");
}

// Launch in clusters of `splits`; `overlap` lets the kernel start before the previous one of
// the stream has ended (it then waits with griddep_wait).
template <class Kernel, class... Args>
inline void launch_clusters(Kernel k, dim3 grid, int splits, int threads, uint32_t smem, bool overlap, cudaStream_t stream,
                            Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = overlap ? 2 : 1;
  GICC_CUDA(cudaLaunchKernelEx(&cfg, k, args...));
}

// Launch that may start before the previous kernel of the stream has ended (its griddep_wait
// comes after its set-up).
template <class Kernel, class... Args>
inline void launch_dependent(Kernel k, dim3 grid, int threads, uint32_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  GICC_CUDA(cudaLaunchKernelEx(&cfg, k, args...));
}

}  // namespace split
}  // namespace gemm
}  // namespace gicc
