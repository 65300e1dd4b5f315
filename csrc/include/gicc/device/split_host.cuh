// split_host.cuh -- host side of the split-K cluster core: tile and split by shape, launch.
#pragma once
#include <algorithm>

#include "gicc/device/split_core.cuh"
#include "gicc/host_util.hpp"

namespace gicc {
namespace gemm {
namespace split {

struct Plan {
  Shape sh;
  int splits = 1;
  dim3 grid;
  uint32_t smem = 0;
};

// The split S and the column count bn that give the shortest stream per CTA: every CTA reads
// its share of the depth of bn weight rows (and of the tile's rows of X, from L2 mostly), and
// CTAs beyond the SM count wait for a second turn.
inline Plan plan(int T, int N, int K, int accs, uint32_t extra_smem) {
  Plan p;
  p.sh.T = T;
  p.sh.N = N;
  p.sh.K = K;
  p.sh.xrows = std::min(kRows, (T + 7) / 8 * 8);
  const int sms = num_sms();
  const int tt = (T + kRows - 1) / kRows;
  const int nkb = (K + BK - 1) / BK;
  double best = -1;
  for (int S = 1; S <= kMaxSplit && S <= nkb; ++S)
    for (int bn = 16; bn <= kMaxCols; bn += 16) {
      const long long tiles = (long long)((N + bn - 1) / bn) * tt;
      const long long turns = (tiles * S + sms - 1) / sms;
      const int steps = (nkb + S - 1) / S;
      // bytes a CTA streams (X weighs less: it comes from L2), plus what a tile costs anyway
      const double cost = turns * (steps * (accs * bn + 0.4 * p.sh.xrows) * 128.0 + 60000.0 + 4000.0 * S);
      if (best < 0 || cost < best) {
        best = cost;
        p.sh.bn = bn;
        p.splits = S;
      }
    }
  const uint32_t per = stage_bytes(accs, p.sh.bn);
  p.sh.stages = std::max(2, std::min<int>(kMaxStages, 128 * 1024 / per));
  p.grid = dim3((N + p.sh.bn - 1) / p.sh.bn * p.splits, tt, 1);
  p.smem = 1024 + ring_bytes(accs, p.sh.bn, p.sh.stages, kRows) + kBarBytes + extra_smem;
  return p;
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

}  // namespace split
}  // namespace gemm
}  // namespace gicc
