// adapter_lanes.cuh -- which adapters a tile's rows use, and the rows (TMEM lanes) of each.
//
// A tile's rows may belong to any adapters in any order.  Instead of sorting rows, the tile
// runs one narrow MMA per distinct adapter and lets it write only that adapter's lanes (the
// MMA's lane mask), so rows stay where they are and rows without an adapter are in no mask.
#pragma once
#include <cstdint>

#include "gicc/error.hpp"

namespace gicc {
namespace lora {

constexpr int kMaxAdapters = 8192;
constexpr int kWords = kMaxAdapters / 32;

template <int ROWS>
struct LaneLists {
  uint32_t used[kWords];            // bit a: some row uses adapter a
  int before[kWords];               // distinct adapters below word w's
  uint32_t skip[ROWS][ROWS / 32];   // per distinct adapter: lanes that are not its
  int list[ROWS];                   // distinct adapters, ascending
  int n;

  // All threads of the block; synchronises.  An index outside [-1, L) is reported and its row
  // treated as having no adapter.
  __device__ void build(const int* adapter, int t0, int T, int L, ErrorRecord* err) {
    const int words = (L + 31) / 32;
    for (int w = threadIdx.x; w < words; w += blockDim.x) used[w] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS; i += blockDim.x) {
      const int a = at(adapter, t0 + i, T, L);
      if (a >= 0) atomicOr(&used[a >> 5], 1u << (a & 31));
      else if (a < -1) report_error(err, GICC_ERANGE, W_ADAPTER, -1, -1, (unsigned)adapter[t0 + i], (unsigned)L);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int run = 0;
      for (int w0 = 0; w0 < words; w0 += 32) {
        uint32_t b = w0 + lane < words ? used[w0 + lane] : 0u;
        const int cnt = __popc(b);
        int incl = cnt;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, incl, d);
          if (lane >= d) incl += o;
        }
        int pos = run + incl - cnt;
        if (w0 + lane < words) before[w0 + lane] = pos;
        for (; b; b &= b - 1) list[pos++] = (w0 + lane) * 32 + __ffs(b) - 1;
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (lane == 0) n = run;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n * (ROWS / 32); i += blockDim.x) skip[0][i] = ~0u;
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS; i += blockDim.x) {
      const int s = slot(at(adapter, t0 + i, T, L));
      if (s >= 0) atomicAnd(&skip[s][i >> 5], ~(1u << (i & 31)));
    }
    __syncthreads();
  }
  // the row's adapter, -1 for none, -2 for an index outside [-1, L)
  __device__ static int at(const int* adapter, int t, int T, int L) {
    if (t >= T) return -1;
    const int a = adapter[t];
    return a >= -1 && a < L ? a : -2;
  }
  __device__ int slot(int a) const {
    return a < 0 ? -1 : before[a >> 5] + __popc(used[a >> 5] & ((1u << (a & 31)) - 1u));
  }
};

}  // namespace lora
}  // namespace gicc
