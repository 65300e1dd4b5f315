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

// MASKS false: only the list and the rows' slots.
template <int ROWS, bool MASKS = true>
struct LaneLists {
  uint32_t skip[MASKS ? ROWS : 1][ROWS / 32];  // per distinct adapter: lanes that are not its
  uint32_t used[kWords];            // bit a: some row uses adapter a
  int before[kWords];               // distinct adapters below word w's
  int list[ROWS];                   // distinct adapters, ascending
  int n;

  // By `threads` threads (whole warps, at least ROWS / 2 threads), this one number `tid` of them,
  // which synchronise on named barrier 1.  An index outside [-1, L) is reported and its row treated
  // as having no adapter.
  __device__ void build(const int* adapter, int t0, int T, int L, ErrorRecord* err, int tid, int threads) {
    auto sync = [&] { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); };
    const int words = (L + 31) / 32;
    int mine[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int i = tid + k * threads, t = t0 + i;
      mine[k] = -1;
      if (i < ROWS && t < T) {
        const int a = adapter[t];
        if (a >= 0 && a < L) mine[k] = a;
        else if (a != -1) report_error(err, GICC_ERANGE, W_ADAPTER, -1, -1, (unsigned)a, (unsigned)L);
      }
    }
    for (int w = tid; w < words; w += threads) used[w] = 0;
    if (MASKS)
      for (int i = tid; i < ROWS * (ROWS / 32); i += threads) skip[0][i] = ~0u;
    sync();
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (mine[k] >= 0) atomicOr(&used[mine[k] >> 5], 1u << (mine[k] & 31));
    sync();
    if (tid < 32) {
      const int lane = tid;
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
    sync();
    if (MASKS) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int i = tid + k * threads;
        if (mine[k] >= 0) atomicAnd(&skip[slot(mine[k])][i >> 5], ~(1u << (i & 31)));
      }
      sync();
    }
  }
  // a's place in the list, for an adapter that some row uses
  __device__ int slot(int a) const { return before[a >> 5] + __popc(used[a >> 5] & ((1u << (a & 31)) - 1u)); }
};

}  // namespace lora
}  // namespace gicc
