// split_core.cuh -- tcgen05 projection core for few rows: one output tile per thread-block
// cluster, the depth K split over the cluster's CTAs.
//
//   D_i[rows, cols] = X[rows, K] * W_i[cols, K]^T,  i = 0 .. kAccs-1, f32 accumulate
//
// With few rows the product is a stream of the weights from HBM, and the output has too few
// tiles to give every SM one.  So a cluster of S CTAs takes one tile of up to 128 rows x bn
// columns, each CTA runs its share of the k-blocks through its own TMA ring and accumulators
// (rows in TMEM lanes, columns of weight i at i * bn), writes its f32 partial to its own
// shared memory, and after a cluster barrier every CTA sums a slice of the tile over all S
// partials (distributed shared memory, in rank order, so results do not depend on timing)
// and hands it to the Op's emit().  One launch, no workspace, no atomics.
//
// Warp roles: 0 producer, 1 TMEM + MMA, 2..5 TMEM readers; all six sum and store.  Every wait
// is bounded; all CTAs of a cluster always reach both cluster barriers.
#pragma once
#include <cstdint>

#include "gicc/device/gemm_core2.cuh"

namespace gicc {
namespace gemm {
namespace split {

constexpr int kRows = 128;              // rows of a tile (TMEM lanes)
constexpr int kThreads = 192;
constexpr int kMaxSplit = 8;            // portable cluster size
constexpr int kMaxCols = 256;           // columns of all weights per tile (the MMA's N)
constexpr int kMaxStages = 12;
constexpr uint32_t kBarBytes = (2 * kMaxStages + 4) * 8 + 8;  // barriers, TMEM address, abort flag

struct Shape {
  int T;         // rows of X
  int bn;        // columns per tile and weight: a multiple of 16
  int mblocks;   // tiles of 128 rows
  int xrows;     // rows of an X box: min(128, T rounded up to 8)
  int group;     // k-blocks per ring stage
  int stages;
};

__host__ __device__ constexpr uint32_t x_bytes(int xrows) { return xrows * BK * 2; }        // of one k-block
__host__ __device__ constexpr uint32_t w_bytes(int accs, int bn) { return accs * bn * BK * 2; }
// floats between two rows of a partial: + 4 keeps the 16-byte writes of 8 lanes on 32 banks
__host__ __device__ constexpr int pitch(int accs, int bn) { return accs * bn + 4; }
// The ring (X of all stages, then W), or the partial that takes its place.  The MMA reads 128
// rows of X whatever xrows is: the rows behind an X box are other data of the ring, and their
// lanes are never read; the last box has 16 KB of ring behind its start.
__host__ __device__ constexpr uint32_t ring_bytes(int accs, int bn, int xrows, int group, int stages) {
  uint32_t ring = stages * group * (x_bytes(xrows) + w_bytes(accs, bn));
  const uint32_t reach = (stages * group - 1) * x_bytes(xrows) + kRows * BK * 2, part = xrows * pitch(accs, bn) * 4;
  if (reach > ring) ring = reach;
  return ((ring > part ? ring : part) + 127) / 128 * 128;
}
__host__ __device__ constexpr uint32_t tmem_cols(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : 256; }

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Four columns of an output row in its 16-bit type: one 8-byte store where C's base and pitch
// allow it (vec) and all four columns exist, else element stores.
__device__ __forceinline__ void store4_16(uint16_t* row, int col, int N, const float* v, int fmt, int vec) {
  const uint32_t a = ptx::pack_16x2(v[0], v[1], fmt), b = ptx::pack_16x2(v[2], v[3], fmt);
  if (vec && col + 4 <= N) {
    *reinterpret_cast<uint2*>(row + col) = make_uint2(a, b);
  } else {
    if (col < N) row[col] = (uint16_t)a;
    if (col + 1 < N) row[col + 1] = (uint16_t)(a >> 16);
    if (col + 2 < N) row[col + 2] = (uint16_t)b;
    if (col + 3 < N) row[col + 3] = (uint16_t)(b >> 16);
  }
}

// Op: kAccs (weights multiplied side by side) and
//   start(smem_extra)              by all threads before the pipeline starts
//   kExtra                         whether there are further k-blocks after the weights'; then
//   prepare(t0, tid)               by the 128 threads of warps 2..5, beside the pipeline
//   loads(kb, t0, n0, x, w, bar)   the loads of k-block kb (x_bytes + w_bytes in all)
//   idesc(n), x_desc(addr, k), w_desc(addr, k)  the MMA descriptors of k-step k of a k-block
//   depth()                        k-blocks
//   extra_blocks(c, S, e0, e1)     this CTA's further k-blocks, once prepare() is done
//   extra_shared(t0, bar)          by the producer before the first of them: waits for what they
//                                  need and loads what all share (arrives on bar with its bytes)
//   extra_loads(e, n0, w, bar)     loads of one (w_bytes)
//   extra_mma(e, d, w, idesc)      its MMAs
//   emit(row, col, v)              v[i][4]: four columns of weight i of one valid row
//   finish()                       by all threads, last
// The K-major operands and no further k-blocks: the base of most Ops.
struct PlainOp {
  int type;                 // 0 = f16, 1 = bf16
  const CUtensorMap* tmX;   // set by the kernel
  const CUtensorMap* tmW;
  static constexpr bool kExtra = false;
  __device__ void start(uint8_t*) {}
  __device__ void prepare(int, int) {}
  __device__ void prefetch_maps() const {
    ptx::prefetch_tmap(tmX);
    ptx::prefetch_tmap(tmW);
  }
  __device__ uint32_t idesc(int n) const { return ptx::idesc_f16_f32(kRows, n, type, 0, 0); }
  __device__ uint64_t x_desc(uint32_t x, int k) const { return ptx::sdesc_kmajor_sw128(x + k * 32); }
  __device__ uint64_t w_desc(uint32_t w, int k) const { return ptx::sdesc_kmajor_sw128(w + k * 32); }
  __device__ void loads(int kb, int t0, int n0, uint8_t* x, uint8_t* w, uint64_t* bar) const {
    ptx::tma_load_2d(w, tmW, bar, kb * BK, n0);
    ptx::tma_load_2d(x, tmX, bar, kb * BK, t0);
  }
  __device__ void extra_blocks(int, int, int& e0, int& e1) const { e0 = e1 = 0; }
  __device__ void extra_shared(int, uint64_t*) const {}
  __device__ void extra_loads(int, int, uint8_t*, uint64_t*) const {}
  __device__ void extra_mma(int, uint32_t, uint32_t, uint32_t) const {}
  __device__ void finish() const {}
};

template <class Op>
__device__ __forceinline__ void split_core(const Shape& sh, Op& op, ErrorRecord* err, uint64_t timeout_ns) {
  constexpr int A = Op::kAccs;
  extern __shared__ uint8_t split_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(split_smem_raw) + 1023) & ~uintptr_t(1023));
  const int stages = sh.stages, group = sh.group;
  const uint32_t xb = x_bytes(sh.xrows), wb = w_bytes(A, sh.bn);
  uint8_t* sX = smem;
  uint8_t* sW = smem + stages * group * xb;  // per k-block: bn rows of each weight
  uint8_t* after = smem + ring_bytes(A, sh.bn, sh.xrows, group, stages);
  uint64_t* full = reinterpret_cast<uint64_t*>(after);
  uint64_t* empty = full + kMaxStages;
  uint64_t* tfull = empty + kMaxStages;
  uint64_t* drain = tfull + 1;
  uint64_t* once = drain + 1;  // what the further k-blocks share has landed
  uint64_t* ready = once + 1;  // prepare() is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* part = reinterpret_cast<float*>(smem);  // after the last MMA: this CTA's partial

  const uint32_t warp = ptx::warp_id();
  const uint32_t lane = ptx::lane_id();
  const int S = (int)cluster_size();
  const int c = (int)pair::cta_rank();
  const int n0 = (int)(blockIdx.x / S) * sh.bn;
  const int t0 = (int)blockIdx.y % sh.mblocks * kRows;  // blockIdx.y / mblocks: the Op's further index
  const int rows = min(kRows, sh.T - t0);
  const int ncol = A * sh.bn;
  const uint32_t tcols = tmem_cols(ncol);

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      ptx::mbar_init(&full[s], 1);
      ptx::mbar_init(&empty[s], 1);
    }
    ptx::mbar_init(tfull, 1);
    ptx::mbar_init(drain, 1);
    ptx::mbar_init(once, 1);
    ptx::mbar_init(ready, 1);
    *abort_flag = 0;
    ptx::fence_mbar_init();
    op.prefetch_maps();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, tcols);
    ptx::tmem_relinquish();
  }
  op.start(after + kBarBytes);
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int nkb = op.depth();
  const int kb0 = (int)((long long)nkb * c / S), nk = (int)((long long)nkb * (c + 1) / S) - kb0;
  // nk >= 1: the host takes S <= nkb.  With further blocks, the steps that hold only the weights'
  // come before prepare() has to be done; then the rest, which it determines.
  int e0 = 0, blocks = nk, steps = Op::kExtra ? nk / group : (nk + group - 1) / group;
  auto all_steps = [&]() -> bool {
    if (!ptx::mbar_wait(ready, 0, timeout_ns, abort_flag)) {
      if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 5, 0);
      *abort_flag = 1;
      return false;
    }
    int e1;
    op.extra_blocks(c, S, e0, e1);
    blocks = nk + (e1 - e0);
    steps = (blocks + group - 1) / group;
    return true;
  };

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool shared = false;
      for (int i = 0;; ++i) {
        if (Op::kExtra && i == nk / group && !all_steps()) break;
        if (i >= steps) break;
        if (!ptx::mbar_wait(&empty[stage], phase ^ 1, timeout_ns, abort_flag)) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 0, 0);
          *abort_flag = 1;
          break;
        }
        const int b0 = i * group, nb = min(group, blocks - b0);
        ptx::mbar_arrive_expect_tx(&full[stage], nb * wb + max(0, min(nb, nk - b0)) * xb);
        for (int j = 0; j < nb; ++j) {
          const int b = b0 + j;
          uint8_t* x = sX + (stage * group + j) * xb;
          uint8_t* w = sW + (stage * group + j) * wb;
          if (b < nk) {
            op.loads(kb0 + b, t0, n0, x, w, &full[stage]);
          } else {
            if (!shared) {
              op.extra_shared(t0, once);
              shared = true;
            }
            op.extra_loads(e0 + b - nk, n0, w, &full[stage]);
          }
        }
        issued = i + 1;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (*abort_flag) {
        // Let the TMA loads already issued land before the CTA's smem is used again.
        for (int i = issued > stages ? issued - stages : 0; i < issued; ++i)
          ptx::mbar_wait(&full[i % stages], (i / stages) & 1, 20000000ull, nullptr);
        if (shared) ptx::mbar_wait(once, 0, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = op.idesc(ncol);
      int stage = 0;
      uint32_t phase = 0;
      int i = 0;
      for (;; ++i) {
        if (Op::kExtra && i == nk / group && !all_steps()) break;
        if (i >= steps) break;
        if (!ptx::mbar_wait(&full[stage], phase, timeout_ns, abort_flag)) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 2, 0);
          *abort_flag = 1;
          break;
        }
        ptx::tc_fence_after();
        const int b0 = i * group, nb = min(group, blocks - b0);
        if (b0 <= nk && b0 + nb > nk && !ptx::mbar_wait(once, 0, timeout_ns, abort_flag)) {
          if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 4, 0);
          *abort_flag = 1;
          break;
        }
        ptx::tc_fence_after();
        for (int j = 0; j < nb; ++j) {
          const uint32_t x = ptx::smem_u32(sX + (stage * group + j) * xb);
          const uint32_t w = ptx::smem_u32(sW + (stage * group + j) * wb);
          if (b0 + j < nk) {
#pragma unroll
            for (int k = 0; k < BK / 16; ++k)
              ptx::mma_f16_ss(tmem, op.x_desc(x, k), op.w_desc(w, k), idesc, (b0 + j > 0 || k > 0) ? 1u : 0u);
          } else {
            op.extra_mma(e0 + b0 + j - nk, tmem, w, idesc);
          }
        }
        ptx::mma_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (!*abort_flag) {
        ptx::mma_commit(tfull);
      } else if (i > 0) {  // aborted: wait for the MMAs in flight before TMEM is released
        ptx::mma_commit(drain);
        ptx::mbar_wait(drain, 0, 20000000ull, nullptr);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3;
    const int row = q * 32 + (int)lane;
    if constexpr (Op::kExtra) {
      op.prepare(t0, (int)threadIdx.x - 64);
      if (threadIdx.x == 64) ptx::mbar_arrive(ready);
    }
    if (!ptx::mbar_wait_long(tfull, 0, timeout_ns, abort_flag)) {
      if (!*abort_flag) report_error(err, GICC_ETIMEDOUT, W_GEMM_PIPE, -1, -1, 3, 0);
      *abort_flag = 1;
    } else if (q * 32 < rows) {
      ptx::tc_fence_after();
      const uint32_t tbase = tmem + (static_cast<uint32_t>(q * 32) << 16);
      float* dst = part + row * pitch(A, sh.bn);
      for (int col = 0; col < ncol; col += 16) {
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
  pair::cluster_sync();  // every CTA's partial is in place
  if (!*abort_flag) {
    const int g4 = sh.bn / 4;  // groups of four columns per row
    const int groups = rows * g4;
    const int j1 = (int)((long long)groups * (c + 1) / S);
    const uint32_t base = ptx::smem_u32(part);
    for (int j = (int)((long long)groups * c / S) + (int)threadIdx.x; j < j1; j += kThreads) {
      const int row = j / g4, col = (j - row * g4) * 4;
      float v[A][4];
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const uint32_t off = base + (row * pitch(A, sh.bn) + a * sh.bn + col) * 4;
        float4 p[kMaxSplit];
#pragma unroll
        for (int s = 0; s < kMaxSplit; ++s)
          if (s < S) p[s] = ld_cluster_f4(pair::map_to(off, s));
        v[a][0] = p[0].x;
        v[a][1] = p[0].y;
        v[a][2] = p[0].z;
        v[a][3] = p[0].w;
#pragma unroll
        for (int s = 1; s < kMaxSplit; ++s)
          if (s < S) {
            v[a][0] += p[s].x;
            v[a][1] += p[s].y;
            v[a][2] += p[s].z;
            v[a][3] += p[s].w;
          }
      }
      op.emit(t0 + row, n0 + col, v);
    }
  }
  op.finish();
  pair::cluster_sync();  // no CTA leaves while its partial is being read
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, tcols);
  }
}

}  // namespace split
}  // namespace gemm
}  // namespace gicc
