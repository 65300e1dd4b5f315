/* projections.h -- C entry points of the gated projection and of the projection with low-rank adapters.
 *
 * All matrices are row-major with unit column stride, on the current device, all f16 (fmt 0) or all
 * bf16 (fmt 1); ld* are row pitches in elements.  x, the weights, lora_a, lora_b and the gradients
 * have 16-byte aligned rows (base and pitch); saved and work are 16-byte aligned.  Sizes are 1 or more,
 * H, K and r multiples of 8.  Outputs, saved and work overlap neither the inputs nor one another.  The
 * calls launch on `stream`, allocate nothing but the device's error record (first call of the library)
 * and can be captured.
 * They return 0, or -1 with the reason on stderr.
 *
 * gicc_gated_linear            h[T,I] = act(x[T,H] w_gate[I,H]^T) * (x w_up[I,H]^T).  saved: null, or
 *                              gicc_gated_saved_floats(T, I) floats that the backward pass needs.
 * gicc_gated_linear_backward   dx[T,H] (null: not wanted), dw_gate and dw_up [I,H] of pitch lddw (null, both
 *                              or none) from dh[T,I] and the forward's saved.  work:
 *                              gicc_gated_grad_bytes(T, I) bytes, free again when the call's work is done.
 * gicc_lora_linear             y[T,N] = x[T,K] w[N,K]^T + scale[a] (x lora_a[a]^T) lora_b[a]^T with
 *                              a = adapter[t] (-1: none); lora_a [L,r,K] and lora_b [L,N,r] dense, adapter
 *                              int32 [T], scale f32 [L] or null (1); r <= 128, L <= 8192, T <= 8388480.  work:
 *                              gicc_lora_work_bytes(T, L, r) bytes, as above.
 *
 * The layouts of saved and work are private; their sizes are 0 for sizes that the calls refuse.
 */
#ifndef GICC_PROJECTIONS_H
#define GICC_PROJECTIONS_H

#include <cuda_runtime.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { GICC_ACT_SILU = 0, GICC_ACT_GELU = 1, GICC_ACT_GELU_TANH = 2 };

size_t gicc_gated_saved_floats(int T, int I);
size_t gicc_gated_grad_bytes(int T, int I);
size_t gicc_lora_work_bytes(int T, int L, int r);

int gicc_gated_linear(const void* x, const void* w_gate, const void* w_up, void* h, int T, int H, int I, long long ldx,
                      long long ldg, long long ldu, long long ldh, int act, int fmt, float* saved, cudaStream_t stream);
int gicc_gated_linear_backward(const void* dh, const void* x, const void* w_gate, const void* w_up, const float* saved,
                               void* work, void* dx, void* dw_gate, void* dw_up, int T, int H, int I, long long lddh,
                               long long ldx, long long ldg, long long ldu, long long lddx, long long lddw, int act, int fmt,
                               cudaStream_t stream);
int gicc_lora_linear(const void* x, const void* w, const void* lora_a, const void* lora_b, const int* adapter,
                     const float* scale, void* y, void* work, int T, int K, int N, int L, int r, long long ldx,
                     long long ldw, long long ldy, int fmt, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* GICC_PROJECTIONS_H */
