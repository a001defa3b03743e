// Internal declarations of the gated feed-forward block and of the 4-bit products, shared
// between their kernels and the C-ABI layer.
#pragma once

#include "moe_internal.h"

namespace cernels {

// ---- pair_gemm.cu: bf16 matrix products over CTA pairs (more than a few tokens, and training)
struct FfnShape {
  int tokens, hidden, inter;
};

// h = silu(x gate^T) * (x up^T); with `gate_up` also both products in 32 bits (layout: gate_up_floats()).
cudaError_t launch_ffn_gate_up(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                               const __nv_bfloat16* up, __nv_bfloat16* h, float* gate_up, cudaStream_t stream);
// out = h down^T
cudaError_t launch_ffn_down(const FfnShape& s, const __nv_bfloat16* h, const __nv_bfloat16* down, __nv_bfloat16* out,
                            cudaStream_t stream);
// d_gate, d_up [T, F]: gradients at the two products, from dy [T, H] and the stored products.
cudaError_t launch_ffn_d_gate_up(const FfnShape& s, const __nv_bfloat16* dy, const __nv_bfloat16* down,
                                 const float* gate_up, __nv_bfloat16* d_gate, __nv_bfloat16* d_up,
                                 cudaStream_t stream);
// dx = d_gate gate + d_up up;  dw_gate = d_gate^T x;  dw_up = d_up^T x;  dw_down = dy^T h. Outputs that are null
// are not computed; one launch for all.
struct FfnGrads {
  __nv_bfloat16 *dx, *dw_gate, *dw_up, *dw_down;
};
cudaError_t launch_ffn_grads(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                             const __nv_bfloat16* up, const __nv_bfloat16* h, const __nv_bfloat16* dy,
                             const __nv_bfloat16* d_gate, const __nv_bfloat16* d_up, const FfnGrads& out,
                             cudaStream_t stream);

// Reads, and clears when nonzero, this device's word for bounded waits of these kernels that gave up.
cudaError_t ffn_status(int* status, cudaStream_t stream);

// 32-bit values in the stored gate/up products: [ceil(T/32)][F/4][gate, up][32 rows][4 columns], so that a
// warp whose lanes hold one row each reads and writes 512 contiguous bytes.
inline size_t gate_up_floats(const FfnShape& s) {
  return (static_cast<size_t>(s.tokens) + 31) / 32 * 32 * 2 * static_cast<size_t>(s.inter);
}

}  // namespace cernels
