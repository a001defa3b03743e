// Internal declarations of the gated feed-forward block and of the 4-bit products, shared
// between their kernels and the C-ABI layer.
#pragma once

#include "moe_internal.h"

namespace cernels {

#ifdef __CUDACC__
// Programmatic dependent launch: every kernel here may start while the one before it on its stream, whichever that
// is, still runs, and waits for its end before it reads or writes what that one might write or read. All CTAs
// wait, so that a kernel's end implies the ends of all before it; and only then do they let the next kernel
// start, so that what a kernel reads before its own wait can be in the hands of its predecessor alone.
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}

template <class K, class... A>
cudaError_t launch_kernel(K kernel, dim3 grid, int threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
#endif

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

// ---- skinny.cu: a few rows of x times bf16 or 4-bit weights
constexpr int kSkinnyMaxColumns = 16;

struct SkinnyArgs {
  const __nv_bfloat16* x;
  size_t x_stride;            // elements between rows of x
  const uint8_t *w0, *w1;     // weight rows; gate/up: w0 gate, w1 up
  size_t w_expert;            // bytes between experts
  const uint16_t *s0, *s1;    // bf16 group scales of the same rows (4 bits)
  size_t s_expert;            // scales between experts
  void* out;                  // bf16 or fp32 [column, rows], out_stride elements apart
  size_t out_stride;
  int out_f32;
  int k, rows;                // reduction length; outputs per column (gate/up: F)
  int cols;                   // columns that a tile takes at once (skinny_columns())
  int tokens;                 // columns without routing
  const int32_t* indices;     // routing: expert of each pair, or null; a pair is a column
  int pairs, topk, experts;
  int x_by_pair;              // x rows belong to pairs (else to tokens, pair / topk)
  int k_warps;                // warps that share a tile (the launcher sets it)
  int x_from_previous;        // x is written by the kernel launched just before, which writes nothing else read here
};

// Columns per tile for a reduction of `k` (group as below; pairs and experts 0 without routing): at
// most `want`, kSkinnyMaxColumns and what shared memory holds of x. 0 when not even one row fits.
int skinny_columns(int want, int k, int group, int pairs, int experts);
// group: 0 for bf16 weights, 32 / 64 / 128 for 4 bits. gate_up: out = silu(w0 x) * (w1 x).
cudaError_t launch_skinny(const SkinnyArgs& a, int group, bool gate_up, cudaStream_t stream);
cudaError_t launch_weighted_rows(const float* rows, const int32_t* indices, const float* weights, int tokens, int topk,
                                 int experts, int hidden, __nv_bfloat16* out, cudaStream_t stream);

}  // namespace cernels
