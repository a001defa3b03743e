// C ABI of the gated feed-forward block: argument checks, workspace carving and the launch
// sequence of each entry point. No entry allocates, synchronises (cernels_ffn_status apart) or
// reads device memory on the host, and none throws.
#include <cstdio>

#include "ffn_internal.h"

using namespace cernels;

namespace {

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int code_of(cudaError_t e) {
  if (e == cudaSuccess) return CERNELS_OK;
  std::fprintf(stderr, "cernels_b200: CUDA error: %s\n", cudaGetErrorString(e));
  return CERNELS_E_CUDA;
}

int check_ffn(const cernels_ffn_shape* s) {
  if (!s) return CERNELS_E_NULL;
  if (s->tokens < 0 || s->hidden <= 0 || s->intermediate <= 0) return CERNELS_E_INVALID_SHAPE;
  if (s->hidden % 8 != 0 || s->intermediate % 8 != 0) return CERNELS_E_ALIGNMENT;
  // tile counts and TMA coordinates are 32-bit
  if (s->tokens > (1 << 28) || s->hidden > (1 << 20) || s->intermediate > (1 << 20)) return CERNELS_E_UNSUPPORTED;
  return CERNELS_OK;
}

int check_call(const cernels_ffn_shape* s, const void* x, int64_t x_stride, const void* gate, const void* up,
               const void* down) {
  if (!x || !gate || !up || !down) return CERNELS_E_NULL;
  if (!aligned(x) || !aligned(gate) || !aligned(up) || !aligned(down)) return CERNELS_E_ALIGNMENT;
  if (x_stride % 8 != 0) return CERNELS_E_ALIGNMENT;
  if (x_stride < s->hidden) return CERNELS_E_INVALID_SHAPE;
  return check_sm100();
}

FfnShape shape_of(const cernels_ffn_shape* s) { return {s->tokens, s->hidden, s->intermediate}; }

size_t act_bytes(const cernels_ffn_shape* s) {
  return align_up(static_cast<size_t>(s->tokens) * s->intermediate * 2, 256);
}

const __nv_bfloat16* in(const void* p) { return static_cast<const __nv_bfloat16*>(p); }
__nv_bfloat16* outp(void* p) { return static_cast<__nv_bfloat16*>(p); }

}  // namespace

extern "C" {

int cernels_gated_ffn_workspace_bytes(const cernels_ffn_shape* shape, int32_t backward, size_t* bytes) {
  const int rc = check_ffn(shape);
  if (rc) return rc;
  if (!bytes) return CERNELS_E_NULL;
  *bytes = (backward ? 2 : 1) * act_bytes(shape);
  return CERNELS_OK;
}

int cernels_gated_ffn_saved_bytes(const cernels_ffn_shape* shape, size_t* bytes) {
  const int rc = check_ffn(shape);
  if (rc) return rc;
  if (!bytes) return CERNELS_E_NULL;
  *bytes = gate_up_floats(shape_of(shape)) * sizeof(float);
  return CERNELS_OK;
}

int cernels_gated_ffn(const cernels_ffn_shape* shape, const void* x, int64_t x_stride, const void* gate_proj,
                      const void* up_proj, const void* down_proj, void* out, void* workspace, size_t workspace_bytes,
                      void* stream) {
  int rc = check_ffn(shape);
  if (rc || shape->tokens == 0) return rc;
  rc = check_call(shape, x, x_stride, gate_proj, up_proj, down_proj);
  if (rc) return rc;
  if (!out) return CERNELS_E_NULL;
  if (!workspace || workspace_bytes < act_bytes(shape)) return CERNELS_E_WORKSPACE;
  if (!aligned(out) || !aligned(workspace)) return CERNELS_E_ALIGNMENT;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const FfnShape s = shape_of(shape);
  cudaError_t err = launch_ffn_gate_up(s, in(x), static_cast<size_t>(x_stride), in(gate_proj), in(up_proj),
                                       outp(workspace), nullptr, st);
  if (err == cudaSuccess) err = launch_ffn_down(s, in(workspace), in(down_proj), outp(out), st);
  return code_of(err);
}

int cernels_gated_ffn_forward(const cernels_ffn_shape* shape, const void* x, int64_t x_stride, const void* gate_proj,
                              const void* up_proj, const void* down_proj, void* out, void* act, void* saved,
                              void* stream) {
  int rc = check_ffn(shape);
  if (rc || shape->tokens == 0) return rc;
  rc = check_call(shape, x, x_stride, gate_proj, up_proj, down_proj);
  if (rc) return rc;
  if (!out || !act || !saved) return CERNELS_E_NULL;
  if (!aligned(out) || !aligned(act) || !aligned(saved)) return CERNELS_E_ALIGNMENT;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const FfnShape s = shape_of(shape);
  cudaError_t err = launch_ffn_gate_up(s, in(x), static_cast<size_t>(x_stride), in(gate_proj), in(up_proj), outp(act),
                                       static_cast<float*>(saved), st);
  if (err == cudaSuccess) err = launch_ffn_down(s, in(act), in(down_proj), outp(out), st);
  return code_of(err);
}

int cernels_gated_ffn_backward(const cernels_ffn_shape* shape, const void* x, int64_t x_stride, const void* gate_proj,
                               const void* up_proj, const void* down_proj, const void* act, const void* saved,
                               const void* dout, void* dx, void* dgate_proj, void* dup_proj, void* ddown_proj,
                               void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_ffn(shape);
  if (rc) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (shape->tokens == 0) {  // sums over no tokens
    const size_t bytes = static_cast<size_t>(shape->hidden) * shape->intermediate * 2;
    cudaError_t err = cudaSuccess;
    for (void* w : {dgate_proj, dup_proj, ddown_proj})
      if (w && err == cudaSuccess) err = cudaMemsetAsync(w, 0, bytes, st);
    return code_of(err);
  }
  rc = check_call(shape, x, x_stride, gate_proj, up_proj, down_proj);
  if (rc) return rc;
  if (!act || !saved || !dout) return CERNELS_E_NULL;
  if (!workspace || workspace_bytes < 2 * act_bytes(shape)) return CERNELS_E_WORKSPACE;
  for (const void* p : {act, saved, dout, const_cast<const void*>(dx), const_cast<const void*>(dgate_proj),
                        const_cast<const void*>(dup_proj), const_cast<const void*>(ddown_proj),
                        const_cast<const void*>(workspace)})
    if (!aligned(p)) return CERNELS_E_ALIGNMENT;
  const FfnShape s = shape_of(shape);
  __nv_bfloat16* d_gate = outp(workspace);
  __nv_bfloat16* d_up = outp(static_cast<uint8_t*>(workspace) + act_bytes(shape));
  cudaError_t err = cudaSuccess;
  if (dx || dgate_proj || dup_proj)
    err = launch_ffn_d_gate_up(s, in(dout), in(down_proj), static_cast<const float*>(saved), d_gate, d_up, st);
  const FfnGrads g{outp(dx), outp(dgate_proj), outp(dup_proj), outp(ddown_proj)};
  if (err == cudaSuccess)
    err = launch_ffn_grads(s, in(x), static_cast<size_t>(x_stride), in(gate_proj), in(up_proj), in(act), in(dout),
                           d_gate, d_up, g, st);
  return code_of(err);
}

int cernels_ffn_status(int* status, void* stream) {
  if (!status) return CERNELS_E_NULL;
  return code_of(ffn_status(status, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
