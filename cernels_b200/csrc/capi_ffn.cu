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

// Times that the weights are read for `tokens` rows of `k`; 0 when not even one row fits.
int passes_of(int tokens, int k, int group) {
  const int most = skinny_columns(kSkinnyMaxColumns, k, group, 0, 0);
  return most == 0 ? 0 : (tokens + most - 1) / most;
}

int balanced_columns(int tokens, int k, int group) {
  const int passes = passes_of(tokens, k, group);
  return passes == 0 ? 0 : (tokens + passes - 1) / passes;
}

// A few tokens: the weights' bytes bound the work, and the kernel that streams them (once per 16 tokens, or as
// many as shared memory holds) beats the tile kernel, whose time is a full tile's for any number. By how much
// more than once it may read them depends on whether L2 keeps them. us, streamed / tiled, at T tokens and that many reads:
//   50 MB (H = F = 2880)           T = 48, 3.0: 23.4 / 29.0    T = 64, 4.0: 35.0 / 29.0
//   100 MB (H = 8192, F = 2048)    T = 30, 2.7: 44.7 / 48.5    T = 32, 3.3: 47.3 / 45.3
//   100 MB (H = F = 4096)          T = 32, 2.0: 39.3 / 38.4    T = 48, 3.0: 54.8 / 38.7
//   302 MB (H = 6144, F = 8192)    T = 10, 1.0: 62.0 / 82.8    T = 20, 2.0: 95.8 / 71.6
//   402 MB (H = 4096, F = 16384)   T = 15, 1.7: 123.4 / 121.0
bool few(const cernels_ffn_shape* s) {
  if (s->tokens > 4 * kSkinnyMaxColumns) return false;
  const int gate_up = passes_of(s->tokens, s->hidden, 0), down = passes_of(s->tokens, s->intermediate, 0);
  if (gate_up == 0 || down == 0) return false;
  const long long weights = 6ll * s->hidden * s->intermediate;
  const int thirds = 2 * gate_up + down;  // of the weights' bytes that are read
  return thirds <= (weights <= (64ll << 20) ? 9 : weights <= (105ll << 20) ? 8 : 5);
}

int check_group(int group, int a, int b) {
  if (group != 32 && group != 64 && group != 128) return CERNELS_E_UNSUPPORTED;
  return a % group == 0 && b % group == 0 ? CERNELS_OK : CERNELS_E_INVALID_SHAPE;
}

int check_moe_w4(const cernels_moe_shape* s, int group) {
  if (!s) return CERNELS_E_NULL;
  if (s->tokens < 0 || s->hidden <= 0 || s->experts <= 0 || s->intermediate <= 0 || s->topk <= 0)
    return CERNELS_E_INVALID_SHAPE;
  if (s->layout != CERNELS_LAYOUT_LINEAR || s->experts > kMaxExperts) return CERNELS_E_UNSUPPORTED;
  if (static_cast<long long>(s->tokens) * s->topk > kDecodeMaxPairs) return CERNELS_E_UNSUPPORTED;
  if (s->hidden > (1 << 15) || s->intermediate > (1 << 15)) return CERNELS_E_UNSUPPORTED;
  const int rc = check_group(group, s->hidden, s->intermediate);
  if (rc) return rc;
  const int pairs = s->tokens * s->topk, longest = s->hidden > s->intermediate ? s->hidden : s->intermediate;
  return skinny_columns(1, longest, group, pairs, s->experts) ? CERNELS_OK : CERNELS_E_UNSUPPORTED;
}

struct MoeW4Workspace {
  __nv_bfloat16* act;  // [T * topk, F]
  float* rows;         // [T * topk, H]
  size_t bytes;
};
MoeW4Workspace carve_moe_w4(const cernels_moe_shape* s, void* base) {
  const size_t pairs = static_cast<size_t>(s->tokens) * s->topk;
  const size_t act = align_up(pairs * s->intermediate * 2, 256);
  uint8_t* p = static_cast<uint8_t*>(base);
  return {reinterpret_cast<__nv_bfloat16*>(p), reinterpret_cast<float*>(p + act), act + pairs * s->hidden * 4};
}

const uint8_t* bytes(const void* p) { return static_cast<const uint8_t*>(p); }
const uint16_t* halves(const void* p) { return static_cast<const uint16_t*>(p); }
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
  if (few(shape)) {
    SkinnyArgs a{};
    a.x = in(x);
    a.x_stride = static_cast<size_t>(x_stride);
    a.w0 = bytes(gate_proj);
    a.w1 = bytes(up_proj);
    a.out = workspace;
    a.out_stride = static_cast<size_t>(s.inter);
    a.k = s.hidden;
    a.rows = s.inter;
    a.tokens = s.tokens;
    a.cols = balanced_columns(s.tokens, s.hidden, 0);
    cudaError_t e = launch_skinny(a, 0, true, st);
    a.x = in(workspace);
    a.x_stride = static_cast<size_t>(s.inter);
    a.w0 = bytes(down_proj);
    a.w1 = nullptr;
    a.out = out;
    a.out_stride = static_cast<size_t>(s.hidden);
    a.k = s.inter;
    a.rows = s.hidden;
    a.cols = balanced_columns(s.tokens, s.inter, 0);
    a.x_from_previous = 1;
    if (e == cudaSuccess) e = launch_skinny(a, 0, false, st);
    return code_of(e);
  }
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

int cernels_linear_w4(int32_t tokens, int32_t out_features, int32_t in_features, int32_t group, const void* x,
                      int64_t x_stride, const void* qweight, const void* scales, void* out, void* stream) {
  if (tokens < 0 || out_features <= 0 || in_features <= 0) return CERNELS_E_INVALID_SHAPE;
  int rc = check_group(group, in_features, in_features);
  if (rc) return rc;
  if (in_features > (1 << 15) || out_features > (1 << 24)) return CERNELS_E_UNSUPPORTED;
  if (tokens == 0) return CERNELS_OK;
  if (!x || !qweight || !scales || !out) return CERNELS_E_NULL;
  if (!aligned(x) || !aligned(qweight) || x_stride % 8 != 0) return CERNELS_E_ALIGNMENT;
  // scales are copied in 4-byte words, outputs written one by one
  if ((reinterpret_cast<uintptr_t>(scales) & 3u) || (reinterpret_cast<uintptr_t>(out) & 1u)) return CERNELS_E_ALIGNMENT;
  if (x_stride < in_features) return CERNELS_E_INVALID_SHAPE;
  SkinnyArgs a{};
  a.x = in(x);
  a.x_stride = static_cast<size_t>(x_stride);
  a.w0 = bytes(qweight);
  a.s0 = halves(scales);
  a.out = out;
  a.out_stride = static_cast<size_t>(out_features);
  a.k = in_features;
  a.rows = out_features;
  a.tokens = tokens;
  a.cols = balanced_columns(tokens, in_features, group);
  if (a.cols == 0) return CERNELS_E_UNSUPPORTED;
  const long long units = (static_cast<long long>(tokens) / a.cols + 1) * (out_features / 16 + 1);
  if (units > 0x7fffffffll) return CERNELS_E_UNSUPPORTED;
  rc = check_sm100();
  if (rc) return rc;
  return code_of(launch_skinny(a, group, false, static_cast<cudaStream_t>(stream)));
}

int cernels_moe_w4_workspace_bytes(const cernels_moe_shape* shape, int32_t group, size_t* bytes) {
  const int rc = check_moe_w4(shape, group);
  if (rc) return rc;
  if (!bytes) return CERNELS_E_NULL;
  *bytes = carve_moe_w4(shape, nullptr).bytes;
  return CERNELS_OK;
}

int cernels_moe_experts_decode_w4(const cernels_moe_shape* shape, int32_t group, const void* x, const void* gate_up_q,
                                  const void* gate_up_scales, const void* down_q, const void* down_scales,
                                  const int32_t* indices, const float* weights, void* out, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  int rc = check_moe_w4(shape, group);
  if (rc || shape->tokens == 0) return rc;
  if (!x || !gate_up_q || !gate_up_scales || !down_q || !down_scales || !indices || !weights || !out)
    return CERNELS_E_NULL;
  for (const void* p : {x, gate_up_q, gate_up_scales, down_q, down_scales, const_cast<const void*>(out)})
    if (!aligned(p)) return CERNELS_E_ALIGNMENT;
  const MoeW4Workspace ws = carve_moe_w4(shape, workspace);
  if (!workspace || workspace_bytes < ws.bytes) return CERNELS_E_WORKSPACE;
  if (!aligned(workspace)) return CERNELS_E_ALIGNMENT;
  rc = check_sm100();
  if (rc) return rc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const size_t H = shape->hidden, F = shape->intermediate;
  SkinnyArgs a{};
  a.indices = indices;
  a.pairs = shape->tokens * shape->topk;
  a.topk = shape->topk;
  a.experts = shape->experts;
  a.tokens = shape->tokens;
  a.x = in(x);
  a.x_stride = H;
  a.w0 = bytes(gate_up_q);
  a.w1 = a.w0 + F * (H / 2);
  a.w_expert = 2 * F * (H / 2);
  a.s0 = halves(gate_up_scales);
  a.s1 = a.s0 + F * (H / group);
  a.s_expert = 2 * F * (H / group);
  a.out = ws.act;
  a.out_stride = F;
  a.k = shape->hidden;
  a.rows = shape->intermediate;
  // 4 columns are the cheapest tile; an expert with more pairs is read again for each 4 (or 8)
  const int want = a.pairs > 4 * a.experts ? 8 : 4;
  a.cols = skinny_columns(want, a.k, group, a.pairs, a.experts);
  cudaError_t err = launch_skinny(a, group, true, st);
  if (err != cudaSuccess) return code_of(err);
  a.x = ws.act;
  a.x_stride = F;
  a.x_by_pair = 1;
  a.w0 = bytes(down_q);
  a.w1 = nullptr;
  a.w_expert = H * (F / 2);
  a.s0 = halves(down_scales);
  a.s1 = nullptr;
  a.s_expert = H * (F / group);
  a.out = ws.rows;
  a.out_stride = H;
  a.k = shape->intermediate;
  a.rows = shape->hidden;
  a.cols = skinny_columns(want, a.k, group, a.pairs, a.experts);
  a.x_from_previous = 1;
  a.out_f32 = 1;
  err = launch_skinny(a, group, false, st);
  if (err == cudaSuccess)
    err = launch_weighted_rows(ws.rows, indices, weights, shape->tokens, shape->topk, shape->experts, shape->hidden,
                               outp(out), st);
  return code_of(err);
}

int cernels_ffn_status(int* status, void* stream) {
  if (!status) return CERNELS_E_NULL;
  return code_of(ffn_status(status, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
