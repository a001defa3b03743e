// Products of a few rows x with a tall matrix of bf16 or 4-bit weights: the feed-forward block at
// single tokens, 4-bit linear layers, and the routed experts' decode call in 4 bits.
//
//   y[t, n] = sum_k x[t, k] W[n, k];   4 bits: W[n, k] = (q[n, k] - 8) s[n, k / G]
//
// Each weight is used for at most 16 columns, so the work is bound by reading W once. A tile is 16
// rows of W (gate/up: 8 gate rows and the 8 up rows of the same outputs) over the whole reduction:
// the 8 warps of a CTA take its K steps in turn, so that neighbouring warps read neighbouring
// bytes, and add their sums in shared memory at the tile's end, in warp order. A CTA walks through
// a contiguous range of tiles with its x rows in shared memory and, per warp, the weights of the next
// kDepth steps already on their way into registers, across tile borders. 256 CTA threads at two CTAs
// per SM keep 64 KB of weights in flight per SM, about what HBM needs for its rate times its latency.
//
// mma.sync m16n8k16 does the products: rows of W are the A operand straight from the registers
// they were loaded into, x columns the B operand. The order of k within the reduction is free as long
// as A and B agree, so each lane takes 16 contiguous bytes of a row and x is stored to match.
// tcgen05 would need W in shared memory in its tile layout, a trip that 4-bit weights would make
// unpacked; the tensor work here is a few percent of the machine either way.
//
// 4 bits: two codes at a time become bf16 128 + q by (word >> 4 i) & 0x000f000f | 0x43004300, and q - 8 by
// one subtraction, all exact. Sums within a group are exact products added in 32 bits; the group's
// scale multiplies that sum in 32 bits, so weights are never rounded.
#include "ffn_internal.h"

namespace cernels {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kDepth = 4;
constexpr int kMaxSmem = 232448;          // per CTA
constexpr int kXSmem = 160 * 1024;        // of it for x rows; the rest holds sums and the largest lists
constexpr int kTwoCtaSmem = 112 * 1024;   // a CTA within this shares its SM with another

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes i and i + 4 of a word of eight, as the bf16 pair (q_i - 8, q_{i+4} - 8).
__device__ __forceinline__ uint32_t codes(uint32_t word, int i) {
  const uint32_t v = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // 128 + q
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.0f));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kFmt 0: bf16 weights; 32, 64, 128: 4-bit weights with that group size. One K step is what a quad of
// lanes reads as 64 contiguous bytes of a row.
template <int kFmt>
struct Format {
  static constexpr int kStep = kFmt == 0 ? 32 : 128;
  static constexpr int kGroups = kFmt == 0 ? 1 : 128 / kFmt;  // per step
  static constexpr int kWords = kFmt == 0 ? 1 : kFmt / 32;    // 8-code words per lane and group
};

// Weights of one step of one row that this lane holds, with the scale it fetched for its quad.
template <int kFmt>
struct Piece {
  uint4 w;
  uint16_t scale;
};

// Bytes in a shared-memory row of x: steps * kStep bf16, an odd multiple of 64 so that the 8 lanes of
// a 16-byte access phase (two rows, four pieces each) fall into different banks.
__host__ __device__ constexpr int x_row_bytes(int padded_k) {
  return padded_k * 2 % 128 == 0 ? padded_k * 2 + 64 : padded_k * 2;
}

struct Item {
  int expert, first, count;  // columns: order[first .. first + count)
};

struct SkinnySmem {
  size_t part, x, count, base, rank, order, items, total;
};

__host__ __device__ inline SkinnySmem carve_smem(int cols, int padded_k, int pairs, int experts) {
  SkinnySmem s;
  size_t off = 0;
  s.part = off;
  off += static_cast<size_t>(2) * kWarps * ((cols + 7) / 8 * 8) * 16 * 4;
  s.x = off;
  off += static_cast<size_t>(cols) * x_row_bytes(padded_k);
  s.count = off;  // the lists exist only with routing
  off += static_cast<size_t>(experts) * 4;
  s.base = off;
  off += static_cast<size_t>(experts) * 4;
  s.items = off;
  off += static_cast<size_t>(pairs) * sizeof(Item);
  s.rank = off;
  off += static_cast<size_t>(pairs) * 2;
  s.order = off;
  off += static_cast<size_t>(pairs) * 2;
  s.total = off + 16;
  return s;
}

// Groups the (token, slot) pairs by expert, experts in order of first use and pairs in their own
// order, into items of at most `cols` columns. Every CTA does this for itself. Returns the items.
__device__ int build_items(const SkinnyArgs& a, uint8_t* smem, const SkinnySmem& lay) {
  int* count = reinterpret_cast<int*>(smem + lay.count);
  int* base = reinterpret_cast<int*>(smem + lay.base);
  uint16_t* rank = reinterpret_cast<uint16_t*>(smem + lay.rank);
  uint16_t* order = reinterpret_cast<uint16_t*>(smem + lay.order);
  Item* items = reinterpret_cast<Item*>(smem + lay.items);
  int* n_items = reinterpret_cast<int*>(smem + lay.total - 16);
  for (int i = threadIdx.x; i < a.experts; i += kThreads) count[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  if (threadIdx.x < 32) {
    for (int p0 = 0; p0 < a.pairs; p0 += 32) {
      const int p = p0 + lane;
      const int e = p < a.pairs ? a.indices[p] : -1;
      const bool live = e >= 0 && e < a.experts;
      const unsigned same = __match_any_sync(0xffffffffu, live ? e : -1);
      const int before = live ? count[e] : 0;
      const int mine = __popc(same & ((1u << lane) - 1u));
      if (live) rank[p] = static_cast<uint16_t>(before + mine);
      __syncwarp();
      if (live && mine == 0) count[e] = before + __popc(same);
      __syncwarp();
    }
    int pos = 0, item = 0;
    for (int p0 = 0; p0 < a.pairs; p0 += 32) {
      const int p = p0 + lane;
      const int e = p < a.pairs ? a.indices[p] : -1;
      const bool first = e >= 0 && e < a.experts && rank[p] == 0;
      const int n = first ? count[e] : 0;
      const int parts = (n + a.cols - 1) / a.cols;
      int pos_incl = n, item_incl = parts;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, pos_incl, d), w = __shfl_up_sync(0xffffffffu, item_incl, d);
        if (lane >= d) {
          pos_incl += v;
          item_incl += w;
        }
      }
      if (first) {
        const int at = pos + pos_incl - n, it = item + item_incl - parts;
        base[e] = at;
        for (int i = 0; i < parts; ++i) items[it + i] = Item{e, at + i * a.cols, min(a.cols, n - i * a.cols)};
      }
      pos += __shfl_sync(0xffffffffu, pos_incl, 31);
      item += __shfl_sync(0xffffffffu, item_incl, 31);
    }
    if (lane == 0) *n_items = item;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += kThreads) {
    const int e = a.indices[p];
    if (e >= 0 && e < a.experts) order[base[e] + rank[p]] = static_cast<uint16_t>(p);
  }
  const int n = *n_items;
  __syncthreads();
  return n;
}

template <int kFmt, bool kGateUp, int NT, bool kOutF32>
__global__ void __launch_bounds__(kThreads, 2) skinny_kernel(const SkinnyArgs a) {
  using F = Format<kFmt>;
  extern __shared__ __align__(16) uint8_t smem[];
  let_next_kernel_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;  // mma row (and x column) of this lane, its quarter of a step
  const int steps = (a.k + F::kStep - 1) / F::kStep;
  const int per_warp = (steps + kWarps - 1) / kWarps;
  const int padded_k = steps * F::kStep;
  const int x_bytes = x_row_bytes(padded_k);
  const bool routed = a.indices != nullptr;
  const SkinnySmem lay = carve_smem(a.cols, padded_k, routed ? a.pairs : 0, routed ? a.experts : 0);
  float* part = reinterpret_cast<float*>(smem + lay.part);
  uint8_t* xs = smem + lay.x;
  const Item* items = reinterpret_cast<const Item*>(smem + lay.items);
  const uint16_t* order = reinterpret_cast<const uint16_t*>(smem + lay.order);

  const int n_items = routed ? build_items(a, smem, lay) : (a.tokens + a.cols - 1) / a.cols;
  const int tiles = kGateUp ? (a.rows + 7) / 8 : (a.rows + 15) / 16;
  const long long units = static_cast<long long>(n_items) * tiles;
  const int begin = static_cast<int>(units * blockIdx.x / gridDim.x);
  const int end = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
  if (begin >= end) {
    if (a.dependent) wait_for_previous_kernel();  // this kernel never ends before the one it follows
    return;
  }

  auto item_of = [&](int i) {
    return routed ? items[i] : Item{0, i * a.cols, min(a.cols, a.tokens - i * a.cols)};
  };

  // ---- weights: this lane's two rows of a unit, and the stream of steps through them
  const size_t row_bytes = kFmt == 0 ? static_cast<size_t>(a.k) * 2 : static_cast<size_t>(a.k) / 2;
  const int row_groups = kFmt == 0 ? 0 : a.k / (kFmt == 0 ? 1 : kFmt);
  const uint8_t *wa = nullptr, *wb = nullptr;
  const uint16_t *sa = nullptr, *sb = nullptr;
  auto point = [&](int unit) {
    const int it = unit / tiles, tile = unit - it * tiles;
    const int e = routed ? items[it].expert : 0;
    const int ra = min(kGateUp ? tile * 8 + g : tile * 16 + g, a.rows - 1);
    const int rb = kGateUp ? ra : min(tile * 16 + 8 + g, a.rows - 1);
    const uint8_t* second = kGateUp ? a.w1 : a.w0;
    wa = a.w0 + static_cast<size_t>(e) * a.w_expert + static_cast<size_t>(ra) * row_bytes;
    wb = second + static_cast<size_t>(e) * a.w_expert + static_cast<size_t>(rb) * row_bytes;
    if constexpr (kFmt != 0) {
      const uint16_t* s_second = kGateUp ? a.s1 : a.s0;
      sa = a.s0 + static_cast<size_t>(e) * a.s_expert + static_cast<size_t>(ra) * row_groups;
      sb = s_second + static_cast<size_t>(e) * a.s_expert + static_cast<size_t>(rb) * row_groups;
    }
  };
  auto fetch = [&](const uint8_t* w, const uint16_t* s, int step) {
    Piece<kFmt> p;
    p.w = make_uint4(0, 0, 0, 0);
    p.scale = 0;
    if constexpr (kFmt == 0) {
      const int k = step * 32 + q * 8;
      if (k < a.k) p.w = __ldcs(reinterpret_cast<const uint4*>(w + static_cast<size_t>(k) * 2));
    } else {
      const int group = step * F::kGroups;
      const uint8_t* src = w + static_cast<size_t>(step) * 64;
      if constexpr (kFmt == 128) {
        if (group < row_groups) p.w = __ldcs(reinterpret_cast<const uint4*>(src) + q);
      } else if constexpr (kFmt == 64) {
        uint2 v[2] = {make_uint2(0, 0), make_uint2(0, 0)};
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (group + i < row_groups) v[i] = __ldcs(reinterpret_cast<const uint2*>(src + 32 * i) + q);
        p.w = make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
      } else {
        uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (group + i < row_groups) v[i] = __ldcs(reinterpret_cast<const uint32_t*>(src + 16 * i) + q);
        p.w = make_uint4(v[0], v[1], v[2], v[3]);
      }
      const int mine = group + (q % F::kGroups);
      if (mine < row_groups) p.scale = __ldg(s + mine);
    }
    return p;
  };

  Piece<kFmt> pa[kDepth], pb[kDepth];
  int load_unit = begin, load_i = 0;
  point(begin);
  auto issue = [&](int d) {
    if (load_unit >= end) return;
    const int step = load_i * kWarps + warp;
    pa[d] = fetch(wa, sa, step);
    pb[d] = fetch(wb, sb, step);
    if (++load_i == per_warp) {
      load_i = 0;
      if (++load_unit < end) point(load_unit);
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) issue(d);

  if (a.dependent) wait_for_previous_kernel();  // x is the previous kernel's output

  // ---- x rows of an item, 8 values at a time, in the order in which the weights lie in the lanes
  auto load_x = [&](const Item& it) {
    const int pieces = padded_k / 8;
    for (int i = threadIdx.x; i < it.count * pieces; i += kThreads) {
      const int c = i / pieces, k8 = i - c * pieces;
      int row = it.first + c;
      if (routed) {
        row = order[row];
        if (!a.x_by_pair) row /= a.topk;
      }
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k8 * 8 < a.k) v = *reinterpret_cast<const uint4*>(a.x + static_cast<size_t>(row) * a.x_stride + k8 * 8);
      int at = k8;
      if constexpr (kFmt != 0) {
        // group | quarter | word  ->  group | word | quarter, and pairs (i, i + 4)
        constexpr int kPer = kFmt / 8;  // pieces per group
        const int in = k8 % kPer;
        at = k8 - in + (in % F::kWords) * 4 + in / F::kWords;
        v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                       __byte_perm(v.y, v.w, 0x7632));
      }
      *reinterpret_cast<uint4*>(xs + static_cast<size_t>(c) * x_bytes + at * 16) = v;
    }
  };
  int item_index = begin / tiles;
  Item item = item_of(item_index);
  load_x(item);
  __syncthreads();

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  int unit = begin, i = 0, buffer = 0;
  while (unit < end) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (unit >= end) break;
      const Piece<kFmt> va = pa[d], vb = pb[d];
      const int step = i * kWarps + warp;
      if (step < steps) {
        const uint8_t* xrow = xs + static_cast<size_t>(step) * (F::kStep * 2) + q * 16;
        const uint32_t aw[4] = {va.w.x, va.w.y, va.w.z, va.w.w}, bw[4] = {vb.w.x, vb.w.y, vb.w.z, vb.w.w};
        if constexpr (kFmt == 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int c = n * 8 + g;
            uint4 x4 = make_uint4(0, 0, 0, 0);
            if (c < item.count) x4 = *reinterpret_cast<const uint4*>(xrow + static_cast<size_t>(c) * x_bytes);
            mma_bf16(acc[n], aw[0], bw[0], aw[1], bw[1], x4.x, x4.y);
            mma_bf16(acc[n], aw[2], bw[2], aw[3], bw[3], x4.z, x4.w);
          }
        } else {
#pragma unroll
          for (int s = 0; s < F::kGroups; ++s) {
            float sum[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) sum[n][j] = 0.f;
#pragma unroll
            for (int w = 0; w < F::kWords; ++w) {
              const uint32_t wa4 = aw[s * F::kWords + w], wb4 = bw[s * F::kWords + w];
              const uint32_t a0 = codes(wa4, 0), a1 = codes(wa4, 1), a2 = codes(wa4, 2), a3 = codes(wa4, 3);
              const uint32_t b0 = codes(wb4, 0), b1 = codes(wb4, 1), b2 = codes(wb4, 2), b3 = codes(wb4, 3);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const int c = n * 8 + g;
                uint4 x4 = make_uint4(0, 0, 0, 0);
                if (c < item.count)
                  x4 = *reinterpret_cast<const uint4*>(xrow + static_cast<size_t>(c) * x_bytes +
                                                       (s * F::kWords + w) * 64);
                mma_bf16(sum[n], a0, b0, a1, b1, x4.x, x4.y);
                mma_bf16(sum[n], a2, b2, a3, b3, x4.z, x4.w);
              }
            }
            const int from = (lane & ~3) | (s % F::kGroups);
            const float fa = __uint_as_float(static_cast<uint32_t>(__shfl_sync(0xffffffffu, static_cast<int>(va.scale), from)) << 16);
            const float fb = __uint_as_float(static_cast<uint32_t>(__shfl_sync(0xffffffffu, static_cast<int>(vb.scale), from)) << 16);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              acc[n][0] += fa * sum[n][0];
              acc[n][1] += fa * sum[n][1];
              acc[n][2] += fb * sum[n][2];
              acc[n][3] += fb * sum[n][3];
            }
          }
        }
      }
      issue(d);
      if (++i < per_warp) continue;

      // ---- end of the tile: add the warps' sums (in warp order) and write
      i = 0;
      constexpr int kCols = NT * 8;
      float* mine = part + (buffer * kWarps + warp) * kCols * 16;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float* p = mine + (n * 8 + 2 * q) * 16 + g;
        p[0] = acc[n][0];
        p[16] = acc[n][1];
        p[8] = acc[n][2];
        p[24] = acc[n][3];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
      }
      __syncthreads();
      const float* all = part + buffer * kWarps * kCols * 16;
      const int tile = unit - item_index * tiles;
      constexpr int kOut = kGateUp ? 8 : 16;  // outputs per column
      const int r = threadIdx.x % kOut, c = threadIdx.x / kOut;
      const int row = tile * kOut + r;
      if (c < item.count && row < a.rows) {
        float v = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          v += all[(w * kCols + c) * 16 + r];
          if constexpr (kGateUp) u += all[(w * kCols + c) * 16 + 8 + r];
        }
        if constexpr (kGateUp) v = v * sigmoid(v) * u;
        const size_t at = static_cast<size_t>(routed ? order[item.first + c] : item.first + c) * a.out_stride + row;
        if constexpr (kOutF32)
          static_cast<float*>(a.out)[at] = v;
        else
          static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
      }
      buffer ^= 1;
      ++unit;
      if (unit < end && unit / tiles != item_index) {  // every warp has used the old x rows
        item_index = unit / tiles;
        item = item_of(item_index);
        load_x(item);
        __syncthreads();
      }
    }
  }
}

// out[t] = sum_j weights[t, j] rows[t * topk + j] over the slots whose expert exists, in slot order.
__global__ void __launch_bounds__(256) weighted_rows_kernel(const float* rows, const int32_t* indices,
                                                            const float* weights, int topk, int experts, int hidden,
                                                            __nv_bfloat16* out) {
  const int h = (blockIdx.x * 256 + threadIdx.x) * 4;
  const size_t t = blockIdx.y;
  wait_for_previous_kernel();
  if (h >= hidden) return;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j < topk; ++j) {
    const int e = indices[t * topk + j];
    if (e < 0 || e >= experts) continue;
    const float w = weights[t * topk + j];
    const float4 v = *reinterpret_cast<const float4*>(rows + (t * topk + j) * hidden + h);
    sum.x += w * v.x;
    sum.y += w * v.y;
    sum.z += w * v.z;
    sum.w += w * v.w;
  }
  __nv_bfloat162 lo = __floats2bfloat162_rn(sum.x, sum.y), hi = __floats2bfloat162_rn(sum.z, sum.w);
  uint2 v;
  v.x = *reinterpret_cast<uint32_t*>(&lo);
  v.y = *reinterpret_cast<uint32_t*>(&hi);
  *reinterpret_cast<uint2*>(out + t * hidden + h) = v;
}

template <class K, class... A>
cudaError_t launch_kernel(K kernel, dim3 grid, int threads, size_t smem, bool dependent, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <int kFmt, bool kGateUp, int NT, bool kOutF32>
cudaError_t launch_tile(SkinnyArgs a, cudaStream_t stream) {
  const int step = Format<kFmt>::kStep;
  const int padded_k = (a.k + step - 1) / step * step;
  const bool routed = a.indices != nullptr;
  const SkinnySmem lay = carve_smem(a.cols, padded_k, routed ? a.pairs : 0, routed ? a.experts : 0);
  static PerDeviceOnce attr;
  cudaError_t err = attr.run([] {
    return cudaFuncSetAttribute(skinny_kernel<kFmt, kGateUp, NT, kOutF32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kMaxSmem);
  });
  if (err != cudaSuccess) return err;
  const long long tiles = kGateUp ? (a.rows + 7) / 8 : (a.rows + 15) / 16;
  const long long most = (routed ? a.pairs : (a.tokens + a.cols - 1) / a.cols) * tiles;
  const int slots = device_sm_count() * (lay.total <= kTwoCtaSmem ? 2 : 1);
  const int grid = static_cast<int>(most < slots ? most : slots);
  return launch_kernel(skinny_kernel<kFmt, kGateUp, NT, kOutF32>, dim3(grid), kThreads, lay.total, a.dependent != 0,
                       stream, a);
}

template <bool kGateUp, bool kOutF32>
cudaError_t launch_format(const SkinnyArgs& a, int group, cudaStream_t stream) {
  const bool wide = a.cols > 8;
  switch (group) {
    case 0: return wide ? launch_tile<0, kGateUp, 2, kOutF32>(a, stream) : launch_tile<0, kGateUp, 1, kOutF32>(a, stream);
    case 32: return wide ? launch_tile<32, kGateUp, 2, kOutF32>(a, stream) : launch_tile<32, kGateUp, 1, kOutF32>(a, stream);
    case 64: return wide ? launch_tile<64, kGateUp, 2, kOutF32>(a, stream) : launch_tile<64, kGateUp, 1, kOutF32>(a, stream);
    case 128:
      return wide ? launch_tile<128, kGateUp, 2, kOutF32>(a, stream) : launch_tile<128, kGateUp, 1, kOutF32>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int skinny_columns(int want, int k) {
  const int row = x_row_bytes((k + 127) / 128 * 128);
  const int fit = kXSmem / row;
  const int cols = want < fit ? want : fit;
  return cols < kSkinnyMaxColumns ? cols : kSkinnyMaxColumns;
}

cudaError_t launch_skinny(const SkinnyArgs& a, int group, bool gate_up, bool out_f32, cudaStream_t stream) {
  if (a.cols < 1 || a.cols > kSkinnyMaxColumns) return cudaErrorInvalidValue;
  if (gate_up) return out_f32 ? cudaErrorInvalidValue : launch_format<true, false>(a, group, stream);
  return out_f32 ? launch_format<false, true>(a, group, stream) : launch_format<false, false>(a, group, stream);
}

cudaError_t launch_weighted_rows(const float* rows, const int32_t* indices, const float* weights, int tokens, int topk,
                                 int experts, int hidden, __nv_bfloat16* out, cudaStream_t stream) {
  return launch_kernel(weighted_rows_kernel, dim3((hidden / 4 + 255) / 256, tokens), 256, 0, true, stream, rows, indices,
                       weights, topk, experts, hidden, out);
}

}  // namespace cernels
