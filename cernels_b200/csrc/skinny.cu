// Products of a few rows x with a tall matrix of bf16 or 4-bit weights: the feed-forward block at
// single tokens, 4-bit linear layers, and the routed experts' decode call in 4 bits.
//
//   y[t, n] = sum_k x[t, k] W[n, k];   4 bits: W[n, k] = (q[n, k] - 8) s[n, k / G]
//
// Each weight is used for at most 16 columns, so the work is bound by reading W once. A tile is 16
// rows of W (gate/up: 8 gate rows and the 8 up rows of the same outputs); a CTA's 8 warps take
// 8 / KW tiles at once, KW warps to a tile: these take the tile's K steps in turn, so that
// neighbouring warps read neighbouring bytes, and their sums are added in shared memory in warp order. A
// CTA walks through a contiguous range of tiles with its x rows in shared memory and, per warp, the
// weights of the next kDepth steps already on their way into registers, across tile borders:
// up to 128 KB of weights in flight per SM.
//
// mma.sync m16n8k16 does the products: rows of W are the A operand straight from the registers
// they were loaded into, x columns the B operand. The order of k within the reduction is free as long
// as A and B agree, so each lane takes 16 contiguous bytes of a row and x is stored to match.
// tcgen05 would need W in shared memory in its tile layout, a trip that 4-bit weights would make
// unpacked; the tensor pipe is a small part of the time either way.
//
// 4 bits: two codes at a time become the bf16 pair 128 + q by (word >> 4 i) & 0x000f000f | 0x43004300,
// exactly. A group's sum starts at -136 sum(x) instead of 0, which turns every 128 + q into q - 8
// without an instruction per weight; it is exact products added in 32 bits, and the group's scale
// multiplies it in 32 bits, so weights are never rounded. (Subtracting 136 from each pair instead
// made the kernel issue-bound: 241 instructions per 16 x 128 weights where HBM's rate leaves 180.)
#include "ffn_internal.h"

namespace cernels {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kMaxSmem = 232448;          // per CTA
constexpr int kTwoCtaSmem = 112 * 1024;   // a CTA within this shares its SM with another

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes i and i + 4 of a word of eight, as the bf16 pair (128 + q_i, 128 + q_{i+4}).
__device__ __forceinline__ uint32_t codes(uint32_t word, int i) { return ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u; }
constexpr float kCodeOffset = 136.0f;  // 128 + 8

__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// kFmt 0: bf16 weights; 32, 64, 128: 4-bit weights with that group size. A K step is 128 bytes of a
// row in two halves, of which a quad of lanes reads 4 x 16 bytes each.
template <int kFmt>
struct Format {
  static constexpr int kHalf = kFmt == 0 ? 32 : 128;
  static constexpr int kStep = 2 * kHalf;
  static constexpr int kGroups = kFmt == 0 ? 1 : 128 / kFmt;  // per half
  static constexpr int kWords = kFmt == 0 ? 1 : kFmt / 32;    // 8-code words per lane and group
  static constexpr int kDepth = kFmt == 0 || kFmt == 128 ? 4 : 3;
};

// One step of one row, as a lane holds it: 16 bytes of each half, and the scales it fetched for its
// quad (low and high half of a word: consecutive groups).
struct Piece {
  uint4 w[2];
  uint32_t scale;
};

// Bytes in a shared-memory row of x: an odd multiple of 64, so that the 8 lanes of a 16-byte
// access phase (two rows, four pieces each) fall into different banks.
__host__ __device__ constexpr int x_row_bytes(int padded_k) {
  return padded_k * 2 % 128 == 0 ? padded_k * 2 + 64 : padded_k * 2;
}

struct Item {
  int expert, first, count;  // columns: order[first .. first + count)
};

struct SkinnySmem {
  size_t part, sums, x, count, base, rank, order, items, total;
};

// groups: scale groups in padded_k (0 for bf16)
__host__ __device__ inline SkinnySmem carve_smem(int cols, int padded_k, int groups, int pairs, int experts) {
  SkinnySmem s;
  size_t off = 0;
  s.part = off;
  off += static_cast<size_t>(2) * kWarps * ((cols + 7) / 8 * 8) * 16 * 4;
  s.sums = off;  // [group][column]: -136 times the group's sum of x
  off += static_cast<size_t>(groups) * ((cols + 7) / 8 * 8) * 4;
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
  constexpr int kDepth = F::kDepth;
  constexpr int kCols = NT * 8;
  constexpr int kOut = kGateUp ? 8 : 16;  // outputs per tile and column
  extern __shared__ __align__(16) uint8_t smem[];
  let_next_kernel_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;  // mma row (and x column) of this lane, its quarter of a half step
  const int kw = warp % a.k_warps, rt = warp / a.k_warps;
  const int tiles_at_once = kWarps / a.k_warps;
  const int steps = (a.k + F::kStep - 1) / F::kStep;
  const int per_warp = (steps + a.k_warps - 1) / a.k_warps;
  const int padded_k = steps * F::kStep;
  const int x_bytes = x_row_bytes(padded_k);
  const bool routed = a.indices != nullptr;
  const SkinnySmem lay = carve_smem(a.cols, padded_k, kFmt == 0 ? 0 : padded_k / (kFmt == 0 ? 1 : kFmt),
                                    routed ? a.pairs : 0, routed ? a.experts : 0);
  float* part = reinterpret_cast<float*>(smem + lay.part);
  float* sums = reinterpret_cast<float*>(smem + lay.sums);
  uint8_t* xs = smem + lay.x;
  const Item* items = reinterpret_cast<const Item*>(smem + lay.items);
  const uint16_t* order = reinterpret_cast<const uint16_t*>(smem + lay.order);

  const int n_items = routed ? build_items(a, smem, lay) : (a.tokens + a.cols - 1) / a.cols;
  const int per_item = (a.rows + kOut * tiles_at_once - 1) / (kOut * tiles_at_once);  // units of an item
  const long long units = static_cast<long long>(n_items) * per_item;
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
  int load_item = begin / per_item, load_unit = begin - load_item * per_item;  // position of the stream
  int load_left = (end - begin) * per_warp, load_step = kw;
  const uint8_t *wa = nullptr, *wb = nullptr;
  const uint16_t *sa = nullptr, *sb = nullptr;
  auto point = [&] {
    const int e = routed ? items[load_item].expert : 0;
    const int first = (load_unit * tiles_at_once + rt) * kOut + g;
    const int ra = min(first, a.rows - 1);
    const int rb = kGateUp ? ra : min(first + 8, a.rows - 1);
    const uint8_t* second = kGateUp ? a.w1 : a.w0;
    wa = a.w0 + static_cast<size_t>(e) * a.w_expert + static_cast<size_t>(ra) * row_bytes + q * (kFmt == 0 ? 16 : kFmt / 8);
    wb = second + static_cast<size_t>(e) * a.w_expert + static_cast<size_t>(rb) * row_bytes + q * (kFmt == 0 ? 16 : kFmt / 8);
    if constexpr (kFmt != 0) {
      const uint16_t* s_second = kGateUp ? a.s1 : a.s0;
      sa = a.s0 + static_cast<size_t>(e) * a.s_expert + static_cast<size_t>(ra) * row_groups;
      sb = s_second + static_cast<size_t>(e) * a.s_expert + static_cast<size_t>(rb) * row_groups;
    }
  };
  // Lane q holds the 16 (128-code groups), 8 (64) or 4 bytes (32) of its quarter of every group, so
  // that an mma never spans two groups.
  auto fetch = [&](const uint8_t* w, const uint16_t* s, int step) {
    Piece p;
    const uint8_t* src = w + static_cast<size_t>(step) * 128;
    p.scale = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      p.w[h] = make_uint4(0, 0, 0, 0);
      if constexpr (kFmt == 0) {
        if (step * 64 + h * 32 + q * 8 < a.k) p.w[h] = __ldcs(reinterpret_cast<const uint4*>(src + h * 64));
      } else {
        const int left = row_groups - (2 * step + h) * F::kGroups;  // groups from this half on
        if constexpr (kFmt == 128) {
          if (left > 0) p.w[h] = __ldcs(reinterpret_cast<const uint4*>(src + h * 64));
        } else if constexpr (kFmt == 64) {
          uint2 v[2] = {make_uint2(0, 0), make_uint2(0, 0)};
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (i < left) v[i] = __ldcs(reinterpret_cast<const uint2*>(src + h * 64 + 32 * i));
          p.w[h] = make_uint4(v[0].x, v[0].y, v[1].x, v[1].y);
        } else {
          uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < left) v[i] = __ldcs(reinterpret_cast<const uint32_t*>(src + h * 64 + 16 * i));
          p.w[h] = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    }
    if constexpr (kFmt != 0) {
      // a step has 2, 4 or 8 groups per row: lane q of the quad fetches one, or two neighbours
      const int first = step * 2 * F::kGroups;
      if constexpr (kFmt == 32) {
        const int at = first + 2 * q;
        if (at < row_groups) p.scale = __ldg(s + at);
        if (at + 1 < row_groups) p.scale |= static_cast<uint32_t>(__ldg(s + at + 1)) << 16;
      } else {
        const int at = first + (q % (2 * F::kGroups));
        if (at < row_groups) p.scale = __ldg(s + at);
      }
    }
    return p;
  };
  // scale of group i of the step (0 .. 2 kGroups - 1) from the lane of the quad that fetched it
  auto scale_of = [&](const Piece& p, int i) {
    if constexpr (kFmt == 32) {
      const uint32_t v = __shfl_sync(0xffffffffu, p.scale, (lane & ~3) | (i >> 1));
      return __uint_as_float(i & 1 ? v & 0xffff0000u : v << 16);
    } else {
      return __uint_as_float(__shfl_sync(0xffffffffu, p.scale, (lane & ~3) | i) << 16);
    }
  };

  Piece pa[kDepth], pb[kDepth];
  point();
  auto issue = [&](int d) {
    if (load_left == 0) return;
    pa[d] = fetch(wa, sa, load_step);
    pb[d] = fetch(wb, sb, load_step);
    --load_left;
    load_step += a.k_warps;
    if (load_step - kw == per_warp * a.k_warps) {
      load_step = kw;
      if (++load_unit == per_item) {
        load_unit = 0;
        ++load_item;
      }
      if (load_left != 0) point();
    }
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) issue(d);

  if (a.dependent) wait_for_previous_kernel();  // x is the previous kernel's output

  // ---- x rows of an item, 8 values at a time, in the order in which the weights lie in the lanes
  auto load_x = [&](const Item& it) {
    const int pieces = padded_k / 8;  // a multiple of 32 with 4-bit weights: a warp stays within a row
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
        constexpr int kPer = kFmt / 8;  // pieces (lanes here) per group
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t u = j == 0 ? v.x : j == 1 ? v.y : j == 2 ? v.z : v.w;
          sum += __uint_as_float(u << 16) + __uint_as_float(u & 0xffff0000u);
        }
#pragma unroll
        for (int d = kPer / 2; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        const int in = k8 % kPer;
        if (in == 0) sums[(k8 / kPer) * kCols + c] = -kCodeOffset * sum;
        // group | quarter | word  ->  group | word | quarter, and pairs (i, i + 4)
        at = k8 - in + (in % F::kWords) * 4 + in / F::kWords;
        v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                       __byte_perm(v.y, v.w, 0x7632));
      }
      *reinterpret_cast<uint4*>(xs + static_cast<size_t>(c) * x_bytes + at * 16) = v;
    }
  };
  int item_index = begin / per_item, unit = begin - item_index * per_item;
  Item item = item_of(item_index);
  load_x(item);
  __syncthreads();
  // Columns past the item's last read its last one again: their sums are never used.
  const uint8_t* xcol[NT];
  auto point_x = [&] {
#pragma unroll
    for (int n = 0; n < NT; ++n) xcol[n] = xs + static_cast<size_t>(min(n * 8 + g, item.count - 1)) * x_bytes + q * 16;
  };
  point_x();

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  int units_left = end - begin, i = 0, buffer = 0;
  while (true) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      const Piece va = pa[d], vb = pb[d];
      const int step = i * a.k_warps + kw;
      if (step < steps) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int x_at = (step * 2 + h) * (F::kHalf * 2);
          const uint32_t aw[4] = {va.w[h].x, va.w[h].y, va.w[h].z, va.w[h].w};
          const uint32_t bw[4] = {vb.w[h].x, vb.w[h].y, vb.w[h].z, vb.w[h].w};
          if constexpr (kFmt == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 x4 = *reinterpret_cast<const uint4*>(xcol[n] + x_at);
              mma_bf16(acc[n], aw[0], bw[0], aw[1], bw[1], x4.x, x4.y);
              mma_bf16(acc[n], aw[2], bw[2], aw[3], bw[3], x4.z, x4.w);
            }
          } else {
#pragma unroll
            for (int s = 0; s < F::kGroups; ++s) {
              float sum[NT][4];
              const int group = (step * 2 + h) * F::kGroups + s;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const float2 start = *reinterpret_cast<const float2*>(sums + group * kCols + n * 8 + 2 * q);
                sum[n][0] = sum[n][2] = start.x;
                sum[n][1] = sum[n][3] = start.y;
              }
#pragma unroll
              for (int w = 0; w < F::kWords; ++w) {
                const uint32_t u = aw[s * F::kWords + w], v = bw[s * F::kWords + w];
                const uint32_t a0 = codes(u, 0), a1 = codes(u, 1), a2 = codes(u, 2), a3 = codes(u, 3);
                const uint32_t b0 = codes(v, 0), b1 = codes(v, 1), b2 = codes(v, 2), b3 = codes(v, 3);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                  const uint4 x4 = *reinterpret_cast<const uint4*>(xcol[n] + x_at + (s * F::kWords + w) * 64);
                  mma_bf16(sum[n], a0, b0, a1, b1, x4.x, x4.y);
                  mma_bf16(sum[n], a2, b2, a3, b3, x4.z, x4.w);
                }
              }
              const float fa = scale_of(va, h * F::kGroups + s), fb = scale_of(vb, h * F::kGroups + s);
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
      }
      issue(d);
      if (++i < per_warp) continue;

      // ---- end of the unit: add the sums of each tile's warps (in warp order) and write
      i = 0;
      float* mine = part + ((buffer * kWarps + warp) * kCols + 2 * q) * 16 + g;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mine[n * 128] = acc[n][0];
        mine[n * 128 + 16] = acc[n][1];
        mine[n * 128 + 8] = acc[n][2];
        mine[n * 128 + 24] = acc[n][3];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
      }
      __syncthreads();
      const float* all = part + buffer * kWarps * kCols * 16;
      // the half of the warps that adds first alternates, as there may be work for one half only
      for (int o = (threadIdx.x + buffer * (kThreads / 2)) % kThreads; o < tiles_at_once * kOut * kCols; o += kThreads) {
        const int r = o % kOut, c = o / kOut % kCols, t = o / (kOut * kCols);
        const int row = (unit * tiles_at_once + t) * kOut + r;
        if (c >= item.count || row >= a.rows) continue;
        const float* from = all + (t * a.k_warps * kCols + c) * 16 + r;
        float v = 0.f, u = 0.f;
        for (int w = 0; w < a.k_warps; ++w) {
          v += from[w * kCols * 16];
          if constexpr (kGateUp) u += from[w * kCols * 16 + 8];
        }
        if constexpr (kGateUp) v = v * sigmoid(v) * u;
        const size_t at = static_cast<size_t>(routed ? order[item.first + c] : item.first + c) * a.out_stride + row;
        if constexpr (kOutF32)
          static_cast<float*>(a.out)[at] = v;
        else
          static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
      }
      buffer ^= 1;
      if (--units_left == 0) return;
      if (++unit == per_item) {  // the next item's x rows; every warp has used the old ones
        unit = 0;
        item = item_of(++item_index);
        load_x(item);
        __syncthreads();
        point_x();
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
  const int steps = (a.k + step - 1) / step;
  const bool routed = a.indices != nullptr;
  const SkinnySmem lay = carve_smem(a.cols, steps * step, kFmt == 0 ? 0 : steps * step / (kFmt == 0 ? 1 : kFmt),
                                    routed ? a.pairs : 0, routed ? a.experts : 0);
  if (lay.total > kMaxSmem) return cudaErrorInvalidValue;
  static PerDeviceOnce attr;
  cudaError_t err = attr.run([] {
    return cudaFuncSetAttribute(skinny_kernel<kFmt, kGateUp, NT, kOutF32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                kMaxSmem);
  });
  if (err != cudaSuccess) return err;
  const int items = routed ? a.pairs : (a.tokens + a.cols - 1) / a.cols;
  const int slots = device_sm_count() * (lay.total <= kTwoCtaSmem ? 2 : 1);
  auto units = [&](int k_warps) {
    const int rows = (kGateUp ? 8 : 16) * (kWarps / k_warps);
    return static_cast<long long>(items) * ((a.rows + rows - 1) / rows);
  };
  // All warps to a tile, unless that leaves a warp fewer than 4 steps a tile and there are tiles
  // enough: the barrier and the additions at a tile's end then cost as much as its products.
  a.k_warps = kWarps;
  while (a.k_warps > 2 && steps < 4 * a.k_warps && units(a.k_warps / 2) >= 2 * slots) a.k_warps /= 2;
  const long long most = units(a.k_warps);
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

int skinny_columns(int want, int k, int group, int pairs, int experts) {
  const int step = group == 0 ? Format<0>::kStep : Format<32>::kStep;
  const int padded = (k + step - 1) / step * step;
  int cols = want < kSkinnyMaxColumns ? want : kSkinnyMaxColumns;
  while (cols > 0 && carve_smem(cols, padded, group == 0 ? 0 : padded / group, pairs, experts).total > kMaxSmem) --cols;
  return cols;
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
