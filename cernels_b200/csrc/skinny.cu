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
// weights of the next kDepth steps on their way into a ring of its own (cp.async, across tile borders): up to
// 96 KB of weights in flight per SM. bf16 weights reach 5.3 of the measured 6.5 TB/s (one row of x, 201 MB in
// 37.7 us). The same ring in registers gave 2.7 TB/s, and a third as much with 4-bit weights: a warp has too
// few load counters to wait for one step and not for those behind it.
//
// mma.sync does the products: rows of W are the A operand, x columns the B operand. The order of k
// within the reduction is free as long as A and B agree, so W is used as it lies in memory and x is
// stored in shared memory to match. tcgen05 would need W in shared memory in its tile layout, a trip
// that 4-bit weights would make unpacked; the tensor pipe is a small part of the time either way.
//
// 4 bits: a byte holds two codes, and (byte & 0xf0) ^ 0x80 is 16 (q - 8) as a signed byte: the A operand
// of the 8-bit mma (m16n8k32), in 3 instructions for 8 codes. (Making bf16 pairs of them took 7 and twice the
// mma's; that version was bound by instructions at 2.3 TB/s.) So x becomes integers too: in each block of
// 128, x = 2^e v with |v| < 2^14, e from the block's largest |x|, as v = 256 hi + lo in two signed bytes and
// two mma's (up to 4 columns: two columns of one mma). This keeps 14 bits below the block's largest value, where
// bf16 x holds 8 bits of each value: every x within 2^-6 of the largest is exact, the others are rounded by at
// most 2^-14 of it. That is far below the rounding of an output that the larger values enter, but the values between
// a few large ones would be lost to an output whose weights are 0 where those stand. So a block of x in which more than half of
// the nonzero values are under 128 units (2^-7 to 2^-6 of the largest) is mixed: it is not taken as integers but
// multiplied in bf16, exactly, as are blocks with an infinity or a NaN (add_mixed: codes from L2 once more; where all
// blocks are mixed a call takes 2 to 3 times as long, 18 -> 44 us for 16384 x 8192 at one row). In the
// other blocks no x is off by more than 2^-8 of the median. Normal x has no mixed block, the halved products of normal
// gates and ups one in a thousand.
//
// The sums of 16 (q - 8) hi and 16 (q - 8) lo over a
// group are exact integers of at most 128 * 128 * 128 < 2^22, and they start at the integer whose bits are the
// float 1.5 * 2^23, so that their own bits are that float plus the sum. From there on it is 32-bit floating
// arithmetic: scales are never rounded and multiply each group's sum. What bounds it now
// is instructions, 180 for 16 x 128 weights in groups of 32: experts at 8 tokens take 86 us against 45 for their bytes (an
// earlier state, at 87, took 80 without the copies and 68 without the products).
#include "ffn_internal.h"

#include <cmath>
#include <cstring>
#include <type_traits>

namespace cernels {
namespace {

constexpr int kMaxSmem = 232448;        // per CTA
constexpr int kSmemPerSm = 228 * 1024;  // 1 KB of it is taken per CTA
constexpr int kDepth = 3;  // steps in flight per warp; 4 measured the same where as many CTAs fit
constexpr int kParts = 2;  // 64-byte parts of a row in a step: whole lines (4, at depth 2, measured the same)
constexpr int kCtas = 2;   // per SM; fewer where x rows need the shared memory

__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// d = c + 16 (q - 8) (rows of W) times bytes of x. c is an operand of its own: the constant start of every
// group's sums then stays in its registers.
__device__ __forceinline__ void mma_bytes(int4& d, const int4& c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d.x), "=r"(d.y), "=r"(d.z), "=r"(d.w)
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c.x), "r"(c.y), "r"(c.z), "r"(c.w));
}

constexpr int kFloatBias = 0x4b400000;       // the bits of 1.5 * 2^23: adding n < 2^22 to them adds n to the float
constexpr float kFloatBiasValue = 12582912.0f;

// Codes 2 i and 2 i + 1 of a word of eight as bf16 values q - 8: 0x4300 | q is 128 + q.
__device__ __forceinline__ uint32_t bf16_codes(uint32_t word, int i) {
  const uint32_t t = word >> 8 * i, biased = (t & 0xfu) | (t << 12 & 0xf0000u) | 0x43004300u;
  const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&biased), __float2bfloat162_rn(136.0f));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Bytes of a word that are not zero, as their top bits.
__device__ __forceinline__ uint32_t nonzero_bytes(uint32_t w) {
  return (((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w) & 0x80808080u;
}

// Two 32-bit values at once (FFMA2 and the like: half the instructions of the scalar forms).
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ Two two(int lo, int hi) { return two(__int_as_float(lo), __int_as_float(hi)); }
__device__ __forceinline__ float2 split(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two add(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two mul(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Copies `bytes` (4, 8 or 16) to shared memory without a register; reads only the first `valid` of
// them (0: none) and fills the rest with zeros.
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(kBytes) : "memory");
}
template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, int valid) {
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(kBytes), "r"(valid)
                 : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void wait_copies() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// kFmt 0: bf16 weights; 32, 64, 128: 4-bit weights with that group size. A K step is kParts parts of 64 bytes
// of a row, of which a quad of lanes reads 16 bytes each.
template <int kFmt>
struct Format {
  static constexpr int kPart = kFmt == 0 ? 32 : 128;  // values
  static constexpr int kStep = kParts * kPart;
  static constexpr int kGroups = kFmt == 0 ? 1 : 128 / kFmt;  // per part
  static constexpr int kWords = kFmt == 0 ? 1 : kFmt / 32;    // 8-code words per lane and group
  // A warp's ring slot: a step's 16 rows, [part][row][64 bytes], and the words that hold the rows' scales, [word][row];
  // rows may start in the middle of a word. Where an mma takes the same group from all lanes (4 kWords bytes
  // each), a row's 16-byte pieces are exchanged so that those reads meet no bank twice: piece ^ swizzle(row).
  static constexpr int kPartBytes = 16 * 64;
  static constexpr int kScaleWords = kFmt == 0 ? 0 : kParts * kGroups / 2 + 1;
  static constexpr int kScaleAt = kParts * kPartBytes;
  __device__ static int swizzle(int row) { return kFmt == 32 ? row >> 1 & 3 : kFmt == 64 ? row & 2 : 0; }
  static constexpr int kSlot = kScaleAt + kScaleWords * 64;
};

// Bytes in a shared-memory row of x: an odd multiple of 64, so that the 8 lanes of a 16-byte
// access phase (two rows, four pieces each) fall into different banks.
__host__ __device__ constexpr int x_row_bytes(int padded_k) {
  return padded_k * 2 % 128 == 0 ? padded_k * 2 + 64 : padded_k * 2;
}

struct Item {
  int expert, first, count;  // columns: order[first .. first + count)
};

// Buffers of the warps' sums: with two, a tile's additions overlap the next tile's products.
__host__ __device__ constexpr int part_buffers(int warps) { return warps == 8 ? 2 : 1; }

// Columns of the tile that `cols` columns are computed with.
__host__ __device__ constexpr int tile_columns(bool bf16, int cols) {
  return cols > 8 ? 16 : cols > 4 || bf16 ? 8 : 4;
}

struct SkinnySmem {
  size_t ring, part, units, x, items, ids, lead, count, first, sums, rank, list, order, total;
};

// tile_cols: columns of the kernel's tile (its template argument), cols of them in use; blocks: of 128 values in
// padded_k (0 for bf16); pairs and experts: 0 without routing
__host__ __device__ inline SkinnySmem carve_smem(int warps, int slot, int tile_cols, int cols, int padded_k,
                                                int blocks, int pairs, int experts) {
  SkinnySmem s;
  size_t off = 0;
  s.ring = off;
  off += static_cast<size_t>(warps) * kDepth * slot;
  s.part = off;
  off += static_cast<size_t>(part_buffers(warps)) * warps * tile_cols * 16 * 4;
  s.units = off;  // per column and block: 2^e / 16, or 0 for a mixed block
  off += (static_cast<size_t>(blocks) * cols * 4 + 15) / 16 * 16;
  s.x = off;
  off += static_cast<size_t>(cols) * x_row_bytes(padded_k);
  const size_t n = (static_cast<size_t>(pairs) + 3) / 4 * 4;
  s.ids = off;
  off += n * 4;
  s.items = off;
  off += n * sizeof(Item);
  s.lead = off;
  off += static_cast<size_t>(experts) * 4;
  s.count = off;
  off += static_cast<size_t>(experts) * 4;
  s.first = off;
  off += static_cast<size_t>(experts) * 4;
  s.sums = off;
  off += (n + 31) / 32 * 4;
  s.rank = off;
  off += n * 2;
  s.list = off;
  off += n * 2;
  s.order = off;
  off += n * 2;
  s.total = off + 16;  // number of items, mark of the last item with a mixed block
  return s;
}

// Groups the (token, slot) pairs by expert, experts in order of first use and pairs in their own order, into
// items of at most `cols` columns. Every CTA does this for itself, and all come to the same lists: what
// the counters' atomics leave open is put in order again by each pair looking through its expert's. (One
// warp walking through all pairs took 4 us for 232 of them.) Returns the number of items.
__device__ int build_items(const SkinnyArgs& a, uint8_t* smem, const SkinnySmem& lay) {
  int* ids = reinterpret_cast<int*>(smem + lay.ids);
  Item* items = reinterpret_cast<Item*>(smem + lay.items);
  int* count = reinterpret_cast<int*>(smem + lay.count);
  int* first = reinterpret_cast<int*>(smem + lay.first);  // an expert's first pair
  int* lead = reinterpret_cast<int*>(smem + lay.lead);    // and its first place in `order`
  uint16_t* rank = reinterpret_cast<uint16_t*>(smem + lay.rank);
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + lay.list);  // places as the atomics gave them out
  uint16_t* order = reinterpret_cast<uint16_t*>(smem + lay.order);
  int* n_items = reinterpret_cast<int*>(smem + lay.total - 16);
  for (int p = threadIdx.x; p < a.pairs; p += blockDim.x) {
    const int e = a.indices[p];
    ids[p] = e >= 0 && e < a.experts ? e : -1;
  }
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) {
    count[e] = 0;
    first[e] = a.pairs;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += blockDim.x)
    if (ids[p] >= 0) {
      rank[p] = static_cast<uint16_t>(atomicAdd(&count[ids[p]], 1));
      atomicMin(&first[ids[p]], p);
    }
  __syncthreads();
  // places and items before each expert: within 32 pairs, then over all of them
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  uint32_t* sums = reinterpret_cast<uint32_t*>(smem + lay.sums);  // items << 16 | places, of 32 pairs each
  for (int chunk = threadIdx.x >> 5; chunk * 32 < a.pairs; chunk += warps) {
    const int p = chunk * 32 + lane;
    const int e = p < a.pairs ? ids[p] : -1;
    const int n = e >= 0 && first[e] == p ? count[e] : 0;
    const uint32_t mine = static_cast<uint32_t>((n + a.cols - 1) / a.cols) << 16 | static_cast<uint32_t>(n);
    uint32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    if (n != 0) lead[e] = static_cast<int>(sum - mine);
    if (lane == 31) sums[chunk] = sum;
  }
  __syncthreads();
  for (int chunk = threadIdx.x >> 5; chunk * 32 < a.pairs; chunk += warps) {
    const int p = chunk * 32 + lane;
    const uint32_t before = __reduce_add_sync(0xffffffffu, lane < chunk ? sums[lane] : 0);
    const int e = p < a.pairs ? ids[p] : -1;
    const int n = e >= 0 && first[e] == p ? count[e] : 0;
    if (n != 0) {
      const uint32_t start = before + static_cast<uint32_t>(lead[e]);
      const int from = start & 0xffff;
      lead[e] = from;
      Item* to = items + (start >> 16);
      for (int i = 0; i * a.cols < n; ++i) to[i] = Item{e, from + i * a.cols, min(a.cols, n - i * a.cols)};
    }
    if ((chunk + 1) * 32 >= a.pairs && lane == 0) *n_items = before + sums[chunk] >> 16;
  }
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += blockDim.x)
    if (ids[p] >= 0) list[lead[ids[p]] + rank[p]] = static_cast<uint16_t>(p);
  __syncthreads();
  for (int p = threadIdx.x; p < a.pairs; p += blockDim.x) {
    const int e = ids[p];
    if (e < 0) continue;
    const int from = lead[e], n = count[e];
    int before = 0;
    for (int i = 0; i < n; ++i) before += list[from + i] < p;
    order[from + before] = static_cast<uint16_t>(p);
  }
  __syncthreads();
  return *n_items;
}

template <int kFmt, bool kGateUp, int kCols, int kWarps>
__global__ void __launch_bounds__(32 * kWarps, kWarps == 8 ? kCtas : 1) skinny_kernel(const SkinnyArgs a) {
  using F = Format<kFmt>;
  constexpr int kThreads = 32 * kWarps;
  // Up to 4 columns of 4-bit products fit one mma: its columns are hi and lo of each.
  constexpr bool kPacked = kCols == 4;
  constexpr int NT = kPacked ? 1 : kCols / 8;
  static_assert(!kPacked || kFmt != 0, "bf16 x has no halves");
  constexpr int kOut = kGateUp ? 8 : 16;  // outputs per tile and column
  extern __shared__ __align__(16) uint8_t smem[];
  if (!a.x_from_previous) wait_for_previous_kernel();  // it may have written anything read here
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;  // mma row (and x column) of this lane, its quarter of a half step
  const int kw = warp % a.k_warps, rt = warp / a.k_warps;
  const int tiles_at_once = kWarps / a.k_warps;
  const int steps = (a.k + F::kStep - 1) / F::kStep;
  const int per_warp = (steps + a.k_warps - 1) / a.k_warps;
  const int padded_k = steps * F::kStep;
  const int x_bytes = x_row_bytes(padded_k);
  const bool routed = a.indices != nullptr;
  const SkinnySmem lay = carve_smem(kWarps, F::kSlot, kCols, a.cols, padded_k, kFmt == 0 ? 0 : padded_k / 128,
                                    routed ? a.pairs : 0, routed ? a.experts : 0);
  float* part = reinterpret_cast<float*>(smem + lay.part);
  const int blocks = padded_k / 128;
  float* units_of_x = reinterpret_cast<float*>(smem + lay.units);  // [column][block]
  int* mixed_mark = reinterpret_cast<int*>(smem + lay.total - 12);
  uint8_t* xs = smem + lay.x;
  const Item* items = reinterpret_cast<const Item*>(smem + lay.items);
  const uint16_t* order = reinterpret_cast<const uint16_t*>(smem + lay.order);

  const int n_items = routed ? build_items(a, smem, lay) : (a.tokens + a.cols - 1) / a.cols;
  const int per_item = (a.rows + kOut * tiles_at_once - 1) / (kOut * tiles_at_once);  // units of an item
  const long long units = static_cast<long long>(n_items) * per_item;
  const int begin = static_cast<int>(units * blockIdx.x / gridDim.x);
  const int end = static_cast<int>(units * (blockIdx.x + 1) / gridDim.x);
  if (begin >= end) {
    if (a.x_from_previous) wait_for_previous_kernel();
    return;
  }

  auto item_of = [&](int i) {
    return routed ? items[i] : Item{0, i * a.cols, min(a.cols, a.tokens - i * a.cols)};
  };

  // ---- weights: this lane's two rows of a unit, and the stream of steps through them
  const size_t row_bytes = kFmt == 0 ? static_cast<size_t>(a.k) * 2 : static_cast<size_t>(a.k) / 2;
  const int row_groups = kFmt == 0 ? 0 : a.k / (kFmt == 0 ? 1 : kFmt);
  constexpr int kPerStep = kFmt == 0 ? F::kStep : kParts * F::kGroups;  // values (bf16) or groups
  int load_item = begin / per_item, load_unit = begin - load_item * per_item;  // position of the stream
  int load_left = (end - begin) * per_warp, load_step = kw;
  // Eight lanes copy a row's 128 bytes of a step, four rows at once: whole lines, half the tag lookups of the
  // lanes' own rows and quarters. Scales: lane (g, q) copies word q of rows g and g + 8.
  const uint8_t *w_first = nullptr, *w_second = nullptr;  // rows lane / 8 of the tile's halves
  int w_next_first = 0, w_next_second = 0;                // distance to rows lane / 8 + 4
  const uint16_t *s_first = nullptr, *s_second = nullptr;  // scales of rows g, g + 8, from a word's start
  int odd_first = 0, odd_second = 0;                       // they start at the word's second half
  uint32_t odd_a = 0, odd_b = 0;  // the same, of the unit being consumed
  const int piece = lane & 7;     // 16 bytes of the 128: part piece / 4, lane of the quad piece % 4
  auto point = [&] {
    const int e = routed ? items[load_item].expert : 0;
    const int base = (load_unit * tiles_at_once + rt) * kOut;
    const int second = kGateUp ? 0 : 8;
    auto row_of = [&](int r) { return static_cast<size_t>(min(base + r, a.rows - 1)); };
    const int r = lane >> 3;
    const uint8_t* from = a.w0 + static_cast<size_t>(e) * a.w_expert + kw * (kParts * 64) + piece * 16;
    const uint8_t* up = (kGateUp ? a.w1 : a.w0) + static_cast<size_t>(e) * a.w_expert + kw * (kParts * 64) + piece * 16;
    w_first = from + row_of(r) * row_bytes;
    w_second = up + row_of(r + second) * row_bytes;
    w_next_first = static_cast<int>((row_of(r + 4) - row_of(r)) * row_bytes);
    w_next_second = static_cast<int>((row_of(r + second + 4) - row_of(r + second)) * row_bytes);
    if constexpr (kFmt != 0) {
      auto scales = [&](const uint16_t* s, size_t row, int& odd) {
        s += static_cast<size_t>(e) * a.s_expert + row * row_groups + kw * kPerStep;
        odd = static_cast<int>(reinterpret_cast<uintptr_t>(s) >> 1 & 1);
        return s - odd + 2 * q;  // this lane's first word
      };
      s_first = scales(a.s0, row_of(g), odd_first);
      s_second = scales(kGateUp ? a.s1 : a.s0, row_of(g + second), odd_second);
    }
  };
  uint8_t* ring = smem + lay.ring + static_cast<size_t>(warp) * kDepth * F::kSlot;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  uint32_t load_at = ring_at;  // slot that the next step goes to
  // rows r and r + 8 share a swizzle, rows r and r + 4 (r < 4) do not
  auto piece_at = [&](int row) { return (piece >> 2) * F::kPartBytes + row * 64 + ((piece & 3) ^ F::swizzle(row)) * 16; };
  const uint32_t lane_at = piece_at(lane >> 3), next_at = piece_at((lane >> 3) + 4);
  const uint32_t scale_at = F::kScaleAt + g * 4 + q * 64;
  const int step_bytes = a.k_warps * (kParts * 64), step_scales = a.k_warps * kPerStep;
  // A row's words of scales beyond the first four (lane q has word q), and its last one, which counts only
  // where the row starts in the middle of the first.
  auto copy_step = [&](auto whole, int left) {
#pragma unroll
    for (int c = 0; c < kParts / 2; ++c) {
      // first value (bf16) or group of this lane's 16 bytes
      const int first = kFmt == 0 ? c * 64 + piece * 8 : (2 * c + (piece >> 2)) * F::kGroups + (piece & 3) * F::kGroups / 4;
      auto row = [&](uint32_t to, const uint8_t* from) {
        to += load_at + 2 * c * F::kPartBytes;
        if constexpr (whole.value)
          copy_async<16>(to, from + c * 128);
        else
          copy_async<16>(to, from + c * 128, first < left ? 16 : 0);
      };
      row(lane_at, w_first);
      row(next_at, w_first + w_next_first);
      row(lane_at + 8 * 64, w_second);
      row(next_at + 8 * 64, w_second + w_next_second);
    }
    if constexpr (kFmt != 0) {
      auto scales = [&](uint32_t to, const uint16_t* from, int odd) {
        const int need = left > 0 ? min(left, kPerStep) + odd : 0;  // from the word's start on
#pragma unroll
        for (int i = 0; i < (F::kScaleWords + 3) / 4; ++i) {
          const int word = 4 * i + q;
          if (word < F::kScaleWords && (word < F::kScaleWords - 1 || odd)) {
            if constexpr (whole.value)
              copy_async<4>(load_at + scale_at + to + i * 256, from + 8 * i);
            else
              copy_async<4>(load_at + scale_at + to + i * 256, from + 8 * i, max(0, min(4, 2 * (need - 2 * word))));
          }
        }
      };
      scales(0, s_first, odd_first);
      scales(32, s_second, odd_second);
    }
  };
  auto issue = [&] {
    if (load_left != 0) {
      const int left = (kFmt == 0 ? a.k : row_groups) - load_step * kPerStep;
      if (left > kPerStep)  // more of the row follows: nothing to cut off, not even half of the last word
        copy_step(std::true_type{}, left);
      else
        copy_step(std::false_type{}, left);
      w_first += step_bytes;
      w_second += step_bytes;
      if constexpr (kFmt != 0) {
        s_first += step_scales;
        s_second += step_scales;
      }
      load_at += F::kSlot;
      if (load_at == ring_at + kDepth * F::kSlot) load_at = ring_at;
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
    }
    commit_copies();
  };
  // ---- x rows of an item, 8 values (a piece) at a time, in the order in which the weights lie
  // 4 bits: a warp takes a row's 256 values at once (a chunk), kBatch chunks on their way together.
  constexpr int kBatch = 8;
  const int row_chunks = padded_k / 256;
  const unsigned inverse_chunks = (1u << 20) / (row_chunks ? row_chunks : 1) + 1;  // chunk / row_chunks, exact for up to 16 * 128
  auto load_piece = [&](const Item& it, unsigned chunk) {
    const int c = static_cast<int>(chunk * inverse_chunks >> 20);
    const int k = (static_cast<int>(chunk) - c * row_chunks) * 256 + lane * 8;
    int row = it.first + c;
    if (routed) {
      row = order[row];
      if (!a.x_by_pair) row /= a.topk;
    }
    return k < a.k ? *reinterpret_cast<const uint4*>(a.x + static_cast<size_t>(row) * a.x_stride + k) : make_uint4(0, 0, 0, 0);
  };
  auto fetch_x = [&](const Item& it, int first_chunk, uint4 (&v)[kBatch]) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const unsigned chunk = first_chunk + b * kWarps;
      v[b] = make_uint4(0, 0, 0, 0);
      if (static_cast<int>(chunk) < it.count * row_chunks) v[b] = load_piece(it, chunk);
    }
  };
  // Gives the mixed blocks of a batch the unit 0, and the item its mark.
  auto mark_mixed = [&](const Item& it, int mark, int first_chunk) {
#pragma unroll 1
    for (int chunk = first_chunk; chunk < min(first_chunk + kBatch * kWarps, it.count * row_chunks); chunk += kWarps) {
      const uint4 v = load_piece(it, chunk);
      const uint32_t words[4] = {v.x, v.y, v.z, v.w};
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) top = max(top, max(words[j] << 16 & 0x7fff0000u, words[j] & 0x7fff0000u));
#pragma unroll
      for (unsigned d = 8; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
      const int least = max(static_cast<int>(top >> 23) - 13, 5) + 7;  // exponent of 128 units
      int votes = 0;  // of the nonzero values: +1 small, -1 large
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t size = j & 1 ? words[j >> 1] & 0x7fff0000u : words[j >> 1] << 16 & 0x7fff0000u;
        votes += size == 0 ? 0 : static_cast<int>(size >> 23) < least ? 1 : -1;
      }
#pragma unroll
      for (unsigned d = 8; d > 0; d /= 2) votes += __shfl_xor_sync(0xffffffffu, votes, d);
      if ((votes > 0 || top >= 0x7f800000u) && lane % 16 == 0) {
        const int c = chunk / row_chunks;
        units_of_x[c * blocks + (chunk - c * row_chunks) * 2 + lane / 16] = 0.f;
        *mixed_mark = mark;
      }
    }
  };
  auto store_x = [&](const Item& it, int mark, int first_chunk, const uint4 (&v)[kBatch]) {
    if constexpr (kFmt != 0) {
      // counts of large values, a byte for each block of two chunks, less the 64 that stand for a chunk which is not there
      uint32_t large[kBatch / 2] = {};
      uint32_t special = 0;
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const unsigned chunk = first_chunk + b * kWarps;
        if (static_cast<int>(chunk) >= it.count * row_chunks) break;
        const int c = static_cast<int>(chunk * inverse_chunks >> 20);
        const unsigned k8 = (chunk - c * row_chunks) * 32 + lane;
        const uint32_t words[4] = {v[b].x, v[b].y, v[b].z, v[b].w};
        uint32_t top = 0;  // the block's largest magnitude, as bits
#pragma unroll
        for (int j = 0; j < 4; ++j) top = max(top, max(words[j] << 16 & 0x7fff0000u, words[j] & 0x7fff0000u));
#pragma unroll
        for (unsigned d = 8; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
        // 2^13 <= largest / 2^e < 2^14 (less for values whose unit, or its 16th, would be subnormal)
        const int unit_exp = max(static_cast<int>(top >> 23) - 13, 5);
        const float inverse = __uint_as_float(static_cast<uint32_t>(254 - unit_exp) << 23);
        uint32_t n[8];  // the nearest integer, in the low half of the float's bits
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t bits = j & 1 ? words[j >> 1] & 0xffff0000u : words[j >> 1] << 16;
          n[j] = __float_as_uint(fmaf(__uint_as_float(bits), inverse, kFloatBiasValue));
        }
        auto bytes = [&](uint32_t selector, int odd, uint32_t add) {  // one byte of n[odd], n[odd + 2], ..
          return __byte_perm(__byte_perm(n[odd] + add, n[odd + 2] + add, selector),
                             __byte_perm(n[odd + 4] + add, n[odd + 6] + add, selector), 0x5410);
        };
        const uint4 split_x = make_uint4(bytes(0x51, 0, 128), bytes(0x51, 1, 128), bytes(0x40, 0, 0), bytes(0x40, 1, 0));
        // values of 128 units or more, by their high byte; past the row's end half of the places count
        const uint32_t found = static_cast<int>(k8) * 8 < a.k ? __popc(nonzero_bytes(split_x.x) | nonzero_bytes(split_x.y) >> 1) : 4;
        large[b / 2] += (found - 4) << (lane / 16 * 8 + b % 2 * 16);
        special = max(special, top);
        if (k8 % 16 == 0) units_of_x[c * blocks + k8 / 16] = __uint_as_float(static_cast<uint32_t>(unit_exp - 4) << 23);
        constexpr unsigned kPer = kFmt / 8;  // pieces per group
        const unsigned in = k8 % kPer;
        // group | lane of the quad | word  ->  group | word | lane
        const unsigned at = k8 - in + (in % F::kWords) * 4 + in / F::kWords;
        *reinterpret_cast<uint4*>(xs + static_cast<size_t>(c) * x_bytes + at * 16) = split_x;
      }
      // a count under 64 in any block: bits 6 and 7 of its byte are clear
      uint32_t enough = 0x40404040u;
#pragma unroll
      for (int j = 0; j < kBatch / 2; ++j) {
        const uint32_t counts = __reduce_add_sync(0xffffffffu, large[j]) + 0x40404040u;
        enough &= counts | counts >> 1;
      }
      if (__any_sync(0xffffffffu, enough != 0x40404040u || special >= 0x7f800000u)) mark_mixed(it, mark, first_chunk);
    }
  };
  auto copy_x = [&](const Item& it) {  // bf16
    const unsigned pieces = static_cast<unsigned>(padded_k) / 8;
    const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(xs));
    for (unsigned i = threadIdx.x; i < it.count * pieces; i += kThreads) {
      const unsigned c = i / pieces, k8 = i - c * pieces;
      const size_t row = it.first + c;
      copy_async<16>(to + c * x_bytes + k8 * 16, a.x + row * a.x_stride + k8 * 8, static_cast<int>(k8) * 8 < a.k ? 16 : 0);
    }
    commit_copies();
  };
  auto load_x = [&](const Item& it, int mark, int first_chunk) {
    if constexpr (kFmt == 0) {
      copy_x(it);
      wait_copies<0>();
    } else {
      for (int chunk = first_chunk; chunk < it.count * row_chunks; chunk += kWarps * kBatch) {
        uint4 v[kBatch];
        fetch_x(it, chunk, v);
        store_x(it, mark, chunk, v);
      }
    }
  };

  // x before the weights where it is there already: its first loads then do not queue behind them
  int item_index = begin / per_item, unit = begin - item_index * per_item;
  Item item = item_of(item_index);
  uint4 first_x[kBatch];
  if (!a.x_from_previous) {
    if constexpr (kFmt == 0)
      copy_x(item);
    else
      fetch_x(item, warp, first_x);
  }
  point();
#pragma unroll
  for (int d = 0; d < kDepth; ++d) issue();
  if (a.x_from_previous) {
    wait_for_previous_kernel();
    if constexpr (kFmt != 0)
      fetch_x(item, warp, first_x);
    else
      load_x(item, 0, 0);
  } else if constexpr (kFmt == 0) {
    wait_copies<kDepth>();
  }
  if constexpr (kFmt != 0) {
    store_x(item, item_index + 1, warp, first_x);
    load_x(item, item_index + 1, warp + kWarps * kBatch);
  }
  __syncthreads();
  // Columns past the item's last read its last one again: their sums are never used.
  const uint8_t* xcol[NT];
  const float* units_at[NT][2];  // of the columns whose sums this lane gets (packed: one)
  auto point_x = [&] {
    const int last = item.count - 1;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int c = kPacked ? g >> 1 : n * 8 + g;
      xcol[n] = xs + static_cast<size_t>(min(c, last)) * x_bytes + q * 16 + (kPacked ? (g & 1) * 8 : 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) units_at[n][j] = units_of_x + min(kPacked ? q : n * 8 + 2 * q + j, last) * blocks;
    }
  };
  point_x();
  // What the word holds before the first mark may look like one: then no block's unit is 0 all the same.
  bool any_mixed = kFmt != 0 && *mixed_mark == item_index + 1;
  // start of every group's sums; opaque, so that it stays in registers
  int4 start;
  asm volatile("mov.b32 %0, %4;\n\tmov.b32 %1, %4;\n\tmov.b32 %2, %4;\n\tmov.b32 %3, %4;"
               : "=r"(start.x), "=r"(start.y), "=r"(start.z), "=r"(start.w)
               : "n"(kFloatBias));

  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;

  const int swizzle = F::swizzle(g);  // of rows g and g + 8
  int units_left = end - begin, i = 0, buffer = 0;
  const uint8_t* at = ring;  // slot of the step being consumed
  auto point_scales = [&] {
    if constexpr (kFmt != 0) {
      const int base = (unit * tiles_at_once + rt) * kOut;
      const int ra = min(base + g, a.rows - 1);
      const int rb = kGateUp ? ra : min(base + g + 8, a.rows - 1);
      const size_t from = static_cast<size_t>(routed ? item.expert : 0) * a.s_expert;
      const uint16_t* second = kGateUp ? a.s1 : a.s0;
      odd_a = reinterpret_cast<uintptr_t>(a.s0 + from + static_cast<size_t>(ra) * row_groups) >> 1 & 1;
      odd_b = reinterpret_cast<uintptr_t>(second + from + static_cast<size_t>(rb) * row_groups) >> 1 & 1;
    }
  };
  point_scales();
  // Adds the products of the unit's mixed blocks in this warp's steps to its sums `to` (in shared memory: registers for it
  // would cost the loop of ordinary x), with codes, scales and x from global memory (L2 has them). The sums of integers
  // left these blocks' columns out: their units are 0.
  auto add_mixed = [&](float* to) {
    if constexpr (kFmt != 0) {
      const int base = (unit * tiles_at_once + rt) * kOut;
      const size_t e = routed ? item.expert : 0;
      const size_t ra = min(base + g, a.rows - 1), rb = kGateUp ? ra : min(base + g + 8, a.rows - 1);
      const uint8_t* wa = a.w0 + e * a.w_expert + ra * row_bytes;
      const uint8_t* wb = (kGateUp ? a.w1 : a.w0) + e * a.w_expert + rb * row_bytes;
      const uint16_t* fa = a.s0 + e * a.s_expert + ra * row_groups;
      const uint16_t* fb = (kGateUp ? a.s1 : a.s0) + e * a.s_expert + rb * row_groups;
      const __nv_bfloat16* x_row[NT];  // of the column whose values this lane gives the mma (packed: its even columns)
      unsigned column[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        column[n] = kPacked ? (g & 1 ? 31 : g >> 1) : n * 8 + g;
        size_t row = item.first + min(static_cast<int>(column[n]), item.count - 1);
        if (routed) {
          row = order[row];
          if (!a.x_by_pair) row /= a.topk;
        }
        x_row[n] = a.x + row * a.x_stride;
      }
#pragma unroll 1
      for (int block = kw * kParts; block < steps * kParts; block += block % kParts == kParts - 1 ? (a.k_warps - 1) * kParts + 1 : 1) {
        const unsigned mixed = __ballot_sync(0xffffffffu, lane < item.count && units_of_x[min(lane, item.count - 1) * blocks + block] == 0.f);
        if (mixed == 0) continue;
        // lane q's words of a group: kWords in a row; groups past the row's end are empty
        uint32_t ca[F::kGroups * F::kWords], cb[F::kGroups * F::kWords];
        float scale_a[F::kGroups], scale_b[F::kGroups];
        const int group = block * F::kGroups, left = row_groups - group;
#pragma unroll
        for (int s = 0; s < F::kGroups; ++s) {
          using Words = std::conditional_t<F::kWords == 4, uint4, std::conditional_t<F::kWords == 2, uint2, uint32_t>>;
          Words u{}, v{};
          scale_a[s] = scale_b[s] = 0.f;
          if (s < left) {
            u = reinterpret_cast<const Words*>(wa + (group + s) * (kFmt / 2))[q];
            v = reinterpret_cast<const Words*>(wb + (group + s) * (kFmt / 2))[q];
            scale_a[s] = __uint_as_float(static_cast<uint32_t>(fa[group + s]) << 16);
            scale_b[s] = __uint_as_float(static_cast<uint32_t>(fb[group + s]) << 16);
          }
          memcpy(ca + s * F::kWords, &u, sizeof(u));
          memcpy(cb + s * F::kWords, &v, sizeof(v));
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const bool mine = mixed >> column[n] & 1;
          uint4 x8[F::kGroups * F::kWords];
#pragma unroll
          for (int j = 0; j < F::kGroups * F::kWords; ++j) {
            const int s = j / F::kWords, piece = (group + s) * (kFmt / 8) + q * F::kWords + j % F::kWords;  // of eight values
            x8[j] = make_uint4(0, 0, 0, 0);
            if (mine && s < left) x8[j] = *reinterpret_cast<const uint4*>(x_row[n] + piece * 8);
          }
#pragma unroll
          for (int s = 0; s < F::kGroups; ++s) {
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < F::kWords; ++w) {
              const int j = s * F::kWords + w;
              mma_bf16(sum, bf16_codes(ca[j], 0), bf16_codes(cb[j], 0), bf16_codes(ca[j], 1), bf16_codes(cb[j], 1), x8[j].x, x8[j].y);
              mma_bf16(sum, bf16_codes(ca[j], 2), bf16_codes(cb[j], 2), bf16_codes(ca[j], 3), bf16_codes(cb[j], 3), x8[j].z, x8[j].w);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if (kPacked ? j == 0 && mixed >> q & 1 : mixed >> (n * 8 + 2 * q + j) & 1) {
                to[n * 128 + j * 16] = fmaf(scale_a[s], sum[j], to[n * 128 + j * 16]);
                to[n * 128 + j * 16 + 8] = fmaf(scale_b[s], sum[j + 2], to[n * 128 + j * 16 + 8]);
              }
            }
          }
        }
      }
    }
  };
  while (true) {
    const int step = i * a.k_warps + kw;
    wait_copies<kDepth - 1>();
    __syncwarp();  // the scales were fetched by other lanes
    if (step < steps) {
      const uint8_t* x_at[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) x_at[n] = xcol[n] + step * (F::kStep * 2);
      uint32_t sa[F::kScaleWords + 1], sb[F::kScaleWords + 1];
#pragma unroll
      for (int j = 0; j < F::kScaleWords; ++j) {
        sa[j] = *reinterpret_cast<const uint32_t*>(at + F::kScaleAt + j * 64 + g * 4);
        sb[j] = *reinterpret_cast<const uint32_t*>(at + F::kScaleAt + j * 64 + 32 + g * 4);
      }
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const uint8_t* ra = at + h * F::kPartBytes + g * 64;
        const uint8_t* rb = ra + 8 * 64;
        if constexpr (kFmt == 0) {
          const uint4 u = *reinterpret_cast<const uint4*>(ra + q * 16), v = *reinterpret_cast<const uint4*>(rb + q * 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const uint4 x4 = *reinterpret_cast<const uint4*>(x_at[n] + h * (F::kPart * 2));
            mma_bf16(acc[n], u.x, v.x, u.y, v.y, x4.x, x4.y);
            mma_bf16(acc[n], u.z, v.z, u.w, v.w, x4.z, x4.w);
          }
        } else {
          uint32_t aw[4], bw[4];  // words of group 0, then of group 1, ..
          if constexpr (kFmt == 128) {
            const uint4 u = *reinterpret_cast<const uint4*>(ra + q * 16), v = *reinterpret_cast<const uint4*>(rb + q * 16);
            aw[0] = u.x, aw[1] = u.y, aw[2] = u.z, aw[3] = u.w;
            bw[0] = v.x, bw[1] = v.y, bw[2] = v.z, bw[3] = v.w;
          } else if constexpr (kFmt == 64) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              const uint2 u = *reinterpret_cast<const uint2*>(ra + ((2 * s + (q >> 1)) ^ swizzle) * 16 + (q & 1) * 8);
              const uint2 v = *reinterpret_cast<const uint2*>(rb + ((2 * s + (q >> 1)) ^ swizzle) * 16 + (q & 1) * 8);
              aw[2 * s] = u.x, aw[2 * s + 1] = u.y;
              bw[2 * s] = v.x, bw[2 * s + 1] = v.y;
            }
          } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
              aw[s] = *reinterpret_cast<const uint32_t*>(ra + (s ^ swizzle) * 16 + q * 4);
              bw[s] = *reinterpret_cast<const uint32_t*>(rb + (s ^ swizzle) * 16 + q * 4);
            }
          }
          // scale of group s of this part, of a row whose first is the low or (odd) the high half of word 0
          auto scale_of = [&](const uint32_t* words, uint32_t odd, int s) {
            const int gi = h * F::kGroups + s;
            const uint32_t v = __funnelshift_r(words[gi >> 1], words[(gi >> 1) + 1], odd * 16);
            return __uint_as_float(gi & 1 ? v & 0xffff0000u : v << 16);
          };
          const Two bias = two(-kFloatBiasValue, -kFloatBiasValue), high_weight = two(256.0f, 256.0f);
          Two block_a[NT], block_b[NT];  // the block's sums over groups, rows g and g + 8
          float block_p[2] = {0.f, 0.f};
#pragma unroll
          for (int n = 0; n < NT; ++n) block_a[n] = block_b[n] = two(0.f, 0.f);
#pragma unroll
          for (int s = 0; s < F::kGroups; ++s) {
            int4 high[NT], low[NT];
#pragma unroll
            for (int w = 0; w < F::kWords; ++w) {
              const uint32_t u = aw[s * F::kWords + w], v = bw[s * F::kWords + w];
              const uint32_t a0 = (u << 4 & 0xf0f0f0f0u) ^ 0x80808080u, a1 = (v << 4 & 0xf0f0f0f0u) ^ 0x80808080u;
              const uint32_t a2 = (u & 0xf0f0f0f0u) ^ 0x80808080u, a3 = (v & 0xf0f0f0f0u) ^ 0x80808080u;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const uint8_t* from = x_at[n] + h * (F::kPart * 2) + (s * F::kWords + w) * 64;
                if constexpr (kPacked) {
                  const uint2 x2 = *reinterpret_cast<const uint2*>(from);
                  mma_bytes(high[n], w == 0 ? start : high[n], a0, a1, a2, a3, x2.x, x2.y);
                } else {
                  const uint4 x4 = *reinterpret_cast<const uint4*>(from);
                  mma_bytes(high[n], w == 0 ? start : high[n], a0, a1, a2, a3, x4.x, x4.y);
                  mma_bytes(low[n], w == 0 ? start : low[n], a0, a1, a2, a3, x4.z, x4.w);
                }
              }
            }
            const float fa = scale_of(sa, odd_a, s), fb = scale_of(sb, odd_b, s);
            if constexpr (kPacked) {
              const float2 va = split(add(two(high[0].x, high[0].y), bias)), vb = split(add(two(high[0].z, high[0].w), bias));
              block_p[0] = fmaf(fa, fmaf(va.x, 256.0f, va.y), block_p[0]);
              block_p[1] = fmaf(fb, fmaf(vb.x, 256.0f, vb.y), block_p[1]);
            } else {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const Two sum_a = fma(add(two(high[n].x, high[n].y), bias), high_weight, add(two(low[n].x, low[n].y), bias));
                const Two sum_b = fma(add(two(high[n].z, high[n].w), bias), high_weight, add(two(low[n].z, low[n].w), bias));
                block_a[n] = fma(two(fa, fa), sum_a, block_a[n]);
                block_b[n] = fma(two(fb, fb), sum_b, block_b[n]);
              }
            }
          }
          const int block = step * kParts + h;
          if constexpr (kPacked) {
            const float unit = units_at[0][0][block];
            acc[0][0] = fmaf(unit, block_p[0], acc[0][0]);
            acc[0][2] = fmaf(unit, block_p[1], acc[0][2]);
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const Two ux = two(units_at[n][0][block], units_at[n][1][block]);
              const float2 ra2 = split(fma(ux, block_a[n], two(acc[n][0], acc[n][1])));
              const float2 rb2 = split(fma(ux, block_b[n], two(acc[n][2], acc[n][3])));
              acc[n][0] = ra2.x, acc[n][1] = ra2.y;
              acc[n][2] = rb2.x, acc[n][3] = rb2.y;
            }
          }
        }
      }
    }
    __syncwarp();  // every lane has read the slot
    issue();
    at += F::kSlot;
    if (at == ring + kDepth * F::kSlot) at = ring;
    if (++i == per_warp) {
      // ---- end of the unit: add the sums of each tile's warps (in warp order) and write
      i = 0;
      float* mine = part + ((buffer * kWarps + warp) * kCols + (kPacked ? q : 2 * q)) * 16 + g;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mine[n * 128] = acc[n][0];
        mine[n * 128 + 8] = acc[n][2];
        if constexpr (!kPacked) {
          mine[n * 128 + 16] = acc[n][1];
          mine[n * 128 + 24] = acc[n][3];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[n][j] = 0.f;
      }
      if (any_mixed) add_mixed(mine);
      __syncthreads();
      const float* all = part + buffer * kWarps * kCols * 16;
      // the half of the warps that adds first alternates, as there may be work for one half only
      for (int o = (threadIdx.x + buffer * (kThreads / 2)) % kThreads; o < tiles_at_once * kOut * kCols; o += kThreads) {
        const int r = o % kOut, c = o / kOut % kCols, t = o / (kOut * kCols);
        const int row = (unit * tiles_at_once + t) * kOut + r;
        if (c >= item.count || row >= a.rows) continue;
        const float* from = all + (t * a.k_warps * kCols + c) * 16 + r;
        float v = 0.f, u = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          if (w >= a.k_warps) break;
          v += from[w * kCols * 16];
          if constexpr (kGateUp) u += from[w * kCols * 16 + 8];
        }
        if constexpr (kGateUp) v = v * sigmoid(v) * u;
        const size_t at = static_cast<size_t>(routed ? order[item.first + c] : item.first + c) * a.out_stride + row;
        if (a.out_f32)
          static_cast<float*>(a.out)[at] = v;
        else
          static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
      }
      if constexpr (part_buffers(kWarps) == 2)
        buffer ^= 1;
      else
        __syncthreads();
      if (--units_left == 0) return;
      if (++unit == per_item) {  // the next item's x rows; every warp has used the old ones
        unit = 0;
        item = item_of(++item_index);
        load_x(item, item_index + 1, warp);
        __syncthreads();
        point_x();
        any_mixed = kFmt != 0 && *mixed_mark == item_index + 1;
      }
      point_scales();
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

template <int kFmt, int kCols>
size_t smem_bytes(const SkinnyArgs& a, int warps) {
  const int step = Format<kFmt>::kStep;
  const int padded = (a.k + step - 1) / step * step;
  const bool routed = a.indices != nullptr;
  return carve_smem(warps, Format<kFmt>::kSlot, kCols, a.cols, padded, kFmt == 0 ? 0 : padded / 128,
                    routed ? a.pairs : 0, routed ? a.experts : 0)
      .total;
}

template <int kFmt, bool kGateUp, int kCols, int kWarps>
cudaError_t launch_warps(SkinnyArgs a, cudaStream_t stream);

// Eight warps a CTA and two CTAs an SM; where x rows leave room for one, sixteen warps if they fit.
template <int kFmt, bool kGateUp, int kCols>
cudaError_t launch_tile(const SkinnyArgs& a, cudaStream_t stream) {
  const size_t two = smem_bytes<kFmt, kCols>(a, 8), one = smem_bytes<kFmt, kCols>(a, 16);
  return 2 * (two + 1024) > kSmemPerSm && one <= kMaxSmem ? launch_warps<kFmt, kGateUp, kCols, 16>(a, stream)
                                                          : launch_warps<kFmt, kGateUp, kCols, 8>(a, stream);
}

template <int kFmt, bool kGateUp, int kCols, int kWarps>
cudaError_t launch_warps(SkinnyArgs a, cudaStream_t stream) {
  const auto kernel = skinny_kernel<kFmt, kGateUp, kCols, kWarps>;
  const int step = Format<kFmt>::kStep;
  const int steps = (a.k + step - 1) / step;
  const bool routed = a.indices != nullptr;
  const size_t smem = smem_bytes<kFmt, kCols>(a, kWarps);
  if (smem > kMaxSmem) return cudaErrorInvalidValue;
  static PerDeviceOnce attr;
  cudaError_t err =
      attr.run([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem); });
  if (err != cudaSuccess) return err;
  const int items = routed ? a.pairs : (a.tokens + a.cols - 1) / a.cols;
  const int slots = device_sm_count() * (kWarps == 8 && 2 * (smem + 1024) <= kSmemPerSm ? 2 : 1);
  // Warps to a tile: a unit costs its steps per warp and about 1.5 more for the barrier and the additions at
  // its end, and the CTA with the most units decides. (On 16384 x 8192 at 7
  // columns 2 warps take 24.4 us and 16 take 29.0.) With routing the expected number of experts stands for
  // the items.
  const double likely = routed ? a.experts * (1.0 - std::exp(-static_cast<double>(a.pairs) / a.experts)) : 0.0;
  const long long expected = routed ? static_cast<long long>(likely) + 1 : items;
  long long best = 0;
  for (int k = 1; k <= kWarps; k *= 2) {
    const int rows = (kGateUp ? 8 : 16) * (kWarps / k);
    const long long n = expected * ((a.rows + rows - 1) / rows);
    const long long cost = (n + slots - 1) / slots * (2 * ((steps + k - 1) / k) + 3);
    if (best == 0 || cost < best) {
      best = cost;
      a.k_warps = k;
    }
  }
  const int unit_rows = (kGateUp ? 8 : 16) * (kWarps / a.k_warps);
  const long long most = static_cast<long long>(items) * ((a.rows + unit_rows - 1) / unit_rows);
  const int grid = static_cast<int>(most < slots ? most : slots);
  return launch_kernel(kernel, dim3(grid), 32 * kWarps, smem, stream, a);
}

template <int kFmt, bool kGateUp>
cudaError_t launch_columns(const SkinnyArgs& a, cudaStream_t stream) {
  const int cols = tile_columns(kFmt == 0, a.cols);
  if constexpr (kFmt != 0)
    if (cols == 4) return launch_tile<kFmt, kGateUp, 4>(a, stream);
  if (cols == 8) return launch_tile<kFmt, kGateUp, 8>(a, stream);
  if constexpr (kFmt == 0 || !kGateUp) return launch_tile<kFmt, kGateUp, 16>(a, stream);
  return cudaErrorInvalidValue;  // 4-bit gate/up products are the experts', at most 8 columns
}

template <bool kGateUp>
cudaError_t launch_format(const SkinnyArgs& a, int group, cudaStream_t stream) {
  switch (group) {
    case 0: return launch_columns<0, kGateUp>(a, stream);
    case 32: return launch_columns<32, kGateUp>(a, stream);
    case 64: return launch_columns<64, kGateUp>(a, stream);
    case 128: return launch_columns<128, kGateUp>(a, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace

int skinny_columns(int want, int k, int group, int pairs, int experts) {
  const int step = group == 0 ? Format<0>::kStep : Format<32>::kStep;
  const int slot = group == 0 ? Format<0>::kSlot : group == 128 ? Format<128>::kSlot : group == 64 ? Format<64>::kSlot : Format<32>::kSlot;
  const int padded = (k + step - 1) / step * step;
  int cols = want < kSkinnyMaxColumns ? want : kSkinnyMaxColumns;
  const int blocks = group == 0 ? 0 : padded / 128;
  while (cols > 0 &&
         carve_smem(8, slot, tile_columns(group == 0, cols), cols, padded, blocks, pairs, experts).total > kMaxSmem)
    --cols;
  return cols;
}

cudaError_t launch_skinny(const SkinnyArgs& a, int group, bool gate_up, cudaStream_t stream) {
  if (a.cols < 1 || a.cols > kSkinnyMaxColumns) return cudaErrorInvalidValue;
  return gate_up ? launch_format<true>(a, group, stream) : launch_format<false>(a, group, stream);
}

cudaError_t launch_weighted_rows(const float* rows, const int32_t* indices, const float* weights, int tokens, int topk,
                                 int experts, int hidden, __nv_bfloat16* out, cudaStream_t stream) {
  return launch_kernel(weighted_rows_kernel, dim3((hidden / 4 + 255) / 256, tokens), 256, 0, stream, rows, indices,
                       weights, topk, experts, hidden, out);
}

}  // namespace cernels
