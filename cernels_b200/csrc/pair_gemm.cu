// Matrix products of the gated feed-forward block and of its backward pass (bf16 operands,
// 32-bit sums) on sm_100a tensor cores, two CTAs to a tile.
//
//   forward    g = x Wg^T, u = x Wu^T, h = silu(g) u         (kGateUp: both products and h in one pass)
//              y = h Wd^T                                     (kPlain)
//   backward   dh = dy Wd; du = dh g s; dg = dh u s (1 + g (1 - s)), s = sigmoid(g)   (kGradGateUp)
//              dx = dg Wg + du Wu; dWg = dg^T x; dWu = du^T x; dWd = dy^T h           (kPlain, one launch)
//
// A CTA pair computes a 256 x BN tile of one product: each CTA stages half of A's rows (128) and
// half of B's rows (BN / 2) of every 64-deep K block by TMA, the pair's first CTA issues
// tcgen05.mma.cta_group::2, and each CTA's TMEM receives its own 128 rows of the sum. Halving B per
// CTA is what this buys: 32 KB per SM and K block instead of 48 KB for the same 128 x 256 result.
// Operands are read where they lie: K-major for x Wg^T, MN-major (64-column boxes) where the
// reduction runs over rows, so no product needs a transposed copy.
//
// Per CTA, 320 threads: warp 0 TMA loads, warp 1 TMEM and (in CTA 0) the MMAs, warps 2-9 the
// epilogue: warp w reads TMEM lanes 32 (w % 4).. of one half of the tile's columns, and writes
// 32 x 64 windows through shared memory with TMA stores, which clip ragged edges. Two
// accumulators let the epilogue of a tile overlap the next tile's MMAs.
//
// The backward pass keeps g and u in 32 bits (8 F bytes a token): recomputing them would cost
// 4 H F operations a token against 16 F bytes of traffic, more for H above about 1000, and
// rounding them to bf16 would add its error to every gradient. h, dg and du are rounded to bf16,
// once each: they are operands of the next product.
#include <algorithm>
#include <cmath>

#include "ffn_internal.h"
#include "pair_drain.h"
#include "pair_gemm.cuh"

namespace cernels {
namespace {

constexpr int kBM = 128;  // rows of A per CTA
constexpr int kBK = 64;
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kABytes = kBM * kBK * 2;
constexpr int kBoxBytes = 64 * kBK * 2;  // 64 columns x 64 K rows
constexpr int kWindowBytes = 32 * 128;   // 32 rows x 64 bf16
constexpr int kSmemLimit = 232448;
constexpr int kMaxProblems = 4;
constexpr int kMaxMaps = 16;
constexpr int kGroupM = 8;  // row tiles that run together, for reuse of B in L2

enum Epilogue : int { kPlain, kGateUp, kGradGateUp };

template <int kEpi, int BN>
struct Config {
  static constexpr int kBBytes = BN / 2 * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kWindows = kEpi == kGradGateUp ? 2 : 1;  // staging windows per epilogue warp
  static constexpr int kStaging = kEpiWarps * kWindows * kWindowBytes;
  static constexpr int kFit = (kSmemLimit - 1024 - 256 - kStaging) / kStageBytes;
  static constexpr int kStages = kFit < 8 ? kFit : 8;
  static constexpr int kSmem = 1024 + kStages * kStageBytes + kStaging + 256;
};

// One product A B^T of the launch: `m` x `n` outputs, reduction over up to two pairs of operands
// (dx adds two products). Maps are indices into Maps::m.
struct Problem {
  int m, n;
  int kb[2];           // 64-deep blocks of each reduction segment
  int m_tiles, n_tiles;
  int tile_begin;
  int a_mn, b_mn;      // operand is MN-major: its rows run along the reduction
  int a_map[2], b_map[2];  // per segment; kGateUp: b_map[0] gate, b_map[1] up, one segment
  int out_map[2];
};

struct alignas(64) Maps {
  CUtensorMap m[kMaxMaps];
};

struct PairArgs {
  Problem p[kMaxProblems];
  int problems, total_tiles;
  float* gate_up;  // stored products (kGateUp writes when not null, kGradGateUp reads)
  int inter;       // F
  int row_blocks;  // ceil(T / 32)
  unsigned long long wait_ns;
};

// Nonzero after a bounded wait of these kernels gave up on this device; see ffn_status().
__device__ int g_ffn_status;

struct Tile {
  int problem, m_tile, n_tile;
};

__device__ __forceinline__ Tile decode(const PairArgs& a, int t) {
  Tile r;
  r.problem = 0;
#pragma unroll
  for (int i = 1; i < kMaxProblems; ++i)
    if (i < a.problems && t >= a.p[i].tile_begin) r.problem = i;
  const Problem& p = a.p[r.problem];
  const int local = t - p.tile_begin;
  const int per_group = kGroupM * p.n_tiles;
  const int group = local / per_group, in = local - group * per_group;
  const int rows = min(kGroupM, p.m_tiles - group * kGroupM);
  r.n_tile = in / rows;
  r.m_tile = group * kGroupM + in - r.n_tile * rows;
  return r;
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 1 / (1 + exp(-g)) to a few units in the last place of 32 bits (far below the bf16 rounding of
// what it enters); 0 once exp(-g) passes the 32-bit range. The exact division costs a branch a
// value, which took a gate/up tile's epilogue from 3,000 to 8,000 cycles.
__device__ __forceinline__ float sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// Writes N values of this lane's row into columns [col, col + N) of a 32 x 64 window that is laid
// out as the 128-byte swizzle of the output maps has it (16-byte pieces exchanged by row % 8).
template <int N>
__device__ __forceinline__ void stage(uint8_t* window, int lane, int col, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    uint4 q;
    q.x = pack2(v[8 * i], v[8 * i + 1]);
    q.y = pack2(v[8 * i + 2], v[8 * i + 3]);
    q.z = pack2(v[8 * i + 4], v[8 * i + 5]);
    q.w = pack2(v[8 * i + 6], v[8 * i + 7]);
    const int piece = (col >> 3) + i;
    *reinterpret_cast<uint4*>(window + lane * 128 + ((piece ^ (lane & 7)) << 4)) = q;
  }
}

// Waits until every load has landed that the CTAs of the pair started (pair_drain.h), kBytes a block and CTA. CTA 0.
template <int kStages, int kBytes>
__device__ void drain_loads(uint64_t* full_bar, long long mine, long long other) {
  for (long long i = drain_first(mine, other, kStages); i < max(mine, other); ++i) {
    uint64_t* bar = &full_bar[i % kStages];
    const Drain action = drain_action(i, mine, other);
    if (action == Drain::kAnnounce) mbar_arrive_expect_tx(bar, kBytes);
    if (action == Drain::kCancel) mbar_complete_tx(bar, kBytes);
    mbar_drain(bar, static_cast<uint32_t>((i / kStages) & 1), kWaitLimitNs);
  }
}

template <int kEpi, int BN>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    pair_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ PairArgs args) {
  using C = Config<kEpi, BN>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages * kABytes;
  uint8_t* staging = smem + kStages * C::kStageBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(staging + C::kStaging);
  uint64_t* full_bar = bars;                  // [kStages] used in CTA 0
  uint64_t* empty_bar = bars + kStages;       // [kStages]
  uint64_t* tfull_bar = bars + 2 * kStages;   // [2]
  uint64_t* tempty_bar = tfull_bar + 2;       // [2] used in CTA 0
  uint64_t* drain_bar = tempty_bar + 2;       // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain_bar + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile long long* issued_count = reinterpret_cast<volatile long long*>(tmem_slot + 2);  // K blocks whose loads started
  volatile int* peer_abort = reinterpret_cast<volatile int*>(tmem_slot + 4);  // the other CTA's abort_flag, when it is over

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = pair_rank();
  const int pair = blockIdx.x >> 1;
  const int pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull_bar[i], 1);
      mbar_init(&tempty_bar[i], 2 * kEpiWarps);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    *issued_count = 0;
    *peer_abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  pair_sync();  // both CTAs' barriers exist before any remote arrive
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  wait_for_previous_kernel();

  if (warp == 0) {
    // ------------------------------------------------------------ TMA loads
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      long long issued = 0;
      for (int t = pair; t < args.total_tiles && ok; t += pairs) {
        const Tile c = decode(args, t);
        const Problem& p = args.p[c.problem];
        const int m0 = c.m_tile * 2 * kBM + static_cast<int>(rank) * kBM;
        const int n0 = kEpi == kGateUp ? c.n_tile * (BN / 2) : c.n_tile * BN + static_cast<int>(rank) * (BN / 2);
        for (int seg = 0; seg < 2 && ok; ++seg) {
          const CUtensorMap* ma = &maps.m[p.a_map[seg]];
          const CUtensorMap* mb = &maps.m[kEpi == kGateUp ? p.b_map[rank] : p.b_map[seg]];
          for (int kb = 0; kb < p.kb[seg]; ++kb) {
            if (!mbar_wait_bounded(&empty_bar[stage], phase ^ 1u, &g_ffn_status, kStatusTimeoutProducer, abort_flag,
                                   args.wait_ns)) {
              ok = false;
              break;
            }
            if (rank == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * C::kStageBytes);
            const uint32_t bar = leader_smem(&full_bar[stage]);
            uint8_t* a_dst = smem_a + stage * kABytes;
            uint8_t* b_dst = smem_b + stage * C::kBBytes;
            const int k0 = kb * kBK;
            if (p.a_mn) {
              tma_load_2d_pair(a_dst, ma, bar, m0, k0);
              tma_load_2d_pair(a_dst + kBoxBytes, ma, bar, m0 + 64, k0);
            } else {
              tma_load_2d_pair(a_dst, ma, bar, k0, m0);
            }
            if (p.b_mn) {
#pragma unroll
              for (int j = 0; j < BN / 128; ++j) tma_load_2d_pair(b_dst + j * kBoxBytes, mb, bar, n0 + 64 * j, k0);
            } else {
              tma_load_2d_pair(b_dst, mb, bar, k0, n0);
            }
            ++issued;
            if (++stage == kStages) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      *issued_count = issued;
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issue
    if (rank == 0 && elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      bool ok = true;
      for (int t = pair; t < args.total_tiles && ok; t += pairs, ++local) {
        const Tile c = decode(args, t);
        const Problem& p = args.p[c.problem];
        const uint32_t idesc = make_idesc_bf16(2 * kBM, BN, p.a_mn, p.b_mn);
        // K-major: 16 K values are 32 bytes along a swizzled row. MN-major: 16 K values are 16 rows
        // of 128 bytes, and the next 64 columns start a box further.
        const uint32_t a_step = p.a_mn ? 2048 : 32, b_step = p.b_mn ? 2048 : 32;
        const uint32_t a_lbo = p.a_mn ? kBoxBytes : 16, b_lbo = p.b_mn ? kBoxBytes : 16;
        const int acc = local & 1;
        if (!mbar_wait_bounded(&tempty_bar[acc], ((local >> 1) & 1) ^ 1u, &g_ffn_status, kStatusTimeoutMma, abort_flag,
                               args.wait_ns))
          break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
        const int blocks = p.kb[0] + p.kb[1];
        for (int kb = 0; kb < blocks; ++kb) {
          if (!mbar_wait_bounded(&full_bar[stage], phase, &g_ffn_status, kStatusTimeoutMma, abort_flag, args.wait_ns)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem_a + stage * kABytes);
          const uint32_t b_addr = smem_u32(smem_b + stage * C::kBBytes);
#pragma unroll
          for (int kk = 0; kk < kBK / 16; ++kk)
            umma_bf16_pair(d_tmem, make_smem_desc_sw128(a_addr + kk * a_step, a_lbo, 1024),
                           make_smem_desc_sw128(b_addr + kk * b_step, b_lbo, 1024), idesc, (kb | kk) != 0 ? 1u : 0u);
          umma_commit_pair(&empty_bar[stage]);
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit_pair(&tfull_bar[acc]);
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ epilogue
    const int quarter = warp & 3;        // TMEM lanes this warp can read
    const int half = (warp - 2) >> 2;    // its half of the tile's columns
    float4* saved = reinterpret_cast<float4*>(args.gate_up);
    uint8_t* window = staging + (warp - 2) * C::kWindows * kWindowBytes;
    int local = 0;
    for (int t = pair; t < args.total_tiles; t += pairs, ++local) {
      const Tile c = decode(args, t);
      const Problem& p = args.p[c.problem];
      const int acc = local & 1;
      const int row0 = c.m_tile * 2 * kBM + static_cast<int>(rank) * kBM + quarter * 32;
      const size_t row_block = static_cast<size_t>(row0 >> 5);
      if (!mbar_wait_bounded(&tfull_bar[acc], (local >> 1) & 1, &g_ffn_status, kStatusTimeoutEpilogue, abort_flag,
                             args.wait_ns))
        break;
      tc_fence_after();
      const uint32_t t_row = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(acc * BN);

      auto reuse = [&] {  // the window's last store has read it
        if (lane == 0) bulk_wait_read();
        __syncwarp();
      };
      auto flush = [&](int map, const uint8_t* from, int col0) {
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row0 < p.m && col0 < p.n) tma_store_2d(&maps.m[map], from, col0, row0);
          bulk_commit_group();
        }
      };

      if constexpr (kEpi == kPlain) {
#pragma unroll 1
        for (int w = 0; w < BN / 128; ++w) {
          const int col = half * (BN / 2) + 64 * w;
          reuse();
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float v[32];
            tmem_ld_32x32b_x32(t_row + col + 32 * i, v);
            stage(window, lane, 32 * i, v);
          }
          flush(p.out_map[0], window, c.n_tile * BN + col);
        }
      } else if constexpr (kEpi == kGateUp) {
        // columns [0, BN / 2) hold gate products, [BN / 2, BN) the up products of the same outputs
        if (half * 64 < BN / 2) {
          const int out0 = c.n_tile * (BN / 2) + half * 64;
          reuse();
#pragma unroll 1
          for (int i = 0; i < 2; ++i) {
            float g[32], u[32];
            tmem_ld_32x32b_x32(t_row + half * 64 + 32 * i, g);
            tmem_ld_32x32b_x32(t_row + BN / 2 + half * 64 + 32 * i, u);
            if (args.gate_up != nullptr && row_block < static_cast<size_t>(args.row_blocks)) {
              const int f = out0 + 32 * i;
              float4* dst = saved + ((row_block * (args.inter >> 2) + (f >> 2)) << 6) + lane;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (f + 4 * j < args.inter) {
                  dst[64 * j] = make_float4(g[4 * j], g[4 * j + 1], g[4 * j + 2], g[4 * j + 3]);
                  dst[64 * j + 32] = make_float4(u[4 * j], u[4 * j + 1], u[4 * j + 2], u[4 * j + 3]);
                }
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) g[j] = g[j] * sigmoid(g[j]) * u[j];
            stage(window, lane, 32 * i, g);
          }
          flush(p.out_map[0], window, out0);
        }
      } else {
// 16 columns at a time; the stored products of the next 16 are on their way meanwhile
        constexpr int kChunks = BN / 32;
        const int f0 = c.n_tile * BN + half * (BN / 2);
        const float4* src = saved + ((row_block * (args.inter >> 2) + (f0 >> 2)) << 6) + lane;
        const int live = row_block < static_cast<size_t>(args.row_blocks) ? args.inter - f0 : 0;  // columns that exist
        float4 g4[2][4], u4[2][4];
        auto fetch = [&](int ch) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool in = 16 * ch + 4 * j < live;
            g4[ch & 1][j] = in ? __ldcs(src + 64 * (4 * ch + j)) : make_float4(0.f, 0.f, 0.f, 0.f);
            u4[ch & 1][j] = in ? __ldcs(src + 64 * (4 * ch + j) + 32) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
        };
        fetch(0);
#pragma unroll
        for (int ch = 0; ch < kChunks; ++ch) {
          if (ch + 1 < kChunks) fetch(ch + 1);
          if (ch % 4 == 0) reuse();
          float d[16], e[16];
          tmem_ld_32x32b_x16(t_row + half * (BN / 2) + 16 * ch, d);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float4 gq = g4[ch & 1][j >> 2], uq = u4[ch & 1][j >> 2];
            const float g = j % 4 == 0 ? gq.x : j % 4 == 1 ? gq.y : j % 4 == 2 ? gq.z : gq.w;
            const float u = j % 4 == 0 ? uq.x : j % 4 == 1 ? uq.y : j % 4 == 2 ? uq.z : uq.w;
            const float dh = d[j], s = sigmoid(g);
            e[j] = dh * (g * s);
            d[j] = dh * u * (s * (1.0f + g * (1.0f - s)));
          }
          stage(window, lane, 16 * (ch % 4), d);
          stage(window + kWindowBytes, lane, 16 * (ch % 4), e);
          if (ch % 4 == 3) {
            const int out0 = f0 + 16 * (ch - 3);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row0 < p.m && out0 < p.n) {
                tma_store_2d(&maps.m[p.out_map[0]], window, out0, row0);
                tma_store_2d(&maps.m[p.out_map[1]], window + kWindowBytes, out0, row0);
              }
              bulk_commit_group();
            }
          }
        }
      }
      // every TMEM read of this accumulator is done
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_leader(leader_smem(&tempty_bar[acc]));
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) store_peer(peer_abort, rank ^ 1u, 1);
  __syncwarp();
  pair_sync();  // neither CTA leaves while the other may still reach its shared memory or TMEM
  // A wait gave up, whichever role's and in whichever CTA (both see the same here): loads and MMAs that it did
  // not wait for may be in flight in both CTAs. They end within this kernel, however short the limit of its waits.
  if (*abort_flag != 0 || *peer_abort != 0) {
    if (warp == 1) {
      if (elect_one()) {
        if (rank == 0) {
          umma_commit_pair(drain_bar);  // of the thread that issued the MMAs: elect_one() has one answer per warp
          drain_loads<kStages, C::kStageBytes>(full_bar, *issued_count, load_peer(issued_count, 1));
        }
        mbar_drain(drain_bar, 0, kWaitLimitNs);
      }
      __syncwarp();
    }
    __syncthreads();
    pair_sync();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 2 * BN);
  }
}

// ---------------------------------------------------------------- host side
struct Builder {
  Maps maps;
  PairArgs args{};
  int count = 0;
  bool ok = true;

  int add(const void* ptr, int cols, int rows, size_t stride, int box_cols, int box_rows) {
    if (count == kMaxMaps) {
      ok = false;
      return 0;
    }
    const uint64_t dims[2] = {static_cast<uint64_t>(cols), static_cast<uint64_t>(rows)};
    const uint64_t strides[1] = {static_cast<uint64_t>(stride) * 2};
    const uint32_t box[2] = {static_cast<uint32_t>(box_cols), static_cast<uint32_t>(box_rows)};
    ok = ok && encode_bf16_map(&maps.m[count], ptr, 2, dims, strides, box);
    return count++;
  }
  // operand of a [rows, cols] matrix whose rows run along the output (K-major) or along the reduction
  int k_major(const void* ptr, int rows, int cols, size_t stride, int tile_rows) {
    return add(ptr, cols, rows, stride, kBK, tile_rows);
  }
  int mn_major(const void* ptr, int rows, int cols, size_t stride) { return add(ptr, cols, rows, stride, 64, kBK); }
  int output(const void* ptr, int rows, int cols) { return add(ptr, cols, rows, cols, 64, 32); }

  Problem& problem(int m, int n, int tile_n) {
    Problem& p = args.p[args.problems++];
    p = Problem{};
    p.m = m;
    p.n = n;
    p.m_tiles = (m + 2 * kBM - 1) / (2 * kBM);
    p.n_tiles = (n + tile_n - 1) / tile_n;
    p.tile_begin = args.total_tiles;
    args.total_tiles += p.m_tiles * p.n_tiles;
    return p;
  }
};

int blocks_of(int k) { return (k + kBK - 1) / kBK; }

template <int kEpi, int BN>
cudaError_t launch(Builder& b, cudaStream_t stream) {
  if (!b.ok) return cudaErrorInvalidValue;
  using C = Config<kEpi, BN>;
  static_assert(C::kStages >= 3 && C::kSmem <= kSmemLimit, "tile does not fit shared memory");
  static PerDeviceOnce attr;
  cudaError_t err = attr.run([] {
    return cudaFuncSetAttribute(pair_gemm_kernel<kEpi, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  });
  if (err != cudaSuccess) return err;
  const int max_pairs = device_sm_count() / 2;
  const int pairs = b.args.total_tiles < max_pairs ? b.args.total_tiles : max_pairs;
  if (pairs <= 0) return cudaSuccess;
  b.args.wait_ns = wait_limit_ns(kWaitLimitNs);
  return launch_kernel(pair_gemm_kernel<kEpi, BN>, dim3(2 * pairs), kThreads, C::kSmem, stream, b.maps, b.args);
}

int tiles_of(int m, int n, int tile_n) { return (m + 2 * kBM - 1) / (2 * kBM) * ((n + tile_n - 1) / tile_n); }

// Whether 128-wide tiles beat 256-wide ones for `wide` and `narrow` tiles of each: a launch takes as many
// rounds as its fullest pair has tiles, and a 128-wide tile costs 0.75 of a 256-wide one: both are bound by the
// 64 bytes a cycle that an SM gets from L2, and it needs 24 KB per K block instead of 32. (Forward at T = 301,
// H = 2048, F = 768: 18.9 us with 128, 24.9 with 256; at T = 4096, F = 1408: 65.0 and 56.4.)
bool narrow_tiles(double wide, double narrow) {
  const int pairs = device_sm_count() / 2;
  return std::ceil(narrow / pairs) * 0.75 < std::ceil(wide / pairs);
}

template <int BN>
cudaError_t gate_up(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                    const __nv_bfloat16* up, __nv_bfloat16* h, float* stored, cudaStream_t stream) {
  Builder b;
  Problem& p = b.problem(s.tokens, s.inter, BN / 2);
  p.kb[0] = blocks_of(s.hidden);
  p.a_map[0] = b.k_major(x, s.tokens, s.hidden, x_stride, kBM);
  p.b_map[0] = b.k_major(gate, s.inter, s.hidden, s.hidden, BN / 2);
  p.b_map[1] = b.k_major(up, s.inter, s.hidden, s.hidden, BN / 2);
  p.out_map[0] = b.output(h, s.tokens, s.inter);
  b.args.gate_up = stored;
  b.args.inter = s.inter;
  b.args.row_blocks = (s.tokens + 31) / 32;
  return launch<kGateUp, BN>(b, stream);
}

template <int BN>
cudaError_t down_product(const FfnShape& s, const __nv_bfloat16* h, const __nv_bfloat16* down, __nv_bfloat16* out,
                         cudaStream_t stream) {
  Builder b;
  Problem& p = b.problem(s.tokens, s.hidden, BN);
  p.kb[0] = blocks_of(s.inter);
  p.a_map[0] = b.k_major(h, s.tokens, s.inter, s.inter, kBM);
  p.b_map[0] = b.k_major(down, s.hidden, s.inter, s.inter, BN / 2);
  p.out_map[0] = b.output(out, s.tokens, s.hidden);
  return launch<kPlain, BN>(b, stream);
}

template <int BN>
cudaError_t d_gate_up(const FfnShape& s, const __nv_bfloat16* dy, const __nv_bfloat16* down, const float* stored,
                      __nv_bfloat16* d_gate, __nv_bfloat16* d_up, cudaStream_t stream) {
  Builder b;
  Problem& p = b.problem(s.tokens, s.inter, BN);
  p.kb[0] = blocks_of(s.hidden);
  p.b_mn = 1;
  p.a_map[0] = b.k_major(dy, s.tokens, s.hidden, s.hidden, kBM);
  p.b_map[0] = b.mn_major(down, s.hidden, s.inter, s.inter);
  p.out_map[0] = b.output(d_gate, s.tokens, s.inter);
  p.out_map[1] = b.output(d_up, s.tokens, s.inter);
  b.args.gate_up = const_cast<float*>(stored);
  b.args.inter = s.inter;
  b.args.row_blocks = (s.tokens + 31) / 32;
  return launch<kGradGateUp, BN>(b, stream);
}

template <int BN>
cudaError_t grads(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                  const __nv_bfloat16* up, const __nv_bfloat16* h, const __nv_bfloat16* dy,
                  const __nv_bfloat16* d_gate, const __nv_bfloat16* d_up, const FfnGrads& out, cudaStream_t stream) {
  Builder b;
  const int T = s.tokens, H = s.hidden, F = s.inter;
  auto weight = [&](__nv_bfloat16* w, const __nv_bfloat16* a, int a_cols, const __nv_bfloat16* bb, int b_cols,
                    size_t b_stride) {
    Problem& p = b.problem(a_cols, b_cols, BN);
    p.kb[0] = blocks_of(T);
    p.a_mn = p.b_mn = 1;
    p.a_map[0] = b.mn_major(a, T, a_cols, a_cols);
    p.b_map[0] = b.mn_major(bb, T, b_cols, b_stride);
    p.out_map[0] = b.output(w, a_cols, b_cols);
  };
  auto input = [&] {
    Problem& p = b.problem(T, H, BN);
    p.kb[0] = p.kb[1] = blocks_of(F);
    p.b_mn = 1;
    p.a_map[0] = b.k_major(d_gate, T, F, F, kBM);
    p.a_map[1] = b.k_major(d_up, T, F, F, kBM);
    p.b_map[0] = b.mn_major(gate, F, H, H);
    p.b_map[1] = b.mn_major(up, F, H, H);
    p.out_map[0] = b.output(out.dx, T, H);
  };
  // the product with the longest reduction first: its tiles are the ones that must not start last
  const bool input_first = 2 * blocks_of(F) > blocks_of(T);
  if (out.dx && input_first) input();
  if (out.dw_gate) weight(out.dw_gate, d_gate, F, x, H, x_stride);
  if (out.dw_up) weight(out.dw_up, d_up, F, x, H, x_stride);
  if (out.dw_down) weight(out.dw_down, dy, H, h, F, F);
  if (out.dx && !input_first) input();
  return launch<kPlain, BN>(b, stream);
}

}  // namespace

cudaError_t launch_ffn_gate_up(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                               const __nv_bfloat16* up, __nv_bfloat16* h, float* stored, cudaStream_t stream) {
  return narrow_tiles(tiles_of(s.tokens, s.inter, 128), tiles_of(s.tokens, s.inter, 64))
             ? gate_up<128>(s, x, x_stride, gate, up, h, stored, stream)
             : gate_up<256>(s, x, x_stride, gate, up, h, stored, stream);
}
cudaError_t launch_ffn_down(const FfnShape& s, const __nv_bfloat16* h, const __nv_bfloat16* down, __nv_bfloat16* out,
                            cudaStream_t stream) {
  return narrow_tiles(tiles_of(s.tokens, s.hidden, 256), tiles_of(s.tokens, s.hidden, 128))
             ? down_product<128>(s, h, down, out, stream)
             : down_product<256>(s, h, down, out, stream);
}
cudaError_t launch_ffn_d_gate_up(const FfnShape& s, const __nv_bfloat16* dy, const __nv_bfloat16* down,
                                 const float* stored, __nv_bfloat16* d_gate, __nv_bfloat16* d_up,
                                 cudaStream_t stream) {
  return narrow_tiles(tiles_of(s.tokens, s.inter, 256), tiles_of(s.tokens, s.inter, 128))
             ? d_gate_up<128>(s, dy, down, stored, d_gate, d_up, stream)
             : d_gate_up<256>(s, dy, down, stored, d_gate, d_up, stream);
}
cudaError_t launch_ffn_grads(const FfnShape& s, const __nv_bfloat16* x, size_t x_stride, const __nv_bfloat16* gate,
                             const __nv_bfloat16* up, const __nv_bfloat16* h, const __nv_bfloat16* dy,
                             const __nv_bfloat16* d_gate, const __nv_bfloat16* d_up, const FfnGrads& out,
                             cudaStream_t stream) {
  // tiles of two lengths: weigh them by their K blocks, in units of the longer ones
  auto rounds = [&](int tile_n) {
    const double t_blocks = blocks_of(s.tokens), f_blocks = 2 * blocks_of(s.inter);
    const double work = (out.dx ? tiles_of(s.tokens, s.hidden, tile_n) * f_blocks : 0.0) +
                        t_blocks * ((out.dw_gate ? tiles_of(s.inter, s.hidden, tile_n) : 0) +
                                    (out.dw_up ? tiles_of(s.inter, s.hidden, tile_n) : 0) +
                                    (out.dw_down ? tiles_of(s.hidden, s.inter, tile_n) : 0));
    return work / std::max(t_blocks, f_blocks);
  };
  return narrow_tiles(rounds(256), rounds(128))
             ? grads<128>(s, x, x_stride, gate, up, h, dy, d_gate, d_up, out, stream)
             : grads<256>(s, x, x_stride, gate, up, h, dy, d_gate, d_up, out, stream);
}

cudaError_t ffn_status(int* status, cudaStream_t stream) {
  cudaError_t err = cudaMemcpyFromSymbolAsync(status, g_ffn_status, sizeof(int), 0, cudaMemcpyDeviceToHost, stream);
  const int zero = 0;
  if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  if (err == cudaSuccess && *status != 0) {
    err = cudaMemcpyToSymbolAsync(g_ffn_status, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, stream);
    if (err == cudaSuccess) err = cudaStreamSynchronize(stream);
  }
  return err;
}

}  // namespace cernels
