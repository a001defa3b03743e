// Which loads a CTA pair that gives up has to wait for, and how (pair_gemm.cu). Plain C++: no CUDA needed.
//
// Both CTAs load every K block into the ring's stage `block % stages`; their bytes are counted on one barrier a
// stage, in CTA 0, whose phase for a block ends when CTA 0 has announced both CTAs' bytes and all have landed.
// CTA 0 has started (and announced) blocks [0, mine), CTA 1 blocks [0, other). A block is loaded over another only
// after the MMAs have read that one, so a stage has one phase open at most: that of its last block.
#pragma once

#ifdef __CUDACC__
#define CERNELS_HD __host__ __device__ __forceinline__
#else
#define CERNELS_HD inline
#endif

namespace cernels {

enum class Drain {
  kWait,      // both started it, or the MMAs already waited for it
  kAnnounce,  // only CTA 1 started it: its bytes still have to be announced
  kCancel,    // only CTA 0 did: CTA 1's announced bytes are not coming
};

// The last block of each stage: [drain_first(), max(mine, other)).
CERNELS_HD long long drain_first(long long mine, long long other, int stages) {
  const long long most = mine > other ? mine : other;
  return most > stages ? most - stages : 0;
}

CERNELS_HD Drain drain_action(long long block, long long mine, long long other) {
  if (block >= mine) return Drain::kAnnounce;
  return block >= other ? Drain::kCancel : Drain::kWait;
}

}  // namespace cernels
