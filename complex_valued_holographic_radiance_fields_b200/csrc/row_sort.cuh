// The block's part of the stable radix sort (row_groups.cu, and the gradient of small tables in
// row_tables.cu): up to kTile keys of a block of kThreads threads, in registers and shared memory.
#pragma once
#include "common.cuh"

namespace cvhrf {
namespace row_sort {

constexpr int kThreads = 1024, kWarps = kThreads / 32, kItems = 8, kTile = kThreads * kItems;
constexpr int kMaxBits = 9, kMaxRadix = 1 << kMaxBits;
constexpr uint32_t kNone = 0xffffffffu;
static_assert(kThreads == 2 * kMaxRadix, "two threads per digit");

struct Source {
  const void* index;         // the caller's indices in the first pass
  int bytes;                 // 4 or 8; 0: sorted keys and entries of the pass before
  const uint32_t* keys;
  const uint32_t* entries;
  uint32_t rows;             // values outside [0, rows) are left out, or become `rows`
  int keep;
};

// Key of item i, kNone if it is left out (keys are below 2^31).
__device__ __forceinline__ uint32_t source_key(const Source& s, uint32_t i) {
  if (s.bytes == 0) return s.keys[i];
  const unsigned long long v = s.bytes == 4 ? (unsigned long long)(long long)((const int*)s.index)[i]
                                            : ((const unsigned long long*)s.index)[i];
  return v < s.rows ? (uint32_t)v : (s.keep ? s.rows : kNone);
}

struct Shared {
  uint32_t cnt[kWarps * kMaxRadix];    // warp x digit
  uint32_t key[kTile], entry[kTile];   // the tile in digit order
  uint32_t base[kMaxRadix];            // place of the chunk's next key with this digit
  uint32_t start[kMaxRadix];           // start of the digit inside the tile
  uint32_t delta[kMaxRadix];           // base - start
  uint32_t lower[kMaxRadix], upper[kMaxRadix];   // keys of the digit in either half of the warps
  uint32_t sh[kMaxRadix / 32 + 1];
};

// Exclusive scan over the values of a block's first kMaxRadix threads; all threads call it.
__device__ __forceinline__ uint32_t scan_radix(uint32_t v, uint32_t* sh /* kMaxRadix / 32 + 1 */, uint32_t& total) {
  constexpr int kParts = kMaxRadix / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (warp < kParts && lane == 31) sh[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    uint32_t t = lane < kParts ? sh[lane] : 0u, run = t;
#pragma unroll
    for (int o = 1; o < kParts; o <<= 1) {
      const uint32_t u = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += u;
    }
    if (lane < kParts) sh[lane] = run - t;
    if (lane == kParts - 1) sh[kParts] = run;
  }
  __syncthreads();
  const uint32_t r = (warp < kParts ? sh[warp] : 0u) + inc - v;
  total = sh[kParts];
  __syncthreads();
  return r;
}

// Sorts one tile by a digit into sh.key / sh.entry.  Warp w holds the `rounds` x 32 keys from
// w * rounds * 32 on (key[r] of lane l is the r * 32 + l-th of them; kNone: no key).  place[r]
// becomes the key's place inside its digit's run.  Returns how many of digit threadIdx.x
// there are; kept = keys in the tile.
__device__ __forceinline__ uint32_t sort_tile(Shared& sh, const uint32_t (&key)[kItems], const uint32_t (&entry)[kItems],
                                              uint32_t (&place)[kItems], int rounds, int shift, int width,
                                              uint32_t& kept) {
  const int radix = 1 << width;
  const uint32_t mask = radix - 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < kWarps * radix / 4; i += kThreads) reinterpret_cast<uint4*>(sh.cnt)[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  const unsigned lt = (1u << lane) - 1u;
  uint32_t* mine = sh.cnt + warp * radix;
  // the lanes with the same digit, bit by bit (__match_any_sync takes a step per distinct digit)
  unsigned peers[kItems];
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if (r >= rounds) break;
    const uint32_t d = key[r] >> shift;
    peers[r] = __ballot_sync(0xffffffffu, key[r] != kNone);
#pragma unroll
    for (int b = 0; b < kMaxBits; ++b) {
      if (b >= width) break;
      const unsigned ones = __ballot_sync(0xffffffffu, d & (1u << b));
      peers[r] &= d & (1u << b) ? ones : ~ones;
    }
  }
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if (r >= rounds) break;
    const bool in = key[r] != kNone;
    const uint32_t d = (key[r] >> shift) & mask;
    uint32_t before = 0;
    if (in) before = mine[d];
    place[r] = before + __popc(peers[r] & lt);
    __syncwarp();
    if (in && (peers[r] & lt) == 0) mine[d] = before + __popc(peers[r]);
    __syncwarp();
  }
  __syncthreads();
  // per digit: where each warp's keys begin, the upper half of the warps by the upper threads
  constexpr int kHalf = kWarps / 2;
  const int d0 = tid & (kMaxRadix - 1), w0 = tid / kMaxRadix * kHalf;
  uint32_t run = 0;
  if (d0 < radix) {
#pragma unroll
    for (int w = 0; w < kHalf; ++w) {
      const uint32_t c = sh.cnt[(w0 + w) * radix + d0];
      sh.cnt[(w0 + w) * radix + d0] = run;
      run += c;
    }
  }
  if (tid < kMaxRadix) sh.lower[tid] = run;
  else sh.upper[tid - kMaxRadix] = run;
  __syncthreads();
  if (tid < kMaxRadix) run += sh.upper[tid];
  const uint32_t start = scan_radix(tid < kMaxRadix ? run : 0u, sh.sh, kept);
  if (tid < kMaxRadix) sh.start[tid] = start;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kItems; ++r) {
    if (r >= rounds) break;
    if (key[r] == kNone) continue;
    const uint32_t d = (key[r] >> shift) & mask;
    place[r] += mine[d] + (warp >= kHalf ? sh.lower[d] : 0u);
    const uint32_t at = sh.start[d] + place[r];
    sh.key[at] = key[r];
    sh.entry[at] = entry[r];
  }
  __syncthreads();
  return run;
}

// All passes on items begin .. begin + n (n up to kTile) of the source: sh.key / sh.entry hold the
// keys that are not left out, in order, and their items.  Returns how many.
__device__ __forceinline__ uint32_t sort_run(Shared& sh, const Source& s, uint32_t begin, uint32_t n, int bits,
                                             int passes) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t key[kItems], entry[kItems], place[kItems];
  uint32_t kept = n;
  int done = 0;
  for (int p = 0; p < passes; ++p) {
    const int width = (bits - done + (passes - p) - 1) / (passes - p);
    const int rounds = (int)((kept + kThreads - 1) / kThreads);
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      key[r] = kNone;
      if (r >= rounds) continue;
      const uint32_t i = warp * (32 * rounds) + r * 32 + lane;
      if (i < kept) {
        key[r] = p == 0 ? source_key(s, begin + i) : sh.key[i];
        entry[r] = p == 0 ? begin + i : sh.entry[i];
      }
    }
    __syncthreads();
    sort_tile(sh, key, entry, place, rounds, done, width, kept);
    done += width;
  }
  return kept;
}

inline int bits_for(unsigned long long values) {   // bits that hold 0 .. values - 1
  int b = 1;
  while ((1ull << b) < values) ++b;
  return b;
}

constexpr int passes_for(int bits) { return (bits + kMaxBits - 1) / kMaxBits; }

}  // namespace row_sort
}  // namespace cvhrf
