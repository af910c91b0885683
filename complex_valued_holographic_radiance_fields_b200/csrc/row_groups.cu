// Integer indices sorted stably by value (see row_groups.cuh), and cvhrf_group_rows.
//
// LSD radix sort, digits of at most 8 bits, the bits shared evenly between the passes.  A
// pass is two launches: chunk_count_kernel counts the digits of each contiguous chunk of
// keys into a chunk x digit matrix, and chunk_scatter_kernel reads that matrix, adds up
// what lies before its own chunk, and writes each key to its place.  No block waits for
// another one and nothing has to be cleared beforehand, so a sort is 2 launches per pass.
// (A look-back between tiles, as in scan_sort.cu, needs a cleared status array, one more
// launch for the histogram, and a walk over the earlier tiles in L2 latency.)
// The first pass reads the caller's indices as they are (4 or 8 bytes).
#include "row_groups.cuh"

namespace cvhrf {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32, kItems = 4, kTile = kThreads * kItems;
constexpr int kMaxChunks = 296;   // two blocks per SM
constexpr int kMaxRadix = 256;

struct Source {
  const void* index;         // the caller's indices in the first pass
  int bytes;                 // 4 or 8; 0: sorted keys and entries of the pass before
  const uint32_t* keys;
  const uint32_t* entries;
  uint32_t rows;             // values outside [0, rows) are left out, or become `rows`
  int keep;
};

// Key of item i; false if it is left out.
__device__ __forceinline__ bool source_key(const Source& s, uint32_t i, uint32_t& key) {
  if (s.bytes == 0) {
    key = s.keys[i];
    return true;
  }
  const unsigned long long v = s.bytes == 4 ? (unsigned long long)(long long)((const int*)s.index)[i]
                                            : ((const unsigned long long*)s.index)[i];
  const bool inside = v < s.rows;
  key = inside ? (uint32_t)v : s.rows;
  return inside || s.keep;
}

// counts[chunk][digit] over the keys of each chunk.
__global__ void __launch_bounds__(kThreads) chunk_count_kernel(Source s, uint32_t n, const uint32_t* __restrict__ n_dev,
                                                               uint32_t chunk, int shift, int radix,
                                                               uint32_t* __restrict__ counts) {
  __shared__ uint32_t h[kWarps][kMaxRadix];
  if (n_dev) n = min(n, *n_dev);
  for (int i = threadIdx.x; i < kWarps * kMaxRadix; i += kThreads) (&h[0][0])[i] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t begin = min(n, blockIdx.x * chunk), end = min(n, begin + chunk);
  const uint32_t mask = radix - 1;
  for (uint32_t base = begin + warp * 32; base < end; base += kThreads) {
    uint32_t key, d = 0xffffffffu;
    if (base + lane < end && source_key(s, base + lane, key)) d = (key >> shift) & mask;
    // one add per distinct digit of the warp: few groups would otherwise add to one word 32 times
    const unsigned peers = __match_any_sync(0xffffffffu, d);
    if (d != 0xffffffffu && (peers & ((1u << lane) - 1u)) == 0) h[warp][d] += __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kThreads) {
    uint32_t c = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) c += h[w][d];
    counts[(size_t)blockIdx.x * radix + d] = c;
  }
}

// Exclusive scan over the 256 values of a block's first 256 threads; all threads call it.
__device__ __forceinline__ uint32_t scan_256(uint32_t v, uint32_t* sh /* 9 */, uint32_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (warp < 8 && lane == 31) sh[warp] = inc;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t run = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint32_t t = sh[w];
      sh[w] = run;
      run += t;
    }
    sh[8] = run;
  }
  __syncthreads();
  const uint32_t r = (warp < 8 ? sh[warp] : 0u) + inc - v;
  total = sh[8];
  __syncthreads();
  return r;
}

struct Target {
  uint32_t* keys;      // null: not wanted
  uint32_t* entries;
  int* slots;          // cvhrf_group_rows in one pass: the place of each entry, -1 behind the last group
  int* offsets;        // ... and where each of the `groups` groups begins, and the last one ends
  int groups;
  uint32_t* count;     // number of sorted items
};

__global__ void __launch_bounds__(kThreads) chunk_scatter_kernel(Source s, uint32_t n,
                                                                 const uint32_t* __restrict__ n_dev, uint32_t chunk,
                                                                 int shift, int radix,
                                                                 const uint32_t* __restrict__ counts, Target out) {
  __shared__ uint32_t s_cnt[kWarps][kMaxRadix];
  __shared__ uint32_t s_base[kMaxRadix];    // place of the chunk's next key with this digit
  __shared__ uint32_t s_start[kMaxRadix];   // start of the digit inside the tile
  __shared__ uint32_t s_key[kTile], s_entry[kTile];
  __shared__ uint32_t sh[9];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (n_dev) n = min(n, *n_dev);
  // the matrix of counts: threads d and d + 256 add the even and the odd chunks of digit d
  {
    uint32_t before = 0, all = 0;
    const int d = tid & 255;
    if (d < radix) {
#pragma unroll 8
      for (int c = tid >> 8; c < (int)gridDim.x; c += 2) {
        const uint32_t v = counts[(size_t)c * radix + d];
        all += v;
        before += c < (int)blockIdx.x ? v : 0u;
      }
    }
    if (tid >= 256) s_cnt[0][d] = before, s_cnt[1][d] = all;
    __syncthreads();
    if (tid < 256) before += s_cnt[0][d], all += s_cnt[1][d];
    uint32_t total;
    const uint32_t first = scan_256(tid < 256 ? all : 0u, sh, total);
    if (tid < 256) s_base[d] = first + before;
    if (blockIdx.x == 0 && tid == 0 && out.count) *out.count = total;
    if (blockIdx.x == 0 && out.offsets) {
      if (tid < 256 && tid < out.groups) out.offsets[tid] = (int)first;
      if (tid == out.groups - 1) out.offsets[out.groups] = (int)(first + all);
    }
  }
  const uint32_t begin = min(n, blockIdx.x * chunk), end = min(n, begin + chunk);
  const uint32_t mask = radix - 1;
  const unsigned lt = (1u << lane) - 1u;
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    for (int i = tid; i < kWarps * kMaxRadix; i += kThreads) (&s_cnt[0][0])[i] = 0;
    __syncthreads();
    // stable ranks inside the warp's run of 32 * kItems keys
    const uint32_t base = tile + warp * (32 * kItems);
    uint32_t key[kItems], rank[kItems], digit[kItems];
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const uint32_t i = base + r * 32 + lane;
      uint32_t k = 0;
      const bool in = i < end && source_key(s, i, k);
      key[r] = k;
      digit[r] = in ? (k >> shift) & mask : 0xffffffffu;
    }
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const unsigned peers = __match_any_sync(0xffffffffu, digit[r]);
      const bool in = digit[r] != 0xffffffffu;
      uint32_t before = 0;
      if (in) before = s_cnt[warp][digit[r]];
      rank[r] = before + __popc(peers & lt);
      __syncwarp();
      if (in && (peers & lt) == 0) s_cnt[warp][digit[r]] = before + __popc(peers);
      __syncwarp();
    }
    __syncthreads();
    // per digit: where each warp's keys begin, then where the digit begins in the tile
    uint32_t run = 0;
    if (tid < 256) {
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t c = s_cnt[w][tid];
        s_cnt[w][tid] = run;
        run += c;
      }
    }
    uint32_t kept;
    const uint32_t start = scan_256(run, sh, kept);
    if (tid < 256) s_start[tid] = start;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      const uint32_t i = base + r * 32 + lane, d = digit[r];
      if (d == 0xffffffffu) continue;
      const uint32_t local = s_cnt[warp][d] + rank[r];
      const uint32_t e = s.bytes ? i : s.entries[i];
      s_key[s_start[d] + local] = key[r];
      s_entry[s_start[d] + local] = e;
      if (out.slots) out.slots[i] = key[r] < (uint32_t)out.groups ? (int)(s_base[d] + local) : -1;
    }
    __syncthreads();
    // the tile is in digit order: each digit's keys go out as one run
    for (uint32_t i = tid; i < kept; i += kThreads) {
      const uint32_t k = s_key[i], d = (k >> shift) & mask;
      const uint32_t at = s_base[d] + i - s_start[d];
      if (out.keys) out.keys[at] = k;
      out.entries[at] = s_entry[i];
    }
    __syncthreads();
    if (tid < 256) s_base[tid] += run;
    __syncthreads();
  }
}

// The places of the entries and the beginnings of the groups from the sorted keys (more than 255 groups).
__global__ void __launch_bounds__(256) places_kernel(const uint32_t* __restrict__ keys,
                                                     const uint32_t* __restrict__ entries, uint32_t n, int groups,
                                                     int* __restrict__ order, int* __restrict__ slots,
                                                     int* __restrict__ offsets) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) {
    const uint32_t e = entries[i];
    order[i] = (int)e;
    slots[e] = keys[i] < (uint32_t)groups ? (int)i : -1;
  }
  if (i <= groups) {
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (keys[mid] < (uint32_t)i) lo = mid + 1;
      else hi = mid;
    }
    offsets[i] = (int)lo;
  }
}

inline int bits_for(unsigned long long values) {   // bits that hold 0 .. values - 1
  int b = 1;
  while ((1ull << b) < values) ++b;
  return b;
}

struct Chunks {
  int count;
  uint32_t size;
};

inline Chunks chunks_for(long long n) {
  // a chunk has 1024 keys at least (two per thread), so small sorts stay on few blocks
  long long c = (n + 1023) / 1024;
  if (c > kMaxChunks) c = kMaxChunks;
  if (c < 1) c = 1;
  const long long size = ((n + c - 1) / c + 31) / 32 * 32;
  return {(int)((n + size - 1) / (size > 0 ? size : 1)), (uint32_t)size};
}

int one_pass(const Source& src, long long n, const uint32_t* n_dev, int shift, int bits, uint32_t* counts, Target out,
             cudaStream_t st) {
  const Chunks c = chunks_for(n);
  chunk_count_kernel<<<c.count, kThreads, 0, st>>>(src, (uint32_t)n, n_dev, c.size, shift, 1 << bits, counts);
  CVHRF_LAUNCH_CHECK();
  chunk_scatter_kernel<<<c.count, kThreads, 0, st>>>(src, (uint32_t)n, n_dev, c.size, shift, 1 << bits, counts, out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

}  // namespace

// scratch: count (64 words), counts matrix, two buffers of keys and entries
size_t group_sort_words(long long n) { return 64 + (size_t)kMaxChunks * kMaxRadix + 4 * (align_up((size_t)n, 64)); }

int group_sort(const void* index, int index_bytes, long long n, long long rows, bool keep_outside, uint32_t* scratch,
               cudaStream_t st, const uint32_t** keys, const uint32_t** entries, const uint32_t** count_dev) {
  uint32_t* count = scratch;
  uint32_t* counts = scratch + 64;
  const size_t len = align_up((size_t)n, 64);
  uint32_t* k[2] = {counts + (size_t)kMaxChunks * kMaxRadix, nullptr};
  k[1] = k[0] + 2 * len;
  const int bits = bits_for((unsigned long long)rows + (keep_outside ? 1 : 0));
  const int npass = (bits + 7) / 8;
  Source src{index, index_bytes, nullptr, nullptr, (uint32_t)rows, keep_outside ? 1 : 0};
  int done = 0;
  for (int p = 0; p < npass; ++p) {
    const int width = (bits - done + (npass - p) - 1) / (npass - p);   // the bits left, shared evenly
    uint32_t* to = k[p & 1];
    Target out{to, to + len, nullptr, nullptr, 0, p == 0 ? count : nullptr};
    const int rc = one_pass(src, n, p == 0 ? nullptr : count, done, width, counts, out, st);
    if (rc) return rc;
    src = Source{nullptr, 0, to, to + len, (uint32_t)rows, 1};
    done += width;
  }
  *keys = src.keys;
  *entries = src.entries;
  *count_dev = count;
  return CVHRF_OK;
}

}  // namespace cvhrf

using namespace cvhrf;

extern "C" size_t cvhrf_group_rows_workspace_bytes(long long entries, int groups) {
  if (entries < 0 || entries > kGroupMaxEntries || groups < 1) return 0;
  return group_sort_words(entries) * sizeof(uint32_t);
}

extern "C" int cvhrf_group_rows(const void* index, int index_bytes, long long entries, int groups, int* order,
                                int* slots, int* offsets, void* workspace, size_t workspace_bytes, void* stream) {
  if (entries < 0 || groups < 1 || groups > 0x7ffffffe || (index_bytes != 4 && index_bytes != 8) || !offsets)
    return CVHRF_EINVAL;
  if (entries > 0 && (!index || !order || !slots)) return CVHRF_EINVAL;
  if (entries > kGroupMaxEntries) return CVHRF_EUNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  if (entries == 0) {
    CVHRF_CUDA_TRY(cudaMemsetAsync(offsets, 0, ((size_t)groups + 1) * sizeof(int), st));
    return CVHRF_OK;
  }
  if (!workspace || workspace_bytes < cvhrf_group_rows_workspace_bytes(entries, groups)) return CVHRF_EWORKSPACE;
  uint32_t* scratch = (uint32_t*)workspace;
  if (groups < kMaxRadix) {   // one pass writes everything
    const Source src{index, index_bytes, nullptr, nullptr, (uint32_t)groups, 1};
    const Target out{nullptr, (uint32_t*)order, slots, offsets, groups, nullptr};
    return one_pass(src, entries, nullptr, 0, bits_for((unsigned long long)groups + 1), scratch + 64, out, st);
  }
  const uint32_t *keys, *sorted, *count;
  const int rc = group_sort(index, index_bytes, entries, groups, true, scratch, st, &keys, &sorted, &count);
  if (rc) return rc;
  const long long most = entries > (long long)groups + 1 ? entries : (long long)groups + 1;
  places_kernel<<<(unsigned)((most + 255) / 256), 256, 0, st>>>(keys, sorted, (uint32_t)entries, groups, order, slots,
                                                               offsets);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}
