// Integer indices sorted stably by value (see row_groups.cuh), and cvhrf_group_rows.
//
// LSD radix sort, digits of at most 9 bits (two passes up to 262144 values), the bits shared
// evenly between the passes.  A pass is two launches: chunk_count_kernel counts the digits of
// each contiguous chunk of keys into a chunk x digit matrix, and chunk_scatter_kernel reads that
// matrix, adds up what lies before its own chunk, and writes each key to its place.  No block
// waits for another one and nothing has to be cleared beforehand.  (Counting a key's next digit
// where it is scattered saves a launch, but its atomics cost 8 us for 1M keys, and the launch 3.)
// (A look-back between tiles, as in scan_sort.cu, needs a cleared status array, one more
// launch for the histogram, and a walk over the earlier tiles in L2 latency.)
// The first pass reads the caller's indices as they are (4 or 8 bytes).
//
// Bound by latency and by the instructions around the keys: one block of 1024 threads per SM
// takes a chunk of up to 8192 keys in registers, so a pass is a handful of dependent steps
// (512 threads: 18 us a pass for 1M keys, against 15).  Up to 8192 keys in all, one block
// does every pass in shared memory (small_sort_kernel, one launch).
#include "row_groups.cuh"
#include "row_sort.cuh"
#include "row_types.cuh"

namespace cvhrf {
namespace {

using namespace row_sort;

constexpr int kMaxChunks = 148;   // one block per SM

struct Target {
  uint32_t* keys;      // null: not wanted
  uint32_t* entries;
  int* slots;          // cvhrf_group_rows: the place of each entry, -1 behind the last group
  int* offsets;        // ... and where each of the `groups` groups begins, and the last one ends
  int groups;
  uint32_t* count;     // number of sorted items
  uint8_t* touched;    // 1 for every key
};

// Zeros into `touched` before the passes set its ones.
__device__ __forceinline__ void clear_touched(uint8_t* touched, uint32_t rows) {
  if (!touched) return;
  const uint32_t head = min((uint32_t)(-(long long)(uintptr_t)touched & 15), rows), words = (rows - head) >> 4;
  uint4* w = reinterpret_cast<uint4*>(touched + head);
  for (uint32_t i = blockIdx.x * kThreads + threadIdx.x; i < words; i += gridDim.x * kThreads)
    w[i] = make_uint4(0u, 0u, 0u, 0u);
  if (blockIdx.x == 0) {
    if (threadIdx.x < head) touched[threadIdx.x] = 0;
    for (uint32_t i = head + (words << 4) + threadIdx.x; i < rows; i += kThreads) touched[i] = 0;
  }
}

// counts[chunk][digit] over the keys of each chunk.
__global__ void __launch_bounds__(kThreads) chunk_count_kernel(Source s, uint32_t n, const uint32_t* n_dev,
                                                               uint32_t chunk, int shift, int radix,
                                                               uint32_t* __restrict__ counts,
                                                               uint8_t* __restrict__ clear) {
  follow();
  let_next_start();
  constexpr int kCopies = 8;   // histograms, so that equal digits of different warps do not meet
  __shared__ uint32_t h[kCopies][kMaxRadix];
  clear_touched(clear, s.rows);
  if (n_dev) n = min(n, *n_dev);
  for (int i = threadIdx.x; i < kCopies * kMaxRadix; i += kThreads) (&h[0][0])[i] = 0;
  __syncthreads();
  const uint32_t begin = min(n, blockIdx.x * chunk), end = min(n, begin + chunk);
  uint32_t* mine = h[(threadIdx.x >> 5) % kCopies];
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    uint32_t key[kItems];
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      key[r] = kNone;
      if (tile + r * kThreads >= end) continue;
      const uint32_t i = tile + r * kThreads + threadIdx.x;
      if (i < end) key[r] = source_key(s, i);
    }
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      if (tile + r * kThreads >= end) break;
      if (key[r] != kNone) atomicAdd(&mine[(key[r] >> shift) & (radix - 1)], 1u);
    }
  }
  __syncthreads();
  for (int d = threadIdx.x; d < radix; d += kThreads) {
    uint32_t c = 0;
#pragma unroll
    for (int w = 0; w < kCopies; ++w) c += h[w][d];
    counts[(size_t)blockIdx.x * radix + d] = c;
  }
}

__global__ void __launch_bounds__(kThreads) chunk_scatter_kernel(Source s, uint32_t n,
                                                                 const uint32_t* n_dev, uint32_t chunk, int shift,
                                                                 int radix, const uint32_t* counts, Target out) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  follow();
  let_next_start();
  const int chunks = gridDim.x;
  if (n_dev) n = min(n, *n_dev);
  const uint32_t begin = min(n, blockIdx.x * chunk), end = min(n, begin + chunk);
  const uint32_t mask = radix - 1;
  uint32_t key[kItems], entry[kItems], place[kItems];
  int rounds = 0;
  auto load = [&](uint32_t tile) {
    const uint32_t len = min(end - tile, (uint32_t)kTile);
    rounds = (int)((len + kThreads - 1) / kThreads);   // equal runs for the warps
    const uint32_t base = tile + warp * (32 * rounds) + lane;
#pragma unroll
    for (int r = 0; r < kItems; ++r) {
      key[r] = kNone;
      if (r >= rounds) continue;
      const uint32_t i = base + r * 32;
      if (i < end) {
        key[r] = source_key(s, i);
        entry[r] = s.bytes ? i : s.entries[i];
      }
    }
  };
  if (begin < end) load(begin);   // on its way while the matrix of counts is added up
  // the matrix of counts: four digits per thread, the chunks shared between the threads
  {
    const int quads = radix >> 2, shares = min(kThreads / quads, 16), share = tid / quads, q = tid - share * quads;
    uint4 before4 = make_uint4(0, 0, 0, 0), all4 = before4;
    constexpr int kLoads = 10;   // in flight: all of them up to 256 digits
    for (int c0 = share; share < shares && c0 < chunks; c0 += kLoads * shares) {
      uint4 v[kLoads];
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int c = c0 + i * shares;
        v[i] = c < chunks ? reinterpret_cast<const uint4*>(counts)[(size_t)c * quads + q] : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        all4.x += v[i].x, all4.y += v[i].y, all4.z += v[i].z, all4.w += v[i].w;
        if (c0 + i * shares < (int)blockIdx.x)
          before4.x += v[i].x, before4.y += v[i].y, before4.z += v[i].z, before4.w += v[i].w;
      }
    }
    if (share < shares) {
      reinterpret_cast<uint4*>(sh.key)[tid] = before4;   // shares x radix
      reinterpret_cast<uint4*>(sh.entry)[tid] = all4;
    }
    __syncthreads();
    uint32_t before = 0, all = 0;
    if (tid < radix) {
#pragma unroll 8
      for (int i = 0; i < shares; ++i) before += sh.key[i * radix + tid], all += sh.entry[i * radix + tid];
    }
    uint32_t total;
    const uint32_t first = scan_radix(all, sh.sh, total);
    if (tid < kMaxRadix) sh.base[tid] = first + before;
    if (blockIdx.x == 0 && tid == 0 && out.count) *out.count = total;
    if (blockIdx.x == 0 && out.offsets) {
      if (tid < out.groups) out.offsets[tid] = (int)first;
      if (tid == out.groups - 1) out.offsets[out.groups] = (int)(first + all);
    }
  }
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    if (tile != begin) load(tile);
    uint32_t kept;
    const uint32_t run = sort_tile(sh, key, entry, place, rounds, shift, 31 - __clz(radix), kept);
    if (out.slots) {   // first and only pass: the entries are the items in order
#pragma unroll
      for (int r = 0; r < kItems; ++r)
        if (r < rounds && key[r] != kNone)
          out.slots[entry[r]] =
              key[r] < (uint32_t)out.groups ? (int)(sh.base[(key[r] >> shift) & mask] + place[r]) : -1;
    }
    // the tile is in digit order: each digit's keys go out as one run
    if (tid < kMaxRadix) sh.delta[tid] = sh.base[tid] - sh.start[tid];
    __syncthreads();
    for (uint32_t i = tid; i < kept; i += kThreads) {
      const uint32_t k = sh.key[i], d = (k >> shift) & mask;
      const uint32_t at = sh.delta[d] + i;
      if (out.keys) out.keys[at] = k;
      out.entries[at] = sh.entry[i];
      // (the tile is in order of the whole key by the last pass)
      if (out.touched && (i == 0 || sh.key[i - 1] != k)) out.touched[k] = 1;
    }
    __syncthreads();
    if (tid < kMaxRadix) sh.base[tid] += run;
    __syncthreads();
  }
}

// All passes on up to kTile keys, in one block.
__global__ void __launch_bounds__(kThreads) small_sort_kernel(Source s, uint32_t n, int bits, int passes, Target out,
                                                              bool clear) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int tid = threadIdx.x;
  let_next_start();
  if (clear) clear_touched(out.touched, s.rows);
  const uint32_t kept = sort_run(sh, s, 0, n, bits, passes);
  for (uint32_t i = tid; i < kept; i += kThreads) {
    const uint32_t k = sh.key[i], e = sh.entry[i];
    if (out.keys) out.keys[i] = k;
    out.entries[i] = e;
    if (out.slots) out.slots[e] = k < (uint32_t)out.groups ? (int)i : -1;
    if (out.touched && (i == 0 || sh.key[i - 1] != k)) out.touched[k] = 1;
  }
  if (tid == 0 && out.count) *out.count = kept;
  if (out.offsets) {
    for (long long g = tid; g <= out.groups; g += kThreads) {   // the first key of group g or a later one
      uint32_t lo = 0, hi = kept;
      while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if (sh.key[mid] < (uint32_t)g) lo = mid + 1;
        else hi = mid;
      }
      out.offsets[g] = (int)lo;
    }
  }
}

// The places of the entries and the beginnings of the groups from the sorted keys (more groups than one pass sorts).
__global__ void __launch_bounds__(256) places_kernel(const uint32_t* keys, const uint32_t* entries, uint32_t n,
                                                     int groups, int* __restrict__ order, int* __restrict__ slots,
                                                     int* __restrict__ offsets) {
  follow();
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

// The beginnings of many groups for few entries, from their order alone: in small_sort_kernel one
// block looks for all of them (5000 entries: 23 us in all at 8192 groups, 23 with this launch
// beside; at 65536 groups 60 and 25).
constexpr int kBlockGroups = 1 << 13;   // most that small_sort_kernel writes itself
__global__ void __launch_bounds__(256) offsets_kernel(Source s, const uint32_t* order, uint32_t n, int groups,
                                                      int* __restrict__ offsets) {
  follow();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i > groups) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = (lo + hi) >> 1;
    if (source_key(s, order[mid]) < (uint32_t)i) lo = mid + 1;
    else hi = mid;
  }
  offsets[i] = (int)lo;
}

struct Chunks {
  int count;
  uint32_t size;
};

inline Chunks chunks_for(long long n) {
  // a chunk has a key per thread at least
  long long c = (n + kThreads - 1) / kThreads;
  if (c > kMaxChunks) c = kMaxChunks;
  if (c < 1) c = 1;
  const long long size = ((n + c - 1) / c + 31) / 32 * 32;
  return {(int)((n + size - 1) / (size > 0 ? size : 1)), (uint32_t)size};
}

// All passes over the low `bits` bits.  The last one writes `out`; the ones before it go to and
// fro between the two buffers of keys and entries at `buffers` (of `len` words each).
int sort_chunks(Source src, long long n, int bits, uint32_t* counts, uint32_t* buffers, size_t len, uint32_t* count,
                Target out, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed{0};
  CVHRF_CUDA_TRY(allow_shared(chunk_scatter_kernel, sizeof(Shared), allowed));
  const Chunks c = chunks_for(n);
  const int passes = passes_for(bits);
  int shift = 0;
  for (int p = 0; p < passes; ++p) {
    int width = (bits - shift + (passes - p) - 1) / (passes - p);   // the bits left, shared evenly
    if (width < 2) width = 2;   // the counts are read four digits at a time
    uint32_t* to = buffers + (p & 1) * 2 * len;
    Target t = out;
    if (p + 1 < passes) t = Target{to, to + len, nullptr, nullptr, 0, nullptr, nullptr};
    t.count = p == 0 ? count : nullptr;
    const uint32_t* n_dev = p == 0 ? nullptr : count;
    if (p == 0) {
      chunk_count_kernel<<<c.count, kThreads, 0, st>>>(src, (uint32_t)n, n_dev, c.size, shift, 1 << width, counts,
                                                       out.touched);
      CVHRF_LAUNCH_CHECK();
    } else {
      CVHRF_CUDA_TRY(launch_after(chunk_count_kernel, dim3(c.count), kThreads, 0, st, src, (uint32_t)n, n_dev, c.size,
                                  shift, 1 << width, counts, nullptr));
      count_launch(1);
    }
    CVHRF_CUDA_TRY(launch_after(chunk_scatter_kernel, dim3(c.count), kThreads, sizeof(Shared), st, src, (uint32_t)n,
                                n_dev, c.size, shift, 1 << width, counts, t));
    count_launch(1);
    src = Source{nullptr, 0, to, to + len, src.rows, 1};
    shift += width;
  }
  return CVHRF_OK;
}

int small_sort(const Source& src, long long n, int bits, Target out, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed{0};
  CVHRF_CUDA_TRY(allow_shared(small_sort_kernel, sizeof(Shared), allowed));
  const bool clear = src.rows <= 1u << 20;   // more marks than the one block clears in a few microseconds
  if (out.touched && !clear) CVHRF_CUDA_TRY(cudaMemsetAsync(out.touched, 0, src.rows, st));
  small_sort_kernel<<<1, kThreads, sizeof(Shared), st>>>(src, (uint32_t)n, bits, passes_for(bits), out, clear);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

}  // namespace

// scratch: count (64 words), the matrix of counts, two buffers of keys and entries (up to kTile
// keys the result alone)
constexpr size_t kCountWords = (size_t)kMaxChunks * kMaxRadix;
size_t group_sort_words(long long n) {
  const size_t len = align_up((size_t)n, 64);
  return n <= kTile ? 64 + 2 * len : 64 + kCountWords + 4 * len;
}

int group_sort(const void* index, int index_bytes, long long n, long long rows, bool keep_outside, uint32_t* scratch,
               uint8_t* touched, cudaStream_t st, const uint32_t** keys, const uint32_t** entries,
               const uint32_t** count_dev) {
  uint32_t* count = scratch;
  *count_dev = count;
  const size_t len = align_up((size_t)n, 64);
  const int bits = bits_for((unsigned long long)rows + (keep_outside ? 1 : 0));
  const Source src{index, index_bytes, nullptr, nullptr, (uint32_t)rows, keep_outside ? 1 : 0};
  uint32_t* buffers = scratch + 64 + (n <= kTile ? 0 : kCountWords);
  uint32_t* to = buffers + (n <= kTile ? 0 : ((passes_for(bits) - 1) & 1) * 2 * len);
  *keys = to;
  *entries = to + len;
  const Target out{to, to + len, nullptr, nullptr, 0, count, touched};
  if (n <= kTile) return small_sort(src, n, bits, out, st);
  return sort_chunks(src, n, bits, scratch + 64, buffers, len, count, out, st);
}

}  // namespace cvhrf

using namespace cvhrf;

extern "C" size_t cvhrf_group_rows_workspace_bytes(long long entries, int groups) {
  if (entries <= kTile || entries > kGroupMaxEntries || groups < 1) return 0;   // a small sort needs none
  return group_sort_words(entries) * sizeof(uint32_t);
}

extern "C" int cvhrf_group_rows(const cvhrf_group_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const auto [index, order, slots, offsets, workspace, workspace_bytes, entries, groups, index_bytes] = *args;
  if (entries < 0 || groups < 1 || groups > 0x7ffffffe || (index_bytes != 4 && index_bytes != 8) || !offsets)
    return CVHRF_EINVAL;
  if (entries > 0 && (!index || !order || !slots)) return CVHRF_EINVAL;
  if (entries > kGroupMaxEntries) return CVHRF_EUNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  if (entries == 0) {
    CVHRF_CUDA_TRY(cudaMemsetAsync(offsets, 0, ((size_t)groups + 1) * sizeof(int), st));
    return CVHRF_OK;
  }
  const size_t need = cvhrf_group_rows_workspace_bytes(entries, groups);
  if (need && (!workspace || workspace_bytes < need)) return CVHRF_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return CVHRF_EINVAL;
  uint32_t* scratch = (uint32_t*)workspace;
  const Source src{index, index_bytes, nullptr, nullptr, (uint32_t)groups, 1};
  const Target out{nullptr, (uint32_t*)order, slots, offsets, groups, nullptr, nullptr};
  const int bits = bits_for((unsigned long long)groups + 1);
  if (entries <= kTile && groups <= kBlockGroups) return small_sort(src, entries, bits, out, st);
  if (entries <= kTile) {
    Target rest = out;
    rest.offsets = nullptr;
    const int rc = small_sort(src, entries, bits, rest, st);
    if (rc) return rc;
    CVHRF_CUDA_TRY(launch_after(offsets_kernel, dim3((unsigned)((groups + 256ll) / 256)), 256, 0, st, src,
                                (const uint32_t*)order, (uint32_t)entries, groups, offsets));
    count_launch(1);
    return CVHRF_OK;
  }
  // up to 511 groups (and the entries left out) one pass writes everything
  if (groups < kMaxRadix) return sort_chunks(src, entries, bits, scratch + 64, nullptr, 0, scratch, out, st);
  const uint32_t *keys, *sorted, *count;
  const int rc = group_sort(index, index_bytes, entries, groups, true, scratch, nullptr, st, &keys, &sorted, &count);
  if (rc) return rc;
  const long long most = entries > (long long)groups + 1 ? entries : (long long)groups + 1;
  CVHRF_CUDA_TRY(launch_after(places_kernel, dim3((unsigned)((most + 255) / 256)), 256, 0, st, keys, sorted,
                              (uint32_t)entries, groups, order, slots, offsets));
  count_launch(1);
  return CVHRF_OK;
}
