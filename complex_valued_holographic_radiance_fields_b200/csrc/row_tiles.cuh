// Rows that do not begin on 16 bytes (an odd width, a slice), gathered into tiles.
//
// Whatever reads rows here writes contiguous ones, so a block puts a run of output rows together
// in shared memory, one element per lane and load (never an element outside a row, whatever its
// alignment), and sends the run, which begins on 16 bytes and is whole lines, with one bulk
// copy.  Written by the lanes themselves, rows that begin anywhere send two requests per store,
// and what is done per row outweighed its words: 63 us against 56 for 1M rows of 59 floats (at
// 4.5 TB/s; L1 68 % busy, DRAM 45 %).  Addresses are worked out by one lane per row and shuffled.
#pragma once
#include <type_traits>
#include "row_types.cuh"

namespace cvhrf {

constexpr int kTileThreads = 256, kTileWarps = kTileThreads / 32;
constexpr int kTileBytes = 32 * 1024;   // of a block's run of rows
constexpr int kTileRowBytes = kTileBytes / kTileWarps;   // widest row: one per warp

// Rows of a tile: a multiple of the warps (so of 16 bytes), 32 per warp at most, and fewer where
// that would leave SMs without work.
inline int tile_rows(long long rows, int width, size_t elem) {
  long long per_warp = kTileBytes / ((long long)width * (long long)elem) / kTileWarps;
  const long long even = rows / (148ll * 6 * kTileWarps);
  if (per_warp > even) per_warp = even;
  per_warp = per_warp < 1 ? 1 : per_warp > 32 ? 32 : per_warp;
  if (per_warp > 4) per_warp = per_warp / 4 * 4;
  return (int)per_warp * kTileWarps;
}
inline bool tile_fits(int width, size_t elem, const void* out) {
  return (size_t)width * elem <= kTileRowBytes && ((uintptr_t)out & 15) == 0;
}

__device__ __forceinline__ unsigned long long shuffle(unsigned long long v, int lane) {
  return (unsigned long long)__shfl_sync(0xffffffffu, (uint32_t)(v >> 32), lane) << 32 |
         __shfl_sync(0xffffffffu, (uint32_t)v, lane);
}

// Sends the first n rows of the tile to out (16-byte aligned); the whole block calls it.
template <typename T>
__device__ __forceinline__ void send_tile(const T* tile, int n, int width, T* out) {
  fence_proxy_async_smem();
  __syncthreads();
  const int total = n * width, whole = total / (16 / (int)sizeof(T)) * (16 / (int)sizeof(T));
  if (threadIdx.x == 0 && whole > 0) bulk_copy_s2g(out, tile, whole * (int)sizeof(T));
  for (int i = whole + threadIdx.x; i < total; i += kTileThreads) out[i] = tile[i];
  if (threadIdx.x == 0) bulk_copy_wait();
}

// What entries without a row read.
static __device__ uint4 g_zero_row[kTileRowBytes / 16];

// ROWS rows into the tile, J elements of each per lane and step; a lane's first elements are at
// from[q] and `to`.  WIDE: rows of more than 32 J elements.
template <typename T, bool SCALE, bool WIDE, int ROWS, int J>
__device__ __forceinline__ void rows_to_tile(const T* (&from)[ROWS], T* to, int width, int left, float scale) {
  // left: elements of the row from the lane's first one on
#pragma unroll 1
  for (int c = 0;; c += 32 * J) {
    T v[ROWS][J];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (32 * j < left) v[q][j] = from[q][32 * j];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (32 * j < left) to[q * width + 32 * j] = SCALE ? from_float<T>(scale * to_float(v[q][j])) : v[q][j];
    if (!WIDE || c + 32 * J >= width) break;
    left -= 32 * J;
    to += 32 * J;
#pragma unroll
    for (int q = 0; q < ROWS; ++q) from[q] += 32 * J;
  }
}

// The same for 16-bit elements by pairs: words of the row that is read, stored as they are or in
// two halves where the tile has them on the other side of a word.
template <typename T, bool SCALE, bool WIDE, int ROWS, int J>
__device__ __forceinline__ void pairs_to_tile(const T* (&from)[ROWS], T* to, int width, int lane, float scale) {
  static_assert(sizeof(T) == 2);
  struct alignas(4) Two { T a, b; };
  int head[ROWS], words[ROWS];   // elements before the first whole word, whole words
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    head[q] = (int)((uintptr_t)from[q] >> 1) & 1;
    words[q] = (width - head[q]) >> 1;
  }
#pragma unroll 1
  for (int c = lane;; c += 32 * J) {
    Two v[ROWS][J];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (c + 32 * j < words[q]) v[q][j] = reinterpret_cast<const Two*>(from[q] + head[q])[c + 32 * j];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      T* d = to + q * width + head[q] + 2 * c;
      const bool whole = ((uintptr_t)d & 2) == 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (c + 32 * j < words[q]) {
          Two o = v[q][j];
          if (SCALE) o = {from_float<T>(scale * to_float(o.a)), from_float<T>(scale * to_float(o.b))};
          if (whole) *reinterpret_cast<Two*>(d + 64 * j) = o;
          else d[64 * j] = o.a, d[64 * j + 1] = o.b;
        }
    }
    if (!WIDE || (c - lane + 32 * J) * 2 >= width) break;
  }
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    const int e = lane == 0 && head[q] ? 0 : lane == 1 && ((width - head[q]) & 1) ? width - 1 : -1;
    if (e >= 0) to[q * width + e] = SCALE ? from_float<T>(scale * to_float(from[q][e])) : from[q][e];
  }
}

// out[i] = scale * (the row get(i), null: zeros), SCALE; else the row bit for bit.  A lane has
// ROWS x J elements (PAIRS: pairs) in flight.
template <typename T, bool SCALE, bool PAIRS, bool WIDE, int ROWS, int J, typename Get>
__device__ __forceinline__ void gather_tile(const Get& get, long long rows, int tile, int width, float scale,
                                            T* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char raw[];
  T* buf = reinterpret_cast<T*>(raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = tile / kTileWarps;
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, rows - first), r0 = warp * each;
  const T* row = nullptr;
  if (lane < each && r0 + lane < n) row = get(first + r0 + lane);
  const unsigned long long mine = (unsigned long long)(uintptr_t)(row ? row : reinterpret_cast<const T*>(g_zero_row));
  T* to = buf + r0 * width + (PAIRS ? 0 : lane);
  auto copy = [&](auto count, int r) {
    constexpr int kCount = decltype(count)::value;
    const T* from[kCount];
#pragma unroll
    for (int q = 0; q < kCount; ++q)
      from[q] = reinterpret_cast<const T*>((uintptr_t)shuffle(mine, r + q)) + (PAIRS ? 0 : lane);
    if constexpr (PAIRS) pairs_to_tile<T, SCALE, WIDE, kCount, J>(from, to, width, lane, scale);
    else rows_to_tile<T, SCALE, WIDE, kCount, J>(from, to, width, width - lane, scale);
    to += kCount * width;
  };
  int r = 0;
  for (; r + ROWS <= each; r += ROWS) copy(std::integral_constant<int, ROWS>(), r);
  for (; ROWS > 1 && r < each; ++r) copy(std::integral_constant<int, 1>(), r);
  send_tile(buf, n, width, out + first * width);
}

// Calls f<PAIRS, WIDE, ROWS, J> for rows of `width` elements: J shares the row evenly between
// the lanes' steps (333 elements in two steps of 6, not of 8 and 3), narrow rows go several at
// a time.
template <int A, int B, int C, int D>
struct Shape4 {
  static constexpr bool kPairs = A, kWide = B;
  static constexpr int kRows = C, kJ = D;
};
template <typename T, typename F>
int with_shape(int width, F f) {
  if constexpr (sizeof(T) == 2) {
    if (width >= 64) {
      const int words = (width + 1) / 2, steps = (words + 255) / 256, j = (words + 32 * steps - 1) / (32 * steps);
      if (steps > 1) return j <= 6 ? f(Shape4<1, 1, 1, 6>()) : f(Shape4<1, 1, 1, 8>());
      if (j > 6) return f(Shape4<1, 0, 1, 8>());
      if (j > 4) return f(Shape4<1, 0, 1, 6>());
      if (j > 2) return f(Shape4<1, 0, 2, 4>());
      return f(Shape4<1, 0, 4, 2>());
    }
  }
  const int steps = (width + 255) / 256, j = (width + 32 * steps - 1) / (32 * steps);
  if (steps > 1) return j <= 6 ? f(Shape4<0, 1, 1, 6>()) : f(Shape4<0, 1, 1, 8>());
  if (j > 4) return f(Shape4<0, 0, 1, 8>());
  if (j > 2) return f(Shape4<0, 0, 2, 4>());
  if (j > 1) return f(Shape4<0, 0, 4, 2>());
  return f(Shape4<0, 0, 8, 1>());
}

// The same for rows of a few elements, where a row would leave most of a warp idle: four bytes
// of the run per lane and step, the rows' addresses in shared memory; reciprocal =
// ceil(2^32 / width) divides what is below 2^32 / width exactly.  The stores are whole lines as
// they are.
constexpr int kFlatWidth = 16;     // widest row
constexpr int kFlatRows = 512;     // most rows of a block
constexpr int kFlatWords = 16;     // words of a thread, about

inline bool flat_fits(int width, const void* out) { return width <= kFlatWidth && ((uintptr_t)out & 3) == 0; }
inline int flat_rows(int width, size_t elem) {
  const int rows = kTileThreads * kFlatWords * (4 / (int)elem) / width / 2 * 2;
  return rows < kFlatRows ? rows : kFlatRows;
}
inline uint32_t flat_reciprocal(int width) {   // of 1 it would be 2^32: not used
  return width == 1 ? 0u : (uint32_t)((0xffffffffull + width) / width);
}

// The row of element e of a run.
__device__ __forceinline__ int flat_row(int e, int width, uint32_t reciprocal) {
  return width == 1 ? e : (int)__umulhi((uint32_t)e, reciprocal);
}
// A lane's word of a run, or its first element where the run ends inside it.
__device__ __forceinline__ void flat_store(float* to, const float (&f)[1], bool) { *to = f[0]; }
template <typename T>
__device__ __forceinline__ void flat_store(T* to, const float (&f)[2], bool whole) {
  struct alignas(4) Two { T a, b; };
  if (whole) *reinterpret_cast<Two*>(to) = Two{from_float<T>(f[0]), from_float<T>(f[1])};
  else *to = from_float<T>(f[0]);
}

template <typename T, bool SCALE, typename Get>
__device__ __forceinline__ void gather_flat(const Get& get, long long rows, int tile, uint32_t reciprocal, int width,
                                            float scale, T* __restrict__ out) {
  constexpr int kEach = 4 / (int)sizeof(T);
  __shared__ const T* row[kFlatRows];
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, rows - first);
  for (int k = threadIdx.x; k < n; k += kTileThreads) {
    const T* r = get(first + k);
    row[k] = r ? r : reinterpret_cast<const T*>(g_zero_row);
  }
  __syncthreads();
  T* to = out + first * width;
  const int total = n * width;
#pragma unroll 4
  for (int p = threadIdx.x * kEach; p < total; p += kTileThreads * kEach) {
    T v[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = min(p + i, total - 1), t = flat_row(e, width, reciprocal);
      const T x = row[t][e - t * width];
      v[i] = SCALE ? from_float<T>(scale * to_float(x)) : x;
    }
    if constexpr (kEach == 1) {
      to[p] = v[0];
    } else if (p + 1 < total) {
      struct alignas(4) Two { T a, b; };
      *reinterpret_cast<Two*>(to + p) = Two{v[0], v[1]};
    } else {
      to[p] = v[0];
    }
  }
}

}  // namespace cvhrf
