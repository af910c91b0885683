// Rows of a table that many entries share: cvhrf_table_lookup and cvhrf_table_gradient.
//
//   lookup    out[t] = scale * table[index[t]]                        (a row of zeros where index[t] is outside)
//   gradient  grad_table[v] = scale * sum_{t : index[t] = v} grad[t]  (fp32, entries in order), row_mask[v] = any
//
// Both are bound by memory: the lookup reads the distinct rows and writes T rows; the
// gradient reads T rows and writes V.
//
// The gradient sorts the entries by row (row_groups.cu, which also marks the rows that occur)
// and adds up runs of entries with the same row.  Every unit of lanes takes an equal share of
// the sorted entries, whatever rows they belong to, so a row with very many entries holds up
// nobody while they are added up.  A row whose entries lie in several units is joined in the order
// of the units: inside a block through shared memory, where the unit in which the row ends walks the
// sums before it one by one, between blocks by table_join_kernel.  That walk is what a popular row
// costs: little where a block has few units (1M entries on 65536 rows of 59 floats: 117 us, 127 if all
// name one row), more with rows of a few elements in the forms of one block's sort, which have 1024 /
// width units (300k on 4096 rows of 3 floats: 27 and 39 us, of 1: 25 and 64; 2048 of 1: 16 and 59;
// replayed from a graph, cold).  The order of every sum
// is fixed, so results repeat.  Blocks between those that add up write zeros into the rows that
// do not occur: they only write and the others mostly read, and every row is written once.
#include <algorithm>
#include "row_groups.cuh"
#include "row_sort.cuh"
#include "row_types.cuh"
#include "row_tiles.cuh"
#include "row_words.cuh"

namespace cvhrf {
namespace {

constexpr int kThreads = 256;

// ---- lookup ---------------------------------------------------------------------------
__device__ __forceinline__ long long table_row(const void* index, int bytes, long long t, long long rows) {
  const long long v = bytes == 4 ? (long long)((const int*)index)[t] : ((const long long*)index)[t];
  return (unsigned long long)v < (unsigned long long)rows ? v : -1;
}

// Aligned rows.  A row is owned by up to a warp of lanes; an owner has ROWS rows in flight (J
// packs of each at a time), the owners of a block neighbouring rows.  Blocks walk over the
// entries, and the indices of the next rows are read while these rows are on their way:
// without that a row waits for two trips to memory, one after the other.
template <typename T, int ROWS, int J>
__global__ void __launch_bounds__(kThreads, 4) table_lookup_kernel(const T* __restrict__ table, long long rows,
                                                                   int width, long long stride,
                                                                   const void* __restrict__ index, int index_bytes,
                                                                   long long entries, int lanes, int owners,
                                                                   float scale, T* __restrict__ out) {
  using R = Row<T, kAligned>;
  const Owner o = Owner::of(lanes);
  const int step = lanes * R::kVec;
  if (!o.live) return;
  const long long walk = (long long)gridDim.x * owners * ROWS;
  long long first = (long long)blockIdx.x * (owners * ROWS) + o.index;
  long long v[ROWS];
  auto load_index = [&](long long from) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const long long t = from + k * owners;
      v[k] = t < entries ? table_row(index, index_bytes, t, rows) : -1;
    }
  };
  load_index(first);
  for (; first < entries; first += walk) {
    const T* from[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) from[k] = v[k] >= 0 ? table + v[k] * stride : nullptr;
    bool next = true;
    for (int c = o.lane * R::kVec + (int)blockIdx.y * step * J; c < width; c += step * J * (int)gridDim.y) {
      typename R::Raw p[ROWS][J];
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (from[k] && c + j * step < width) p[k][j] = R::load(from[k] + c + j * step);
      if (next) load_index(first + walk);
      next = false;
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (first + k * owners < entries && c + j * step < width) {
            float f[R::kVec];
            R::floats(p[k][j], f);
#pragma unroll
            for (int i = 0; i < R::kVec; ++i) f[i] *= scale;
            R::store(out + (first + k * owners) * width + c + j * step, from[k] ? R::words(f) : zero_words());
          }
    }
  }
}

// Rows that are not aligned, up to 4 KB.
template <typename T, typename S>
__global__ void __launch_bounds__(kTileThreads) table_lookup_tile_kernel(const T* __restrict__ table, long long rows,
                                                                         int width, long long stride,
                                                                         const void* __restrict__ index,
                                                                         int index_bytes, long long entries, int tile,
                                                                         float scale, T* __restrict__ out) {
  gather_tile<T, true, S::kPairs, S::kWide, S::kRows, S::kJ>(
      [&](long long t) -> const T* {
        const long long v = table_row(index, index_bytes, t, rows);
        return v >= 0 ? table + v * stride : nullptr;
      },
      entries, tile, width, scale, out);
}

// ... of a few elements.
template <typename T>
__global__ void __launch_bounds__(kTileThreads) table_lookup_flat_kernel(const T* __restrict__ table, long long rows,
                                                                         int width, long long stride,
                                                                         const void* __restrict__ index,
                                                                         int index_bytes, long long entries, int tile,
                                                                         uint32_t reciprocal, float scale,
                                                                         T* __restrict__ out) {
  gather_flat<T, true>(
      [&](long long t) -> const T* {
        const long long v = table_row(index, index_bytes, t, rows);
        return v >= 0 ? table + v * stride : nullptr;
      },
      entries, tile, reciprocal, width, scale, out);
}

// ... and wider ones, or an output that does not begin on 16 bytes.
template <typename T, int LANES, int FLIGHT, int J>
__global__ void __launch_bounds__(kWordThreads) table_lookup_words_kernel(const T* __restrict__ table, Source4 source,
                                                                          long long rows, int width,
                                                                          const void* __restrict__ index,
                                                                          int index_bytes, long long entries,
                                                                          int rounds, int lanes, float scale,
                                                                          T* __restrict__ out) {
  copy_rows<T, true, LANES, FLIGHT, J>(
      [&](long long e, int& from, int& to) {
        from = (int)table_row(index, index_bytes, e, rows);
        to = (int)e;
      },
      entries, rounds, lanes, width, table, source, scale, out);
}

template <typename T, int LANES, int FLIGHT, int J>
int launch_lookup_words(const void* table, long long rows, int width, long long stride, const void* index,
                        int index_bytes, long long entries, float scale, void* out, cudaStream_t st) {
  const int lanes = word_lanes(words_of<T>(width)), owners = 32 / lanes, rounds = rounds_for(entries, owners, FLIGHT);
  const unsigned blocks = word_blocks(entries, rounds, owners);
  const unsigned parts = parts_for(blocks, (words_of<T>(width) + lanes * J - 1) / (lanes * J));
  table_lookup_words_kernel<T, LANES, FLIGHT, J><<<dim3(blocks, parts), kWordThreads, 0, st>>>(
      (const T*)table, source4_of(table, rows, stride, width, sizeof(T)), rows, width, index, index_bytes, entries,
      rounds, lanes, scale, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T, int ROWS, int J>
int launch_lookup(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
                  long long entries, int lanes, float scale, void* out, cudaStream_t st) {
  static const int resident = [] {
    int blocks = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, table_lookup_kernel<T, ROWS, J>, kThreads, 0);
    return e == cudaSuccess && blocks > 0 ? blocks : 4;
  }();
  const int owners = owners_of(kThreads, lanes);
  const long long per_block = (long long)owners * ROWS, blocks = (entries + per_block - 1) / per_block;
  const long long most = 148 * resident;
  const unsigned parts = parts_for((unsigned)(blocks < most ? blocks : most),
                                   (packs_of<T, kAligned>(width) + lanes * J - 1) / (lanes * J));
  table_lookup_kernel<T, ROWS, J><<<dim3((unsigned)(blocks < most ? blocks : most), parts), kThreads, 0, st>>>(
      (const T*)table, rows, width, stride, index, index_bytes, entries, lanes, owners, scale, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T>
int lookup(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
           long long entries, float scale, void* out, cudaStream_t st) {
  if (rows_16(table, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0) {
    const int packs = packs_of<T, kAligned>(width), lanes = lanes_for(packs);
    if (packs > 64)
      return launch_lookup<T, 1, 4>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
    if (packs > 32)
      return launch_lookup<T, 2, 2>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
    return launch_lookup<T, 4, 1>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
  }
  if (flat_fits(width, out)) {
    const int tile = flat_rows(width, sizeof(T));
    table_lookup_flat_kernel<T><<<(unsigned)((entries + tile - 1) / tile), kTileThreads, 0, st>>>(
        (const T*)table, rows, width, stride, index, index_bytes, entries, tile, flat_reciprocal(width), scale,
        (T*)out);
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  if (tile_fits(width, sizeof(T), out)) {
    const int tile = tile_rows(entries, width, sizeof(T));
    return with_shape<T>(width, [&](auto shape) {
      table_lookup_tile_kernel<T, decltype(shape)>
          <<<(unsigned)((entries + tile - 1) / tile), kTileThreads, (size_t)tile * width * sizeof(T), st>>>(
              (const T*)table, rows, width, stride, index, index_bytes, entries, tile, scale, (T*)out);
      CVHRF_LAUNCH_CHECK();
      return CVHRF_OK;
    });
  }
  const int words = words_of<T>(width);
  if (words > 64)
    return launch_lookup_words<T, 32, 2, 4>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  if (words >= 32)
    return launch_lookup_words<T, 32, 4, 2>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  return launch_lookup_words<T, 0, 4, 1>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
}

// ---- gradient -------------------------------------------------------------------------
constexpr int kBlockItems = 2048;   // most entries of a block, staged in shared memory

// What a block leaves for table_join_kernel: the part of a row that began in an earlier
// block and ends in this one (head), and of the row that goes on behind its end (tail).
struct Joins {
  float* head;        // block x width
  float* tail;        // block x width
  int* head_row;      // -1: none
  int* tail_row;      // -1: none
  int* tail_begun;    // the row's first entry is in this block
};

struct Gradient {
  const uint32_t* keys;      // sorted rows
  const uint32_t* entries;   // the entry of each
  const uint32_t* count;     // how many
  long long stride;          // elements between the rows of grad
  int width;
  int lanes, units;          // lanes of a unit (up to 32), units of a block
  int items;                 // entries of a unit
  float scale;
  const uint8_t* touched;    // rows that occur
  uint32_t table_rows;
  int blocks, tiles;         // that add up: runs of entries x tiles of columns
  int clear_blocks;          // that clear, spread between them
  int clear_step;            // rows that a warp of theirs looks at together, 32 at most
};

// Columns per lane: one pack of aligned rows, or J single elements `lanes` apart (so that a
// warp's loads are whole lines wherever a row begins).
template <typename T, bool ALIGNED, int J>
struct Columns {
  using R = Row<T, ALIGNED ? kAligned : kElement>;
  static constexpr int kVec = R::kVec, kEach = ALIGNED ? kVec : J;
  static constexpr int kBatch = ALIGNED ? 8 : 16 / J;   // rows in flight
  struct Raw {
    typename R::Raw v[J];
  };
};
template <int EACH>
constexpr size_t gradient_shared() {   // staged rows and keys, heads and tails of the units, their rows
  return (kBlockItems + 1) * (sizeof(uint64_t) + sizeof(uint32_t)) + 4 + 2 * kThreads * EACH * sizeof(float) +
         3 * kThreads * sizeof(int);
}

// Zeros into a share of the rows that do not occur, a warp per row.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void clear_rows(const Gradient& g, int share, T* __restrict__ out) {
  const uint32_t warps = (uint32_t)g.clear_blocks * (kThreads / 32), lane = threadIdx.x & 31;
  const uint32_t warp = (uint32_t)share * (kThreads / 32) + (threadIdx.x >> 5);
  const uint32_t step = g.clear_step;
  for (unsigned long long r0 = (unsigned long long)warp * step; r0 < g.table_rows; r0 += (unsigned long long)warps * step) {
    unsigned empty = __ballot_sync(0xffffffffu, lane < step && r0 + lane < g.table_rows && !g.touched[r0 + lane]);
    if (!ALIGNED && g.width < 32) {   // narrow rows as one run of elements
      T* to = out + (long long)r0 * g.width;
      for (int e = lane; e < (int)step * g.width; e += 32)
        if (empty >> (e / g.width) & 1) to[e] = from_float<T>(0.f);
    } else {
      for (; empty; empty &= empty - 1)
        clear_row<T, ALIGNED ? kAligned : kSpan>(out + (long long)(r0 + __ffs(empty) - 1) * g.width, g.width, lane, 32);
    }
  }
}

template <typename T, bool ALIGNED, int J>
__global__ void __launch_bounds__(kThreads) table_gradient_kernel(Gradient g, const T* __restrict__ grad,
                                                                  T* __restrict__ out, Joins joins) {
  using C = Columns<T, ALIGNED, J>;
  using R = typename C::R;
  constexpr int kEach = C::kEach, kBatch = C::kBatch;
  extern __shared__ __align__(16) unsigned char raw[];
  const int lanes = g.lanes, units = g.units;
  const int unit = threadIdx.x / lanes, lane = threadIdx.x - unit * lanes;
  const bool live = unit < units;   // a few threads are left over where the lanes do not divide them
  const int tile_width = lanes * kEach;
  const T** rows = reinterpret_cast<const T**>(raw);
  float* heads = reinterpret_cast<float*>(rows + kBlockItems + 1);   // units x tile_width
  float* tails = heads + kThreads * kEach;
  int* head_row = reinterpret_cast<int*>(tails + kThreads * kEach);
  int* tail_row = head_row + kThreads;
  int* tail_begun = tail_row + kThreads;
  uint32_t* keys = reinterpret_cast<uint32_t*>(tail_begun + kThreads);
  follow();
  let_next_start();
  // block b adds up, or clears where b's share of the clearing blocks goes up by one
  const int add_blocks = g.blocks * g.tiles;
  const long long all = add_blocks + g.clear_blocks;
  const int clears = (int)((long long)blockIdx.x * g.clear_blocks / all);
  if ((int)(((long long)blockIdx.x + 1) * g.clear_blocks / all) > clears) return clear_rows<T, ALIGNED>(g, clears, out);
  const int block = ((int)blockIdx.x - clears) / g.tiles, tile = ((int)blockIdx.x - clears) - block * g.tiles;
  const uint32_t n = *g.count;
  const uint32_t block_items = units * g.items, first = min(n, block * block_items);
  const int count = (int)min(block_items, n - first);
  const uint32_t before_first = first > 0 ? g.keys[first - 1] : 0xffffffffu;
  for (int i = threadIdx.x; i <= count; i += kThreads) {   // one more: whether the last row goes on
    const bool in = first + i < n;
    keys[i] = in ? g.keys[first + i] : 0xffffffffu;
    if (in && i < count) rows[i] = grad + (long long)g.entries[first + i] * g.stride;
  }
  __syncthreads();
  const int p0 = live ? min(unit * g.items, count) : count, p1 = min(p0 + g.items, count);
  const int first_col = tile * tile_width + lane * C::kVec;
  const int left = live ? g.width - first_col : 0;   // columns from the lane's first one on
  auto in = [&](int j) { return ALIGNED ? left > 0 : j * lanes < left; };
  float acc[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) acc[i] = 0.f;
  uint32_t row = p0 < p1 ? keys[p0] : 0xffffffffu;
  bool begun_before = p0 < p1 && (p0 > 0 ? keys[p0 - 1] : before_first) == row;   // in earlier units
  int my_head = -1;
  // a lane's columns of the unit's head and tail, kEach floats apart
  float* my_head_sum = heads + (unit * lanes + lane) * kEach;
  float* my_tail_sum = tails + (unit * lanes + lane) * kEach;
  auto write = [&](uint32_t r, const float (&sum)[kEach]) {
    T* to = out + (long long)r * g.width + first_col;
    if constexpr (ALIGNED) {
      float f[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) f[i] = g.scale * sum[i];
      if (left > 0) R::store(to, R::words(f));
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (in(j)) to[j * lanes] = from_float<T>(g.scale * sum[j]);
    }
  };
  auto end_row = [&]() {
    if (begun_before) {   // its other entries are elsewhere: leave the sum for the join
      my_head = (int)row;
#pragma unroll
      for (int i = 0; i < kEach; ++i) my_head_sum[i] = acc[i];
    } else {
      write(row, acc);
    }
    begun_before = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i) acc[i] = 0.f;
  };
  auto load = [&](int p, typename C::Raw& v) {
    const T* from = rows[p] + first_col;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (in(j)) v.v[j] = R::load(from + j * lanes);
  };
  auto add = [&](int p, const typename C::Raw& v) {
    const uint32_t key = keys[p];
    if (key != row) {
      end_row();
      row = key;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (in(j)) {
        float f[C::kVec];
        R::floats(v.v[j], f);
#pragma unroll
        for (int i = 0; i < C::kVec; ++i) acc[j * C::kVec + i] += f[i];
      }
  };
  int p = p0;
  for (; p + kBatch <= p1; p += kBatch) {
    typename C::Raw v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) load(p + b, v[b]);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) add(p + b, v[b]);
  }
  if (p < p1) {
    typename C::Raw v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) load(p + b, v[b]);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) add(p + b, v[b]);
  }
  // the last row, which may go on behind the unit
  bool open = false;
  if (p0 < p1) {
    open = keys[p1] == row;
    if (!open) {
      end_row();
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) my_tail_sum[i] = acc[i];
    }
  }
  if (live && lane == 0) {
    head_row[unit] = my_head;
    tail_row[unit] = open ? (int)row : -1;
    tail_begun[unit] = open && !begun_before;
  }
  __syncthreads();
  // a row that ends in this unit and began in an earlier one: add the tails before it
  bool unfinished = false;
  if (my_head >= 0) {
    float sum[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum[i] = my_head_sum[i];
    bool whole = false;
    for (int q = unit - 1; q >= 0 && !whole; --q) {
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum[i] += tails[(q * lanes + lane) * kEach + i];
      whole = tail_begun[q];
    }
    if (whole) {
      write((uint32_t)my_head, sum);
    } else {   // it began before this block
      unfinished = true;
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (in(i)) joins.head[(long long)block * g.width + first_col + (ALIGNED ? i : i * lanes)] = sum[i];
      if (lane == 0 && tile == 0) joins.head_row[block] = my_head;
    }
  }
  const int block_head = __syncthreads_or(unfinished);
  if (!block_head && threadIdx.x == 0 && tile == 0) joins.head_row[block] = -1;
  // the row that goes on behind the block: the tail of its last unit with entries
  const int last = count > 0 ? (count - 1) / g.items : 0;
  if (unit == last) {
    const int r = tail_row[unit];
    bool begun = false;
    if (r >= 0) {
      float sum[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum[i] = 0.f;
      for (int q = unit; q >= 0 && !begun; --q) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum[i] += tails[(q * lanes + lane) * kEach + i];
        begun = tail_begun[q];
      }
#pragma unroll
      for (int i = 0; i < kEach; ++i)
        if (in(i)) joins.tail[(long long)block * g.width + first_col + (ALIGNED ? i : i * lanes)] = sum[i];
    }
    if (lane == 0 && tile == 0) {
      joins.tail_row[block] = r;
      joins.tail_begun[block] = begun;
    }
  }
}

// Rows whose entries lie in several blocks: block x's head plus the tails before it, the
// blocks shared between `slices` threads of a column and then added in the slices' order.
template <typename T>
__global__ void __launch_bounds__(kThreads) table_join_kernel(Joins joins, int width, int columns, float scale,
                                                              T* __restrict__ out) {
  __shared__ float part[kThreads];
  __shared__ int s_first;
  follow();
  const int block = blockIdx.x, row = joins.head_row[block];
  if (row < 0) return;
  // the chain of open tails of this row: it begins at the nearest block where the row begins
  if (threadIdx.x == 0) s_first = 0;
  __syncthreads();
  for (int q0 = block - 1; q0 >= 0; q0 -= kThreads) {
    const int q = q0 - (int)threadIdx.x;
    const bool begin = q >= 0 && joins.tail_begun[q] && joins.tail_row[q] == row;
    if (begin) s_first = q;   // one block at most begins the row
    if (__syncthreads_or(begin)) break;
  }
  __syncthreads();
  const int first = s_first;
  const int slices = kThreads / columns, slice = threadIdx.x / columns;
  const int c = blockIdx.y * columns + (threadIdx.x & (columns - 1));
  float sum = 0.f;
  if (c < width)
    for (int q = first + slice; q < block; q += slices) sum += joins.tail[(long long)q * width + c];
  part[threadIdx.x] = sum;
  __syncthreads();
  if (slice == 0 && c < width) {
    for (int s = 1; s < slices; ++s) sum += part[s * columns + threadIdx.x];
    sum += joins.head[(long long)block * width + c];
    out[(long long)row * width + c] = from_float<T>(scale * sum);
  }
}

// ---- gradient of few entries -----------------------------------------------------------------
// A small batch is bound by its launches: every block sorts all entries for itself, then takes a
// share of the table's rows and a tile of their columns, adds up the rows that occur and clears
// some of the others.  One launch, nothing in global memory between (512 entries on 4096 rows of
// 64 floats: 9.7 us, 11.7 in three launches).  Shares x tiles fill the SMs once: a second wave
// would sort again (2048 entries on 5000 rows of 1024 floats: 16 us; 80 in 8 waves, 21 in three
// launches).  Tables of more elements, mostly to be cleared, are left to more blocks (50000 rows of
// 2047 floats: 130 us against 95; of 1023: 61 against 58).
constexpr int kFewEntries = 2 * row_sort::kThreads;
constexpr int kFewBlocks = 148, kFewWidth = 32 * kFewBlocks;   // a tile has 32 columns at least
constexpr long long kFewElements = 1ll << 26;
inline bool few(long long entries, long long rows, int width) {
  return entries <= kFewEntries && width <= kFewWidth && rows * width <= kFewElements;
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(row_sort::kThreads) few_entries_kernel(row_sort::Source index, uint32_t n, int bits,
                                                                         int rows_each, int lanes, int width,
                                                                         const T* __restrict__ grad, long long stride,
                                                                         float scale, T* __restrict__ out,
                                                                         uint8_t* __restrict__ mask) {
  using namespace row_sort;
  using C = Columns<T, ALIGNED, 1>;
  using Rw = typename C::R;
  constexpr int kVec = C::kVec, kBatch = 4;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const uint32_t count = sort_run(sh, index, 0, n, bits, passes_for(bits));
  __syncthreads();
  auto first_of = [&](uint32_t row) {   // the first entry of this row or a later one
    uint32_t lo = 0, hi = count;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) >> 1;
      if (sh.key[mid] < row) lo = mid + 1;
      else hi = mid;
    }
    return lo;
  };
  const uint32_t r0 = (uint32_t)min((unsigned long long)blockIdx.x * rows_each, (unsigned long long)index.rows);
  const uint32_t r1 = (uint32_t)min((unsigned long long)r0 + rows_each, (unsigned long long)index.rows);
  const int begin = (int)first_of(r0), end = (int)first_of(r1);
  // the rows that do not occur, whole, `step` at a time per warp (shared evenly between the warps
  // of all tiles)
  {
    const int in_warp = threadIdx.x & 31, warps = kWarps * gridDim.y;
    const int warp = blockIdx.y * kWarps + (threadIdx.x >> 5), step = max(1, min(32, rows_each / warps));
    for (uint32_t r = r0 + warp * step; r < r1; r += warps * step) {
      const bool mine = in_warp < step && r + in_warp < r1;
      uint32_t at = 0;
      if (mine) at = first_of(r + in_warp);
      const bool occurs = mine && at < count && sh.key[at] == r + in_warp;
      if (mask && mine) mask[r + in_warp] = occurs;
      for (unsigned empty = __ballot_sync(0xffffffffu, mine && !occurs); empty; empty &= empty - 1)
        clear_row<T, ALIGNED ? kAligned : kSpan>(out + (long long)(r + __ffs(empty) - 1) * width, width, in_warp, 32);
    }
  }
  // units of the entries in this share, as table_gradient_kernel's; none goes on in another block
  const int units = row_sort::kThreads / lanes, unit = threadIdx.x / lanes, lane = threadIdx.x - unit * lanes;
  const int items = (end - begin + units - 1) / units;
  const int p0 = unit < units ? min(begin + unit * items, end) : end, p1 = min(p0 + items, end);
  float* heads = reinterpret_cast<float*>(sh.cnt);   // the sort's counters have done their work
  float* tails = heads + row_sort::kThreads * kVec;
  int* begun = reinterpret_cast<int*>(sh.base);
  static_assert(sizeof(sh.cnt) >= 2 * row_sort::kThreads * kVec * sizeof(float));
  static_assert(sizeof(sh.base) + sizeof(sh.start) >= row_sort::kThreads * sizeof(int));
  const int first_col = (blockIdx.y * lanes + lane) * kVec;
  const bool in = unit < units && first_col < width;
  float acc[kVec];
#pragma unroll
  for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
  uint32_t row = p0 < p1 ? sh.key[p0] : kNone;
  bool begun_before = p0 < p1 && p0 > begin && sh.key[p0 - 1] == row;
  int my_head = -1;
  auto write = [&](uint32_t r, float (&sum)[kVec]) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum[i] *= scale;
    if (in) Rw::store(out + (long long)r * width + first_col, Rw::words(sum));
  };
  auto end_row = [&]() {
    if (begun_before) {
      my_head = (int)row;
#pragma unroll
      for (int i = 0; i < kVec; ++i) heads[threadIdx.x * kVec + i] = acc[i];
    } else {
      write(row, acc);
    }
    begun_before = false;
#pragma unroll
    for (int i = 0; i < kVec; ++i) acc[i] = 0.f;
  };
  for (int p = p0; p < p1; p += kBatch) {
    typename Rw::Raw v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1 && in) v[b] = Rw::load(grad + (long long)sh.entry[p + b] * stride + first_col);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) {
        const uint32_t k = sh.key[p + b];
        if (k != row) {
          end_row();
          row = k;
        }
        if (in) {
          float f[kVec];
          Rw::floats(v[b], f);
#pragma unroll
          for (int i = 0; i < kVec; ++i) acc[i] += f[i];
        }
      }
  }
  bool open = false;
  if (p0 < p1) {
    open = p1 < end && sh.key[p1] == row;
    if (!open) {
      end_row();
    } else {
#pragma unroll
      for (int i = 0; i < kVec; ++i) tails[threadIdx.x * kVec + i] = acc[i];
    }
  }
  if (unit < units && lane == 0) begun[unit] = open && !begun_before;
  __syncthreads();
  if (my_head >= 0) {
    float sum[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) sum[i] = heads[threadIdx.x * kVec + i];
    for (int q = unit - 1; q >= 0; --q) {
#pragma unroll
      for (int i = 0; i < kVec; ++i) sum[i] += tails[(q * lanes + lane) * kVec + i];
      if (begun[q]) break;
    }
    write((uint32_t)my_head, sum);
  }
}

template <typename T>
int few_entries(const void* grad, long long stride, int width, const void* index, int index_bytes, long long n,
                long long rows, float scale, void* out, uint8_t* mask, cudaStream_t st) {
  const row_sort::Source source{index, index_bytes, nullptr, nullptr, (uint32_t)rows, 0};
  const int bits = row_sort::bits_for((unsigned long long)rows);
  auto launch = [&](auto aligned) {
    constexpr bool kAlignedRows = decltype(aligned)::value;
    static std::atomic<unsigned long long> allowed{0};
    CVHRF_CUDA_TRY(allow_shared(few_entries_kernel<T, kAlignedRows>, sizeof(row_sort::Shared), allowed));
    const int packs = width / Columns<T, kAlignedRows, 1>::kVec, lanes = packs < 32 ? packs : 32;
    const int tiles = (packs + lanes - 1) / lanes, shares = kFewBlocks / tiles;
    const long long rows_each = std::max(32ll, (rows + shares - 1) / shares);
    few_entries_kernel<T, kAlignedRows>
        <<<dim3((unsigned)((rows + rows_each - 1) / rows_each), tiles), row_sort::kThreads, sizeof(row_sort::Shared), st>>>(
            source, (uint32_t)n, bits, (int)rows_each, lanes, width, (const T*)grad, stride, scale, (T*)out, mask);
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  };
  if (rows_16(grad, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0) return launch(std::true_type());
  return launch(std::false_type());
}

// ---- gradient of small tables ---------------------------------------------------------------
// A codebook's whole gradient fits in shared memory: a block sorts its share of the entries there
// (row_sort.cuh), adds the runs up into a table of its own, and table_sum_kernel adds the blocks'
// tables in their order.  2 launches; by way of the sorted list of all entries it is 6 (300k
// entries on 4096 rows of 3 floats: 33 us against 19).
constexpr int kSmallElements = 16384;   // rows x width
constexpr int kSmallWidth = 32;         // one lane per column
constexpr int kSmallBlocks = 148;

struct SmallTable {
  row_sort::Source index;
  uint32_t n, chunk;        // entries, of a block
  int bits;
  long long stride;
  int width;
  float* sums;              // block x rows x width
  uint8_t* touched;         // block x rows
};

constexpr size_t small_shared() { return sizeof(row_sort::Shared) + kSmallElements * (sizeof(float) + 1); }

template <typename T>
__global__ void __launch_bounds__(row_sort::kThreads) small_table_kernel(SmallTable t, const T* __restrict__ grad) {
  using namespace row_sort;
  constexpr int kBatch = 4;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  float* table = reinterpret_cast<float*>(raw + sizeof(Shared));
  uint8_t* touched = reinterpret_cast<uint8_t*>(table + kSmallElements);
  const int rows = (int)t.index.rows, width = t.width, elements = rows * width;
  let_next_start();
  for (int i = threadIdx.x; i < elements; i += row_sort::kThreads) table[i] = 0.f;
  for (int i = threadIdx.x; i < rows; i += row_sort::kThreads) touched[i] = 0;
  // units of one lane per column; heads and tails of the units take the place of the sort's counters
  const int units = row_sort::kThreads / width, unit = threadIdx.x / width, lane = threadIdx.x - unit * width;
  float* heads = reinterpret_cast<float*>(sh.cnt);
  float* tails = heads + row_sort::kThreads;
  int* begun = reinterpret_cast<int*>(tails + row_sort::kThreads);
  static_assert(sizeof(sh.cnt) >= 3 * row_sort::kThreads * sizeof(float));
  const uint32_t begin = min(t.n, blockIdx.x * t.chunk), end = min(t.n, begin + t.chunk);
  for (uint32_t tile = begin; tile < end; tile += kTile) {
    const int count = (int)sort_run(sh, t.index, tile, min(end - tile, (uint32_t)kTile), t.bits, passes_for(t.bits));
    __syncthreads();
    const int items = (count + units - 1) / units;
    const int p0 = unit < units ? min(unit * items, count) : count, p1 = min(p0 + items, count);
    float acc = 0.f;
    uint32_t row = p0 < p1 ? sh.key[p0] : kNone;
    bool begun_before = p0 < p1 && p0 > 0 && sh.key[p0 - 1] == row;
    int my_head = -1;
    auto end_row = [&]() {
      if (begun_before) {
        my_head = (int)row;
        heads[threadIdx.x] = acc;
      } else {   // the run lies in this unit alone
        table[row * width + lane] += acc;
        touched[row] = 1;
      }
      begun_before = false;
      acc = 0.f;
    };
    for (int p = p0; p < p1; p += kBatch) {
      float v[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (p + b < p1) v[b] = to_float(grad[(long long)sh.entry[p + b] * t.stride + lane]);
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (p + b < p1) {
          const uint32_t k = sh.key[p + b];
          if (k != row) {
            end_row();
            row = k;
          }
          acc += v[b];
        }
    }
    bool open = false;
    if (p0 < p1) {
      open = p1 < count && sh.key[p1] == row;
      if (open) tails[threadIdx.x] = acc;
      else end_row();
    }
    if (unit < units && lane == 0) begun[unit] = open && !begun_before;
    __syncthreads();
    if (my_head >= 0) {   // a run over several units: from its first one on
      float sum = heads[threadIdx.x];
      for (int q = unit - 1; q >= 0; --q) {
        sum += tails[q * width + lane];
        if (begun[q]) break;
      }
      table[my_head * width + lane] += sum;
      touched[my_head] = 1;
    }
    __syncthreads();
  }
  __syncthreads();
  for (int i = threadIdx.x; i < elements; i += row_sort::kThreads) t.sums[(size_t)blockIdx.x * elements + i] = table[i];
  for (int i = threadIdx.x; i < rows; i += row_sort::kThreads) t.touched[(size_t)blockIdx.x * rows + i] = touched[i];
}

// Sums over the blocks' tables, `slices` threads per element.
constexpr int kSumSlices = 8, kSumElements = kThreads / kSumSlices;
template <typename T>
__global__ void __launch_bounds__(kThreads) table_sum_kernel(const float* sums, const uint8_t* touched, int blocks,
                                                             int rows, int width, float scale, T* __restrict__ out,
                                                             uint8_t* __restrict__ mask) {
  __shared__ float part[kSumSlices][kSumElements];
  __shared__ int any[kSumElements];
  follow();
  const int slice = threadIdx.x / kSumElements, k = threadIdx.x - slice * kSumElements;
  const int elements = rows * width, e = blockIdx.x * kSumElements + k;
  float sum = 0.f;
  if (e < elements)
#pragma unroll 8
    for (int b = slice; b < blocks; b += kSumSlices) sum += sums[(size_t)b * elements + e];
  part[slice][k] = sum;
  if (slice == 0) any[k] = 0;
  __syncthreads();
  if (slice == 0 && e < elements) {
#pragma unroll
    for (int s = 1; s < kSumSlices; ++s) sum += part[s][k];
    out[e] = from_float<T>(scale * sum);
  }
  if (mask && e < rows) {   // the first `rows` elements' threads look after a row each
    int t = 0;
#pragma unroll 8
    for (int b = slice; b < blocks; b += kSumSlices) t |= touched[(size_t)b * rows + e];
    if (t) any[k] = 1;
  }
  __syncthreads();
  if (mask && slice == 0 && e < rows) mask[e] = (uint8_t)any[k];
}

inline bool small_table(long long rows, int width) { return width <= kSmallWidth && rows * width <= kSmallElements; }
inline int small_blocks(long long n) {   // two entries per thread at least
  const long long b = (n + 2 * row_sort::kThreads - 1) / (2 * row_sort::kThreads);
  return (int)(b < kSmallBlocks ? b : kSmallBlocks);
}

template <typename T>
int small_gradient(const void* grad, long long stride, int width, const void* index, int index_bytes, long long n,
                   long long rows, float scale, void* out, uint8_t* mask, void* workspace, cudaStream_t st) {
  static std::atomic<unsigned long long> allowed{0};
  CVHRF_CUDA_TRY(allow_shared(small_table_kernel<T>, small_shared(), allowed));
  const int blocks = small_blocks(n), elements = (int)rows * width;
  float* sums = (float*)workspace;
  uint8_t* touched = (uint8_t*)(sums + (size_t)blocks * elements);
  const SmallTable t{{index, index_bytes, nullptr, nullptr, (uint32_t)rows, 0}, (uint32_t)n,
                     (uint32_t)((n + blocks - 1) / blocks), row_sort::bits_for((unsigned long long)rows), stride, width,
                     sums, touched};
  small_table_kernel<T><<<blocks, row_sort::kThreads, small_shared(), st>>>(t, (const T*)grad);
  CVHRF_LAUNCH_CHECK();
  CVHRF_CUDA_TRY(launch_after(table_sum_kernel<T>, dim3((elements + kSumElements - 1) / kSumElements), kThreads, 0, st,
                              sums, touched, blocks, (int)rows, width, scale, (T*)out, mask));
  count_launch(1);
  return CVHRF_OK;
}

constexpr int kMinItems = 4;        // entries of a unit at least

// Most blocks a gradient can have (x dimension): its joins' rows.
inline long long most_blocks(long long n) {
  constexpr long long share = kBlockItems - kThreads;        // of a block whose units do not divide kBlockItems
  const long long full = (n + share - 1) / share + 148 * 8;
  const long long tiny = (n + 8 * kMinItems - 1) / (8 * kMinItems);   // 8 units at least in a block
  return full < tiny ? full : tiny;
}

template <typename T, bool ALIGNED, int J>
int launch_gradient(Gradient g, int lanes, long long n, const void* grad, void* out, float* joins_at, cudaStream_t st) {
  constexpr int kEach = Columns<T, ALIGNED, J>::kEach;
  constexpr size_t shared = gradient_shared<kEach>();
  static_assert(shared <= 48 * 1024, "the default limit of shared memory");
  static const int resident = [] {
    int blocks = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, table_gradient_kernel<T, ALIGNED, J>, kThreads, shared);
    return e == cudaSuccess && blocks > 0 ? (blocks < 8 ? blocks : 8) : 2;
  }();
  g.lanes = lanes;
  const int units = g.units = kThreads / lanes, tile_width = lanes * kEach;
  const int tiles = (g.width + tile_width - 1) / tile_width;
  // equal blocks that fill the SMs a whole number of times
  long long slots = 148 * resident / tiles;
  if (slots < 1) slots = 1;
  const long long waves = (n + slots * kBlockItems - 1) / (slots * kBlockItems);
  long long items = (n + slots * waves * units - 1) / (slots * waves * units);
  if (items < kMinItems) items = kMinItems;
  if (items * units > kBlockItems) items = kBlockItems / units;
  g.items = (int)items;
  const long long blocks = (n + items * units - 1) / (items * units);
  Joins joins;
  joins.head = joins_at;
  joins.tail = joins.head + blocks * g.width;
  joins.head_row = (int*)(joins.tail + blocks * g.width);
  joins.tail_row = joins.head_row + blocks;
  joins.tail_begun = joins.tail_row + blocks;
  g.blocks = (int)blocks;
  g.tiles = tiles;
  // enough blocks that clear for every SM, each warp with 4 to 32 rows
  g.clear_step = (int)std::min(32ll, std::max(4ll, (long long)g.table_rows / (148 * 32)));
  const long long per_block = g.clear_step * (kThreads / 32);
  g.clear_blocks = (int)std::min((g.table_rows + per_block - 1) / per_block, 148ll * 64);
  if (blocks * tiles > 0x7fffffff - g.clear_blocks) return CVHRF_EUNSUPPORTED;
  CVHRF_CUDA_TRY(launch_after(table_gradient_kernel<T, ALIGNED, J>, dim3((unsigned)(blocks * tiles + g.clear_blocks)),
                              kThreads, shared, st, g, (const T*)grad, (T*)out, joins));
  count_launch(1);
  if (blocks == 1) return CVHRF_OK;
  const int columns = next_pow2(g.width < kThreads ? g.width : kThreads);
  CVHRF_CUDA_TRY(launch_after(table_join_kernel<T>, dim3((unsigned)blocks, (g.width + columns - 1) / columns), kThreads,
                              0, st, joins, g.width, columns, g.scale, (T*)out));
  count_launch(1);
  return CVHRF_OK;
}

// Units of as many lanes as a row has packs or elements, a warp at most; wider rows have several
// elements per lane, then tiles.
template <typename T>
int gradient(const void* grad, long long stride, int width, long long n, long long rows, float scale, void* out,
             const uint8_t* touched, const uint32_t* keys, const uint32_t* entries, const uint32_t* count, float* joins, cudaStream_t st) {
  const Gradient g{keys, entries, count, stride, width, 0, 0, 0, scale, touched, (uint32_t)rows, 0, 0, 0};
  if (rows_16(grad, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0) {
    const int packs = packs_of<T, kAligned>(width);
    return launch_gradient<T, true, 1>(g, packs < 32 ? packs : 32, n, grad, out, joins, st);
  }
  if (width <= 32) return launch_gradient<T, false, 1>(g, width, n, grad, out, joins, st);
  // tiles of equal width: 257 columns are two of 192, not one of 256 and one of a column
  const int tiles = (width + 255) / 256, each = (width + 32 * tiles - 1) / (32 * tiles);
  if (each <= 2) return launch_gradient<T, false, 2>(g, 32, n, grad, out, joins, st);
  if (each <= 3) return launch_gradient<T, false, 3>(g, 32, n, grad, out, joins, st);
  if (each <= 4) return launch_gradient<T, false, 4>(g, 32, n, grad, out, joins, st);
  if (each <= 6) return launch_gradient<T, false, 6>(g, 32, n, grad, out, joins, st);
  return launch_gradient<T, false, 8>(g, 32, n, grad, out, joins, st);
}

constexpr long long kMaxRows = 0x7ffffffe;

}  // namespace
}  // namespace cvhrf

using namespace cvhrf;

extern "C" int cvhrf_table_lookup(const cvhrf_lookup_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const auto [table, index, out, rows, row_stride, entries, width, dtype, index_bytes, scale] = *args;
  if (!row_type_ok(dtype) || rows < 0 || rows > kMaxRows || width < 1 || width > kMaxWidth || row_stride < 0 ||
      (index_bytes != 4 && index_bytes != 8) || entries < 0)
    return CVHRF_EINVAL;
  if (entries == 0) return CVHRF_OK;
  if ((rows > 0 && !table) || !index || !out) return CVHRF_EINVAL;
  if (entries > kGroupMaxEntries) return CVHRF_EUNSUPPORTED;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == CVHRF_F32)
    return lookup<float>(table, rows, width, row_stride, index, index_bytes, entries, scale, out, st);
  if (dtype == CVHRF_BF16)
    return lookup<__nv_bfloat16>(table, rows, width, row_stride, index, index_bytes, entries, scale, out, st);
  return lookup<__half>(table, rows, width, row_stride, index, index_bytes, entries, scale, out, st);
}

extern "C" size_t cvhrf_table_gradient_workspace_bytes(long long entries, long long rows, int width) {
  if (entries < 0 || entries > kGroupMaxEntries || rows < 0 || rows > kMaxRows || width < 1 || width > kMaxWidth)
    return 0;
  if (few(entries, rows, width)) return 0;
  if (small_table(rows, width))
    return align_up((size_t)small_blocks(entries) * ((size_t)rows * width * sizeof(float) + (size_t)rows), 256);
  return align_up(group_sort_words(entries) * sizeof(uint32_t), 256) + align_up((size_t)rows, 256) +
         align_up((size_t)most_blocks(entries) * (2 * (size_t)width * sizeof(float) + 3 * sizeof(int)), 256);
}

extern "C" int cvhrf_table_gradient(const cvhrf_gradient_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const auto [grad, index, grad_table, row_mask, workspace, workspace_bytes, grad_stride, entries, rows, width, dtype,
              index_bytes, scale] = *args;
  if (!row_type_ok(dtype) || rows < 0 || rows > kMaxRows || width < 1 || width > kMaxWidth || grad_stride < 0 ||
      (index_bytes != 4 && index_bytes != 8) || entries < 0)
    return CVHRF_EINVAL;
  if (entries > kGroupMaxEntries) return CVHRF_EUNSUPPORTED;
  if (rows == 0) return CVHRF_OK;
  if (!grad_table || (entries > 0 && (!grad || !index))) return CVHRF_EINVAL;
  cudaStream_t st = (cudaStream_t)stream;
  const size_t elem = row_type_bytes(dtype);
  if (entries == 0) {
    CVHRF_CUDA_TRY(cudaMemsetAsync(grad_table, 0, (size_t)rows * width * elem, st));
    if (row_mask) CVHRF_CUDA_TRY(cudaMemsetAsync(row_mask, 0, (size_t)rows, st));
    return CVHRF_OK;
  }
  if (few(entries, rows, width)) {
    if (dtype == CVHRF_F32)
      return few_entries<float>(grad, grad_stride, width, index, index_bytes, entries, rows, scale, grad_table,
                                row_mask, st);
    if (dtype == CVHRF_BF16)
      return few_entries<__nv_bfloat16>(grad, grad_stride, width, index, index_bytes, entries, rows, scale,
                                        grad_table, row_mask, st);
    return few_entries<__half>(grad, grad_stride, width, index, index_bytes, entries, rows, scale, grad_table,
                               row_mask, st);
  }
  if (!workspace || workspace_bytes < cvhrf_table_gradient_workspace_bytes(entries, rows, width))
    return CVHRF_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return CVHRF_EINVAL;
  if (small_table(rows, width)) {
    if (dtype == CVHRF_F32)
      return small_gradient<float>(grad, grad_stride, width, index, index_bytes, entries, rows, scale, grad_table,
                                   row_mask, workspace, st);
    if (dtype == CVHRF_BF16)
      return small_gradient<__nv_bfloat16>(grad, grad_stride, width, index, index_bytes, entries, rows, scale,
                                           grad_table, row_mask, workspace, st);
    return small_gradient<__half>(grad, grad_stride, width, index, index_bytes, entries, rows, scale, grad_table,
                                  row_mask, workspace, st);
  }
  uint32_t* scratch = (uint32_t*)workspace;
  const uint32_t *keys, *sorted, *count;
  char* after = (char*)workspace + align_up(group_sort_words(entries) * sizeof(uint32_t), 256);
  uint8_t* touched = row_mask ? row_mask : (uint8_t*)after;
  float* joins = (float*)(after + align_up((size_t)rows, 256));
  const int rc = group_sort(index, index_bytes, entries, rows, false, scratch, touched, st, &keys, &sorted, &count);
  if (rc) return rc;
  if (dtype == CVHRF_F32)
    return gradient<float>(grad, grad_stride, width, entries, rows, scale, grad_table, touched, keys, sorted, count,
                           joins, st);
  if (dtype == CVHRF_BF16)
    return gradient<__nv_bfloat16>(grad, grad_stride, width, entries, rows, scale, grad_table, touched, keys, sorted,
                                   count, joins, st);
  return gradient<__half>(grad, grad_stride, width, entries, rows, scale, grad_table, touched, keys, sorted, count,
                          joins, st);
}
