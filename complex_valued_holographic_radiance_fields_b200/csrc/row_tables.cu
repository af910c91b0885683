// Rows of a table that many entries share: cvhrf_table_lookup and cvhrf_table_gradient.
//
//   lookup    out[t] = scale * table[index[t]]                        (a row of zeros where index[t] is outside)
//   gradient  grad_table[v] = scale * sum_{t : index[t] = v} grad[t]  (fp32, entries in order), row_mask[v] = any
//
// Both are bound by memory: the lookup reads the distinct rows and writes T rows; the
// gradient reads T rows and writes V.
//
// The gradient sorts the entries by row (row_groups.cu) and merges the sorted list with the
// list of row ends 0 .. V-1: an item is either an entry (add its row) or a row end (write the
// sum, zeros for a row without entries, and start the next).  Every unit of lanes takes an
// equal share of the T + V items, found by one binary search on its diagonal of the merge, so
// neither a row with very many entries nor a long stretch of rows with none holds up a block,
// and the table is written once without being cleared first.  A row whose entries lie in
// several units is joined in the order of the units: inside a block through shared memory,
// between blocks by table_join_kernel.  The order of every sum is fixed, so results repeat.
#include "row_groups.cuh"
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
    for (int c = o.lane * R::kVec; c < width; c += step * J) {
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
template <typename T, bool WIDE, int ROWS, int J>
__global__ void __launch_bounds__(kTileThreads) table_lookup_tile_kernel(const T* __restrict__ table, long long rows,
                                                                         int width, long long stride,
                                                                         const void* __restrict__ index,
                                                                         int index_bytes, long long entries, int tile,
                                                                         float scale, T* __restrict__ out) {
  gather_tile<T, true, WIDE, ROWS, J>(
      [&](long long t) -> const T* {
        const long long v = table_row(index, index_bytes, t, rows);
        return v >= 0 ? table + v * stride : nullptr;
      },
      entries, tile, width, scale, out);
}

template <typename T, bool WIDE, int ROWS, int J>
int launch_lookup_tile(const void* table, long long rows, int width, long long stride, const void* index,
                       int index_bytes, long long entries, float scale, void* out, cudaStream_t st) {
  const int tile = tile_rows(entries, width, sizeof(T));
  table_lookup_tile_kernel<T, WIDE, ROWS, J>
      <<<(unsigned)((entries + tile - 1) / tile), kTileThreads, (size_t)tile * width * sizeof(T), st>>>(
          (const T*)table, rows, width, stride, index, index_bytes, entries, tile, scale, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
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
  table_lookup_words_kernel<T, LANES, FLIGHT, J><<<word_blocks(entries, rounds, owners), kWordThreads, 0, st>>>(
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
  table_lookup_kernel<T, ROWS, J><<<(unsigned)(blocks < most ? blocks : most), kThreads, 0, st>>>(
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
#define CVHRF_LOOKUP_TILE(WIDE, ROWS, J) \
  launch_lookup_tile<T, WIDE, ROWS, J>(table, rows, width, stride, index, index_bytes, entries, scale, out, st)
    if (width > 128) return CVHRF_LOOKUP_TILE(true, 1, 8);
    if (width > 64) return CVHRF_LOOKUP_TILE(false, 2, 4);
    if (width > 32) return CVHRF_LOOKUP_TILE(false, 4, 2);
    return CVHRF_LOOKUP_TILE(false, 8, 1);
#undef CVHRF_LOOKUP_TILE
  }
  const int words = words_of<T>(width);
  if (words > 64)
    return launch_lookup_words<T, 32, 2, 4>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  if (words >= 32)
    return launch_lookup_words<T, 32, 4, 2>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  return launch_lookup_words<T, 0, 4, 1>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
}

// ---- gradient -------------------------------------------------------------------------
constexpr int kBlockItems = 2048;   // most items of a block: its entries are staged in shared memory

// What a block leaves for table_join_kernel: the part of a row that began in an earlier
// block and ends in this one (head), and of the row that is open at its end (tail).
struct Joins {
  float* head;        // block x width
  float* tail;        // block x width
  int* head_row;      // -1: none
  int* tail_row;      // -1: none
  int* tail_begun;    // the open row's first entry is in this block
};

struct Gradient {
  const uint32_t* keys;      // sorted rows
  const uint32_t* entries;   // the entry of each
  const uint32_t* count;     // how many
  long long stride;          // elements between the rows of grad
  int rows, width;
  int lanes, units;          // lanes of a unit (up to 32), units of a block
  int items;                 // items of a unit
  float scale;
  uint8_t* mask;             // may be null
};

// Entries among the first d items of the merge: entry i comes before row end j iff keys[i] <= j,
// so it is the first i with keys[i] > d - 1 - i.  32 probes at a time; the whole warp calls it.
__device__ __forceinline__ uint32_t entries_before(const uint32_t* __restrict__ keys, uint32_t n, uint32_t rows,
                                                   long long d) {
  long long lo = d > rows ? d - rows : 0, hi = d < n ? d : n;
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const long long step = (hi - lo + 31) >> 5, at = lo + (lane + 1) * step - 1;
    const bool before = at < hi && (long long)keys[at] <= d - 1 - at;
    const int whole = __popc(__ballot_sync(0xffffffffu, before));
    const long long next = lo + (whole + 1) * step - 1;
    lo += whole * step;
    hi = next < hi ? next : hi;
  }
  return (uint32_t)lo;
}

template <int VEC>
constexpr size_t gradient_shared() {   // staged entries, heads and tails (units x lanes = kThreads), their rows
  return kBlockItems * 2 * sizeof(uint32_t) + 2 * kThreads * VEC * sizeof(float) + 3 * kThreads * sizeof(int);
}

// Units of `lanes` lanes; a lane holds one pack of columns; blockIdx.y: column tile.
template <typename T, Layout L>
__global__ void __launch_bounds__(kThreads, 4) table_gradient_kernel(Gradient g, const T* __restrict__ grad, Extent extent,
                                                                  T* __restrict__ out, Joins joins) {
  using R = Row<T, L>;
  constexpr int VEC = R::kVec;
  constexpr int kBatch = L == kSpan ? 4 : 8;   // rows of grad in flight per unit
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint32_t s_bound[2];
  const int lanes = g.lanes, units = g.units;
  const int unit = threadIdx.x / lanes, lane = threadIdx.x - unit * lanes;
  const bool live = unit < units;   // a few threads are left over where the lanes do not divide them
  const int tile_width = lanes * VEC;
  uint32_t* keys = reinterpret_cast<uint32_t*>(raw);
  uint32_t* entries = keys + kBlockItems;
  float* heads = reinterpret_cast<float*>(entries + kBlockItems);   // units x tile_width
  float* tails = heads + kThreads * VEC;
  int* head_row = reinterpret_cast<int*>(tails + kThreads * VEC);
  int* tail_row = head_row + kThreads;
  int* tail_begun = tail_row + kThreads;
  follow();
  let_next_start();
  const uint32_t n = *g.count;
  const long long total = (long long)n + g.rows;
  // the block's share of the merge, its entries brought into shared memory
  const long long block_items = (long long)units * g.items;
  const long long b0 = min((long long)blockIdx.x * block_items, total), b1 = min(b0 + block_items, total);
  if (threadIdx.x < 64) {
    const uint32_t p = entries_before(g.keys, n, g.rows, threadIdx.x < 32 ? b0 : b1);
    if ((threadIdx.x & 31) == 0) s_bound[threadIdx.x >> 5] = p;
  }
  __syncthreads();
  const uint32_t first = s_bound[0], last = s_bound[1];
  const uint32_t before_first = first > 0 ? g.keys[first - 1] : 0xffffffffu;
  for (uint32_t i = threadIdx.x; i < last - first; i += kThreads) {
    keys[i] = g.keys[first + i];
    entries[i] = g.entries[first + i];
  }
  __syncthreads();
  // the unit's share, places counted from `first`
  const long long d0 = live ? min(b0 + (long long)unit * g.items, b1) : b1, d1 = min(d0 + g.items, b1);
  uint32_t p0, p1;
  {
    auto search = [&](long long d) {
      long long lo = max(d - g.rows, (long long)first) - first, hi = min(d, (long long)last) - first;
      while (lo < hi) {
        const long long mid = (lo + hi) >> 1;
        if ((long long)keys[mid] <= d - 1 - mid - first) lo = mid + 1;
        else hi = mid;
      }
      return (uint32_t)lo;
    };
    p0 = search(d0);
    p1 = search(d1);
  }
  uint32_t r = (uint32_t)(d0 - first - p0);
  const uint32_t r1 = (uint32_t)(d1 - first - p1);
  // whether row r has entries in earlier units
  bool begun_before = d0 < d1 && (p0 > 0 ? keys[p0 - 1] : before_first) == r;
  // the lane's first column; a last pack that would end behind the row is moved back into it
  // (its first columns are then the lane's before, added up twice and written twice, alike)
  const int first_col = blockIdx.y * tile_width + lane * VEC;
  const bool in = live && first_col < g.width;
  const int col = L == kSpan ? min(first_col, g.width - VEC) : first_col;
  float acc[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
  bool any = false;
  int my_head = -1;
  float* my_heads = heads + unit * tile_width + lane * VEC;
  float* my_tails = tails + unit * tile_width + lane * VEC;
  auto write = [&](uint32_t row, float (&sum)[VEC]) {   // columns of a row that may begin anywhere
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] *= g.scale;
    if (!in) return;
    T* to = out + (long long)row * g.width + col;
    if (L == kSpan && ((uintptr_t)to & 15)) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) to[i] = from_float<T>(sum[i]);
    } else {
      R::store(to, R::words(sum));
    }
  };

  auto end_row = [&]() {
    if (begun_before) {   // its other entries are elsewhere: leave the sum for the join
      my_head = (int)r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) my_heads[i] = acc[i];
    } else {
      if (any || L != kSpan) {
        write(r, acc);
      } else if (r % gridDim.y == blockIdx.y) {   // the tiles share the rows without entries
        clear_row<T, L>(out + (long long)r * g.width, g.width, lane, lanes);
      }
      if (g.mask && lane == 0 && blockIdx.y == 0) g.mask[r] = any;
    }
    begun_before = false;
    any = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    ++r;
  };

  // the rows of the next batches are called into L2 ahead of their loads, which costs no registers
  const int tile_bytes = (int)sizeof(T) * min(tile_width, g.width - (int)blockIdx.y * tile_width);
  const int lines = (tile_bytes + 127) / 128 + (L == kAligned ? 0 : 1);
  auto call = [&](uint32_t from) {
    for (int i = lane; i < kBatch * lines; i += lanes) {
      const int b = i / lines, at = min((i - b * lines) * 128, tile_bytes - (int)sizeof(T));
      if (from + b < p1)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(
            grad + (long long)entries[from + b] * g.stride + blockIdx.y * tile_width) + at));
    }
  };
  if (live) call(p0 + kBatch);
  for (uint32_t p = p0; p < p1; p += kBatch) {
    if (live) call(p + 2 * kBatch);
    typename R::Raw v[kBatch];
    auto load = [&](auto read) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (p + b < p1 && in) v[b] = read(grad + (long long)entries[p + b] * g.stride + col);
    };
    bool inside = true;
    if (L == kSpan && extent.checked) {
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (p + b < p1) inside = inside && extent.inside(grad + (long long)entries[p + b] * g.stride, g.width);
    }
    if (L != kSpan || inside) load([](const T* at) { return R::load(at); });
    else load([](const T* at) { return R::load_elements(at); });
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) {
        const uint32_t key = keys[p + b];
        while (r < key) end_row();
        if (in) {
          float f[VEC];
          R::floats(v[b], f);
#pragma unroll
          for (int i = 0; i < VEC; ++i) acc[i] += f[i];
        }
        any = true;
      }
  }
  while (r < r1) end_row();

  // the row that is open at the unit's end
  const bool open = any || begun_before;
  if (open) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) my_tails[i] = acc[i];
  }
  if (live && lane == 0) {
    head_row[unit] = my_head;
    tail_row[unit] = open ? (int)r : -1;
    tail_begun[unit] = open && !begun_before;
  }
  __syncthreads();
  // a row that ends in this unit and began in an earlier one: add the tails before it
  bool unfinished = false;
  if (my_head >= 0) {
    float sum[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sum[i] = my_heads[i];
    bool whole = false;
    for (int q = unit - 1; q >= 0 && !whole; --q) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] += tails[q * tile_width + lane * VEC + i];
      whole = tail_begun[q];
    }
    if (whole) {
      write((uint32_t)my_head, sum);
      if (g.mask && lane == 0 && blockIdx.y == 0) g.mask[my_head] = 1;
    } else {   // it began before this block
      unfinished = true;
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (in) joins.head[(long long)blockIdx.x * g.width + col + i] = sum[i];
      if (lane == 0 && blockIdx.y == 0) joins.head_row[blockIdx.x] = my_head;
    }
  }
  const int block_head = __syncthreads_or(unfinished);
  if (!block_head && threadIdx.x == 0 && blockIdx.y == 0) joins.head_row[blockIdx.x] = -1;
  // the row that is open at the block's end
  if (unit == units - 1) {
    const int row = tail_row[unit];
    bool begun = false;
    if (row >= 0) {
      float sum[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] = 0.f;
      for (int q = unit; q >= 0 && !begun; --q) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[i] += tails[q * tile_width + lane * VEC + i];
        begun = tail_begun[q];
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (in) joins.tail[(long long)blockIdx.x * g.width + col + i] = sum[i];
    }
    if (lane == 0 && blockIdx.y == 0) {
      joins.tail_row[blockIdx.x] = row;
      joins.tail_begun[blockIdx.x] = begun;
    }
  }
}

// Rows whose entries lie in several blocks: block x's head plus the tails before it, the
// blocks shared between `slices` threads of a column and then added in the slices' order.
template <typename T>
__global__ void __launch_bounds__(kThreads) table_join_kernel(Joins joins, int width, int columns, float scale,
                                                              T* __restrict__ out, uint8_t* __restrict__ mask) {
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
    if (mask && c == 0) mask[row] = 1;
  }
}

constexpr int kMinItems = 8;        // items of a unit at least, or the searches outweigh the rows

// Most blocks a gradient can have (x dimension): its joins' rows.
inline long long most_blocks(long long n, long long rows) {
  const long long total = n + rows, fewest = 8 * kMinItems;   // 8 units at least in a block
  constexpr long long share = kBlockItems - kThreads;       // of a block whose units do not divide kBlockItems
  const long long full = (total + share - 1) / share + 148 * 8;
  const long long tiny = (total + fewest - 1) / fewest;
  return full < tiny ? full : tiny;
}

template <typename T, Layout L>
int launch_gradient(Gradient g, long long n, const void* grad, void* out, float* joins_at, cudaStream_t st) {
  constexpr int VEC = Row<T, L>::kVec;
  constexpr size_t shared = gradient_shared<VEC>();
  static_assert(shared <= 48 * 1024, "the default limit of shared memory");
  static const int resident = [] {
    int blocks = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, table_gradient_kernel<T, L>, kThreads, shared);
    return e == cudaSuccess && blocks > 0 ? (blocks < 8 ? blocks : 8) : 2;
  }();
  const int packs = (g.width + VEC - 1) / VEC;
  g.lanes = packs < 32 ? packs : 32;
  const int units = g.units = kThreads / g.lanes, tile_width = g.lanes * VEC;
  const int tiles = (g.width + tile_width - 1) / tile_width;
  // equal blocks that fill the SMs a whole number of times
  const long long total = n + g.rows;
  long long slots = 148 * resident / tiles;
  if (slots < 1) slots = 1;
  const long long waves = (total + slots * kBlockItems - 1) / (slots * kBlockItems);
  long long items = (total + slots * waves * units - 1) / (slots * waves * units);
  if (items < kMinItems) items = kMinItems;
  if (items * units > kBlockItems) items = kBlockItems / units;
  g.items = (int)items;
  const long long blocks = (total + items * units - 1) / (items * units);
  Joins joins;
  joins.head = joins_at;
  joins.tail = joins.head + blocks * g.width;
  joins.head_row = (int*)(joins.tail + blocks * g.width);
  joins.tail_row = joins.head_row + blocks;
  joins.tail_begun = joins.tail_row + blocks;
  CVHRF_CUDA_TRY(launch_after(table_gradient_kernel<T, L>, dim3((unsigned)blocks, tiles), kThreads, shared, st, g,
                              (const T*)grad, extent_of(grad, n, g.stride, g.width, sizeof(T)), (T*)out, joins));
  count_launch(1);
  if (blocks == 1) return CVHRF_OK;
  const int columns = next_pow2(g.width < kThreads ? g.width : kThreads);
  CVHRF_CUDA_TRY(launch_after(table_join_kernel<T>, dim3((unsigned)blocks, (g.width + columns - 1) / columns), kThreads,
                              0, st, joins, g.width, columns, g.scale, (T*)out, g.mask));
  count_launch(1);
  return CVHRF_OK;
}

// Units of as many lanes as a row has packs, a warp at most; wider rows are cut into tiles.
template <typename T>
int gradient(const void* grad, long long stride, int width, long long n, long long rows, float scale, void* out,
             uint8_t* mask, const uint32_t* keys, const uint32_t* entries, const uint32_t* count, float* joins,
             cudaStream_t st) {
  const Gradient g{keys, entries, count, stride, (int)rows, width, 0, 0, 0, scale, mask};
  if (rows_16(grad, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0)
    return launch_gradient<T, kAligned>(g, n, grad, out, joins, st);
  if (width >= kSpanWidth) return launch_gradient<T, kSpan>(g, n, grad, out, joins, st);
  return launch_gradient<T, kElement>(g, n, grad, out, joins, st);
}

constexpr long long kMaxRows = 0x7ffffffe;
constexpr int kMaxWidth = 1 << 20;

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
  return align_up(group_sort_words(entries) * sizeof(uint32_t), 256) +
         (size_t)most_blocks(entries, rows) * (2 * (size_t)width * sizeof(float) + 3 * sizeof(int));
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
  if (!workspace || workspace_bytes < cvhrf_table_gradient_workspace_bytes(entries, rows, width))
    return CVHRF_EWORKSPACE;
  if ((uintptr_t)workspace & 15) return CVHRF_EINVAL;
  uint32_t* scratch = (uint32_t*)workspace;
  const uint32_t *keys, *sorted, *count;
  const int rc = group_sort(index, index_bytes, entries, rows, false, scratch, st, &keys, &sorted, &count);
  if (rc) return rc;
  float* joins = (float*)((char*)workspace + align_up(group_sort_words(entries) * sizeof(uint32_t), 256));
  if (dtype == CVHRF_F32)
    return gradient<float>(grad, grad_stride, width, entries, rows, scale, grad_table, row_mask, keys, sorted, count,
                           joins, st);
  if (dtype == CVHRF_BF16)
    return gradient<__nv_bfloat16>(grad, grad_stride, width, entries, rows, scale, grad_table, row_mask, keys, sorted,
                                   count, joins, st);
  return gradient<__half>(grad, grad_stride, width, entries, rows, scale, grad_table, row_mask, keys, sorted, count,
                          joins, st);
}
