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

namespace cvhrf {
namespace {

constexpr int kThreads = 256;

// ---- lookup ---------------------------------------------------------------------------
__device__ __forceinline__ long long table_row(const void* index, int bytes, long long t, long long rows) {
  const long long v = bytes == 4 ? (long long)((const int*)index)[t] : ((const long long*)index)[t];
  return (unsigned long long)v < (unsigned long long)rows ? v : -1;
}

// A row is owned by a power of two of lanes, up to a warp.  An owner has ROWS rows in flight
// (J packs of each at a time), the owners of a block neighbouring rows; blocks walk over the
// entries, and the indices of the next rows are read while these rows are on their way:
// without that a row waits for two trips to memory, one after the other.
template <typename T, Layout L, int ROWS, int J>
__global__ void __launch_bounds__(kThreads, 4) table_lookup_kernel(const T* __restrict__ table, Extent extent,
                                                                   long long rows, int width, long long stride,
                                                                   const void* __restrict__ index, int index_bytes,
                                                                   long long entries, int lanes, float scale,
                                                                   T* __restrict__ out) {
  using R = Row<T, L>;
  const int owners = kThreads / lanes, lane = threadIdx.x & (lanes - 1), step = lanes * R::kVec;
  const long long walk = (long long)gridDim.x * owners * ROWS;
  long long first = (long long)blockIdx.x * (owners * ROWS) + threadIdx.x / lanes;
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
    T* to[ROWS];
    int e0[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      from[k] = v[k] >= 0 ? table + v[k] * stride : nullptr;
      to[k] = out + (first + k * owners) * width;
      e0[k] = lane * R::kVec - R::ahead(to[k]);
    }
    bool next = true;
    for (int c = 0; c - (L == kSpan ? R::kVec - 1 : 0) < width; c += step * J) {
      typename R::Raw p[ROWS][J];
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (from[k] && e0[k] + c + j * step < width) p[k][j] = R::load(from[k], e0[k] + c + j * step, width, extent);
      if (next) load_index(first + walk);
      next = false;
#pragma unroll
      for (int k = 0; k < ROWS; ++k)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (first + k * owners < entries && e0[k] + c + j * step < width) {
            if (from[k]) {
              float f[R::kVec];
              R::floats(p[k][j], f);
#pragma unroll
              for (int i = 0; i < R::kVec; ++i) f[i] *= scale;
              R::store(to[k], e0[k] + c + j * step, width, R::words(f));
            } else {
              R::store(to[k], e0[k] + c + j * step, width, zero_pack<T, L>());
            }
          }
    }
  }
}

template <typename T, Layout L, int ROWS, int J>
int launch_lookup(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
                  long long entries, int lanes, float scale, void* out, cudaStream_t st) {
  static const int resident = [] {
    int blocks = 0;
    const cudaError_t e =
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, table_lookup_kernel<T, L, ROWS, J>, kThreads, 0);
    return e == cudaSuccess && blocks > 0 ? blocks : 4;
  }();
  const long long per_block = kThreads / lanes * ROWS, blocks = (entries + per_block - 1) / per_block;
  const long long most = 148 * resident;
  table_lookup_kernel<T, L, ROWS, J><<<(unsigned)(blocks < most ? blocks : most), kThreads, 0, st>>>(
      (const T*)table, extent_of(table, rows, stride, width, sizeof(T)), rows, width, stride, index, index_bytes,
      entries, lanes, scale, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T, Layout L>
int lookup_rows(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
                long long entries, float scale, void* out, cudaStream_t st) {
  const int packs = packs_of<T, L>(width), lanes = next_pow2(packs < 32 ? packs : 32);
  if constexpr (L == kSpan) {   // twice the registers per pack
    if (packs > 32)
      return launch_lookup<T, L, 1, 2>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
    return launch_lookup<T, L, 2, 1>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
  } else {
    if (packs > 64)
      return launch_lookup<T, L, 1, 4>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
    if (packs > 32)
      return launch_lookup<T, L, 2, 2>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
    return launch_lookup<T, L, 4, 1>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out, st);
  }
}

template <typename T>
int lookup(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
           long long entries, float scale, void* out, cudaStream_t st) {
  if (rows_16(table, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0)
    return lookup_rows<T, kAligned>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  if (width >= kSpanWidth)
    return lookup_rows<T, kSpan>(table, rows, width, stride, index, index_bytes, entries, scale, out, st);
  // rows of one element per lane: a warp's worth of lanes at most, so one step
  const int lanes = next_pow2(width);
  return launch_lookup<T, kElement, 4, 1>(table, rows, width, stride, index, index_bytes, entries, lanes, scale, out,
                                          st);
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
  int lanes;                 // lanes of a unit (a power of two up to 32)
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
__global__ void __launch_bounds__(kThreads) table_gradient_kernel(Gradient g, const T* __restrict__ grad, Extent extent,
                                                                  T* __restrict__ out, Joins joins) {
  using R = Row<T, L>;
  constexpr int VEC = R::kVec;
  constexpr int kBatch = L == kSpan ? 4 : 8;   // rows of grad in flight per unit
  extern __shared__ __align__(16) unsigned char raw[];
  __shared__ uint32_t s_bound[2];
  const int lanes = g.lanes, units = kThreads / lanes;
  const int unit = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  const int tile_width = lanes * VEC;
  uint32_t* keys = reinterpret_cast<uint32_t*>(raw);
  uint32_t* entries = keys + kBlockItems;
  float* heads = reinterpret_cast<float*>(entries + kBlockItems);   // units x tile_width
  float* tails = heads + kThreads * VEC;
  int* head_row = reinterpret_cast<int*>(tails + kThreads * VEC);
  int* tail_row = head_row + kThreads;
  int* tail_begun = tail_row + kThreads;
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
  const long long d0 = min(b0 + (long long)unit * g.items, b1), d1 = min(d0 + g.items, b1);
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
  const int col = blockIdx.y * tile_width + lane * VEC;   // the lane's first column
  const bool in = col < g.width;
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
    T* to = out + (long long)row * g.width;
    if (in) {
      if (L == kSpan && R::ahead(to) != 0) R::store_by_element(to, col, g.width, R::words(sum));
      else R::store(to, col, g.width, R::words(sum));
    }
  };

  auto end_row = [&]() {
    if (begun_before) {   // its other entries are elsewhere: leave the sum for the join
      my_head = (int)r;
#pragma unroll
      for (int i = 0; i < VEC; ++i) my_heads[i] = acc[i];
    } else {
      if (any) {
        write(r, acc);
      } else {
        // zeros may be shifted: whole packs wherever the row begins, one more at its end
        T* to = out + (long long)r * g.width;
        const int e = col - R::ahead(to);
        if (e < g.width) R::store(to, e, g.width, zero_pack<T, L>());
        if (L == kSpan && lane == lanes - 1 && blockIdx.y + 1 == gridDim.y && e + VEC < g.width)
          R::store(to, e + VEC, g.width, zero_pack<T, L>());
      }
      if (g.mask && lane == 0 && blockIdx.y == 0) g.mask[r] = any;
    }
    begun_before = false;
    any = false;
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
    ++r;
  };

  for (uint32_t p = p0; p < p1; p += kBatch) {
    typename R::Raw v[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1 && in) v[b] = R::load(grad + (long long)entries[p + b] * g.stride, col, g.width, extent);
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
  if (lane == 0) {
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
        if (col + i < g.width) joins.head[(long long)blockIdx.x * g.width + col + i] = sum[i];
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
        if (col + i < g.width) joins.tail[(long long)blockIdx.x * g.width + col + i] = sum[i];
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
  const long long full = (total + kBlockItems - 1) / kBlockItems + 148 * 8;
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
  g.lanes = next_pow2(packs < 32 ? packs : 32);
  const int units = kThreads / g.lanes, tile_width = g.lanes * VEC;
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
  table_gradient_kernel<T, L><<<dim3((unsigned)blocks, tiles), kThreads, shared, st>>>(
      g, (const T*)grad, extent_of(grad, n, g.stride, g.width, sizeof(T)), (T*)out, joins);
  CVHRF_LAUNCH_CHECK();
  if (blocks == 1) return CVHRF_OK;
  const int columns = next_pow2(g.width < kThreads ? g.width : kThreads);
  table_join_kernel<T><<<dim3((unsigned)blocks, (g.width + columns - 1) / columns), kThreads, 0, st>>>(
      joins, g.width, columns, g.scale, (T*)out, g.mask);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

// Units of the smallest power of two of lanes that holds a row, a warp at most; wider rows are
// cut into tiles.
template <typename T>
int gradient(const void* grad, long long stride, int width, long long n, long long rows, float scale, void* out,
             uint8_t* mask, const uint32_t* keys, const uint32_t* entries, const uint32_t* count, float* joins,
             cudaStream_t st) {
  const Gradient g{keys, entries, count, stride, (int)rows, width, 0, 0, scale, mask};
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

extern "C" int cvhrf_table_lookup(const void* table, long long rows, int width, long long row_stride, int dtype,
                                  const void* index, int index_bytes, long long entries, float scale, void* out,
                                  void* stream) {
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

extern "C" int cvhrf_table_gradient(const void* grad, long long grad_stride, int dtype, int width, const void* index,
                                    int index_bytes, long long entries, float scale, void* grad_table, long long rows,
                                    uint8_t* row_mask, void* workspace, size_t workspace_bytes, void* stream) {
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
