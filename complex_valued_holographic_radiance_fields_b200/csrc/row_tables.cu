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

// One pack per thread and step; kSteps rows in flight per thread.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) table_lookup_kernel(const T* __restrict__ table, long long rows, int packs,
                                                                long long stride, const void* __restrict__ index,
                                                                int index_bytes, long long total, float scale,
                                                                T* __restrict__ out) {
  constexpr int kSteps = 4;
  const long long base = (long long)blockIdx.x * (kThreads * kSteps) + threadIdx.x;
  Pack<T, VEC> p[kSteps];
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long e = base + s * kThreads;
    if (e < total) {
      const long long t = e / packs;
      const int c = (int)(e - t * packs);
      const long long v = table_row(index, index_bytes, t, rows);
      if (v >= 0) {
        p[s] = *(const Pack<T, VEC>*)(table + v * stride + (long long)c * VEC);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p[s].v[i] = from_float<T>(0.f);
      }
    }
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    const long long e = base + s * kThreads;
    if (e < total) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[s].v[i] = from_float<T>(scale * to_float(p[s].v[i]));
      *(Pack<T, VEC>*)(out + e * VEC) = p[s];
    }
  }
}

template <typename T>
int lookup(const void* table, long long rows, int width, long long stride, const void* index, int index_bytes,
           long long entries, float scale, void* out, cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const bool wide = rows_16(table, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0;
  const int packs = wide ? width / kVec : width;
  const long long total = entries * packs, blocks = (total + kThreads * 4 - 1) / (kThreads * 4);
  if (blocks > 0x7fffffff) return CVHRF_EUNSUPPORTED;
  if (wide)
    table_lookup_kernel<T, kVec><<<(unsigned)blocks, kThreads, 0, st>>>((const T*)table, rows, packs, stride, index,
                                                                        index_bytes, total, scale, (T*)out);
  else
    table_lookup_kernel<T, 1><<<(unsigned)blocks, kThreads, 0, st>>>((const T*)table, rows, packs, stride, index,
                                                                     index_bytes, total, scale, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

// ---- gradient -------------------------------------------------------------------------
constexpr int kMaxBlocks = 148 * 8;

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

// Entries among the first d items of the merge.
__device__ __forceinline__ uint32_t entries_before(const uint32_t* __restrict__ keys, uint32_t n, uint32_t rows,
                                                   long long d) {
  long long lo = d > rows ? d - rows : 0, hi = d < n ? d : n;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if ((long long)keys[mid] <= d - 1 - mid) lo = mid + 1;
    else hi = mid;
  }
  return (uint32_t)lo;
}

template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* __restrict__ to, const float* acc, float scale) {
  Pack<T, VEC> p;
#pragma unroll
  for (int i = 0; i < VEC; ++i) p.v[i] = from_float<T>(scale * acc[i]);
  *(Pack<T, VEC>*)to = p;
}

// Units of `lanes` lanes; a lane holds J packs of VEC columns; blockIdx.y: column tile.
template <typename T, int VEC, int J>
__global__ void __launch_bounds__(kThreads) table_gradient_kernel(Gradient g, const T* __restrict__ grad,
                                                                  T* __restrict__ out, Joins joins) {
  constexpr int kBatch = 4;
  extern __shared__ float shared[];
  const int lanes = g.lanes, units = kThreads / lanes;
  const int unit = threadIdx.x / lanes, lane = threadIdx.x & (lanes - 1);
  const int tile_width = lanes * J * VEC;
  float* heads = shared;                          // units x tile_width
  float* tails = heads + units * tile_width;
  int* head_row = (int*)(tails + units * tile_width);
  int* tail_row = head_row + units;
  int* tail_begun = tail_row + units;
  const uint32_t n = *g.count;
  const long long total = (long long)n + g.rows;
  const long long first = ((long long)blockIdx.x * units + unit) * g.items;
  const long long d0 = first < total ? first : total, d1 = first + g.items < total ? first + g.items : total;
  const uint32_t p0 = entries_before(g.keys, n, g.rows, d0), p1 = entries_before(g.keys, n, g.rows, d1);
  uint32_t r = (uint32_t)(d0 - p0);
  const uint32_t r1 = (uint32_t)(d1 - p1);
  bool begun_before = d0 < d1 && p0 > 0 && g.keys[p0 - 1] == r;   // row r has entries in earlier units
  int col[J];
  bool in[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    col[j] = blockIdx.y * tile_width + (j * lanes + lane) * VEC;
    in[j] = col[j] < g.width;
  }
  float acc[J][VEC];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[j][i] = 0.f;
  bool any = false;
  int my_head = -1;

  auto end_row = [&]() {
    if (begun_before) {   // its other entries are elsewhere: leave the sum for the join
      my_head = (int)r;
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) heads[unit * tile_width + (j * lanes + lane) * VEC + i] = acc[j][i];
    } else {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (in[j]) write_row<T, VEC>(out + (long long)r * g.width + col[j], acc[j], g.scale);
      if (g.mask && lane == 0 && blockIdx.y == 0) g.mask[r] = any;
    }
    begun_before = false;
    any = false;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[j][i] = 0.f;
    ++r;
  };

  for (uint32_t p = p0; p < p1; p += kBatch) {
    Pack<T, VEC> v[kBatch][J];
    uint32_t key[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) {
        key[b] = g.keys[p + b];
        const T* row = grad + (long long)g.entries[p + b] * g.stride;
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (in[j]) v[b][j] = *(const Pack<T, VEC>*)(row + col[j]);
      }
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (p + b < p1) {
        while (r < key[b]) end_row();
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (in[j])
#pragma unroll
            for (int i = 0; i < VEC; ++i) acc[j][i] += to_float(v[b][j].v[i]);
        any = true;
      }
  }
  while (r < r1) end_row();

  // the row that is open at the unit's end
  const bool open = any || begun_before;
  if (open)
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) tails[unit * tile_width + (j * lanes + lane) * VEC + i] = acc[j][i];
  if (lane == 0) {
    head_row[unit] = my_head;
    tail_row[unit] = open ? (int)r : -1;
    tail_begun[unit] = open && !begun_before;
  }
  __syncthreads();
  // rows that end in this unit and began in an earlier one: add the tails before it
  if (my_head >= 0) {
    int q = unit - 1;
    bool whole = false;
    while (q >= 0 && !whole) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const int at = (j * lanes + lane) * VEC + i;
          heads[unit * tile_width + at] += tails[q * tile_width + at];
        }
      whole = tail_begun[q];
      --q;
    }
    float sum[J][VEC];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[j][i] = heads[unit * tile_width + (j * lanes + lane) * VEC + i];
    if (whole) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (in[j]) write_row<T, VEC>(out + (long long)my_head * g.width + col[j], sum[j], g.scale);
      if (g.mask && lane == 0 && blockIdx.y == 0) g.mask[my_head] = 1;
    } else {   // it began before this block
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (in[j])
#pragma unroll
          for (int i = 0; i < VEC; ++i) joins.head[(long long)blockIdx.x * g.width + col[j] + i] = sum[j][i];
      if (lane == 0 && blockIdx.y == 0) joins.head_row[blockIdx.x] = my_head;
    }
    my_head = whole ? -1 : my_head;
  }
  const int block_head = __syncthreads_or(my_head >= 0);
  if (!block_head && threadIdx.x == 0 && blockIdx.y == 0) joins.head_row[blockIdx.x] = -1;
  // the row that is open at the block's end
  if (unit == units - 1) {
    const int row = tail_row[unit];
    bool begun = false;
    if (row >= 0) {
      float sum[J][VEC];
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) sum[j][i] = 0.f;
      for (int q = unit; q >= 0 && !begun; --q) {
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int i = 0; i < VEC; ++i) sum[j][i] += tails[q * tile_width + (j * lanes + lane) * VEC + i];
        begun = tail_begun[q];
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (in[j])
#pragma unroll
          for (int i = 0; i < VEC; ++i) joins.tail[(long long)blockIdx.x * g.width + col[j] + i] = sum[j][i];
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

struct Shape {
  int lanes, j, vec, tiles, blocks, items;
  size_t shared;
};

// Units of the smallest power of two of lanes that holds a row, a warp at most; wider rows
// take several packs per lane (16 columns at most, so that the joins fit 32 KB), then tiles.
inline Shape shape_for(long long n, long long rows, int width, int vec) {
  Shape s{};
  s.vec = vec;
  const int packs = (width + vec - 1) / vec;
  s.lanes = next_pow2(packs < 32 ? packs : 32);
  const int most = 16 / vec < 4 ? 16 / vec : 4;
  s.j = next_pow2((packs + s.lanes - 1) / s.lanes);
  if (s.j > most) s.j = most;
  s.tiles = (packs + s.lanes * s.j - 1) / (s.lanes * s.j);
  const int units = kThreads / s.lanes;
  const long long total = n + rows;
  long long items = 8;   // at least, or the searches outweigh the rows
  const long long even = (total + (long long)kMaxBlocks * units - 1) / ((long long)kMaxBlocks * units);
  if (items < even) items = even;
  s.items = (int)items;
  s.blocks = (int)((total + items * units - 1) / (items * units));
  s.shared = (size_t)units * (2 * s.lanes * s.j * vec * sizeof(float) + 3 * sizeof(int));
  return s;
}

template <typename T, int VEC, int J>
int launch_gradient(const Shape& s, const Gradient& g, const void* grad, void* out, const Joins& joins,
                    cudaStream_t st) {
  table_gradient_kernel<T, VEC, J><<<dim3(s.blocks, s.tiles), kThreads, s.shared, st>>>(g, (const T*)grad, (T*)out,
                                                                                       joins);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T, int VEC>
int launch_gradient_j(const Shape& s, const Gradient& g, const void* grad, void* out, const Joins& joins,
                      cudaStream_t st) {
  if (s.j == 1) return launch_gradient<T, VEC, 1>(s, g, grad, out, joins, st);
  if (s.j == 2) return launch_gradient<T, VEC, 2>(s, g, grad, out, joins, st);
  if constexpr (VEC * 4 <= 16) return launch_gradient<T, VEC, 4>(s, g, grad, out, joins, st);
  return CVHRF_EUNSUPPORTED;
}

template <typename T>
int gradient(const void* grad, long long stride, int width, long long n, long long rows, float scale, void* out,
             uint8_t* mask, const uint32_t* keys, const uint32_t* entries, const uint32_t* count, float* joins_at,
             cudaStream_t st) {
  constexpr int kVec = 16 / sizeof(T);
  const bool wide = rows_16(grad, stride, width, sizeof(T)) && ((uintptr_t)out & 15) == 0;
  const Shape s = shape_for(n, rows, width, wide ? kVec : 1);
  const Gradient g{keys, entries, count, stride, (int)rows, width, s.lanes, s.items, scale, mask};
  Joins joins;
  joins.head = joins_at;
  joins.tail = joins.head + (size_t)kMaxBlocks * width;
  joins.head_row = (int*)(joins.tail + (size_t)kMaxBlocks * width);
  joins.tail_row = joins.head_row + kMaxBlocks;
  joins.tail_begun = joins.tail_row + kMaxBlocks;
  const int rc = wide ? launch_gradient_j<T, kVec>(s, g, grad, out, joins, st)
                      : launch_gradient_j<T, 1>(s, g, grad, out, joins, st);
  if (rc || s.blocks == 1) return rc;
  const int columns = next_pow2(width < kThreads ? width : kThreads);
  table_join_kernel<T><<<dim3(s.blocks, (width + columns - 1) / columns), kThreads, 0, st>>>(joins, width, columns,
                                                                                            scale, (T*)out, mask);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
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
         (size_t)kMaxBlocks * (2 * (size_t)width * sizeof(float) + 3 * sizeof(int));
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
