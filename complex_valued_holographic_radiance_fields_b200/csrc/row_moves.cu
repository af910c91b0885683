// Rows taken to their groups and back: cvhrf_rows_to_groups, cvhrf_groups_to_rows and the
// gradient of the latter.  With slot[n, j] the place of row n's j-th choice (-1: left out):
//
//   to groups  out[slot[n, j]] = x[n]                                    (rows behind the last group: zeros)
//   to rows    out[n] = sum_j w[n, j] y[slot[n, j]]                      (fp32, in the order of j)
//   gradient   dy[slot[n, j]] = w[n, j] dout[n],  dw[n, j] = <dout[n], y[slot[n, j]]>
//
// (The gradient of "to groups" is "to rows" without weights.)  Aligned rows go by n: a row is
// owned by up to a warp of lanes that hold its columns, so a row of x or dout is read once however
// many groups it goes to, and no two owners write to one place.  Other rows go by the rows that
// are written, in tiles (row_tiles.cuh).
// Bound by memory: each touches N + N k rows once.  16384 rows of 2048 bf16 to 4 of 64 groups:
// 51 us there (6.6 TB/s), 60 back (5.6), 101 for the gradient (5.3, y read for dw).  100003 odd
// rows of 333 f16 to 2 of 7: 45, 57 and 87 us, where 2-byte loads are what is waited for.
#include <algorithm>
#include <type_traits>
#include "row_groups.cuh"
#include "row_tiles.cuh"
#include "row_types.cuh"

namespace cvhrf {
namespace {

constexpr int kThreads = 256;

struct Moves {
  long long n;          // rows
  int choices, width;
  int lanes, owners;    // lanes that own a row, owners in a block
  const int* slots;     // n x choices
  const int* used;      // (device) places that belong to a group; the rest is behind the last group
};

// Zeros into the rows behind the last group, shared out between the owners of the rows or the
// entries (owner x of `owners` takes every `owners`-th of them).
template <typename T, Layout L>
__device__ __forceinline__ void clear_behind(const Moves& m, int used, long long x, long long owners, int lane,
                                             T* __restrict__ out) {
  const long long places = m.n * m.choices;
  for (long long p = used + x; p < places; p += owners) clear_row<T, L>(out + p * m.width, m.width, lane, m.lanes);
}

// Aligned rows: an owner has ROWS rows (owners apart, so that the owners of a block touch
// neighbouring rows) with J packs of each in flight; each pack is read once and written once
// per choice.
template <typename T, int ROWS, int J>
__global__ void __launch_bounds__(kThreads) rows_to_groups_kernel(Moves m, const T* __restrict__ x, long long stride,
                                                                  T* __restrict__ out) {
  using R = Row<T, kAligned>;
  const Owner o = Owner::of(m.lanes);
  const int owners = m.owners, lane = o.lane, step = m.lanes * R::kVec;
  const long long first = (long long)blockIdx.x * (owners * ROWS) + o.index;
  if (!o.live) return;
  const int used = *m.used;
  for (int c0 = lane * R::kVec + (int)blockIdx.y * step * J; c0 < m.width; c0 += step * J * (int)gridDim.y) {
    uint4 p[ROWS][J];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (first + q * owners < m.n && c0 + j * step < m.width)
          p[q][j] = *(const uint4*)(x + (first + q * owners) * stride + c0 + j * step);
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long row = first + q * owners;
      if (row < m.n) {
#pragma unroll 4
        for (int i = 0; i < m.choices; ++i) {
          const int s = m.slots[row * m.choices + i];
          if (s < 0) continue;
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (c0 + j * step < m.width) *(uint4*)(out + (long long)s * m.width + c0 + j * step) = p[q][j];
        }
      }
    }
  }
#pragma unroll
  for (int q = 0; q < ROWS; ++q)
    if (first + q * owners < m.n && blockIdx.y == 0)
      clear_behind<T, kAligned>(m, used, first + q * owners, m.n, lane, out);
}

// Other rows: packs follow the row that is written, which begins elsewhere for every choice,
// so each owner copies ENTRIES entries (a row's choices are neighbours: its row is read from
// DRAM once).
template <typename T, Layout L, int ENTRIES>
__global__ void __launch_bounds__(kThreads) entries_to_groups_kernel(Moves m, const T* __restrict__ x, Extent extent,
                                                                     long long stride, T* __restrict__ out) {
  using R = Row<T, L>;
  const Owner o = Owner::of(m.lanes);
  const int owners = m.owners, lane = o.lane;
  const long long entries = m.n * m.choices;
  const long long first = (long long)blockIdx.x * (owners * ENTRIES) + o.index;
  if (!o.live) return;
  const int used = *m.used;
  bool inside = true;
  const T* from[ENTRIES];
  T* to[ENTRIES];
  Edges edges[ENTRIES];
#pragma unroll
  for (int q = 0; q < ENTRIES; ++q) {
    const long long e = first + q * owners;
    const int s = e < entries ? m.slots[e] : -1;
    from[q] = x + (long long)((uint32_t)e / (uint32_t)m.choices) * stride;   // entries are below 2^30
    to[q] = out + (long long)(s >= 0 ? s : 0) * m.width;
    edges[q] = Edges::of<R>(to[q], m.width);
    if (s < 0) edges[q].packs = edges[q].count = 0;
    else inside = inside && extent.inside(from[q], m.width);
  }
  for (int k = lane + (int)blockIdx.y * m.lanes; k < packs_of<T, L>(m.width); k += m.lanes * (int)gridDim.y) {
    typename R::Raw p[ENTRIES];
    if (inside) {
#pragma unroll
      for (int q = 0; q < ENTRIES; ++q)
        if (k < edges[q].packs) p[q] = R::load(from[q] + edges[q].head + k * R::kVec);
    } else {
#pragma unroll
      for (int q = 0; q < ENTRIES; ++q)
        if (k < edges[q].packs) p[q] = R::load_elements(from[q] + edges[q].head + k * R::kVec);
    }
#pragma unroll
    for (int q = 0; q < ENTRIES; ++q)
      if (k < edges[q].packs) R::store(to[q] + edges[q].head + k * R::kVec, R::words(p[q]));
  }
  if (blockIdx.y) return;
#pragma unroll
  for (int q = 0; q < ENTRIES; ++q) {
    if (L == kSpan)
      for (int i = lane; i < edges[q].count; i += m.lanes) to[q][edges[q].edge(i)] = from[q][edges[q].edge(i)];
    if (first + q * owners < entries) clear_behind<T, L>(m, used, first + q * owners, entries, lane, out);
  }
}

// ... gathered into runs of places.
struct Places {
  const int* order;     // the entry at each place
  const int* used;
  int choices;
  __device__ __forceinline__ long long row(long long place) const {   // -1: behind the last group
    return place < *used ? (long long)((uint32_t)order[place] / (uint32_t)choices) : -1;   // entries are below 2^30
  }
};

template <typename T, typename S>
__global__ void __launch_bounds__(kTileThreads) rows_to_groups_tile_kernel(Places places, long long count, int tile,
                                                                           int width, const T* __restrict__ x,
                                                                           long long stride, T* __restrict__ out) {
  gather_tile<T, false, S::kPairs, S::kWide, S::kRows, S::kJ>(
      [&](long long p) -> const T* {
        const long long n = places.row(p);
        return n >= 0 ? x + n * stride : nullptr;
      },
      count, tile, width, 1.f, out);
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads) rows_to_groups_flat_kernel(Places places, long long count, int tile,
                                                                           uint32_t reciprocal, int width,
                                                                           const T* __restrict__ x, long long stride,
                                                                           T* __restrict__ out) {
  gather_flat<T, false>(
      [&](long long p) -> const T* {
        const long long n = places.row(p);
        return n >= 0 ? x + n * stride : nullptr;
      },
      count, tile, reciprocal, width, 1.f, out);
}

// The weights are float32 or of the rows' type.
struct Weights {
  const void* at;   // null: ones
  bool same;        // of the rows' type
};

template <typename T>
__device__ __forceinline__ float weight_at(const Weights& w, long long e) {
  if (!w.at) return 1.f;
  return w.same ? to_float(((const T*)w.at)[e]) : ((const float*)w.at)[e];
}

// Slots and weights of CHOICES choices from i0 on of the owner's rows; a slot is -1 where
// there is no entry or it is left out.
template <typename T, int ROWS, int CHOICES>
__device__ __forceinline__ void load_choices(const Moves& m, const Weights& weights, long long first, int owners, int i0,
                                             int (&slot)[ROWS][CHOICES], float (&w)[ROWS][CHOICES]) {
#pragma unroll
  for (int q = 0; q < ROWS; ++q)
#pragma unroll
    for (int i = 0; i < CHOICES; ++i) {
      const long long row = first + q * owners, e = row * m.choices + i0 + i;
      const bool in = row < m.n && i0 + i < m.choices;
      slot[q][i] = in ? m.slots[e] : -1;
      w[q][i] = in ? weight_at<T>(weights, e) : 0.f;
    }
}

// An owner has one pack of CHOICES choices of each of ROWS rows in flight.  Five blocks per SM leave
// 48 registers, which the 16-bit forms of two rows and of four choices, and spans of two, spill 48 to
// 92 bytes of: 97656 aligned rows of 1024 f16 from one choice take 84 us, the same bytes as floats 71.
template <typename T, Layout L, int ROWS, int CHOICES>
__global__ void __launch_bounds__(kThreads, 5) groups_to_rows_kernel(Moves m, const T* __restrict__ y, Extent extent,
                                                                     long long stride, Weights weights,
                                                                     T* __restrict__ out) {
  using R = Row<T, L>;
  const Owner o = Owner::of(m.lanes);
  const int owners = m.owners, lane = o.lane;
  const long long first = (long long)blockIdx.x * (owners * ROWS) + o.index;
  if (!o.live) return;
  int slot[ROWS][CHOICES];
  float w[ROWS][CHOICES];
  Edges edges[ROWS];
  load_choices<T>(m, weights, first, owners, 0, slot, w);
  bool inside = true;
#pragma unroll
  for (int q = 0; q < ROWS; ++q) {
    edges[q] = Edges::of<R>(out + (first + q * owners) * m.width, m.width);
    if (first + q * owners >= m.n) edges[q].packs = edges[q].count = 0;
    if (L == kSpan && extent.checked)
      for (int i = 0; i < m.choices; ++i) {
        const int s = first + q * owners < m.n ? m.slots[(first + q * owners) * m.choices + i] : -1;
        if (s >= 0) inside = inside && extent.inside(y + (long long)s * stride, m.width);
      }
  }
  for (int k = lane + (int)blockIdx.y * m.lanes; k < packs_of<T, L>(m.width); k += m.lanes * (int)gridDim.y) {
    float acc[ROWS][R::kVec];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int v = 0; v < R::kVec; ++v) acc[q][v] = 0.f;
    for (int i0 = 0; i0 < m.choices; i0 += CHOICES) {
      if (m.choices > CHOICES) load_choices<T>(m, weights, first, owners, i0, slot, w);
      typename R::Raw p[ROWS][CHOICES];
      auto load = [&](auto read) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
#pragma unroll
          for (int i = 0; i < CHOICES; ++i)
            if (slot[q][i] >= 0 && k < edges[q].packs)
              p[q][i] = read(y + (long long)slot[q][i] * stride + edges[q].head + k * R::kVec);
      };
      if (L != kSpan || inside) load([](const T* at) { return R::load(at); });
      else load([](const T* at) { return R::load_elements(at); });
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0 && k < edges[q].packs) {   // an entry left out counts nothing, whatever its weight holds
            float f[R::kVec];
            R::floats(p[q][i], f);
#pragma unroll
            for (int v = 0; v < R::kVec; ++v) acc[q][v] = fmaf(w[q][i], f[v], acc[q][v]);
          }
    }
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
      if (k < edges[q].packs)
        R::store(out + (first + q * owners) * m.width + edges[q].head + k * R::kVec, R::words(acc[q]));
  }
  if (L == kSpan && blockIdx.y == 0) {
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const long long row = first + q * owners;
      for (int i = lane; i < edges[q].count; i += m.lanes) {
        const int e = edges[q].edge(i);
        float acc = 0.f;
#pragma unroll 4
        for (int j = 0; j < m.choices; ++j) {
          const int s = m.slots[row * m.choices + j];
          if (s >= 0) acc = fmaf(weight_at<T>(weights, row * m.choices + j), to_float(y[(long long)s * stride + e]), acc);
        }
        out[row * m.width + e] = from_float<T>(acc);
      }
    }
  }
}

// Rows that are not aligned, up to 4 KB: a warp puts its rows into the block's tile, J elements
// per lane of CHOICES choices in flight.  Its slots and weights are 32 at a time, one per lane.
// (Two rows at once: 75 us against 57 for 100003 rows of 333 f16 from 2 choices.)
template <typename T, bool WIDE, int CHOICES, int J>
__global__ void __launch_bounds__(kTileThreads) groups_to_rows_tile_kernel(long long rows, int choices, int tile,
                                                                           int width, const int* __restrict__ slots,
                                                                           const T* __restrict__ y, long long stride,
                                                                           Weights weights, T* __restrict__ out) {
  extern __shared__ __align__(16) unsigned char raw[];
  T* buf = reinterpret_cast<T*>(raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = tile / kTileWarps;
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, rows - first), r0 = warp * each, mine = max(0, min(each, n - r0));
  const long long e0 = (first + r0) * choices;
  const int entries = mine * choices;   // of this warp
  int chunk = -32;
  unsigned long long my_row = 0;
  float my_weight = 0.f;
  auto entry = [&](int e, const T*& row, float& w) {   // the same entry for the whole warp
    if (e < chunk || e >= chunk + 32) {
      chunk = e & ~31;
      const int i = chunk + lane, s = i < entries ? slots[e0 + i] : -1;
      my_row = (unsigned long long)(uintptr_t)(s >= 0 ? y + (long long)s * stride : reinterpret_cast<const T*>(g_zero_row));
      my_weight = s >= 0 ? weight_at<T>(weights, e0 + i) : 0.f;   // left out: whatever its weight holds
    }
    row = reinterpret_cast<const T*>((uintptr_t)shuffle(my_row, e & 31)) + lane;
    w = __shfl_sync(0xffffffffu, my_weight, e & 31);
  };
  for (int r = 0; r < mine; ++r) {
    T* to = buf + (r0 + r) * width + lane;
    for (int c = 0; c < width; c += 32 * J) {
      const int left = width - lane - c;
      float acc[J];
#pragma unroll
      for (int j = 0; j < J; ++j) acc[j] = 0.f;
      for (int i = 0; i < choices; i += CHOICES) {
        const T *a, *b;
        float wa, wb = 0.f;
        entry(r * choices + i, a, wa);
        // (a row of zeros for a choice too many: loads under a branch would wait one by one)
        if (CHOICES > 1 && i + 1 < choices) entry(r * choices + i + 1, b, wb);
        else b = reinterpret_cast<const T*>(g_zero_row) + lane;
        T va[J], vb[J];
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (32 * j < left) {
            va[j] = a[c + 32 * j];
            if (CHOICES > 1) vb[j] = b[c + 32 * j];
          }
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (32 * j < left) {
            acc[j] = fmaf(wa, to_float(va[j]), acc[j]);
            if (CHOICES > 1) acc[j] = fmaf(wb, to_float(vb[j]), acc[j]);
          }
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (32 * j < left) to[c + 32 * j] = from_float<T>(acc[j]);
      if (!WIDE) break;
    }
  }
  send_tile(buf, n, width, out + first * width);
}

// The same for narrow rows, flat as gather_flat: an element (16 bits: two) of the block's run of
// rows per lane and step, kFlatSteps steps at once, the places and weights in shared memory.
// (1.6M rows of 31 floats from a choice: 99 us, 135 by warps with two rows each; of 59: 97 and 97.
// 4M rows of 12 f16: 108 us, 303 by an element per lane and row.)
constexpr int kFlatSumWidth = 64, kFlatSteps = 4;
constexpr int kFlatEntries = 1024;   // rows x choices of a block at most

template <typename T>
__global__ void __launch_bounds__(kTileThreads) groups_to_rows_flat_kernel(long long rows, int choices, int tile,
                                                                           uint32_t reciprocal, int width,
                                                                           const int* __restrict__ slots,
                                                                           const T* __restrict__ y, long long stride,
                                                                           Weights weights, T* __restrict__ out) {
  constexpr int kEach = 4 / (int)sizeof(T);
  __shared__ const T* row[kFlatEntries];
  __shared__ float weight[kFlatEntries];
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, rows - first);
  for (int k = threadIdx.x; k < n * choices; k += kTileThreads) {
    const int s = slots[first * choices + k];
    row[k] = s >= 0 ? y + (long long)s * stride : reinterpret_cast<const T*>(g_zero_row);
    weight[k] = s >= 0 ? weight_at<T>(weights, first * choices + k) : 0.f;   // left out: whatever its weight holds
  }
  __syncthreads();
  T* to = out + first * width;
  const int total = n * width;
  for (int p0 = threadIdx.x * kEach; p0 < total; p0 += kTileThreads * kEach * kFlatSteps) {
    int at[kFlatSteps][kEach], col[kFlatSteps][kEach];
    float acc[kFlatSteps][kEach];
#pragma unroll
    for (int u = 0; u < kFlatSteps; ++u)
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int e = min(p0 + u * kTileThreads * kEach + i, total - 1), t = flat_row(e, width, reciprocal);
        at[u][i] = t * choices;
        col[u][i] = e - t * width;
        acc[u][i] = 0.f;
      }
    for (int j = 0; j < choices; ++j) {
      T v[kFlatSteps][kEach];
#pragma unroll
      for (int u = 0; u < kFlatSteps; ++u)
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[u][i] = row[at[u][i] + j][col[u][i]];
#pragma unroll
      for (int u = 0; u < kFlatSteps; ++u)
#pragma unroll
        for (int i = 0; i < kEach; ++i) acc[u][i] = fmaf(weight[at[u][i] + j], to_float(v[u][i]), acc[u][i]);
    }
#pragma unroll
    for (int u = 0; u < kFlatSteps; ++u) {
      const int p = p0 + u * kTileThreads * kEach;
      if (p < total) flat_store(to + p, acc[u], p + kEach <= total);
    }
  }
}

// ... and its gradient, by places: dy[p] = w dout[n], dw = <dout[n], y[p]> for the entry at p.
template <typename T, bool WIDE, int ROWS, int J>
__global__ void __launch_bounds__(kTileThreads) groups_to_rows_backward_tile_kernel(
    Places places, long long count, int tile, int width, const T* __restrict__ grad, long long grad_stride,
    const T* __restrict__ y, long long stride, Weights weights, T* __restrict__ grad_y,
    void* __restrict__ grad_weights) {
  extern __shared__ __align__(16) unsigned char raw[];
  T* buf = reinterpret_cast<T*>(raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, each = tile / kTileWarps;
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, count - first), r0 = warp * each;
  const T* zeros = reinterpret_cast<const T*>(g_zero_row);
  const T *grad_row = zeros, *y_row = zeros;
  float weight = 0.f, my_dot = 0.f;
  int entry = -1;
  if (lane < each && r0 + lane < n) {
    const long long p = first + r0 + lane, row = places.row(p);
    entry = places.order[p];
    if (row >= 0) {
      grad_row = grad + row * grad_stride;
      y_row = y + p * stride;
      weight = weight_at<T>(weights, entry);
    }
  }
  for (int r = 0; r < each; r += ROWS) {
    const T *g[ROWS], *h[ROWS];
    float w[ROWS], dot[ROWS];
#pragma unroll
    for (int q = 0; q < ROWS; ++q) {
      const int src = (r + q) & 31;
      g[q] = reinterpret_cast<const T*>((uintptr_t)shuffle((unsigned long long)(uintptr_t)grad_row, src)) + lane;
      h[q] = reinterpret_cast<const T*>((uintptr_t)shuffle((unsigned long long)(uintptr_t)y_row, src)) + lane;
      w[q] = __shfl_sync(0xffffffffu, weight, src);
      dot[q] = 0.f;
    }
    for (int c = 0; c < width; c += 32 * J) {
      const int left = width - lane - c;
      T vg[ROWS][J], vh[ROWS][J];
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (32 * j < left) {
            vg[q][j] = g[q][c + 32 * j];
            if (grad_weights) vh[q][j] = h[q][c + 32 * j];
          }
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (32 * j < left) {
            const float f = to_float(vg[q][j]);
            if (grad_weights) dot[q] = fmaf(f, to_float(vh[q][j]), dot[q]);
            if (grad_y && r + q < each) buf[(r0 + r + q) * width + lane + c + 32 * j] = from_float<T>(w[q] * f);
          }
      if (!WIDE) break;
    }
    if (grad_weights) {
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], o);
        if (lane == r + q) my_dot = dot[q];
      }
    }
  }
  if (grad_weights && entry >= 0) {
    if (weights.same) ((T*)grad_weights)[entry] = from_float<T>(my_dot);
    else ((float*)grad_weights)[entry] = my_dot;
  }
  if (grad_y) send_tile(buf, n, width, grad_y + first * width);
}

// The same for narrow rows, flat; the products of a place's dot product go through shared memory
// to one thread, which adds them up in order.  (4M rows of 12 f16: 162 us, 545 by an element per
// lane and row; 3M of 33: 230, 289 by warps; 1.7M of 59: 225 and 190.  From 3 elements on: 4M rows
// of 3 floats 90 and 117, of 2: 78 and 74, of 1: 72 and 45; 1M rows of 4 choices of 3 floats 74 and
// 82, of 2: 70 and 57; 4M of 3 bf16 102 and 100, of 2: 96 and 66.)
constexpr int kFlatGradWidth = 40;
template <typename T>
__global__ void __launch_bounds__(kTileThreads) groups_to_rows_backward_flat_kernel(
    Places places, long long count, int tile, uint32_t reciprocal, int width, const T* __restrict__ grad,
    long long grad_stride, const T* __restrict__ y, long long stride, Weights weights, T* __restrict__ grad_y,
    void* __restrict__ grad_weights) {
  constexpr int kEach = 4 / (int)sizeof(T);
  __shared__ const T* grad_row[kFlatRows];
  __shared__ float weight[kFlatRows];
  __shared__ float product[kTileThreads * kFlatWords * kEach / 2];
  const T* zeros = reinterpret_cast<const T*>(g_zero_row);
  const long long first = (long long)blockIdx.x * tile;
  const int n = (int)min((long long)tile, count - first);
  const int used = (int)max(0ll, min((long long)n, *places.used - first));   // the others' rows are not read
  const T* const y0 = y + first * stride;
  for (int k = threadIdx.x; k < n; k += kTileThreads) {
    const long long p = first + k, r = places.row(p);
    grad_row[k] = r >= 0 ? grad + r * grad_stride : zeros;
    weight[k] = r >= 0 ? weight_at<T>(weights, places.order[p]) : 0.f;
  }
  __syncthreads();
  const int total = n * width;
  for (int p0 = threadIdx.x * kEach; p0 < total; p0 += kTileThreads * kEach * kFlatSteps) {
    T g[kFlatSteps][kEach], h[kFlatSteps][kEach];
    int row[kFlatSteps][kEach];
#pragma unroll
    for (int u = 0; u < kFlatSteps; ++u)
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int e = min(p0 + u * kTileThreads * kEach + i, total - 1), t = flat_row(e, width, reciprocal);
        row[u][i] = t;
        g[u][i] = grad_row[t][e - t * width];
        if (grad_weights) h[u][i] = *(t < used ? y0 + t * stride + (e - t * width) : zeros);
      }
#pragma unroll
    for (int u = 0; u < kFlatSteps; ++u) {
      const int p = p0 + u * kTileThreads * kEach;
      float f[kEach];
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        f[i] = to_float(g[u][i]);
        if (grad_weights && p + i < total) product[p + i] = f[i] * to_float(h[u][i]);
        f[i] *= weight[row[u][i]];
      }
      if (grad_y && p < total) flat_store(grad_y + first * width + p, f, p + kEach <= total);
    }
  }
  if (!grad_weights) return;
  __syncthreads();
  for (int k = threadIdx.x; k < n; k += kTileThreads) {
    float dot = 0.f;
    for (int c = 0; c < width; ++c) dot += product[k * width + c];
    const int entry = places.order[first + k];
    if (weights.same) ((T*)grad_weights)[entry] = from_float<T>(dot);
    else ((float*)grad_weights)[entry] = dot;
  }
}

// Packs follow the row of grad_y that is written (with unaligned rows each choice's begins
// elsewhere, so the row of grad is read again for it, from L1).  BLOCK: a whole block owns a row,
// its warps' dot products are joined in their order.
template <typename T, Layout L, int ROWS, int CHOICES, bool BLOCK>
__global__ void __launch_bounds__(kThreads, 4) groups_to_rows_backward_kernel(
    Moves m, const T* __restrict__ grad, Extent grad_extent, long long grad_stride, const T* __restrict__ y,
    Extent extent, long long stride, Weights weights, T* __restrict__ grad_y, void* __restrict__ grad_weights) {
  using R = Row<T, L>;
  constexpr bool kShared = L != kSpan;   // one pack of grad for all choices
  const Owner o = BLOCK ? Owner{0, (int)threadIdx.x, true} : Owner::of(m.lanes);
  const int owners = m.owners, lane = o.lane;
  // lanes without an owner stay for the shuffles, behind the last row
  const long long first = o.live ? (long long)blockIdx.x * (owners * ROWS) + o.index : m.n;
  for (int i0 = (int)blockIdx.y * CHOICES; i0 < m.choices; i0 += CHOICES * (int)gridDim.y) {
    int slot[ROWS][CHOICES];
    float w[ROWS][CHOICES], dot[ROWS][CHOICES];
    Edges edges[ROWS][CHOICES];
    load_choices<T>(m, weights, first, owners, i0, slot, w);
    bool inside = true;
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int i = 0; i < CHOICES; ++i) {
        dot[q][i] = 0.f;
        edges[q][i] = Edges::of<R>((grad_y ? grad_y : grad) + (long long)max(slot[q][i], 0) * m.width, m.width);
        if (L == kSpan && slot[q][i] >= 0)
          inside = inside && grad_extent.inside(grad + (first + q * owners) * grad_stride, m.width) &&
                   (!grad_weights || extent.inside(y + (long long)slot[q][i] * stride, m.width));
      }
    for (int k = lane; k < packs_of<T, L>(m.width); k += m.lanes) {
      typename R::Raw g[ROWS][kShared ? 1 : CHOICES], p[ROWS][CHOICES];
      auto load = [&](auto read) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
          const T* row = grad + (first + q * owners) * grad_stride;
          if (kShared && first + q * owners < m.n) g[q][0] = read(row + k * R::kVec);
#pragma unroll
          for (int i = 0; i < CHOICES; ++i)
            if (slot[q][i] >= 0 && k < edges[q][i].packs) {
              const int e = edges[q][i].head + k * R::kVec;
              if (!kShared) g[q][kShared ? 0 : i] = read(row + e);
              if (grad_weights) p[q][i] = read(y + (long long)slot[q][i] * stride + e);
            }
        }
      };
      if (L != kSpan || inside) load([](const T* at) { return R::load(at); });
      else load([](const T* at) { return R::load_elements(at); });
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0 && k < edges[q][i].packs) {
            float f[R::kVec];
            R::floats(g[q][kShared ? 0 : i], f);
            if (grad_weights) {
              float h[R::kVec];
              R::floats(p[q][i], h);
#pragma unroll
              for (int v = 0; v < R::kVec; ++v) dot[q][i] = fmaf(f[v], h[v], dot[q][i]);
            }
            if (grad_y) {
#pragma unroll
              for (int v = 0; v < R::kVec; ++v) f[v] *= w[q][i];
              R::store(grad_y + (long long)slot[q][i] * m.width + edges[q][i].head + k * R::kVec, R::words(f));
            }
          }
    }
    if (L == kSpan) {
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0)
            for (int j = lane; j < edges[q][i].count; j += m.lanes) {
              const int e = edges[q][i].edge(j);
              const float f = to_float(grad[(first + q * owners) * grad_stride + e]);
              if (grad_weights) dot[q][i] = fmaf(f, to_float(y[(long long)slot[q][i] * stride + e]), dot[q][i]);
              if (grad_y) grad_y[(long long)slot[q][i] * m.width + e] = from_float<T>(w[q][i] * f);
            }
    }
    if (grad_weights) {
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i) {
          float d = dot[q][i];
          if constexpr (BLOCK) {
            __shared__ float part[kThreads / 32];
#pragma unroll
            for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
            if ((lane & 31) == 0) part[lane >> 5] = d;
            __syncthreads();
            d = part[0];
#pragma unroll
            for (int x = 1; x < kThreads / 32; ++x) d += part[x];
            __syncthreads();
          } else if ((m.lanes & (m.lanes - 1)) == 0) {
            for (int x = m.lanes >> 1; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
          } else {   // lanes beside one another: halve what is left, an odd one waits for its turn
            for (int left = m.lanes; left > 1; left = (left + 1) >> 1) {
              const float other = __shfl_down_sync(0xffffffffu, d, (left + 1) >> 1);
              if (lane < left >> 1) d += other;
            }
          }
          const long long row = first + q * owners, e = row * m.choices + i0 + i;
          if (lane == 0 && row < m.n && i0 + i < m.choices) {
            if (weights.same) ((T*)grad_weights)[e] = from_float<T>(d);
            else ((float*)grad_weights)[e] = d;
          }
        }
    }
  }
  if (grad_y && blockIdx.y == 0) {
    const int used = *m.used;
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
      if (first + q * owners < m.n) clear_behind<T, L>(m, used, first + q * owners, m.n, lane, grad_y);
  }
}

inline unsigned blocks_for(long long n, int owners, int rows) {
  const long long per_block = (long long)owners * rows;
  return (unsigned)((n + per_block - 1) / per_block);
}

// Calls f<layout>(lanes) for rows that are all aligned, and for others by their width.
template <typename T, typename F>
int with_layout(bool aligned, int width, F f) {
  if (aligned) return f(std::integral_constant<Layout, kAligned>(), lanes_for(packs_of<T, kAligned>(width)));
  if (width >= kSpanWidth) return f(std::integral_constant<Layout, kSpan>(), lanes_for(packs_of<T, kSpan>(width)));
  return f(std::integral_constant<Layout, kElement>(), lanes_for(width));
}

template <typename T>
int to_groups(bool aligned, const void* x, long long stride, Moves m, const int* order, void* out, cudaStream_t st) {
  const Places places{order, m.used, m.choices};
  const long long count = m.n * m.choices;
  if (!aligned && flat_fits(m.width, out)) {
    const int tile = flat_rows(m.width, sizeof(T));
    rows_to_groups_flat_kernel<T><<<(unsigned)((count + tile - 1) / tile), kTileThreads, 0, st>>>(
        places, count, tile, flat_reciprocal(m.width), m.width, (const T*)x, stride, (T*)out);
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  if (!aligned && tile_fits(m.width, sizeof(T), out)) {
    const int tile = tile_rows(count, m.width, sizeof(T));
    const unsigned blocks = (unsigned)((count + tile - 1) / tile);
    const size_t shared = (size_t)tile * m.width * sizeof(T);
    return with_shape<T>(m.width, [&](auto shape) {
      rows_to_groups_tile_kernel<T, decltype(shape)><<<blocks, kTileThreads, shared, st>>>(
          places, count, tile, m.width, (const T*)x, stride, (T*)out);
      CVHRF_LAUNCH_CHECK();
      return CVHRF_OK;
    });
  }
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    m.owners = owners_of(kThreads, lanes);
    const T* from = (const T*)x;
    if constexpr (L == kAligned) {
      const int packs = packs_of<T, L>(m.width);
      if (packs > 64) {
        // (2 per SM: 2000 rows of 4096 floats to 4 places each 33 us, 35 in two parts)
        const unsigned blocks = blocks_for(m.n, m.owners, 1);
        const unsigned parts = parts_for(blocks, (packs + lanes * 4 - 1) / (lanes * 4), 2);
        rows_to_groups_kernel<T, 1, 4><<<dim3(blocks, parts), kThreads, 0, st>>>(m, from, stride, (T*)out);
      } else if (packs > 32) {
        rows_to_groups_kernel<T, 2, 2><<<blocks_for(m.n, m.owners, 2), kThreads, 0, st>>>(m, from, stride, (T*)out);
      } else {
        rows_to_groups_kernel<T, 4, 1><<<blocks_for(m.n, m.owners, 4), kThreads, 0, st>>>(m, from, stride, (T*)out);
      }
    } else {
      constexpr int kEntries = L == kSpan ? 2 : 4;
      const unsigned blocks = blocks_for(m.n * m.choices, m.owners, kEntries);
      const unsigned parts = parts_for(blocks, (packs_of<T, L>(m.width) + lanes - 1) / lanes);
      entries_to_groups_kernel<T, L, kEntries><<<dim3(blocks, parts), kThreads, 0, st>>>(
          m, from, extent_of(x, m.n, stride, m.width, sizeof(T)), stride, (T*)out);
    }
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

template <typename T>
int to_rows(bool aligned, const void* y, long long stride, Moves m, Weights weights, void* out, cudaStream_t st) {
  const bool pairs = ((uintptr_t)out & 3) == 0;
  // (Very narrow rows of many choices read their places again for every element: 22 us against 48
  // for 500000 rows of 2 f16 from 8 choices; of 12: 110 against 83.)
  if (!aligned && m.width >= (m.choices > 2 ? 8 : 3) && m.width <= kFlatSumWidth && m.choices <= kFlatEntries / 8 && pairs) {
    const int most = kFlatEntries / m.choices / 2 * 2, rows = flat_rows(m.width, sizeof(T));
    const int tile = rows < most ? rows : most;
    groups_to_rows_flat_kernel<T><<<(unsigned)((m.n + tile - 1) / tile), kTileThreads, 0, st>>>(
        m.n, m.choices, tile, flat_reciprocal(m.width), m.width, m.slots, (const T*)y, stride, weights, (T*)out);
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  if (!aligned && m.width > kFlatWidth && tile_fits(m.width, sizeof(T), out)) {
    const int tile = tile_rows(m.n, m.width, sizeof(T));
    const unsigned blocks = (unsigned)((m.n + tile - 1) / tile);
    const size_t shared = (size_t)tile * m.width * sizeof(T);
#define CVHRF_SHAPE(WIDE, CHOICES, J)                                                       \
  groups_to_rows_tile_kernel<T, WIDE, CHOICES, J><<<blocks, kTileThreads, shared, st>>>(    \
      m.n, m.choices, tile, m.width, m.slots, (const T*)y, stride, weights, (T*)out)
#define CVHRF_LAUNCH(WIDE, J)                      \
  do {                                             \
    if (m.choices == 1) CVHRF_SHAPE(WIDE, 1, J);   \
    else CVHRF_SHAPE(WIDE, 2, J);                  \
  } while (0)
    const int steps = (m.width + 255) / 256;   // J shares the row evenly between them
    if (m.width > 128 && m.width <= steps * 192) CVHRF_LAUNCH(true, 6);
    else if (m.width > 128) CVHRF_LAUNCH(true, 8);
    else if (m.width > 64) CVHRF_LAUNCH(false, 4);
    else if (m.width > 32) CVHRF_LAUNCH(false, 2);
    else CVHRF_LAUNCH(false, 1);
#undef CVHRF_SHAPE
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    m.owners = owners_of(kThreads, lanes);
    const Extent extent = extent_of(y, m.n * m.choices, stride, m.width, sizeof(T));
    const int steps = (packs_of<T, L>(m.width) + lanes - 1) / lanes;
#define CVHRF_LAUNCH(ROWS, CHOICES)                                                                      \
  groups_to_rows_kernel<T, L, ROWS, CHOICES>                                                             \
      <<<dim3(blocks_for(m.n, m.owners, ROWS), parts_for(blocks_for(m.n, m.owners, ROWS), steps)), kThreads, 0, st>>>( \
          m, (const T*)y, extent, stride, weights, (T*)out)
    if constexpr (L == kSpan) {   // twice the registers per pack
      if (m.choices > 1) CVHRF_LAUNCH(1, 2);
      else CVHRF_LAUNCH(1, 1);
    } else {
      if (m.choices > 2) CVHRF_LAUNCH(1, 4);
      else if (m.choices > 1) CVHRF_LAUNCH(1, 2);
      else CVHRF_LAUNCH(2, 1);
    }
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

template <typename T>
int to_rows_backward(bool aligned, const void* grad, long long grad_stride, const void* y, long long stride, Moves m,
                     const int* order, Weights weights, void* grad_y, void* grad_weights, cudaStream_t st) {
  const Places places{order, m.used, m.choices};
  const long long count = m.n * m.choices;
  if (!aligned && m.width >= 3 && m.width <= kFlatGradWidth && ((uintptr_t)grad_y & 3) == 0) {
    const int tile = flat_rows(m.width, sizeof(T)) / 4 * 2;
    groups_to_rows_backward_flat_kernel<T><<<(unsigned)((count + tile - 1) / tile), kTileThreads, 0, st>>>(
        places, count, tile, flat_reciprocal(m.width), m.width, (const T*)grad, grad_stride, (const T*)y, stride,
        weights, (T*)grad_y, grad_weights);
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  if (!aligned && m.width > kFlatGradWidth && tile_fits(m.width, sizeof(T), grad_y)) {
    const int tile = tile_rows(count, m.width, sizeof(T));
    const unsigned blocks = (unsigned)((count + tile - 1) / tile);
    const size_t shared = (size_t)tile * m.width * sizeof(T);
#define CVHRF_LAUNCH(WIDE, ROWS, J)                                                               \
  groups_to_rows_backward_tile_kernel<T, WIDE, ROWS, J><<<blocks, kTileThreads, shared, st>>>(    \
      places, count, tile, m.width, (const T*)grad, grad_stride, (const T*)y, stride, weights, (T*)grad_y, grad_weights)
    const int steps = (m.width + 255) / 256;
    if (m.width > 128 && m.width <= steps * 192) CVHRF_LAUNCH(true, 1, 6);
    else if (m.width > 128) CVHRF_LAUNCH(true, 1, 8);
    else if (m.width > 64) CVHRF_LAUNCH(false, 1, 4);
    else CVHRF_LAUNCH(false, 2, 2);
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  }
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    m.owners = owners_of(kThreads, lanes);
    const Extent grad_extent = extent_of(grad, m.n, grad_stride, m.width, sizeof(T));
    const Extent extent = extent_of(y, m.n * m.choices, stride, m.width, sizeof(T));
    // Few rows: the choices are shared between blocks, and long rows are a whole block's, the longer
    // the more of them (64 rows of 9000 floats to 8 places: 7.5 us, 75 by warps, 148 without either;
    // 2000 of 4096 floats to one: 19 and 30; of 1024 floats to 4: 14 and 11).
#define CVHRF_LAUNCH(ROWS, CHOICES, BLOCK)                                                                 \
  groups_to_rows_backward_kernel<T, L, ROWS, CHOICES, BLOCK>                                               \
      <<<dim3(blocks_for(m.n, m.owners, ROWS),                                                             \
              parts_for(blocks_for(m.n, m.owners, ROWS), (m.choices + CHOICES - 1) / CHOICES)),            \
         kThreads, 0, st>>>(                                                                               \
      m, (const T*)grad, grad_extent, grad_stride, (const T*)y, extent, stride, weights, (T*)grad_y, grad_weights)
    if constexpr (L != kElement) {
      const long long packs = packs_of<T, L>(m.width), entries = (long long)blocks_for(m.n, m.owners, 1) * m.choices;
      if (packs >= 128 && entries < 148 * std::min(8ll, packs / 128)) {
        m.lanes = kThreads;
        m.owners = 1;
        if (L == kAligned && m.choices > 1) CVHRF_LAUNCH(1, 2, true);
        else CVHRF_LAUNCH(1, 1, true);
        CVHRF_LAUNCH_CHECK();
        return CVHRF_OK;
      }
    }
    if constexpr (L == kSpan) {   // four times: the pack of grad and of y
      CVHRF_LAUNCH(1, 1, false);
    } else {
      if (m.choices > 2) CVHRF_LAUNCH(1, 4, false);
      else if (m.choices > 1) CVHRF_LAUNCH(1, 2, false);
      else CVHRF_LAUNCH(2, 1, false);
    }
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

int check_moves(int dtype, long long n, int choices, int width) {
  if (!row_type_ok(dtype) || n < 0 || choices < 1 || width < 1 || width > kMaxWidth) return CVHRF_EINVAL;
  if (n > kGroupMaxEntries / choices) return CVHRF_EUNSUPPORTED;
  return CVHRF_OK;
}

template <typename F>
int with_type(int dtype, F f) {
  if (dtype == CVHRF_F32) return f(float());
  if (dtype == CVHRF_BF16) return f(__nv_bfloat16());
  return f(__half());
}

}  // namespace
}  // namespace cvhrf

using namespace cvhrf;

extern "C" int cvhrf_rows_to_groups(const cvhrf_moves_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const cvhrf_moves_args a = *args;
  const int rc = check_moves(a.dtype, a.n, a.choices, a.width);
  if (rc) return rc;
  if (a.stride < 0) return CVHRF_EINVAL;
  if (a.n == 0) return CVHRF_OK;
  if (!a.from || !a.order || !a.slots || !a.used || !a.to) return CVHRF_EINVAL;
  const bool aligned = rows_16(a.from, a.stride, a.width, row_type_bytes(a.dtype)) && ((uintptr_t)a.to & 15) == 0;
  const Moves m{a.n, a.choices, a.width, 0, 0, a.slots, a.used};
  return with_type(a.dtype, [&](auto type) {
    return to_groups<decltype(type)>(aligned, a.from, a.stride, m, a.order, a.to, (cudaStream_t)stream);
  });
}

extern "C" int cvhrf_groups_to_rows(const cvhrf_moves_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const cvhrf_moves_args a = *args;
  const int rc = check_moves(a.dtype, a.n, a.choices, a.width);
  if (rc) return rc;
  if (a.stride < 0 || (a.weights && a.weights_dtype != CVHRF_F32 && a.weights_dtype != a.dtype)) return CVHRF_EINVAL;
  if (a.n == 0) return CVHRF_OK;
  if (!a.from || !a.slots || !a.to) return CVHRF_EINVAL;
  const bool aligned = rows_16(a.from, a.stride, a.width, row_type_bytes(a.dtype)) && ((uintptr_t)a.to & 15) == 0;
  const Moves m{a.n, a.choices, a.width, 0, 0, a.slots, nullptr};
  const Weights w{a.weights, a.weights && a.weights_dtype == a.dtype};
  return with_type(a.dtype, [&](auto type) {
    return to_rows<decltype(type)>(aligned, a.from, a.stride, m, w, a.to, (cudaStream_t)stream);
  });
}

extern "C" int cvhrf_groups_to_rows_backward(const cvhrf_moves_backward_args* args, void* stream) {
  if (!args) return CVHRF_EINVAL;
  const cvhrf_moves_backward_args a = *args;
  const int rc = check_moves(a.dtype, a.n, a.choices, a.width);
  if (rc) return rc;
  if (a.grad_stride < 0 || a.y_stride < 0 ||
      (a.weights && a.weights_dtype != CVHRF_F32 && a.weights_dtype != a.dtype) || (a.grad_weights && !a.weights))
    return CVHRF_EINVAL;
  if (a.n == 0 || (!a.grad_y && !a.grad_weights)) return CVHRF_OK;
  if (!a.grad || !a.order || !a.slots || !a.used || (a.grad_weights && !a.y)) return CVHRF_EINVAL;
  const size_t elem = row_type_bytes(a.dtype);
  const bool aligned = rows_16(a.grad, a.grad_stride, a.width, elem) &&
                       (!a.grad_weights || rows_16(a.y, a.y_stride, a.width, elem)) && ((uintptr_t)a.grad_y & 15) == 0;
  const Moves m{a.n, a.choices, a.width, 0, 0, a.slots, a.used};
  const Weights w{a.weights, a.weights && a.weights_dtype == a.dtype};
  return with_type(a.dtype, [&](auto type) {
    return to_rows_backward<decltype(type)>(aligned, a.grad, a.grad_stride, a.y, a.y_stride, m, a.order, w,
                                            a.grad_y,
                                            a.grad_weights, (cudaStream_t)stream);
  });
}
