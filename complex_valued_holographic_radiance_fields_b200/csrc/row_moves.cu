// Rows taken to their groups and back: cvhrf_rows_to_groups, cvhrf_groups_to_rows and the
// gradient of the latter.  With slot[n, j] the place of row n's j-th choice (-1: left out):
//
//   to groups  out[slot[n, j]] = x[n]                                    (rows behind the last group: zeros)
//   to rows    out[n] = sum_j w[n, j] y[slot[n, j]]                      (fp32, in the order of j)
//   gradient   dy[slot[n, j]] = w[n, j] dout[n],  dw[n, j] = <dout[n], y[slot[n, j]]>
//
// (The gradient of "to groups" is "to rows" without weights.)  All three go by rows n: a row
// is owned by a power of two of lanes, up to a warp, that hold its columns, so a row of x or
// dout is read once however many groups it goes to, and no two owners write to one place.
// Bound by memory: each touches N + N k rows once.
#include <type_traits>
#include "row_groups.cuh"
#include "row_types.cuh"

namespace cvhrf {
namespace {

constexpr int kThreads = 256;

struct Moves {
  long long n;          // rows
  int choices, width;
  int lanes;            // lanes that own a row
  const int* slots;     // n x choices
  const int* used;      // (device) places that belong to a group; the rest is behind the last group
};

// Zeros into the rows behind the last group, shared out between the owners of the rows or the
// entries (owner x of `owners` takes every `owners`-th of them).
template <typename T, Layout L>
__device__ __forceinline__ void clear_behind(const Moves& m, int used, long long x, long long owners, int lane,
                                             T* __restrict__ out) {
  using R = Row<T, L>;
  const long long places = m.n * m.choices;
  for (long long p = used + x; p < places; p += owners) {
    T* to = out + p * m.width;
    for (int e = lane * R::kVec - R::ahead(to); e < m.width; e += m.lanes * R::kVec)
      R::store(to, e, m.width, zero_pack<T, L>());
  }
}

// Aligned rows: an owner has ROWS rows (owners apart, so that the owners of a block touch
// neighbouring rows) with J packs of each in flight; each pack is read once and written once
// per choice.
template <typename T, int ROWS, int J>
__global__ void __launch_bounds__(kThreads) rows_to_groups_kernel(Moves m, const T* __restrict__ x, long long stride,
                                                                  T* __restrict__ out) {
  using R = Row<T, kAligned>;
  const int owners = kThreads / m.lanes, lane = threadIdx.x & (m.lanes - 1), step = m.lanes * R::kVec;
  const long long first = (long long)blockIdx.x * (owners * ROWS) + threadIdx.x / m.lanes;
  const int used = *m.used;
  for (int c0 = lane * R::kVec; c0 < m.width; c0 += step * J) {
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
    if (first + q * owners < m.n) clear_behind<T, kAligned>(m, used, first + q * owners, m.n, lane, out);
}

// Other rows: packs follow the row that is written, which begins elsewhere for every choice,
// so each owner copies ENTRIES entries (a row's choices are neighbours: its row is read from
// DRAM once).
template <typename T, Layout L, int ENTRIES>
__global__ void __launch_bounds__(kThreads) entries_to_groups_kernel(Moves m, const T* __restrict__ x, Extent extent,
                                                                     long long stride, T* __restrict__ out) {
  using R = Row<T, L>;
  const int owners = kThreads / m.lanes, lane = threadIdx.x & (m.lanes - 1), step = m.lanes * R::kVec;
  const long long entries = m.n * m.choices;
  const long long first = (long long)blockIdx.x * (owners * ENTRIES) + threadIdx.x / m.lanes;
  const int used = *m.used;
  const T* from[ENTRIES];
  T* to[ENTRIES];
  int e0[ENTRIES];
#pragma unroll
  for (int q = 0; q < ENTRIES; ++q) {
    const long long e = first + q * owners;
    const int s = e < entries ? m.slots[e] : -1;
    from[q] = s >= 0 ? x + (long long)((uint32_t)e / (uint32_t)m.choices) * stride : nullptr;   // entries are below 2^30
    to[q] = out + (long long)(s >= 0 ? s : 0) * m.width;
    e0[q] = lane * R::kVec - R::ahead(to[q]);
  }
  for (int c = 0; c - (R::kVec - 1) < m.width; c += step) {
    typename R::Raw p[ENTRIES];
#pragma unroll
    for (int q = 0; q < ENTRIES; ++q)
      if (from[q] && e0[q] + c < m.width) p[q] = R::load(from[q], e0[q] + c, m.width, extent);
#pragma unroll
    for (int q = 0; q < ENTRIES; ++q)
      if (from[q] && e0[q] + c < m.width) R::store(to[q], e0[q] + c, m.width, R::words(p[q]));
  }
#pragma unroll
  for (int q = 0; q < ENTRIES; ++q)
    if (first + q * owners < entries) clear_behind<T, L>(m, used, first + q * owners, entries, lane, out);
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

// An owner has one pack of CHOICES choices of each of ROWS rows in flight.
template <typename T, Layout L, int ROWS, int CHOICES>
__global__ void __launch_bounds__(kThreads, 4) groups_to_rows_kernel(Moves m, const T* __restrict__ y, Extent extent,
                                                                     long long stride, Weights weights,
                                                                     T* __restrict__ out) {
  using R = Row<T, L>;
  const int owners = kThreads / m.lanes, lane = threadIdx.x & (m.lanes - 1), step = m.lanes * R::kVec;
  const long long first = (long long)blockIdx.x * (owners * ROWS) + threadIdx.x / m.lanes;
  int slot[ROWS][CHOICES], e0[ROWS];
  float w[ROWS][CHOICES];
  load_choices<T>(m, weights, first, owners, 0, slot, w);
#pragma unroll
  for (int q = 0; q < ROWS; ++q) e0[q] = lane * R::kVec - R::ahead(out + (first + q * owners) * m.width);
  for (int c = 0; c - (L == kSpan ? R::kVec - 1 : 0) < m.width; c += step) {
    float acc[ROWS][R::kVec];
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int v = 0; v < R::kVec; ++v) acc[q][v] = 0.f;
    for (int i0 = 0; i0 < m.choices; i0 += CHOICES) {
      if (m.choices > CHOICES) load_choices<T>(m, weights, first, owners, i0, slot, w);
      typename R::Raw p[ROWS][CHOICES];
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0 && e0[q] + c < m.width)
            p[q][i] = R::load(y + (long long)slot[q][i] * stride, e0[q] + c, m.width, extent);
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0 && e0[q] + c < m.width) {   // an entry left out counts nothing, whatever its weight holds
            float f[R::kVec];
            R::floats(p[q][i], f);
#pragma unroll
            for (int v = 0; v < R::kVec; ++v) acc[q][v] = fmaf(w[q][i], f[v], acc[q][v]);
          }
    }
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
      if (first + q * owners < m.n && e0[q] + c < m.width)
        R::store(out + (first + q * owners) * m.width, e0[q] + c, m.width, R::words(acc[q]));
  }
}

// Packs follow the row of grad_y that is written (with unaligned rows each choice's begins
// elsewhere, so the row of grad is read again for it, from L1).
template <typename T, Layout L, int ROWS, int CHOICES>
__global__ void __launch_bounds__(kThreads, 4) groups_to_rows_backward_kernel(
    Moves m, const T* __restrict__ grad, Extent grad_extent, long long grad_stride, const T* __restrict__ y,
    Extent extent, long long stride, Weights weights, T* __restrict__ grad_y, void* __restrict__ grad_weights) {
  using R = Row<T, L>;
  const int owners = kThreads / m.lanes, lane = threadIdx.x & (m.lanes - 1), step = m.lanes * R::kVec;
  const long long first = (long long)blockIdx.x * (owners * ROWS) + threadIdx.x / m.lanes;
  for (int i0 = 0; i0 < m.choices; i0 += CHOICES) {
    int slot[ROWS][CHOICES], e0[ROWS][CHOICES];
    float w[ROWS][CHOICES], dot[ROWS][CHOICES];
    load_choices<T>(m, weights, first, owners, i0, slot, w);
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
#pragma unroll
      for (int i = 0; i < CHOICES; ++i) {
        dot[q][i] = 0.f;
        e0[q][i] = lane * R::kVec - (grad_y ? R::ahead(grad_y + (long long)slot[q][i] * m.width) : 0);
      }
    for (int c = 0; c - (L == kSpan ? R::kVec - 1 : 0) < m.width; c += step) {
      typename R::Raw g[ROWS][L == kSpan ? CHOICES : 1], p[ROWS][CHOICES];
#pragma unroll
      for (int q = 0; q < ROWS; ++q) {
        const T* row = grad + (first + q * owners) * grad_stride;
        if (L != kSpan && first + q * owners < m.n && e0[q][0] + c < m.width)
          g[q][0] = R::load(row, e0[q][0] + c, m.width, grad_extent);
#pragma unroll
        for (int i = 0; i < CHOICES; ++i)
          if (slot[q][i] >= 0 && e0[q][i] + c < m.width) {
            if (L == kSpan) g[q][L == kSpan ? i : 0] = R::load(row, e0[q][i] + c, m.width, grad_extent);
            if (grad_weights) p[q][i] = R::load(y + (long long)slot[q][i] * stride, e0[q][i] + c, m.width, extent);
          }
      }
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i) {
          const int e = e0[q][i] + c;
          if (slot[q][i] >= 0 && e < m.width) {
            float f[R::kVec];
            R::floats(g[q][L == kSpan ? i : 0], f);
            if (grad_weights) {
              float h[R::kVec];
              R::floats(p[q][i], h);
#pragma unroll
              for (int v = 0; v < R::kVec; ++v)
                if (L != kSpan || (e + v >= 0 && e + v < m.width)) dot[q][i] = fmaf(f[v], h[v], dot[q][i]);
            }
            if (grad_y) {
#pragma unroll
              for (int v = 0; v < R::kVec; ++v) f[v] *= w[q][i];
              R::store(grad_y + (long long)slot[q][i] * m.width, e, m.width, R::words(f));
            }
          }
        }
    }
    if (grad_weights) {
#pragma unroll
      for (int q = 0; q < ROWS; ++q)
#pragma unroll
        for (int i = 0; i < CHOICES; ++i) {
          float d = dot[q][i];
          for (int o = m.lanes >> 1; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
          const long long row = first + q * owners, e = row * m.choices + i0 + i;
          if (lane == 0 && row < m.n && i0 + i < m.choices) {
            if (weights.same) ((T*)grad_weights)[e] = from_float<T>(d);
            else ((float*)grad_weights)[e] = d;
          }
        }
    }
  }
  if (grad_y) {
    const int used = *m.used;
#pragma unroll
    for (int q = 0; q < ROWS; ++q)
      if (first + q * owners < m.n) clear_behind<T, L>(m, used, first + q * owners, m.n, lane, grad_y);
  }
}

// Lanes that own a row of `packs` packs, and the blocks for `rows` rows per owner.
inline int lanes_for(int packs) { return next_pow2(packs < 32 ? packs : 32); }
inline unsigned blocks_for(long long n, int lanes, int rows) {
  const int per_block = kThreads / lanes * rows;
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
int to_groups(bool aligned, const void* x, long long stride, Moves m, void* out, cudaStream_t st) {
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    const T* from = (const T*)x;
    if constexpr (L == kAligned) {
      const int packs = packs_of<T, L>(m.width);
      if (packs > 64) rows_to_groups_kernel<T, 1, 4><<<blocks_for(m.n, lanes, 1), kThreads, 0, st>>>(m, from, stride, (T*)out);
      else if (packs > 32) rows_to_groups_kernel<T, 2, 2><<<blocks_for(m.n, lanes, 2), kThreads, 0, st>>>(m, from, stride, (T*)out);
      else rows_to_groups_kernel<T, 4, 1><<<blocks_for(m.n, lanes, 4), kThreads, 0, st>>>(m, from, stride, (T*)out);
    } else {
      constexpr int kEntries = L == kSpan ? 2 : 4;
      entries_to_groups_kernel<T, L, kEntries><<<blocks_for(m.n * m.choices, lanes, kEntries), kThreads, 0, st>>>(
          m, from, extent_of(x, m.n, stride, m.width, sizeof(T)), stride, (T*)out);
    }
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

template <typename T>
int to_rows(bool aligned, const void* y, long long stride, Moves m, Weights weights, void* out, cudaStream_t st) {
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    const Extent extent = extent_of(y, m.n * m.choices, stride, m.width, sizeof(T));
#define CVHRF_LAUNCH(ROWS, CHOICES)                                                               \
  groups_to_rows_kernel<T, L, ROWS, CHOICES><<<blocks_for(m.n, lanes, ROWS), kThreads, 0, st>>>(  \
      m, (const T*)y, extent, stride, weights, (T*)out)
    if constexpr (L == kSpan) {   // twice the registers per pack
      if (m.choices > 1) CVHRF_LAUNCH(1, 2);
      else CVHRF_LAUNCH(2, 1);
    } else {
      if (m.choices > 2) CVHRF_LAUNCH(1, 4);
      else if (m.choices > 1) CVHRF_LAUNCH(2, 2);
      else CVHRF_LAUNCH(4, 1);
    }
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

template <typename T>
int to_rows_backward(bool aligned, const void* grad, long long grad_stride, const void* y, long long stride, Moves m,
                     Weights weights, void* grad_y, void* grad_weights, cudaStream_t st) {
  return with_layout<T>(aligned, m.width, [&](auto layout, int lanes) {
    constexpr Layout L = decltype(layout)::value;
    m.lanes = lanes;
    const Extent grad_extent = extent_of(grad, m.n, grad_stride, m.width, sizeof(T));
    const Extent extent = extent_of(y, m.n * m.choices, stride, m.width, sizeof(T));
#define CVHRF_LAUNCH(ROWS, CHOICES)                                                                        \
  groups_to_rows_backward_kernel<T, L, ROWS, CHOICES><<<blocks_for(m.n, lanes, ROWS), kThreads, 0, st>>>(  \
      m, (const T*)grad, grad_extent, grad_stride, (const T*)y, extent, stride, weights, (T*)grad_y, grad_weights)
    if constexpr (L == kSpan) {   // four times: the pack of grad and of y
      CVHRF_LAUNCH(1, 1);
    } else {
      if (m.choices > 2) CVHRF_LAUNCH(1, 4);
      else if (m.choices > 1) CVHRF_LAUNCH(2, 2);
      else CVHRF_LAUNCH(4, 1);
    }
#undef CVHRF_LAUNCH
    CVHRF_LAUNCH_CHECK();
    return CVHRF_OK;
  });
}

int check_moves(int dtype, long long n, int choices, int width) {
  if (!row_type_ok(dtype) || n < 0 || choices < 1 || width < 1) return CVHRF_EINVAL;
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

extern "C" int cvhrf_rows_to_groups(const void* x, long long x_stride, int dtype, long long n, int choices, int width,
                                    const int* slots, const int* used, void* out, void* stream) {
  const int rc = check_moves(dtype, n, choices, width);
  if (rc) return rc;
  if (x_stride < 0) return CVHRF_EINVAL;
  if (n == 0) return CVHRF_OK;
  if (!x || !slots || !used || !out) return CVHRF_EINVAL;
  const bool aligned = rows_16(x, x_stride, width, row_type_bytes(dtype)) && ((uintptr_t)out & 15) == 0;
  const Moves m{n, choices, width, 0, slots, used};
  return with_type(dtype, [&](auto type) {
    return to_groups<decltype(type)>(aligned, x, x_stride, m, out, (cudaStream_t)stream);
  });
}

extern "C" int cvhrf_groups_to_rows(const void* y, long long y_stride, int dtype, long long n, int choices, int width,
                                    const int* slots, const void* weights, int weights_dtype, void* out,
                                    void* stream) {
  const int rc = check_moves(dtype, n, choices, width);
  if (rc) return rc;
  if (y_stride < 0 || (weights && weights_dtype != CVHRF_F32 && weights_dtype != dtype)) return CVHRF_EINVAL;
  if (n == 0) return CVHRF_OK;
  if (!y || !slots || !out) return CVHRF_EINVAL;
  const bool aligned = rows_16(y, y_stride, width, row_type_bytes(dtype)) && ((uintptr_t)out & 15) == 0;
  const Moves m{n, choices, width, 0, slots, nullptr};
  const Weights w{weights, weights && weights_dtype == dtype};
  return with_type(dtype, [&](auto type) {
    return to_rows<decltype(type)>(aligned, y, y_stride, m, w, out, (cudaStream_t)stream);
  });
}

extern "C" int cvhrf_groups_to_rows_backward(const void* grad, long long grad_stride, const void* y,
                                             long long y_stride, int dtype, long long n, int choices, int width,
                                             const int* slots, const int* used, const void* weights,
                                             int weights_dtype, void* grad_y, void* grad_weights, void* stream) {
  const int rc = check_moves(dtype, n, choices, width);
  if (rc) return rc;
  if (grad_stride < 0 || y_stride < 0 || (weights && weights_dtype != CVHRF_F32 && weights_dtype != dtype) ||
      (grad_weights && !weights))
    return CVHRF_EINVAL;
  if (n == 0 || (!grad_y && !grad_weights)) return CVHRF_OK;
  if (!grad || !slots || !used || (grad_weights && !y)) return CVHRF_EINVAL;
  const size_t elem = row_type_bytes(dtype);
  const bool aligned = rows_16(grad, grad_stride, width, elem) &&
                       (!grad_weights || rows_16(y, y_stride, width, elem)) && ((uintptr_t)grad_y & 15) == 0;
  const Moves m{n, choices, width, 0, slots, used};
  const Weights w{weights, weights && weights_dtype == dtype};
  return with_type(dtype, [&](auto type) {
    return to_rows_backward<decltype(type)>(aligned, grad, grad_stride, y, y_stride, m, w, grad_y, grad_weights,
                                            (cudaStream_t)stream);
  });
}
