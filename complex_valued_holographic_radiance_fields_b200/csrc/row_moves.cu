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

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> zero_pack() {
  Pack<T, VEC> z;
#pragma unroll
  for (int i = 0; i < VEC; ++i) z.v[i] = from_float<T>(0.f);
  return z;
}

// Zeros into the rows behind the last group, shared out between the owners (row n takes
// every n-th of them, `choices` at most).
template <typename T, int VEC>
__device__ __forceinline__ void clear_behind(const Moves& m, long long row, int lane, T* __restrict__ out) {
  const long long places = m.n * m.choices;
  for (long long p = *m.used + row; p < places; p += m.n)
    for (int c = lane * VEC; c < m.width; c += m.lanes * VEC)
      *(Pack<T, VEC>*)(out + p * m.width + c) = zero_pack<T, VEC>();
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) rows_to_groups_kernel(Moves m, const T* __restrict__ x, long long stride,
                                                                  T* __restrict__ out) {
  const long long row = (long long)blockIdx.x * (kThreads / m.lanes) + threadIdx.x / m.lanes;
  const int lane = threadIdx.x & (m.lanes - 1);
  if (row >= m.n) return;
  const int* slots = m.slots + row * m.choices;
  for (int c = lane * VEC; c < m.width; c += m.lanes * VEC) {
    const Pack<T, VEC> p = *(const Pack<T, VEC>*)(x + row * stride + c);
    for (int j = 0; j < m.choices; ++j) {
      const int s = slots[j];
      if (s >= 0) *(Pack<T, VEC>*)(out + (long long)s * m.width + c) = p;
    }
  }
  clear_behind<T, VEC>(m, row, lane, out);
}

template <typename T, int VEC, typename W>
__global__ void __launch_bounds__(kThreads) groups_to_rows_kernel(Moves m, const T* __restrict__ y, long long stride,
                                                                  const W* __restrict__ weights,
                                                                  T* __restrict__ out) {
  const long long row = (long long)blockIdx.x * (kThreads / m.lanes) + threadIdx.x / m.lanes;
  const int lane = threadIdx.x & (m.lanes - 1);
  if (row >= m.n) return;
  const int* slots = m.slots + row * m.choices;
  for (int c = lane * VEC; c < m.width; c += m.lanes * VEC) {
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (int j = 0; j < m.choices; ++j) {
      const int s = slots[j];
      if (s < 0) continue;   // whatever its weight holds
      const Pack<T, VEC> p = *(const Pack<T, VEC>*)(y + (long long)s * stride + c);
      const float w = weights ? to_float(weights[row * m.choices + j]) : 1.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) acc[i] = fmaf(w, to_float(p.v[i]), acc[i]);
    }
    Pack<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = from_float<T>(acc[i]);
    *(Pack<T, VEC>*)(out + row * m.width + c) = o;
  }
}

template <typename T, int VEC, typename W>
__global__ void __launch_bounds__(kThreads) groups_to_rows_backward_kernel(
    Moves m, const T* __restrict__ grad, long long grad_stride, const T* __restrict__ y, long long stride,
    const W* __restrict__ weights, T* __restrict__ grad_y, W* __restrict__ grad_weights) {
  const long long row = (long long)blockIdx.x * (kThreads / m.lanes) + threadIdx.x / m.lanes;
  const int lane = threadIdx.x & (m.lanes - 1);
  const bool live = row < m.n;
  const int* slots = m.slots + row * m.choices;
  for (int j = 0; j < m.choices; ++j) {
    const int s = live ? slots[j] : -1;
    float dot = 0.f;
    if (s >= 0) {
      const float w = weights ? to_float(weights[row * m.choices + j]) : 1.f;
#pragma unroll 2
      for (int c = lane * VEC; c < m.width; c += m.lanes * VEC) {
        const Pack<T, VEC> g = *(const Pack<T, VEC>*)(grad + row * grad_stride + c);
        if (grad_weights) {
          const Pack<T, VEC> p = *(const Pack<T, VEC>*)(y + (long long)s * stride + c);
#pragma unroll
          for (int i = 0; i < VEC; ++i) dot = fmaf(to_float(g.v[i]), to_float(p.v[i]), dot);
        }
        if (grad_y) {
          Pack<T, VEC> o;
#pragma unroll
          for (int i = 0; i < VEC; ++i) o.v[i] = from_float<T>(w * to_float(g.v[i]));
          *(Pack<T, VEC>*)(grad_y + (long long)s * m.width + c) = o;
        }
      }
    }
    if (grad_weights) {
      for (int o = m.lanes >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (live && lane == 0) grad_weights[row * m.choices + j] = from_float<W>(dot);
    }
  }
  if (live && grad_y) clear_behind<T, VEC>(m, row, lane, grad_y);
}

struct Launch {
  Moves m;
  unsigned blocks;
};

template <int VEC>
Launch launch_for(long long n, int choices, int width, const int* slots, const int* used) {
  const int packs = (width + VEC - 1) / VEC;
  const int lanes = next_pow2(packs < 32 ? packs : 32);
  const int rows = kThreads / lanes;
  return {{n, choices, width, lanes, slots, used}, (unsigned)((n + rows - 1) / rows)};
}

template <typename T, int VEC>
int to_groups(const void* x, long long stride, long long n, int choices, int width, const int* slots, const int* used,
              void* out, cudaStream_t st) {
  const Launch l = launch_for<VEC>(n, choices, width, slots, used);
  rows_to_groups_kernel<T, VEC><<<l.blocks, kThreads, 0, st>>>(l.m, (const T*)x, stride, (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T, int VEC, typename W>
int to_rows(const void* y, long long stride, long long n, int choices, int width, const int* slots,
            const void* weights, void* out, cudaStream_t st) {
  const Launch l = launch_for<VEC>(n, choices, width, slots, nullptr);
  groups_to_rows_kernel<T, VEC, W><<<l.blocks, kThreads, 0, st>>>(l.m, (const T*)y, stride, (const W*)weights,
                                                                 (T*)out);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

template <typename T, int VEC, typename W>
int to_rows_backward(const void* grad, long long grad_stride, const void* y, long long stride, long long n,
                     int choices, int width, const int* slots, const int* used, const void* weights, void* grad_y,
                     void* grad_weights, cudaStream_t st) {
  const Launch l = launch_for<VEC>(n, choices, width, slots, used);
  groups_to_rows_backward_kernel<T, VEC, W><<<l.blocks, kThreads, 0, st>>>(
      l.m, (const T*)grad, grad_stride, (const T*)y, stride, (const W*)weights, (T*)grad_y, (W*)grad_weights);
  CVHRF_LAUNCH_CHECK();
  return CVHRF_OK;
}

int check_moves(int dtype, long long n, int choices, int width) {
  if (!row_type_ok(dtype) || n < 0 || choices < 1 || width < 1) return CVHRF_EINVAL;
  if (n > kGroupMaxEntries / choices) return CVHRF_EUNSUPPORTED;
  return CVHRF_OK;
}

// CALL<type, packed>(...) for the element type and whether rows move 16 bytes at a time
#define CVHRF_ROW_DISPATCH(dtype, wide, CALL32, CALL32W, CALLB, CALLBW, CALLH, CALLHW) \
  (dtype == CVHRF_F32    ? (wide ? CALL32W : CALL32)                                   \
   : dtype == CVHRF_BF16 ? (wide ? CALLBW : CALLB)                                     \
                         : (wide ? CALLHW : CALLH))

}  // namespace
}  // namespace cvhrf

using namespace cvhrf;
using bf16 = __nv_bfloat16;
using f16 = __half;

extern "C" int cvhrf_rows_to_groups(const void* x, long long x_stride, int dtype, long long n, int choices, int width,
                                    const int* slots, const int* used, void* out, void* stream) {
  const int rc = check_moves(dtype, n, choices, width);
  if (rc) return rc;
  if (x_stride < 0) return CVHRF_EINVAL;
  if (n == 0) return CVHRF_OK;
  if (!x || !slots || !used || !out) return CVHRF_EINVAL;
  const bool wide = rows_16(x, x_stride, width, row_type_bytes(dtype)) && ((uintptr_t)out & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
#define CVHRF_CALL(T, V) to_groups<T, V>(x, x_stride, n, choices, width, slots, used, out, st)
  return CVHRF_ROW_DISPATCH(dtype, wide, CVHRF_CALL(float, 1), CVHRF_CALL(float, 4), CVHRF_CALL(bf16, 1),
                            CVHRF_CALL(bf16, 8), CVHRF_CALL(f16, 1), CVHRF_CALL(f16, 8));
#undef CVHRF_CALL
}

extern "C" int cvhrf_groups_to_rows(const void* y, long long y_stride, int dtype, long long n, int choices, int width,
                                    const int* slots, const void* weights, int weights_dtype, void* out,
                                    void* stream) {
  const int rc = check_moves(dtype, n, choices, width);
  if (rc) return rc;
  if (y_stride < 0 || (weights && weights_dtype != CVHRF_F32 && weights_dtype != dtype)) return CVHRF_EINVAL;
  if (n == 0) return CVHRF_OK;
  if (!y || !slots || !out) return CVHRF_EINVAL;
  const bool wide = rows_16(y, y_stride, width, row_type_bytes(dtype)) && ((uintptr_t)out & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
#define CVHRF_CALL(T, V)                                                                                     \
  (!weights || weights_dtype == CVHRF_F32 ? to_rows<T, V, float>(y, y_stride, n, choices, width, slots, weights, out, st) \
                                          : to_rows<T, V, T>(y, y_stride, n, choices, width, slots, weights, out, st))
  return CVHRF_ROW_DISPATCH(dtype, wide, CVHRF_CALL(float, 1), CVHRF_CALL(float, 4), CVHRF_CALL(bf16, 1),
                            CVHRF_CALL(bf16, 8), CVHRF_CALL(f16, 1), CVHRF_CALL(f16, 8));
#undef CVHRF_CALL
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
  const bool wide = rows_16(grad, grad_stride, width, elem) && (!grad_weights || rows_16(y, y_stride, width, elem)) &&
                    ((uintptr_t)grad_y & 15) == 0;
  cudaStream_t st = (cudaStream_t)stream;
#define CVHRF_CALL(T, V)                                                                                        \
  (!weights || weights_dtype == CVHRF_F32                                                                       \
       ? to_rows_backward<T, V, float>(grad, grad_stride, y, y_stride, n, choices, width, slots, used, weights, \
                                       grad_y, grad_weights, st)                                                \
       : to_rows_backward<T, V, T>(grad, grad_stride, y, y_stride, n, choices, width, slots, used, weights,     \
                                   grad_y, grad_weights, st))
  return CVHRF_ROW_DISPATCH(dtype, wide, CVHRF_CALL(float, 1), CVHRF_CALL(float, 4), CVHRF_CALL(bf16, 1),
                            CVHRF_CALL(bf16, 8), CVHRF_CALL(f16, 1), CVHRF_CALL(f16, 8));
#undef CVHRF_CALL
}
