// Element types and row layouts shared by the row kernels (row_tables.cu, row_moves.cu).
//
// A row of `width` elements is moved in packs.  Three layouts:
//   kAligned  every row begins on 16 bytes and is a multiple of 16 bytes long: a pack is 16 bytes
//             of the row, one load or store.
//   kSpan     rows begin anywhere (an odd width, a slice).  Packs are 16-byte aligned on the side
//             that is written, so that stores stay whole; the first and the last pack of a row
//             are partial and stored by element.  A pack's elements lie in two aligned 16-byte
//             words of the row that is read, which are shifted together.  By element, a warp needs
//             4 (float32) or 8 (16 bits) times the instructions, and was bound by them: 141 us
//             against 55 us for 1M rows of 59 floats.
//   kElement  rows of a few elements: one element per lane (a span would be all edges).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace cvhrf {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

enum Layout { kAligned, kSpan, kElement };

// A tensor that is read: its first byte and the byte behind its last one.  A 16-byte word that
// is not wholly inside is read by element.
struct Extent {
  const char* begin;
  const char* end;
};

inline Extent extent_of(const void* p, long long rows, long long stride, int width, size_t elem) {
  const char* b = (const char*)p;
  return {b, rows > 0 ? b + ((rows - 1) * stride + width) * (long long)elem : b};
}

__device__ __forceinline__ uint4 zero_words() { return make_uint4(0u, 0u, 0u, 0u); }

// Elements of type T in 16 bytes, as floats and back.
__device__ __forceinline__ void unpack(uint4 w, float (&f)[4], const float*) {
  f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack(uint4 w, float (&f)[8], const __nv_bfloat16*) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {   // a bfloat16 is the upper half of its float
    f[2 * i] = __uint_as_float(x[i] << 16);
    f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack(uint4 w, float (&f)[8], const __half*) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
    f[2 * i] = v.x, f[2 * i + 1] = v.y;
  }
}
__device__ __forceinline__ uint4 pack(const float (&f)[4], const float*) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __nv_bfloat16*) {
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    x[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ uint4 pack(const float (&f)[8], const __half*) {
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    x[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(x[0], x[1], x[2], x[3]);
}

// How packs of a row are read and written.  A pack is named by its first element `e` of the
// row; it may begin before the row or end behind it (kSpan), what lies outside is undefined
// when read and not written.
template <typename T, Layout L>
struct Row {
  static constexpr int kVec = 16 / (int)sizeof(T);
  struct Raw {   // what one pack's loads bring; joined by words()
    uint4 a, b;
    uint32_t shift;
  };
  // elements by which the written row is ahead of a 16-byte boundary
  static __device__ __forceinline__ int ahead(const T* row) {
    return L == kSpan ? (int)(((uintptr_t)row & 15) / sizeof(T)) : 0;
  }
  static __device__ __forceinline__ Raw load(const T* row, int e, int width, const Extent& x) {
    Raw r;
    if (L == kAligned) {
      r.a = *reinterpret_cast<const uint4*>(row + e);
      return r;
    }
    const char* p = reinterpret_cast<const char*>(row) + (long long)e * (int)sizeof(T);
    r.shift = (uint32_t)((uintptr_t)p & 15);
    const char* at = p - r.shift;
    if (at >= x.begin && at + 32 <= x.end) {
      r.a = *reinterpret_cast<const uint4*>(at);
      r.b = r.shift ? *reinterpret_cast<const uint4*>(at + 16) : zero_words();
    } else {   // at the tensor's ends
      r.shift = 0;
      r.a = zero_words();
      uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < kVec; ++i)
        if (e + i >= 0 && e + i < width) {
          if (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t*>(row)[e + i];
          else w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(row)[e + i] << ((i & 1) * 16);
        }
      r.a = make_uint4(w[0], w[1], w[2], w[3]);
      r.b = zero_words();
    }
    return r;
  }
  static __device__ __forceinline__ uint4 words(const Raw& r) {
    if (L == kAligned) return r.a;
    uint32_t x[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
    if (r.shift & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) x[i] = x[i + 2];
    }
    if (r.shift & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) x[i] = x[i + 1];
    }
    if (sizeof(T) == 2) {
      const uint32_t bits = (r.shift & 2) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = __funnelshift_r(x[i], x[i + 1], bits);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
  }
  static __device__ __forceinline__ void store(T* row, int e, int width, uint4 w) {
    if (L == kAligned || (e >= 0 && e + kVec <= width)) {
      *reinterpret_cast<uint4*>(row + e) = w;
    } else {
      store_by_element(row, e, width, w);
    }
  }
  static __device__ __forceinline__ void store_by_element(T* row, int e, int width, uint4 w) {
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < kVec; ++i)
      if (e + i >= 0 && e + i < width) {
        if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(row)[e + i] = x[i];
        else reinterpret_cast<uint16_t*>(row)[e + i] = (uint16_t)(x[i >> 1] >> ((i & 1) * 16));
      }
  }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[kVec]) { unpack(words(r), f, (const T*)nullptr); }
  static __device__ __forceinline__ uint4 words(const float (&f)[kVec]) { return pack(f, (const T*)nullptr); }
};

template <typename T>
struct Row<T, kElement> {
  static constexpr int kVec = 1;
  using Raw = T;
  static __device__ __forceinline__ int ahead(const T*) { return 0; }
  static __device__ __forceinline__ Raw load(const T* row, int e, int, const Extent&) { return row[e]; }
  static __device__ __forceinline__ T words(const Raw& r) { return r; }
  static __device__ __forceinline__ void store(T* row, int e, int, T w) { row[e] = w; }
  static __device__ __forceinline__ void store_by_element(T* row, int e, int, T w) { row[e] = w; }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[1]) { f[0] = to_float(r); }
  static __device__ __forceinline__ T words(const float (&f)[1]) { return from_float<T>(f[0]); }
};

template <typename T, Layout L>
__device__ __forceinline__ auto zero_pack() {
  if constexpr (L == kElement) return from_float<T>(0.f);
  else return zero_words();
}

// Packs that cover a row wherever it begins.
template <typename T, Layout L>
__host__ __device__ constexpr int packs_of(int width) {
  constexpr int vec = 16 / (int)sizeof(T);
  return L == kElement ? width : L == kAligned ? width / vec : (width + vec - 1) / vec + 1;
}

inline size_t row_type_bytes(int dtype) { return dtype == CVHRF_F32 ? 4 : 2; }
inline bool row_type_ok(int dtype) { return dtype == CVHRF_F32 || dtype == CVHRF_BF16 || dtype == CVHRF_F16; }
inline int next_pow2(int x) {
  int p = 1;
  while (p < x) p <<= 1;
  return p;
}

// Whether rows of `width` elements every `stride` elements from p all begin on 16 bytes and
// end there (torch's own allocations are aligned; slices and odd widths need not be).
inline bool rows_16(const void* p, long long stride, int width, size_t elem) {
  return ((uintptr_t)p & 15) == 0 && (stride * (long long)elem) % 16 == 0 && ((size_t)width * elem) % 16 == 0;
}

// A span's edges are up to two packs' worth of single elements, so it pays from this many on.
constexpr int kSpanWidth = 32;

}  // namespace cvhrf
