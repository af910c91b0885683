// Element types and row layouts shared by the row kernels (row_tables.cu, row_moves.cu).
//
// A row of `width` elements is moved in packs.  Three layouts:
//   kAligned  every row begins on 16 bytes and is a multiple of 16 bytes long: a pack is 16 bytes
//             of the row, one load or store.
//   kSpan     rows begin anywhere (an odd width, a slice).  Packs are 16-byte aligned on the side
//             that is written, so that stores stay whole; the elements before the first and
//             behind the last boundary (the edges) are moved one per lane.  A pack's elements lie
//             in two aligned 16-byte words of the row that is read, which are shifted together.
//   kElement  rows of a few elements: one element per lane (a span would be all edges).
#pragma once
#include <atomic>
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

// A tensor that is read.  Where it does not begin and end on 16 bytes, the words at its ends are
// not wholly inside, and the rows that touch them are read by element (Row::load_elements).
struct Extent {
  const char* begin;   // its first byte
  const char* end;     // the byte behind its last one
  bool checked;
  template <typename T>
  __device__ __forceinline__ bool inside(const T* row, int width) const {
    return !checked || (reinterpret_cast<const char*>(row) - 15 >= begin &&
                        reinterpret_cast<const char*>(row + width) + 15 <= end);
  }
};

inline Extent extent_of(const void* p, long long rows, long long stride, int width, size_t elem) {
  const char* b = (const char*)p;
  const char* e = rows > 0 ? b + ((rows - 1) * stride + width) * (long long)elem : b;
  return {b, e, (((uintptr_t)b | (uintptr_t)e) & 15) != 0};
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

// How packs of a row are read and written.  A pack is named by its first element of the row and
// lies wholly inside it.
template <typename T, Layout L>
struct Row {
  static constexpr int kVec = 16 / (int)sizeof(T);
  struct Raw {   // what one pack's loads bring; joined by words()
    uint4 a, b;
    uint32_t shift;
  };
  // elements of a row before its first boundary of 16 bytes
  static __device__ __forceinline__ int head(const T* row, int width) {
    if (L != kSpan) return 0;
    const int ahead = (int)(((uintptr_t)row & 15) / sizeof(T));
    return min(ahead ? kVec - ahead : 0, width);
  }
  static __device__ __forceinline__ Raw load(const T* from) {
    Raw r;
    if (L == kAligned) {
      r.a = *reinterpret_cast<const uint4*>(from);
      return r;
    }
    const char* p = reinterpret_cast<const char*>(from);
    r.shift = (uint32_t)((uintptr_t)p & 15);
    p -= r.shift;
    r.a = *reinterpret_cast<const uint4*>(p);
    // the word with the pack's last element (the same one again if the pack is aligned)
    r.b = *reinterpret_cast<const uint4*>(p + (r.shift ? 16 : 0));
    return r;
  }
  static __device__ __noinline__ uint4 load_words(const T* from) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      if (sizeof(T) == 4) w[i] = reinterpret_cast<const uint32_t*>(from)[i];
      else w[i >> 1] |= (uint32_t) reinterpret_cast<const uint16_t*>(from)[i] << ((i & 1) * 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ Raw load_elements(const T* from) {
    Raw r;
    r.a = load_words(from);
    r.b = r.a;
    r.shift = 0;
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
  static __device__ __forceinline__ void store(T* to, uint4 w) { *reinterpret_cast<uint4*>(to) = w; }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[kVec]) { unpack(words(r), f, (const T*)nullptr); }
  static __device__ __forceinline__ uint4 words(const float (&f)[kVec]) { return pack(f, (const T*)nullptr); }
};

template <typename T>
struct Row<T, kElement> {
  static constexpr int kVec = 1;
  using Raw = T;
  static __device__ __forceinline__ int head(const T*, int) { return 0; }
  static __device__ __forceinline__ Raw load(const T* from) { return *from; }
  static __device__ __forceinline__ Raw load_elements(const T* from) { return *from; }
  static __device__ __forceinline__ T words(const Raw& r) { return r; }
  static __device__ __forceinline__ void store(T* to, T w) { *to = w; }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[1]) { f[0] = to_float(r); }
  static __device__ __forceinline__ T words(const float (&f)[1]) { return from_float<T>(f[0]); }
};

// Where a row's whole packs begin (after `head` elements) and how many there are, and the `count`
// elements outside them: edge(i) for i < count.
struct Edges {
  int head, packs, count, width;
  template <typename R, typename T>
  static __device__ __forceinline__ Edges of(const T* row, int width) {
    Edges e;
    e.head = R::head(row, width);
    e.packs = (width - e.head) / R::kVec;
    e.count = width - e.packs * R::kVec;
    e.width = width;
    return e;
  }
  __device__ __forceinline__ int edge(int i) const { return i < head ? i : width - count + i; }
};

template <typename T, Layout L>
__device__ __forceinline__ auto zero_pack() {
  if constexpr (L == kElement) return from_float<T>(0.f);
  else return zero_words();
}

// Zeros into a row.
template <typename T, Layout L>
__device__ __forceinline__ void clear_row(T* row, int width, int lane, int lanes) {
  using R = Row<T, L>;
  const Edges e = Edges::of<R>(row, width);
  for (int q = lane; q < e.packs; q += lanes) R::store(row + e.head + q * R::kVec, zero_pack<T, L>());
  if (L == kSpan)
    for (int i = lane; i < e.count; i += lanes) row[e.edge(i)] = from_float<T>(0.f);
}

// Whole packs of a row at most.
template <typename T, Layout L>
constexpr int packs_of(int width) {
  return width / Row<T, L>::kVec;
}

constexpr int kMaxWidth = 1 << 20;   // elements of a row at most: columns are counted in int

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

// Rows are owned by `lanes` neighbouring lanes of a warp (not a power of two: rows of 5 packs
// would leave 3 of 8 lanes idle); a warp has 32 / lanes owners.
struct Owner {
  int index, lane;   // the owner in its block, the lane in its owner
  bool live;
  static __device__ __forceinline__ Owner of(int lanes) {
    const int in_warp = threadIdx.x & 31, each = 32 / lanes, o = in_warp / lanes;
    return {(int)(threadIdx.x >> 5) * each + o, in_warp - o * lanes, o < each};
  }
};
inline int owners_of(int threads, int lanes) { return threads / 32 * (32 / lanes); }
// A row's lanes: its packs, a warp at most, or half of one where that leaves fewer idle.
inline int lanes_for(int packs) {
  if (packs <= 32) return packs < 1 ? 1 : packs;
  return (packs + 31) / 32 * 2 > (packs + 15) / 16 ? 16 : 32;
}

// Blocks that share the columns of one block's rows (the y dimension), where the rows alone leave
// SMs without work, so that there are about `per_sm` of them per SM; `steps`: the parts that a row
// can be taken in.  (The sum of 64 rows of 4096 bf16 from 8 choices: 3.9 us, 23.5 by a warp per row.)
inline unsigned parts_for(unsigned blocks, int steps, unsigned per_sm = 4) {
  const unsigned want = 148u * per_sm / (blocks ? blocks : 1u);
  return want <= 1 || steps <= 1 ? 1u : want < (unsigned)steps ? want : (unsigned)steps;
}

// ---- launches that follow one another ----------------------------------------------------
// A kernel launched with launch_after may start while the one before it ends; it calls
// follow() before it touches memory, which waits until that one is done and its writes seen.
// What the kernel before writes is written while this one is already on the GPU, so it must not be
// read as `const ... __restrict__`: that lets the compiler take it for constant as long as the
// kernel runs and read it by the read-only path, whose loads neither follow() orders nor the
// writes reach.  Only what the caller hands in may be (the first kernel of a chain, launched
// plainly, has waited for it).
__device__ __forceinline__ void follow() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
// ... and the one before it says early that the next one may start.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... P, typename... A>
inline cudaError_t launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t st, A... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Lets a kernel use `bytes` of dynamic shared memory, once per device.
template <typename K>
inline cudaError_t allow_shared(K* kernel, size_t bytes, std::atomic<unsigned long long>& devices) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = 1ull << (dev & 63);
  if (devices.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess) devices.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace cvhrf
