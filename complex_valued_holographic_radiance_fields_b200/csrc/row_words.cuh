// Rows that do not begin on 16 bytes, moved in 4-byte words where they do not go through a tile
// (row_tiles.cuh): rows of more than 4 KB, and outputs that do not begin on 16 bytes.
//
// A word is one float32 or two 16-bit elements, aligned on the row that is written; with 16-bit
// elements the row that is read may begin on the other half of a word, and then two of its
// words are shifted together.  The element before the first word and the one behind the last
// (the edges) are moved by themselves.  Neighbouring lanes hold neighbouring words, so loads and
// stores are whole lines up to their ends.  What is done per row (its place, its address, its
// edges) is as much work as the words of a short row, so a warp takes up to 32 entries, each
// lane works out one of them, and the owners of rows get them by shuffle.
#pragma once
#include "row_tiles.cuh"

namespace cvhrf {

constexpr int kWordThreads = 256;

// The tensor that is read.  Where it does not begin and end on 4 bytes, the words at its ends
// are not wholly inside it; `ends`: 0 they are, 1 the first and the last row are read by element,
// 2 every row is (rows that overlap).
struct Source4 {
  long long stride;   // bytes between its rows
  int last;           // index of the last row
  int ends;
  __device__ __forceinline__ bool by_element(int i) const { return ends != 0 && (ends == 2 || i == 0 || i == last); }
};

inline Source4 source4_of(const void* p, long long rows, long long stride, int width, size_t elem) {
  const long long bytes = stride * (long long)elem;
  const uintptr_t b = (uintptr_t)p, e = b + (size_t)((rows > 0 ? (rows - 1) * bytes : 0) + width * (long long)elem);
  return {bytes, (int)(rows - 1), ((b | e) & 3) == 0 ? 0 : bytes >= 4 ? 1 : 2};
}

// Words of a row at most.
template <typename T>
inline int words_of(int width) {
  return width / (4 / (int)sizeof(T));
}

// Where a row that is read has the elements of the words of the row that is written: words of
// memory and the bits by which they are shifted.  Packed into its address: the address of the
// first element (its bit 1 is the shift, which 4-byte elements never have), bit 0: to be read by
// element; 0: no row.
struct From {
  const uint32_t* at;
  uint32_t shift;   // 0 or 16
  bool by_element;
  __device__ __forceinline__ explicit From(unsigned long long packed)
      : at(reinterpret_cast<const uint32_t*>(packed & ~3ull)), shift((uint32_t)(packed & 2) * 8), by_element(packed & 1) {}
  static __device__ __forceinline__ unsigned long long pack(const void* first, bool by_element) {
    return (unsigned long long)(uintptr_t)first | (by_element ? 1u : 0u);
  }
};
// A row that is written, packed into the address of its first word; bit 0: an element before it;
// 0: no row.
template <typename T>
struct To {
  uint32_t* at;
  int head, words, tail;
  __device__ __forceinline__ To(unsigned long long packed, int width) {
    at = reinterpret_cast<uint32_t*>(packed & ~1ull);
    head = sizeof(T) == 4 ? 0 : (int)(packed & 1);
    words = !packed ? 0 : sizeof(T) == 4 ? width : (width - head) >> 1;
    tail = sizeof(T) == 4 || !packed ? 0 : (width - head) & 1;
  }
  static __device__ __forceinline__ unsigned long long pack(const T* row) {
    if (sizeof(T) == 4) return (unsigned long long)(uintptr_t)row;
    const unsigned long long head = (uintptr_t)row >> 1 & 1;
    return (unsigned long long)(uintptr_t)(row + head) | head;
  }
};

struct RawWord {
  uint32_t a, b;
};
// The same word by element, for words at the ends of the tensor.
__device__ __noinline__ RawWord load_word_elements(const uint32_t* at, uint32_t shift) {
  const uint16_t* p = reinterpret_cast<const uint16_t*>(at) + (shift >> 4);
  const uint32_t v = (uint32_t)p[0] | (uint32_t)p[1] << 16;
  return {v << shift, v >> (shift ? 16 : 0)};   // as the two words it would lie in
}
template <typename T>
__device__ __forceinline__ RawWord load_word(const From& f, const uint32_t* at, bool slow) {
  if (sizeof(T) == 4) return {*at, 0u};
  if (slow && f.by_element) return load_word_elements(at, f.shift);
  return {at[0], at[f.shift ? 1 : 0]};   // b holds the word's second element
}
template <typename T>
__device__ __forceinline__ uint32_t join_word(const From& f, const RawWord& r) {
  return sizeof(T) == 4 ? r.a : __funnelshift_r(r.a, r.b, f.shift);
}

// The elements of a word.
__device__ __forceinline__ void word_floats(uint32_t w, float (&f)[1], const float*) { f[0] = __uint_as_float(w); }
__device__ __forceinline__ void word_floats(uint32_t w, float (&f)[2], const __nv_bfloat16*) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xffff0000u);
}
__device__ __forceinline__ void word_floats(uint32_t w, float (&f)[2], const __half*) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = v.x, f[1] = v.y;
}
__device__ __forceinline__ uint32_t floats_word(const float (&f)[1], const float*) { return __float_as_uint(f[0]); }
__device__ __forceinline__ uint32_t floats_word(const float (&f)[2], const __nv_bfloat16*) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t floats_word(const float (&f)[2], const __half*) {
  const __half2 v = __floats2half2_rn(f[0], f[1]);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Entries of a warp: 32, or fewer where that would leave SMs without work (`rounds` rounds of
// the warp's owners).
inline int rounds_for(long long entries, int owners, int in_flight) {
  const int most = (32 + owners - 1) / owners;
  long long r = entries / (148ll * 24 * owners);
  r = r / in_flight * in_flight;
  if (r < in_flight) r = in_flight;
  return (int)(r < most ? r : most);
}

// Copies rows: entry e's row `from` (-1: zeros) to place `to` (-1: nowhere), as get(e, from, to)
// says, times scale (SCALE; else bit for bit).  An owner has FLIGHT rows in flight, J words of
// each; LANES: the lanes of an owner where they are a whole warp, else 0.
template <typename T, bool SCALE, int LANES, int FLIGHT, int J, typename Get>
__device__ __forceinline__ void copy_rows(const Get& get, long long entries, int rounds, int any_lanes, int width,
                                          const T* __restrict__ x, const Source4& source, float scale,
                                          T* __restrict__ out) {
  constexpr int kEach = 4 / (int)sizeof(T);
  const int lanes = LANES ? LANES : any_lanes, owners = LANES ? 1 : 32 / lanes;
  const int lane = threadIdx.x & 31, owner = LANES ? 0 : lane / lanes, word = LANES ? lane : lane - owner * lanes;
  const int tile = min(rounds * owners, 32);
  const long long first = ((long long)blockIdx.x * (kWordThreads / 32) + (threadIdx.x >> 5)) * tile;
  const int n = (int)min((long long)tile, entries - first);
  if (n <= 0) return;
  unsigned long long my_from = 0, my_to = 0;
  if (lane < n) {
    int from = -1, to = -1;
    get(first + lane, from, to);
    if (to >= 0) my_to = To<T>::pack(out + (long long)to * width);
    if (to >= 0 && from >= 0)
      my_from = From::pack(reinterpret_cast<const char*>(x) + from * source.stride + (sizeof(T) == 2 ? 2 * (my_to & 1) : 0),
                           sizeof(T) == 2 && source.by_element(from));
  }
  const bool slow = sizeof(T) == 2 && __any_sync(0xffffffffu, my_from & 1);
  for (int r = 0; r < n; r += owners * FLIGHT) {
    unsigned long long from[FLIGHT], to[FLIGHT];
#pragma unroll
    for (int q = 0; q < FLIGHT; ++q) {
      const int src = r + q * owners + owner;   // a lane at or behind n has no row
      from[q] = shuffle(my_from, src & 31);
      to[q] = shuffle(my_to, src & 31);
      if (!LANES && (owner >= owners || src > 31)) from[q] = to[q] = 0;
    }
    for (int c = word + (int)blockIdx.y * lanes * J; c < width / kEach; c += lanes * J * (int)gridDim.y) {
      RawWord v[FLIGHT][J];
#pragma unroll
      for (int q = 0; q < FLIGHT; ++q) {
        const From f(from[q]);
        const int words = To<T>(to[q], width).words;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          v[q][j] = {0u, 0u};
          if (from[q] && c + j * lanes < words) v[q][j] = load_word<T>(f, f.at + c + j * lanes, slow);
        }
      }
#pragma unroll
      for (int q = 0; q < FLIGHT; ++q) {
        const From f(from[q]);
        const To<T> t(to[q], width);
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (c + j * lanes < t.words) {
            uint32_t o = join_word<T>(f, v[q][j]);
            if (SCALE) {
              float e[kEach];
              word_floats(o, e, (const T*)nullptr);
#pragma unroll
              for (int i = 0; i < kEach; ++i) e[i] *= scale;
              o = from[q] ? floats_word(e, (const T*)nullptr) : 0u;
            }
            t.at[c + j * lanes] = o;
          }
      }
    }
    if (sizeof(T) == 2 && blockIdx.y == 0) {
#pragma unroll
      for (int q = 0; q < FLIGHT; ++q) {
        const To<T> t(to[q], width);
        const T* s = reinterpret_cast<const T*>(from[q] & ~1ull);
        auto edge = [&](int e) {   // e: counted from the first word
          T* d = reinterpret_cast<T*>(t.at) + e;
          if (!from[q]) *d = from_float<T>(0.f);
          else *d = SCALE ? from_float<T>(scale * to_float(s[e])) : s[e];
        };
        if (t.head && word == 0) edge(-1);
        if (t.tail && word == lanes - 1) edge(2 * t.words);
      }
    }
  }
}

// Lanes of a row of `words` words; a row of none has one lane for its edges.
inline int word_lanes(int words) { return words < 1 ? 1 : words < 32 ? words : 32; }
inline unsigned word_blocks(long long entries, int rounds, int owners) {
  const int tile = rounds * owners < 32 ? rounds * owners : 32;
  const long long warps = (entries + tile - 1) / tile, per_block = kWordThreads / 32;
  return (unsigned)((warps + per_block - 1) / per_block);
}

}  // namespace cvhrf
