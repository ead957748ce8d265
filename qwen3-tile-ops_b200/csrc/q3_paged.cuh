// Device helpers of the ragged paged-cache operators (q3_rope.cu,
// q3_attention_chunk*.cu): 16-bit and 32-bit element rows, and the lookup of a
// row's sequence.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "q3_common.cuh"

namespace q3 {

// bits of the device error word (q3_device_status) that these operators set
constexpr unsigned kBadPage = 1u << 1;       // page index beyond the pool
constexpr unsigned kBadTable = 1u << 2;      // more pages than the table holds
constexpr unsigned kBadPosition = 1u << 4;   // position outside the rotary tables
constexpr unsigned kBadRagged = 1u << 5;     // row0 / kv_len / max_rows do not fit

template <int BYTES>
struct Chunk;
template <>
struct Chunk<1> { using type = uint8_t; };
template <>
struct Chunk<2> { using type = uint16_t; };
template <>
struct Chunk<4> { using type = uint32_t; };
template <>
struct Chunk<8> { using type = uint2; };
template <>
struct Chunk<16> { using type = uint4; };

// N consecutive elements of T as float32 (one vector access of at most 16 bytes each)
template <typename T, int N>
struct Elems {
  static constexpr int BYTES = N * static_cast<int>(sizeof(T)) > 16 ? 16 : N * static_cast<int>(sizeof(T));
  static constexpr int PER = BYTES / static_cast<int>(sizeof(T)), CH = N / PER;
  using V = typename Chunk<BYTES>::type;
  union {
    V v[CH];
    T e[N];
  };
  __device__ __forceinline__ Elems() {}
  __device__ __forceinline__ void load(const void *p) {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = reinterpret_cast<const V *>(p)[i];
  }
  // read and written once: past the caches
  __device__ __forceinline__ void load_stream(const void *p) {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = __ldcs(reinterpret_cast<const V *>(p) + i);
  }
  __device__ __forceinline__ void store_stream(void *p) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) __stcs(reinterpret_cast<V *>(p) + i, v[i]);
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < CH; ++i) v[i] = V{};
  }
  __device__ __forceinline__ void store(void *p) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) reinterpret_cast<V *>(p)[i] = v[i];
  }
};
// float32 of the elements; 16-bit ones two at a time, as a word holds them
template <typename T, int N>
__device__ __forceinline__ void to_f32(const Elems<T, N> &e, float (&x)[N]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = e.e[i];
  } else {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(e.v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(w + i));
        x[2 * i] = y.x, x[2 * i + 1] = y.y;
      } else {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ Elems<T, N> from_f32(const float (&x)[N]) {
  Elems<T, N> e;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) e.e[i] = x[i];
  } else {
    uint32_t *w = reinterpret_cast<uint32_t *>(e.v);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 y = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&y);
      } else {
        const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&y);
      }
    }
  }
  return e;
}
template <typename T, int N>
__device__ __forceinline__ void store_row(const float (&x)[N], void *p) {
  from_f32<T>(x).store(p);
}
template <typename T, int N>
__device__ __forceinline__ void store_row_stream(const float (&x)[N], void *p) {
  from_f32<T>(x).store_stream(p);
}

// Rows first .. end-1 of a sequence do not all exist (none: nothing is missing)
__device__ __forceinline__ bool rows_missing(int first, int end, int rows) {
  return first != end && (first < 0 || end < first || end > rows);
}

// Sequence of row r (whole warp): the last s with row0[s] <= r, or -1 when r
// belongs to nobody.  Each round a warp looks at 32 places of the ascending
// array, so 1024 sequences take two rounds.  Whatever row0 holds, reads stay in
// [0, n_seqs] and the range that comes back contains r.
__device__ __forceinline__ int find_seq(const int32_t *row0, int n_seqs, int r, int lane, int &first,
                                        int &count) {
  int lo = 0, n = n_seqs;   // candidates lo .. lo + n - 1
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lane * step;
    const bool le = at < n && row0[lo + at] <= r;
    const unsigned m = __ballot_sync(0xffffffffu, le);
    const int k = m ? 31 - __clz(m) : 0;
    lo += k * step;
    n = min(step, n - k * step);
  }
  first = row0[lo];
  const int end = row0[lo + 1];
  count = end - first;
  return first >= 0 && first <= r && r < end ? lo : -1;
}

}  // namespace q3
