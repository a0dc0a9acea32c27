// Device helpers of the ragged steps: packed rows, and the checks of the
// starts, lengths and page-table entries that live in device memory.
#pragma once
#include "common.cuh"

namespace spock {

// The first report stays until the host reads it.
__device__ __forceinline__ void report_bad_index(int* err) { atomicCAS(err, 0, kErrBadIndex); }

// Rows [lo, lo + n) of sequence b, cut to the `total` rows that exist.
struct RowSpan {
  int lo, n;
};
__device__ __forceinline__ RowSpan row_span(const int32_t* __restrict__ start, int b, int total, int* err) {
  const int lo = start[b], hi = start[b + 1];
  if (lo < 0 || hi < lo || hi > total) {
    report_bad_index(err);
    return {0, 0};
  }
  return {lo, hi - lo};
}

// The sequence that owns packed row `row`, by all 32 lanes of a warp: each
// round narrows the candidates [lo, hi) 32-fold. -1 for a row behind the last
// sequence (or before the first, or in starts that do not ascend).
__device__ __forceinline__ int seq_of_row(const int32_t* __restrict__ start, int batch, int row, int lane) {
  int lo = 0, hi = batch;  // the first b with start[b + 1] > row, if any, is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int probe = min(lo + (lane + 1) * step, hi) - 1;  // the last of this lane's slice
    const unsigned hit = __ballot_sync(0xffffffffu, start[probe + 1] > row);
    if (!hit) return -1;
    lo += (__ffs(hit) - 1) * step;
    hi = min(hi, lo + step);
  }
  return start[lo] <= row && row < start[lo + 1] ? lo : -1;
}

// 16-bit storage types.
template <typename T>
struct Io;
template <>
struct Io<__half> {
  static __device__ __forceinline__ float2 up2(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
  static __device__ __forceinline__ uint32_t down2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Io<__nv_bfloat16> {
  static __device__ __forceinline__ float2 up2(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t down2(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N 32-bit words (2 N values) at a 4 N-byte aligned address.
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
template <int N>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[N]) {
  if constexpr (N == 4) {
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  } else {
    *reinterpret_cast<uint32_t*>(p) = w[0];
  }
}

}  // namespace spock
