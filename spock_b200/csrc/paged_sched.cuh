// How spock_paged_attention cuts a ragged batch into equal shares.
//
// A row tile is `tp` whole tokens of one sequence times the G query heads of one
// kv head (tp = R / G; R = 128, or 16 in the kernel for few rows); its work is
// the KV tiles of kTile positions that its last token sees, at least one (a row
// tile that sees nothing still has zeros to write). Starting and finishing a row
// tile takes as long as `extra` KV tiles. All row tiles' units (extra, then KV tiles), in the
// order sequence, kv head, row tile, form one line; share c of C is units
// [U c / C, U (c + 1) / C); where parts are dear its borders are moved off short
// row tiles (enter_share). A row tile cut by a border is computed in parts and
// joined afterwards, so one long sequence, many short ones and any mix all keep
// every SM busy without the host knowing any length.
#pragma once
#include <stdint.h>

namespace spock {
namespace sched {

constexpr int kTile = 128;

// sum of floor(j / p) over j in [0, x)
__host__ __device__ inline int64_t steps_sum(uint32_t x, uint32_t p) {
  const uint32_t k = x / p;
  return (int64_t)((uint64_t)k * (k > 0 ? k - 1 : 0) / 2) * p + (int64_t)k * (x - k * p);
}
// sum of floor((b + i a) / kTile) over i in [0, n), a <= kTile, without divisions
// of 64 bits. Where a divides kTile (group sizes that are powers of two) the terms
// rise by one every kTile / a: floor((b + i a) / kTile) = floor((b / a + i) / (kTile / a)).
// Otherwise Euclid's steps on (a, m), some 3000 cycles.
__host__ __device__ __noinline__ inline int64_t floor_sum(uint32_t n, uint32_t a, uint32_t b) {
  int64_t s = (int64_t)n * (b / kTile);
  b %= kTile;
  if (kTile % a == 0) {
    const uint32_t c = b / a, p = kTile / a;
    return s + steps_sum(c + n, p) - steps_sum(c, p);
  }
  uint32_t m = kTile;
#pragma unroll 1
  while (n > 0) {
    if (a >= m) {
      s += (int64_t)((uint64_t)n * (n - 1) / 2) * (a / m);
      a %= m;
    }
    s += (int64_t)n * (b / m);
    b %= m;
    // y = a n + b = m (a (n / m)) + (a (n % m) + b)
    const uint32_t low = a * (n % m) + b;
    n = a * (n / m) + low / m;  // 0: y < m
    b = low % m;
    const uint32_t t = a;
    a = m;
    m = t;
  }
  return s;
}

// KV tiles of row tile j of a sequence with n new tokens out of len positions
__host__ __device__ inline int row_tile_units(int n, int len, int tp, int j) {
  const int64_t end = (int64_t)(j + 1) * tp;
  const int seen = len - n + (end < n ? (int)end : n);
  return seen <= kTile ? 1 : (int)(((uint32_t)seen + kTile - 1) / kTile);
}
// the same summed over row tiles 0 .. j-1, none of them the last
__host__ __device__ __noinline__ inline int64_t units_before(int n, int len, int tp, int j) {
  if (j == 0) return 0;
  const int off = len - n;
  int j0 = off < 0 ? -off / tp : 0;  // row tiles that see nothing: one unit each
  if (j0 >= j) return j;
  return j0 + floor_sum(j - j0, tp, (uint32_t)off + (uint32_t)(j0 + 1) * tp + kTile - 1);
}
__host__ __device__ inline int row_tiles(int n, int tp) { return n <= 0 ? 0 : (n + tp - 1) / tp; }
__host__ __device__ inline int64_t head_units(int n, int len, int tp) {
  if (n <= 0) return 0;
  const int last = row_tiles(n, tp) - 1;
  if (last == 0) return row_tile_units(n, len, tp, 0);
  return units_before(n, len, tp, last) + row_tile_units(n, len, tp, last);
}
// units c / shares, in divisions of 32 bits: units < 2^51, shares <= 2^12
__host__ __device__ inline int64_t share_begin(int64_t units, int c, int shares) {
  const uint32_t hi = (uint32_t)(units >> 20), lo = (uint32_t)units & 0xfffffu, m = (uint32_t)shares;
  const uint32_t low = hi % m << 20 | lo;
  const int64_t q = (int64_t)(hi / m) << 20 | low / m;
  return q * c + low % m * (uint32_t)c / m;
}

}  // namespace sched
}  // namespace spock
