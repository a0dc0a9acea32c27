// How spock_paged_attention cuts a ragged batch into equal shares.
//
// A row tile is `tp` whole tokens of one sequence times the G query heads of one
// kv head (tp = R / G, at most R = 128 rows, or 16 or 32 in the kernel for few
// rows); its work is the KV tiles of kTile
// positions that its last token sees, at least one (a row tile that sees
// nothing still has zeros to write). Starting and finishing a row tile takes as
// long as `extra` KV tiles. All row tiles' units (extra, then KV tiles), in the
// order sequence, kv head, row tile, form one line; share c of C is units
// [U c / C, U (c + 1) / C), its borders moved off short row tiles. A row tile cut by a border is computed in parts and joined afterwards, so one long
// sequence, many short ones and any mix all keep every SM busy without the host
// knowing any length.
#pragma once
#include <stdint.h>

namespace spock {
namespace sched {

constexpr int kTile = 128;

// sum of floor((b + i a) / m) over i in [0, n): Euclid's steps on (a, m)
__host__ __device__ __noinline__ inline int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t s = 0;
  while (n > 0) {
    if (a >= m) {
      s += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      s += n * (b / m);
      b %= m;
    }
    const int64_t y = a * n + b;
    if (y < m) break;
    n = y / m;
    b = y % m;
    const int64_t t = a;
    a = m;
    m = t;
  }
  return s;
}

// KV tiles of row tile j of a sequence with n new tokens out of len positions
__host__ __device__ inline int row_tile_units(int n, int len, int tp, int j) {
  const int64_t end = (int64_t)(j + 1) * tp;
  const int64_t seen = (int64_t)len - n + (end < n ? end : n);
  return seen <= kTile ? 1 : (int)((seen + kTile - 1) / kTile);
}
// the same summed over row tiles 0 .. j-1, none of them the last
__host__ __device__ __noinline__ inline int64_t units_before(int n, int len, int tp, int64_t j) {
  if (j == 0) return 0;
  const int64_t off = (int64_t)len - n;
  int64_t j0 = off < 0 ? -off / tp : 0;  // row tiles that see nothing: one unit each
  if (j0 > j) j0 = j;
  if (j0 == j) return j0;
  return j0 + floor_sum(j - j0, kTile, tp, off + (j0 + 1) * tp + kTile - 1);
}
__host__ __device__ inline int64_t head_units(int n, int len, int tp) {
  if (n <= 0) return 0;
  const int last = (n + tp - 1) / tp - 1;
  if (last == 0) return row_tile_units(n, len, tp, 0);
  return units_before(n, len, tp, last) + row_tile_units(n, len, tp, last);
}
__host__ __device__ inline int row_tiles(int n, int tp) { return n <= 0 ? 0 : (n + tp - 1) / tp; }
// the row tile that unit r of a head falls into (r becomes the unit within it),
// each with `extra` units before its KV tiles
__host__ __device__ inline int find_row_tile(int n, int len, int tp, int extra, int64_t& r) {
  int lo = 0, hi = row_tiles(n, tp) - 1;
  if (hi == 0) return 0;
  while (lo < hi) {
    const int mid = lo + (hi - lo + 1) / 2;
    if (units_before(n, len, tp, mid) + (int64_t)extra * mid <= r)
      lo = mid;
    else
      hi = mid - 1;
  }
  r -= units_before(n, len, tp, lo) + (int64_t)extra * lo;
  return lo;
}

__host__ __device__ inline int64_t share_begin(int64_t units, int c, int shares) {
  if (units < (1 << 20) && shares <= 1024) return (uint32_t)units * (uint32_t)c / (uint32_t)shares;  // fits 32 bits
  return units * c / shares;
}

}  // namespace sched
}  // namespace spock
