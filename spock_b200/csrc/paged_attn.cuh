// What the two kernels of spock_paged_attention share: their arguments, a CTA's
// share of the batch and the walk through it, the K and V loads, and the parts
// that paged_join_kernel adds up.
#pragma once
#include <cuda.h>

#include "paged_sched.cuh"
#include "ragged.cuh"
#include "tc.cuh"

namespace spock {
namespace paged {

using sched::kTile;
constexpr uint32_t kWait = 1u << 20;    // polls before a wait gives up
constexpr uint32_t kSleep = 20000;      // ns that one poll may sleep
constexpr int kThreads = 384;
constexpr int kFewRows = 16;  // rows of a row tile of the few-row kernel
constexpr float kLazy = 8.0f;  // log2 of how far weights may exceed 1
// Weights (and so their sums and O) are 2^kUp times as large where they are rounded
// to fp16: the largest stay below 2^15, and those far below a row's largest keep
// their bits down to 2^-21 of it and are lost below 2^-32. Without, a position
// e^16 below the largest had 2 of its 11 bits, and one e^18 below none, although
// thousands of them may weigh more than the largest.
template <typename T>
constexpr float kUp = std::is_same<T, __half>::value ? 7.0f : 0.0f;

struct AttnArgs {
  const int32_t *start, *table, *kv_len;
  int64_t table_stride;
  int batch, total, table_width, num_pages, page_size, kv_heads, G, tp, piece_k, piece_v, whole, extra;
  int64_t head_blk;  // 64-element blocks from one kv head to the next
  const uint8_t *q, *gate;
  int64_t q_row, q_head, g_row, g_head;  // bytes
  uint8_t* out;
  float scale_log2;
  float* ws;
  int* err;
};

// Workspace: per CTA a Meta and two parts (its first and its last row tile).
// A part: O [128][D] fp32, then the references (part_reference) and sums [128].
struct Meta {
  int slot;      // part of the row tile that begins in this CTA and ends in a later one, or -1
  int row0;      // its first packed row
  int rows;      // valid rows (token, head of the group)
  int head;      // kv head
  int have, nt;  // KV tiles done here, in all
  int units;     // of this CTA
  int before;    // KV tiles of its first row tile that are in earlier CTAs
  int last;      // the last position that the part's first token sees (negative: none)
};
// What a part says its weights refer to (a score before its scale): -inf where it has none, so
// that the join passes it over; a part whose scores are all NaN has weights (NaN),
// relative to 0.
__device__ __forceinline__ float part_reference(float m, float sum) {
  return m == -INFINITY && sum != 0.f ? 0.f : m;
}
template <int D>
__host__ __device__ constexpr size_t part_floats() {
  return (size_t)128 * D + 256;
}
__host__ __device__ constexpr size_t meta_bytes(int ctas) { return ((size_t)ctas * sizeof(Meta) + 127) / 128 * 128; }

// What runs once per CTA or row tile, and every wait, is kept out of line: with
// all of it inlined the kernels had 260 KB of code and every role's hot loop ran
// at the rate its instructions could be fetched (an MMA issued every 250 cycles).

// Bounded wait for a phase, by one thread; gives up at once when another role has
// (*fail), and says so to the others when it does itself.
static __device__ __noinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* fail) {
#pragma unroll 1
  for (uint32_t i = 0; i < kWait; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n"
        " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
        " selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kSleep)
        : "memory");
    if (ok) return true;
    if (*fail) return false;
  }
  *fail = 1;
  return false;
}

struct Seq {
  int lo, n, len;
};
__device__ __forceinline__ Seq load_seq(const AttnArgs& A, int b, bool report) {
  Seq s;
  s.lo = A.start[b];
  const int hi = A.start[b + 1];
  s.n = hi - s.lo;
  s.len = A.kv_len[b];
  const bool bad_n = s.lo < 0 || hi < s.lo || hi > A.total, bad_len = s.len < 0 || s.len > A.table_width * A.page_size;
  if (report && (bad_n || bad_len)) report_bad_index(A.err);
  if (bad_n) s.n = 0;
  if (bad_len) s.len = 0;
  return s;
}
// inclusive sums of a and b over the warp's lanes
__device__ __forceinline__ void warp_sums(int64_t& a, int64_t& b) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, a, o), z = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) a += y, b += z;
  }
}

// A role's way through the CTA's units. The sequence after the current one is
// loaded ahead: its lengths are a memory latency away.
struct Walk {
  int b, h, rt;
  int k0, k1, nt;  // KV tiles of the current row tile: [k0, k1) here, nt in all
  int left;        // units from this row tile's first one on
  Seq s, after;
  __device__ __forceinline__ void fit(const AttnArgs& A) {
    nt = sched::row_tile_units(s.n, s.len, A.tp, rt);
    k1 = min(nt, k0 + left);
  }
  __device__ __forceinline__ void enter(const AttnArgs& A, const Seq& now) {
    s = now;
    after = b + 1 < A.batch ? load_seq(A, b + 1, false) : Seq{0, 0, 0};
  }
  __device__ __noinline__ bool next(const AttnArgs& A) {
    left -= k1 - k0;
    if (left <= 0) return false;
    k0 = 0;
    if (++rt * A.tp >= s.n) {
      rt = 0;
      if (++h == A.kv_heads) {
        h = 0;
        do {
          ++b;
          enter(A, after);
        } while (s.n <= 0 && b + 1 < A.batch);
      }
    }
    fit(A);
    return true;
  }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}


// The row tile that unit r of a head falls into, each with `extra` units before
// its KV tiles (r becomes the unit within it), by all lanes of a warp: a search
// in 32 parts, since one step costs up to 3000 cycles (with halves, and one
// thread, 8 prompts spent 16 us in it).
__device__ __forceinline__ int find_row_tile(int n, int len, int tp, int extra, int64_t& r) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = sched::row_tiles(n, tp) - 1;
  int64_t before = 0;  // of row tile lo
#pragma unroll 1
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32, j = lo + lane * step;
    const int64_t u = j <= hi ? sched::units_before(n, len, tp, j) + (int64_t)extra * j : 0;
    const int at = __popc(__ballot_sync(0xffffffffu, j <= hi && u <= r)) - 1;  // >= 0: row tile lo is one of them
    before = __shfl_sync(0xffffffffu, u, at);
    lo += at * step;
    hi = min(hi, lo + step - 1);
  }
  r -= before;
  return lo;
}

// This CTA's share: the first row tile and KV tile in w; the KV tiles it has. All
// threads (it synchronises). scan: 2 kThreads / 32 + 4 words, first: 4.
//
// Prefix sums of the sequences' KV tiles and row tiles over the block, then the
// borders. Where a part is dear (A.whole: 128 rows of it make a round trip through
// the workspace) a border inside a row tile of at most half a share moves to the
// row tile's nearer end: shares grow or shrink by a quarter at most, and short row
// tiles are not cut. Parts of few rows are cheap, and equal shares worth more (256
// decode tokens: 18 KV tiles a CTA, 24 at most with moved borders).
//
// A share holds a KV tile at least: without `extra` as there are no more shares
// than units, and with it as a share is 2 (extra + 1) units or more (otherwise it
// does not count: few tiles are spread as far as they go), half of which the
// moved borders leave.
static __device__ __noinline__ int enter_share(const AttnArgs& A, int64_t* scan, int* first, Walk& w) {
  constexpr int W = kThreads / 32;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
  const int per = (A.batch + kThreads - 1) / kThreads;
  int64_t mine = 0, rts = 0;  // KV tiles, row tiles
#pragma unroll 1
  for (int b = tid * per; b < min(A.batch, (tid + 1) * per); ++b) {
    const Seq s = load_seq(A, b, cta == 0);
    mine += sched::head_units(s.n, s.len, A.tp) * A.kv_heads;
    rts += (int64_t)sched::row_tiles(s.n, A.tp) * A.kv_heads;
  }
  int64_t incl = mine, rincl = rts;
  warp_sums(incl, rincl);
  if (lane == 31) scan[warp] = incl, scan[W + warp] = rincl;
  __syncthreads();
  // the same over the warps, by each warp
  int64_t w_incl = lane < W ? scan[lane] : 0, w_rincl = lane < W ? scan[W + lane] : 0;
  warp_sums(w_incl, w_rincl);
  int64_t units = __shfl_sync(0xffffffffu, w_incl, 31), base = __shfl_sync(0xffffffffu, w_incl, warp) - scan[warp];
  const int64_t rall = __shfl_sync(0xffffffffu, w_rincl, 31);
  const int64_t rbase = __shfl_sync(0xffffffffu, w_rincl, warp) - scan[W + warp];
  const int64_t all = units;  // KV tiles
  int extra = A.extra;
  if (units + extra * rall < (int64_t)ctas * 2 * (extra + 1)) extra = 0;
  units += extra * rall;
  mine += extra * rts;
  const int64_t rfrom = rbase + rincl - rts, from = base + incl + extra * (rbase + rincl) - mine;
  const int shares = units < ctas ? (int)units : ctas;
  if (cta >= shares) return 0;
  const int64_t share = sched::share_begin(units, 1, shares);
  int64_t* border = scan + 2 * W;  // [2], then the KV tiles before them [2]
  if (tid < 2) {
    border[tid] = sched::share_begin(units, cta + tid, shares);
    border[2 + tid] = all;  // of a border behind the last unit
  }
  __syncthreads();
  // Each border by the warp that holds it. The finder moves it (A.whole); both
  // shares beside it come to the same place.
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const int64_t u = border[i];
    const bool finds = from <= u && u < from + mine;
    const unsigned finder = __ballot_sync(0xffffffffu, finds);
    if (!finder) continue;  // of all warps, one has it (none: behind the last unit)
    int64_t r = u - from, rt_before = rfrom;
    int b = tid * per, h = 0;
    Seq s{0, 0, 0};
    if (finds) {
#pragma unroll 1
      for (;; ++b) {
        s = load_seq(A, b, false);
        const int64_t tiles = sched::row_tiles(s.n, A.tp), hu = sched::head_units(s.n, s.len, A.tp) + extra * tiles;
#pragma unroll 1
        for (h = 0; h < A.kv_heads && r >= hu; ++h) r -= hu, rt_before += tiles;
        if (h < A.kv_heads) break;
      }
    }
    const int who = __ffs(finder) - 1;
    s.n = __shfl_sync(0xffffffffu, s.n, who);
    s.len = __shfl_sync(0xffffffffu, s.len, who);
    r = __shfl_sync(0xffffffffu, r, who);
    int rt = find_row_tile(s.n, s.len, A.tp, extra, r);
    if (finds) {
      const int nt = sched::row_tile_units(s.n, s.len, A.tp, rt), all_of = nt + extra;
      rt_before += rt;
      int64_t at = r;  // of the row tile's units
      if (A.whole && u > 0 && 2 * all_of <= share) at = 2 * r <= all_of ? 0 : all_of;
      int k = max((int)at - extra, 0);
      border[2 + i] = u - r - extra * rt_before + k;
      if (i == 0) {
        if (k == nt) {  // the next row tile's begin
          k = 0;
          if (++rt == sched::row_tiles(s.n, A.tp)) {
            rt = 0;
            if (++h == A.kv_heads) {
              h = 0;
              do ++b;
              while (b + 1 < A.batch && load_seq(A, b, false).n <= 0);
              b = min(b, A.batch - 1);
            }
          }
        }
        first[0] = b, first[1] = h, first[2] = rt, first[3] = k;
      }
    }
  }
  __syncthreads();
  const int n = (int)(border[3] - border[2]);
  w.left = n;
  if (n > 0) {
    w.b = first[0];
    w.h = first[1];
    w.rt = first[2];
    w.k0 = first[3];
    w.enter(A, load_seq(A, w.b, false));
    w.fit(A);
  }
  return n;
}

// The loads of a share's K (or V) tiles into the ring, by one warp each: issuing
// a copy costs its thread some 190 cycles and a wait as much, and one warp for
// both was slower than HBM. The ring's order is K0, K1, V0, K2, V1, .. (load_of_k,
// load_of_v); a stage is 128 positions x DB dims of K or VP positions x all dims
// of V, in [8-position group][64-dim block][8][128 B].
//
// A barrier must not be waited for while it is two phases behind (the parities
// would agree). With 5 stages and two per tile, or 6 or 8 and one per tile, the
// load before the last one into a stage is always known to have been read by
// then: by the loads that the same warp has already made, and because O += P V of
// tile g is issued after S of tiles <= g, and S of tile g after O += P V of tile
// g - 2. (Not so with 6 stages and two per tile.)
//
// A tile is fetched in pieces that lie in one page, a lane each. The page table is
// read two tiles ahead and looked at only when the tile is loaded: a lookup is a
// memory latency away. armed[st]: loads into the stage so far.
template <bool kV, int D, int NST, int kStage, class Wait>
__device__ __forceinline__ void load_tiles(const CUtensorMap& map, const AttnArgs& A, Walk& w, int N, uint8_t* ring,
                                           uint64_t* full, uint64_t* empty, volatile int* armed, Wait wait) {
  constexpr int DB = D < 128 ? D : 128, KS = D / DB;
  constexpr int kPos = kV ? kTile / KS : kTile;  // positions of a stage
  constexpr int kRow = kV ? D * 2 : DB * 2;      // bytes of a position in it
  static_assert((KS == 2 && NST == 5) || (KS == 1 && (NST == 6 || NST == 8)), "see above");
  const int lane = threadIdx.x & 31;
  const int piece = kV ? A.piece_v : A.piece_k, per_stage = kPos / piece;
  struct Src {
    int page, group, live, h;  // of this lane's piece; pieces that hold positions; kv head
  };
  auto look_up = [&](int k) -> Src {
    const int pos = k * kTile + lane * piece;
    Src r{-1, 0, 0, w.h};
    const bool live = lane * piece < kTile && pos < w.s.len;
    if (live) {
      const int slot = pos / A.page_size;
      r.page = A.table[w.b * A.table_stride + slot];
      r.group = (pos - slot * A.page_size) >> 3;
    }
    r.live = __popc(__ballot_sync(0xffffffffu, live));
    return r;
  };
  int k = w.k0, seen = 1;
  auto advance = [&](Src& into) {
    if (seen++ >= N) return;
    if (++k == w.k1) {
      w.next(A);
      k = w.k0;
    }
    into = look_up(k);
  };
  Src cur = look_up(k), nxt = cur, far = cur;
  advance(nxt);
#pragma unroll 1
  for (int g = 0; g < N; ++g) {
    advance(far);
    if (lane < cur.live && (cur.page < 0 || cur.page >= A.num_pages)) {  // reported, and page 0 read in its place
      report_bad_index(A.err);
      cur.page = 0;
    }
    const int first = kV ? (g + 1 < N ? 2 * g + 2 : 2 * N - 1) * KS : (g == 0 ? 0 : 2 * g - 1) * KS;
#pragma unroll 1
    for (int s = 0; s < KS; ++s) {
      const int use = first + s, st = use % NST, round = use / NST;
      const int n = kV ? max(0, min(cur.live - s * per_stage, per_stage)) : cur.live;
      if (lane == 0) {
        if (round == 0 || wait(&empty[st], (round - 1) & 1)) {
          armed[st] = round + 1;
          tc::mbar_arrive_expect_tx(&full[st], n * piece * kRow);
        }
      }
      __syncwarp();
      if (armed[st] <= round) return;  // gave up
      const int i = kV ? lane - s * per_stage : lane;
      if (i >= 0 && i < n)
        tc::tma_load_5d(ring + st * kStage + i * piece * kRow, &map, &full[st], 0, 0,
                        (int)(cur.h * A.head_blk) + (kV ? 0 : s * (DB / 64)), cur.group, cur.page);
    }
    cur = nxt;
    nxt = far;
  }
}
// After a wait that gave up: lets every stage's last copy land.
__device__ __forceinline__ void drain_ring(uint64_t* full, const volatile int* armed, int stages) {
  for (int st = 0; st < stages; ++st)
    if (armed[st]) tc::mbar_wait_bounded(&full[st], (armed[st] - 1) & 1, kWait);
}
// The number of a tile's first load in the ring's order.
__device__ __forceinline__ int load_of_k(int g, int KS) { return (g == 0 ? 0 : 2 * g - 1) * KS; }
__device__ __forceinline__ int load_of_v(int g, int N, int KS) { return (g + 1 < N ? 2 * g + 2 : 2 * N - 1) * KS; }

// V rows of positions behind the sequence become zero (rows from `first` of the
// tile on), by `n` threads, each `t` of them: 0 * NaN would reach every query.
template <int D, int VP>
static __device__ __noinline__ void zero_rows(uint8_t* stage, int from, int t, int n) {
#pragma unroll 1
  for (int i = t; i < (VP - from) * (D / 8); i += n) {
    const int r = from + i / (D / 8), ch = i % (D / 8);
    *reinterpret_cast<uint4*>(stage + (r >> 3) * (D / 64) * 1024 + (ch >> 3) * 1024 + (r & 7) * 128 + (ch & 7) * 16) =
        make_uint4(0, 0, 0, 0);
  }
}

}  // namespace paged
}  // namespace spock
