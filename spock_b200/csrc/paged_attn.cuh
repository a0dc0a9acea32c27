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
constexpr float kLazy = 8.0f;  // log2 of how far weights may exceed 1

struct AttnArgs {
  const int32_t *start, *table, *kv_len;
  int64_t table_stride;
  int batch, total, table_width, num_pages, page_size, kv_heads, G, tp, piece_k, piece_v;
  int64_t head_blk;  // 64-element blocks from one kv head to the next
  const uint8_t *q, *gate;
  int64_t q_row, q_head, g_row, g_head;  // bytes
  uint8_t* out;
  float scale_log2;
  float* ws;
  int* err;
};

// Workspace: per CTA a Meta and two parts (its first and its last row tile).
// A part: O [128][D] fp32, then the reference maxima (log2 units) and sums [128].
struct Meta {
  int slot;      // part of the row tile that begins in this CTA and ends in a later one, or -1
  int row0;      // its first packed row
  int rows;      // valid rows (token, head of the group)
  int head;      // kv head
  int have, nt;  // KV tiles done here, in all
  int units;     // of this CTA
  int pad;
};
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
  if (s.lo < 0 || hi < s.lo || hi > A.total) {
    if (report) report_bad_index(A.err);
    s.n = 0;
  }
  if (s.len < 0 || s.len > A.table_width * A.page_size) {
    if (report) report_bad_index(A.err);
    s.len = 0;
  }
  return s;
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


// This CTA's share: the first row tile and KV tile in w; the KV tiles it has. All
// threads (it synchronises). scan: kThreads / 32 + 2 words, first: 4.
//
// Prefix sums of the sequences' units over the block, then the borders. A border
// inside a row tile of at most half a share moves to the row tile's nearer end:
// shares grow or shrink by a quarter at most, and short row tiles are not cut
// (a part costs a round trip through the workspace and the join).
static __device__ __noinline__ int enter_share(const AttnArgs& A, int64_t* scan, int* first, Walk& w) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x, ctas = gridDim.x;
  const int per = (A.batch + kThreads - 1) / kThreads;
  int64_t mine = 0;
  for (int b = tid * per; b < min(A.batch, (tid + 1) * per); ++b) {
    const Seq s = load_seq(A, b, cta == 0);
    mine += sched::head_units(s.n, s.len, A.tp) * A.kv_heads;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t base = 0, units = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < warp) base += scan[i];
    units += scan[i];
  }
  const int64_t from = base + incl - mine;
  const int shares = units < ctas ? (int)units : ctas;  // none of them empty
  if (cta >= shares) return 0;
  int64_t* border = scan + kThreads / 32;
  // sequence, head, row tile and KV tile of unit u (in this thread's range); the row tile's units
  auto locate = [&](int64_t u, int& b, int& h, int& rt, int& k) -> int {
    int64_t r = u - from;
    for (b = tid * per;; ++b) {
      const Seq s = load_seq(A, b, false);
      const int64_t hu = sched::head_units(s.n, s.len, A.tp);
      if (r < hu * A.kv_heads) {
        for (h = 0; r >= hu; ++h) r -= hu;
        rt = sched::find_row_tile(s.n, s.len, A.tp, r);
        k = (int)r;
        return sched::row_tile_units(s.n, s.len, A.tp, rt);
      }
      r -= hu * A.kv_heads;
    }
  };
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const int64_t u = sched::share_begin(units, cta + i, shares);
    if (u == 0 || u == units) {
      if (tid == 0) border[i] = u;
    } else if (from <= u && u < from + mine) {
      int b, h, rt, k;
      const int nt = locate(u, b, h, rt, k);
      border[i] = 2 * nt > units / shares ? u : 2 * k <= nt ? u - k : u - k + nt;
    }
  }
  __syncthreads();
  const int64_t u0 = border[0], u1 = border[1];
  if (from <= u0 && u0 < from + mine && u1 > u0) {
    int b, h, rt, k;
    locate(u0, b, h, rt, k);
    first[0] = b, first[1] = h, first[2] = rt, first[3] = k;
  }
  __syncthreads();
  const int n = (int)(u1 - u0);
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

// The loads of a share's K and V tiles, by one warp, in the order K0, K1, V0,
// K2, V1, .. A stage is KP positions x KD dims of K or VP positions x all dims
// of V, in [8-position group][64-dim block][8][128 B].
//
// A tile is fetched in pieces that lie in one page: of V piece_v positions, one
// lane each, of K piece_k (a multiple, since a V stage has fewer positions). The
// page table is read two tiles ahead and looked at only when the tile is loaded:
// a lookup is a memory latency away.
template <int D, int NST, int kStage, class Wait>
__device__ __forceinline__ void load_tiles(const CUtensorMap& tmk, const CUtensorMap& tmv, const AttnArgs& A, Walk& w,
                                           int N, uint8_t* ring, uint64_t* full, uint64_t* empty, volatile int* issued,
                                           Wait wait) {
  constexpr int DB = D < 128 ? D : 128, KS = D / DB, VP = kTile / KS;
  const int lane = threadIdx.x & 31;
  struct Src {
    int page, group, live, h;  // of this lane's piece; pieces that hold positions; kv head
  };
  auto look_up = [&](int k) -> Src {
    const int pos = k * kTile + lane * A.piece_v;
    Src r{-1, 0, 0, w.h};
    const bool live = lane * A.piece_v < kTile && pos < w.s.len;
    if (live) {
      const int slot = pos / A.page_size;
      r.page = A.table[w.b * A.table_stride + slot];
      r.group = (pos - slot * A.page_size) >> 3;
    }
    r.live = __popc(__ballot_sync(0xffffffffu, live));
    return r;
  };
  const int per_k = A.piece_k / A.piece_v, per_stage = VP / A.piece_v;  // V pieces per K piece, per V stage
  auto check = [&](Src& r) {  // an entry out of range is reported and page 0 read in its place
    if (lane < r.live && (r.page < 0 || r.page >= A.num_pages)) {
      report_bad_index(A.err);
      r.page = 0;
    }
  };
  int ld = 0;
  auto stage = [&](int bytes) -> int {  // the next load's stage, once it is free; -1: gave up
    const int st = ld % NST, round = ld / NST;
    bool ok = true;
    if (lane == 0) {
      ok = round == 0 || wait(&empty[st], (round - 1) & 1);
      if (ok) {
        tc::mbar_arrive_expect_tx(&full[st], bytes);
        *issued = ld + 1;
      }
    }
    ++ld;
    return __shfl_sync(0xffffffffu, ok, 0) ? st : -1;
  };
  auto load_k = [&](const Src& src) -> bool {
    const int n = (src.live + per_k - 1) / per_k;  // K pieces
    const int page = __shfl_sync(0xffffffffu, src.page, (lane * per_k) & 31);
    const int group = __shfl_sync(0xffffffffu, src.group, (lane * per_k) & 31);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int st = stage(n * A.piece_k * DB * 2);
      if (st < 0) return false;
      if (lane < n)
        tc::tma_load_5d(ring + st * kStage + lane * A.piece_k * DB * 2, &tmk, &full[st], 0, 0,
                        (int)(src.h * A.head_blk) + s * (DB / 64), group, page);
    }
    return true;
  };
  auto load_v = [&](const Src& src) -> bool {
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int n = max(0, min(src.live - s * per_stage, per_stage)), i = lane - s * per_stage;
      const int st = stage(n * A.piece_v * D * 2);
      if (st < 0) return false;
      if (i >= 0 && i < n)
        tc::tma_load_5d(ring + st * kStage + i * A.piece_v * D * 2, &tmv, &full[st], 0, 0, (int)(src.h * A.head_blk),
                        src.group, src.page);
    }
    return true;
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
  check(cur);
  bool ok = load_k(cur);
  for (int g = 0; g < N && ok; ++g) {
    advance(far);
    if (g + 1 < N) {
      check(nxt);
      ok = load_k(nxt);
    }
    if (ok) ok = load_v(cur);
    cur = nxt;
    nxt = far;
  }
}
// The number of a tile's first load in that order.
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
