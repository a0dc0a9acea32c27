// spock_paged_attention for batches of decode tokens with small groups at head
// size 256: the tensor-core tile turned over.
//
// With 128 query rows on the M side (paged_attn_tc.cu) a decode token's 4 rows
// leave 124 lanes of every softmax and output instruction idle, which shows where
// row tiles are short (launch_paged_attention has both kernels' times, and the
// rule between them). Here M is the cache's side,
// and N the rows, 16:
//   S^T = K Q^T   M = 128 positions  N = rows  K = head dims
//   O^T += V^T P^T  M = 128 dims, twice  N = rows  K = positions
// K and V come straight from their tiles as the A operands (V M-major), the
// queries and the weights are the small B operands in shared memory. A softmax
// thread takes one position's scores, four rows at a time; no maximum crosses
// lanes unless a score exceeds its row's reference by 2^8, which one barrier with
// a vote finds out for the block. O^T has dims on the lanes, so outputs and gates
// are read and written in whole rows. Meant to be bound by the cache's bytes: an
// SM streams a tile (128 positions, 128 KB) in some 5700 cycles
// of HBM's time, its MMAs take 2300. 256 sequences of 65 to 1150 positions take 1.5
// times those bytes' time: starting, the last tiles and the join are some 15 us, and the ring holds
// little more than one tile, so every wait on the way shows. Separate rings for K
// and V (3 + 3 or 4 + 2 stages) were slower (81 and 83 us against 75).
//
// One CTA per SM walks its share (paged_attn.cuh). Warp roles:
//   warps 0, 3  K tiles and V tiles by TMA into a ring
//   warps 1, 2  issue S^T = K Q^T and O^T += V^T P^T
//   warps 4-7   softmax, a position per thread
//   warps 8-11  the queries of the row tile after the next, and the outputs of the
//               finished one (O^T has two buffers), while the others are at the next
// Parts of cut row tiles, masked slots and bounded waits as in paged_attn_tc.cu.
#include <atomic>

#include "paged_attn.cuh"
#include "ragged.h"

namespace spock {
namespace {

using namespace paged;

constexpr int NR = kFewRows;

template <int D>
struct Few {
  static_assert(D == 256, "head size");
  static constexpr int DB = 128, KS = D / DB, VP = kTile / KS;
  static constexpr int kStage = kTile * DB * 2;
  static constexpr int kQ = NR * D * 2;       // one of two query buffers: [64-dim block][row][128 B]
  static constexpr int kP = NR * kTile * 2;   // one of two weight buffers: [64-position block][row][128 B]
  static constexpr int NST = 5;
  static constexpr int kRing = 2 * kQ + 2 * kP;
  static constexpr int kBar = kRing + NST * kStage;
  static constexpr int kStat = kBar + 576;    // [2 row tiles][4 warps][NR] sums, [2][2][NR] references
  static constexpr int kMax = kStat + 2 * 6 * NR * 4;  // [4 warps][NR] maxima
  static constexpr int kSums = kMax + 4 * NR * 4;        // [NR][128] each softmax thread's sums
  static constexpr int kSmem = kSums + NR * 128 * 4;
  static constexpr int kBlocks = D / 128;     // M blocks of O^T
  static constexpr int kO = 2 * NR;           // TMEM: S^T [2][NR], then O^T [2][kBlocks][NR]
};
static_assert(Few<256>::kSmem <= 227 * 1024, "shared memory of one SM");

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_few_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                     const __grid_constant__ AttnArgs A) {
  using Sh = Few<D>;
  constexpr int DB = Sh::DB, KS = Sh::KS, NST = Sh::NST, NB = Sh::kBlocks;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t sm[];  // no static shared memory beside it, so it starts on 1024 bytes
  // [2] barriers are indexed by a tile's or row tile's parity, so that a waiter
  // that comes late never finds one a whole phase further on
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + Sh::kBar);
  uint64_t* empty = full + NST;
  uint64_t* q_full = empty + NST;    // [2]
  uint64_t* q_empty = q_full + 2;    // [2]
  uint64_t* s_full = q_full + 4;     // [2]
  uint64_t* p_full = q_full + 6;     // [2]
  uint64_t* p_free = q_full + 8;     // [2] also: O^T += V^T P^T of the tile is done
  uint64_t* o_full = q_full + 10;    // [2]
  uint64_t* o_free = q_full + 12;    // [2]
  uint64_t* stats = q_full + 14;     // [2]
  uint64_t* drain = q_full + 16;
  volatile int* s_fail = reinterpret_cast<volatile int*>(q_full + 17);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(q_full + 17) + 1;
  int64_t* s_scan = reinterpret_cast<int64_t*>(sm + Sh::kBar + 264);  // [2 warps + 4]
  int* s_first = reinterpret_cast<int*>(s_scan + 2 * (kThreads / 32) + 4);  // [4]
  volatile int* s_armed = s_first + 4;  // [NST]
  static_assert((2 * NST + 18) * 8 <= 264 && 264 + (2 * (kThreads / 32) + 4) * 8 + (4 + NST) * 4 <= 576, "barrier area");
  float* s_sum = reinterpret_cast<float*>(sm + Sh::kStat);
  // [2 row tiles]: of the vote, -inf for a row without scores yet; then of the weights, 0 for one
  float* s_ref = s_sum + 2 * 4 * NR;
  float* s_max = reinterpret_cast<float*>(sm + Sh::kMax);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int cta = blockIdx.x, ctas = gridDim.x;
  Meta* meta = reinterpret_cast<Meta*>(A.ws);
  float* parts = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(A.ws) + meta_bytes(ctas));

  if (tc::smem_u32(sm) & 1023) {  // never on this toolchain; the operand layouts need it
    if (tid == 0) {
      atomicExch(A.err, 6);
      pdl_wait();
      meta[cta].slot = -1, meta[cta].units = 0, meta[cta].before = 0;  // for the join: nothing here
    }
    return;
  }
  if (tid == 0) {
    for (int i = 0; i < NST; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&q_full[i], 4);
      tc::mbar_init(&q_empty[i], 1);
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 4);
      tc::mbar_init(&p_free[i], 1);
      tc::mbar_init(&o_full[i], 1);
      tc::mbar_init(&o_free[i], 4);
      tc::mbar_init(&stats[i], 4);
    }
    tc::mbar_init(drain, 2);
    *s_fail = 0;
    for (int i = 0; i < NST; ++i) s_armed[i] = 0;
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tmk);
    tc::prefetch_tmap(&tmv);
  }
  if (warp == 1) {
    tc::tmem_alloc(s_tmem, 256);
    tc::tmem_relinquish();
  }
  pdl_wait();
  pdl_launch();

  Walk w;
  const int N = enter_share(A, s_scan, s_first, w);  // KV tiles of this CTA
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tb = *s_tmem;
  const uint32_t sbase = tc::smem_u32(sm);
  auto o_at = [&](int item, int blk) { return tb + Sh::kO + ((item & 1) * NB + blk) * NR; };

  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(tc::smem_u32(bar), parity, s_fail); };
  // For warps that meet at named barriers: a wait that gives up does not leave
  // the loop (each later wait returns at once; the outputs are unspecified).
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
    if (lane == 0) wait(bar, parity);  // one lane polls: 32 would crowd the pipe that MMAs and loads go through
    __syncwarp();
    tc::tc_fence_after();
  };

  if (N == 0) {
    if (tid == 0) meta[cta].slot = -1, meta[cta].units = 0, meta[cta].before = 0;
  } else if (warp == 0) {
    load_tiles<false, D, NST, Sh::kStage>(tmk, A, w, N, sm + Sh::kRing, full, empty, s_armed, wait);
  } else if (warp == 1) {
    // ---- S^T = K Q^T ----
    if (tc::elect_one()) {
      constexpr uint32_t ID_S = tc::idesc_f16(128, NR, false, false, kBf16);
      int item = 0, k = w.k0;
      for (int g = 0; g < N; ++g) {
        if (k == w.k0 && !wait(&q_full[item & 1], (item >> 1) & 1)) break;
        if (g >= 2 && !wait(&p_free[g & 1], ((g - 2) >> 1) & 1)) break;  // S^T(g - 2) has been read long before
        bool ok = true;
#pragma unroll 1
        for (int s = 0; s < KS; ++s) {
          const int use = load_of_k(g, KS) + s, st = use % NST;
          if (!(ok = wait(&full[st], (use / NST) & 1))) break;
          tc::tc_fence_after();
          const uint32_t kd = tc::sdesc_lo(sbase + Sh::kRing + st * Sh::kStage, 16);
          const uint32_t qd = tc::sdesc_lo(sbase + (item & 1) * Sh::kQ + s * 2 * NR * 128, 16);
#pragma unroll 2
          for (int ks = 0; ks < DB / 16; ++ks)
            tc::mma_f16(tb + (g & 1) * NR, kd + (ks >> 2) * 64 + (ks & 3) * 2, tc::sdesc_hi((DB / 64) * 1024),
                        qd + (ks >> 2) * NR * 8 + (ks & 3) * 2, tc::sdesc_hi(1024), ID_S, (s | ks) > 0);
          tc::mma_commit(&empty[st]);
        }
        if (!ok) break;
        tc::mma_commit(&s_full[g & 1]);
        if (++k == w.k1) {
          tc::mma_commit(&q_empty[item & 1]);
          if (w.next(A)) k = w.k0;
          ++item;
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---- O^T += V^T P^T ----
    if (tc::elect_one()) {
      constexpr uint32_t ID_O = tc::idesc_f16(128, NR, true, false, kBf16);
      constexpr uint32_t kGroup = (D / 64) * 1024;  // bytes from one 8-position group of a stage to the next
      int item = 0, k = w.k0;
      bool first = true;
      for (int g = 0; g < N; ++g) {
        if (!wait(&p_full[g & 1], (g >> 1) & 1)) break;
        if (first && item >= 2 && !wait(&o_free[item & 1], ((item - 2) >> 1) & 1)) break;
        tc::tc_fence_after();
        bool ok = true;
#pragma unroll 1
        for (int s = 0; s < KS; ++s) {
          const int use = load_of_v(g, N, KS) + s, st = use % NST;
          if (!(ok = wait(&full[st], (use / NST) & 1))) break;
          tc::tc_fence_after();
          const uint32_t vd = tc::sdesc_lo(sbase + Sh::kRing + st * Sh::kStage, 1024);
          const uint32_t pd = tc::sdesc_lo(sbase + 2 * Sh::kQ + (g & 1) * Sh::kP, 16);
          const uint32_t od = o_at(item, 0);
#pragma unroll 1
          for (int ks = 0; ks < Sh::VP / 16; ++ks) {
            const int kk = s * (Sh::VP / 16) + ks;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
              tc::mma_f16(od + blk * NR, vd + (ks * 2 * kGroup + blk * 2048) / 16, tc::sdesc_hi(kGroup),
                          pd + (kk >> 2) * NR * 8 + (kk & 3) * 2, tc::sdesc_hi(1024), ID_O, kk > 0 || !first);
          }
          tc::mma_commit(&empty[st]);
        }
        if (!ok) break;
        tc::mma_commit(&p_free[g & 1]);
        first = false;
        if (++k == w.k1) {
          tc::mma_commit(&o_full[item & 1]);
          if (w.next(A)) k = w.k0;
          ++item;
          first = true;
        }
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    load_tiles<true, D, NST, Sh::kStage>(tmv, A, w, N, sm + Sh::kRing, full, empty, s_armed, wait);
  } else if (warp < 8) {
    // ---- softmax: thread = position of the tile ----
    const int quad = warp & 3, at = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const float c = A.scale_log2, lazy = kLazy / c;  // an infinite one (c < 2^-125): weights refer to 0 throughout
    // Rows in blocks of 4, of which a row tile has one to four; the loops over them
    // stay rolled and what they carry (references, sums) in shared memory: unrolled,
    // the kernel had 116 KB of code and waited for instructions first of all.
    float* const sum = reinterpret_cast<float*>(sm + Sh::kSums) + at;  // + r * 128
    float* ref = s_ref;  // in scores, before their scale (which could overflow); the row tile's
    int k = w.k0, item = 0, rows = 0;
    auto meet = [] { asm volatile("bar.sync 1, 128;" ::: "memory"); };
    auto enter = [&] {
      rows = min(A.tp, w.s.n - w.rt * A.tp) * A.G;
      ref = s_ref + (item & 1) * NR;
      if (item >= 2) wait_warp(&o_free[item & 1], ((item - 2) >> 1) & 1);
      // rows behind the last, in its block of 4, have whatever scores: none is above their reference, all weights are 0
      if (at < NR) ref[at] = at < rows ? -INFINITY : INFINITY, ref[2 * NR + at] = at < rows ? 0.f : INFINITY;
#pragma unroll 1
      for (int r = 0; r < rows; ++r) sum[r * 128] = 0.f;
      meet();
    };
    enter();
#pragma unroll 1
    for (int g = 0; g < N; ++g) {
      const int buf = g & 1, p0 = k * kTile;
      const int lim0 = w.s.len - w.s.n + w.rt * A.tp;  // the last position the first row sees
      const bool masked = p0 + kTile - 1 > lim0;
      wait_warp(&s_full[buf], (g >> 1) & 1);
      if (p0 + kTile > w.s.len) {  // slots behind the sequence: their V rows become zero
        const int first = max(0, w.s.len - p0);
        // O^T of tile g - 1 is done, so every earlier load of V(g)'s stages is over:
        // their barriers are at most one phase behind and the parities are V(g)'s
        if (g > 0) wait_warp(&p_free[buf ^ 1], ((g - 1) >> 1) & 1);
#pragma unroll 1
        for (int st = 0; st < KS; ++st) {
          const int use = load_of_v(g, N, KS) + st;
          wait_warp(&full[use % NST], (use / NST) & 1);
          zero_rows<D, Sh::VP>(sm + Sh::kRing + use % NST * Sh::kStage, max(0, first - st * Sh::VP), at, 128);
        }
        tc::fence_async_smem();
      }
      // f(r, scores of rows r .. r + 3)
      auto each = [&](auto f) {
        int lim = lim0 - (p0 + at), n = 0;  // >= 0: this position is seen by the row
#pragma unroll 1
        for (int r = 0; r < rows; r += 4) {
          float s[4];
          tc::tmem_ld4(tb + buf * NR + lane_off + r, s);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (masked) {
              s[i] = lim >= 0 ? s[i] : -INFINITY;
              if (++n == A.G) n = 0, ++lim;
            }
          }
          f(r, s);
        }
      };
      bool over = false;
      each([&](int r, const float(&s)[4]) {
        const float4 m = *reinterpret_cast<const float4*>(ref + r);
        over |= s[0] - m.x > lazy || s[1] - m.y > lazy || s[2] - m.z > lazy || s[3] - m.w > lazy;
      });
      uint32_t any;
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
          : "=r"(any)
          : "r"((uint32_t)over)
          : "memory");
      if (any) {  // some row's reference moves: the rows' maxima over the tile
        each([&](int r, const float(&s)[4]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float m = s[i];
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (lane == 0) s_max[quad * NR + r + i] = m;
          }
        });
        meet();
        auto top_of = [&](int r) {
          return fmaxf(fmaxf(s_max[r], s_max[NR + r]), fmaxf(s_max[2 * NR + r], s_max[3 * NR + r]));
        };
        const bool begun = k > w.k0;
        if (begun) wait_warp(&p_free[buf ^ 1], ((g - 1) >> 1) & 1);
#pragma unroll 1
        for (int r = 0; r < rows; r += 4) {
          float corr[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float m = top_of(r + i), was = ref[r + i];
            corr[i] = m - was > lazy ? ex2((was - m) * c) : 1.0f;
            sum[(r + i) * 128] *= corr[i];
          }
          if (begun) {
#pragma unroll 1
            for (int blk = 0; blk < NB; ++blk) {
              float o[4];
              tc::tmem_ld4(o_at(item, blk) + lane_off + r, o);
#pragma unroll
              for (int i = 0; i < 4; ++i) o[i] *= corr[i];
              tc::tmem_st4(o_at(item, blk) + lane_off + r, o);
            }
          }
        }
        tc::tmem_st_wait();
        meet();  // all have read the references
        if (at < rows) {
          const float m = top_of(at);
          if (m - ref[at] > lazy) ref[at] = ref[2 * NR + at] = m;
        }
        meet();
      }
      if (g >= 2) wait_warp(&p_free[buf], ((g - 2) >> 1) & 1);
      uint8_t* const pw = sm + 2 * Sh::kQ + buf * Sh::kP + (at >> 6) * NR * 128 + (at & 7) * 2;
      const int ch = (at & 63) >> 3;
      each([&](int r, const float(&s)[4]) {
        const float4 m = *reinterpret_cast<const float4*>(ref + 2 * NR + r);
        const float x[4] = {ex2(fmaf(s[0] - m.x, c, kUp<T>)), ex2(fmaf(s[1] - m.y, c, kUp<T>)),
                            ex2(fmaf(s[2] - m.z, c, kUp<T>)), ex2(fmaf(s[3] - m.w, c, kUp<T>))};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const T p = from_float<T>(x[i]);
          sum[(r + i) * 128] += to_float(p);  // of the weights that V gets: they add up to 1
          *reinterpret_cast<T*>(pw + (r + i) * 128 + ((ch ^ ((r + i) & 7)) << 4)) = p;
        }
      });
      tc::fence_async_smem();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[buf]);
      if (++k < w.k1) continue;

      // ---- the row tile's last KV tile here: sums over this warp's positions ----
#pragma unroll 1
      for (int r = 0; r < rows; ++r) {
        float l = sum[r * 128];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) s_sum[((item & 1) * 4 + quad) * NR + r] = l;
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&stats[item & 1]);
      if (w.next(A)) {
        k = w.k0;
        ++item;
        enter();
      }
    }
  } else {
    // ---- queries, two row tiles ahead; outputs: thread = dim ----
    const int quad = warp & 3, dim = quad * 32 + lane, heads = A.kv_heads * A.G;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    Walk ahead = w;
    bool more = true;
    auto load_q = [&](int item) {  // rows behind the row tile's last only reach results nobody looks at
      const int t0 = ahead.rt * A.tp, rows = min(A.tp, ahead.s.n - t0) * A.G;
      constexpr int CH = D / 8, RW = 128 / CH;  // 16-byte chunks of a row; rows per pass of the 128 threads
      const int c = dim % CH;
      const uint32_t qb = sbase + (item & 1) * Sh::kQ;
      int r = dim / CH, tt = r / A.G, gh = r - tt * A.G;
#pragma unroll 1
      for (; r < rows; r += RW) {
        const uint32_t dst = qb + (c >> 3) * NR * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4);
        cp_async16(dst, A.q + (int64_t)(ahead.s.lo + t0 + tt) * A.q_row + (int64_t)(ahead.h * A.G + gh) * A.q_head + c * 16);
        gh += RW;
        while (gh >= A.G) gh -= A.G, ++tt;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&q_full[item & 1]);
      more = ahead.next(A);
    };
    load_q(0);
    if (more) load_q(1);
    if (tid == 256) meta[cta].slot = -1, meta[cta].units = N, meta[cta].before = w.k0;
    for (int item = 0;; ++item) {
      const int t0 = w.rt * A.tp, rows = min(A.tp, w.s.n - t0) * A.G, row0 = w.s.lo + t0;
      const bool whole = w.k0 == 0 && w.k1 == w.nt;
      const int slot = item == 0 ? 0 : 1;
      if (!whole && w.k0 == 0 && tid == 256) {
        Meta& mt = meta[cta];
        mt.slot = slot;
        mt.row0 = row0;
        mt.rows = rows;
        mt.head = w.h;
        mt.have = w.k1;
        mt.nt = w.nt;
        mt.last = w.s.len - w.s.n + t0;
      }
      wait_warp(&stats[item & 1], (item >> 1) & 1);
      wait_warp(&o_full[item & 1], (item >> 1) & 1);
      const float* sums = s_sum + (item & 1) * 4 * NR;
      float* part = parts + ((size_t)cta * 2 + slot) * part_floats<D>();
#pragma unroll 1
      for (int blk = 0; blk < NB; ++blk) {
        const uint8_t* gp = A.gate + row0 * A.g_row + (int64_t)w.h * A.G * A.g_head + (blk * 128 + dim) * 2;
        T* op = reinterpret_cast<T*>(A.out) + ((int64_t)row0 * heads + w.h * A.G) * D + blk * 128 + dim;
        int ng = 0, no = 0;  // head of the group: of gp, of op
        int last = w.s.len - w.s.n + t0;  // the last position that op's row sees
#pragma unroll 1
        for (int r = 0; r < rows; r += 4) {
          T gate[4];
          if (A.gate && whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (r + i < rows) gate[i] = *reinterpret_cast<const T*>(gp);
              gp += A.g_head;
              if (++ng == A.G) ng = 0, gp += A.g_row - A.G * A.g_head;
            }
          }
          float o[4];
          tc::tmem_ld4(o_at(item, blk) + lane_off + r, o);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (r + i >= rows) break;
            if (whole) {
              const float* l = sums + r + i;
              const float lt = (l[0] + l[NR]) + (l[2 * NR] + l[3 * NR]);
              float x = last < 0 ? 0.f : __fdividef(o[i], lt);
              if (A.gate) x = __fdividef(x, 1.0f + __expf(-to_float(gate[i])));
              *op = from_float<T>(x);
              op += D;
              if (++no == A.G) no = 0, ++last, op += (int64_t)(heads - A.G) * D;
            } else {
              part[(r + i) * D + blk * 128 + dim] = o[i];
            }
          }
        }
      }
      if (!whole && dim < rows) {  // the part's references and sums, a row per thread
        const float l = (sums[dim] + sums[NR + dim]) + (sums[2 * NR + dim] + sums[3 * NR + dim]);
        part[128 * D + dim] = part_reference(s_ref[(item & 1) * NR + dim], l);
        part[128 * D + 128 + dim] = l;
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&o_free[item & 1]);
      if (more) {
        wait_warp(&q_empty[item & 1], (item >> 1) & 1);
        load_q(item + 2);
      }
      if (!w.next(A)) break;
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (*s_fail) {
    // let the copies and MMAs in flight land before shared memory and TMEM go
    if (tid == 0) {
      atomicExch(A.err, 5);
      drain_ring(full, s_armed, NST);
    }
    if ((warp == 1 || warp == 2) && tc::elect_one()) {  // the threads that issued the MMAs: a commit is for its own
      tc::mma_commit(drain);
      tc::mbar_wait_bounded(drain, 0, kWait);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tb, 256);
  }
}

template <typename T, int D>
Status launch(const CUtensorMap& mk, const CUtensorMap& mv, const AttnArgs& A, int sms, cudaStream_t st) {
  // the attribute belongs to the kernel on the current device: set once on each
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "spock_paged_attention");
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load() & bit)) {
    e = cudaFuncSetAttribute(paged_few_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Few<D>::kSmem);
    if (e != cudaSuccess) return cuda_status(e, "paged_few_kernel attribute");
    done.fetch_or(bit);
  }
  e = launch_k(paged_few_kernel<T, D>, dim3(sms), dim3(kThreads), Few<D>::kSmem, st, mk, mv, A);
  if (e != cudaSuccess) return cuda_status(e, "paged_few_kernel");
  SPOCK_LAUNCH_CHECK("paged_few_kernel");
  return Status::ok();
}

}  // namespace

Status launch_paged_few(int dtype, const CUtensorMap& mk, const CUtensorMap& mv, const paged::AttnArgs& A, int sms,
                        cudaStream_t st) {
  if (dtype == SPOCK_F16) return launch<__half, 256>(mk, mv, A, sms, st);
  return launch<__nv_bfloat16, 256>(mk, mv, A, sms, st);
}

}  // namespace spock
