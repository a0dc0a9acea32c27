// Causal attention of several new tokens per sequence over a KV cache in pages
// (spock_paged_attention) on the tcgen05 tensor cores.
//
//   o_r = sum_p w_rp v_p / sum_p w_rp,  w_rp = exp(scale (q_r . k_p) - m_r),
//   p = 0 .. len - n + t(r);  out_r = o_r sigmoid(gate_r)
//
// paged_attn_kernel: one CTA per SM walks its share of the batch
// (paged_sched.cuh): row tiles of up to 128 (token, query head) rows of one
// sequence and kv head, times KV tiles of 128 positions. Warp roles:
//   warps 0, 2  K tiles and V tiles by TMA from the pages into a ring of stages
//   warp 1      issues the MMAs: S = Q K^T (M128 N128 K=D) into one of two TMEM
//               buffers, O += P V (M128 N=D K128) with P read from TMEM
//   warp 3      the next row tile's queries, into shared memory
//   warps 4-11  softmax, two threads per row (64 of a tile's positions each), and
//               the output of finished row tiles
// S(i+1) is issued before O += P(i) V(i), so the tensor pipe has work while the
// softmax of a tile runs; the ring and the walk run on across row tiles. P
// overwrites its S in TMEM, in the operand type. The running maximum a row's
// weights refer to moves only when a tile's exceeds it by 2^8 (weights stay
// below 2^8, times kUp; sums in fp32), so O is rarely rescaled.
// A row tile that is one CTA's alone is finished there; a cut one leaves its
// unnormalised O (fp32), maximum and sum in the workspace, and
// paged_join_kernel adds the parts in order (no atomics: results repeat).
//
// Bound, at head size 256 with long sequences, by the K and V tiles' way from L2
// and the one and a quarter tiles that the ring holds: 2048 tokens of 8 heads over
// 16384 positions take 286 us where inputs change from call to call, 0.52 of the
// measured rate of large matrix products (247 us, 0.61, the same call again and again);
// of a tile's 3900 cycles the MMAs take 2100, the softmax 2000 beside them, and
// 1700 are waits for tiles. At head size 128 with short prompts (8 of 301 to 1021
// tokens: 59 us) by starting and finishing row tiles of some three KV tiles each.
// The MMA thread is the one elected by the warp: the same code under `lane == 0`
// goes through a loop over the lanes for each descriptor (333 us instead of 285).
//
// Slots behind kv_len may hold anything: their scores are masked, and their V
// rows are zeroed in shared memory, since 0 * NaN would reach every row.
// Every wait is bounded; one that gives up sets the context's error word, and
// the CTA lets its copies and MMAs land, frees its TMEM and leaves.
#include <cuda.h>

#include <atomic>

#include "paged_attn.cuh"
#include "ragged.h"
#include "tmap.h"

namespace spock {
Status launch_paged_few(int dtype, const CUtensorMap& mk, const CUtensorMap& mv, const paged::AttnArgs& A, int sms,
                        cudaStream_t st);

namespace {

using namespace paged;

// A row tile of this CTA, for the roles that do not walk by themselves (a walk's
// steps cost the softmax warps 1900 cycles each).
struct Item {
  int lo, n, len;  // its sequence: first packed row, new tokens, positions
  int h, rt;       // kv head, row tile
  int k0, k1, nt;  // KV tiles here, in all
};

template <int D>
struct Shape {
  // A stage is 32 KB (16 KB at head size 64): of K 128 positions x DB dims, of V
  // VP positions x all dims, so that each MMA of O += P V is as wide as O.
  static constexpr int DB = D < 128 ? D : 128;
  static constexpr int KS = D / DB;  // stages per K (or V) tile
  static constexpr int VP = kTile / KS;
  static constexpr int kStage = kTile * DB * 2;
  static constexpr int kQ = 128 * D * 2;
  static constexpr int NST = D == 256 ? 5 : D == 128 ? 6 : 8;
  static constexpr int kBar = kQ + NST * kStage;
  static constexpr int kRed = kBar + 576;
  static constexpr int kItem = kRed + 4 * 128 * 4;
  static constexpr int kSmem = kItem + 2 * sizeof(Item);
};
static_assert(Shape<256>::kSmem <= 227 * 1024 && Shape<128>::kSmem <= 227 * 1024, "shared memory of one SM");

// x[v]: piece v of this lane's row -> piece (lane & 3) of row v of its 4 lanes; and back
__device__ __forceinline__ void trade(uint32_t (&x)[4][4], int lane) {
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      if (v & b) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & b ? x[v][e] : x[v | b][e], b);
        if (lane & b)
          x[v][e] = got;
        else
          x[v | b][e] = got;
      }
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                      const __grid_constant__ CUtensorMap tmq, const __grid_constant__ AttnArgs A) {
  using Sh = Shape<D>;
  constexpr int DB = Sh::DB, KS = Sh::KS, NST = Sh::NST;
  constexpr bool kBf16 = sizeof(T) == 2 && !std::is_same<T, __half>::value;
  extern __shared__ __align__(1024) uint8_t sm[];  // no static shared memory beside it, so it starts on 1024 bytes
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + Sh::kBar);
  uint64_t* empty = full + NST;
  uint64_t* q_full = empty + NST;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_full + 2;   // [2]
  uint64_t* p_full = q_full + 4;   // [2]
  // [2], by tile parity: a waiter that comes late must not find the barrier a
  // whole phase further on
  uint64_t* o_done = q_full + 6;
  uint64_t* drain = q_full + 8;
  uint64_t* entered = q_full + 9;  // [2], by row tile parity: its Item is there
  volatile int* s_fail = reinterpret_cast<volatile int*>(q_full + 11);
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(q_full + 11) + 1;
  int64_t* s_scan = reinterpret_cast<int64_t*>(sm + Sh::kBar + 256);  // [2 warps + 4]
  int* s_first = reinterpret_cast<int*>(s_scan + 2 * (kThreads / 32) + 4);  // [4]
  volatile int* s_armed = s_first + 4;  // [NST + 1]
  Item* s_item = reinterpret_cast<Item*>(sm + Sh::kItem);  // [2], by row tile parity
  float* red = reinterpret_cast<float*>(sm + Sh::kRed);  // [2 tiles][2 halves][128] maxima (and sums)
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
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&s_full[i], 1);
      tc::mbar_init(&p_full[i], 8);
      tc::mbar_init(&o_done[i], 1);
      tc::mbar_init(&entered[i], 1);
    }
    tc::mbar_init(drain, 1);
    *s_fail = 0;
    for (int i = 0; i <= NST; ++i) s_armed[i] = 0;
    tc::fence_mbar_init();
    tc::prefetch_tmap(&tmk);
    tc::prefetch_tmap(&tmv);
    tc::prefetch_tmap(&tmq);
  }
  if (warp == 1) {
    tc::tmem_alloc(s_tmem, 512);
    tc::tmem_relinquish();
  }
  pdl_wait();
  pdl_launch();

  Walk w;
  const int N = enter_share(A, s_scan, s_first, w);  // KV tiles of this CTA
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tb = *s_tmem, tO = tb + 256;
  const uint32_t sbase = tc::smem_u32(sm);

  auto wait = [&](uint64_t* bar, uint32_t parity) { return wait_for(tc::smem_u32(bar), parity, s_fail); };

  if (N == 0) {
    if (tid == 0) meta[cta].slot = -1, meta[cta].units = 0, meta[cta].before = 0;
  } else if (warp == 0) {
    load_tiles<false, D, NST, Sh::kStage>(tmk, A, w, N, sm + Sh::kQ, full, empty, s_armed, wait);
  } else if (warp == 2) {
    load_tiles<true, D, NST, Sh::kStage>(tmv, A, w, N, sm + Sh::kQ, full, empty, s_armed, wait);
  } else if (warp == 1) {
    // ---- MMAs ----
    if (tc::elect_one()) {
      constexpr uint32_t ID_S = tc::idesc_f16(128, kTile, false, false, kBf16);
      constexpr uint32_t ID_O = tc::idesc_f16(128, D, false, true, kBf16);
      constexpr uint32_t kGroup = (D / 64) * 1024;  // bytes from one 8-position group of a V stage to the next
      int item = 0, left = 0, gs = 0, go = 0;  // the next S and O; S tiles left of the row tile
      bool fresh = true;    // S(gs) is its row tile's first
      uint32_t starts = 0;  // bit g & 1: O(g) starts from zero
      while (go < N) {
        // S(g + 1) goes before O(g), unless it waits for the next row tile's queries
        if (gs < N && (gs == go || (gs == go + 1 && !fresh))) {
          const int g = gs++;
          if (fresh) {
            if (!wait(q_full, item & 1)) break;
            left = s_item[item & 1].k1 - s_item[item & 1].k0;
            tc::mbar_arrive(&entered[item & 1]);
          }
          starts = (starts & ~(1u << (g & 1))) | (uint32_t)fresh << (g & 1);
          bool ok = true;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int use = load_of_k(g, KS) + s, st = use % NST;
            if (!(ok = wait(&full[st], (use / NST) & 1))) break;
            tc::tc_fence_after();
            const uint32_t kd = tc::sdesc_lo(sbase + Sh::kQ + st * Sh::kStage, 16);
            const uint32_t qd = tc::sdesc_lo(sbase + s * (DB / 64) * 16384, 16);
#pragma unroll
            for (int ks = 0; ks < DB / 16; ++ks)
              tc::mma_f16(tb + (g & 1) * kTile, qd + (ks >> 2) * 1024 + (ks & 3) * 2, tc::sdesc_hi(1024),
                          kd + (ks >> 2) * 64 + (ks & 3) * 2, tc::sdesc_hi((DB / 64) * 1024), ID_S, (s | ks) > 0);
            tc::mma_commit(&empty[st]);
          }
          if (!ok) break;
          tc::mma_commit(&s_full[g & 1]);
          fresh = --left == 0;
          if (fresh) {
            tc::mma_commit(q_empty);
            ++item;
          }
        } else {
          const int g = go++;
          const bool first = starts >> (g & 1) & 1;
          if (!wait(&p_full[g & 1], (g >> 1) & 1)) break;
          bool ok = true;
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            const int use = load_of_v(g, N, KS) + s, st = use % NST;
            if (!(ok = wait(&full[st], (use / NST) & 1))) break;
            tc::tc_fence_after();
            const uint32_t vd = tc::sdesc_lo(sbase + Sh::kQ + st * Sh::kStage, 1024);
#pragma unroll
            for (int ks = 0; ks < Sh::VP / 16; ++ks)
              tc::mma_f16_ta(tO, tb + (g & 1) * kTile + (s * (Sh::VP / 16) + ks) * 8, vd + ks * 2 * kGroup / 16,
                             tc::sdesc_hi(kGroup), ID_O, (s | ks) > 0 || !first);
            tc::mma_commit(&empty[st]);
          }
          if (!ok) break;
          tc::mma_commit(&o_done[g & 1]);
        }
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // ---- queries: a box of tp tokens x G heads for each 64 dims ----
    if (tc::elect_one()) {
      const uint32_t bytes = (uint32_t)(A.tp * A.G) * 128;
      for (int item = 0;; ++item) {
        if (item > 0 && !wait(q_empty, (item - 1) & 1)) break;
        s_item[item & 1] = {w.s.lo, w.s.n, w.s.len, w.h, w.rt, w.k0, w.k1, w.nt};
        s_armed[NST] = item + 1;
        tc::mbar_arrive_expect_tx(q_full, bytes * (D / 64));
#pragma unroll
        for (int blk = 0; blk < D / 64; ++blk)
          tc::tma_load_3d(sm + blk * 16384, &tmq, q_full, blk * 64, w.h * A.G, w.s.lo + w.rt * A.tp);
        if (!w.next(A)) break;
      }
    }
    __syncwarp();
  } else {
    // ---- softmax and outputs ----
    const int quad = warp & 3, half = (warp - 4) >> 2, row = quad * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const float c = A.scale_log2;
    // A wait that gives up does not leave the loop: the warps of a pair meet at
    // named barriers, so all of them walk on (each later wait returns at once),
    // with empty row tiles from the next one on; the outputs are unspecified.
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
      if (lane == 0) wait(bar, parity);  // one lane polls: 32 would crowd the pipe that MMAs and loads go through
      __syncwarp();
      tc::tc_fence_after();
    };
    auto pair_sync = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + quad) : "memory"); };
    if (tid == 128) meta[cta].slot = -1, meta[cta].units = N, meta[cta].before = w.k0;
    float m = -INFINITY, l = 0.f;
    int k = 0, item = 0;
    int t0 = 0, rows = 0, lim = 0, lim0 = 0;
    const int tt = row / A.G;
    Item it;
    auto enter = [&] {  // O of the row tile before cannot be issued without this one's warps: never two phases behind
      bool ok = true;
      if (lane == 0) ok = wait(&entered[item & 1], (item >> 1) & 1);
      uint32_t both;  // the pair agrees
      asm volatile(
          "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.and.pred q, %2, 64, p;\n selp.u32 %0, 1, 0, q;\n}"
          : "=r"(both)
          : "r"((uint32_t)ok), "r"(1 + quad)
          : "memory");
      if (both)
        it = s_item[item & 1];
      else
        it = Item{0, 0, 0, 0, 0, 0, 0, 0};
      k = it.k0;
      t0 = it.rt * A.tp;
      rows = min(A.tp, it.n - t0) * A.G;
      lim = row < rows ? it.len - it.n + t0 + tt : 0x7fffffff;
      lim0 = __shfl_sync(0xffffffffu, lim, 0);
      m = -INFINITY;
      l = 0.f;
    };
    enter();
    for (int g = 0; g < N; ++g) {
      const int buf = g & 1, p0 = k * kTile;
      const bool live = quad * 32 < rows;
      wait_warp(&s_full[buf], (g >> 1) & 1);
      if (p0 + kTile > it.len) {  // slots behind the sequence: their V rows become zero
        const int first = max(0, it.len - p0);
        // V(g - 1) has been read, so every earlier load of V(g)'s stages is over:
        // their barriers are at most one phase behind and the parities are V(g)'s
        if (g > 0) wait_warp(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          const int use = load_of_v(g, N, KS) + s, st = use % NST, from = max(0, first - s * Sh::VP);
          wait_warp(&full[st], (use / NST) & 1);
          zero_rows<D, Sh::VP>(sm + Sh::kQ + st * Sh::kStage, from, tid - 128, 256);
        }
        tc::fence_async_smem();
      }
      if (live) {
        float s[64];
        tc::tmem_ld64(tb + buf * kTile + lane_off + half * 64, s);
        if (p0 + kTile - 1 > lim0) {
          const int d = lim - p0 - half * 64;  // the last column this row sees
#pragma unroll
          for (int j = 0; j < 64; ++j) s[j] = j <= d ? s[j] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int j = 4; j < 64; ++j) mx[j & 3] = fmaxf(mx[j & 3], s[j]);
        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        red[buf * 256 + half * 128 + row] = top;
        pair_sync();  // also: both halves have read S before P overwrites it
        top = fmaxf(top, red[buf * 256 + (half ^ 1) * 128 + row]);
        const bool move = (top - m) * c > kLazy;
        if (__any_sync(0xffffffffu, move)) {
          const float corr = move ? ex2((m - top) * c) : 1.0f;
          if (move) m = top;
          l *= corr;
          if (k > it.k0) {
            wait_warp(&o_done[(g - 1) & 1], ((g - 1) >> 1) & 1);
#pragma unroll 1
            for (int cb = 0; cb < D / 64; ++cb) {
              float o[32];
              const uint32_t at = tO + lane_off + half * (D / 2) + cb * 32;
              tc::tmem_ld32(at, o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] *= corr;
              tc::tmem_st32(at, o);
            }
          }
        }
        // (s - m) c and not s c - m c: at scores of 2^31 a rounding of m c is 2^7, weights of 2^+-128
        const float from = m == -INFINITY ? 0.f : m;
        uint32_t p[32];
        float2 sum[2] = {};
#pragma unroll
        for (int j = 0; j < 32; ++j) {  // in pairs, so that this costs no more than the one multiply-add
          const float2 x = __ffma2_rn(__fadd2_rn(make_float2(s[2 * j], s[2 * j + 1]), make_float2(-from, -from)),
                                      make_float2(c, c), make_float2(kUp<T>, kUp<T>));
          const float2 w = make_float2(ex2(x.x), ex2(x.y));
          p[j] = Io<T>::down2(w.x, w.y);
          sum[j & 1] = __fadd2_rn(sum[j & 1], Io<T>::up2(p[j]));  // of the weights that V gets: they add up to 1
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tc::tmem_st32u(tb + buf * kTile + lane_off + half * 32, p);
        tc::tmem_st_wait();
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[buf]);
      if (++k < it.k1) continue;

      // ---- the row tile's last KV tile here ----
      const bool whole = it.k0 == 0 && it.k1 == it.nt;
      const int64_t tok = it.lo + t0 + tt;
      const int hq = it.h * A.G + row - tt * A.G;
      wait_warp(&o_done[buf], (g >> 1) & 1);
      const int slot = item == 0 ? 0 : 1;
      if (!whole && it.k0 == 0 && tid == 128) {
        Meta& mt = meta[cta];
        mt.slot = slot;
        mt.row0 = it.lo + t0;
        mt.rows = rows;
        mt.head = it.h;
        mt.have = it.k1;
        mt.nt = it.nt;
        mt.last = lim0;
      }
      if (live) {
        float* rl = red + (buf ^ 1) * 256;  // idle: the maxima of the tile before, read by both halves
        rl[half * 128 + row] = l;
        pair_sync();
        const float lt = l + rl[(half ^ 1) * 128 + row];
        pair_sync();  // read before the next tile's maxima go there
        if (whole) {
          const float inv = lim < 0 ? 0.f : 1.0f / lt;
          // 4 lanes trade their rows' 16-byte pieces, so that each store (and load of
          // gates) has 64 bytes of a row beside each other, 8 rows and not 32 at a time
          const int64_t op = (tok * (A.kv_heads * A.G) + hq) * (D * 2) + half * D;
          const int64_t gp = tok * A.g_row + hq * A.g_head + half * D;
          const int piece = (lane & 3) * 16, first = row & ~3;
          int64_t ops[4], gps[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            ops[t] = __shfl_sync(0xffffffffu, op, (lane & ~3) + t) + piece;
            gps[t] = __shfl_sync(0xffffffffu, gp, (lane & ~3) + t) + piece;
          }
#pragma unroll 1
          for (int cb = 0; cb < D / 64; ++cb) {
            uint32_t x[4][4];
            if (A.gate) {
#pragma unroll
              for (int t = 0; t < 4; ++t)
                if (first + t < rows) load_words(A.gate + gps[t] + cb * 64, x[t]);
              trade(x, lane);
            }
            float o[32];
            tc::tmem_ld32(tO + lane_off + half * (D / 2) + cb * 32, o);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float a = o[v * 8 + 2 * e] * inv, b = o[v * 8 + 2 * e + 1] * inv;
                if (A.gate) {
                  const float2 z = Io<T>::up2(x[v][e]);
                  a = __fdividef(a, 1.0f + __expf(-z.x));
                  b = __fdividef(b, 1.0f + __expf(-z.y));
                }
                x[v][e] = Io<T>::down2(a, b);
              }
            }
            trade(x, lane);
#pragma unroll
            for (int t = 0; t < 4; ++t)
              if (first + t < rows) store_words(A.out + ops[t] + cb * 64, x[t]);
          }
        } else {
          float* part = parts + ((size_t)cta * 2 + slot) * part_floats<D>();
          if (half == 0 && row < rows) {
            part[128 * D + row] = part_reference(m, lt);
            part[128 * D + 128 + row] = lt;
          }
#pragma unroll 1
          for (int cb = 0; cb < D / 64; ++cb) {
            float o[32];
            tc::tmem_ld32(tO + lane_off + half * (D / 2) + cb * 32, o);
            if (row < rows) {
              float4* dst = reinterpret_cast<float4*>(part + row * D + half * (D / 2) + cb * 32);
#pragma unroll
              for (int v = 0; v < 8; ++v) dst[v] = make_float4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            }
          }
        }
      }
      ++item;
      if (g + 1 < N) enter();
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
      if (s_armed[NST]) tc::mbar_wait_bounded(q_full, (s_armed[NST] - 1) & 1, kWait);
    }
    if (warp == 1 && tc::elect_one()) {  // the thread that issued the MMAs: a commit is for its own
      tc::mma_commit(drain);
      tc::mbar_wait_bounded(drain, 0, kWait);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tb, 512);
  }
}

// Joins the parts of each cut row tile, in share order: o = sum e_i O_i /
// sum e_i l_i, e_i = exp(scale (m_i - m)). The blocks of all its n shares (blockIdx.x) do it, the rows
// dealt to the n gridDim.y of them: the one that continues in a share, then the
// one that begins there. (With the first share's blocks alone, a call that ends in
// 12 row tiles of 13 parts and 128 rows took 80 us, and 46 so.) Few parts: a warp
// per row; many (a long sequence over the whole GPU): the block's 8 warps share
// each row's.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ AttnArgs A) {
  constexpr int V = D / 32, kMany = 12;
  const int cta = blockIdx.x, ctas = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float s_o[8][D];
  __shared__ float s_l[8], s_m[8];
  pdl_wait();
  pdl_launch();
  const Meta* meta = reinterpret_cast<const Meta*>(A.ws);
  const float* parts = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(A.ws) + meta_bytes(ctas));
  // shares from `at` on (by dir), 32 at a time, until their units cover `want`: how many
  auto cover = [&](int at, int dir, int want) -> int {
    int n = 0;
    for (int have = 0; have < want && at >= 0 && at < ctas;) {
      const int i = at + dir * lane;
      int u = i >= 0 && i < ctas ? meta[i].units : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, u, o);
        if (lane >= o) u += y;
      }
      const unsigned enough = __ballot_sync(0xffffffffu, have + u >= want);
      if (enough) return n + __ffs(enough);
      have += __shfl_sync(0xffffffffu, u, 31);
      n += 32;
      at += dir * 32;
    }
    return n;
  };
  const Meta own = meta[cta];
#pragma unroll 1
  for (int job = 0; job < 2; ++job) {
    if (job == 0 ? own.before <= 0 : own.slot < 0) continue;
    const int c0 = job == 0 ? max(0, cta - cover(cta - 1, -1, own.before)) : cta;
    const Meta mt = job == 0 ? meta[c0] : own;
    if (mt.slot < 0) continue;  // only after a wait that gave up
    const int n = min(1 + cover(c0 + 1, 1, mt.nt - mt.have), ctas - c0);
    const int rank = (cta - c0) * gridDim.y + blockIdx.y, ranks = n * gridDim.y;
    auto part = [&](int i) {
      return parts + ((size_t)(c0 + i) * 2 + (i == 0 ? mt.slot : 0)) * part_floats<D>();
    };
    // parts i0, i0 + step, .. < n of row r, four in flight; l and acc relative to the running maximum m
    auto add = [&](int i0, int step, int r, float& m, float (&acc)[V], float& l) {
      constexpr int U = 4;
#pragma unroll 1
      for (int i = i0; i < n; i += U * step) {
        float mi[U], li[U], x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = i + u * step;
          mi[u] = -INFINITY;
          if (j < n) {
            const float* p = part(j);
            mi[u] = p[128 * D + r];
            li[u] = p[128 * D + 128 + r];
#pragma unroll
            for (int v = 0; v < V; v += 2) {
              const float2 y = *reinterpret_cast<const float2*>(p + r * D + lane * V + v);
              x[u][v] = y.x, x[u][v + 1] = y.y;
            }
          }
        }
        const float to = fmaxf(fmaxf(fmaxf(mi[0], mi[1]), fmaxf(mi[2], mi[3])), m);
        if (to > m) {
          const float f = ex2((m - to) * A.scale_log2);
          l *= f;
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] *= f;
          m = to;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (mi[u] > -INFINITY) {  // not one without weights
            const float f = ex2((mi[u] - m) * A.scale_log2);
            l = fmaf(f, li[u], l);
            if (f != 0.f) {
#pragma unroll
              for (int v = 0; v < V; ++v) acc[v] = fmaf(f, x[u][v], acc[v]);
            }
          }
      }
    };
    const bool many = n > kMany;
#pragma unroll 1
    for (int r = many ? rank : rank * 8 + warp; r < mt.rows; r += many ? ranks : ranks * 8) {
      const int tt = r / A.G, hq = mt.head * A.G + r - tt * A.G;
      const int64_t tok = mt.row0 + tt;
      uint32_t w[V / 2], gw[V / 2];
      if (A.gate) load_words(A.gate + tok * A.g_row + hq * A.g_head + lane * V * 2, gw);
      float m = -INFINITY, acc[V] = {}, l = 0.f;
      add(many ? warp : 0, many ? 8 : 1, r, m, acc, l);
      if (many) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; ++v) s_o[warp][lane * V + v] = acc[v];
        if (lane == 0) s_m[warp] = m, s_l[warp] = l;
        __syncthreads();
        if (warp) continue;
        float to = s_m[0];
        for (int k = 1; k < 8; ++k) to = fmaxf(to, s_m[k]);
        l = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.f;
        for (int k = 0; k < 8; ++k) {
          const float f = s_m[k] > -INFINITY ? ex2((s_m[k] - to) * A.scale_log2) : 0.f;
          l = fmaf(f, s_l[k], l);
#pragma unroll
          for (int v = 0; v < V; ++v) acc[v] = fmaf(f, s_o[k][lane * V + v], acc[v]);
        }
      }
      const float inv = mt.last + tt < 0 ? 0.f : 1.0f / l;
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        float a = acc[2 * e] * inv, b = acc[2 * e + 1] * inv;
        if (A.gate) {
          const float2 z = Io<T>::up2(gw[e]);
          a = __fdividef(a, 1.0f + __expf(-z.x));
          b = __fdividef(b, 1.0f + __expf(-z.y));
        }
        w[e] = Io<T>::down2(a, b);
      }
      store_words(A.out + (tok * (A.kv_heads * A.G) + hq) * (D * 2) + lane * V * 2, w);
    }
  }
}

// Pages as [page][8-position group][64-dim block][position in group][64]: one
// box of a piece's groups lands as [group][block][8][128 B], which both the
// K-major and the MN-major operand layouts read with constant strides whatever
// the page size. The blocks of head h start at h * head_stride / 64.
CUresult encode_pages(EncodeFn fn, CUtensorMap* map, const spock_paged_kv& kv, void* base, int piece, int dims_box) {
  const int64_t blocks = (kv.kv_heads - 1) * (kv.head_stride / 64) + kv.head_dim / 64;
  cuuint64_t dims[5] = {64, 8, (cuuint64_t)blocks, (cuuint64_t)kv.page_size / 8, (cuuint64_t)kv.num_pages};
  cuuint64_t strides[4] = {(cuuint64_t)kv.pos_stride * 2, 128, (cuuint64_t)kv.pos_stride * 16,
                           (cuuint64_t)kv.page_stride * 2};
  cuuint32_t box[5] = {64, 8, (cuuint32_t)dims_box / 64, (cuuint32_t)piece / 8, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn(map, kv.dtype == SPOCK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, base,
            dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

template <typename T, int D>
Status launch(const spock_paged_kv& kv, AttnArgs& A, bool few, int sms, cudaStream_t st) {
  EncodeFn fn = tensor_map_encoder();
  if (!fn) return Status::err(SPOCK_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  A.tp = (few ? kFewRows : 128) / A.G;
  // A part of 128 rows is dear, one of 20 (five drafts of 4 heads) not. us with moved borders / equal shares by the
  // rows of a sequence, back to back, 256 sequences of 65 to 1150 positions: head size 256, groups of 4: 20 rows
  // 86.2 / 80.6, 48 89.0 / 86.9, 64 90.4 / 90.5, 96 91.8 / 96.7, 128 93.4 / 104, 512 262 / 280; head size 128: 32
  // 94.4 / 92.4, 48 96.5 / 99.0, 64 96.2 / 97.6, 128 100 / 109. Of longer ones (64 of 130 to 4000) equal shares are
  // ahead up to 200 rows (head size 256: 64 71.6 / 71.4, 200 127 / 115; 128: 64 81.5 / 71.8, 200 149 / 127).
  A.whole = !few && A.total * (int64_t)A.G > 64 * (int64_t)A.batch;
  A.extra = 3;
  A.piece_k = gcd(kv.page_size, kTile);
  A.piece_v = gcd(kv.page_size, Shape<D>::VP);
  CUtensorMap mk, mv, mq;
  if (encode_pages(fn, &mk, kv, kv.k, A.piece_k, Shape<D>::DB) != CUDA_SUCCESS ||
      encode_pages(fn, &mv, kv, kv.v, A.piece_v, D) != CUDA_SUCCESS)
    return Status::err(SPOCK_ERR_CUDA, "spock_paged_attention: tensor map encoding failed");
  cudaError_t e;
  if (D == 256 && few) {
    const Status s = launch_paged_few(kv.dtype, mk, mv, A, sms, st);
    if (s.code) return s;
  } else {
    // the attribute belongs to the kernel on the current device: set once on each
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return cuda_status(e, "spock_paged_attention");
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
      e = cudaFuncSetAttribute(paged_attn_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
      if (e != cudaSuccess) return cuda_status(e, "paged_attn_kernel attribute");
      done.fetch_or(bit);
    }
    // queries as [token][head][dim]
    const int heads = A.kv_heads * A.G;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)A.total};
    cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? A.q_head : D * 2), (cuuint64_t)(A.total > 1 ? A.q_row : D * 2)};
    cuuint32_t box[3] = {64, (cuuint32_t)A.G, (cuuint32_t)A.tp}, estr[3] = {1, 1, 1};
    if (fn(&mq, kv.dtype == SPOCK_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
           const_cast<uint8_t*>(A.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return Status::err(SPOCK_ERR_CUDA, "spock_paged_attention: tensor map encoding failed");
    e = launch_k(paged_attn_kernel<T, D>, dim3(sms), dim3(kThreads), Shape<D>::kSmem, st, mk, mv, mq, A);
    if (e != cudaSuccess) return cuda_status(e, "paged_attn_kernel");
    SPOCK_LAUNCH_CHECK("paged_attn_kernel");
  }
  pdl_scope overlap;  // the join's launch runs under the main kernel
  e = launch_k(paged_join_kernel<T, D>, dim3(sms, 2), dim3(256), 0, st, A);
  if (e != cudaSuccess) return cuda_status(e, "paged_join_kernel");
  SPOCK_LAUNCH_CHECK("paged_join_kernel");
  return Status::ok();
}

}  // namespace

size_t paged_attention_workspace(int, int, int head_dim, int sms) {
  const size_t part = head_dim == 64 ? part_floats<64>() : head_dim == 128 ? part_floats<128>() : part_floats<256>();
  return meta_bytes(sms) + (size_t)sms * 2 * part * sizeof(float);
}

Status launch_paged_attention(const spock_paged_kv& kv, int batch, const int32_t* start, int64_t total, int q_heads,
                              const void* q, int64_t q_row, int64_t q_head, const void* gate, int64_t g_row,
                              int64_t g_head, float scale, void* out, void* ws, int sms, int* err, cudaStream_t st) {
  AttnArgs A{};
  A.start = start;
  A.table = kv.page_table;
  A.kv_len = kv.kv_len;
  A.table_stride = kv.table_stride;
  A.batch = batch;
  A.total = (int)total;
  A.table_width = kv.table_width;
  A.num_pages = kv.num_pages;
  A.page_size = kv.page_size;
  A.kv_heads = kv.kv_heads;
  A.G = q_heads / kv.kv_heads;
  A.head_blk = kv.head_stride / 64;
  A.q = (const uint8_t*)q;
  A.gate = (const uint8_t*)gate;
  A.q_row = q_row * 2;
  A.q_head = q_head * 2;
  A.g_row = g_row * 2;
  A.g_head = g_head * 2;
  A.out = (uint8_t*)out;
  A.scale_log2 = scale * kLog2e;
  A.ws = (float*)ws;
  A.err = err;
  // Either kernel is right for every batch. us of the few-row / the wide one, back to
  // back over caches beyond L2, 2 kv heads, "short" 65 to 1150 positions, "long" 130
  // to 4000:
  //   head size 256, one token each, 4 query heads a group
  //     sequences          64          128          192          256          512
  //     short       33.2 / 37.0  47.0 / 47.1  59.9 / 61.8  74.4 / 76.1  130.9 / 132.8
  //     long        62.4 / 61.5   101 / 101    142 / 143    184 / 187    350 / 365
  //     1 sequence of 577 18.6 / 17.6; 8 of 8000 43.1 / 43.1; 1000 of up to 300 129 / 137
  //   other groups, 256 short: 1 73.9 / 76.3, 3 73.8 / 76.4, 6 78.3 / 77.4, 8 79.9 / 77.7,
  //     16 99.0 / 79.3
  //   more tokens each, 256 short, group of 4: 2 79.6 / 77.2, 3 89.4 / 77.6, 4 98.4 / 78.6
  //   head size 128, group of 4: 64 short 32.9 / 32.8, long 44.8 / 42.0; 256 short
  //     57.2 / 56.1, long 114 / 106; group of 8, 256 short 67.5 / 56.4
  // At head size 64 half of the few-row kernel's output tile would be empty.
  const bool few = kv.head_dim == 256 && total <= batch && batch >= 64 && A.G <= 4;
  if (kv.dtype == SPOCK_F16) {
    if (kv.head_dim == 64) return launch<__half, 64>(kv, A, few, sms, st);
    if (kv.head_dim == 128) return launch<__half, 128>(kv, A, few, sms, st);
    return launch<__half, 256>(kv, A, few, sms, st);
  }
  if (kv.head_dim == 64) return launch<__nv_bfloat16, 64>(kv, A, few, sms, st);
  if (kv.head_dim == 128) return launch<__nv_bfloat16, 128>(kv, A, few, sms, st);
  return launch<__nv_bfloat16, 256>(kv, A, few, sms, st);
}

}  // namespace spock
