// Several tokens per sequence through a Gated DeltaNet layer's mixer core
// (spock_deltanet_decode_span). Per token t of a head, with S the 128 x 128
// state (key x value), sums, norms and states in fp32:
//   y = silu(conv4(x)), q = y_q / |y_q| / sqrt(128), k = y_k / |y_k|, v = y_v
//   S <- e^{g_t} S;  d_t = beta_t (v_t - S^T k_t);  S <- S + k_t d_t^T;  o_t = S^T q_t
//   out = rmsnorm(o) * w * silu(z)
// Up to kChunk tokens are taken at once. With E(t,s) = e^{g_{s+1} + .. + g_t}
// and S_0 the state before them,
//   d_t = beta_t (v_t - E(t,-1) S_0^T k_t - sum_{s<t} E(t,s) (k_s . k_t) d_s)
//   o_t =               E(t,-1) S_0^T q_t + sum_{s<=t} E(t,s) (k_s . q_t) d_s
//   S_T = E(T-1,-1) S_0 + sum_s E(T-1,s) k_s d_s^T
// so the state is read for the products S_0^T [k_t, q_t] of all tokens in one
// sweep, and touched again only where it has to be written. E is a product of
// decays (differences of summed logarithms lose a small decay behind a large
// one).
//
// The 64 KiB head states are the traffic, one read (and one write) each; what
// competes with it is issue slots, not arithmetic. The products therefore run
// as mma.sync m16n8k8 tiles with every fp32 operand split into two tf32 parts
// (hi hi + hi lo + lo hi: about 21 bits a product, fp32 sums): 8 tokens fill the
// N side, and no sum crosses lanes by shuffles. As fp32 multiply-adds with
// shuffle sums the kernel issued twice the instructions (64 sequences x 5
// tokens, outputs only: 54 us).
//
// CTAs walk the (sequence, head) items, two CTAs an SM. A head's state comes
// into shared memory by TMA, issued as soon as the previous item's is
// done with; the other inputs of the next item are loaded into registers while
// this one is computed. Warp w owns value columns 16w .. 16w+15, which no other
// column depends on; lane (g = l/4, c = l%4) takes S[8x+2c, 8x+2c+1][16w+2g,
// 16w+2g+1], x < 16: the A fragment of S^T [k, q] (M = column, K = key row) and
// the C fragment of S^T += d k^T (M = column, N = key row) under the same
// relabelling of rows and columns.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "chunk_common.cuh"
#include "ragged.cuh"
#include "ragged.h"
#include "tc.cuh"
#include "tmap.h"

namespace spock {
namespace {

using chunk::mma_tf32;

constexpr int kDim = 128, kThreads = 256, kChunk = 8;

struct SpanArgs {
  int H, batch, total, items;
  const int32_t *start, *counts;
  const __half *qkv, *a, *b, *z;
  int64_t qkv_ld, ab_ld, z_ld;
  const __half *conv_w, *conv;
  const float *a_log_bias, *norm_w, *state;
  __half* conv_out;
  float* state_out;
  __half* out;
  float eps;
  int* err;
};

// Keys and queries of a chunk, before their norms: row t, pair of dims (2p,
// 2p+1) as (hi, hi, lo, lo). The row stride keeps the fragment loads (rows g,
// pairs c) free of bank conflicts.
constexpr int kRow = 68;   // float4 per row
constexpr uint32_t kWait = 1u << 22;
struct __align__(1024) SpanSmem {
  // The state as TMA leaves it: 4 blocks of 32 columns, each [128 rows][128 B]
  // with the 16-byte chunks of row i exchanged by i & 7, so that a fragment's
  // rows 2c (or 2c + 1) fall into different banks.
  float s[4][kDim][32];
  float4 k[kChunk][kRow], q[kChunk][kRow];
  float v[kChunk][kDim];
  float d[2][kChunk][kDim];           // S_0^T k_t, S_0^T q_t; then o in d[1]
  float dd[kChunk][kDim];             // d_s E(T-1, s) / |k_s|
  float part[kThreads / 32][16][10];  // per warp: k.k and q.k over its dims (row stride: see below)
  float gram[16][kChunk];             // rows 0-7 k_t . k_s, 8-15 q_t . k_s
  float qq[kChunk];
  float m[2][kChunk][kChunk];         // E(t,s) (k_s . k_t), E(t,s) (k_s . q_t)
  float c[2][kChunk];                 // E(t,-1) / |k_t|, E(t,-1) / |q_t| / sqrt(128)
  float eg[kChunk], beta[kChunk], last[kChunk];  // last: E(T-1, s) / |k_s|
  uint64_t full;                      // the state has arrived
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

// x as two tf32 parts, hi rounded towards zero and lo what remains, likewise:
// 3 instructions where the rounding conversion takes several more (it was two
// thirds of the products' instructions).
__device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}
// The three products of a split tile, each into sums of its own: a chain of
// dependent MMAs costs their latency.
struct Acc3 {
  float hh[4] = {0.f, 0.f, 0.f, 0.f}, hl[4] = {0.f, 0.f, 0.f, 0.f}, lh[4] = {0.f, 0.f, 0.f, 0.f};
  __device__ __forceinline__ void add(const uint32_t (&ah)[4], const uint32_t (&al)[4], const float4& b) {
    mma_tf32(lh, al, __float_as_uint(b.x), __float_as_uint(b.y));
    mma_tf32(hl, ah, __float_as_uint(b.z), __float_as_uint(b.w));
    mma_tf32(hh, ah, __float_as_uint(b.x), __float_as_uint(b.y));
  }
  __device__ __forceinline__ float sum(int i) const { return hh[i] + (hl[i] + lh[i]); }
};

template <bool kOut>
__global__ void __launch_bounds__(kThreads, 2) dn_span_kernel(const __grid_constant__ CUtensorMap tmap,
                                                                  const __grid_constant__ SpanArgs A) {
  extern __shared__ __align__(1024) uint8_t span_smem[];
  SpanSmem& m = *reinterpret_cast<SpanSmem*>(span_smem);
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, g = lane >> 2, c = lane & 3;
  const int col = warp * 16 + 2 * g;  // and col + 1
  const int conv_dim = A.H * 3 * kDim, step = gridDim.x;
  if (tc::smem_u32(&m) & 1023) {  // never on this toolchain; the exchanged chunks need it
    if (t == 0) atomicExch(A.err, 6);
    return;
  }
  // an item's state (one thread)
  auto load_state = [&](int item) {
    tc::mbar_arrive_expect_tx(&m.full, kDim * kDim * 4);
#pragma unroll
    for (int b = 0; b < 4; ++b) tc::tma_load_2d(m.s[b], &tmap, &m.full, b * 32, item * kDim);
  };
  // rows 8x + 2c + e, columns col, col + 1: block, and chunk before the exchange
  const int chunk = (warp & 1) * 4 + (g >> 1);
  auto state_at = [&](int x, int e) {
    return reinterpret_cast<float2*>(&m.s[warp >> 1][8 * x + 2 * c + e][((chunk ^ (2 * c + e)) << 2) + 2 * (g & 1)]);
  };
  if (t == 0) {
    tc::mbar_init(&m.full, 1);
    tc::fence_mbar_init();
  }
  pdl_wait();
  pdl_launch();
  if (t == 0) load_state(blockIdx.x);
  struct Rows {
    int lo, n;
  };
  auto rows_of = [&](int item) -> Rows {
    const int s = item / A.H;
    const RowSpan r = row_span(A.start, s, A.total, A.err);
    return {r.lo, A.counts ? max(0, min(A.counts[s], r.n)) : r.n};
  };
  // the first chunk's inputs of this thread: channels t (queries, keys) and
  // t + 256 (values, threads 0-127); threads 128 .. hold a token's gates
  struct In {
    __half x[2][kChunk], a, b;
    uint2 conv[2], cw[2];
    float a_log, dt;
  };
  auto channel = [&](int h, int u) {
    const int e = t + u * kThreads;
    return (e / kDim) * A.H * kDim + h * kDim + e % kDim;
  };
  auto load_x = [&](In& in, int h, int row0, int nt) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u * kThreads >= 3 * kDim) continue;
      const __half* xp = A.qkv + row0 * A.qkv_ld + channel(h, u);
#pragma unroll
      for (int j = 0; j < kChunk; ++j)
        if (j < nt) in.x[u][j] = xp[j * A.qkv_ld];
    }
    if (t >= 128 && t < 128 + nt) {
      const int64_t at = (row0 + t - 128) * A.ab_ld + h;
      in.a = A.a[at];
      in.b = A.b[at];
    }
  };
  auto load_in = [&](In& in, int item, const Rows& r) {
    const int s = item / A.H, h = item - s * A.H;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (t + u * kThreads >= 3 * kDim) continue;
      in.conv[u] = *reinterpret_cast<const uint2*>(A.conv + ((size_t)s * conv_dim + channel(h, u)) * 4);
      in.cw[u] = *reinterpret_cast<const uint2*>(A.conv_w + (size_t)channel(h, u) * 4);
    }
    in.a_log = A.a_log_bias[h * 2];
    in.dt = A.a_log_bias[h * 2 + 1];
    load_x(in, h, r.lo, min(kChunk, r.n));
  };
  In in;
  Rows rows = rows_of(blockIdx.x), rows1{0, 0};
  load_in(in, blockIdx.x, rows);
  if (blockIdx.x + step < A.items) rows1 = rows_of(blockIdx.x + step);
  // by single floats, as spock_deltanet_decode_step: a weight need not start on 16 bytes
  float4 norm = make_float4(0.f, 0.f, 0.f, 0.f);
  if (kOut) {
    const float* w = A.norm_w + lane * 4;
    norm = make_float4(w[0], w[1], w[2], w[3]);
  }
  bool ok = true, waited = false;
  int phase = 0;
  __syncthreads();  // the barrier's initialisation
  for (int item = blockIdx.x; item < A.items; item += step) {
    const int s = item / A.H, h = item - s * A.H, n = rows.n;
    const bool more = item + step < A.items;
    waited = false;
    float win[2][4];
    uint2 cw[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const float2 a = Io<__half>::up2(in.conv[u].x), b = Io<__half>::up2(in.conv[u].y);
      win[u][0] = a.x, win[u][1] = a.y, win[u][2] = b.x, win[u][3] = b.y;
      cw[u] = in.cw[u];
    }
    const float a_log = in.a_log, a_dt = in.dt;
    for (int t0 = 0; t0 < n; t0 += kChunk) {
      const int nt = min(kChunk, n - t0);
      const bool last = t0 + nt == n, keep = A.state_out || !last;  // keep: the state is needed after this chunk
      if (t0 > 0) {
        __syncthreads();  // the shared arrays are free again
        load_x(in, h, rows.lo + t0, nt);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t + u * kThreads >= 3 * kDim) continue;
        const float2 c0 = Io<__half>::up2(cw[u].x), c1 = Io<__half>::up2(cw[u].y);
        const int i = t & (kDim - 1);
        float* dst = reinterpret_cast<float*>(t < kDim ? &m.q[0][i >> 1] : &m.k[0][i >> 1]) + (i & 1);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          float y = 0.f;
          if (j < nt) {
            win[u][0] = win[u][1];
            win[u][1] = win[u][2];
            win[u][2] = win[u][3];
            win[u][3] = __half2float(in.x[u][j]);
            y = silu(fmaf(win[u][3], c1.y, fmaf(win[u][2], c1.x, fmaf(win[u][1], c0.y, win[u][0] * c0.x))));
          } else if (!keep) {
            break;  // rows of tokens that are not there only reach their own results, but for the state's update
          }
          if (u == 1) {
            m.v[j][t] = y;
          } else if (kOut || t >= kDim) {
            uint32_t hi, lo;
            split(y, hi, lo);
            dst[j * kRow * 4] = __uint_as_float(hi);
            dst[j * kRow * 4 + 2] = __uint_as_float(lo);
          }
        }
      }
      if (t >= 128 && t < 128 + nt) {  // gates (these threads have no value channel)
        const float x = __half2float(in.a) + a_dt;
        const float sp = fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
        m.eg[t - 128] = expf(-expf(a_log) * sp);
        m.beta[t - 128] = 1.0f / (1.0f + expf(-__half2float(in.b)));
      }
      // the gated norm's inputs, and the next item's, while this chunk is computed
      __half z[4];
      if (kOut && warp < nt) {
        const __half* zp = A.z + (rows.lo + t0 + warp) * A.z_ld + h * kDim + lane * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = zp[i];
      }
      if (last && more) load_in(in, item + step, rows1);
      __syncthreads();
      // products of the tokens' keys and queries: rows k_t (M 0-7) and q_t (8-15)
      // against columns k_s, this warp's 16 dims; and |q_t|^2
      {
        Acc3 p;
#pragma unroll
        for (int x = 2 * warp; x < 2 * warp + 2; ++x) {
          const float4 k = m.k[g][4 * x + c], q = kOut ? m.q[g][4 * x + c] : make_float4(0.f, 0.f, 0.f, 0.f);
          const uint32_t ah[4] = {__float_as_uint(k.x), __float_as_uint(q.x), __float_as_uint(k.y), __float_as_uint(q.y)};
          const uint32_t al[4] = {__float_as_uint(k.z), __float_as_uint(q.z), __float_as_uint(k.w), __float_as_uint(q.w)};
          p.add(ah, al, k);
        }
        *reinterpret_cast<float2*>(&m.part[warp][g][2 * c]) = make_float2(p.sum(0), p.sum(1));
        *reinterpret_cast<float2*>(&m.part[warp][g + 8][2 * c]) = make_float2(p.sum(2), p.sum(3));
        if (kOut && warp < nt) {
          const float4 u = m.q[warp][lane], w = m.q[warp][lane + 32];
          const float y0 = u.x + u.z, y1 = u.y + u.w, y2 = w.x + w.z, y3 = w.y + w.w;
          const float qq = warp_sum(fmaf(y0, y0, y1 * y1) + fmaf(y2, y2, y3 * y3));
          if (lane == 0) m.qq[warp] = qq;
        }
      }
      __syncthreads();
      if (t < 128) {
        float x = 0.f;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) x += m.part[w][t >> 3][t & 7];
        m.gram[t >> 3][t & 7] = x;
      }
      // the state: it has had the conv and the products above to arrive
      if (!waited) {
        ok = tc::mbar_wait_bounded(&m.full, phase & 1, kWait);
        waited = true;
        ++phase;
      }
      if (__syncthreads_or(!ok)) {  // the copy has not arrived: give it as long again to land, and leave
        if (t == 0) {
          atomicExch(A.err, 7);
          tc::mbar_wait_bounded(&m.full, (phase - 1) & 1, kWait);
        }
        return;
      }
      if (t < kChunk * (kChunk + 1)) {
        const int j = t / (kChunk + 1), i = t % (kChunk + 1) - 1;  // i = -1: from before the chunk
        if (j < nt && i <= j) {
          float e = 1.0f;
          for (int u = i + 1; u <= j; ++u) e *= m.eg[u];
          const float ks = rsqrtf(m.gram[j][j] + 1e-6f), qs = kOut ? rsqrtf(m.qq[j] + 1e-6f) * 0.08838834764831845f : 0.f;
          if (i < 0) {
            m.c[0][j] = e * ks;
            m.c[1][j] = e * qs;
          } else {
            const float ki = rsqrtf(m.gram[i][i] + 1e-6f);
            m.m[0][j][i] = e * ks * ki * m.gram[j][i];
            m.m[1][j][i] = e * qs * ki * m.gram[8 + j][i];
            if (j == nt - 1) m.last[i] = e * ki;
          }
        }
      }
      // S_0^T [k, q] of this warp's columns
      {
        Acc3 pk, pq;
#pragma unroll 4
        for (int x = 0; x < 16; ++x) {
          const float2 r0 = *state_at(x, 0), r1 = *state_at(x, 1);
          uint32_t ah[4], al[4];
          split(r0.x, ah[0], al[0]);
          split(r0.y, ah[1], al[1]);
          split(r1.x, ah[2], al[2]);
          split(r1.y, ah[3], al[3]);
          pk.add(ah, al, m.k[g][4 * x + c]);
          if (kOut) pq.add(ah, al, m.q[g][4 * x + c]);
        }
        // rows g, g + 8 of a fragment are columns col, col + 1; its columns the tokens
        *reinterpret_cast<float2*>(&m.d[0][2 * c][col]) = make_float2(pk.sum(0), pk.sum(2));
        *reinterpret_cast<float2*>(&m.d[0][2 * c + 1][col]) = make_float2(pk.sum(1), pk.sum(3));
        if (kOut) {
          *reinterpret_cast<float2*>(&m.d[1][2 * c][col]) = make_float2(pq.sum(0), pq.sum(2));
          *reinterpret_cast<float2*>(&m.d[1][2 * c + 1][col]) = make_float2(pq.sum(1), pq.sum(3));
        }
      }
      __syncthreads();
      if (!keep && more && t == 0) load_state(item + step);
      // d_t and o_t, a column per lane: lanes 0-15 form d_t, lanes 16-31 o_t
      {
        const int type = lane >> 4, mycol = warp * 16 + (lane & 15);
        float dt[kChunk];
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          if (j < nt) {
            float acc = m.c[type][j] * m.d[kOut ? type : 0][j][mycol];
#pragma unroll
            for (int i = 0; i < j; ++i) acc = fmaf(m.m[type][j][i], dt[i], acc);
            const float x = m.beta[j] * (m.v[j][mycol] - acc);
            dt[j] = __shfl_sync(0xffffffffu, x, lane & 15);
            if (type == 1) {
              if (kOut) m.d[1][j][mycol] = fmaf(m.m[1][j][j], dt[j], acc);
            } else {
              m.dd[j][mycol] = dt[j] * m.last[j];
            }
          } else {
            dt[j] = 0.f;
            if (keep && type == 0) m.dd[j][mycol] = 0.f;
          }
        }
      }
      // S_T, where it is needed: for the next tokens or for the caller
      if (keep) {
        float e = 1.0f;
        for (int u = 0; u < nt; ++u) e *= m.eg[u];
        __syncwarp();  // dd: this warp's own columns
        uint32_t ah[4], al[4];
        const float2 d0 = *reinterpret_cast<const float2*>(&m.dd[c][col]);
        const float2 d1 = *reinterpret_cast<const float2*>(&m.dd[c + 4][col]);
        split(d0.x, ah[0], al[0]);
        split(d0.y, ah[1], al[1]);
        split(d1.x, ah[2], al[2]);
        split(d1.y, ah[3], al[3]);
        const float* k0 = reinterpret_cast<const float*>(&m.k[c][g >> 1]) + (g & 1);
        const float* k1 = reinterpret_cast<const float*>(&m.k[c + 4][g >> 1]) + (g & 1);
        float* p = A.state_out ? A.state_out + (size_t)item * kDim * kDim + (size_t)(2 * c) * kDim + col : nullptr;
#pragma unroll 4
        for (int x = 0; x < 16; ++x) {
          float2 *s0 = state_at(x, 0), *s1 = state_at(x, 1);
          const float2 r0 = *s0, r1 = *s1;
          Acc3 a;
          a.add(ah, al, make_float4(k0[16 * x], k1[16 * x], k0[16 * x + 2], k1[16 * x + 2]));
          const float2 n0 = make_float2(fmaf(r0.x, e, a.sum(0)), fmaf(r0.y, e, a.sum(2)));
          const float2 n1 = make_float2(fmaf(r1.x, e, a.sum(1)), fmaf(r1.y, e, a.sum(3)));
          if (last) {
            *reinterpret_cast<float2*>(p + x * 8 * kDim) = n0;
            *reinterpret_cast<float2*>(p + x * 8 * kDim + kDim) = n1;
          } else {
            *s0 = n0;
            *s1 = n1;
          }
        }
        if (!last) tc::fence_async_smem();  // before the next item's copy overwrites it
      }
      if (kOut) {
        __syncthreads();
        if (warp < nt) {  // warp j: the gated norm of token j
          const float4 o = reinterpret_cast<float4*>(m.d[1][warp])[lane];
          const float nf = rsqrtf(warp_sum(o.x * o.x + o.y * o.y + o.z * o.z + o.w * o.w) * (1.0f / kDim) + A.eps);
          const int64_t row = rows.lo + t0 + warp;
          uint2 r;
          r.x = Io<__half>::down2(o.x * nf * norm.x * silu(__half2float(z[0])), o.y * nf * norm.y * silu(__half2float(z[1])));
          r.y = Io<__half>::down2(o.z * nf * norm.z * silu(__half2float(z[2])), o.w * nf * norm.w * silu(__half2float(z[3])));
          *reinterpret_cast<uint2*>(A.out + (row * A.H + h) * kDim + lane * 4) = r;
        }
      }
    }
    if (n == 0) {
      // nothing taken: the state as it was
      ok = tc::mbar_wait_bounded(&m.full, phase & 1, kWait);
      ++phase;
      if (__syncthreads_or(!ok)) {
        if (t == 0) {
          atomicExch(A.err, 7);
          tc::mbar_wait_bounded(&m.full, (phase - 1) & 1, kWait);
        }
        return;
      }
      if (A.state_out) {
        float* p = A.state_out + (size_t)item * kDim * kDim;
        for (int i = t; i < kDim * kDim / 4; i += kThreads)
          reinterpret_cast<float4*>(p)[i] =
              *reinterpret_cast<const float4*>(&m.s[(i >> 3) & 3][i >> 5][((i & 7) ^ ((i >> 5) & 7)) << 2]);
      }
      if (more) load_in(in, item + step, rows1);
    }
    if (A.state_out) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (t + u * kThreads >= 3 * kDim) continue;
        uint2 r;
        r.x = Io<__half>::down2(win[u][0], win[u][1]);
        r.y = Io<__half>::down2(win[u][2], win[u][3]);
        *reinterpret_cast<uint2*>(A.conv_out + ((size_t)s * conv_dim + channel(h, u)) * 4) = r;
      }
    }
    __syncthreads();  // the shared arrays (and a state that was kept) are free again
    if ((A.state_out || n == 0) && more && t == 0) load_state(item + step);
    rows = rows1;
    if (item + 2 * step < A.items) rows1 = rows_of(item + 2 * step);
  }
}

// All heads' states as [items * 128 rows][128], in boxes of 128 rows x 32 columns.
bool encode_states(CUtensorMap* map, const float* state, int items) {
  EncodeFn fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {kDim, (cuuint64_t)items * kDim}, strides[1] = {kDim * 4};
  cuuint32_t box[2] = {32, kDim}, estr[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<float*>(state), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

Status launch_decode_span(const spock_dn_layer& L, int batch, const int32_t* start, const int32_t* counts,
                          int64_t total, const void* qkv, int64_t qkv_ld, const void* a, const void* b, int64_t ab_ld,
                          const void* z, int64_t z_ld, const void* conv, const float* state, void* conv_out,
                          float* state_out, void* out, int sms, int* err, cudaStream_t st) {
  SpanArgs A{};
  A.H = L.num_heads;
  A.batch = batch;
  A.total = (int)total;
  A.start = start;
  A.counts = counts;
  A.qkv = (const __half*)qkv;
  A.a = (const __half*)a;
  A.b = (const __half*)b;
  A.z = (const __half*)z;
  A.qkv_ld = qkv_ld;
  A.ab_ld = ab_ld;
  A.z_ld = z_ld;
  A.conv_w = (const __half*)L.conv_weight;
  A.conv = (const __half*)conv;
  A.a_log_bias = L.a_log_bias;
  A.norm_w = L.norm_weight;
  A.state = state;
  A.conv_out = (__half*)conv_out;
  A.state_out = state_out;
  A.out = (__half*)out;
  A.eps = L.eps;
  A.err = err;
  A.items = L.num_heads * batch;
  CUtensorMap map;
  if (!encode_states(&map, state, A.items))
    return Status::err(SPOCK_ERR_CUDA, "spock_deltanet_decode_span: tensor map encoding failed");
  // the attribute belongs to the kernels on the current device: set once on each
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, "spock_deltanet_decode_span");
  const uint64_t bit = 1ull << (dev & 63);
  if (!(done.load() & bit)) {
    e = cudaFuncSetAttribute(dn_span_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SpanSmem));
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(dn_span_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SpanSmem));
    if (e != cudaSuccess) return cuda_status(e, "dn_span_kernel attribute");
    done.fetch_or(bit);
  }
  e = launch_k(out ? dn_span_kernel<true> : dn_span_kernel<false>, dim3(std::min(A.items, 2 * sms)),
                                 dim3(kThreads), sizeof(SpanSmem), st, map, A);
  if (e != cudaSuccess) return cuda_status(e, "dn_span_kernel");
  SPOCK_LAUNCH_CHECK("dn_span_kernel");
  return Status::ok();
}

}  // namespace spock
