// Acceptance of drafted tokens from given random numbers (spock_draft_verify).
// With e_j = exp((x_j - max) / T), Z = sum e_j, p_j = e_j / Z:
//   draft x accepted  iff  u q(x) Z < e(x)
//   next token: the lowest j with w_j > 0 and w_0 + .. + w_j > u W, W = sum w,
//   w = max(e / Z - q, 0) at a rejection, e at the last row.
// A token is decided by the side of a border that a sum of up to vocab terms
// falls on, and neighbouring borders can be 1e-6 W apart, so decisions are made
// in 64 bits; what 32 bits can decide for certain is decided there.
//
// verify_stats_kernel: one pass over all logits, several CTAs per row, in fp32:
//   each CTA's maximum, its lowest index (greedy rows) or sum of e (sampled).
//   Bound by bandwidth: each logit is read once.
// verify_pick_kernel: one cluster per sequence. A draft whose u q Z and e differ
//   by more than the fp32 sum's error bound is settled; one that does not gets
//   its Z summed again in 64 bits. Then one row per sequence is read for the
//   next token: weights in 64 bits, sums per warp and per 32-lane step kept in
//   shared memory, so that locating the token rescans one step.
#include <cooperative_groups.h>

#include <algorithm>

#include "ragged.cuh"
#include "ragged.h"

namespace cg = cooperative_groups;

namespace spock {
namespace {

constexpr int kT = 256, kW = kT / 32;
constexpr int kCluster = 8;
constexpr int kSteps = 64;  // step sums kept per warp
// The fp32 Z is off by less than this part of itself: each e by 3 roundings of
// its exponent (up to 126 * 2^-24 * 3 ln 2 < 2^-15.8 of e) and ex2's 2^-22, the
// sums by one rounding of 2^-24 per term of a thread (kThreadTerms = 2^11, so
// 2^-13) and some more for joining them.
constexpr double kSure = 1.0 / (1 << 12);
constexpr int64_t kThreadTerms = 2048;

struct Part {  // of one row, by one CTA
  float top;   // largest logit (-inf if none)
  int best;    // its lowest index (greedy)
  float z;     // sum of e relative to top (sampled)
  int pad;
};

template <typename T>
constexpr int kChunk = 16 / (int)sizeof(T);  // elements of a 16-byte load

// Chunk k of a row starts at element k * kChunk - a, a = how far the row's
// first element is behind a 16-byte boundary, so inner chunks are one aligned
// load; elements outside [0, vocab) read as -inf, NaN logits too (fix = true).
template <typename T>
__device__ __forceinline__ int row_shift(const T* row) {
  return (int)(((uintptr_t)row & 15) / sizeof(T));
}
template <typename T, bool kFix>
__device__ __forceinline__ void load_chunk(const T* row, int64_t j0, int64_t vocab, float (&x)[kChunk<T>]) {
  constexpr int C = kChunk<T>;
  if (j0 >= 0 && j0 + C <= vocab) {
    const uint4 u = *reinterpret_cast<const uint4*>(row + j0);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        x[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = Io<T>::up2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = j0 + i >= 0 && j0 + i < vocab ? load_as_f32(row, j0 + i) : -INFINITY;
  }
  if constexpr (kFix) {
#pragma unroll
    for (int i = 0; i < C; ++i) x[i] = fmaxf(x[i], -INFINITY);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a sum relative to maximum m, taken to maximum to >= m
__device__ __forceinline__ float rebase(float z, float m, float to, float c) {
  return m == to ? z : z * ex2((m - to) * c);
}

int stat_splits(int64_t total, int64_t vocab) {
  // enough CTAs for several waves of 8 an SM, at least 8192 logits each; and no
  // thread sums more than kThreadTerms terms
  const int64_t want = total > 0 ? (148 * 32 + total - 1) / total : 1, most = (vocab + 8191) / 8192;
  const int64_t least = (vocab + kThreadTerms * kT / 2 - 1) / (kThreadTerms * kT / 2);
  return (int)std::max(least, std::min(want, most));
}

template <typename T>
__global__ void __launch_bounds__(kT) verify_stats_kernel(const VerifyArgs A, int splits) {
  constexpr int C = kChunk<T>, U = 4;
  __shared__ float s_top[kW], s_z[kW];
  __shared__ int s_best[kW];
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x / splits, part = blockIdx.x % splits, t = threadIdx.x;
  const int b = seq_of_row(A.start, A.batch, row, t & 31);
  if (b < 0) return;
  const float temp = A.temperature ? A.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const float c = 1.44269504088896341f / temp;
  const T* x = static_cast<const T*>(A.logits) + row * A.logits_ld;
  const int a = row_shift(x);
  const int64_t chunks = (A.vocab + a + C - 1) / C;
  const int64_t k0 = chunks * part / splits, k1 = chunks * (part + 1) / splits;
  float top = -INFINITY, z = 0.f;
  int64_t at = -1;  // chunk of the thread's first maximum
  for (int64_t k = k0 + t; k < k1; k += U * kT) {
    float v[U][C];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k + u * kT < k1) {
        load_chunk<T, false>(x, (k + u * kT) * C - a, A.vocab, v[u]);
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) v[u][i] = -INFINITY;
      }
    float m = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float cm = v[u][0];
#pragma unroll
      for (int i = 1; i < C; ++i) cm = fmaxf(cm, v[u][i]);
      if (greedy && cm > m) at = k + u * kT;
      m = fmaxf(m, cm);
    }
    if (!greedy) {
      if (m > top) z = rebase(z, top, m, c);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < C; ++i) z += ex2((v[u][i] - m) * c);
    }
    top = m;
  }
  if (!greedy && !(z < INFINITY)) {  // NaN or +inf among the logits (or none above -inf): once more, with care
    z = 0.f;
    for (int64_t k = k0 + t; k < k1; k += kT) {
      float v[C];
      load_chunk<T, true>(x, k * C - a, A.vocab, v);
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (v[i] > -INFINITY) z += v[i] == top ? 1.0f : ex2((v[i] - top) * c);
    }
  }
  int best = 0x7fffffff;
  if (greedy && at >= 0) {
    float v[C];
    load_chunk<T, true>(x, at * C - a, A.vocab, v);
#pragma unroll
    for (int i = C - 1; i >= 0; --i)
      if (v[i] == top) best = (int)(at * C - a + i);
  }
  // the warp's, then the block's
  const float mine = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, top, o);
    const int i = __shfl_xor_sync(0xffffffffu, best, o);
    if (v > top || (v == top && i < best)) best = i;
    top = fmaxf(top, v);
  }
  z = z > 0.f ? rebase(z, mine, top, c) : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  if ((t & 31) == 0) {
    s_top[t >> 5] = top;
    s_z[t >> 5] = z;
    s_best[t >> 5] = best;
  }
  __syncthreads();
  if (t == 0) {
    for (int w = 1; w < kW; ++w) {
      if (s_top[w] > top || (s_top[w] == top && s_best[w] < best)) best = s_best[w];
      top = fmaxf(top, s_top[w]);
    }
    z = 0.f;
    for (int w = 0; w < kW; ++w) z += s_z[w] > 0.f ? rebase(s_z[w], s_top[w], top, c) : 0.f;
    static_cast<Part*>(A.ws)[(int64_t)row * splits + part] = {top, best, z, 0};
  }
}

// fp32 -> fp64 with integer operations (the conversion instruction runs at a
// fraction of the fp64 rate); zeros and subnormals become about +-2^-127.
__device__ __forceinline__ double widen(float x) {
  const uint32_t u = __float_as_uint(x);
  return __hiloint2double((int)((u & 0x80000000u) | (((u >> 3) & 0x0fffffffu) + (896u << 20))), (int)(u << 29));
}
// 2^(t / 256) for t <= 0: t = n + f with |f| <= 1/2, 2^(n/256) from a table,
// e^r with r = f ln 2 / 256 (|r| < 2^-9.5) as 1 + r + r^2/2 + r^3/6: the next
// term, r^4 / 24, is below 1.4e-13.
__device__ __forceinline__ double exp2_neg(double t, const double* tab) {
  if (t < -256000.0) return 0.0;
  const double big = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
  const double k = t + big;
  const int n = __double2loint(k);
  const double r = (t - (k - big)) * (0.69314718055994530942 / 256.0);
  const double p = fma(fma(r, 1.0 / 6.0, 0.5), r * r, r);
  const double s = tab[n & 255];
  const double y = fma(s, p, s);
  return __hiloint2double(__double2hiint(y) + ((n >> 8) << 20), __double2loint(y));
}

// Combines a row's parts, by one warp.
__device__ __forceinline__ Part join_parts(const Part* p, int splits, float c, int lane) {
  Part r{-INFINITY, 0x7fffffff, 0.f, 0};
  for (int i = lane; i < splits; i += 32) {
    const float top = __ldcg(&p[i].top);
    const int best = __ldcg(&p[i].best);
    if (top > r.top || (top == r.top && best < r.best)) r.best = best;
    r.top = fmaxf(r.top, top);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, r.top, o);
    const int i = __shfl_xor_sync(0xffffffffu, r.best, o);
    if (v > r.top || (v == r.top && i < r.best)) r.best = i;
    r.top = fmaxf(r.top, v);
  }
  for (int i = lane; i < splits; i += 32) {
    const float z = __ldcg(&p[i].z);
    if (z > 0.f) r.z += rebase(z, __ldcg(&p[i].top), r.top, c);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
  return r;
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

enum { kAccept = 0, kReject = 1, kUnsure = 2 };

template <typename T>
__global__ void __launch_bounds__(kT) verify_pick_kernel(const VerifyArgs A, int splits) {
  constexpr int C = kChunk<T>;
  __shared__ double s_tab[256], s_step[kW][kSteps], s_warp[kW], s_all[kCluster * kW];
  __shared__ int s_say[kW];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / ranks, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  s_tab[t] = exp2(t / 256.0);
  pdl_wait();
  pdl_launch();
  const RowSpan rows = row_span(A.start, b, (int)A.total, A.err);
  if (rows.n == 0) {  // all of the cluster
    if (t == 0 && rank == 0) A.emitted[b] = 0;
    return;
  }
  const Part* parts = static_cast<const Part*>(A.ws);
  const T* logits = static_cast<const T*>(A.logits);
  const float temp = A.temperature ? A.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const float c = 1.44269504088896341f / temp;
  const double c256 = 256.0 * 1.44269504088896340736 / (double)temp;
  __syncthreads();

  // e of one logit: 1 at the top (also where it is +inf), 0 for -inf
  auto weight = [&](float x, float top) -> double {
    if (x == -INFINITY) return 0.0;
    if (x == top) return 1.0;
    return exp2_neg((widen(x) - widen(top)) * c256, s_tab);
  };
  const int nw = ranks * kW, me = rank * kW + warp;
  // Sums f over this warp's chunks of row x, step by step; the cluster's sum is
  // in s_all afterwards. f(chunk's first element, logits) -> the chunk's sum.
  int64_t k0 = 0, k1 = 0, per_step = 0;
  auto sum_row = [&](const T* x, auto f) -> double {
    const int a = row_shift(x);
    const int64_t chunks = (A.vocab + a + C - 1) / C;
    k0 = chunks * me / nw;
    k1 = chunks * (me + 1) / nw;
    const int64_t most = (chunks + nw - 1) / nw;  // a warp's most
    per_step = (most + 32 * kSteps - 1) / (32 * kSteps) * 32;
    double all = 0.0;
    int step = 0;
    for (int64_t k = k0; k < k1; k += per_step, ++step) {
      double s = 0.0;
      for (int64_t q = k + lane; q < min(k1, k + per_step); q += 32) {
        float v[C];
        load_chunk<T, true>(x, q * C - a, A.vocab, v);
        s += f(q * C - a, v);
      }
      s = warp_sum(s);
      if (lane == 0) s_step[warp][step] = s;
      all += s;
    }
    cluster.sync();  // the last sums have been read
    if (lane == 0) s_warp[warp] = all;
    cluster.sync();
    for (int i = t; i < nw; i += kT) s_all[i] = cluster.map_shared_rank(s_warp, i / kW)[i % kW];
    __syncthreads();
    double total = 0.0;
    for (int i = 0; i < nw; ++i) total += s_all[i];
    return total;
  };
  auto sum_e = [&](int r, float top) -> double {
    return sum_row(logits + r * A.logits_ld, [&](int64_t, const float(&v)[C]) {
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < C; ++i) s += weight(v[i], top);
      return s;
    });
  };
  auto draft_of = [&](int i) -> int {
    const int d = A.tokens[rows.lo + i + 1];
    return d >= 0 && d < A.vocab ? d : -1;
  };
  // what row i says of its draft, given Z within a factor 1 +- sure
  auto say = [&](int i, const Part& p, double z, double sure) -> int {
    const int r = rows.lo + i, d = draft_of(i);
    if (d < 0) {
      if (lane == 0) report_bad_index(A.err);
      return kReject;
    }
    if (greedy) return (p.best == 0x7fffffff ? 0 : p.best) == d ? kAccept : kReject;
    const double e = weight(fmaxf(load_as_f32(logits + r * A.logits_ld, d), -INFINITY), p.top);
    const double q = A.probs ? (double)A.probs[r * A.probs_ld + d] : 1.0;
    const double uqz = (double)A.u_accept[r] * q * z;
    if (uqz * (1.0 + sure) < e && uqz * (1.0 - sure) < e) return kAccept;
    if (uqz * (1.0 - sure) < e || uqz * (1.0 + sure) < e) return kUnsure;
    return kReject;
  };

  // the first draft that is not accepted
  int i = 0;
  for (const int drafts = rows.n - 1; i < drafts;) {
    const int mine = i + warp;
    Part p{};
    int said = kReject;
    if (mine < drafts) {
      p = join_parts(parts + (int64_t)(rows.lo + mine) * splits, splits, c, lane);
      said = say(mine, p, (double)p.z, kSure);
    }
    __syncthreads();
    if (lane == 0) s_say[warp] = said;
    __syncthreads();
    int w = 0;
    while (w < kW && i + w < drafts && s_say[w] == kAccept) ++w;
    i += w;
    if (w == kW || i >= drafts) continue;
    if (s_say[w] == kReject) break;
    // too near to tell in 32 bits: Z again in 64, by the whole cluster
    p = join_parts(parts + (int64_t)(rows.lo + i) * splits, splits, c, lane);
    const double z = sum_e(rows.lo + i, p.top);
    if (say(i, p, z, 0.0) != kAccept) break;
    ++i;
  }

  const int r = rows.lo + i;
  const bool drafted = i < rows.n - 1;
  const Part p = join_parts(parts + (int64_t)r * splits, splits, c, lane);
  const int drop = drafted ? A.tokens[r + 1] : -1;
  int pick = -1;  // known to one warp of the cluster
  bool mine = rank == 0 && warp == 0;
  if (greedy) {
    pick = p.best == 0x7fffffff ? 0 : p.best;
  } else {
    const T* x = logits + r * A.logits_ld;
    const float* q = drafted && A.probs ? A.probs + r * A.probs_ld : nullptr;
    const double inv_z = q ? 1.0 / sum_e(r, p.top) : 0.0;
    bool rest = drafted;
    auto weights = [&](int64_t j0, const float(&v)[C], double(&w)[C]) {
      float qv[C];
      if (rest && q) {
        if (j0 >= 0 && j0 + C <= A.vocab && ((uintptr_t)(q + j0) & 15) == 0) {
#pragma unroll
          for (int k = 0; k < C; k += 4) {
            const float4 f = *reinterpret_cast<const float4*>(q + j0 + k);
            qv[k] = f.x, qv[k + 1] = f.y, qv[k + 2] = f.z, qv[k + 3] = f.w;
          }
        } else {
#pragma unroll
          for (int k = 0; k < C; ++k) qv[k] = j0 + k >= 0 && j0 + k < A.vocab ? q[j0 + k] : 0.f;
        }
      }
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const double e = weight(v[k], p.top);
        w[k] = !rest ? e : q ? fmax(fma(e, inv_z, -(double)qv[k]), 0.0) : j0 + k == drop ? 0.0 : e;
      }
    };
    auto sum_w = [&]() {
      return sum_row(x, [&](int64_t j0, const float(&v)[C]) {
        double w[C], s = 0.0;
        weights(j0, v, w);
#pragma unroll
        for (int k = 0; k < C; ++k) s += w[k];
        return s;
      });
    };
    double W = sum_w();
    if (rest && !(W > 0.0)) {
      rest = false;
      W = sum_w();
    }
    // the warp whose sums cross u W, or the last that has any weight
    const double at = (double)A.u_sample[b] * W;
    double before = 0.0, b4 = 0.0;
    int owner = -1, last = -1;
    for (int k = 0; k < nw; ++k) {
      if (s_all[k] > 0.0) {
        if (before + s_all[k] > at) {
          owner = k;
          break;
        }
        last = k;
        b4 = before;
      }
      before += s_all[k];
    }
    if (owner < 0) owner = last, before = b4;
    mine = owner < 0 ? mine : me == owner;
    if (owner < 0) pick = 0;  // no weight anywhere
    if (owner >= 0 && mine) {
      const int steps = (int)((k1 - k0 + per_step - 1) / per_step);
      int step = -1, back = -1;
      double sb = before, bb = before;
      for (int k = 0; k < steps; ++k) {
        if (s_step[warp][k] > 0.0) {
          if (sb + s_step[warp][k] > at) {
            step = k;
            break;
          }
          back = k;
          bb = sb;
        }
        sb += s_step[warp][k];
      }
      if (step < 0) step = back, sb = bb;
      // one step's chunks again, in order
      const int a = row_shift(x);
      const int64_t end = min(k1, k0 + (step + 1) * per_step);
      int found = 0x7fffffff, seen = -1;
      for (int64_t k = k0 + step * per_step; k < end && found == 0x7fffffff; k += 32) {
        float v[C];
        double w[C], s = 0.0;
#pragma unroll
        for (int e = 0; e < C; ++e) w[e] = 0.0;
        const int64_t j0 = (k + lane) * C - a;
        if (k + lane < end) {
          load_chunk<T, true>(x, j0, A.vocab, v);
          weights(j0, v, w);
        }
#pragma unroll
        for (int e = 0; e < C; ++e) s += w[e];
        double incl = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        double run = sb + (incl - s);
        int here = 0x7fffffff, tail = -1;
#pragma unroll
        for (int e = 0; e < C; ++e) {
          if (w[e] > 0.0) {
            run += w[e];
            tail = (int)(j0 + e);
            if (run > at && here == 0x7fffffff) here = tail;
          }
        }
        found = __reduce_min_sync(0xffffffffu, here);
        seen = max(seen, __reduce_max_sync(0xffffffffu, tail));
        sb += __shfl_sync(0xffffffffu, incl, 31);
      }
      pick = found != 0x7fffffff ? found : max(seen, 0);
    }
  }
  if (mine && lane == 0) {
    A.out_tokens[r] = pick;
    A.emitted[b] = i + 1;
  }
  if (rank == 0)
    for (int k = t; k < rows.n; k += kT)
      if (k != i) A.out_tokens[rows.lo + k] = k < i ? A.tokens[rows.lo + k + 1] : -1;
  cluster.sync();  // the other CTAs' shared memory stays until all have read it
}

template <typename T>
Status launch(const VerifyArgs& a, cudaStream_t st) {
  const int splits = stat_splits(a.total, a.vocab);
  cudaError_t e = cudaSuccess;
  if (a.total > 0) {
    e = launch_k(verify_stats_kernel<T>, dim3((unsigned)(a.total * splits)), dim3(kT), 0, st, a, splits);
    if (e != cudaSuccess) return cuda_status(e, "verify_stats_kernel");
    SPOCK_LAUNCH_CHECK("verify_stats_kernel");
  }
  // a CTA per 8192 logits of a row, at most the portable cluster size
  int ranks = 1;
  while (ranks < kCluster && (int64_t)ranks * 8192 < a.vocab) ranks *= 2;
  pdl_scope overlap;  // its launch and table run under the first kernel
  e = launch_k_cluster(verify_pick_kernel<T>, dim3((unsigned)a.batch * ranks), dim3(kT), dim3(ranks), 0, st, a,
                       splits);
  if (e != cudaSuccess) return cuda_status(e, "verify_pick_kernel");
  SPOCK_LAUNCH_CHECK("verify_pick_kernel");
  return Status::ok();
}

}  // namespace

size_t draft_verify_workspace(int64_t total, int64_t vocab, int) {
  return (size_t)total * stat_splits(total, vocab) * sizeof(Part) + 16;
}

Status launch_draft_verify(int dtype, const VerifyArgs& a, cudaStream_t st) {
  if (dtype == SPOCK_F16) return launch<__half>(a, st);
  if (dtype == SPOCK_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<float>(a, st);
}

}  // namespace spock
