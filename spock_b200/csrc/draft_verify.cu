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
//   its Z summed again in 64 bits (weights good to 1.5e-13: Top). Then one row
//   per sequence is read for the next token: weights in 64 bits, sums per warp
//   and per 32-lane step kept in shared memory, so that locating the token
//   rescans one step.
#include <cooperative_groups.h>

#include <algorithm>

#include "ragged.cuh"
#include "ragged.h"

namespace cg = cooperative_groups;

namespace spock {
namespace {

constexpr int kT = 256, kW = kT / 32;
constexpr int kCluster = 8;
// CTAs of verify_pick_kernel on an SM: its arithmetic needs independent chains
// more than warps (248320 logits x 64 rows: 110 us at 3 with 80 registers and two
// chunks at a time, 129 at 4 with 64).
constexpr int kResident = 3;
constexpr int kSteps = 64;  // step sums kept per warp
constexpr int U = 2;        // chunks in flight, and of independent 64-bit arithmetic
constexpr int kBatch = 32 * U;
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

// A row in 16-byte chunks: chunk k is elements k C - a .. + C - 1, a = how far
// the row's first element is behind a 16-byte boundary, so the inner chunks
// [f0, f1) are one aligned load each; of the others (the first and the last, at
// most) the elements that do not exist read as -inf.
template <typename T>
struct Row {
  static constexpr int C = kChunk<T>;
  const T* x;
  const uint4* base;  // chunk 0 (only inner ones are read as such)
  int a, f0, f1, chunks, vocab;
  __device__ __forceinline__ Row(const T* row, int n) : x(row), vocab(n) {
    a = (int)(((uintptr_t)row & 15) / sizeof(T));
    base = reinterpret_cast<const uint4*>(row - a);
    chunks = (int)(((int64_t)n + a + C - 1) / C);
    f0 = a ? 1 : 0;
    f1 = (int)(((int64_t)n + a) / C);
  }
  __device__ __forceinline__ int first(int k) const { return k * C - a; }  // chunk k's first element
  __device__ __forceinline__ bool inner(int k) const { return k >= f0 && k < f1; }
  __device__ __forceinline__ void open(const uint4& u, float (&v)[C]) const {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[i] = __uint_as_float(w[i]);
      } else {
        const float2 f = Io<T>::up2(w[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  static constexpr uint32_t kNone =  // -inf in each element
      sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
  static __device__ __forceinline__ uint4 none() { return make_uint4(kNone, kNone, kNone, kNone); }
  // any chunk
  __device__ __forceinline__ uint4 fetch(int k) const {
    if (inner(k)) return __ldg(base + k);
    return ragged(x, a, vocab, k);
  }
  static __device__ __noinline__ uint4 ragged(const T* x, int a, int vocab, int k) {
    using Bits = typename std::conditional<sizeof(T) == 4, uint32_t, uint16_t>::type;
    const int64_t j0 = (int64_t)k * C - a;
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const bool there = j0 + i >= 0 && j0 + i < vocab;
      const uint32_t bits = there ? (uint32_t)reinterpret_cast<const Bits*>(x)[j0 + i] : (uint32_t)(Bits)kNone;
      const int at = i * (int)sizeof(T);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u == at >> 2) w[u] |= bits << (at & 3) * 8;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void load(int k, float (&v)[C]) const { open(fetch(k), v); }
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// a sum relative to maximum m, taken to maximum to >= m
__device__ __forceinline__ float rebase(float z, float m, float to, float c) {
  return m == to ? z : z * ex2((m - to) * c);
}

int stat_splits(int64_t total, int64_t vocab, int sms) {
  // a wave of 8 CTAs an SM (more cost more than they hide), at least 8192 logits each; and no
  // thread sums more than kThreadTerms terms
  const int64_t want = total > 0 ? (sms * 8 + total - 1) / total : 1, most = (vocab + 8191) / 8192;
  const int64_t least = (vocab + kThreadTerms * kT / 2 - 1) / (kThreadTerms * kT / 2);
  return (int)std::max(least, std::min(want, most));
}

template <typename T>
__global__ void __launch_bounds__(kT) verify_stats_kernel(const VerifyArgs A, int splits) {
  constexpr int C = kChunk<T>;
  __shared__ float s_top[kW], s_z[kW];
  __shared__ int s_best[kW];
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x / splits, part = blockIdx.x % splits, t = threadIdx.x;
  const Row<T> x(static_cast<const T*>(A.logits) + row * A.logits_ld, (int)A.vocab);
  const int k0 = (int)((int64_t)x.chunks * part / splits), k1 = (int)((int64_t)x.chunks * (part + 1) / splits);
  int k = max(k0, x.f0) + t;
  const int kf = min(k1, x.f1);
  // the first loads go out before the row's sequence is known
  uint4 raw[U];
  const bool full = k + (U - 1) * kT < kf;
  if (full) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __ldg(x.base + k + u * kT);
  }
  const int b = seq_of_row(A.start, A.batch, row, t & 31);
  if (b < 0) return;
  const float temp = A.temperature ? A.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const float c = 1.44269504088896341f / temp;
  float top = -INFINITY, z = 0.f;
  int at = -1;  // chunk of the thread's first maximum
  // a thread's chunks are kT apart, U of them in flight at a time
  auto take = [&](const float(&v)[U][C], int n, int k) {
    float m = top;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= n) break;
      float cm = fmaxf(v[u][0], v[u][1]);
#pragma unroll
      for (int i = 2; i < C; ++i) cm = fmaxf(cm, v[u][i]);
      if (greedy && cm > m) at = k + u * kT;
      m = fmaxf(m, cm);
    }
    if (!greedy) {
      if (m > top) z = rebase(z, top, m, c);
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= n) break;
#pragma unroll
        for (int i = 0; i < C; ++i) s[i & 1] += ex2((v[u][i] - m) * c);
      }
      z += s[0] + s[1];
    }
    top = m;
  };
  float v[U][C];
  for (bool more = full; more;) {
#pragma unroll
    for (int u = 0; u < U; ++u) x.open(raw[u], v[u]);
    const int at_k = k;
    k += U * kT;
    more = k + (U - 1) * kT < kf;
    if (more) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = __ldg(x.base + k + u * kT);
    }
    take(v, U, at_k);
  }
  for (; k < kf; k += kT) {
    x.open(__ldg(x.base + k), v[0]);
    take(v, 1, k);
  }
  // the row's ragged first and last chunks: threads 0 and 1, where this CTA has them
  int edge = t == 0 ? 0 : t == 1 && x.chunks > 1 ? x.chunks - 1 : -1;
  if (edge < k0 || edge >= k1 || x.inner(edge)) edge = -1;
  if (edge >= 0) {
    x.load(edge, v[0]);
    const float was = top;
    const int before = at;
    take(v, 1, edge);
    // among equals the lowest chunk counts, and the first one comes last here
    if (greedy && edge < before && top == was) {
      bool tie = false;
#pragma unroll
      for (int i = 0; i < C; ++i) tie |= v[0][i] == top;
      if (tie) at = edge;
    }
  }
  if (!greedy && !(z < INFINITY)) {  // NaN or +inf among the logits (or none above -inf): once more, with care
    z = 0.f;
    auto add = [&](int q) {
      x.load(q, v[0]);
#pragma unroll
      for (int i = 0; i < C; ++i)
        if (v[0][i] > -INFINITY) z += v[0][i] == top ? 1.0f : ex2((v[0][i] - top) * c);
    };
    for (int q = max(k0, x.f0) + t; q < kf; q += kT) add(q);
    if (edge >= 0) add(edge);
  }
  int best = 0x7fffffff;
  if (greedy && at >= 0) {
    x.load(at, v[0]);
#pragma unroll
    for (int i = C - 1; i >= 0; --i)
      if (v[0][i] == top) best = x.first(at) + i;
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

// What e is relative to, in 64 bits. With t = x c (c = 256 log2(e) / T) and I = rint(max c):
//   e = 2^((t - I) / 256), which is `one` (within 2^(1/512) of 1) at the maximum.
// n = rint(t) - I and f = t - rint(t), |f| <= 1/2, cost three operations as t is
// never rounded by itself: adding 1.5 * 2^52 - I to the exact product leaves n in
// the low word. 2^(n/256) comes from a table, 2^(f/256) as a cubic of f: with
// r = f ln 2 / 256 (|r| < 2^-9.5) the next term, r^4 / 24, is below 1.4e-13. Entry
// i of the table is 2^(i/256) with i * 4096 taken off its high word, so that
// adding n * 4096 (n = 256 k + i) leaves k in the exponent.
struct Top {
  double c, magic;  // 1.5 * 2^52 - I
  float least;      // logits up to this one have no weight (e below 2^-1000, -inf, NaN)
  bool count;       // those above it weigh 1 each: they are +inf, or T is so small
                    // that only logits equal to the largest have any weight
  __device__ __forceinline__ double weight(float x, const double* tab) const {
    constexpr double h = 0.69314718055994530942 / 256.0;
    const double xd = (double)x, k = fma(xd, c, magic), f = fma(xd, c, magic - k);
    const int n = __double2loint(k);
    const double e = tab[n & 255];
    const double s = __hiloint2double(__double2hiint(e) + n * 4096, __double2loint(e));
    const double w = fma(s * f, fma(fma(f, h * h * h / 6.0, h * h / 2.0), f, h), s);
    return x > least ? w : 0.0;
  }
};

__device__ __forceinline__ double warp_scan(double x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}
// 64 sums (two per lane: i = lane, lane + 32) and their running sums: the first
// positive one whose running sum exceeds `at`, or the last positive one, and the
// running sum before it; -1 if none is positive.
__device__ __forceinline__ int first_over(const double (&x)[2], const double (&upto)[2], double at, int lane,
                                          double& before) {
  int i = -1;
#pragma unroll
  for (int h = 1; h >= 0; --h) {
    const unsigned over = __ballot_sync(0xffffffffu, x[h] > 0.0 && upto[h] > at);
    if (over) i = h * 32 + __ffs(over) - 1;
  }
  if (i < 0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned some = __ballot_sync(0xffffffffu, x[h] > 0.0);
      if (some) i = h * 32 + 31 - __clz(some);
    }
  }
  const double b = i < 32 ? upto[0] - x[0] : upto[1] - x[1];
  before = __shfl_sync(0xffffffffu, b, i & 31);
  return i;
}

enum { kAccept = 0, kReject = 1, kUnsure = 2 };

template <typename T>
__global__ void __launch_bounds__(kT, kResident) verify_pick_kernel(const VerifyArgs A, int splits) {
  constexpr int C = kChunk<T>;
  __shared__ double s_tab[256], s_step[kW][kSteps], s_warp[kW];
  __shared__ int s_say[kW];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int b = blockIdx.x / ranks, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  {
    const double e = exp2(t / 256.0);
    s_tab[t] = __hiloint2double(__double2hiint(e) - t * 4096, __double2loint(e));
  }
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
  const double c256 = fmin(256.0 * 1.44269504088896340736 / (double)temp, 1e300);
  __syncthreads();

  auto top_of = [&](float top) -> Top {
    constexpr double big = 6755399441055744.0;  // 1.5 * 2^52
    if (top == INFINITY) return {0.0, big, 3.4028235e38f, true};
    if (top == -INFINITY) return {0.0, big, INFINITY, false};  // no weights
    const float below = nextafterf(top, -INFINITY);
    const double t = (double)top * c256;
    // neighbours of the maximum are 2^-24 of it away, and 2^-24 * 2^49 / 256 octaves down
    if (!(fabs(t) < 562949953421312.0)) return {0.0, big, below, true};
    const double least = (double)top - 256000.0 / c256;
    return {c256, big - rint(t), fminf((float)least, below), false};
  };
  const int nw = ranks * kW, me = rank * kW + warp;
  // Sums f(chunk, logits) over this warp's chunks of a row, step by step; the
  // cluster's sums are in mine2 and upto (running) afterwards.
  int k0 = 0, k1 = 0, per_step = 0;
  double mine2[2], upto[2];
  auto sum_row = [&](const Row<T>& x, auto f) -> double {
    k0 = (int)((int64_t)x.chunks * me / nw);
    k1 = (int)((int64_t)x.chunks * (me + 1) / nw);
    const int most = (x.chunks + nw - 1) / nw;  // a warp's most
    per_step = (most + kBatch * kSteps - 1) / (kBatch * kSteps) * kBatch;
    double all = 0.0;
    int step = 0;
    for (int k = k0; k < k1; k += per_step, ++step) {
      const int end = min(k1, k + per_step);
      double s = 0.0;
      for (int q = k + lane; q - lane < end; q += 32 * U) {
        uint4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = q + u * 32 < end ? x.fetch(q + u * 32) : Row<T>::none();
        s += f(q, end, raw);
      }
      s = warp_sum(s);
      if (lane == 0) s_step[warp][step] = s;
      all += s;
    }
    cluster.sync();  // the last sums have been read
    if (lane == 0) s_warp[warp] = all;
    cluster.sync();
    // every warp: the sums of warps lane and lane + 32, their running sums
    mine2[0] = lane < nw ? cluster.map_shared_rank(s_warp, lane / kW)[lane % kW] : 0.0;
    mine2[1] = lane + 32 < nw ? cluster.map_shared_rank(s_warp, (lane + 32) / kW)[lane % kW] : 0.0;
    upto[0] = warp_scan(mine2[0], lane);
    const double half = __shfl_sync(0xffffffffu, upto[0], 31);
    upto[1] = half + warp_scan(mine2[1], lane);
    return __shfl_sync(0xffffffffu, upto[1], 31);
  };
  auto row_of = [&](int r) { return Row<T>(logits + r * A.logits_ld, (int)A.vocab); };
  // a chunk's weights: e; e without the draft's; max(e / Z - q, 0)
  auto plain = [&](const Row<T>& x, const Top& top, const uint4& raw, double(&w)[C]) {
    float v[C];
    x.open(raw, v);
    if (top.count) {
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = v[i] > top.least ? 1.0 : 0.0;
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) w[i] = top.weight(v[i], s_tab);
    }
  };
  auto add_up = [](const double(&w)[C]) {
    double s[2] = {0.0, 0.0};
#pragma unroll
    for (int i = 0; i < C; ++i) s[i & 1] += w[i];
    return s[0] + s[1];
  };
  auto sum_e = [&](const Row<T>& x, const Top& top) -> double {
    return sum_row(x, [&](int, int, const uint4(&raw)[U]) {
      double s = 0.0, w[C];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        plain(x, top, raw[u], w);
        s += add_up(w);
      }
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
    if (sure > 0.0 && !(c < INFINITY)) return kUnsure;  // T below 2^-127: the Z of 32 bits counts equal logits only
    const Top top = top_of(p.top);
    const float x = load_as_f32(logits + r * A.logits_ld, d);
    const double e = top.count ? (double)(x > top.least) : top.weight(x, s_tab);
    if (sure > 0.0 && !top.count) z *= top.weight(p.top, s_tab);  // Z of 32 bits is relative to e = 1 at the maximum
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
    const double z = sum_e(row_of(rows.lo + i), top_of(p.top));
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
    const Row<T> x = row_of(r);
    const float* q = drafted && A.probs ? A.probs + r * A.probs_ld - x.a : nullptr;  // chunk k's start at q + k C
    const Top top = top_of(p.top);
    const double inv_z = q ? 1.0 / sum_e(x, top) : 0.0;
    const bool q16 = ((uintptr_t)q & 15) == 0;  // whether they are aligned too
    auto fetch_q = [&](int k, float(&qv)[C]) {  // 0 where the chunk has no element
      if (q16 && x.inner(k)) {
#pragma unroll
        for (int i = 0; i < C; i += 4) {
          const float4 f = __ldg(reinterpret_cast<const float4*>(q + (int64_t)k * C + i));
          qv[i] = f.x, qv[i + 1] = f.y, qv[i + 2] = f.z, qv[i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < C; ++i) {
          const int64_t j = (int64_t)k * C - x.a + i;
          qv[i] = j >= 0 && j < A.vocab ? __ldg(q + (int64_t)k * C + i) : 0.f;
        }
      }
    };
    auto without = [&](int k, double(&w)[C]) {
      const int64_t at = (int64_t)drop + x.a - (int64_t)k * C;
      if (at >= 0 && at < C) {
#pragma unroll
        for (int i = 0; i < C; ++i) w[i] = i == at ? 0.0 : w[i];
      }
    };
    auto beyond = [&](const float(&qv)[C], double(&w)[C]) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const double y = fma(w[i], inv_z, -(double)qv[i]);
        w[i] = y > 0.0 ? y : 0.0;
      }
    };
    auto sum_plain = [&] { return sum_e(x, top); };
    auto sum_without = [&] {
      return sum_row(x, [&](int k, int, const uint4(&raw)[U]) {
        double s = 0.0, w[C];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          plain(x, top, raw[u], w);
          without(k + u * 32, w);
          s += add_up(w);
        }
        return s;
      });
    };
    auto sum_beyond = [&] {
      return sum_row(x, [&](int k, int end, const uint4(&raw)[U]) {
        double s = 0.0, w[C];
        float qv[C];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (k + u * 32 < end) {
            fetch_q(k + u * 32, qv);
          } else {
#pragma unroll
            for (int i = 0; i < C; ++i) qv[i] = 0.f;
          }
          plain(x, top, raw[u], w);
          beyond(qv, w);
          s += add_up(w);
        }
        return s;
      });
    };
    bool rest = drafted;
    double W = rest ? (q ? sum_beyond() : sum_without()) : sum_plain();
    if (rest && !(W > 0.0)) {
      rest = false;
      W = sum_plain();
    }
    // the warp whose sums cross u W, or the last that has any weight
    const double at = (double)A.u_sample[b] * W;
    double before = 0.0;
    int owner = first_over(mine2, upto, at, lane, before);
    mine = owner < 0 ? mine : me == owner;
    if (owner < 0) pick = 0;  // no weight anywhere
    if (owner >= 0 && mine) {
      const int steps = (k1 - k0 + per_step - 1) / per_step;
      const double sums[2] = {lane < steps ? s_step[warp][lane] : 0.0, lane + 32 < steps ? s_step[warp][lane + 32] : 0.0};
      double run2[2], sb = 0.0;
      run2[0] = before + warp_scan(sums[0], lane);
      run2[1] = __shfl_sync(0xffffffffu, run2[0], 31) + warp_scan(sums[1], lane);
      const int step = max(first_over(sums, run2, at, lane, sb), 0);
      // one step's chunks again, in order
      const int end = min(k1, k0 + (step + 1) * per_step);
      int found = 0x7fffffff, seen = -1;
      for (int k = k0 + step * per_step; k < end && found == 0x7fffffff; k += 32) {
        double w[C], s = 0.0;
#pragma unroll
        for (int e = 0; e < C; ++e) w[e] = 0.0;
        const int j0 = x.first(k + lane);
        if (k + lane < end) {
          plain(x, top, x.fetch(k + lane), w);
          if (rest && q) {
            float qv[C];
            fetch_q(k + lane, qv);
            beyond(qv, w);
          } else if (rest) {
            without(k + lane, w);
          }
        }
#pragma unroll
        for (int e = 0; e < C; ++e) s += w[e];
        const double incl = warp_scan(s, lane);
        double run = sb + (incl - s);
        int here = 0x7fffffff, tail = -1;
#pragma unroll
        for (int e = 0; e < C; ++e) {
          if (w[e] > 0.0) {
            run += w[e];
            tail = j0 + e;
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
  const int splits = stat_splits(a.total, a.vocab, a.sms);
  cudaError_t e = cudaSuccess;
  if (a.total > 0) {
    e = launch_k(verify_stats_kernel<T>, dim3((unsigned)(a.total * splits)), dim3(kT), 0, st, a, splits);
    if (e != cudaSuccess) return cuda_status(e, "verify_stats_kernel");
    SPOCK_LAUNCH_CHECK("verify_stats_kernel");
  }
  // a CTA per 8192 logits of a row, up to the portable cluster size, while all are resident at once
  const int64_t most = std::min<int64_t>(kCluster, (a.vocab + 8191) / 8192);
  const int ranks = (int)std::max<int64_t>(1, std::min<int64_t>(most, a.sms * kResident / a.batch));
  pdl_scope overlap;  // its launch and table run under the first kernel
  e = launch_k_cluster(verify_pick_kernel<T>, dim3((unsigned)a.batch * ranks), dim3(kT), dim3(ranks), 0, st, a,
                       splits);
  if (e != cudaSuccess) return cuda_status(e, "verify_pick_kernel");
  SPOCK_LAUNCH_CHECK("verify_pick_kernel");
  return Status::ok();
}

}  // namespace

size_t draft_verify_workspace(int64_t total, int64_t vocab, int sms) {
  return (size_t)total * stat_splits(total, vocab, sms) * sizeof(Part) + 16;
}

Status launch_draft_verify(int dtype, const VerifyArgs& a, cudaStream_t st) {
  if (dtype == SPOCK_F16) return launch<__half>(a, st);
  if (dtype == SPOCK_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<float>(a, st);
}

}  // namespace spock
