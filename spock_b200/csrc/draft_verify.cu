// Acceptance of drafted tokens from given random numbers (spock_draft_verify).
// With e_j = exp((x_j - max) / T), Z = sum e_j, p_j = e_j / Z:
//   draft x accepted  iff  u q(x) Z < e(x)
//   next token: the lowest j with w_j > 0 and w_0 + .. + w_j > u W, W = sum w,
//   w = max(e / Z - q, 0) at a rejection, e at the last row.
// All of it in 64 bits: a token is decided by the side of a border that a sum
// of up to vocab terms falls on, and neighbouring borders can be 1e-6 W apart.
#include "ragged.cuh"
#include "ragged.h"

namespace spock {
namespace {

constexpr int kT = 512;

struct RowStat {
  double z;    // sum of e
  float top;   // largest logit (-inf if none)
  int best;    // its lowest index
};

template <typename T>
__device__ __forceinline__ float logit(const T* p, int64_t i) {
  const float x = load_as_f32(p, i);
  return x != x ? -INFINITY : x;
}
// e of one logit: 1 at the top (also where it is +inf), 0 for -inf
__device__ __forceinline__ double weight(float x, float top, double inv_t) {
  if (x == -INFINITY) return 0.0;
  if (x == top) return 1.0;
  return exp(((double)x - (double)top) * inv_t);
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ double block_sum(double x, double* red) {
  x = warp_sum(x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < kT / 32; ++w) t += red[w];
  return t;
}

// One CTA per row: top, its index, Z.
template <typename T>
__global__ void __launch_bounds__(kT) verify_stats_kernel(const VerifyArgs A) {
  __shared__ double red[kT / 32];
  __shared__ float sv[kT / 32];
  __shared__ int si[kT / 32];
  const int row = blockIdx.x, t = threadIdx.x;
  const int b = seq_of_row(A.start, A.batch, row, t & 31);
  if (b < 0) return;
  const T* x = static_cast<const T*>(A.logits) + row * A.logits_ld;
  float top = -INFINITY;
  int best = 0x7fffffff;
  for (int64_t j = t; j < A.vocab; j += kT) {
    const float v = logit(x, j);
    if (v > top) top = v, best = (int)j;
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, top, o);
    const int i = __shfl_xor_sync(0xffffffffu, best, o);
    if (v > top || (v == top && i < best)) top = v, best = i;
  }
  if ((t & 31) == 0) sv[t >> 5] = top, si[t >> 5] = best;
  __syncthreads();
  for (int w = 0; w < kT / 32; ++w)
    if (sv[w] > top || (sv[w] == top && si[w] < best)) top = sv[w], best = si[w];
  const float temp = A.temperature ? A.temperature[b] : 1.0f;
  double z = 0.0;
  if (temp > 0.f) {
    const double inv_t = 1.0 / (double)temp;
    for (int64_t j = t; j < A.vocab; j += kT) z += weight(logit(x, j), top, inv_t);
    z = block_sum(z, red);
  }
  if (t == 0) static_cast<RowStat*>(A.ws)[row] = {z, top, best == 0x7fffffff ? 0 : best};
}

// One CTA per sequence: the accepted drafts, the next token.
template <typename T>
__global__ void __launch_bounds__(kT) verify_pick_kernel(const VerifyArgs A) {
  __shared__ double red[kT / 32], part[kT];
  __shared__ int s_pick, s_last;
  const int b = blockIdx.x, t = threadIdx.x;
  const RowSpan rows = row_span(A.start, b, (int)A.total, A.err);
  if (rows.n == 0) {
    if (t == 0) A.emitted[b] = 0;
    return;
  }
  const RowStat* stat = static_cast<const RowStat*>(A.ws);
  const float temp = A.temperature ? A.temperature[b] : 1.0f;
  const bool greedy = !(temp > 0.f);
  const double inv_t = 1.0 / (double)temp;
  int i = 0;
  for (; i < rows.n - 1; ++i) {
    const int r = rows.lo + i, d = A.tokens[r + 1];
    if (d < 0 || d >= A.vocab) {
      if (t == 0) report_bad_index(A.err);
      break;
    }
    if (greedy) {
      if (stat[r].best != d) break;
      continue;
    }
    const double e = weight(logit(static_cast<const T*>(A.logits) + r * A.logits_ld, d), stat[r].top, inv_t);
    const double q = A.probs ? (double)A.probs[r * A.probs_ld + d] : 1.0;
    if (!((double)A.u_accept[r] * q * stat[r].z < e)) break;
  }
  const int r = rows.lo + i;
  const bool drafted = i < rows.n - 1;
  int pick = stat[r].best;
  if (!greedy) {
    const T* x = static_cast<const T*>(A.logits) + r * A.logits_ld;
    const float* q = A.probs ? A.probs + r * A.probs_ld : nullptr;
    const int dropped = drafted ? A.tokens[r + 1] : -1;
    const float top = stat[r].top;
    const double z = stat[r].z;
    bool rest = drafted;
    auto w = [&](int64_t j) -> double {
      const double e = weight(logit(x, j), top, inv_t);
      if (!rest) return e;
      if (!q) return j == dropped ? 0.0 : e;
      return fmax(e / z - (double)q[j], 0.0);
    };
    const int64_t span = (A.vocab + kT - 1) / kT, lo = min(A.vocab, t * span), hi = min(A.vocab, lo + span);
    double mine = 0.0, W = 0.0;
    for (int pass = 0; pass < 2; ++pass) {
      mine = 0.0;
      for (int64_t j = lo; j < hi; ++j) mine += w(j);
      W = block_sum(mine, red);
      if (W > 0.0 || !rest) break;
      rest = false;
    }
    part[t] = mine;
    if (t == 0) s_pick = 0x7fffffff, s_last = 0;
    __syncthreads();
    double before = 0.0;
    for (int k = 0; k < t; ++k) before += part[k];
    const double at = (double)A.u_sample[b] * W;
    int last = -1;
    for (int64_t j = lo; j < hi; ++j) {
      const double v = w(j);
      if (v <= 0.0) continue;
      before += v;
      last = (int)j;
      if (before > at) {
        atomicMin(&s_pick, (int)j);
        break;
      }
    }
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    pick = s_pick == 0x7fffffff ? s_last : s_pick;
  }
  for (int k = t; k < rows.n; k += kT)
    A.out_tokens[rows.lo + k] = k < i ? A.tokens[rows.lo + k + 1] : k == i ? pick : -1;
  if (t == 0) A.emitted[b] = i + 1;
}

template <typename T>
Status launch(const VerifyArgs& a, cudaStream_t st) {
  cudaError_t e = cudaSuccess;
  if (a.total > 0) {
    e = launch_k(verify_stats_kernel<T>, dim3((unsigned)a.total), dim3(kT), 0, st, a);
    if (e != cudaSuccess) return cuda_status(e, "verify_stats_kernel");
    SPOCK_LAUNCH_CHECK("verify_stats_kernel");
  }
  e = launch_k(verify_pick_kernel<T>, dim3(a.batch), dim3(kT), 0, st, a);
  if (e != cudaSuccess) return cuda_status(e, "verify_pick_kernel");
  SPOCK_LAUNCH_CHECK("verify_pick_kernel");
  return Status::ok();
}

}  // namespace

size_t draft_verify_workspace(int64_t total, int64_t, int) { return (size_t)total * sizeof(RowStat) + 16; }

Status launch_draft_verify(int dtype, const VerifyArgs& a, cudaStream_t st) {
  if (dtype == SPOCK_F16) return launch<__half>(a, st);
  if (dtype == SPOCK_BF16) return launch<__nv_bfloat16>(a, st);
  return launch<float>(a, st);
}

}  // namespace spock
