// Several tokens per sequence through a Gated DeltaNet layer's mixer core
// (spock_deltanet_decode_span). Per token t of a head, with S the 128 x 128
// state (key x value), in fp32 throughout:
//   y = silu(conv4(x)), q = y_q / |y_q| / sqrt(128), k = y_k / |y_k|, v = y_v
//   S <- e^{g_t} S;  d = beta_t (v - S^T k);  S <- S + k d^T;  o = S^T q
//   out = rmsnorm(o) * w * silu(z)
// One CTA per (sequence, head): the 64 KiB state is read once, kept in
// registers over all tokens and written once, and only where the caller asks.
// Warp w owns value columns 16w .. 16w+15, which no other column depends on;
// lane l holds rows i*8 + l/4 (i < 16) of columns 4(l%4) .. +3 of them.
#include "ragged.cuh"
#include "ragged.h"

namespace spock {
namespace {

constexpr int kDim = 128, kThreads = 256, kChunk = 8;

struct SpanArgs {
  int H, batch, total;
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

struct SpanSmem {
  float q[kChunk][kDim], k[kChunk][kDim], v[kChunk][kDim], o[kChunk][kDim];
  float eg[kChunk], beta[kChunk];
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ float silu(float x) { return x / (1.0f + expf(-x)); }

__global__ void __launch_bounds__(kThreads, 2) dn_span_kernel(const __grid_constant__ SpanArgs A) {
  __shared__ __align__(16) SpanSmem m;
  const int s = blockIdx.x / A.H, h = blockIdx.x % A.H, t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const RowSpan rows = row_span(A.start, s, A.total, A.err);
  const int n = A.counts ? max(0, min(A.counts[s], rows.n)) : rows.n;
  const int conv_dim = A.H * 3 * kDim;
  if (n == 0 && !A.state_out) return;
  // state -> registers
  const int rg = lane >> 2, col = warp * 16 + (lane & 3) * 4;
  const size_t sbase = ((size_t)s * A.H + h) * kDim * kDim;
  float4 S[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    S[i] = *reinterpret_cast<const float4*>(A.state + sbase + (size_t)(i * 8 + rg) * kDim + col);
  // conv windows of channels t and t + 256
  float win[2][4], cw[2][4];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int c = t + u * kThreads;
    if (c >= 3 * kDim) continue;
    const int ch = (c / kDim) * A.H * kDim + h * kDim + c % kDim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      win[u][i] = __half2float(A.conv[((size_t)s * conv_dim + ch) * 4 + i]);
      cw[u][i] = __half2float(A.conv_w[(size_t)ch * 4 + i]);
    }
  }
  for (int t0 = 0; t0 < n; t0 += kChunk) {
    const int nt = min(kChunk, n - t0);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = t + u * kThreads;
      if (c >= 3 * kDim) continue;
      const int blk = c / kDim, off = c % kDim, ch = blk * A.H * kDim + h * kDim + off;
      float* dst = blk == 0 ? &m.q[0][off] : blk == 1 ? &m.k[0][off] : &m.v[0][off];
      for (int j = 0; j < nt; ++j) {
        win[u][0] = win[u][1];
        win[u][1] = win[u][2];
        win[u][2] = win[u][3];
        win[u][3] = __half2float(A.qkv[(rows.lo + t0 + j) * A.qkv_ld + ch]);
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) y = fmaf(win[u][i], cw[u][i], y);
        dst[j * kDim] = silu(y);
      }
    }
    __syncthreads();
    if (warp < nt) {  // warp j: norms and gates of token j
      float4 q = reinterpret_cast<float4*>(m.q[warp])[lane], k = reinterpret_cast<float4*>(m.k[warp])[lane];
      const float qs = rsqrtf(warp_sum(q.x * q.x + q.y * q.y + q.z * q.z + q.w * q.w) + 1e-6f) * 0.08838834764831845f;
      const float ks = rsqrtf(warp_sum(k.x * k.x + k.y * k.y + k.z * k.z + k.w * k.w) + 1e-6f);
      reinterpret_cast<float4*>(m.q[warp])[lane] = make_float4(q.x * qs, q.y * qs, q.z * qs, q.w * qs);
      reinterpret_cast<float4*>(m.k[warp])[lane] = make_float4(k.x * ks, k.y * ks, k.z * ks, k.w * ks);
      if (lane == 0) {
        const int64_t at = (rows.lo + t0 + warp) * A.ab_ld + h;
        const float x = __half2float(A.a[at]) + A.a_log_bias[h * 2 + 1];
        const float sp = fmaxf(x, 0.f) + log1pf(expf(-fabsf(x)));
        m.eg[warp] = expf(-expf(A.a_log_bias[h * 2]) * sp);
        m.beta[warp] = 1.0f / (1.0f + expf(-__half2float(A.b[at])));
      }
    }
    __syncthreads();
    for (int j = 0; j < nt; ++j) {
      const float eg = m.eg[j], beta = m.beta[j];
      float4 kv = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float k = m.k[j][i * 8 + rg];
        S[i].x *= eg, S[i].y *= eg, S[i].z *= eg, S[i].w *= eg;
        kv.x = fmaf(S[i].x, k, kv.x);
        kv.y = fmaf(S[i].y, k, kv.y);
        kv.z = fmaf(S[i].z, k, kv.z);
        kv.w = fmaf(S[i].w, k, kv.w);
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        kv.x += __shfl_xor_sync(0xffffffffu, kv.x, o);
        kv.y += __shfl_xor_sync(0xffffffffu, kv.y, o);
        kv.z += __shfl_xor_sync(0xffffffffu, kv.z, o);
        kv.w += __shfl_xor_sync(0xffffffffu, kv.w, o);
      }
      const float4 v = *reinterpret_cast<const float4*>(&m.v[j][col]);
      const float4 d = make_float4(beta * (v.x - kv.x), beta * (v.y - kv.y), beta * (v.z - kv.z), beta * (v.w - kv.w));
      float4 ov = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float k = m.k[j][i * 8 + rg], q = m.q[j][i * 8 + rg];
        S[i].x = fmaf(k, d.x, S[i].x);
        S[i].y = fmaf(k, d.y, S[i].y);
        S[i].z = fmaf(k, d.z, S[i].z);
        S[i].w = fmaf(k, d.w, S[i].w);
        ov.x = fmaf(S[i].x, q, ov.x);
        ov.y = fmaf(S[i].y, q, ov.y);
        ov.z = fmaf(S[i].z, q, ov.z);
        ov.w = fmaf(S[i].w, q, ov.w);
      }
      if (A.out) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          ov.x += __shfl_xor_sync(0xffffffffu, ov.x, o);
          ov.y += __shfl_xor_sync(0xffffffffu, ov.y, o);
          ov.z += __shfl_xor_sync(0xffffffffu, ov.z, o);
          ov.w += __shfl_xor_sync(0xffffffffu, ov.w, o);
        }
        if (rg == 0) *reinterpret_cast<float4*>(&m.o[j][col]) = ov;
      }
    }
    if (A.out) {
      __syncthreads();
      if (warp < nt) {
        const float4 o = reinterpret_cast<float4*>(m.o[warp])[lane];
        const float nf =
            rsqrtf(warp_sum(o.x * o.x + o.y * o.y + o.z * o.z + o.w * o.w) * (1.0f / kDim) + A.eps);
        const float ov[4] = {o.x, o.y, o.z, o.w};
        const int64_t row = rows.lo + t0 + warp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int d = lane * 4 + i;
          const float z = __half2float(A.z[row * A.z_ld + h * kDim + d]);
          A.out[(row * A.H + h) * kDim + d] = __float2half_rn(ov[i] * nf * A.norm_w[d] * silu(z));
        }
      }
    }
  }
  if (A.state_out) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      *reinterpret_cast<float4*>(A.state_out + sbase + (size_t)(i * 8 + rg) * kDim + col) = S[i];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = t + u * kThreads;
      if (c >= 3 * kDim) continue;
      const int ch = (c / kDim) * A.H * kDim + h * kDim + c % kDim;
#pragma unroll
      for (int i = 0; i < 4; ++i) A.conv_out[((size_t)s * conv_dim + ch) * 4 + i] = __float2half_rn(win[u][i]);
    }
  }
}

}  // namespace

Status launch_decode_span(const spock_dn_layer& L, int batch, const int32_t* start, const int32_t* counts,
                          int64_t total, const void* qkv, int64_t qkv_ld, const void* a, const void* b, int64_t ab_ld,
                          const void* z, int64_t z_ld, const void* conv, const float* state, void* conv_out,
                          float* state_out, void* out, int* err, cudaStream_t st) {
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
  const cudaError_t e = launch_k(dn_span_kernel, dim3((unsigned)(L.num_heads * batch)), dim3(kThreads), 0, st, A);
  if (e != cudaSuccess) return cuda_status(e, "dn_span_kernel");
  SPOCK_LAUNCH_CHECK("dn_span_kernel");
  return Status::ok();
}

}  // namespace spock
