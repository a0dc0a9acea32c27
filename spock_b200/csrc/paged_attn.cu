// Gated full attention of several new tokens per sequence over a KV cache in
// pages: the prep + store of the new tokens' rows (spock_paged_attention_prep)
// and the attention (spock_paged_attention).
//
// paged_prep_kernel, per (token, head), in fp32 with one rounding at the end:
//   y = x / sqrt(mean(x^2) + eps) * (1 + w)
//   (y_d, y_{d+r/2}) <- (y_d c - y_{d+r/2} s, y_{d+r/2} c + y_d s), d < r/2
// with (c, s) the table's row of the token's position. Bound by bandwidth:
// each projected value is read once and each output written once.
#include <algorithm>

#include "ragged.cuh"
#include "ragged.h"

namespace spock {
namespace {

struct Cache {  // spock_paged_kv with typed strides
  uint8_t *k, *v;
  int64_t page_stride, pos_stride, head_stride;  // bytes
  const int32_t* table;
  int64_t table_stride;
  const int32_t* kv_len;
  int table_width, num_pages, page_size, kv_heads;
};
Cache cache_of(const spock_paged_kv& kv) {
  Cache c;
  c.k = static_cast<uint8_t*>(kv.k);
  c.v = static_cast<uint8_t*>(kv.v);
  c.page_stride = kv.page_stride * 2;
  c.pos_stride = kv.pos_stride * 2;
  c.head_stride = kv.head_stride * 2;
  c.table = kv.page_table;
  c.table_stride = kv.table_stride;
  c.kv_len = kv.kv_len;
  c.table_width = kv.table_width;
  c.num_pages = kv.num_pages;
  c.page_size = kv.page_size;
  c.kv_heads = kv.kv_heads;
  return c;
}

// The first CTA's share of a row-parallel kernel's checks: starts that ascend
// within the rows there are, lengths within what the table can hold.
__device__ __forceinline__ void check_ragged(const Cache& c, int batch, const int32_t* __restrict__ start, int total,
                                             int* err) {
  if (blockIdx.x) return;
  bool bad = false;
  for (int b = threadIdx.x; b < batch; b += blockDim.x)
    bad |= start[b] < 0 || start[b + 1] < start[b] || start[b + 1] > total || c.kv_len[b] < 0 ||
           c.kv_len[b] > c.table_width * c.page_size;
  if (bad) report_bad_index(err);
}

// A warp per token and gridDim.y-th of its heads, 8 tokens per CTA; heads
// 0 .. q_heads-1 are queries, the rest kv heads (k and v in one warp). Lane l
// holds dims l*V .. l*V+V-1, V = D/32, so loads and stores are one vector per
// lane and a pair's two halves sit (r/2)/V lanes apart. The token's sequence,
// position and table row are found once for all heads of a warp. Bound by issued
// instructions, then by latency: 4112 tokens of 8 + 2 heads take 15.4 us with 3
// or 4 heads a warp, 18.0 with one and 17.4 with all of them (the same call again and
// again; 17.5 us where inputs change from call to call).
template <typename T, int D>
__global__ void __launch_bounds__(256, 6)
    paged_prep_kernel(Cache c, int batch, const int32_t* __restrict__ start, int total, const T* __restrict__ proj,
                      int64_t proj_ld, int q_heads, int gated, const T* __restrict__ q_norm,
                      const T* __restrict__ k_norm, float eps, const float* __restrict__ rope, int64_t rope_len,
                      int half_rot, T* __restrict__ q_out, int* __restrict__ err) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31, nh = q_heads + c.kv_heads, q_step = gated ? 2 * D : D;
  if (blockIdx.y == 0) check_ragged(c, batch, start, total, err);
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= total) return;
  proj += row * proj_ld + lane * V;
  auto fetch = [&](int hh, uint32_t(&w)[V / 2]) {
    load_words(proj + (hh < q_heads ? (int64_t)hh * q_step : (int64_t)q_heads * q_step + (int64_t)(hh - q_heads) * D), w);
  };
  int hh = blockIdx.y;
  uint32_t w[V / 2];
  fetch(hh, w);
  const int b = seq_of_row(start, batch, (int)row, lane);
  if (b < 0) return;
  const int pos = c.kv_len[b] - (start[b + 1] - start[b]) + ((int)row - start[b]);
  if (pos < 0) return;
  if (half_rot && pos >= rope_len) {
    if (lane == 0) report_bad_index(err);
    return;
  }
  const int hl = half_rot / V;  // lanes per half
  const bool lo = lane < hl, rot = lane < 2 * hl;
  const int other = rot ? (lo ? lane + hl : lane - hl) : lane;
  const float2* const cs =
      reinterpret_cast<const float2*>(rope) + ((int64_t)pos * half_rot + (rot ? (lo ? lane : lane - hl) * V : 0));
  q_out += row * q_heads * D + lane * V;
#pragma unroll 1
  for (;;) {
    const bool is_q = hh < q_heads;
    float x[V];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = Io<T>::up2(w[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
    const T* nw = is_q ? q_norm : k_norm;
    if (nw) {
      load_words(nw + lane * V, w);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float nf = rsqrtf(ss * (1.0f / D) + eps);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 f = Io<T>::up2(w[i]);
        x[2 * i] *= nf * (1.0f + f.x);
        x[2 * i + 1] *= nf * (1.0f + f.y);
      }
    }
    if (half_rot) {
      const float sign = lo ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float y = __shfl_sync(0xffffffffu, x[i], other);
        if (rot) {
          const float2 t = cs[i];
          x[i] = x[i] * t.x + sign * (y * t.y);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = Io<T>::down2(x[2 * i], x[2 * i + 1]);
    if (is_q) {
      store_words(q_out + (int64_t)hh * D, w);
    } else {
      const int slot = pos / c.page_size, kvh = hh - q_heads;
      const int page = slot < c.table_width ? c.table[b * c.table_stride + slot] : -1;
      if (page < 0 || page >= c.num_pages) {
        if (lane == 0) report_bad_index(err);
        return;
      }
      const int64_t at =
          page * c.page_stride + (pos - slot * c.page_size) * c.pos_stride + kvh * c.head_stride + lane * V * 2;
      store_words(c.k + at, w);
      load_words(proj + (int64_t)q_heads * q_step + (int64_t)(c.kv_heads + kvh) * D, w);
      store_words(c.v + at, w);
    }
    hh += gridDim.y;
    if (hh >= nh) return;
    fetch(hh, w);
  }
}

template <typename F>
Status by_type(int dtype, int head_dim, F f) {
  if (dtype == SPOCK_F16) {
    if (head_dim == 64) return f(__half(), std::integral_constant<int, 64>());
    if (head_dim == 128) return f(__half(), std::integral_constant<int, 128>());
    return f(__half(), std::integral_constant<int, 256>());
  }
  if (head_dim == 64) return f(__nv_bfloat16(), std::integral_constant<int, 64>());
  if (head_dim == 128) return f(__nv_bfloat16(), std::integral_constant<int, 128>());
  return f(__nv_bfloat16(), std::integral_constant<int, 256>());
}

}  // namespace

Status launch_paged_prep(const spock_paged_kv& kv, int batch, const int32_t* start, int64_t total, const void* proj,
                         int64_t proj_ld, int q_heads, bool gated, const void* q_norm, const void* k_norm, float eps,
                         const float* rope, int64_t rope_len, int rotary, void* q_out, int sms, int* err,
                         cudaStream_t st) {
  return by_type(kv.dtype, kv.head_dim, [&](auto t, auto d) -> Status {
    using T = decltype(t);
    // two waves of 6 CTAs an SM; a head each while there are few tokens
    const int64_t heads = q_heads + kv.kv_heads, ctas = (total + 7) / 8;
    const int64_t split = std::max<int64_t>(1, std::min<int64_t>(heads, 2 * sms * 6 / ctas));
    const cudaError_t e =
        launch_k(paged_prep_kernel<T, decltype(d)::value>, dim3((unsigned)ctas, (unsigned)split), dim3(256), 0, st,
                 cache_of(kv), batch, start, (int)total, (const T*)proj, proj_ld, q_heads, (int)gated,
                 (const T*)q_norm, (const T*)k_norm, eps, rope, rope_len, rotary / 2, (T*)q_out, err);
    if (e != cudaSuccess) return cuda_status(e, "paged_prep_kernel");
    SPOCK_LAUNCH_CHECK("paged_prep_kernel");
    return Status::ok();
  });
}

}  // namespace spock
