// Host interface of the ragged steps (paged_attn.cu, dn_span.cu,
// draft_verify.cu): several new tokens per sequence in packed rows.
#pragma once
#include "common.cuh"

namespace spock {

constexpr float kLog2e = 1.44269504088896341f;

Status launch_paged_prep(const spock_paged_kv& kv, int batch, const int32_t* start, int64_t total, const void* proj,
                         int64_t proj_ld, int q_heads, bool gated, const void* q_norm, const void* k_norm, float eps,
                         const float* rope, int64_t rope_len, int rotary, void* q_out, int sms, int* err,
                         cudaStream_t st);

size_t paged_attention_workspace(int q_heads, int kv_heads, int head_dim, int sms);
Status launch_paged_attention(const spock_paged_kv& kv, int batch, const int32_t* start, int64_t total, int q_heads,
                              const void* q, int64_t q_row, int64_t q_head, const void* gate, int64_t g_row,
                              int64_t g_head, float scale, void* out, void* ws, int sms, int* err, cudaStream_t st);

Status launch_decode_span(const spock_dn_layer& L, int batch, const int32_t* start, const int32_t* counts,
                          int64_t total, const void* qkv, int64_t qkv_ld, const void* a, const void* b, int64_t ab_ld,
                          const void* z, int64_t z_ld, const void* conv, const float* state, void* conv_out,
                          float* state_out, void* out, int sms, int* err, cudaStream_t st);

struct VerifyArgs {
  const void* logits;
  int64_t logits_ld, total, vocab;
  int batch;
  const int32_t *start, *tokens;
  const float* probs;
  int64_t probs_ld;
  const float *temperature, *u_accept, *u_sample;
  int32_t *emitted, *out_tokens;
  void* ws;
  int sms;
  int* err;
};
size_t draft_verify_workspace(int64_t total, int64_t vocab, int sms);
Status launch_draft_verify(int dtype, const VerifyArgs& a, cudaStream_t st);

}  // namespace spock
