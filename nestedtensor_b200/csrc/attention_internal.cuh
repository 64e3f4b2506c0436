// Internal interface between the attention entry point (attention.cu) and the tcgen05 kernel
// (attention_tcgen05.cu), and between the error-flag query (gemm_bias.cu) and both.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ntb200 {

// Where the sequences lie in the query and key / value matrices: B+1 offsets in elements, row_elems of them per token; lse:
// NULL, or [H, q_tokens] fp32 for the base-2 logarithms of the softmax denominators.
struct AttnRows {
  const int64_t *offsets_q, *offsets_k;
  int64_t row_elems_q, row_elems_k;
  float* lse;
};

int64_t attn_tcgen05_item_capacity(int64_t batch, int64_t total_tokens);
size_t attn_tcgen05_workspace_bytes(int64_t batch, int64_t total_tokens);
// head_dim 64, and with row statistics also 128
bool attn_tcgen05_supported(int64_t batch, int64_t total_tokens, int num_heads, int head_dim, int dtype, bool stats);
// skip_short > 0 (then it must be 32): sequences of at most that many tokens get no work item; single warps of the
// launch that builds the work list compute them
int attn_tcgen05_launch(const void* qkv, void* out, const AttnRows& rows, int64_t batch, int64_t total_tokens, int H, int d, float scaling,
                        int dtype, void* workspace, cudaStream_t st, int skip_short);
// queries of sequence b over the keys / values of sequence b of other matrices (row strides in elements, multiples of 8;
// k_tokens = rows of the key / value matrices); workspace as for the self-attention launch with (batch, q_tokens)
int attn_tcgen05_cross_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* out,
                              const AttnRows& rows, int64_t batch, int64_t q_tokens, int64_t k_tokens, int H, int d, float scaling,
                              int dtype, void* workspace, cudaStream_t st);
// attention_backward.cu: forward pass of training calls in 32-bit tiles (any dtype, head_dim <= 256; tokens and batch < 2^31 - 256)
size_t attn_fwd_tiles_workspace_bytes(int64_t batch, int64_t q_tokens);
int attn_fwd_tiles_launch(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v, int64_t ldv, void* out, const AttnRows& rows,
                          int64_t batch, int64_t q_tokens, int H, int d, float scaling, int dtype, void* workspace, cudaStream_t st);
int attn_tcgen05_error_flags_read_and_clear();
int attn_bwd_tcgen05_error_flags_read_and_clear();  // attention_backward_tcgen05.cu
int construct_error_flags_read_and_clear();  // construct.cu: bit 0 = embedding index out of range

}  // namespace ntb200
