// Host entry points of the operators around whole prompts and packed texts: causal attention of sequences that lie one behind the other,
// rotary positions, and the choice of tokens from logits.  All enqueue on the given stream and return the launch status; nothing here
// allocates.  The reference has no counterpart (it has collectives and no model operators).
#pragma once

#include <cuda_runtime.h>

#include "serving.hpp"

namespace mccl {
namespace ops {

// ---- causal attention of packed sequences.  Sequence s has the queries offsets[s] .. offsets[s + 1] - 1 and the keys k_offsets[s] ..
// k_offsets[s + 1] - 1; its last query stands at its last key.  A query at position p sees keys j <= p with j > p - window or j < sinks
// (window <= 0: all).  o [tokens, heads, head_dim] = softmax(scale q.K) V, zero where nothing is seen and in rows of no sequence; lse [heads,
// tokens] (may be null): log of the sum of exponentials, -inf there.  Offsets are clamped to the tensors; they must not decrease.
// heads % kv_heads == 0, head_dim % 8 == 0 and <= 128, strides as TokenView has them.
struct PackedAttentionArgs {
  TokenView q, k, v;
  const int* offsets = nullptr;
  const int* k_offsets = nullptr;
  void* o = nullptr;
  float* lse = nullptr;
  int tokens = 0, k_tokens = 0, sequences = 0;
  int heads = 0, kv_heads = 0, head_dim = 0;
  float scale = 1.f;
  int window = 0, sinks = 0;
  Half16 type = Half16::bf16;
};
cudaError_t packed_attention(const PackedAttentionArgs& a, cudaStream_t stream);

// ---- its gradients, bf16.  o and lse are what the forward call left (f.o is not written), d_o [tokens, heads, head_dim]; dq, dk and dv are contiguous and
// zero in rows of no sequence.  delta: [heads, tokens] fp32 of room.  Every sum is taken in an order that depends on the sizes only.
struct PackedAttentionGradArgs {
  PackedAttentionArgs f;
  TokenView o, d_o;
  void* dq = nullptr;
  void* dk = nullptr;
  void* dv = nullptr;
  float* delta = nullptr;
};
cudaError_t packed_attention_grad(const PackedAttentionGradArgs& a, cudaStream_t stream);

}  // namespace ops
}  // namespace mccl
