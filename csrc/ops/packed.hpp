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
  void* o_rest = nullptr;   // [tokens, heads, head_dim], may be null: what rounding o to 16 bits left, rounded to 16 bits (zero in rows of no sequence or not written)
  int tokens = 0, k_tokens = 0, sequences = 0;
  int heads = 0, kv_heads = 0, head_dim = 0;
  float scale = 1.f;
  int window = 0, sinks = 0;
  Half16 type = Half16::bf16;
  void* workspace = nullptr;   // packed_attention_workspace() bytes, on a 16-byte boundary
};
size_t packed_attention_workspace(const PackedAttentionArgs& a);
cudaError_t packed_attention(const PackedAttentionArgs& a, cudaStream_t stream);

// ---- its gradients, bf16.  f.o, f.o_rest and f.lse are what the forward call left, d_o [tokens, heads, head_dim]; dq, dk and dv are contiguous and
// zero in rows of no sequence.  delta: [heads, tokens] fp32 of room.  Every sum is taken in an order that depends on the sizes only.
struct PackedAttentionGradArgs {
  PackedAttentionArgs f;
  TokenView d_o;
  void* dq = nullptr;
  void* dk = nullptr;
  void* dv = nullptr;
  float* delta = nullptr;
};
cudaError_t packed_attention_grad(const PackedAttentionGradArgs& a, cudaStream_t stream);

// ---- rotary positions.  x [tokens, heads, head_dim] and, where its `heads` is not zero, k of the same tokens: the first 2 * width elements of every head are
// turned by row positions[t] (null: t) of cos / sin (fp32 [rope_rows, width]) into contiguous out; the others are copied.  Pairs are neighbours or, with `halves`,
// `width` apart; `inverse` turns the other way.  A token whose position lies outside the tables becomes zeros.  head_dim % 8 == 0, width % 4 == 0.
struct RotaryPart {
  TokenView x;
  void* out = nullptr;
  int heads = 0;
};
struct RotaryArgs {
  RotaryPart q, k;
  const float* cos = nullptr;
  const float* sin = nullptr;
  const int* positions = nullptr;
  int rope_rows = 0, width = 0;
  int tokens = 0, head_dim = 0;
  bool halves = false, inverse = false;
  Half16 type = Half16::bf16;
};
cudaError_t rotary(const RotaryArgs& a, cudaStream_t stream);

// ---- one token per row of logits [rows, vocab] (stride elements apart).  With w_i = exp((l_i - max) / temperature): the top_k likeliest (<= 0: all; the lowest
// numbers among equals), of these the fewest likeliest whose weights reach top_p times the sum of these (>= 1: all), of these the ones with w >= min_p; then the
// lowest i for which the sum of the kept w_j, j <= i, exceeds uniform[row] times their whole sum.  temperature 0: the likeliest.  -1 for a row that holds a NaN
// or +inf or nothing finite, or whose temperature is negative or NaN.  vocab <= 2^20.
enum class Logits : int { bf16 = 0, fp16 = 1, fp32 = 2 };
template <typename T>
struct RowSetting {
  const T* each = nullptr;   // one per row, or
  T all = T(0);              // one for all
};
struct SampleArgs {
  const void* logits = nullptr;
  long long stride = 0;
  Logits type = Logits::bf16;
  int rows = 0, vocab = 0;
  const void* uniform = nullptr;   // fp32, or fp64
  bool uniform64 = false;
  RowSetting<float> temperature, top_p, min_p;
  RowSetting<int> top_k;
  long long* tokens = nullptr;
};
cudaError_t sample(const SampleArgs& a, cudaStream_t stream);

}  // namespace ops
}  // namespace mccl
