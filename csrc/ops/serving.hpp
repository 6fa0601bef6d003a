// Host entry points of the operators that answer token by token: a paged key-value cache, attention of single new tokens over
// it, and products with 4-bit weights.  All enqueue on the given stream and return the launch status; nothing here allocates.
// The reference has no counterpart (it has collectives and no model operators).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mccl {
namespace ops {

enum class Half16 : int { bf16 = 0, fp16 = 1 };

// Keys or values of a cache: [pages, kv_heads, page_size, head_dim] with head_dim contiguous; strides in elements, multiples of 8,
// and a base on a 16-byte boundary.
struct PagedTensor {
  void* p = nullptr;
  long long page = 0, head = 0, token = 0;
};
// Row r of the table holds the pages of sequence r in order: position j is in page table[r * stride + j / page_size].
struct PageTable {
  const int* p = nullptr;
  long long stride = 0;
  int rows = 0, width = 0;
  int page_size = 0;
  int pages = 0;   // pages the cache has: entries outside [0, pages) are never followed
};
// [tokens, heads, head_dim] with head_dim contiguous; strides in elements, multiples of 8, base on a 16-byte boundary.
struct TokenView {
  const void* p = nullptr;
  long long token = 0, head = 0;
};

// ---- keys and values of new tokens into their pages.  Token t belongs to table row rows[t] (rows null: t) and has position
// positions[t]; one whose row, position or page lies outside the table, the cache or the rotation tables writes nothing into the cache.
// cos / sin (fp32 [rope_rows, head_dim / 2], may be null): k, and q (into q_out [tokens, heads, head_dim], may be null), are rotated in
// pairs of (even, odd) elements; q_out is zero for a token that writes nothing.  head_dim % 8 == 0.
struct AppendArgs {
  TokenView k, v, q;
  PagedTensor k_pages, v_pages;
  PageTable table;
  const int* positions = nullptr;
  const int* rows = nullptr;
  const float* cos = nullptr;
  const float* sin = nullptr;
  int rope_rows = 0;
  void* q_out = nullptr;
  long long tokens = 0;
  int heads = 0, kv_heads = 0, head_dim = 0;
  Half16 type = Half16::bf16;
};
cudaError_t paged_append(const AppendArgs& a, cudaStream_t stream);

// ---- pages[o, dst[i], :] = pages[o, src[i], :] for every o < outer and i < count.  Strides and sizes in bytes.  No page may be named
// twice among dst, nor as dst of one copy and src of another; pairs with an index outside [0, pages) are skipped.
cudaError_t copy_pages(void* base, long long outer, long long outer_stride, long long page_stride, long long page_bytes, int pages,
                       const int* src, const int* dst, long long count, cudaStream_t stream);

// ---- attention of one new token per sequence over the cache.  Sequence b sees positions j < lengths[b] with j >= lengths[b] - window or
// j < sinks (window <= 0: all).  o [batch, heads, head_dim] = softmax(scale q.K) V, zero where nothing is seen; lse [batch, heads] (may be
// null): log of the sum of exponentials, -inf where nothing is seen.  heads % kv_heads == 0, head_dim % 8 == 0 and <= 256.
struct PagedAttentionArgs {
  TokenView q;
  PagedTensor k_pages, v_pages;
  PageTable table;
  const int* lengths = nullptr;
  void* o = nullptr;
  float* lse = nullptr;
  void* workspace = nullptr;   // paged_attention_workspace() bytes
  int batch = 0, heads = 0, kv_heads = 0, head_dim = 0;
  float scale = 1.f;
  int window = 0, sinks = 0;
  Half16 type = Half16::bf16;
};
size_t paged_attention_workspace(const PagedAttentionArgs& a);
cudaError_t paged_attention(const PagedAttentionArgs& a, cudaStream_t stream);

// ---- y[m, n] = act(sum_k x[m, k] scale[n, k / group] (code[n, k] - zero[n, k / group]) + bias[n]) + residual[m, n], bf16.
// Weights as laid out by mccl_b200/ops/w4.py: tiles of 16 rows and 64 columns, 512 bytes each, [ceil(n / 16), ceil(k / 64)]; a lane's 16
// bytes are the A fragments of four m16n8k16 products.  params [ceil(n / 16), k / group, 8, 2]: for rows r and r + 8 of a tile the
// scale as bf16 bits and above them those of 128 + zero.  k % 32 == 0, group 32, 64, 128 or 256 and a divisor of k.
struct W4Args {
  const void* x = nullptr;   // [m, k] bf16, rows ldx elements apart (a multiple of 8), 16-byte aligned
  long long ldx = 0;
  const void* codes = nullptr;
  const void* params = nullptr;
  const float* bias = nullptr;        // [n], may be null
  const void* residual = nullptr;     // [m, n] bf16, rows ldr apart, may be null
  long long ldr = 0;
  void* y = nullptr;                  // [m, n] bf16, contiguous
  int m = 0, n = 0, k = 0, group = 0;
  bool gelu = false;
};
cudaError_t w4_linear(const W4Args& a, cudaStream_t stream);
// Lays out codes [n, k] (one per byte, from an even address on), scales [n, k / group] bf16 and zeros (bytes, may be null: 8); *bad becomes nonzero when one is above 15.
cudaError_t w4_pack(const uint8_t* codes, const void* scales, const uint8_t* zeros, void* packed, void* params, int* bad, int n, int k, int group, cudaStream_t stream);
// w [n, k] bf16 = scale (code - zero), rounded once.
cudaError_t w4_dequantize(const void* codes, const void* params, void* w, int n, int k, int group, cudaStream_t stream);

}  // namespace ops
}  // namespace mccl
