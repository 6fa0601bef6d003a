// Writing into a paged key-value cache and copying its pages.  Both are bound by memory: every value is read once and written once,
// 16 bytes per thread and access.
#include "../core/launch.hpp"
#include "divisor.cuh"
#include "half16.cuh"
#include "ops.hpp"
#include "serving.hpp"

namespace mccl {
namespace ops {

namespace {

constexpr int kThreads = 256;

// Four (even, odd) pairs rotated.  Products are rounded before they are added, as the training path's rotation does, so a key in the
// cache has the bits of the key that scoring the whole text would use.
__device__ __forceinline__ void rotate_pairs(float (&f)[8], const float4& c, const float4& s) {
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = f[2 * i], b = f[2 * i + 1];
    f[2 * i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
    f[2 * i + 1] = __fadd_rn(__fmul_rn(a, ss[i]), __fmul_rn(b, cc[i]));
  }
}

// A token's heads are k's, v's and, where q is rotated, q's.  A thread has eight elements of a head, the same eight of every `rows`-th head of one token: it
// follows the token's place (position, row, page), takes its part of the rotation and works out addresses once, and its loads are all under way before
// that and the first result.  A block has one token, or as many as it has threads for.  64 tokens of 48 heads of 128: 2.5 us (3.2 with a place per 16 bytes),
// 1537 of them, 38 MB: 9.5 us, of which 2.5 are the launch: 5.4 TB/s.  (Four loads ahead 9.4; loads behind the position's 11.0; blocks that go from token to token and
// look two places ahead 10.8, and 2.9 for the 64.)
template <typename H>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a, int per_block, int rows, int all_heads, Divisor by_heads, Divisor by_hd8) {
  constexpr int kDeep = 3;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const int at_row = by_hd8.of(threadIdx.x), d8 = threadIdx.x - at_row * by_hd8.d;
  const int in_block = per_block > 1 ? by_heads.of(at_row) : 0;
  const long long t = static_cast<long long>(blockIdx.x) * per_block + in_block;
  if (at_row >= rows || in_block >= per_block || t >= a.tokens) return;
  using T = typename H::T;
  const int kv = a.kv_heads;
  const T* k = static_cast<const T*>(a.k.p) + t * a.k.token + d8 * 8;
  const T* v = static_cast<const T*>(a.v.p) + t * a.v.token + d8 * 8;
  const T* q = static_cast<const T*>(a.q.p) + t * a.q.token + d8 * 8;
  int h0 = at_row - in_block * all_heads;
  uint4 raw[kDeep];
  auto load = [&]() {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int h = h0 + i * rows;
      if (h < all_heads) raw[i] = __ldg(reinterpret_cast<const uint4*>(h < kv ? k + h * a.k.head : (h < 2 * kv ? v + (h - kv) * a.v.head : q + (h - 2 * kv) * a.q.head)));
    }
  };
  load();   // before anything is waited for
  const int pos = __ldg(a.positions + t), row = a.rows ? __ldg(a.rows + t) : static_cast<int>(t);
  const int ps = a.table.page_size, slot = pos >= 0 ? pos / ps : 0;
  const bool inside = pos >= 0 && row >= 0 && row < a.table.rows && slot < a.table.width && (a.cos == nullptr || pos < a.rope_rows);
  int page = -1;
  float4 c = make_float4(1.f, 1.f, 1.f, 1.f), s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (inside) {
    page = __ldg(a.table.p + row * a.table.stride + slot);
    if (a.cos != nullptr) {
      const size_t at = (static_cast<size_t>(pos) * by_hd8.d + d8) * 4;
      c = __ldg(reinterpret_cast<const float4*>(a.cos + at));
      s = __ldg(reinterpret_cast<const float4*>(a.sin + at));
    }
  }
  const bool good = page >= 0 && page < a.table.pages;
  const long long place = static_cast<long long>(good ? page : 0), at = good ? pos - slot * ps : 0;
  T* to_k = static_cast<T*>(a.k_pages.p) + place * a.k_pages.page + at * a.k_pages.token + d8 * 8;
  T* to_v = static_cast<T*>(a.v_pages.p) + place * a.v_pages.page + at * a.v_pages.token + d8 * 8;
  T* to_q = static_cast<T*>(a.q_out) + t * a.heads * a.head_dim + d8 * 8;
  while (true) {
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int h = h0 + i * rows;
      if (h >= all_heads) break;
      const bool value = h >= kv && h < 2 * kv;
      if (a.cos != nullptr && !value) {
        float f[8];
        unpack8_as<H>(raw[i], f);
        rotate_pairs(f, c, s);
        raw[i] = pack8_as<H>(f);
      }
      if (h >= 2 * kv)
        *reinterpret_cast<uint4*>(to_q + (h - 2 * kv) * static_cast<long long>(a.head_dim)) = good ? raw[i] : make_uint4(0, 0, 0, 0);
      else if (good)
        *reinterpret_cast<uint4*>(value ? to_v + (h - kv) * a.v_pages.head : to_k + h * a.k_pages.head) = raw[i];
    }
    h0 += kDeep * rows;
    if (h0 >= all_heads) break;
    load();
  }
}

// Block (x, y): piece x of the pages, pairs y, y + gridDim.y, ... of outer index and copy.  Four accesses in flight per thread.  61 pages of 12 layers of 16 heads
// of 128 (384 MB read and written): 115 us, 6.7 TB/s, the rate of a plain copy.
template <typename V>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(char* base, long long outer_stride, long long page_stride, long long words, int pages,
                                                              const int* __restrict__ src, const int* __restrict__ dst, long long count, long long pairs) {
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  constexpr int kDeep = 4;
  for (long long y = blockIdx.y; y < pairs; y += gridDim.y) {
    const long long o = y / count, i = y - o * count;
    const int s = __ldg(src + i), d = __ldg(dst + i);
    if (s < 0 || s >= pages || d < 0 || d >= pages) continue;
    const V* from = reinterpret_cast<const V*>(base + o * outer_stride + s * page_stride);
    V* to = reinterpret_cast<V*>(base + o * outer_stride + d * page_stride);
    for (long long w = static_cast<long long>(blockIdx.x) * (kThreads * kDeep) + threadIdx.x; w < words; w += static_cast<long long>(gridDim.x) * (kThreads * kDeep)) {
      V v[kDeep];
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (w + k * kThreads < words) v[k] = from[w + k * kThreads];
#pragma unroll
      for (int k = 0; k < kDeep; ++k)
        if (w + k * kThreads < words) to[w + k * kThreads] = v[k];
    }
  }
}

template <typename V>
cudaError_t launch_copy(void* base, long long outer, long long outer_stride, long long page_stride, long long page_bytes, int pages, const int* src,
                        const int* dst, long long count, cudaStream_t stream) {
  const long long words = page_bytes / static_cast<long long>(sizeof(V)), pairs = outer * count;
  const long long bx = (words + kThreads * 4 - 1) / (kThreads * 4);
  dim3 grid(static_cast<unsigned>(bx < 1024 ? bx : 1024), static_cast<unsigned>(pairs < 65535 ? pairs : 65535));
  MCCL_LAUNCH_PDL(copy_pages_kernel<V>, grid, kThreads, 0, stream, static_cast<char*>(base), outer_stride, page_stride, words, pages, src, dst, count, pairs);
  count_launch();
  return ::mccl::launch_status();
}

}  // namespace

cudaError_t paged_append(const AppendArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  const int hd8 = a.head_dim / 8, all_heads = 2 * a.kv_heads + (a.q_out ? a.heads : 0);
  if (hd8 <= 0 || all_heads <= 0) return cudaSuccess;
  if (hd8 > kThreads) return cudaErrorNotSupported;
  // Tokens for several rounds of SMs take half as many threads each, whose blocks come and go more evenly (1537 tokens of 48 heads of 128 9.2 us, 9.8 with
  // all; 2048 of 36 heads of 64 5.1 and 7.5); fewer tokens finish sooner with all (64 tokens 2.5 and 3.2 us, 600 4.4 and 4.7).
  const int threads = a.tokens >= 5 * 148 && hd8 <= kThreads / 2 ? kThreads / 2 : kThreads;
  const int rows = threads / hd8, per_block = all_heads < rows ? rows / all_heads : 1;
  const long long blocks = (a.tokens + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (a.type == Half16::bf16)
    MCCL_LAUNCH_PDL(paged_append_kernel<Bf16>, static_cast<unsigned>(blocks), threads, 0, stream, a, per_block, rows, all_heads, Divisor(all_heads), Divisor(hd8));
  else
    MCCL_LAUNCH_PDL(paged_append_kernel<Fp16>, static_cast<unsigned>(blocks), threads, 0, stream, a, per_block, rows, all_heads, Divisor(all_heads), Divisor(hd8));
  count_launch();
  return ::mccl::launch_status();
}

cudaError_t copy_pages(void* base, long long outer, long long outer_stride, long long page_stride, long long page_bytes, int pages, const int* src,
                       const int* dst, long long count, cudaStream_t stream) {
  if (outer <= 0 || count <= 0 || page_bytes <= 0) return cudaSuccess;
  const unsigned long long align = reinterpret_cast<uintptr_t>(base) | outer_stride | page_stride | page_bytes;
  if (align % 16 == 0) return launch_copy<uint4>(base, outer, outer_stride, page_stride, page_bytes, pages, src, dst, count, stream);
  if (align % 4 == 0) return launch_copy<uint32_t>(base, outer, outer_stride, page_stride, page_bytes, pages, src, dst, count, stream);
  return launch_copy<uint8_t>(base, outer, outer_stride, page_stride, page_bytes, pages, src, dst, count, stream);
}

}  // namespace ops
}  // namespace mccl
