// Writing into a paged key-value cache and copying its pages.  Both are bound by memory: every value is read once and written once,
// 16 bytes per thread and access.
#include "../core/launch.hpp"
#include "half16.cuh"
#include "ops.hpp"
#include "serving.hpp"

namespace mccl {
namespace ops {

namespace {

constexpr int kThreads = 256;

// Four (even, odd) pairs rotated.  Products are rounded before they are added, as the training path's rotation does, so a key in the
// cache has the bits of the key that scoring the whole text would use.
__device__ __forceinline__ void rotate_pairs(float (&f)[8], const float* cos_row, const float* sin_row) {
  const float4 c = __ldg(reinterpret_cast<const float4*>(cos_row)), s = __ldg(reinterpret_cast<const float4*>(sin_row));
  const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = f[2 * i], b = f[2 * i + 1];
    f[2 * i] = __fsub_rn(__fmul_rn(a, cc[i]), __fmul_rn(b, ss[i]));
    f[2 * i + 1] = __fadd_rn(__fmul_rn(a, ss[i]), __fmul_rn(b, cc[i]));
  }
}

// A unit is 8 elements of one head of one token.  A block takes `per_block` consecutive tokens, so that the units of a token are
// counted in 32 bits whatever the number of tokens.
template <typename H>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a, int per_block, int units) {
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const int hd8 = a.head_dim / 8, kv_units = a.kv_heads * hd8;
  const long long first = static_cast<long long>(blockIdx.x) * per_block;
  for (int i = threadIdx.x; i < per_block * units; i += kThreads) {
    const int in_block = i / units, u = i - in_block * units;
    const long long t = first + in_block;
    if (t >= a.tokens) break;
    const int part = u < kv_units ? 0 : (u < 2 * kv_units ? 1 : 2);   // k, v, q
    const int r = u - part * kv_units;
    const int h = r / hd8, d8 = r - h * hd8;
    const TokenView& from = part == 0 ? a.k : (part == 1 ? a.v : a.q);
    uint4 raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const typename H::T*>(from.p) + t * from.token + h * from.head) + d8);
    const int pos = __ldg(a.positions + t), row = a.rows ? __ldg(a.rows + t) : static_cast<int>(t);
    const int ps = a.table.page_size;
    int page = -1;
    if (pos >= 0 && row >= 0 && row < a.table.rows && pos / ps < a.table.width && (a.cos == nullptr || pos < a.rope_rows))
      page = __ldg(a.table.p + row * a.table.stride + pos / ps);
    const bool good = page >= 0 && page < a.table.pages;
    if (a.cos != nullptr && part != 1 && good) {
      float f[8];
      unpack8_as<H>(raw, f);
      const size_t at = (static_cast<size_t>(pos) * hd8 + d8) * 4;
      rotate_pairs(f, a.cos + at, a.sin + at);
      raw = pack8_as<H>(f);
    }
    if (part == 2) {
      if (!good) raw = make_uint4(0, 0, 0, 0);
      reinterpret_cast<uint4*>(static_cast<typename H::T*>(a.q_out) + t * a.heads * a.head_dim)[r] = raw;
    } else if (good) {
      const PagedTensor& to = part == 0 ? a.k_pages : a.v_pages;
      reinterpret_cast<uint4*>(static_cast<typename H::T*>(to.p) + page * to.page + h * to.head + (pos % ps) * to.token)[d8] = raw;
    }
  }
}

// Block (x, y): piece x of the pages, pairs y, y + gridDim.y, ... of outer index and copy.  Four accesses in flight per thread.
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
  const int units = (2 * a.kv_heads + (a.q_out ? a.heads : 0)) * (a.head_dim / 8);
  if (units <= 0) return cudaSuccess;
  int per_block = kThreads / units;
  if (per_block < 1) per_block = 1;
  const long long blocks = (a.tokens + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  if (a.type == Half16::bf16)
    MCCL_LAUNCH_PDL(paged_append_kernel<Bf16>, static_cast<unsigned>(blocks), kThreads, 0, stream, a, per_block, units);
  else
    MCCL_LAUNCH_PDL(paged_append_kernel<Fp16>, static_cast<unsigned>(blocks), kThreads, 0, stream, a, per_block, units);
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
