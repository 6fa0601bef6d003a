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

// A unit is 8 elements of one head of one token: the token's units are k's, v's and, where q is rotated, q's.  A block has one token of many units, or as many
// tokens as it has threads for, so a thread has one token and follows its place (position, row, page) once; its loads are all under way before the first
// result.  1537 tokens of 48 heads of 128, 38 MB: 12.4 us with a unit at a time, 11.0 us so (5.8 at the rate of a copy).
template <typename H>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a, int per_block, Divisor units, Divisor kv_units, Divisor hd8) {
  constexpr int kDeep = 4;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const int in_block = units.of(threadIdx.x);   // zero where a token's units are more than the threads
  const long long t = static_cast<long long>(blockIdx.x) * per_block + in_block;
  if (in_block >= per_block || t >= a.tokens) return;
  using V = uint4;
  auto source = [&](int u) -> const V* {
    const int part = kv_units.of(u), r = u - (part > 2 ? 2 : part) * kv_units.d, h = hd8.of(r);
    const TokenView& from = part == 0 ? a.k : (part == 1 ? a.v : a.q);
    return reinterpret_cast<const V*>(static_cast<const typename H::T*>(from.p) + t * from.token + h * from.head) + (r - h * hd8.d);
  };
  const int pos = __ldg(a.positions + t), row = a.rows ? __ldg(a.rows + t) : static_cast<int>(t);
  const int ps = a.table.page_size, slot = pos >= 0 ? pos / ps : 0;
  const bool inside = pos >= 0 && row >= 0 && row < a.table.rows && slot < a.table.width && (a.cos == nullptr || pos < a.rope_rows);
  int page = -1;
  if (inside) page = __ldg(a.table.p + row * a.table.stride + slot);
  const bool good = page >= 0 && page < a.table.pages;
  for (int u0 = threadIdx.x - in_block * units.d; u0 < static_cast<int>(units.d); u0 += kThreads * kDeep) {
    V raw[kDeep];
#pragma unroll
    for (int i = 0; i < kDeep; ++i)
      if (u0 + i * kThreads < static_cast<int>(units.d)) raw[i] = __ldg(source(u0 + i * kThreads));
#pragma unroll
    for (int i = 0; i < kDeep; ++i) {
      const int u = u0 + i * kThreads;
      if (u >= static_cast<int>(units.d)) break;
      const int part = min(static_cast<int>(kv_units.of(u)), 2), r = u - part * kv_units.d, h = hd8.of(r), d8 = r - h * hd8.d;
      if (a.cos != nullptr && part != 1 && good) {
        float f[8];
        unpack8_as<H>(raw[i], f);
        const size_t at = (static_cast<size_t>(pos) * hd8.d + d8) * 4;
        rotate_pairs(f, a.cos + at, a.sin + at);
        raw[i] = pack8_as<H>(f);
      }
      if (part == 2) {
        if (!good) raw[i] = make_uint4(0, 0, 0, 0);
        reinterpret_cast<V*>(static_cast<typename H::T*>(a.q_out) + t * a.heads * a.head_dim)[r] = raw[i];
      } else if (good) {
        const PagedTensor& to = part == 0 ? a.k_pages : a.v_pages;
        reinterpret_cast<V*>(static_cast<typename H::T*>(to.p) + page * to.page + h * to.head + (pos - slot * ps) * to.token)[d8] = raw[i];
      }
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
  const int per_block = units < kThreads ? kThreads / units : 1;
  const long long blocks = (a.tokens + per_block - 1) / per_block;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidValue;
  const Divisor by_units(units), by_kv(a.kv_heads * (a.head_dim / 8)), by_hd8(a.head_dim / 8);
  if (a.type == Half16::bf16)
    MCCL_LAUNCH_PDL(paged_append_kernel<Bf16>, static_cast<unsigned>(blocks), kThreads, 0, stream, a, per_block, by_units, by_kv, by_hd8);
  else
    MCCL_LAUNCH_PDL(paged_append_kernel<Fp16>, static_cast<unsigned>(blocks), kThreads, 0, stream, a, per_block, by_units, by_kv, by_hd8);
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
