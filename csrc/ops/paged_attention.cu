// Attention of one new token per sequence over a paged key-value cache.
//
// The formula, for one sequence and head with query q: o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j over the visible
// positions j and m their maximum.  Sums over any split of the positions join exactly: parts (m, l, o) combine with weights exp(m_part - m).
#include "../core/launch.hpp"
#include "half16.cuh"
#include "ops.hpp"
#include "serving.hpp"

namespace mccl {
namespace ops {

namespace {

constexpr int kWarps = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// One block per sequence and query head, a warp per key: lane l holds elements l, l + 32, ... of the head.
template <typename H>
__global__ void __launch_bounds__(kWarps * 32) paged_attention_kernel(PagedAttentionArgs a) {
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  using T = typename H::T;
  constexpr int kMost = 8;   // elements per lane
  __shared__ float part[kWarps][256];
  __shared__ float part_m[kWarps], part_l[kWarps];
  const int b = blockIdx.x, h = blockIdx.y, kvh = h / (a.heads / a.kv_heads);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long room = static_cast<long long>(a.table.width) * a.table.page_size;
  const int length = static_cast<int>(min(static_cast<long long>(max(a.lengths[b], 0)), room));
  const T* q = static_cast<const T*>(a.q.p) + b * a.q.token + h * a.q.head;
  float qf[kMost], acc[kMost];
  const int mine = (a.head_dim - lane + 31) / 32;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    qf[i] = i < mine ? H::up(q[lane + 32 * i]) * a.scale * kLog2e : 0.f;
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int first = a.window > 0 ? max(length - a.window, 0) : 0;
  for (int j = warp; j < length; j += kWarps) {
    if (j < first && j >= a.sinks) continue;
    const int page = a.table.p[b * a.table.stride + j / a.table.page_size], at = j % a.table.page_size;
    if (page < 0 || page >= a.table.pages) continue;
    const T* k = static_cast<const T*>(a.k_pages.p) + page * a.k_pages.page + kvh * a.k_pages.head + at * a.k_pages.token;
    const T* v = static_cast<const T*>(a.v_pages.p) + page * a.v_pages.page + kvh * a.v_pages.head + at * a.v_pages.token;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine) s += qf[i] * H::up(k[lane + 32 * i]);
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float m_new = fmaxf(m, s);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float keep = exp2f(m - base), p = exp2f(s - base);
    l = l * keep + p;
#pragma unroll
    for (int i = 0; i < kMost; ++i)
      if (i < mine) acc[i] = acc[i] * keep + p * H::up(v[lane + 32 * i]);
    m = m_new;
  }
  if (lane == 0) {
    part_m[warp] = m;
    part_l[warp] = l;
  }
  for (int i = 0; i < kMost; ++i)
    if (i < mine) part[warp][lane + 32 * i] = acc[i];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, part_m[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < kWarps; ++w) sum += part_l[w] * exp2f(part_m[w] - base);
  for (int d = threadIdx.x; d < a.head_dim; d += blockDim.x) {
    float o = 0.f;
    for (int w = 0; w < kWarps; ++w) o += part[w][d] * exp2f(part_m[w] - base);
    static_cast<T*>(a.o)[(static_cast<long long>(b) * a.heads + h) * a.head_dim + d] = H::down(length == 0 ? 0.f : o / sum);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[static_cast<long long>(b) * a.heads + h] = length == 0 ? -INFINITY : (base + log2f(sum)) * kLn2;
}

}  // namespace

size_t paged_attention_workspace(const PagedAttentionArgs&) { return 0; }

cudaError_t paged_attention(const PagedAttentionArgs& a, cudaStream_t stream) {
  if (a.batch <= 0 || a.heads <= 0) return cudaSuccess;
  dim3 grid(static_cast<unsigned>(a.batch), static_cast<unsigned>(a.heads));
  if (a.type == Half16::bf16)
    MCCL_LAUNCH_PDL(paged_attention_kernel<Bf16>, grid, kWarps * 32, 0, stream, a);
  else
    MCCL_LAUNCH_PDL(paged_attention_kernel<Fp16>, grid, kWarps * 32, 0, stream, a);
  count_launch();
  return ::mccl::launch_status();
}

}  // namespace ops
}  // namespace mccl
