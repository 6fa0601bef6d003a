// Products of few rows with 4-bit weights.
//
// y = x W^T with W[n, k] = scale[n, k / g] (code - zero): a group's sum is scale * sum x (code - zero), so the codes go into the product as
// whole numbers and the scale is applied once per group to a sum in fp32.  Nothing but x and y is rounded to 16 bits.
// The weights are read once, 0.5 bytes each, and bound the time.  They are the A operand of m16n8k16 products (16 weight rows, 8 rows of x
// as columns): the tensor cores of this generation's own instruction take 64 to 256 rows of x at a time and operands in shared or tensor
// memory, which single tokens do not fill, while here a code goes from its load through one mask and one subtraction into the product.
#include "../core/launch.hpp"
#include "bf16x8.cuh"
#include "ops.hpp"
#include "serving.hpp"

namespace mccl {
namespace ops {

namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Two codes (bits 0-3 and 16-19 of w >> 4 j) as bf16 pair code - zero: 0x4300 is 128, whose last mantissa bit is worth one.
__device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t zero2) { return sub2((w & 0x000f000fu) | 0x43004300u, zero2); }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// A block has kR tiles of 16 weight rows and kN tiles of 8 rows of x; its warps share out K in chunks of 64 and add up at the end.
template <int kR, int kN, bool kG32>
__global__ void __launch_bounds__(kWarps * 32) w4_linear_kernel(W4Args a) {
  extern __shared__ float sums[];   // [warp][token][weight row]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_tiles = (a.n + 15) / 16, chunks = (a.k + 63) / 64, groups = a.k / a.group;
  const int tile0 = blockIdx.x * kR, token0 = blockIdx.y * (8 * kN);
  const uint4* codes = static_cast<const uint4*>(a.codes);
  const uint2* params = static_cast<const uint2*>(a.params);
  const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(a.x);
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  float total[kR][kN][4] = {};
  for (int c = warp; c < chunks; c += kWarps) {
    uint4 w[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r)
      w[r] = tile0 + r < row_tiles ? __ldg(codes + (static_cast<size_t>(tile0 + r) * chunks + c) * 32 + lane) : make_uint4(0, 0, 0, 0);
    uint4 xv[kN][2];
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int token = token0 + n * 8 + g, k = c * 64 + h * 32 + t * 8;
        xv[n][h] = token < a.m && k < a.k ? __ldg(reinterpret_cast<const uint4*>(x + token * a.ldx + k)) : make_uint4(0, 0, 0, 0);
      }
    constexpr int kParts = kG32 ? 2 : 1;   // groups that a chunk touches
    uint2 prm[kR][kParts];
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const int group = min((c * 64 + h * 32) / a.group, groups - 1);
        prm[r][h] = tile0 + r < row_tiles ? __ldg(params + (static_cast<size_t>(tile0 + r) * groups + group) * 8 + g) : make_uint2(0, 0);
      }
#pragma unroll
    for (int r = 0; r < kR; ++r) {
      float acc[kN][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint2 p = prm[r][kG32 ? h : 0];
        const uint32_t z0 = __byte_perm(p.x, 0, 0x3232), z8 = __byte_perm(p.y, 0, 0x3232);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const uint32_t word = h == 0 ? (s == 0 ? w[r].x : w[r].y) : (s == 0 ? w[r].z : w[r].w);
          const uint32_t a0 = codes2(word, z0), a1 = codes2(word >> 4, z8), a2 = codes2(word >> 8, z0), a3 = codes2(word >> 12, z8);
#pragma unroll
          for (int n = 0; n < kN; ++n) mma16816(acc[n], a0, a1, a2, a3, s == 0 ? xv[n][h].x : xv[n][h].z, s == 0 ? xv[n][h].y : xv[n][h].w);
        }
        if (kG32 || h == 1) {
          const float s0 = __uint_as_float(p.x << 16), s8 = __uint_as_float(p.y << 16);
#pragma unroll
          for (int n = 0; n < kN; ++n) {
            total[r][n][0] += s0 * acc[n][0];
            total[r][n][1] += s0 * acc[n][1];
            total[r][n][2] += s8 * acc[n][2];
            total[r][n][3] += s8 * acc[n][3];
            acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
          }
        }
      }
    }
  }
  constexpr int kRows = kR * 16, kTokens = kN * 8;
#pragma unroll
  for (int r = 0; r < kR; ++r)
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[(warp * kTokens + n * 8 + 2 * t + (i & 1)) * kRows + r * 16 + g + (i >> 1) * 8] = total[r][n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kTokens; i += kWarps * 32) {
    const int n = tile0 * 16 + i % kRows, m = token0 + i / kRows;
    if (n >= a.n || m >= a.m) continue;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += sums[w * (kRows * kTokens) + i];
    if (a.bias) v += a.bias[n];
    if (a.gelu) v = 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    if (a.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.residual)[m * a.ldr + n]);
    static_cast<__nv_bfloat16*>(a.y)[static_cast<long long>(m) * a.n + n] = __float2bfloat16_rn(v);
  }
}

template <int kR, int kN>
cudaError_t launch(const W4Args& a, cudaStream_t stream) {
  const int smem = kWarps * kR * 16 * kN * 8 * static_cast<int>(sizeof(float));
  const dim3 grid((a.n + 16 * kR - 1) / (16 * kR), (a.m + 8 * kN - 1) / (8 * kN));
  if (a.group == 32) {
    static const cudaError_t rc = cudaFuncSetAttribute(w4_linear_kernel<kR, kN, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    MCCL_LAUNCH_PDL((w4_linear_kernel<kR, kN, true>), grid, kWarps * 32, smem, stream, a);
  } else {
    static const cudaError_t rc = cudaFuncSetAttribute(w4_linear_kernel<kR, kN, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (rc != cudaSuccess) return rc;
    MCCL_LAUNCH_PDL((w4_linear_kernel<kR, kN, false>), grid, kWarps * 32, smem, stream, a);
  }
  count_launch();
  return ::mccl::launch_status();
}

// A warp per tile of 16 x 64: lane (g, t) writes 8 neighbouring values of rows g and g + 8, in both halves.
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint4* __restrict__ codes, const uint2* __restrict__ params, __nv_bfloat16* __restrict__ w,
                                                            int n, int k, int group) {
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = (k + 63) / 64, groups = k / group;
  const long long tiles = static_cast<long long>((n + 15) / 16) * chunks;
  for (long long i = blockIdx.x * 8ll + (threadIdx.x >> 5); i < tiles; i += gridDim.x * 8ll) {
    const int tile = static_cast<int>(i / chunks), c = static_cast<int>(i - static_cast<long long>(tile) * chunks);
    const uint4 raw = __ldg(codes + i * 32 + lane);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = c * 64 + h * 32 + t * 8;
      if (at >= k) continue;
      const uint2 p = __ldg(params + (static_cast<size_t>(tile) * groups + at / group) * 8 + g);
      const uint32_t lo = h == 0 ? raw.x : raw.z, hi = h == 0 ? raw.y : raw.w;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = tile * 16 + r * 8 + g;
        if (row >= n) continue;
        const uint32_t prm = r == 0 ? p.x : p.y, z = __byte_perm(prm, 0, 0x3232);
        const float s = __uint_as_float(prm << 16);
        const uint32_t v[4] = {codes2(lo >> (4 * r), z), codes2(lo >> (8 + 4 * r), z), codes2(hi >> (4 * r), z), codes2(hi >> (8 + 4 * r), z)};
        float f[8];
        unpack8(make_uint4(v[0], v[1], v[2], v[3]), f);
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] *= s;
        *reinterpret_cast<uint4*>(w + static_cast<size_t>(row) * k + at) = pack8(f);
      }
    }
  }
}

}  // namespace

cudaError_t w4_linear(const W4Args& a, cudaStream_t stream) {
  if (a.m <= 0 || a.n <= 0) return cudaSuccess;
  if (a.m <= 8) return launch<2, 1>(a, stream);
  if (a.m <= 16) return launch<2, 2>(a, stream);
  return launch<2, 4>(a, stream);
}

cudaError_t w4_dequantize(const void* codes, const void* params, void* w, int n, int k, int group, cudaStream_t stream) {
  if (n <= 0 || k <= 0) return cudaSuccess;
  const long long tiles = static_cast<long long>((n + 15) / 16) * ((k + 63) / 64), blocks = (tiles + 7) / 8;
  MCCL_LAUNCH_PDL(w4_dequantize_kernel, static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, stream, static_cast<const uint4*>(codes),
                  static_cast<const uint2*>(params), static_cast<__nv_bfloat16*>(w), n, k, group);
  count_launch();
  return ::mccl::launch_status();
}

}  // namespace ops
}  // namespace mccl
