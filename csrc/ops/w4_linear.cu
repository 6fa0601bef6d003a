// Products with 4-bit weights: y = x W^T, W[n, k] = scale[n, k / g] (code - zero).
//
// Three kernels.  For up to 16 rows of x that fit shared memory the weights are read once, half a byte each: the narrow kernel multiplies codes as whole
// numbers (bf16 holds -15 to 15 exactly) and applies a group's scale to its sum in fp32, scale * sum x (code - zero), so nothing but x and y is rounded to
// 16 bits.  Neither memory (28 % of its rate under the profiler) nor issue (53 % of the slots, 49 % of the ALU pipe: some 190 instructions per KB, most of
// them to take codes apart) is full: four warps per scheduler wait for their own chains as much as for slots.  For more rows bf16 weights, scale * (code - zero) rounded once, are
// made on the way into tensor memory, where they are the left operand of tcgen05 products: a block per tile and part of K where that fills the SMs (the wide
// kernel), a block per SM that runs on from tile to tile where there are several for each (the stream kernel).  For 16384 x 2048 the
// narrow kernel takes 7.4 us for 8 rows and 10.3 for 16, the wide one 9.6 for up to 32: where they meet the narrow one stays, which rounds no weights.
// Measured (codes from memory): 4 x 32000 x 2048, 36 MB: 12.7 us, 2.8 TB/s; 1 x 16384 x 2048: 6.5 us; 1 x 2048 x 2048: 2.6 us, a launch and one chain of loads;
// 48 x 3072 x 768: 5.0 us; 128 x 16384 x 2048: 11.3 us, 0.76 PFLOP/s; 256: 16.0 us; 1537: 95 us, 1.09 PFLOP/s, among calls that go on for seconds (80 us, 1.29
// PFLOP/s, in a burst, before the power limit lowers the clock).
#include <cuda.h>

#include <array>
#include <limits>

#include "../core/launch.hpp"
#include "bf16x8.cuh"
#include "gemm_common.cuh"
#include "ops.hpp"
#include "serving.hpp"
#include "smem_limit.hpp"
#include "tcgen05.cuh"

namespace mccl {
namespace ops {

namespace {

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// Two codes (bits 0-3 and 16-19) as a bf16 pair code - zero, from 128 + zero: 0x4300 is 128, whose last mantissa bit is worth one.  Both steps are written
// out, one instruction each: the mask and the exponent in one three-input operation, the difference (exact) as a product with minus one and a sum, on the
// pipe that does no logic.
__device__ __forceinline__ uint32_t codes2(uint32_t w, uint32_t zero2) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(0x000f000fu), "r"(0x43004300u));
  asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(r) : "r"(zero2), "r"(0xbf80bf80u));
  return r;
}
// Of a row's parameters (scale, and above it 128 + zero) the scale, and either of them twice.
__device__ __forceinline__ float scale_of(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ uint32_t scale2(uint32_t p) { return __byte_perm(p, 0, 0x1010); }
__device__ __forceinline__ uint32_t zero2(uint32_t p) { return __byte_perm(p, 0, 0x3232); }

template <int kBytes>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from, bool real = true) {
  if (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(kBytes), "r"(real ? kBytes : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void load_matrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first product of a sum.
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float finished(const W4Args& a, float v, int m, int n) {
  if (a.bias) v += __ldg(a.bias + n);
  if (a.gelu) v = 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
  if (a.residual) v += __bfloat162float(static_cast<const __nv_bfloat16*>(a.residual)[m * a.ldr + n]);
  return v;
}

// ----------------------------------------------------------- up to 16 rows of x --
constexpr int kNarrowWarps = 8, kNarrowThreads = kNarrowWarps * 32;
template <int kR>
constexpr int kDeep = kR == 2 ? 3 : 4;   // stages of 128 columns that a warp has on their way
template <int kR, int kParams>
constexpr int kNarrowSlot = kR * (1024 + kParams * 256);
template <int kR, int kN>
constexpr int kNarrowSums = 2 * kNarrowWarps * kR * kN * 128 * 4;
constexpr int kNarrowX = 128 * 1024;   // most bytes of x: m rows of 256 per 128 columns
template <int kR, int kN, int kParams>
constexpr int narrow_smem(int x_bytes) { return kNarrowWarps * kDeep<kR> * kNarrowSlot<kR, kParams> + kNarrowSums<kR, kN> + x_bytes + 16; }
constexpr int kSmemLimit = 227 * 1024;
static_assert(narrow_smem<1, 1, 4>(kNarrowX) <= kSmemLimit && narrow_smem<1, 2, 4>(kNarrowX) <= kSmemLimit);   // one tile per warp always fits

// A warp takes kR tiles of 16 weight rows at a time, a block 8 / along times as many, gridDim.x such groups apart; `along` warps share out K for each, a
// run of stages of 128 columns, and add up at its end.  A lane's 16 bytes of 64 columns are its own A fragments of four m16n8k16 products: it copies them
// ahead into its own place and waits for nobody, and so it does with its two rows' parameters (kParams groups in a stage).  x lies in shared memory, 128
// bytes of every row per 64 columns, in the order of the 128-byte swizzle; kN is how many times 8 rows it has.
// Two blocks of 8 warps per SM: one of 16 warps took 14.2 us for 4 x 32000 x 2048 and 6.1 for a small product, whose next launch then finds no room.
// kEven: no tile and no half stage is missing at the end of N or K.
template <int kR, int kN, int kParams, bool kEven>
__global__ void __launch_bounds__(kNarrowThreads, 2) w4_narrow_kernel(W4Args a, int tiles, int chunks, int group_shift, int along_shift) {
  extern __shared__ __align__(128) unsigned char smem[];
  constexpr int kSlot = kNarrowSlot<kR, kParams>, kTile = 1024 + kParams * 256, kDeep = ops::kDeep<kR>, kOut = kR * kN * 128;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = tc::smem_u32(smem) + warp * (kDeep * kSlot);
  float* sums = reinterpret_cast<float*>(smem + kNarrowWarps * kDeep * kSlot);   // [2][warp][row of x][weight row]
  const int pairs = (chunks + 1) / 2;
  const uint32_t xs = tc::smem_u32(smem) + kNarrowWarps * kDeep * kSlot + kNarrowSums<kR, kN>, nothing = xs + a.m * pairs * 256;
  const int along = 1 << along_shift, at_once = kR * (kNarrowWarps >> along_shift), part = warp & (along - 1);
  const int c0 = pairs * part >> along_shift, slice = (pairs * (part + 1) >> along_shift) - c0;
  const int groups = a.k >> group_shift, tile0 = blockIdx.x * at_once + (warp >> along_shift) * kR, step = gridDim.x * at_once;   // this warp's tiles
  const int rounds = (tiles - static_cast<int>(blockIdx.x) * at_once + step - 1) / step, mine = tile0 < tiles ? (tiles - tile0 + step - 1) / step : 0;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  for (int i = threadIdx.x; i < a.m * pairs * 16; i += kNarrowThreads) {
    const int row = i / (pairs * 16), piece = i - row * (pairs * 16);
    const bool real = piece * 8 < a.k;
    copy_async<16>(xs + (piece >> 3) * (a.m * 128) + row * 128 + (((piece ^ row) & 7) << 4), static_cast<const __nv_bfloat16*>(a.x) + (real ? row * a.ldx + piece * 8 : 0), real);
  }
  if (threadIdx.x == 0) *reinterpret_cast<uint4*>(smem + (nothing - tc::smem_u32(smem))) = make_uint4(0, 0, 0, 0);   // rows of x that there are not
  copy_commit();

  // ---- the loading side
  int to_load = slice * mine, at = c0, load_tile = tile0;
  const size_t tile_codes = static_cast<size_t>(chunks) * 32;
  const uint4* codes = static_cast<const uint4*>(a.codes) + (static_cast<size_t>(tile0) * chunks + 2 * c0) * 32 + lane;
  const uint2* params = static_cast<const uint2*>(a.params) + static_cast<size_t>(tile0) * groups * 8 + g;
  const size_t codes_on = (static_cast<size_t>(step) * chunks - 2 * slice) * 32, params_on = static_cast<size_t>(step) * groups * 8;
  auto issue = [&](int slot) {
    if (to_load > 0) {
      const bool second = kEven || 2 * at + 1 < chunks;
      const uint32_t to = ring + slot * kSlot;
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        const bool there = kEven || r == 0 || load_tile + r < tiles;
        const uint4* from = there ? codes + r * tile_codes : codes;
        copy_async<16>(to + r * kTile + lane * 16, from, there);
        copy_async<16>(to + r * kTile + 512 + lane * 16, second ? from + 32 : from, second && there);
        const uint2* with = params + (there ? r * groups * 8 : 0);
#pragma unroll
        for (int i = 0; i < kParams; ++i) {
          const int group = kParams == 1 ? at >> (group_shift - 7) : (kEven ? kParams * at + i : min(kParams * at + i, groups - 1));
          copy_async<8>(to + r * kTile + 1024 + i * 256 + lane * 8, with + group * 8, there);
        }
      }
      --to_load;
      codes += 64;
      if (++at == c0 + slice) {
        at = c0;
        load_tile += step;
        codes += codes_on;
        params += params_on;
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int i = 0; i < kDeep - 1; ++i) issue(i);
  copy_wait<kDeep - 1>();   // x
  __syncthreads();

  const int row = lane & 7;
  uint32_t x_lane[kN], x_step[kN], x_half[kN];   // pieces 0 to 3 of the first chunk; 4 to 7 are 64 bytes on, the next chunk x_step
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    const bool real = n * 8 + row < a.m;
    x_step[n] = real ? a.m * 128 : 0;
    x_half[n] = real ? 64 : 0;
    x_lane[n] = real ? xs + c0 * (a.m * 256) + (n * 8 + row) * 128 + (((lane >> 3) ^ row) << 4) : nothing;
  }
  int slot = 0;
  for (int i = 0; i < rounds; ++i) {
    float total[kR][kN][4] = {};
    uint32_t x_at[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) x_at[n] = x_lane[n];
    for (int c = i < mine ? slice : 0; c > 0; --c) {
      copy_wait<kDeep - 2>();
      const uint32_t from = ring + slot * kSlot;
      uint4 w[kR][2];
      uint2 p[kR][kParams];
#pragma unroll
      for (int r = 0; r < kR; ++r) {
        w[r][0] = shared16(from + r * kTile + lane * 16);
        w[r][1] = shared16(from + r * kTile + 512 + lane * 16);
#pragma unroll
        for (int j = 0; j < kParams; ++j) p[r][j] = shared8(from + r * kTile + 1024 + j * 256 + lane * 8);
      }
      issue(slot == 0 ? kDeep - 1 : slot - 1);
      slot = slot == kDeep - 1 ? 0 : slot + 1;
      float acc[kR][2][kN][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t b[kN][2][4];
#pragma unroll
        for (int n = 0; n < kN; ++n) {
          load_matrix(b[n][0], x_at[n]);
          load_matrix(b[n][1], x_at[n] ^ x_half[n]);
          x_at[n] += x_step[n];
        }
#pragma unroll
        for (int r = 0; r < kR; ++r) {
          const uint32_t word[4] = {w[r][j].x, w[r][j].y, w[r][j].z, w[r][j].w};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint2 q = p[r][kParams == 4 ? 2 * j + (s >> 1) : (kParams == 2 ? j : 0)];
            const uint32_t z0 = zero2(q.x), z8 = zero2(q.y);
            const uint32_t a0 = codes2(word[s], z0), a1 = codes2(word[s] >> 4, z8), a2 = codes2(word[s] >> 8, z0), a3 = codes2(word[s] >> 12, z8);
            const bool begins = kParams == 4 ? (s & 1) == 0 : s == 0, ends = kParams == 4 ? (s & 1) == 1 : s == 3;
#pragma unroll
            for (int n = 0; n < kN; ++n) {
              float (&c)[4] = acc[r][j][n];
              if (begins) {
                mma16816_first(c, a0, a1, a2, a3, b[n][s >> 1][(s & 1) * 2], b[n][s >> 1][(s & 1) * 2 + 1]);
              } else {
                mma16816(c, a0, a1, a2, a3, b[n][s >> 1][(s & 1) * 2], b[n][s >> 1][(s & 1) * 2 + 1]);
              }
              if (ends && (kParams > 1 || j == 1)) {
                if (kParams == 1) {
#pragma unroll
                  for (int e = 0; e < 4; ++e) c[e] += acc[r][0][n][e];
                }
                const float s0 = scale_of(q.x), s8 = scale_of(q.y);
                total[r][n][0] += s0 * c[0];
                total[r][n][1] += s0 * c[1];
                total[r][n][2] += s8 * c[2];
                total[r][n][3] += s8 * c[3];
              }
            }
          }
        }
      }
    }
    float* to = sums + ((i & 1) * kNarrowWarps + warp) * kOut;
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[(n * 8 + 2 * t + (e & 1)) * (16 * kR) + r * 16 + g + 8 * (e >> 1)] = total[r][n][e];
    __syncthreads();
    for (int o = threadIdx.x; o < (kNarrowWarps >> along_shift) * kOut; o += kNarrowThreads) {
      const int which = o / kOut, out = o % kOut, m = out / (16 * kR), n = (static_cast<int>(blockIdx.x) * at_once + i * step + which * kR) * 16 + out % (16 * kR);
      if (m < a.m && n < a.n) {
        float v = 0.f;
        for (int w = 0; w < along; ++w) v += sums[((i & 1) * kNarrowWarps + which * along + w) * kOut + out];
        static_cast<__nv_bfloat16*>(a.y)[static_cast<long long>(m) * a.n + n] = __float2bfloat16_rn(finished(a, v, m, n));
      }
    }
  }
  copy_wait<0>();
}

// --------------------------------------------------------------- more rows of x --
constexpr int kWideRows = 128;             // weight rows of a block: the lanes of tensor memory
// Warp 0 brings x, warp 1 issues the products, sixteen make weights and write results.  Four warps share a chunk (32 weight rows each) and take
// chunks in turn with three other fours: a warp's part is mostly latency (copy, shared memory, arithmetic, tensor memory, barrier), and four under way hide it.
constexpr int kTurns = 4;
constexpr int kWideThreads = (2 + 4 * kTurns) * 32;
constexpr int kWideStages = 4;
// A weight-making warp copies the codes and parameters of its two tiles ahead, each lane its own: so many chunks are on their way (3 KB or 4 KB each, 96 KB of all).
template <bool kG32>
constexpr int kCodeTile = 512 + (kG32 ? 512 : 256);
template <bool kG32>
constexpr int kCodeDeep = kG32 ? 3 : 4;
constexpr int kCodeRing = 4 * kTurns * 2 * kCodeDeep<false> * kCodeTile<false>;
static_assert(kCodeRing == 4 * kTurns * 2 * kCodeDeep<true> * kCodeTile<true>);
constexpr int kWideSmem = 226 * 1024;      // the rest is for the barriers
constexpr int kMostTokens = 256;           // rows of x of a block
constexpr int kMostRows = 0x7fffffff - kMostTokens;   // of x: a tile's last row is counted in 32 bits

struct Wide {
  W4Args a;
  int tokens = 0, chunks, group_shift;   // rows of x per block, a multiple of 16; chunks of 64 columns in K
  int columns;          // of tensor memory that the sums take; the weights' ring lies behind them
  int allocated;
  int splits, share;    // blocks of a cluster that share out K, and rows of x whose sums each of them finishes
  int vector, rows8;    // y and residual can be accessed four elements at a time, y eight
  int tiles, row_tiles; // of the stream: tiles of weight rows and rows of x, and how many of the latter
  uint32_t idesc;
  int* err;
};

// Bounded wait that leaves the issue slots to others: a poll may sleep for two microseconds, or until the phase ends (a third of the stream kernel's instructions were
// polls without that).  Some two seconds in all.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity) {
  const uint32_t at = tc::smem_u32(bar);
  for (int i = 0; i < (1 << 20); ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(at), "r"(parity), "r"(2000)
        : "memory");
    if (done) return true;
  }
  return false;
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_cols, uint64_t desc_b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a_cols), "l"(desc_b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
// 16 lanes x 64 bf16: register 2 i + r of lane 4 g + t is elements 8 i + 2 t and + 1 of row g + 8 r.
__device__ __forceinline__ void tmem_st_16x64(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_32x16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(at)
               : "memory");
}
// A store to the same place of shared memory in block `rank` of the cluster.
__device__ __forceinline__ void store_peer(uint32_t at, int rank, float v) {
  uint32_t there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(v) : "memory");
}

// Where a lane's codes and parameters of a chunk of a tile are.  The next chunk of the same warp is kTurns, 256 columns, on: a step that is the same for all.
struct Ahead {
  const uint4* codes;
  const uint2* params;
  uint32_t size;   // 16, or 0 for a tile that there is not: zeros
};
__device__ __forceinline__ void copy_sized16(uint32_t to, const void* from, uint32_t size) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
__device__ __forceinline__ void copy_sized8(uint32_t to, const void* from, uint32_t size) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(size) : "memory");
}
template <bool kG32>
__device__ __forceinline__ Ahead ahead_of(const W4Args& a, int chunks, int groups, int group_shift, int tile, int tiles, int c, int lane) {
  Ahead at;
  const bool there = tile < tiles;
  at.codes = static_cast<const uint4*>(a.codes) + (static_cast<size_t>(there ? tile : 0) * chunks + c) * 32 + lane;
  at.params = static_cast<const uint2*>(a.params) + (static_cast<size_t>(there ? tile : 0) * groups + (kG32 ? 2 * c : c * 64 >> group_shift)) * 8 + (lane >> 2);
  at.size = there ? 16 : 0;
  return at;
}
// A chunk's to `to` and 512 bytes on; `both`: with groups of 32, whether there is a second one.
template <bool kG32>
__device__ __forceinline__ void copy_tile(uint32_t to, int lane, Ahead& at, int params_step, bool both) {
  copy_sized16(to + lane * 16, at.codes, at.size);
  if (kG32) {
    copy_sized8(to + 512 + lane * 16, at.params, at.size >> 1);
    copy_sized8(to + 520 + lane * 16, at.params + (both ? 8 : 0), both ? at.size >> 1 : 0);
  } else {
    copy_sized8(to + 512 + lane * 8, at.params, at.size >> 1);
  }
  at.codes += kTurns * 32;
  at.params += params_step;
}
template <bool kG32>
__device__ __forceinline__ void take_tile(uint32_t from, int lane, uint4& codes, uint2 (&params)[2]) {
  codes = shared16(from + lane * 16);
  if (kG32) {
    const uint4 both = shared16(from + 512 + lane * 16);
    params[0] = make_uint2(both.x, both.y);
    params[1] = make_uint2(both.z, both.w);
  } else {
    params[0] = shared8(from + 512 + lane * 8);
  }
}
// A lane's part of 16 x 64 weights for tmem_st_16x64, rounded to bf16 once: scale times whole number.
template <bool kG32>
__device__ __forceinline__ void make_weights(uint32_t (&r)[16], const uint4& w, const uint2 (&prm)[2]) {
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int step = 0; step < 4; ++step) {
    const uint2 q = prm[kG32 ? step >> 1 : 0];
    r[4 * step] = mul2(codes2(word[step], zero2(q.x)), scale2(q.x));
    r[4 * step + 1] = mul2(codes2(word[step] >> 4, zero2(q.y)), scale2(q.y));
    r[4 * step + 2] = mul2(codes2(word[step] >> 8, zero2(q.x)), scale2(q.x));
    r[4 * step + 3] = mul2(codes2(word[step] >> 12, zero2(q.y)), scale2(q.y));
  }
}
__device__ __forceinline__ void load_bias(float (&bias)[4], const W4Args& a, int n4) {
#pragma unroll
  for (int e = 0; e < 4; ++e) bias[e] = a.bias && n4 + e < a.n ? __ldg(a.bias + n4 + e) : 0.f;
}
// Four neighbouring results of a row; `vector`: y and residual can be accessed four elements at a time.
__device__ __forceinline__ void finish4(const W4Args& a, const float4& v, const float (&bias)[4], int m, int n4, int vector) {
  float f[4] = {v.x + bias[0], v.y + bias[1], v.z + bias[2], v.w + bias[3]};
  if (a.gelu) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = 0.5f * f[e] * (1.f + erff(f[e] * 0.70710678118654752f));
  }
  __nv_bfloat16* y = static_cast<__nv_bfloat16*>(a.y) + static_cast<long long>(m) * a.n + n4;
  const __nv_bfloat16* residual = static_cast<const __nv_bfloat16*>(a.residual) + (a.residual ? m * a.ldr + n4 : 0);
  if (vector && n4 + 3 < a.n) {
    if (a.residual) {
      const uint2 raw = __ldg(reinterpret_cast<const uint2*>(residual));
      const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x)), hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
      f[0] += lo.x, f[1] += lo.y, f[2] += hi.x, f[3] += hi.y;
    }
    __nv_bfloat162 out[2] = {__floats2bfloat162_rn(f[0], f[1]), __floats2bfloat162_rn(f[2], f[3])};
    *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(out);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n4 + e < a.n) y[e] = __float2bfloat16_rn(f[e] + (a.residual ? __bfloat162float(residual[e]) : 0.f));
  }
}

// Whether any of the 128 threads at a barrier says so.
__device__ __forceinline__ bool any_of_128(int barrier, bool mine) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(any) : "r"(mine ? 1u : 0u), "r"(barrier) : "memory");
  return any != 0;
}

// Sums of 128 weight rows and 16 rows of x, from tensor memory to y, by four warps: a lane has a weight row, and through shared memory (`to`, [row of x][weight
// row]) a row of y leaves in one piece.  rows8: rows of y are made of eights.  Branches stand around all sixteen values: around each of them they cost 1100 clocks.
constexpr int kStaged = 16 * kWideRows * 2;
__device__ __forceinline__ void finish16(const W4Args& a, int rows8, uint32_t sums, __nv_bfloat16* to, int barrier, int m0, int n0, int quarter, int lane, float bias) {
  uint32_t r[16];
  tmem_ld_32x16(sums, r);
  tc::tmem_ld_wait();
  float v[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = __uint_as_float(r[e]) + bias;
  if (a.gelu) {
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = 0.5f * v[e] * (1.f + erff(v[e] * 0.70710678118654752f));
  }
  const int n = n0 + quarter * 32 + lane;
  if (a.residual && n < a.n) {
    const __nv_bfloat16* residual = static_cast<const __nv_bfloat16*>(a.residual) + n;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] += __bfloat162float(residual[min(m0 + e, a.m - 1) * a.ldr]);
  }
#pragma unroll
  for (int e = 0; e < 16; ++e) to[e * kWideRows + quarter * 32 + lane] = __float2bfloat16_rn(v[e]);
  asm volatile("bar.sync %0, 128;" ::"r"(barrier) : "memory");
#pragma unroll
  for (int e = 0; e < 2; ++e) {   // 8 rows at a time, 8 elements per thread
    const int row = e * 8 + quarter * 2 + (lane >> 4), m = m0 + row, n8 = n0 + (lane & 15) * 8;
    if (m < a.m && n8 < a.n) {
      const __nv_bfloat16* from = to + row * kWideRows + (lane & 15) * 8;
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.y) + static_cast<long long>(m) * a.n + n8;
      if (rows8) {
        *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(from);
      } else {
        for (int k = 0; k < min(8, a.n - n8); ++k) out[k] = from[k];
      }
    }
  }
}

// Block (x, y, z): weight rows 128 x and on, rows of x from `tokens` y on, part z of K.  D[weight row, row of x] = W x^T: the weights of a chunk of 64
// columns go from a lane's 16 bytes through registers into tensor memory (the lanes of an m16n8k16 A fragment are those of a 16x128b store), x comes
// by TMA.  The weights are rounded to bf16 once, scale times whole number, as a stored bf16 weight would be.
// Results go through shared memory so that a row of y leaves in one piece; with K shared out every block of the cluster finishes `share` rows of x, whose
// sums the others store into it, and adds them in the order of the parts.
template <bool kG32>
__global__ void __launch_bounds__(kWideThreads, 1) w4_wide_kernel(const __grid_constant__ CUtensorMap x_map, Wide p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kWideStages], empty[kWideStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ int bad;
  const W4Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int first = p.chunks * static_cast<int>(blockIdx.z) / p.splits, last = p.chunks * (static_cast<int>(blockIdx.z) + 1) / p.splits;
  const int stage_bytes = p.tokens * 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kWideStages; ++i) {
      tc::mbar_init(full + i, 5);   // x's bytes and their announcement, and the weights of each 32 rows
      tc::mbar_init(empty + i, 1);
    }
    tc::mbar_init(&done, 1);
    tc::mbar_init_fence();
    bad = 0;
    tc::tma_prefetch_desc(&x_map);
  }
  __syncwarp();
  if (warp == 1) tc::tmem_alloc(&tmem_slot, p.allocated);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  if (p.splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block has started: its memory may be written
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  if (warp == 0) {   // ---- x
    if (tc::elect_one()) {
      int c = first, s = 0, round = 0;
      for (; c < last; ++c) {
        if (round > 0 && !wait_for(empty + s, (round - 1) & 1)) {
          bad = 1;
          break;
        }
        tc::mbar_expect_tx(full + s, stage_bytes);
        tc::tma_load_2d(smem + s * stage_bytes, &x_map, full + s, c * 64, blockIdx.y * p.tokens);
        if (++s == kWideStages) s = 0, ++round;
      }
      if (bad)   // what was issued must land before the block retires
        for (int i = max(c - first - kWideStages, 0); i < c - first; ++i) tc::mbar_wait(full + i % kWideStages, (i / kWideStages) & 1, 1u << 20);
    }
    __syncwarp();
  } else if (warp == 1) {   // ---- products
    // One thread from wait to commit: with the warp voting on every wait a chunk took 450 clocks at any number of rows of x.
    if (tc::elect_one()) {
      const uint64_t desc = tc::smem_desc_k_sw128(smem), stage_step = static_cast<uint64_t>(stage_bytes >> 4);
      const uint32_t weights = tmem + p.columns;
      uint32_t parity = 0;
      for (int c = first; c < last && !bad; parity ^= 1) {
        uint64_t db = desc;
#pragma unroll
        for (int s = 0; s < kWideStages; ++s, db += stage_step) {
          if (c == last) break;
          if (!wait_for(full + s, parity)) {
            bad = 1;
            break;
          }
          tc::fence_after_sync();
          if (s == 0 && c == first) {
            mma_ts(tmem, weights, db, p.idesc, false);
          } else {
            mma_ts(tmem, weights + s * 32, db, p.idesc, true);
          }
#pragma unroll
          for (int k = 1; k < 4; ++k) mma_ts(tmem, weights + s * 32 + k * 8, db + 2 * k, p.idesc, true);
          tc::mma_commit(empty + s);
          ++c;
        }
      }
      tc::mma_commit(&done);   // also after a failure: it releases the waiters
    }
    __syncwarp();
  } else {   // ---- weights: kTurns warps for each 32 rows take chunks in turn
    static_assert(kTurns == kWideStages);   // a warp's stage is always the same
    const int quarter = warp & 3, turn = (warp - 2) >> 2;
    const int row_tiles = (a.n + 15) / 16, groups = a.k >> p.group_shift, tile0 = blockIdx.x * (kWideRows / 16) + quarter * 2;
    constexpr int kDeep = kCodeDeep<kG32>, kTile = kCodeTile<kG32>;
    const uint32_t ring = tc::smem_u32(smem) + kWideStages * stage_bytes + (warp - 2) * (kDeep * 2 * kTile);
    const uint32_t place = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + p.columns + turn * 32;
    const int params_step = kTurns * 64 >> p.group_shift << 3;
    Ahead at[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) at[k] = ahead_of<kG32>(a, p.chunks, groups, p.group_shift, tile0 + k, row_tiles, first + turn, lane);
    auto issue = [&](int c, int slot) {
      if (c < last) {
#pragma unroll
        for (int k = 0; k < 2; ++k) copy_tile<kG32>(ring + (slot * 2 + k) * kTile, lane, at[k], params_step, 2 * c + 1 < groups);
      }
      copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kDeep - 1; ++i) issue(first + turn + kTurns * i, i);
    int slot = 0;
    uint32_t parity = 1;   // of the use before, once there was one
    for (int c = first + turn; c < last; c += kTurns, parity ^= 1) {
      copy_wait<kDeep - 2>();
      uint4 w[2];
      uint2 prm[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) take_tile<kG32>(ring + (slot * 2 + k) * kTile, lane, w[k], prm[k]);
      issue(c + kTurns * (kDeep - 1), slot == 0 ? kDeep - 1 : slot - 1);
      slot = slot == kDeep - 1 ? 0 : slot + 1;
      // the weights are ready in registers before their place in tensor memory is awaited: making them is not part of the loop from one use of a
      // place to the next (490 clocks per chunk when it was, at any number of rows of x)
      uint32_t r[2][16];
#pragma unroll
      for (int k = 0; k < 2; ++k) make_weights<kG32>(r[k], w[k], prm[k]);
      const bool ok = c - first < kWideStages || wait_for(empty + turn, parity);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) bad = 1;
        break;
      }
      tc::fence_after_sync();
#pragma unroll
      for (int k = 0; k < 2; ++k) tmem_st_16x64(place + (static_cast<uint32_t>(k * 16) << 16), r[k]);
      tmem_st_wait();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full + turn);
    }
    copy_wait<0>();
  }

  // ---- results
  __syncwarp();
  const int n0 = blockIdx.x * kWideRows, token0 = blockIdx.y * p.tokens, quarter = warp & 3, turn = (warp - 2) >> 2, row = quarter * 32 + lane;
  float bias[4] = {};
  if (p.splits > 1) {
    load_bias(bias, a, n0 + lane * 4);
  } else {
    bias[0] = a.bias && n0 + row < a.n ? __ldg(a.bias + n0 + row) : 0.f;
  }
  const bool ok = wait_for(&done, 0);
  tc::fence_after_sync();
  __syncwarp();
  const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  if (p.splits == 1) {
    if (warp >= 2 && !any_of_128(1 + turn, !ok))   // four warps leave together or not at all
      for (int c = turn; c < p.tokens / 16; c += kTurns)   // through where x was
        finish16(a, p.rows8, lanes + c * 16, reinterpret_cast<__nv_bfloat16*>(smem + c * kStaged), 1 + turn, token0 + c * 16, n0, quarter, lane, bias[0]);
  } else {
    float* sums = reinterpret_cast<float*>(smem + kWideStages * stage_bytes + kCodeRing);   // [part][row of x][weight row], behind everything else: other blocks write too
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp >= 2 && ok) {
      for (int c = turn; c < p.tokens / 16; c += kTurns) {
        uint32_t r[16];
        tmem_ld_32x16(lanes + c * 16, r);
        tc::tmem_ld_wait();
        int owner = c * 16 / p.share, at = c * 16 - owner * p.share;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          store_peer(tc::smem_u32(sums + (static_cast<int>(blockIdx.z) * p.share + at) * kWideRows + row), owner, __uint_as_float(r[i]));
          if (++at == p.share) {
            at = 0;
            ++owner;
          }
        }
      }
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int from = static_cast<int>(blockIdx.z) * p.share, rows = min(min(p.share, p.tokens - from), a.m - token0 - from);
    for (int i = warp; i < rows; i += kWideThreads / 32) {
      float4 v = *reinterpret_cast<const float4*>(sums + i * kWideRows + lane * 4);
      for (int r = 1; r < p.splits; ++r) {
        const float4 o = *reinterpret_cast<const float4*>(sums + (r * p.share + i) * kWideRows + lane * 4);
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      finish4(a, v, bias, token0 + from + i, n0 + lane * 4, p.vector);
    }
  }
  if ((!ok || bad) && threadIdx.x == 0) atomicExch(p.err, 22);
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, p.allocated);
  }
}

// ------------------------------------------------- tiles for several rounds of SMs --
// The same products for more tiles than there are SMs: a block takes tiles gridDim.x apart, and its four roles run on from one to the next.  Two sets of
// sums in tensor memory (up to 176 rows of x each, behind them five chunks of weights: 512 columns) let eight warps of their own write a tile's results beside
// the next one's products.  1537 x 16384 x 2048 takes 80 us in a burst, 1.29 PFLOP/s (95, 1.09, when calls go on for seconds and the power limit lowers the clock): 500 clocks per
// chunk, of which the products want 352.  No role alone is the rest: with a quarter of the products it takes 69 us, with weights that cost no arithmetic 71,
// with x that need not come 73.  (As one block per tile each round of SMs took 5 us before its first and after its last product: 103 us; four stages 83, six and
// fewer rows 87; rings of their own for x and weights, whose stages are then variables to the issuing thread, 99.)
constexpr int kResultWarps = 8;   // in two fours that take 16 rows of x in turn
constexpr int kStreamThreads = (2 + 4 * kTurns + kResultWarps) * 32;
constexpr int kStages = 5;   // of x and weights
constexpr int kStreamTokens = (512 - 32 * kStages) / 2;
constexpr int kStreamDeep = 3;   // chunks of codes of a warp
template <bool kG32>
constexpr int kStreamCodes = 4 * kTurns * 2 * kStreamDeep * kCodeTile<kG32>;
template <bool kG32>
int stream_smem(int tokens) { return kStages * tokens * 128 + kStreamCodes<kG32> + 4 * kStaged + 1024; }

template <bool kG32>
__global__ void __launch_bounds__(kStreamThreads, 1) w4_stream_kernel(const __grid_constant__ CUtensorMap x_map, Wide p) {
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  __shared__ uint64_t full[kStages], empty[kStages], sums_full[2], sums_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int bad;
  const W4Args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stage_bytes = p.tokens * 128;
  constexpr int kWeights = 2 * kStreamTokens;   // first column of the weights' ring
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(full + i, 5);
      tc::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(sums_full + i, 1);
      tc::mbar_init(sums_empty + i, kResultWarps);
    }
    tc::mbar_init_fence();
    bad = 0;
    tc::tma_prefetch_desc(&x_map);
  }
  __syncwarp();
  if (warp == 1) tc::tmem_alloc(&tmem_slot, 512);
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  if (warp == 0) {   // ---- x
    if (tc::elect_one()) {
      int s = 0, issued = 0;
      uint32_t parity = 1;   // of a stage's use before
      for (int tile = blockIdx.x; tile < p.tiles && !bad; tile += gridDim.x) {
        const int row0 = tile % p.row_tiles * p.tokens;
        for (int c = 0; c < p.chunks; ++c, ++issued) {
          if (issued >= kStages && !wait_for(empty + s, parity)) {
            bad = 1;
            break;
          }
          tc::mbar_expect_tx(full + s, stage_bytes);
          tc::tma_load_2d(smem + s * stage_bytes, &x_map, full + s, c * 64, row0);
          if (++s == kStages) s = 0, parity ^= 1;
        }
      }
      if (bad)   // what was issued must land before the block retires
        for (int i = max(issued - kStages, 0); i < issued; ++i) tc::mbar_wait(full + i % kStages, (i / kStages) & 1, 1u << 20);
    }
    __syncwarp();
  } else if (warp == 1) {   // ---- products
    // Chunks are counted through all tiles, and the loop is written out stage by stage: barriers and operands that are known when it is compiled leave
    // the thread some 140 clocks per chunk, a stage that is a variable 360 (and more beside warps that compute).
    if (tc::elect_one()) {
      const uint64_t desc = tc::smem_desc_k_sw128(smem), stage_step = static_cast<uint64_t>(stage_bytes >> 4);
      int left = (p.tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), c = 0;
      uint32_t parity = 0, set = 0, sums = tmem, used = 0, set_parity = 1;   // set_parity: of a set's use before
      while (left > 0 && !bad) {
        uint64_t db = desc;
#pragma unroll
        for (int s = 0; s < kStages; ++s, db += stage_step) {
          if (left == 0) break;
          if (c == 0 && used >= 2 && !wait_for(sums_empty + set, set_parity)) {
            bad = 1;
            break;
          }
          if (!wait_for(full + s, parity)) {
            bad = 1;
            break;
          }
          tc::fence_after_sync();
          mma_ts(sums, tmem + kWeights + s * 32, db, p.idesc, c > 0);
#pragma unroll
          for (int k = 1; k < 4; ++k) mma_ts(sums, tmem + kWeights + s * 32 + k * 8, db + 2 * k, p.idesc, true);
          tc::mma_commit(empty + s);
          if (++c == p.chunks) {
            tc::mma_commit(sums_full + set);
            c = 0;
            --left;
            ++used;
            set ^= 1;
            set_parity ^= set ^ 1;
            sums = tmem + set * kStreamTokens;
          }
        }
        parity ^= 1;
      }
      if (bad)   // releases the waiters
        for (int i = 0; i < 2; ++i) tc::mma_commit(sums_full + i);
    }
    __syncwarp();
  } else if (warp < 2 + 4 * kTurns) {   // ---- weights; chunks are counted through all tiles, so that a warp's stage is always the same
    const int quarter = warp & 3, turn = (warp - 2) >> 2;
    const int tiles16 = (a.n + 15) / 16, groups = a.k >> p.group_shift;
    constexpr int kDeep = kStreamDeep, kTile = kCodeTile<kG32>;
    const uint32_t ring = tc::smem_u32(smem) + kStages * stage_bytes + (warp - 2) * (kDeep * 2 * kTile);
    const uint32_t place = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + kWeights;
    // the loading side: a chunk of a tile, and where its codes and parameters are
    int tile = blockIdx.x, c = turn;
    const int params_step = kTurns * 64 >> p.group_shift << 3;
    Ahead at[2];
    auto settle = [&]() {   // after a tile's end: on to the tile that chunk c is one of
      while (c >= p.chunks) {
        c -= p.chunks;
        tile += gridDim.x;
      }
      if (tile < p.tiles) {
        const int tile0 = tile / p.row_tiles * (kWideRows / 16) + quarter * 2;
#pragma unroll
        for (int k = 0; k < 2; ++k) at[k] = ahead_of<kG32>(a, p.chunks, groups, p.group_shift, tile0 + k, tiles16, c, lane);
      }
    };
    // this warp's chunks among those of all the block's tiles
    const int mine = (p.tiles - static_cast<int>(blockIdx.x) + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x) * p.chunks;
    settle();
    auto issue = [&](int slot) {
      if (tile < p.tiles) {
        const uint32_t to = ring + slot * (2 * kTile);
#pragma unroll
        for (int k = 0; k < 2; ++k) copy_tile<kG32>(to + k * kTile, lane, at[k], params_step, 2 * c + 1 < groups);
        c += kTurns;
        if (c >= p.chunks) settle();
      }
      copy_commit();
    };
#pragma unroll
    for (int i = 0; i < kDeep - 1; ++i) issue(i);
    int slot = 0;
    int s = turn;
    uint32_t parity = 1;   // of a stage's use before
    for (int n = turn; n < mine; n += kTurns) {
      copy_wait<kDeep - 2>();
      uint4 w[2];
      uint2 prm[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) take_tile<kG32>(ring + (slot * 2 + k) * kTile, lane, w[k], prm[k]);
      issue(slot == 0 ? kDeep - 1 : slot - 1);
      slot = slot == kDeep - 1 ? 0 : slot + 1;
      uint32_t r[2][16];
#pragma unroll
      for (int k = 0; k < 2; ++k) make_weights<kG32>(r[k], w[k], prm[k]);
      const bool ok = n < kStages || wait_for(empty + s, parity);
      if (!__all_sync(0xffffffffu, ok)) {
        if (lane == 0) bad = 1;
        break;
      }
      tc::fence_after_sync();
#pragma unroll
      for (int k = 0; k < 2; ++k) tmem_st_16x64(place + s * 32 + (static_cast<uint32_t>(k * 16) << 16), r[k]);
      tmem_st_wait();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full + s);
      s += kTurns;
      if (s >= kStages) s -= kStages, parity ^= 1;
    }
    copy_wait<0>();
  } else {   // ---- results
    const int quarter = warp & 3, four = (warp - 2 - 4 * kTurns) >> 2;
    unsigned char* staged = smem + kStages * stage_bytes + kStreamCodes<kG32> + four * (2 * kStaged);   // [2][row of x][weight row]
    int i = 0, half = 0;
    for (int tile = blockIdx.x; tile < p.tiles; tile += gridDim.x, ++i) {
      const int block = tile / p.row_tiles, row0 = (tile - block * p.row_tiles) * p.tokens, n0 = block * kWideRows, n = n0 + quarter * 32 + lane;
      const float bias = a.bias && n < a.n ? __ldg(a.bias + n) : 0.f;
      if (any_of_128(1 + four, !wait_for(sums_full + (i & 1), (i >> 1) & 1))) {   // these four warps leave together or not at all
        bad = 1;
        break;
      }
      tc::fence_after_sync();
      const uint32_t sums = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (i & 1) * kStreamTokens;
      for (int c = four; c < p.tokens / 16; c += 2, half ^= 1)
        finish16(a, p.rows8, sums + c * 16, reinterpret_cast<__nv_bfloat16*>(staged + half * kStaged), 1 + four, row0 + c * 16, n0, quarter, lane, bias);
      // the products of the tile after next may begin
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(sums_empty + (i & 1));
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (bad && threadIdx.x == 0) atomicExch(p.err, 23);
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// A warp per tile of 16 x 64: lane (g, t) writes pairs of rows g and g + 8.
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
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int at = c * 64 + s * 16 + 2 * t;
      if (at >= k) continue;
      const uint2 p = __ldg(params + (static_cast<size_t>(tile) * groups + at / group) * 8 + g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // nibble j: row g + 8 (j & 1), columns 8 (j >> 1) on
        const int row = tile * 16 + (j & 1) * 8 + g;
        const uint32_t prm = j & 1 ? p.y : p.x;
        if (row < n) *reinterpret_cast<uint32_t*>(w + static_cast<size_t>(row) * k + at + (j >> 1) * 8) = mul2(codes2(word[s] >> (4 * j), zero2(prm)), scale2(prm));
      }
    }
  }
}

// A warp per tile of 16 x 64, a lane its 16 bytes; behind the tiles, a thread per row and group of the parameters.  (k and the address of the codes are even: two neighbouring codes are one access.)
__global__ void __launch_bounds__(256) w4_pack_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales, const uint8_t* __restrict__ zeros, uint4* __restrict__ packed,
                                                      uint32_t* __restrict__ params, int* bad, int n, int k, int group) {
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const int chunks = (k + 63) / 64, groups = k / group, tiles = (n + 15) / 16;
  const long long pieces = static_cast<long long>(tiles) * chunks * 32, entries = static_cast<long long>(tiles) * groups * 16;
  uint32_t seen = 0;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < pieces + entries; i += gridDim.x * 256ll) {
    if (i < pieces) {
      const int lane = static_cast<int>(i & 31), g = lane >> 2, t = lane & 3;
      const long long at = i >> 5;
      const int tile = static_cast<int>(at / chunks), c = static_cast<int>(at - static_cast<long long>(tile) * chunks);
      uint32_t word[4] = {};
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // row g + 8 (j & 1), columns 8 (j >> 1) on
          const int row = tile * 16 + g + 8 * (j & 1), col = c * 64 + 16 * s + 8 * (j >> 1) + 2 * t;
          if (row < n && col < k) {
            const uint32_t two = *reinterpret_cast<const uint16_t*>(codes + static_cast<size_t>(row) * k + col);
            seen |= two;
            word[s] |= ((two & 15u) | (two & 0xf00u) << 8) << (4 * j);
          }
        }
      packed[i] = make_uint4(word[0], word[1], word[2], word[3]);
    } else {
      const long long e = i - pieces, at = e >> 4;   // [tile][group][8 g][2]
      const int tile = static_cast<int>(at / groups), group_at = static_cast<int>(at - static_cast<long long>(tile) * groups), row = tile * 16 + static_cast<int>(e >> 1 & 7) + 8 * static_cast<int>(e & 1);
      uint32_t v = 0x43000000u;
      if (row < n) {
        const size_t from = static_cast<size_t>(row) * groups + group_at;
        const uint32_t zero = zeros ? zeros[from] : 8u;
        seen |= zero;
        v = scales[from] | (0x4300u + (zero & 15u)) << 16;
      }
      params[e] = v;
    }
  }
  if ((seen & 0xf0f0u) != 0) *bad = 1;
}

int sm_count() {
  static const int n = [] {
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return sms;
  }();
  return n;
}

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

template <int kR, int kN, int kParams, bool kEven>
cudaError_t launch_narrow(const W4Args& a, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(w4_narrow_kernel<kR, kN, kParams, kEven>, kSmemLimit, allowed);
  if (rc != cudaSuccess) return rc;
  const int chunks = (a.k + 63) / 64, smem = narrow_smem<kR, kN, kParams>(a.m * ((chunks + 1) / 2) * 256);
  if (smem > kSmemLimit) return cudaErrorNotSupported;
  const int tiles = ((a.n + 15) / 16 + kR - 1) / kR, blocks = sm_count() * (smem <= 113 * 1024 ? 2 : 1);
  // as few warps along K as give every warp a tile: adding up costs a barrier and a pass through shared memory
  int along = 3;
  while (along > 0 && tiles << (along - 1) >= blocks * kNarrowWarps * 3 / 4) --along;
  const int groups = (tiles + (kNarrowWarps >> along) - 1) / (kNarrowWarps >> along);
  MCCL_LAUNCH_PDL((w4_narrow_kernel<kR, kN, kParams, kEven>), groups < blocks ? groups : blocks, kNarrowThreads, smem, stream, a, (a.n + 15) / 16, chunks, log2_of(a.group), along);
  count_launch();
  return ::mccl::launch_status();
}
template <int kR, int kN, int kParams>
cudaError_t narrow_by_size(const W4Args& a, cudaStream_t stream) {
  return a.k % 128 == 0 && (a.n + 15) / 16 % kR == 0 ? launch_narrow<kR, kN, kParams, true>(a, stream) : launch_narrow<kR, kN, kParams, false>(a, stream);
}
template <int kR, int kN>
cudaError_t narrow(const W4Args& a, cudaStream_t stream) {
  return a.group == 32 ? narrow_by_size<kR, kN, 4>(a, stream) : (a.group == 64 ? narrow_by_size<kR, kN, 2>(a, stream) : narrow_by_size<kR, kN, 1>(a, stream));
}

int wide_smem(const Wide& p) { return kWideStages * p.tokens * 128 + kCodeRing + (p.splits > 1 ? p.splits * p.share * kWideRows * 4 : 0) + 1024; }

// Blocks that the GPU holds at a time, in clusters of `splits`: a cluster lies in one group of SMs, and what is left over in each group stays idle (148, 148,
// 135, 132, 130, 132, 105 and 120 for clusters of one to eight).
int resident(int splits) {
  static const std::array<int, 9> counts = [] {
    std::array<int, 9> c = {};
    for (int n = 1; n <= 8; ++n) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1, 1, n);
      cfg.blockDim = dim3(kWideThreads);
      cfg.dynamicSmemBytes = kWideSmem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = n;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      int clusters = 0;
      cudaError_t rc = cudaFuncSetAttribute(w4_wide_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, kWideSmem);
      if (rc == cudaSuccess) rc = cudaOccupancyMaxActiveClusters(&clusters, w4_wide_kernel<false>, &cfg);
      if (rc != cudaSuccess) cudaGetLastError();
      c[n] = rc == cudaSuccess && clusters > 0 ? clusters * n : sm_count() * 3 / 4;
    }
    return c;
  }();
  return counts[splits];
}

// Rows of x per block and parts of K.  A chunk of 64 columns costs the making of its weights (some 400 clocks) or its products (two clocks per row of x), a
// block some 5000 clocks before its first and after its last chunk.  (Measured beside all other choices for 27 sizes from 20 x 512 x 512 to
// 1537 x 16384 x 2048: within 4 % of the best.)
// With more tiles than SMs they run on from one to the next (returns true), so that no round has a beginning and an end of its own: 1537 x 16384 x 2048 took
// 103 us in rounds.  More rows than a grid has blocks for, 256 x 65535, always run on: they are enough for several rounds.  (p.tokens stays 0 where nothing fits.)
bool choose_wide(int m, int blocks, Wide& p) {
  constexpr double kMake = 400, kRound = 5000, kSplit = 2200, kToken = 20;
  double best = std::numeric_limits<double>::infinity();
  Wide w = p;
  for (int most = 16, before = 0; most <= kMostTokens && before != 1; most += 16) {
    const int tiles = (m + most - 1) / most;
    if (tiles == before || tiles > 65535) continue;
    before = tiles;
    w.tokens = ((m + tiles - 1) / tiles + 15) / 16 * 16;
    const int row_tiles = (m + w.tokens - 1) / w.tokens;
    for (w.splits = 1; w.splits <= 8 && (w.splits == 1 || w.splits * 2 <= p.chunks); ++w.splits) {
      w.share = (w.tokens + w.splits - 1) / w.splits;
      if (wide_smem(w) > kWideSmem) continue;
      const long long all = static_cast<long long>(blocks) * row_tiles * w.splits;
      const int at_once = resident(w.splits);
      if (w.splits > 1 && all > at_once) break;
      const long long waves = (all + at_once - 1) / at_once;
      const double products = 2.0 * w.tokens;
      const double cost = waves * ((p.chunks + w.splits - 1) / w.splits * (kMake > products ? kMake : products) + kRound + (w.splits > 1 ? kSplit : 0.0) + kToken * w.tokens);
      if (cost < best) {
        best = cost;
        p.tokens = w.tokens;
        p.splits = w.splits;
        p.share = w.share;
      }
    }
  }
  bool stream = false;
  for (int most = 32, before = 0; most <= kStreamTokens && before != 1; most += 16) {
    const int tiles = (m + most - 1) / most, tokens = ((m + tiles - 1) / tiles + 15) / 16 * 16, row_tiles = (m + tokens - 1) / tokens;
    if (tiles == before) continue;
    before = tiles;
    if (tokens > kStreamTokens || static_cast<long long>(blocks) * row_tiles > 0x7fffffff || (p.a.group == 32 ? stream_smem<true>(tokens) : stream_smem<false>(tokens)) > kWideSmem) continue;
    const int all = blocks * row_tiles, rounds = (all + sm_count() - 1) / sm_count();
    if (rounds < 2) continue;
    const double products = 2.0 * tokens;
    const double cost = rounds * (p.chunks * (kMake > products ? kMake : products) + 300.0) + kRound + kToken * tokens;
    if (cost < best) {
      best = cost;
      stream = true;
      p.tokens = tokens;
      p.splits = 1;
      p.share = tokens;
      p.tiles = all;
      p.row_tiles = row_tiles;
    }
  }
  return stream;
}

template <bool kG32>
cudaError_t start_wide(const Wide& p, dim3 grid, const CUtensorMap& map, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(w4_wide_kernel<kG32>, kWideSmem, allowed);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL_CLUSTER(w4_wide_kernel<kG32>, grid, kWideThreads, wide_smem(p), stream, static_cast<unsigned>(p.splits), map, p);
  count_launch();
  return ::mccl::launch_status();
}

template <bool kG32>
cudaError_t start_stream(const Wide& p, const CUtensorMap& map, cudaStream_t stream) {
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(w4_stream_kernel<kG32>, kWideSmem, allowed);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL(w4_stream_kernel<kG32>, p.tiles < sm_count() ? p.tiles : sm_count(), kStreamThreads, stream_smem<kG32>(p.tokens), stream, map, p);
  count_launch();
  return ::mccl::launch_status();
}

cudaError_t launch_wide(const W4Args& a, cudaStream_t on) {
  Wide p;
  p.a = a;
  p.chunks = (a.k + 63) / 64;
  p.group_shift = log2_of(a.group);
  const int blocks = (a.n + kWideRows - 1) / kWideRows;
  if (a.m > kMostRows) return cudaErrorInvalidValue;
  const bool stream = choose_wide(a.m, blocks, p);
  if (p.tokens == 0) return cudaErrorInvalidValue;
  p.columns = p.tokens <= 32 ? 32 : (p.tokens <= 64 ? 64 : (p.tokens <= 128 ? 128 : 256));
  p.allocated = p.columns + kWideStages * 32 <= 256 ? 256 : 512;
  p.vector = a.n % 4 == 0 && (a.residual == nullptr || (a.ldr % 4 == 0 && reinterpret_cast<uintptr_t>(a.residual) % 8 == 0));
  p.rows8 = a.n % 8 == 0;
  p.idesc = tc::idesc_bf16(kWideRows, p.tokens);
  p.err = gemm_error_device_ptr();
  const CuDriver& cu = CuDriver::get();
  if (!cu.loaded || !cu.TensorMapEncodeTiled) return cudaErrorNotSupported;
  CUtensorMap map;
  const cuuint64_t size[2] = {static_cast<cuuint64_t>(a.k), static_cast<cuuint64_t>(a.m)}, stride[1] = {static_cast<cuuint64_t>((a.m > 1 ? a.ldx : a.k) * 2)};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(p.tokens)}, step[2] = {1, 1};
  if (cu.TensorMapEncodeTiled(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.x), size, stride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return cudaErrorNotSupported;
  if (stream) return a.group == 32 ? start_stream<true>(p, map, on) : start_stream<false>(p, map, on);
  const dim3 grid(blocks, (a.m + p.tokens - 1) / p.tokens, p.splits);
  return a.group == 32 ? start_wide<true>(p, grid, map, on) : start_wide<false>(p, grid, map, on);
}

}  // namespace

cudaError_t w4_linear(const W4Args& a, cudaStream_t stream) {
  if (a.m <= 0 || a.n <= 0) return cudaSuccess;
  const long long x_bytes = static_cast<long long>(a.m) * ((a.k + 127) / 128) * 256;
  if (a.m <= 16 && x_bytes <= kNarrowX) {
    // two tiles of weights per warp share what is read of x (1 x 16384 x 2048 6.5 us, 7.9 with one; 4 x 32000 x 2048 12.7 and 14.3), if that leaves every SM some
    // warps' work (1 x 2048 x 2048: 2.6 with one) and x its room (with groups of 32 the parameters leave 115 KB); 16 rows' sums leave no registers for it
    const int bytes = static_cast<int>(x_bytes), smem = a.group == 32 ? narrow_smem<2, 1, 4>(bytes) : (a.group == 64 ? narrow_smem<2, 1, 2>(bytes) : narrow_smem<2, 1, 1>(bytes));
    const bool two = a.n >= 16 * 3 * sm_count() && smem <= kSmemLimit;
    if (a.m <= 8) return two ? narrow<2, 1>(a, stream) : narrow<1, 1>(a, stream);
    return narrow<1, 2>(a, stream);
  }
  return launch_wide(a, stream);
}

cudaError_t w4_pack(const uint8_t* codes, const void* scales, const uint8_t* zeros, void* packed, void* params, int* bad, int n, int k, int group, cudaStream_t stream) {
  if (n <= 0 || k <= 0) return cudaSuccess;
  const long long tiles = (n + 15) / 16, all = tiles * ((k + 63) / 64) * 32 + tiles * (k / group) * 16, blocks = (all + 255) / 256;
  MCCL_LAUNCH_PDL(w4_pack_kernel, static_cast<unsigned>(blocks < 148 * 16 ? blocks : 148 * 16), 256, 0, stream, codes, static_cast<const uint16_t*>(scales), zeros,
                  static_cast<uint4*>(packed), static_cast<uint32_t*>(params), bad, n, k, group);
  count_launch();
  return ::mccl::launch_status();
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
