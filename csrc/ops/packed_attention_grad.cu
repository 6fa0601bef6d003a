// Gradients of packed attention (bf16), on the 5th-generation tensor cores.
//
// With P = exp(S - lse), the forward pass's weights, and delta_i = sum_d dO_id O_id:
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta) scale,  dQ = dS K,  dK = dS^T Q
// Two kernels, each with its sums in tensor memory from beginning to end, so that nothing is added in memory and every sum has one order:
//   keys     a block of 128 keys and the queries that see it (of all heads that share it): S^T = K Q^T, dP^T = V dO^T, then dV += P^T dO and dK += dS^T Q.
//            The transposed scores have a key per lane, so P^T and dS^T are left operands straight from tensor memory and never pass through shared memory.
//   queries  a block of 128 queries and the keys they see: S = Q K^T, dP = dO V^T, dQ += dS K, in the same way.
// S and dP are computed twice for that (7 products instead of 5): without it dQ's parts would be added in memory as they arrive, in an order that changes.
// delta comes first, from a kernel of its own.
//
// Both loops are two chains that overlap: while threads make P of a block, the tensor cores multiply dS of the one before, and the other way round.
#include "packed_tiles.cuh"

#include "smem_limit.hpp"

#include <climits>

namespace mccl {
namespace ops {

namespace {

using namespace packed;
using H = Bf16;

constexpr int kThreads = 12 * 32;   // warps 0-3 and 4-7: rows, half of the columns each; 8: products; 9: loads; 10: rows behind the sequence, statistics; 11: nothing
// 256 x 208 + 128 x 80 of the launch's 384 x 168 registers.
constexpr int kRowRegisters = 208, kOtherRegisters = 80;
constexpr int kStage = 8 * 2048;    // results on their way out, 32 rows x 64 bytes per warp

struct Grad {
  Problem p;
  const float* lse;     // [heads, tokens]
  const float* delta;   // [heads, tokens]
  void* dq;
  void* dk;
  void* dv;
  int units;
};

// Rows row .. 127 of a tile: zeros.  Whole-warp call.
template <int DP>
__device__ __forceinline__ void zero_rows(uint8_t* tile, int row) {
  for (int i = (threadIdx.x & 31); i < DP / 64 * (kRows - row) * 8; i += 32) {
    const int sub = i / ((kRows - row) * 8), in = i - sub * (kRows - row) * 8;
    *reinterpret_cast<uint4*>(tile + sub * kSub + row * 128 + in * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ----------------------------------------------------------------------------------------------------- delta ----
// delta[h, t] = sum_d dO[t, h, d] O[t, h, d], with O as it was before it was rounded (its rounding would be the same for all of a row's scores: dQ and dK were off
// by 1.5 to 1.6 times what their own rounding leaves, now by 1.4).  A warp per 32 rows of a head, a half-warp per row at a time.
__global__ void __launch_bounds__(256) packed_delta_kernel(const H::T* o, const H::T* o_rest, TokenView d_o, float* delta, int tokens, int heads, int head_dim) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = lane >> 4, c = (lane & 15) * 8;
  const int h = blockIdx.y * 8 + warp, t0 = blockIdx.x * 32;
  if (h >= heads) return;
  float mine = 0.f;
#pragma unroll 4
  for (int i = 0; i < 16; ++i) {
    const int t = t0 + 2 * i + half;
    float sum = 0.f;
    if (t < tokens && c < head_dim) {
      const long long at = (static_cast<long long>(t) * heads + h) * head_dim + c;
      float x[8], rest[8], y[8];
      unpack8_as<H>(__ldg(reinterpret_cast<const uint4*>(o + at)), x);
      unpack8_as<H>(__ldg(reinterpret_cast<const uint4*>(o_rest + at)), rest);
      unpack8_as<H>(__ldg(reinterpret_cast<const uint4*>(static_cast<const H::T*>(d_o.p) + t * d_o.token + h * d_o.head + c)), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = fmaf(x[e] + rest[e], y[e], sum);
    }
#pragma unroll
    for (int s = 8; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    const float other = __shfl_xor_sync(0xffffffffu, sum, 16);
    if ((lane >> 1) == i) mine = (lane & 1) == half ? sum : other;
  }
  if (t0 + lane < tokens) delta[static_cast<long long>(h) * tokens + t0 + lane] = mine;
}

// ------------------------------------------------------------------------------------------------------ keys ----
// The queries that see a block of keys: tiles of 128 rows from `row` on, of each of the heads that share it.
struct KeyUnit {
  Sequence s;
  int block, kv;         // first key 128 * block
  int row, end, tiles;   // rows row .. end - 1 of the sequence, per head
  int place;             // position of a query minus its row
  bool any;
};
__device__ __forceinline__ KeyUnit key_unit(const Grad& a, int u) {
  const Problem& p = a.p;
  KeyUnit r;
  r.any = false;
  const int slot = u / p.kv_heads;   // a sequence's first keys have the most queries: first
  r.kv = u - slot * p.kv_heads;
  const int s = find_sequence(p.k_offsets, p.sequences, p.k_tokens, slot, kRows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  r.block = slot - (r.s.k0 / kRows + s);
  if (r.block < 0 || r.block * kRows >= r.s.m) return r;
  r.any = true;
  r.place = r.s.m - r.s.n;
  r.row = max(0, r.block * kRows - r.place);
  const int last_key = min(r.block * kRows + kRows, r.s.m) - 1;
  r.end = r.block * kRows < p.sinks ? r.s.n : static_cast<int>(min(static_cast<long long>(r.s.n), static_cast<long long>(last_key) + p.window - r.place));
  r.tiles = r.end > r.row ? (r.end - r.row + kRows - 1) / kRows : 0;
  return r;
}

template <int DP>
constexpr int key_smem() { return 6 * (DP / 64) * kSub + kStage + 2 * 2 * kRows * 4 + 512 + 1024; }

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_grad_keys_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const __grid_constant__ CUtensorMap tm_do, const Grad a) {
  constexpr int kTile = (DP / 64) * kSub;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_k = smem;
  uint8_t* s_v = s_k + kTile;
  uint8_t* s_q = s_v + kTile;        // [2]
  uint8_t* s_do = s_q + 2 * kTile;   // [2]
  uint8_t* s_out = s_do + 2 * kTile;
  float* s_lse = reinterpret_cast<float*>(s_out + kStage);   // [2][128], times log2 e
  float* s_delta = s_lse + 2 * kRows;                        // [2][128]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_delta + 2 * kRows);
  uint64_t* v_full = k_full + 1;
  uint64_t* q_raw = v_full + 1;      // [2]: brought
  uint64_t* do_raw = q_raw + 2;      // [2]
  uint64_t* q_full = do_raw + 2;     // [2]: and rows behind the sequence cleared, statistics there
  uint64_t* empty = q_full + 2;      // [2]: both have been read
  uint64_t* s_full = empty + 2;
  uint64_t* p_full = s_full + 1;
  uint64_t* dp_full = p_full + 1;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);
  KeyUnit* s_unit = reinterpret_cast<KeyUnit*>(tmem_slot + 4);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (uint64_t* b = k_full; b <= done; ++b) tc::mbar_init(b, b == p_full || b == ds_full ? 256 : 1);
    *bad = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(tmem_slot, 512);
  pdl_wait();
  if (warp == 0) {
    const KeyUnit found = key_unit(a, static_cast<int>(blockIdx.x));
    if (lane == 0) *s_unit = found;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const KeyUnit& u = *s_unit;
  pdl_trigger();
  // tensor memory: S^T (then P^T) 0, dP^T (then dS^T) 128, dV 256, dK 256 + DP.  Each half of the threads keeps to its own 64 columns of the first two.
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 256 + DP;
  const int items = u.any ? u.tiles * p.group : 0;

  if (items > 0 && warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 9) {
      // ----------------------------------------------------------------------------------------- loads ----
      if (tc::elect_one()) {
        tc::mbar_expect_tx(k_full, kTile);
        load_tile<DP>(s_k, &tm_k, k_full, u.kv, u.s.k0 + u.block * kRows);
        int n = 0;
        bool ok = true;
        for (int g = 0; g < p.group && ok; ++g) {
          for (int t = 0; t < u.tiles; ++t, ++n) {
            const int st = n & 1;
            if (n >= 2) ok = wait(&empty[st], (n / 2 - 1) & 1, bad);
            if (!ok) break;
            const int row = u.s.q0 + u.row + t * kRows;
            tc::mbar_expect_tx(&q_raw[st], kTile);
            load_tile<DP>(s_q + st * kTile, &tm_q, &q_raw[st], u.kv * p.group + g, row);
            if (n == 0) {
              tc::mbar_expect_tx(v_full, kTile);
              load_tile<DP>(s_v, &tm_v, v_full, u.kv, u.s.k0 + u.block * kRows);
            }
            tc::mbar_expect_tx(&do_raw[st], kTile);
            load_tile<DP>(s_do + st * kTile, &tm_do, &do_raw[st], u.kv * p.group + g, row);
          }
        }
        if (!ok) {   // loads that were issued must land before the block retires
          tc::mbar_wait(k_full, 0, 1u << 18);
          tc::mbar_wait(v_full, 0, 1u << 18);
          for (int i = max(0, n - 2); i < n; ++i) {
            tc::mbar_wait(&q_raw[i & 1], (i / 2) & 1, 1u << 18);
            tc::mbar_wait(&do_raw[i & 1], (i / 2) & 1, 1u << 18);
          }
        }
      }
      __syncwarp();
    } else if (warp == 10) {
      // ---------------------------------- statistics of the queries; rows behind the sequence must not be NaN ----
      for (int n = 0; n < items; ++n) {
        const int st = n & 1, g = n / u.tiles, row = u.row + (n - g * u.tiles) * kRows, rows = min(kRows, u.s.n - row);
        const long long at = static_cast<long long>(u.kv * p.group + g) * p.tokens + u.s.q0 + row;
        float l[4], d[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 32 + lane;
          l[i] = r < rows ? a.lse[at + r] * kLog2e : INFINITY;
          d[i] = r < rows ? a.delta[at + r] : 0.f;
          if (l[i] == -INFINITY) l[i] = INFINITY;   // sees nothing
        }
        bool ok = n < 2 || wait(&empty[st], (n / 2 - 1) & 1, bad);
        if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s_lse[st * kRows + i * 32 + lane] = l[i];
          s_delta[st * kRows + i * 32 + lane] = d[i];
        }
        ok = wait(&q_raw[st], (n / 2) & 1, bad) && wait(&do_raw[st], (n / 2) & 1, bad);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (rows < kRows) {
          zero_rows<DP>(s_q + st * kTile, rows);
          zero_rows<DP>(s_do + st * kTile, rows);
          fence_async_smem();
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_full[st]);
        __syncwarp();
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------------------------------- products ----
      constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false);
      const uint32_t idesc_g = idesc16<H>(kRows, (p.head_dim + 15) / 16 * 16, false, true);
      const int steps = (p.head_dim + 15) / 16;
      bool ok = true;
      auto all_wait = [&](uint64_t* bar, uint32_t parity) {
        const bool w = ok && wait(bar, parity, bad);
        ok = __all_sync(0xffffffffu, w);
        tc::fence_after_sync();
        return ok;
      };
      if (all_wait(k_full, 0) && all_wait(&q_full[0], 0)) {
        if (tc::elect_one()) {
          mma_rows(t_s, s_k, s_q, idesc_s, steps);
          tc::mma_commit(s_full);
        }
        __syncwarp();
        if (all_wait(v_full, 0) && tc::elect_one()) {
          mma_rows(t_dp, s_v, s_do, idesc_s, steps);
          tc::mma_commit(dp_full);
        }
        __syncwarp();
      }
      for (int n = 0; n < items && ok; ++n) {
        const int st = n & 1, next = st ^ 1;
        const bool more = n + 1 < items;
        if (!all_wait(p_full, n & 1)) break;
        if (tc::elect_one()) mma_weights<128, 64>(t_dv, t_s, s_do + st * kTile, idesc_g, n > 0);
        __syncwarp();
        if (more) {
          if (!all_wait(&q_full[next], ((n + 1) / 2) & 1)) break;
          if (tc::elect_one()) {
            mma_rows(t_s, s_k, s_q + next * kTile, idesc_s, steps);
            tc::mma_commit(s_full);
          }
          __syncwarp();
        }
        if (!all_wait(ds_full, n & 1)) break;
        if (tc::elect_one()) {
          mma_weights<128, 64>(t_dk, t_dp, s_q + st * kTile, idesc_g, n > 0);
          tc::mma_commit(&empty[st]);
          if (more) {
            mma_rows(t_dp, s_v, s_do + next * kTile, idesc_s, steps);
            tc::mma_commit(dp_full);
          } else {
            tc::mma_commit(done);
          }
        }
        __syncwarp();
      }
    }
  } else if (items > 0) {
    // -------------------------------------------------------------------- a key per thread, half of the queries ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_s = t_s + lanes + half * 64, my_dp = t_dp + lanes + half * 64;
    const int key = u.block * kRows + row, first_key = u.block * kRows;
    const bool sink = key < p.sinks;
    bool ok = true;
    for (int n = 0; n < items; ++n) {
      const int st = n & 1, t = n % u.tiles;
      const int first = u.place + u.row + t * kRows + half * 64;   // position of my first column
      // the columns that see my key: low <= c < high
      const bool partly = !(first >= first_key + kRows - 1 && (first + 63 - p.window < first_key || first_key + kRows <= p.sinks));
      const int low = key - first, high = sink ? 64 : static_cast<int>(min(64ll, static_cast<long long>(key) + p.window - first));
      ok = wait(&q_full[st], (n / 2) & 1, bad) && wait(s_full, n & 1, bad);   // statistics and scores
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      float w[64];
      {
        uint32_t r[2][32];
        tc::tmem_ld_32x32(my_s, r[0]);
        tc::tmem_ld_32x32(my_s + 32, r[1]);
        tc::tmem_ld_wait();
        const float4* l4 = reinterpret_cast<const float4*>(s_lse + st * kRows + half * 64);
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          const float4 l = l4[c];
          w[4 * c] = exp2f(fmaf(__uint_as_float(r[c / 8][c % 8 * 4]), p.scale_log2, -l.x));
          w[4 * c + 1] = exp2f(fmaf(__uint_as_float(r[c / 8][c % 8 * 4 + 1]), p.scale_log2, -l.y));
          w[4 * c + 2] = exp2f(fmaf(__uint_as_float(r[c / 8][c % 8 * 4 + 2]), p.scale_log2, -l.z));
          w[4 * c + 3] = exp2f(fmaf(__uint_as_float(r[c / 8][c % 8 * 4 + 3]), p.scale_log2, -l.w));
        }
      }
      if (partly) {
#pragma unroll
        for (int c = 0; c < 64; ++c) w[c] = c >= low && c < high ? w[c] : 0.f;
      }
      {
        uint32_t x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const H::T2 h = H::down(w[2 * e], w[2 * e + 1]);
          x[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st32(my_s, x);
      }
      tmem_st_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(p_full);
      ok = wait(dp_full, n & 1, bad);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      {
        uint32_t x[32];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t r[32];
          tc::tmem_ld_32x32(my_dp + 32 * g, r);
          tc::tmem_ld_wait();
          const float4* d4 = reinterpret_cast<const float4*>(s_delta + st * kRows + half * 64 + g * 32);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const float4 d = d4[c];
            float f[4] = {__uint_as_float(r[4 * c]) - d.x, __uint_as_float(r[4 * c + 1]) - d.y, __uint_as_float(r[4 * c + 2]) - d.z, __uint_as_float(r[4 * c + 3]) - d.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = g * 32 + 4 * c + e;
              f[e] = partly && !(at >= low && at < high) ? 0.f : f[e] * w[at];
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const H::T2 h = H::down(f[2 * e], f[2 * e + 1]);
              x[g * 16 + c * 2 + e] = *reinterpret_cast<const uint32_t*>(&h);
            }
          }
        }
        tmem_st32(my_dp, x);
      }
      tmem_st_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(ds_full);
    }
    if (ok) {
      ok = wait(done, 0, bad);
      ok = __all_sync(0xffffffffu, ok);
      tc::fence_after_sync();
    }
    if (ok) {   // one half takes dV out, the other dK
      const uint32_t from = (half == 0 ? t_dv : t_dk) + lanes;
      const float scale = half == 0 ? 1.f : p.scale;
      const long long stride = static_cast<long long>(p.kv_heads) * p.head_dim;
      const int first_row = first_key + (warp & 3) * 32;
      H::T* to = static_cast<H::T*>(half == 0 ? a.dv : a.dk) + (u.s.k0 + first_row) * stride + u.kv * p.head_dim;
      for (int c0 = 0; c0 < p.head_dim; c0 += 32) {
        uint32_t r[32];
        tc::tmem_ld_32x32(from + c0, r);
        tc::tmem_ld_wait();
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = __uint_as_float(r[e]) * scale;
        rows_out<H>(s_out + warp * 2048, f, to, stride, u.s.m - first_row, c0, p.head_dim);
      }
    }
    tc::fence_before_sync();
  } else if (u.any) {
    // nobody sees these keys
    const int rows = min(kRows, u.s.m - u.block * kRows), d8 = p.head_dim / 8;
    const long long at = (static_cast<long long>(u.s.k0 + u.block * kRows) * p.kv_heads + u.kv) * p.head_dim;
    for (int i = tid; i < rows * d8; i += kThreads) {
      const long long to = at + static_cast<long long>(i / d8) * p.kv_heads * p.head_dim + i % d8 * 8;
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dk) + to) = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dv) + to) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 32);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
  zero_outside<H::T>(a.dk, p.kv_heads * p.head_dim, nullptr, 0, p.k_offsets, p.sequences, p.k_tokens, blockIdx.x, gridDim.x, tid, kThreads);
  zero_outside<H::T>(a.dv, p.kv_heads * p.head_dim, nullptr, 0, p.k_offsets, p.sequences, p.k_tokens, blockIdx.x, gridDim.x, tid, kThreads);
}

// --------------------------------------------------------------------------------------------------- queries ----
struct QueryUnit {
  Sequence s;
  int head, row, first, last;   // positions of the tile's rows
  Blocks b;
  bool any;
};
__device__ __forceinline__ QueryUnit query_unit(const Grad& a, int u) {
  const Problem& p = a.p;
  QueryUnit r;
  r.any = false;
  const int slots = a.units / p.heads, slot = slots - 1 - u / p.heads;   // long rows first
  r.head = u % p.heads;
  const int s = find_sequence(p.offsets, p.sequences, p.tokens, slot, kRows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  r.row = (slot - (r.s.q0 / kRows + s)) * kRows;
  if (r.row < 0 || r.row >= r.s.n) return r;
  r.any = true;
  r.first = r.s.m - r.s.n + r.row;
  r.last = min(r.first + kRows, r.s.m) - 1;
  r.b = blocks_of(p, r.first, r.last);
  return r;
}

template <int DP>
constexpr int query_smem() { return 6 * (DP / 64) * kSub + kStage + 512 + 1024; }

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_grad_queries_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                               const __grid_constant__ CUtensorMap tm_do, const Grad a) {
  constexpr int kTile = (DP / 64) * kSub;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;
  uint8_t* s_do = s_q + kTile;
  uint8_t* s_k = s_do + kTile;      // [2]
  uint8_t* s_v = s_k + 2 * kTile;   // [2]
  uint8_t* s_out = s_v + 2 * kTile;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_out + kStage);
  uint64_t* do_full = q_full + 1;
  uint64_t* k_raw = do_full + 1;    // [2]: brought
  uint64_t* k_full = k_raw + 2;     // [2]: and rows behind the sequence cleared
  uint64_t* v_full = k_full + 2;    // [2]
  uint64_t* k_empty = v_full + 2;   // [2]
  uint64_t* v_empty = k_empty + 2;  // [2]
  uint64_t* s_full = v_empty + 2;   // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* done = ds_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);
  QueryUnit* s_unit = reinterpret_cast<QueryUnit*>(tmem_slot + 4);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (uint64_t* b = q_full; b <= done; ++b) tc::mbar_init(b, b == ds_full ? 256 : 1);
    *bad = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(tmem_slot, 512);
  pdl_wait();
  if (warp == 0) {
    const QueryUnit found = query_unit(a, static_cast<int>(blockIdx.x));
    if (lane == 0) *s_unit = found;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const QueryUnit& u = *s_unit;
  pdl_trigger();
  // tensor memory: S of even and odd blocks 0 and 128, dP (then dS) 256, dQ 384
  const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;
  const bool work = u.any && u.b.hi > 0;
  const int kv = u.any ? u.head / p.group : 0;

  if (work && warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 9) {
      // ----------------------------------------------------------------------------------------- loads ----
      if (tc::elect_one()) {
        tc::mbar_expect_tx(q_full, kTile);
        load_tile<DP>(s_q, &tm_q, q_full, u.head, u.s.q0 + u.row);
        int n = 0;
        bool ok = true;
        for (int b = u.b.next(-1); b < u.b.hi; b = u.b.next(b), ++n) {
          const int st = n & 1, row = u.s.k0 + b * kRows;
          if (n >= 2) ok = wait(&k_empty[st], (n / 2 - 1) & 1, bad);
          if (!ok) break;
          tc::mbar_expect_tx(&k_raw[st], kTile);
          load_tile<DP>(s_k + st * kTile, &tm_k, &k_raw[st], kv, row);
          if (n == 0) {
            tc::mbar_expect_tx(do_full, kTile);
            load_tile<DP>(s_do, &tm_do, do_full, u.head, u.s.q0 + u.row);
          }
          // (values are read before the keys of their block are read for the last time: k_empty says that both are free)
          tc::mbar_expect_tx(&v_full[st], kTile);
          load_tile<DP>(s_v + st * kTile, &tm_v, &v_full[st], kv, row);
        }
        if (!ok) {   // loads that were issued must land before the block retires
          tc::mbar_wait(q_full, 0, 1u << 18);
          tc::mbar_wait(do_full, 0, 1u << 18);
          for (int i = max(0, n - 2); i < n; ++i) {
            tc::mbar_wait(&k_raw[i & 1], (i / 2) & 1, 1u << 18);
            tc::mbar_wait(&v_full[i & 1], (i / 2) & 1, 1u << 18);
          }
        }
      }
      __syncwarp();
    } else if (warp == 10) {
      // --------------------------------------------------------------- rows behind the sequence must not be NaN ----
      int n = 0;
      for (int b = u.b.next(-1); b < u.b.hi; b = u.b.next(b), ++n) {
        const int st = n & 1, rows = min(kRows, u.s.m - b * kRows);
        const bool ok = wait(&k_raw[st], (n / 2) & 1, bad);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (rows < kRows) {
          zero_rows<DP>(s_k + st * kTile, rows);
          fence_async_smem();
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&k_full[st]);
        __syncwarp();
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------------------------------- products ----
      constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false);
      const uint32_t idesc_g = idesc16<H>(kRows, (p.head_dim + 15) / 16 * 16, false, true);
      const int steps = (p.head_dim + 15) / 16;
      bool ok = true;
      auto all_wait = [&](uint64_t* bar, uint32_t parity) {
        const bool w = ok && wait(bar, parity, bad);
        ok = __all_sync(0xffffffffu, w);
        tc::fence_after_sync();
        return ok;
      };
      auto scores = [&](int n) {
        if (all_wait(&k_full[n & 1], (n / 2) & 1) && tc::elect_one()) {
          mma_rows(tmem + (n & 1) * 128, s_q, s_k + (n & 1) * kTile, idesc_s, steps);
          tc::mma_commit(&s_full[n & 1]);
        }
        __syncwarp();
      };
      auto gradients = [&](int n) {
        if (all_wait(&v_full[n & 1], (n / 2) & 1) && tc::elect_one()) {
          mma_rows(t_dp, s_do, s_v + (n & 1) * kTile, idesc_s, steps);
          tc::mma_commit(dp_full);
        }
        __syncwarp();
      };
      all_wait(q_full, 0);
      scores(0);
      all_wait(do_full, 0);
      gradients(0);
      int n = 0;
      for (int b = u.b.next(-1); b < u.b.hi && ok; ++n) {
        const int st = n & 1;
        b = u.b.next(b);
        const bool more = b < u.b.hi;
        if (more) scores(n + 1);
        if (!all_wait(ds_full, n & 1)) break;
        if (tc::elect_one()) {
          mma_weights<128, 64>(t_dq, t_dp, s_k + st * kTile, idesc_g, n > 0);
          tc::mma_commit(&k_empty[st]);
          if (!more) tc::mma_commit(done);
        }
        __syncwarp();
        if (more) gradients(n + 1);
      }
    }
  } else if (work) {
    // ----------------------------------------------------------------------- a row per thread, half of the keys ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_dp = t_dp + lanes + half * 64;
    const int pos = u.first + row, first = u.first, last = u.last;
    const Blocks blocks = u.b;
    const bool mine = u.row + row < u.s.n;
    const long long at = static_cast<long long>(u.head) * p.tokens + u.s.q0 + u.row + row;
    float lse = mine ? a.lse[at] * kLog2e : INFINITY;
    if (lse == -INFINITY) lse = INFINITY;   // sees nothing
    const float delta = mine ? a.delta[at] : 0.f;
    bool ok = true;
    int n = 0;
    for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b), ++n) {
      const bool partly = !all_seen(p, b, first, last);
      const int high = pos - b * kRows - half * 64, low = high - p.window, sink = p.sinks - b * kRows - half * 64;   // columns seen: c <= high and (c > low or c < sink)
      ok = wait(&s_full[n & 1], (n / 2) & 1, bad);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      float w[64];
      {
        uint32_t r[2][32];
        tc::tmem_ld_32x32(tmem + (n & 1) * 128 + lanes + half * 64, r[0]);
        tc::tmem_ld_32x32(tmem + (n & 1) * 128 + lanes + half * 64 + 32, r[1]);
        tc::tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 64; ++c) w[c] = exp2f(fmaf(__uint_as_float(r[c / 32][c % 32]), p.scale_log2, -lse));
      }
      ok = wait(dp_full, n & 1, bad);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc::fence_after_sync();
      uint32_t x[32];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t r[32];
        tc::tmem_ld_32x32(my_dp + 32 * g, r);
        tc::tmem_ld_wait();
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = (__uint_as_float(r[e]) - delta) * w[g * 32 + e];
        if (partly) {
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = g * 32 + e <= high && (g * 32 + e > low || g * 32 + e < sink) ? f[e] : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const H::T2 h = H::down(f[2 * e], f[2 * e + 1]);
          x[g * 16 + e] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      tmem_st32(my_dp, x);
      tmem_st_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(ds_full);
    }
    if (ok) {
      ok = wait(done, 0, bad);
      ok = __all_sync(0xffffffffu, ok);
      tc::fence_after_sync();
    }
    if (ok) {   // each half takes half of the columns out
      const long long stride = static_cast<long long>(p.heads) * p.head_dim;
      const int first_row = u.row + (warp & 3) * 32;
      H::T* to = static_cast<H::T*>(a.dq) + (u.s.q0 + first_row) * stride + u.head * p.head_dim;
      for (int c0 = half * 32; c0 < p.head_dim; c0 += 64) {
        uint32_t r[32];
        tc::tmem_ld_32x32(t_dq + lanes + c0, r);
        tc::tmem_ld_wait();
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = pos < 0 ? 0.f : __uint_as_float(r[e]) * p.scale;
        rows_out<H>(s_out + warp * 2048, f, to, stride, u.s.n - first_row, c0, p.head_dim);
      }
    }
    tc::fence_before_sync();
  } else if (u.any) {
    // these rows see nothing
    const int rows = min(kRows, u.s.n - u.row), d8 = p.head_dim / 8;
    const long long at = (static_cast<long long>(u.s.q0 + u.row) * p.heads + u.head) * p.head_dim;
    for (int i = tid; i < rows * d8; i += kThreads)
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dq) + at + static_cast<long long>(i / d8) * p.heads * p.head_dim + i % d8 * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 33);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
  zero_outside<H::T>(a.dq, p.heads * p.head_dim, nullptr, 0, p.offsets, p.sequences, p.tokens, blockIdx.x, gridDim.x, tid, kThreads);
}

template <int DP>
cudaError_t launch(const PackedAttentionGradArgs& args, cudaStream_t stream) {
  const PackedAttentionArgs& f = args.f;
  Grad g;
  g.p = problem_of(f);
  g.lse = f.lse;
  g.delta = args.delta;
  g.dq = args.dq;
  g.dk = args.dk;
  g.dv = args.dv;
  const long long keys = slots_of(f.k_tokens, f.sequences, kRows) * f.kv_heads, queries = slots_of(f.tokens, f.sequences, kRows) * f.heads;
  if (g.p.err == nullptr || keys > INT_MAX || queries > INT_MAX) return cudaErrorInvalidValue;
  CUtensorMap q, k, v, d_o;
  if (!encode_rows(&q, f.type, f.q, f.tokens, f.heads, f.head_dim) || !encode_rows(&k, f.type, f.k, f.k_tokens, f.kv_heads, f.head_dim) ||
      !encode_rows(&v, f.type, f.v, f.k_tokens, f.kv_heads, f.head_dim) || !encode_rows(&d_o, f.type, args.d_o, f.tokens, f.heads, f.head_dim))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed_keys{0}, allowed_queries{0};
  cudaError_t rc = raise_smem_limit(packed_grad_keys_kernel<DP>, key_smem<DP>(), allowed_keys);
  if (rc == cudaSuccess) rc = raise_smem_limit(packed_grad_queries_kernel<DP>, query_smem<DP>(), allowed_queries);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL(packed_delta_kernel, dim3((f.tokens + 31) / 32, (f.heads + 7) / 8), 256, 0, stream, static_cast<const H::T*>(f.o), static_cast<const H::T*>(f.o_rest),
                  args.d_o, args.delta, f.tokens, f.heads, f.head_dim);
  g.units = static_cast<int>(keys);
  MCCL_LAUNCH_PDL(packed_grad_keys_kernel<DP>, g.units, kThreads, key_smem<DP>(), stream, q, k, v, d_o, g);
  g.units = static_cast<int>(queries);
  MCCL_LAUNCH_PDL(packed_grad_queries_kernel<DP>, g.units, kThreads, query_smem<DP>(), stream, q, k, v, d_o, g);
  count_launch(3);
  return ::mccl::launch_status();
}

}  // namespace

cudaError_t packed_attention_grad(const PackedAttentionGradArgs& a, cudaStream_t stream) {
  if (a.f.tokens <= 0 || a.f.heads <= 0) return cudaSuccess;
  return a.f.head_dim <= 64 ? launch<64>(a, stream) : launch<128>(a, stream);
}

}  // namespace ops
}  // namespace mccl
