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

constexpr int kThreads = 12 * 32;   // warps 0-3 and 4-7: rows, half of the columns each; 8: products; 9: loads; 10: rows behind the sequence, statistics; 11: what comes next
// 256 x 208 + 128 x 80 of the launch's 384 x 168 registers.
constexpr int kRowRegisters = 208, kOtherRegisters = 80;
constexpr int kRoles = 8 + 3;       // warps that take a unit from the planning one

// Where the 16-bit weights (or score gradients) of a tile are in tensor memory: in columns of their own where head_dim leaves room, otherwise in those of the scores,
// each half of the threads in its own.  In the latter case the next scores (dP) are written right behind the product that reads the weights (score gradients).  Promised is the order of
// products of one shape into one accumulator; these have one shape, 128 x 128 x 16, and two accumulators, whose order is what has been seen: waits in between changed no bit of 432
// calls of 6 head dimensions (and 8192 x 16 heads over 4 of 128 took 1268 us instead of 1185).
template <int DP>
constexpr int kApart = DP == 64 ? 32 : 64;

struct Grad {
  Problem p;
  const float* lse;     // [heads, tokens]
  const float* delta;   // [heads, tokens]
  void* dq;
  void* dk;
  void* dv;
  int units;
};

// Every query sees one key: weights of one, no gradient of any score.
__device__ __forceinline__ bool one_key(const Problem& p) { return p.window == 1 && p.sinks == 0; }

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
// by 1.5 to 1.6 times what their own rounding leaves, now by 1.4).  A warp per 32 rows of a head, LANES lanes per row.
// Rows that see up to kFew keys: O's weights were rounded to 16 bits, which few keys do not even out (gradients off by 1.53 times their own rounding where rows see 2 to 4
// keys); delta is the sum of p dP itself there, from q, k and v (1.42).  Each row's own number of keys decides, not what else is in the batch; a warp finds its rows' texts by 32 probes at
// a time, the first of which are under way beside the rows.
constexpr int kFew = 8;
template <int LANES>
__global__ void __launch_bounds__(256) packed_delta_kernel(const Problem p, const H::T* o, const H::T* o_rest, TokenView q, TokenView k, TokenView v, TokenView d_o, float* delta) {
  pdl_wait();
  pdl_trigger();
  constexpr int kAtOnce = 32 / LANES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, in = lane / LANES, c = (lane % LANES) * 8;
  const int h = blockIdx.y * 8 + warp, t0 = blockIdx.x * 32, tokens = p.tokens, heads = p.heads, head_dim = p.head_dim;
  if (h >= heads) return;
  int text = 0, texts = p.sequences, step = (texts + 31) / 32;   // the last text that begins at t0 or before is one of `texts` from `text` on
  int begins = lane * step < texts ? __ldg(p.offsets + lane * step) : INT_MAX;
  float mine = 0.f;
#pragma unroll 8
  for (int i = 0; i < LANES; ++i) {
    const int t = t0 + kAtOnce * i + in;
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
    for (int s = LANES / 2; s >= 1; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
    sum = __shfl_sync(0xffffffffu, sum, (lane % kAtOnce) * LANES);
    if (lane / kAtOnce == i) mine = sum;
  }
  for (;;) {
    const int before = max(1, __popc(__ballot_sync(0xffffffffu, begins <= t0)));   // (offsets do not decrease)
    text += (before - 1) * step;
    texts = min(step, texts - (before - 1) * step);
    if (texts <= 1) break;
    step = (texts + 31) / 32;
    begins = lane * step < texts ? __ldg(p.offsets + text + lane * step) : INT_MAX;
  }
  // this lane's row: its text is the last one that begins at it or before, one of the 31 from here on or else (texts without tokens) looked for; keys first[0 .. head) and
  // from[0 .. count - head)
  int count = 0, head = 0, from = 0, first = 0;
  {
    const int t = t0 + lane, here = min(text + lane, p.sequences), begin = __ldg(p.offsets + here), k_begin = __ldg(p.k_offsets + here);
    const int later = text + lane < p.sequences ? begin : INT_MAX;
    int s = 0;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1)
      if (__shfl_sync(0xffffffffu, later, s + o) <= t) s += o;
    Sequence x;
    x.q0 = clamp(__shfl_sync(0xffffffffu, begin, s), 0, tokens);
    x.n = clamp(__shfl_sync(0xffffffffu, begin, s + 1), x.q0, tokens) - x.q0;
    x.k0 = clamp(__shfl_sync(0xffffffffu, k_begin, s), 0, p.k_tokens);
    x.m = clamp(__shfl_sync(0xffffffffu, k_begin, s + 1), x.k0, p.k_tokens) - x.k0;
    if (s == 31) {
      int lo = text + s, n = p.sequences - lo;
      while (n > 1) {
        const int half = n >> 1;
        if (__ldg(p.offsets + lo + half) <= t) lo += half, n -= half;
        else n = half;
      }
      x = sequence_of(p, lo);
    }
    const int row = t - x.q0, pos = x.m - x.n + row;
    if (t < tokens && row >= 0 && row < x.n && pos >= 0) {
      from = max(0, pos - p.window + 1);
      head = min(p.sinks, from);
      count = pos - from + 1 <= kFew && pos - from + 1 + head <= kFew ? pos - from + 1 + head : 0;
      first = x.k0;
    }
  }
  // kAtOnce of these rows at a time (one key has a weight of one, and its score no gradient)
  for (unsigned rows = __ballot_sync(0xffffffffu, count > 1); rows != 0;) {
    int of[kAtOnce], r = -1;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      of[i] = __ffs(rows) - 1;
      rows &= rows - 1;
      if (i == in) r = of[i];
    }
    const int n_ = __shfl_sync(0xffffffffu, count, max(r, 0)), n_head = __shfl_sync(0xffffffffu, head, max(r, 0)), n_from = __shfl_sync(0xffffffffu, from, max(r, 0)),
              n_first = __shfl_sync(0xffffffffu, first, max(r, 0)), n = r < 0 ? 0 : n_;
    float score[kFew] = {}, dp[kFew] = {};
    if (n > 0 && c < head_dim) {   // (all loads under way together: those of keys behind the last one are of that one again)
      const long long t = t0 + r;
      const uint4 q_raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const H::T*>(q.p) + t * q.token + h * q.head + c));
      const uint4 d_raw = __ldg(reinterpret_cast<const uint4*>(static_cast<const H::T*>(d_o.p) + t * d_o.token + h * d_o.head + c));
      uint4 k_raw[kFew], v_raw[kFew];
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        const int at = min(j, n - 1);
        const long long key = n_first + (at < n_head ? at : n_from + at - n_head);
        k_raw[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const H::T*>(k.p) + key * k.token + h / p.group * k.head + c));
        v_raw[j] = __ldg(reinterpret_cast<const uint4*>(static_cast<const H::T*>(v.p) + key * v.token + h / p.group * v.head + c));
      }
      float x[8], y[8];
      unpack8_as<H>(q_raw, x);
      unpack8_as<H>(d_raw, y);
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        float a[8], b[8];
        unpack8_as<H>(k_raw[j], a);
        unpack8_as<H>(v_raw[j], b);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          score[j] = fmaf(x[e], a[e], score[j]);
          dp[j] = fmaf(y[e], b[e], dp[j]);
        }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
#pragma unroll
      for (int s = LANES / 2; s >= 1; s >>= 1) {
        score[j] += __shfl_xor_sync(0xffffffffu, score[j], s);
        dp[j] += __shfl_xor_sync(0xffffffffu, dp[j], s);
      }
      if (j < n) top = fmaxf(top, score[j]);
    }
    float sum = 0.f, all = 0.f;
#pragma unroll
    for (int j = 0; j < kFew; ++j) {
      if (j >= n) continue;
      const float w = exp2f((score[j] - top) * p.scale_log2);
      sum = fmaf(w, dp[j], sum);
      all += w;
    }
    sum /= all;
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const float its = __shfl_sync(0xffffffffu, sum, i * LANES);
      if (lane == of[i]) mine = its;
    }
  }
  if (t0 + lane < tokens) delta[static_cast<long long>(h) * tokens + t0 + lane] = mine;
}

// ------------------------------------------------------------------------------------------------------ keys ----
// The queries that see a block of keys: tiles of 128 rows from `row` on, of each of the heads that share it.
struct KeyUnit {
  Sequence s;
  int block, kv;         // first key 128 * block
  int row, end_row, tiles;   // rows row .. end_row - 1 of the sequence, per head
  int place;             // position of a query minus its row
  bool any, end;
};
__device__ __forceinline__ KeyUnit key_unit(const Grad& a, int u) {
  const Problem& p = a.p;
  KeyUnit r;
  r.any = r.end = false;
  const int slot = u / p.kv_heads;   // a sequence's first keys have the most queries: first
  r.kv = u - slot * p.kv_heads;
  const int s = find_sequence(p.k_offsets, p.sequences, p.k_tokens, slot, kRows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  r.block = slot - (r.s.k0 / kRows + s);
  if (r.block < 0 || r.block * kRows >= r.s.m) return r;
  r.place = r.s.m - r.s.n;
  r.row = max(0, r.block * kRows - r.place);
  const int last_key = min(r.block * kRows + kRows, r.s.m) - 1;
  r.end_row = r.block * kRows < p.sinks ? r.s.n : static_cast<int>(min(static_cast<long long>(r.s.n), static_cast<long long>(last_key) + p.window - r.place));
  r.tiles = r.end_row > r.row ? (r.end_row - r.row + kRows - 1) / kRows : 0;
  r.any = r.tiles > 0;
  if (!r.any) {   // nobody sees these keys
    const int rows = last_key + 1 - r.block * kRows, d8 = p.head_dim / 8;
    const long long at = (static_cast<long long>(r.s.k0 + r.block * kRows) * p.kv_heads + r.kv) * p.head_dim;
    for (int i = threadIdx.x & 31; i < rows * d8; i += 32) {
      const long long to = at + static_cast<long long>(i / d8) * p.kv_heads * p.head_dim + i % d8 * 8;
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dk) + to) = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dv) + to) = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  return r;
}

template <int DP>
constexpr int key_smem() { return 6 * (DP / 64) * kSub + 8 * kOut + 2 * 2 * kRows * 4 + 512; }

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_grad_keys_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_out, const __grid_constant__ CUtensorMap tm_out2, const Grad a) {
  constexpr int kTile = (DP / 64) * kSub;
  extern __shared__ __align__(1024) uint8_t smem_aligned[];   // (no room to move the beginning: all but 512 bytes are in use)
  uint8_t* s_k = smem_aligned;
  uint8_t* s_v = s_k + kTile;
  uint8_t* s_q = s_v + kTile;        // [2]
  uint8_t* s_do = s_q + 2 * kTile;   // [2]
  uint8_t* s_out = s_do + 2 * kTile;   // a warp's rows on their way out
  float* s_lse = reinterpret_cast<float*>(s_out + 8 * kOut);   // [2][128], times log2 e
  float* s_delta = s_lse + 2 * kRows;                        // [2][128]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(s_delta + 2 * kRows);
  uint64_t* v_full = k_full + 1;
  uint64_t* kv_empty = v_full + 1;   // their last products are done: so are the unit's sums
  uint64_t* raw = kv_empty + 1;      // [2]: queries and gradients of a tile that ends behind the sequence: here, to be cleared there
  uint64_t* q_full = raw + 2;        // [2]
  uint64_t* q_empty = q_full + 2;    // [2]
  uint64_t* do_full = q_empty + 2;   // [2]
  uint64_t* do_empty = do_full + 2;  // [2]
  uint64_t* s_full = do_empty + 2;   // [2]: scores and the queries' statistics
  uint64_t* dp_full = s_full + 2;
  uint64_t* p_full = dp_full + 1;    // [2]: halves of each half's columns
  uint64_t* ds_full = p_full + 2;    // [2]
  uint64_t* plan_barriers = ds_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(plan_barriers + Plan::kBarriers);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [2]
  uint4* s_next = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(tmem_slot + 3) + 15) & ~static_cast<uintptr_t>(15));
  KeyUnit* s_unit = reinterpret_cast<KeyUnit*>(s_next + 1);   // [2]
  const Plan plan = Plan::at(plan_barriers, s_next, bad);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (uint64_t* b = k_full; b < plan_barriers; ++b) tc::mbar_init(b, b >= p_full ? 8 : (b == s_full || b == s_full + 1 ? 2 : 1));
    plan.init(kRoles);
    bad[0] = bad[1] = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(tmem_slot, 512);
  pdl_wait();
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  // tensor memory: S^T 0, dP^T 128, dV 256, dK 256 + DP; P^T and dS^T behind these or where the scores were
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 256 + DP, t_p = DP == 64 ? tmem + 384 : t_s, t_ds = DP == 64 ? tmem + 448 : t_dp;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 11) {
      // ------------------------------------------------------------------------------- what comes next ----
      plan.run(s_unit, [&](int id) {
        zero_outside<H::T>(a.dk, p.kv_heads * p.head_dim, nullptr, 0, p.k_offsets, p.sequences, p.k_tokens, id, a.units, lane, 32);
        zero_outside<H::T>(a.dv, p.kv_heads * p.head_dim, nullptr, 0, p.k_offsets, p.sequences, p.k_tokens, id, a.units, lane, 32);
        return key_unit(a, id);
      });
    } else if (warp == 9) {
      // ----------------------------------------------------------------------------------------- loads ----
      int n = 0;
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const KeyUnit& u = s_unit[k & 1];
        if (tc::elect_one()) {
          const int head = u.kv * p.group, first = u.s.q0 + u.row, tiles = u.tiles, key = u.s.k0 + u.block * kRows;
          const bool ragged = u.s.n - u.row < tiles * kRows;
          for (int g = 0; g < p.group && ok; ++g) {
            for (int t = 0; t < tiles && ok; ++t, ++n) {
              const int st = n & 1;
              const bool look = ragged && t + 1 == tiles, begin = g + t == 0;
              auto free = [&](uint64_t* empty) { ok = ok && (n < 2 || wait(&empty[st], (n / 2 - 1) & 1, bad)); };
              auto bring = [&](uint8_t* to, const CUtensorMap* map, uint64_t* full) {
                if (!look) tc::mbar_expect_tx(full, kTile);
                load_tile<DP>(to + st * kTile, map, look ? &raw[st] : full, head + g, first + t * kRows);
              };
              if (begin) {
                if (k > 0) ok = wait(kv_empty, (k - 1) & 1, bad);
                if (!ok) break;
                tc::mbar_expect_tx(k_full, kTile);
                load_tile<DP>(s_k, &tm_k, k_full, u.kv, key);
              }
              // gradients first, theirs is the stage that is free earlier; the first queries have nothing to wait for
              if (!begin || look) free(do_empty);
              if (begin || look) free(q_empty);
              if (!ok) break;
              if (look) tc::mbar_expect_tx(&raw[st], 2 * kTile);   // not before the stage's last use is over: a barrier counts one phase at a time
              if (begin) bring(s_q, &tm_q, &q_full[st]);
              if (begin) {
                tc::mbar_expect_tx(v_full, kTile);
                load_tile<DP>(s_v, &tm_v, v_full, u.kv, key);
                if (!look) free(do_empty);
                if (!ok) break;
              }
              bring(s_do, &tm_do, &do_full[st]);
              if (!begin) {
                if (!look) free(q_empty);
                if (!ok) break;
                bring(s_q, &tm_q, &q_full[st]);
              }
              if ((n & 15) == 0) goes_on(bad);
            }
          }
          if (!ok) {   // loads that were issued must land before the block retires
            for (uint64_t* b = k_full; b < s_full; ++b) {
              tc::mbar_wait(b, 0, 1u << 14);
              tc::mbar_wait(b, 1, 1u << 14);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        n = __reduce_max_sync(0xffffffffu, n);
        if (lane == 0) tc::mbar_arrive(plan.loads_done);
        plan.give_back(k);
      }
    } else if (warp == 10) {
      // ---------------------------------- statistics of the queries; rows behind the sequence must not be NaN ----
      int n = 0;
      uint32_t looked = 0;   // a bit per stage
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const KeyUnit& u = s_unit[k & 1];
        for (int g = 0; g < p.group && ok; ++g) {
          for (int t = 0; t < u.tiles; ++t, ++n) {
            const int st = n & 1, row = u.row + t * kRows, rows = min(kRows, u.s.n - row);
            const long long at = static_cast<long long>(u.kv * p.group + g) * p.tokens + u.s.q0 + row;
            float l[4], d[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 32 + lane;
              l[i] = r < rows ? a.lse[at + r] * kLog2e : INFINITY;
              d[i] = r < rows ? a.delta[at + r] : 0.f;
              if (l[i] == -INFINITY) l[i] = INFINITY;   // sees nothing
            }
            ok = n < 2 || wait(&q_empty[st], (n / 2 - 1) & 1, bad);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              s_lse[st * kRows + i * 32 + lane] = l[i];
              s_delta[st * kRows + i * 32 + lane] = d[i];
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s_full[st]);
            if (rows < kRows) {
              ok = wait(&raw[st], (looked >> st) & 1, bad);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              looked ^= 1u << st;
              zero_rows<DP>(s_q + st * kTile, rows);
              zero_rows<DP>(s_do + st * kTile, rows);
              fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                tc::mbar_arrive(&q_full[st]);
                tc::mbar_arrive(&do_full[st]);
              }
            }
          }
        }
        plan.give_back(k);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------------------------------- products ----
      constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false), idesc_g = idesc16<H>(kRows, DP, false, true);
      const int steps = (p.head_dim + 15) / 16;
      int n = 0;
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const int items = s_unit[k & 1].tiles * p.group;
        if (tc::elect_one()) {
          ok = wait(k_full, k & 1, bad) && wait(&q_full[n & 1], (n / 2) & 1, bad);
          if (ok) {
            mma_rows<DP>(t_s, s_k, s_q + (n & 1) * kTile, idesc_s, steps);
            tc::mma_commit(&s_full[n & 1]);
            ok = wait(v_full, k & 1, bad) && wait(&do_full[n & 1], (n / 2) & 1, bad);
          }
          if (ok) {
            mma_rows<DP>(t_dp, s_v, s_do + (n & 1) * kTile, idesc_s, steps);
            tc::mma_commit(dp_full);
          }
          for (int i = 0; i < items && ok; ++i, ++n) {
            const int st = n & 1, next = st ^ 1;
            const bool more = i + 1 < items;
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) {
              ok = wait(&p_full[h], n & 1, bad);
              tc::fence_after_sync();
              if (ok) mma_half<kApart<DP>>(t_dv, t_p, s_do + st * kTile, h, idesc_g, i + h > 0);
            }
            if (ok) tc::mma_commit(&do_empty[st]);
            if (ok && more) ok = wait(&q_full[next], ((n + 1) / 2) & 1, bad);
            if (!ok) break;
            if (more) {
              mma_rows<DP>(t_s, s_k, s_q + next * kTile, idesc_s, steps);
              tc::mma_commit(&s_full[next]);
            }
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) {
              ok = wait(&ds_full[h], n & 1, bad);
              tc::fence_after_sync();
              if (ok) mma_half<kApart<DP>>(t_dk, t_ds, s_q + st * kTile, h, idesc_g, i + h > 0);
            }
            if (ok) tc::mma_commit(&q_empty[st]);
            if (ok && more) ok = wait(&do_full[next], ((n + 1) / 2) & 1, bad);
            if (!ok) break;
            if (more) {
              mma_rows<DP>(t_dp, s_v, s_do + next * kTile, idesc_s, steps);
              tc::mma_commit(dp_full);
            } else {
              tc::mma_commit(kv_empty);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        n = __reduce_max_sync(0xffffffffu, n);
        plan.give_back(k);
      }
    }
  } else {
    // -------------------------------------------------------------------- a key per thread, half of the queries ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_s = t_s + lanes + half * 64, my_dp = t_dp + lanes + half * 64, my_p = t_p + lanes + half * kApart<DP>, my_ds = t_ds + lanes + half * kApart<DP>;
    const F2 scale2 = f2(p.scale_log2, p.scale_log2);
    int n = 0;
    bool ok = true;
    for (int k = 0; ok && plan.take(s_unit, k); ++k) {
      const KeyUnit& u = s_unit[k & 1];
      const int first_key = u.block * kRows, key = first_key + row, place = u.place + u.row + half * 64, tiles = u.tiles;
      const bool sink = key < p.sinks, all_sinks = first_key + kRows <= p.sinks;
      const int far = key > INT_MAX - p.window ? INT_MAX : key + p.window;   // the first position that does not see the key any more
      int t = 0;
      for (int i = tiles * p.group; i > 0; --i, ++n) {
        const int st = n & 1;
        const int first = place + t * kRows;   // position of my first column
        if (++t == tiles) t = 0;
        // the columns that see my key: low <= c < high
        const bool partly = !(first >= first_key + kRows - 1 && (first + 63 - p.window < first_key || all_sinks));
        const int low = key - first, high = sink ? 64 : min(64, far - first);
        // (the first position sees one key, with a weight of one: its score has no gradient, of which dP - delta would leave rounding)
        const int low_ds = key == 0 ? low + 1 : low;
        ok = wait(&s_full[st], (n / 2) & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
        float w[64];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tc::tmem_ld_32x32(my_s + 32 * h, r);
          const float4* l4 = reinterpret_cast<const float4*>(s_lse + st * kRows + half * 64 + 32 * h);
          float4 l[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) l[c] = l4[c];
          tc::tmem_ld_wait();
          uint32_t x[16];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            float* y = w + 32 * h + 4 * c;
            split(fma2(f2(__uint_as_float(r[4 * c]), __uint_as_float(r[4 * c + 1])), scale2, f2(-l[c].x, -l[c].y)), y[0], y[1]);
            split(fma2(f2(__uint_as_float(r[4 * c + 2]), __uint_as_float(r[4 * c + 3])), scale2, f2(-l[c].z, -l[c].w)), y[2], y[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = exp2f(y[e]);
          }
          if (partly) {
#pragma unroll
            for (int c = 0; c < 32; ++c) w[32 * h + c] = 32 * h + c >= low && 32 * h + c < high ? w[32 * h + c] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const H::T2 h2 = H::down(w[32 * h + 2 * e], w[32 * h + 2 * e + 1]);
            x[e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          tmem_st16(my_p + 16 * h, x);
          tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&p_full[h]);
        }
        ok = wait(dp_full, n & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tc::tmem_ld_32x32(my_dp + 32 * h, r);
          const float4* d4 = reinterpret_cast<const float4*>(s_delta + st * kRows + half * 64 + 32 * h);
          float4 d[8];
#pragma unroll
          for (int c = 0; c < 8; ++c) d[c] = d4[c];
          tc::tmem_ld_wait();
          float f[32];
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            f[4 * c] = (__uint_as_float(r[4 * c]) - d[c].x) * w[32 * h + 4 * c];
            f[4 * c + 1] = (__uint_as_float(r[4 * c + 1]) - d[c].y) * w[32 * h + 4 * c + 1];
            f[4 * c + 2] = (__uint_as_float(r[4 * c + 2]) - d[c].z) * w[32 * h + 4 * c + 2];
            f[4 * c + 3] = (__uint_as_float(r[4 * c + 3]) - d[c].w) * w[32 * h + 4 * c + 3];
          }
          if (partly) {
#pragma unroll
            for (int c = 0; c < 32; ++c) f[c] = 32 * h + c >= low_ds && 32 * h + c < high ? f[c] : 0.f;
          }
          uint32_t x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const H::T2 h2 = H::down(f[2 * e], f[2 * e + 1]);
            x[e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          tmem_st16(my_ds + 16 * h, x);
          tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&ds_full[h]);
        }
      }
      if (ok) {
        ok = wait(kv_empty, k & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
      }
      if (ok) {   // one half takes dV out, the other dK
        const uint32_t from = (half == 0 ? t_dv : t_dk) + lanes;
        const float scale = half == 0 ? 1.f : (one_key(p) ? 0.f : p.scale);
        const int first_row = first_key + (warp & 3) * 32;
#pragma unroll 1
        for (int c0 = 0; c0 < p.head_dim; c0 += 64) {
          uint32_t r[2][32];
          tc::tmem_ld_32x32(from + c0, r[0]);
          tc::tmem_ld_32x32(from + c0 + 32, r[1]);
          tc::tmem_ld_wait();
          float f[64];
#pragma unroll
          for (int e = 0; e < 64; ++e) f[e] = __uint_as_float(r[e / 32][e % 32]) * scale;
          rows_out<H>(s_out + warp * kOut, half == 0 ? &tm_out2 : &tm_out, f, half == 0 ? a.dv : a.dk, p.kv_heads, p.head_dim, u.kv, u.s.k0 + first_row, u.s.m - first_row, c0);
        }
      }
      tc::fence_before_sync();   // the next unit's first products overwrite the sums
      plan.give_back(k);
    }
    rows_sent();
    tc::fence_before_sync();
  }
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 32);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// --------------------------------------------------------------------------------------------------- queries ----
struct QueryUnit {
  Sequence s;
  int head, row, first, last;   // positions of the tile's rows
  Blocks b;
  bool any, end;
};
__device__ __forceinline__ QueryUnit query_unit(const Grad& a, int u) {
  const Problem& p = a.p;
  QueryUnit r;
  r.any = r.end = false;
  const int slots = a.units / p.heads, slot = slots - 1 - u / p.heads;   // long rows first
  r.head = u % p.heads;
  const int s = find_sequence(p.offsets, p.sequences, p.tokens, slot, kRows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  r.row = (slot - (r.s.q0 / kRows + s)) * kRows;
  if (r.row < 0 || r.row >= r.s.n) return r;
  r.first = r.s.m - r.s.n + r.row;
  r.last = min(r.first + kRows, r.s.m) - 1;
  r.b = blocks_of(p, r.first, r.last);
  r.any = r.b.hi > 0;
  if (!r.any) {   // these rows see nothing
    const int rows = min(kRows, r.s.n - r.row), d8 = p.head_dim / 8;
    const long long at = (static_cast<long long>(r.s.q0 + r.row) * p.heads + r.head) * p.head_dim;
    for (int i = threadIdx.x & 31; i < rows * d8; i += 32)
      *reinterpret_cast<uint4*>(static_cast<H::T*>(a.dq) + at + static_cast<long long>(i / d8) * p.heads * p.head_dim + i % d8 * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
  return r;
}

static_assert(key_smem<128>() <= 227 * 1024, "shared memory of a block");

template <int DP>
constexpr int query_smem() { return 6 * (DP / 64) * kSub + 8 * kOut + 512 + 1024; }

template <int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_grad_queries_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                               const __grid_constant__ CUtensorMap tm_do, const __grid_constant__ CUtensorMap tm_out, const Grad a) {
  constexpr int kTile = (DP / 64) * kSub;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;
  uint8_t* s_do = s_q + kTile;
  uint8_t* s_k = s_do + kTile;      // [2]
  uint8_t* s_v = s_k + 2 * kTile;   // [2]
  uint8_t* s_out = s_v + 2 * kTile;   // a warp's rows on their way out
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_out + 8 * kOut);
  uint64_t* do_full = q_full + 1;
  uint64_t* q_empty = do_full + 1;  // the unit's last products are done: so are its sums
  uint64_t* raw = q_empty + 1;      // [2]: keys of a block that ends behind the sequence: here, to be cleared there
  uint64_t* k_full = raw + 2;       // [2]
  uint64_t* k_empty = k_full + 2;   // [2]
  uint64_t* v_full = k_empty + 2;   // [2]
  uint64_t* v_empty = v_full + 2;   // [2]
  uint64_t* s_full = v_empty + 2;   // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;  // [2]: halves of each half's columns
  uint64_t* plan_barriers = ds_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(plan_barriers + Plan::kBarriers);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [2]
  uint4* s_next = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(tmem_slot + 3) + 15) & ~static_cast<uintptr_t>(15));
  QueryUnit* s_unit = reinterpret_cast<QueryUnit*>(s_next + 1);   // [2]
  const Plan plan = Plan::at(plan_barriers, s_next, bad);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (uint64_t* b = q_full; b < plan_barriers; ++b) tc::mbar_init(b, b >= ds_full ? 8 : 1);
    plan.init(kRoles);
    bad[0] = bad[1] = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(tmem_slot, 512);
  // No wait for the kernel before, which is the one for keys: nothing here reads what that writes or writes what it reads.  A block of this kernel begins when all blocks of that
  // one have triggered, which they do behind their own wait for delta and everything earlier: all of that has been written.  So blocks of this kernel fill the SMs that the other's
  // last units leave (8192 tokens of 16 heads over 4 of 128, all gradients: 847 -> 800 us; windows of 1024, 4 texts up to 8192 of 8 heads over 4: 534 -> 434).  Its own end waits for
  // the other's, so that what comes later finds both done.
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  pdl_trigger();
  // tensor memory: S of even and odd blocks 0 and 128, dP 256, dQ 384; dS behind it or where dP was
  const uint32_t t_dp = tmem + 256, t_dq = tmem + 384, t_ds = DP == 64 ? tmem + 448 : t_dp;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 11) {
      // ------------------------------------------------------------------------------- what comes next ----
      plan.run(s_unit, [&](int id) {
        zero_outside<H::T>(a.dq, p.heads * p.head_dim, nullptr, 0, p.offsets, p.sequences, p.tokens, id, a.units, lane, 32);
        return query_unit(a, id);
      });
    } else if (warp == 9) {
      // ----------------------------------------------------------------------------------------- loads ----
      int n = 0;
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const QueryUnit& u = s_unit[k & 1];
        if (tc::elect_one()) {
          const Blocks blocks = u.b;
          const int kv = u.head / p.group, begin = blocks.next(-1);
          for (int b = begin; b < blocks.hi; b = blocks.next(b), ++n) {
            const int st = n & 1, row = u.s.k0 + b * kRows;
            const bool look = u.s.m - b * kRows < kRows;
            if (b == begin) {
              if (k > 0) ok = wait(q_empty, (k - 1) & 1, bad);
              if (!ok) break;
              tc::mbar_expect_tx(q_full, kTile);
              load_tile<DP>(s_q, &tm_q, q_full, u.head, u.s.q0 + u.row);
            }
            ok = n < 2 || wait(&k_empty[st], (n / 2 - 1) & 1, bad);
            if (!ok) break;
            uint64_t* full = look ? &raw[st] : &k_full[st];
            tc::mbar_expect_tx(full, kTile);
            load_tile<DP>(s_k + st * kTile, &tm_k, full, kv, row);
            if (b == begin) {
              tc::mbar_expect_tx(do_full, kTile);
              load_tile<DP>(s_do, &tm_do, do_full, u.head, u.s.q0 + u.row);
            }
            ok = n < 2 || wait(&v_empty[st], (n / 2 - 1) & 1, bad);
            if (!ok) break;
            tc::mbar_expect_tx(&v_full[st], kTile);
            load_tile<DP>(s_v + st * kTile, &tm_v, &v_full[st], kv, row);
            if ((n & 15) == 0) goes_on(bad);
          }
          if (!ok) {   // loads that were issued must land before the block retires
            for (uint64_t* b = q_full; b < s_full; ++b) {
              tc::mbar_wait(b, 0, 1u << 14);
              tc::mbar_wait(b, 1, 1u << 14);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        n = __reduce_max_sync(0xffffffffu, n);
        if (lane == 0) tc::mbar_arrive(plan.loads_done);
        plan.give_back(k);
      }
    } else if (warp == 10) {
      // --------------------------------------------------------------- rows behind the sequence must not be NaN ----
      int n = 0;
      uint32_t looked = 0;   // a bit per stage
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const QueryUnit& u = s_unit[k & 1];
        for (int b = u.b.next(-1); b < u.b.hi; b = u.b.next(b), ++n) {
          const int st = n & 1, rows = u.s.m - b * kRows;
          if (rows >= kRows) continue;
          ok = wait_unit(&raw[st], (looked >> st) & 1, bad);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          looked ^= 1u << st;
          zero_rows<DP>(s_k + st * kTile, rows);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&k_full[st]);
        }
        plan.give_back(k);
      }
    } else if (warp == 8) {
      // -------------------------------------------------------------------------------------- products ----
      constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false), idesc_g = idesc16<H>(kRows, DP, false, true);
      const int steps = (p.head_dim + 15) / 16;
      int n = 0;
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const Blocks blocks = s_unit[k & 1].b;
        if (tc::elect_one()) {
          auto scores = [&](int n) {
            ok = ok && wait(&k_full[n & 1], (n / 2) & 1, bad);
            if (!ok) return;
            mma_rows<DP>(tmem + (n & 1) * 128, s_q, s_k + (n & 1) * kTile, idesc_s, steps);
            tc::mma_commit(&s_full[n & 1]);
          };
          ok = wait(q_full, k & 1, bad);
          scores(n);
          ok = ok && wait(do_full, k & 1, bad);
          bool begun = false;
          for (int b = blocks.next(-1); b < blocks.hi && ok; ++n) {
            const int st = n & 1;
            b = blocks.next(b);
            const bool more = b < blocks.hi;
            ok = wait(&v_full[st], (n / 2) & 1, bad);
            if (!ok) break;
            tc::fence_after_sync();
            mma_rows<DP>(t_dp, s_do, s_v + st * kTile, idesc_s, steps);
            tc::mma_commit(dp_full);
            tc::mma_commit(&v_empty[st]);
            if (more) scores(n + 1);
#pragma unroll 1
            for (int h = 0; h < 2 && ok; ++h) {
              ok = wait(&ds_full[h], n & 1, bad);
              tc::fence_after_sync();
              if (ok) mma_half<kApart<DP>>(t_dq, t_ds, s_k + st * kTile, h, idesc_g, begun || h > 0);
            }
            if (!ok) break;
            begun = true;
            tc::mma_commit(&k_empty[st]);
            if (!more) tc::mma_commit(q_empty);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        n = __reduce_max_sync(0xffffffffu, n);
        plan.give_back(k);
      }
    }
  } else {
    // ----------------------------------------------------------------------- a row per thread, half of the keys ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    const int half = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t my_dp = t_dp + lanes + half * 64, my_ds = t_ds + lanes + half * kApart<DP>;
    const F2 scale2 = f2(p.scale_log2, p.scale_log2);
    int n = 0;
    bool ok = true;
    for (int k = 0; ok && plan.take(s_unit, k); ++k) {
      const QueryUnit& u = s_unit[k & 1];
      const int pos = u.first + row, first = u.first, last = u.last;
      const Blocks blocks = u.b;
      const bool mine = u.row + row < u.s.n;
      const long long at = static_cast<long long>(u.head) * p.tokens + u.s.q0 + u.row + row;
      float lse = mine ? a.lse[at] * kLog2e : INFINITY;
      if (lse == -INFINITY || ((pos == 0 || one_key(p)) && lse == lse)) lse = INFINITY;   // sees nothing, or one key, whose score has no gradient
      const float delta = mine ? a.delta[at] : 0.f;
      const F2 lse2 = f2(-lse, -lse);
      for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b), ++n) {
        const bool partly = !all_seen(p, b, first, last);
        const int high = pos - b * kRows - half * 64, low = high - p.window, sink = p.sinks - b * kRows - half * 64;   // columns seen: c <= high and (c > low or c < sink)
        ok = wait(&s_full[n & 1], (n / 2) & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
        float w[64];
        {
          uint32_t r[2][32];
          tc::tmem_ld_32x32(tmem + (n & 1) * 128 + lanes + half * 64, r[0]);
          tc::tmem_ld_32x32(tmem + (n & 1) * 128 + lanes + half * 64 + 32, r[1]);
          tc::tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 64; c += 2) {
            split(fma2(f2(__uint_as_float(r[c / 32][c % 32]), __uint_as_float(r[c / 32][c % 32 + 1])), scale2, lse2), w[c], w[c + 1]);
            w[c] = exp2f(w[c]);
            w[c + 1] = exp2f(w[c + 1]);
          }
        }
        ok = wait(dp_full, n & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
          tc::tmem_ld_32x32(my_dp + 32 * h, r);
          tc::tmem_ld_wait();
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] = (__uint_as_float(r[e]) - delta) * w[h * 32 + e];
          if (partly) {
#pragma unroll
            for (int e = 0; e < 32; ++e) f[e] = h * 32 + e <= high && (h * 32 + e > low || h * 32 + e < sink) ? f[e] : 0.f;
          }
          uint32_t x[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const H::T2 h2 = H::down(f[2 * e], f[2 * e + 1]);
            x[e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          tmem_st16(my_ds + 16 * h, x);
          tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&ds_full[h]);
        }
      }
      if (ok) {
        ok = wait(q_empty, k & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
      }
      if (ok) {   // each half takes half of the columns out
        const int first_row = u.row + (warp & 3) * 32, c0 = 64 * half;
        if (c0 < p.head_dim) {
          uint32_t r[2][32];
          tc::tmem_ld_32x32(t_dq + lanes + c0, r[0]);
          tc::tmem_ld_32x32(t_dq + lanes + c0 + 32, r[1]);
          tc::tmem_ld_wait();
          float f[64];
#pragma unroll
          for (int e = 0; e < 64; ++e) f[e] = pos < 0 ? 0.f : __uint_as_float(r[e / 32][e % 32]) * p.scale;
          rows_out<H>(s_out + warp * kOut, &tm_out, f, a.dq, p.heads, p.head_dim, u.head, u.s.q0 + first_row, u.s.n - first_row, c0);
        }
      }
      tc::fence_before_sync();   // the next unit's first products overwrite the sums
      plan.give_back(k);
    }
    rows_sent();
    tc::fence_before_sync();
  }
  pdl_wait();   // (see above)
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 33);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
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
  CUtensorMap q, k, v, d_o, dq, dk, dv;
  if (!encode_rows(&q, f.type, f.q, f.tokens, f.heads, f.head_dim) || !encode_rows(&k, f.type, f.k, f.k_tokens, f.kv_heads, f.head_dim) ||
      !encode_rows(&v, f.type, f.v, f.k_tokens, f.kv_heads, f.head_dim) || !encode_rows(&d_o, f.type, args.d_o, f.tokens, f.heads, f.head_dim) ||
      !encode_result(&dq, f.type, args.dq, f.tokens, f.heads, f.head_dim) || !encode_result(&dk, f.type, args.dk, f.k_tokens, f.kv_heads, f.head_dim) ||
      !encode_result(&dv, f.type, args.dv, f.k_tokens, f.kv_heads, f.head_dim))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed_keys{0}, allowed_queries{0};
  cudaError_t rc = raise_smem_limit(packed_grad_keys_kernel<DP>, key_smem<DP>(), allowed_keys);
  if (rc == cudaSuccess) rc = raise_smem_limit(packed_grad_queries_kernel<DP>, query_smem<DP>(), allowed_queries);
  if (rc != cudaSuccess) return rc;
  const dim3 groups((f.tokens + 31) / 32, (f.heads + 7) / 8);
  MCCL_LAUNCH_PDL(packed_delta_kernel<DP / 8>, groups, 256, 0, stream, g.p, static_cast<const H::T*>(f.o), static_cast<const H::T*>(f.o_rest), f.q, f.k, f.v, args.d_o, args.delta);
  g.units = static_cast<int>(keys);
  MCCL_LAUNCH_PDL(packed_grad_keys_kernel<DP>, g.units, kThreads, key_smem<DP>(), stream, q, k, v, d_o, dk, dv, g);
  g.units = static_cast<int>(queries);
  MCCL_LAUNCH_PDL(packed_grad_queries_kernel<DP>, g.units, kThreads, query_smem<DP>(), stream, q, k, v, d_o, dq, g);
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
