// Causal attention of packed sequences, forward, on the 5th-generation tensor cores.
//
// A block has two tiles of 128 queries that read the same keys and values: the same rows of two query heads that share them, or 256
// neighbouring rows of one head.  Per tile and block of 128 keys:
//   S = Q K^T (tcgen05, operands in shared memory, sums in tensor memory)
//   m' = max(m, rowmax S),  P = exp2((S - m') c),  l = l 2^((m - m') c) + sum P,  O = O 2^((m - m') c) + P V
// P goes to tensor memory in 16 bits (columns of S, or its own where there are some) and is the left operand of the second product from there, so no weight passes through shared memory.
// One warpgroup per tile has a row per thread; one warp issues the products of both tiles in turn, so that the tensor cores work on one
// tile while the other's exponentials are computed; one warp brings tiles by TMA; one looks after blocks that not every row sees in whole;
// one finds out what the block does next: a block stays, and takes units of two tiles as long as there are any, the long ones first.
//
// What bounds it: a block of 128 x 128 scores of 128 columns takes the tensor cores some 1024 clocks in both products, and its 16384 exponentials take the special
// function units as long, behind which the threads of a tile have maxima, differences and conversions to do; two tiles in turn reach three quarters of the rate of a library
// product (16381 tokens of 32 heads over 8 of 128: 1.73 ms, 1270 TFLOP/s; 2.0 ms where calls follow one another and the card's power is drawn).  A step of both tiles takes
// 3400 clocks; per tile 200 until the scores are in registers, 500 for the maximum, 720 for each half of the exponentials, 1250 for the product with V and the next scores.
// One thread with all products, which waits once a step, and blocks that stay: with two such threads and a unit per block 2.54 ms.  Results by TMA: 8 texts of 2048 tokens, 16
// heads of 128, 171 us, 190 from registers.
#include "packed_tiles.cuh"

#include "smem_limit.hpp"

#include <climits>

namespace mccl {
namespace ops {

namespace {

using namespace packed;

constexpr int kStages = 2;                 // pairs of tiles under way: values of a block and keys of the next one, which are used together
constexpr int kThreads = 12 * 32;          // warps 0-3 and 4-7: rows of tiles 0 and 1; 8: products; 9: loads; 10: blocks seen in part; 11: what comes next
// A row's scores need more registers than an even share: 256 x 208 + 128 x 80 of the launch's 384 x 168.
constexpr int kRowRegisters = 208, kOtherRegisters = 80;
constexpr int kRoles = 8 + 3;              // warps that take a unit from the planning one

struct Forward {
  Problem p;
  void* o;
  void* o_rest;      // may be null
  float* lse;
  TokenView v;       // for values that are not finite
  int pair_heads;    // a block's tiles are two heads, otherwise two times 128 rows
  int head_units;    // blocks per slot
  int units;
  int parts;         // blocks that share out a unit's keys; with more than one, results go here:
  float* part_o;     // [parts, tokens, heads, head_dim]
  float* part_lse;   // [parts, heads, tokens]
};

template <int DP>
constexpr int smem_bytes() { return (2 + 2 * kStages) * (DP / 64) * kSub + 8 * kOut + 512 + 1024; }

// Weights are kept 2^kBias times larger in fp16: below 2^-21 they are subnormal there and off by 2^-32 at most, which over 2^17 keys is 2^-15 of the sum.  The running
// maximum may be exceeded by 2^kSlack before sums are rescaled (exact in fp32 either way), so that the largest weight is 2^8 in bf16 and 2^15 in fp16.  (With 2^11 and
// 2^4, windows of 1024 and 4 first positions, 4 texts up to 8192 of 16 heads over 4 of 128, took 317 us in fp16: a window's first block is seen in part, and its maximum
// is soon passed.  With 2^7 and 2^8 251.)
template <typename H>
struct Weights {
  static constexpr float kBias = 0.f, kSlack = 8.f;
};
template <>
struct Weights<Fp16> {
  static constexpr float kBias = 7.f, kSlack = 8.f;
};

// The tiles of a unit.
struct Unit {
  Sequence s;
  int row[2], head[2];       // first row within the sequence; row >= s.n: nothing
  int first[2], last[2];     // positions of the tile's rows
  Blocks b[2], all;
  int seen_from, seen_below, seen_first;
  int part;
  bool any, end;
  int odd;                   // values that are not finite were met
  // Whether all rows of the unit see all keys of a block.
  __device__ __forceinline__ bool whole(int block) const { return block < seen_below && (block >= seen_from || block < seen_first); }
};
__device__ __forceinline__ Unit unit_of(const Forward& a, int u) {
  const Problem& p = a.p;
  const int rows = a.pair_heads ? kRows : 2 * kRows;
  const int slots = a.units / a.parts / a.head_units, part = u % a.parts;
  u /= a.parts;
  const int in = u % a.head_units, slot = slots - 1 - u / a.head_units;   // long rows first
  Unit r;
  r.any = r.end = false;
  r.odd = 0;
  const int s = find_sequence(p.offsets, p.sequences, p.tokens, slot, rows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  const int row = (slot - (r.s.q0 / rows + s)) * rows;
  if (row < 0 || row >= r.s.n) return r;
  r.any = true;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (a.pair_heads) {
      const int pairs = (p.group + 1) / 2, kv = in / pairs, head = 2 * (in - kv * pairs) + t;
      r.row[t] = head < p.group ? row : r.s.n;   // (of an odd number the last one is alone)
      r.head[t] = kv * p.group + head;
    } else {
      r.row[t] = row + t * kRows;
      r.head[t] = in;
    }
    r.first[t] = r.s.m - r.s.n + r.row[t];
    r.last[t] = min(r.first[t] + kRows, r.s.m) - 1;
    r.b[t] = r.row[t] < r.s.n ? blocks_of(p, r.first[t], r.last[t]) : Blocks{0, 0, 0};
  }
  r.part = part;
  if (a.parts > 1) {
    // an even share of the blocks from the first one that either tile's last positions see on; the first positions' blocks go with the first share
    const int lo = r.b[1].hi == 0 ? r.b[0].lo : (r.b[0].hi == 0 ? r.b[1].lo : min(r.b[0].lo, r.b[1].lo)), hi = max(r.b[0].hi, r.b[1].hi), count = hi - lo;
    const int from = lo + static_cast<int>(static_cast<long long>(count) * part / a.parts), to = lo + static_cast<int>(static_cast<long long>(count) * (part + 1) / a.parts);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      Blocks& b = r.b[t];
      const int first = max(b.lo, from), last = min(b.hi, to);
      if (part > 0) b.sink = 0;
      if (first < last) b = {min(b.sink, first), first, last};
      else if (b.sink > 0) b = {b.sink, max(b.sink, from), max(b.sink, from)};   // none but the first positions' (and no run of blocks up to the other tile's)
      else b = {0, 0, 0};
    }
  }
  r.all.hi = max(r.b[0].hi, r.b[1].hi);
  r.all.lo = r.b[1].hi == 0 ? r.b[0].lo : (r.b[0].hi == 0 ? r.b[1].lo : min(r.b[0].lo, r.b[1].lo));
  r.all.sink = max(r.b[0].sink, r.b[1].sink);
  if (r.all.sink >= r.all.lo) r.all.sink = r.all.lo = 0;   // one run
  const bool both = r.b[1].hi > 0, only = r.b[0].hi == 0;   // tiles that have blocks: the last one always does if any
  const int from = only ? r.first[1] : r.first[0], to = both ? r.last[1] : r.last[0];
  r.seen_below = from < 0 ? 0 : (from + 1) / kRows;                                      // keys up to the first position
  r.seen_from = to < p.window ? 0 : (to - p.window) / kRows + 1;                         // keys within the last position's window
  r.seen_first = min(p.sinks, 1 << 30) / kRows;
  return r;
}

// The columns, of 64 from c0 on, in which a value that a row of the text sees in one of the blocks that were looked at is not finite.
template <typename H>
__device__ __noinline__ unsigned long long odd_columns(const Problem& p, const TokenView& v, const Unit& u, const Blocks& blocks, int pos, int c0) {
  unsigned long long marks = 0;
  const typename H::T* from = static_cast<const typename H::T*>(v.p) + u.head[0] / p.group * v.head + static_cast<long long>(u.s.k0) * v.token + c0;
  for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b)) {
    if (u.whole(b)) continue;
    const BlockKeys keys = block_keys(b, pos, u.s.m);
    for (int j = keys.first; j < keys.end; ++j) {
      if (j <= pos - p.window && j >= p.sinks) continue;
      for (int e = 0; e < 64 && c0 + e < p.head_dim; ++e)
        if (!(fabsf(H::up(from[j * v.token + e])) < INFINITY)) marks |= 1ull << e;
    }
  }
  return marks;
}

template <typename H, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const __grid_constant__ CUtensorMap tm_o, const __grid_constant__ CUtensorMap tm_rest, const Forward a) {
  constexpr int kTile = (DP / 64) * kSub;
  constexpr uint32_t kP = DP == 64 ? 384 : 0, kPStep = DP == 64 ? 64 : 128;   // columns of the weights
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;                        // [2] tiles
  uint8_t* s_kv = s_q + 2 * kTile;            // [kStages][2] tiles: values, keys
  uint8_t* s_out = s_kv + 2 * kStages * kTile;   // a warp's rows on their way out
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_out + 8 * kOut);   // [2]
  uint64_t* kv_full = q_full + 2;             // [kStages]
  uint64_t* kv_empty = kv_full + kStages;     // [kStages]
  uint64_t* raw_full = kv_empty + kStages;    // [kStages]: values that are looked at before they are used are here, ...
  uint64_t* looked = raw_full + kStages;      // [kStages]: ... and have been
  uint64_t* s_full = looked + kStages;        // [2]
  uint64_t* p_full = s_full + 2;              // [2][2]: tile, half of a block's keys
  uint64_t* o_full = p_full + 4;              // [2]
  uint64_t* q_empty = o_full + 2;
  uint64_t* plan_barriers = q_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(plan_barriers + Plan::kBarriers);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);   // [2]
  uint4* s_next = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(tmem_slot + 3) + 15) & ~static_cast<uintptr_t>(15));
  Unit* s_unit = reinterpret_cast<Unit*>(s_next + 1);   // [2]
  const Plan plan = Plan::at(plan_barriers, s_next, bad);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&q_full[t], 1);
      tc::mbar_init(&s_full[t], 1);
      for (int h = 0; h < 2; ++h) tc::mbar_init(&p_full[2 * t + h], 4);
      tc::mbar_init(&o_full[t], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
      tc::mbar_init(&raw_full[i], 1);
      tc::mbar_init(&looked[i], 1);
    }
    tc::mbar_init(q_empty, 1);
    tc::tma_prefetch_desc(&tm_q);
    tc::tma_prefetch_desc(&tm_k);
    tc::tma_prefetch_desc(&tm_v);
    tc::tma_prefetch_desc(&tm_o);
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
  // tensor memory: S of tile t in columns 128 t .. 128 t + 127, O in 256 + DP t .., P in 384 + 64 t .. where O leaves room for it.  Otherwise P is in the first 64
  // columns of S, and the next scores are written there right behind the product that reads it.  What is promised is the order of products of one shape into one accumulator; these
  // have one shape (128 x 128 x 16) and two accumulators, and that they too are carried out as they were issued is what has been seen: with a wait for the product with V in between
  // 864 calls of 6 head dimensions gave the same bits, and 16381 x 32 heads over 8 took 2.16 ms instead of 1.99.  (Of different shapes they are not: 128 x 64 behind 128 x 128
  // overwrote weights that were still to be read.)
  // Each role takes the units as they come; what they share in stages and phases goes on from one to the next, so that the loads and first products of a unit
  // are under way while the results of the one before are on their way out.
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
    if (warp == 11) {
      // ----------------------------------------------------------------------------------- what comes next ----
      plan.run(s_unit, [&](int id) {
        if (a.parts == 1) {
          zero_outside<typename H::T>(a.o, p.heads * p.head_dim, a.lse, p.heads, p.offsets, p.sequences, p.tokens, id, a.units, lane, 32);
        } else {
          const int width = p.heads * p.head_dim;   // (of floats: two 16-bit numbers each)
          for (int i = 0; i < a.parts; ++i)
            zero_outside<uint16_t>(a.part_o + static_cast<long long>(i) * p.tokens * width, 2 * width, a.part_lse + static_cast<long long>(i) * p.tokens * p.heads, p.heads, p.offsets,
                                   p.sequences, p.tokens, id, a.units, lane, 32);
        }
        return unit_of(a, id);
      });
    } else if (warp == 9) {
      // ------------------------------------------------------------------------------------------- loads ----
      uint32_t raw_uses = 0, q_uses = 0;   // a bit per stage, a bit per tile
      int i = 0, units = 0;                // steps, and units with keys, so far
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const Unit& u = s_unit[k & 1];
        if (tc::elect_one()) {
          const int kv = u.head[0] / p.group;
          if (u.all.hi > 0) {
            if (units > 0) ok = wait(q_empty, (units - 1) & 1, bad);
            ++units;
          }
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (ok && u.b[t].hi > 0) {
              tc::mbar_expect_tx(&q_full[t], kTile);
              load_tile<DP>(s_q + t * kTile, &tm_q, &q_full[t], u.head[t], u.s.q0 + u.row[t]);
              q_uses ^= 1u << t;
            }
          // a step brings the values of the block before and the keys of the next one
          for (int before = -1, b = u.all.next(-1); ok && (b < u.all.hi || before >= 0); ++i) {
            const int st = i % kStages;
            const bool more = b < u.all.hi, look = before >= 0 && !u.whole(before);
            if (i >= kStages) ok = wait(&kv_empty[st], (i / kStages - 1) & 1, bad);
            if (!ok) break;
            tc::mbar_expect_tx(&kv_full[st], (more ? kTile : 0) + (before >= 0 && !look ? kTile : 0));
            if (before >= 0) {
              if (look) {
                tc::mbar_expect_tx(&raw_full[st], kTile);
                raw_uses ^= 1u << st;
              }
              load_tile<DP>(s_kv + 2 * st * kTile, &tm_v, look ? &raw_full[st] : &kv_full[st], kv, u.s.k0 + before * kRows);
            }
            if (more) load_tile<DP>(s_kv + (2 * st + 1) * kTile, &tm_k, &kv_full[st], kv, u.s.k0 + b * kRows);
            if ((i & 15) == 0) goes_on(bad);
            before = more ? b : -1;
            if (more) b = u.all.next(b);
          }
          if (!ok) {   // loads that were issued must land before the block retires
            for (int t = 0; t < 2; ++t) tc::mbar_wait(&q_full[t], ((q_uses >> t) & 1) ^ 1, 1u << 16);
            for (int j = max(0, i - kStages); j < i; ++j) {
              const int st = j % kStages;
              tc::mbar_wait(&kv_full[st], (j / kStages) & 1, 1u << 16);
              tc::mbar_wait(&raw_full[st], ((raw_uses >> st) & 1) ^ 1, 1u << 16);
            }
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (lane == 0) tc::mbar_arrive(plan.loads_done);
        plan.give_back(k);
      }
    } else if (warp == 10) {
      // --------------------------------------------------------- blocks of keys that not every row sees ----
      // A weight of zero times a value that is not finite would be NaN in rows that do not see the value: such values become zeros, and rows that do see
      // them are put right at the end.  Rows behind the sequence are another sequence's.
      int steps = 0;
      uint32_t phase = 0;   // a bit per stage
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const Unit& u = s_unit[k & 1];
        int i = steps + 1;
        for (int b = u.all.next(-1); b < u.all.hi; b = u.all.next(b), ++i) {
          if (u.whole(b)) continue;
          const int st = i % kStages, rows = min(kRows, u.s.m - b * kRows);
          ok = wait_unit(&raw_full[st], (phase >> st) & 1, bad);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          phase ^= 1u << st;
          uint8_t* tile = s_kv + 2 * st * kTile;
          using T2 = typename H::T2;
          const T2 zero = H::down(0.f, 0.f);
          T2 sum = zero;   // products with zero add up to zero, or to NaN
#pragma unroll 4
          for (int i = lane; i < kTile / 16; i += 32) {
            const int r = (i / 8) % kRows;
            uint4* at = reinterpret_cast<uint4*>(tile + i * 16);
            if (r < rows) {
              const uint4 x = *at;
              const T2* h = reinterpret_cast<const T2*>(&x);
#pragma unroll
              for (int e = 0; e < 4; ++e) sum = __hfma2(h[e], zero, sum);
            } else {
              *at = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          const float2 s2 = H::up(sum);
          if (__any_sync(0xffffffffu, !(s2.x == 0.f && s2.y == 0.f))) {
            for (int i = lane; i < kTile / 16; i += 32) {
              if ((i / 8) % kRows >= rows) continue;
              uint4* at = reinterpret_cast<uint4*>(tile + i * 16);
              uint4 x = *at;
              uint16_t* e = reinterpret_cast<uint16_t*>(&x);
              constexpr uint16_t kExponent = std::is_same<H, Bf16>::value ? 0x7f80 : 0x7c00;
#pragma unroll
              for (int k = 0; k < 8; ++k) e[k] = (e[k] & kExponent) == kExponent ? static_cast<uint16_t>(0) : e[k];
              *at = x;
            }
            if (lane == 0) *reinterpret_cast<volatile int*>(&s_unit[k & 1].odd) = 1;
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&looked[st]);
        }
        if (u.all.hi > 0) steps = i;   // a step more than blocks
        plan.give_back(k);
      }
    } else if (warp == 8) {
      // ---------------------------------------------------------------------------------------- products ----
      // One thread.  What it does between the last product of one tile and the first of the other has some 500 clocks, the time of those under way; a barrier's
      // state takes 250 while the products read shared memory.  Hence one barrier for values and keys of a step, and nothing else on the way.
      constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false);
      constexpr uint32_t idesc_o = idesc16<H>(kRows, DP, false, true);   // (columns behind head_dim are zeros: TMA fills them in)
      const int steps = (p.head_dim + 15) / 16;
      uint32_t q_phase = 0, p_phase = 0, looked_phase = 0;   // a bit per tile; the last: per stage
      int i = 0;                                             // steps so far
      bool ok = true;
      for (int k = 0; ok && plan.take(s_unit, k); ++k) {
        const Unit m = s_unit[k & 1];
        if (tc::elect_one()) {
          uint32_t begun = 0;
          bool look = false;
          for (int before = -1, b = m.all.next(-1); b < m.all.hi || before >= 0; ++i) {
            const int st = i % kStages;
            const bool more = b < m.all.hi;
            ok = wait(&kv_full[st], (i / kStages) & 1, bad);
            if (look) {
              ok = ok && wait(&looked[st], (looked_phase >> st) & 1, bad);
              looked_phase ^= 1u << st;
            }
            if (!ok) break;
#pragma unroll 1
            for (int t = 0; t < 2; ++t) {
              const Blocks mine = t == 0 ? m.b[0] : m.b[1];
              if (before >= 0 && mine.has(before)) {
#pragma unroll 1
                for (int h = 0; h < 2; ++h) {   // the first half of the weights is multiplied while the second is made
                  ok = ok && wait(&p_full[2 * t + h], (p_phase >> t) & 1, bad);
                  if (!ok) break;
                  tc::fence_after_sync();
                  mma_weights<64>(tmem + 256 + t * DP, tmem + kP + kPStep * t + 32 * h, s_kv + 2 * st * kTile + h * 64 * 128, idesc_o, h != 0 || ((begun >> t) & 1));
                }
                p_phase ^= 1u << t;
                begun |= 1u << t;
              } else if (more && mine.has(b) && ((begun >> t) & 1) == 0) {
                ok = ok && wait(&q_full[t], (q_phase >> t) & 1, bad);
                q_phase ^= 1u << t;
              }
              if (!ok) break;
              if (more && mine.has(b)) {
                tc::fence_after_sync();
                mma_rows<DP>(tmem + t * 128, s_q + t * kTile, s_kv + (2 * st + 1) * kTile, idesc_s, steps);
                tc::mma_commit(&s_full[t]);
              }
              if (before >= 0 && mine.has(before)) tc::mma_commit(&o_full[t]);
            }
            if (!ok) break;
            tc::mma_commit(&kv_empty[st]);
            look = more && !m.whole(b);
            before = more ? b : -1;
            if (more) b = m.all.next(b);
            if (more && b >= m.all.hi) tc::mma_commit(q_empty);   // those were the last scores
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        plan.give_back(k);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    // ------------------------------------------------------------------------------------------ a row per thread ----
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = lane_base + t * 128, t_o = lane_base + 256 + t * DP, t_p = lane_base + kP + kPStep * t;
    const F2 scale2 = f2(p.scale_log2, p.scale_log2);
    uint32_t phase = 0;   // of the next S
    int total = 0;        // blocks so far, of all units
    bool ok = true;
    for (int k = 0; ok && plan.take(s_unit, k); ++k) {
      const Unit& u = s_unit[k & 1];
      const int pos = u.first[t] + row, first = u.first[t], last = u.last[t];
      const Blocks blocks = u.b[t];
      float m = -INFINITY, l = 0.f;
      bool sees = false;
      int done = 0;         // blocks so far
      for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b), phase ^= 1) {
        ok = wait(&s_full[t], phase, bad);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::fence_after_sync();
        float s[128];
        {
          uint32_t r[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tc::tmem_ld_32x32(t_s + 32 * c, r[c]);
          tc::tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(r[c / 32][c % 32]);
        }
        if (all_seen(p, b, first, last)) {
          sees = true;
        } else {
          const int high = pos - b * kRows, low = high - p.window, sink = p.sinks - b * kRows;   // columns seen: c <= high and (c > low or c < sink)
          sees = sees || (high >= 0 && (low < min(high, kRows - 1) || sink > 0));
#pragma unroll
          for (int c = 0; c < 128; ++c) s[c] = c <= high && (c > low || c < sink) ? s[c] : -INFINITY;
        }
        float m8[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m8[i] = fmaxf(s[2 * i], s[2 * i + 1]);
#pragma unroll
        for (int c = 16; c < 128; c += 16) {
#pragma unroll
          for (int i = 0; i < 8; ++i) m8[i] = max3(m8[i], s[c + 2 * i], s[c + 2 * i + 1]);
        }
        const float mx = max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), fmaxf(m8[6], m8[7]));
        // a row's maximum stays until it is passed by 2^kSlack.  (Each row's own: its bits do not depend on what else is in the tile.)
        const bool raise = (mx - m) * p.scale_log2 > Weights<H>::kSlack || (m == -INFINITY && mx > m);
        if (__any_sync(0xffffffffu, raise)) {
          const float next = raise ? mx : m, f = raise ? (m == -INFINITY ? 0.f : exp2f((m - next) * p.scale_log2)) : 1.f;
          if (done > 0) {
            ok = wait(&o_full[t], (total - 1) & 1, bad);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc::fence_after_sync();
#pragma unroll 1
            for (int c = 0; c < DP / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + 16 * c, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(t_o + 16 * c, o);
            }
          }
          l *= f;
          m = next;
        }
        const float base = (m == -INFINITY ? 0.f : m * p.scale_log2) - Weights<H>::kBias;
        const F2 base2 = f2(-base, -base);
        F2 sums[4] = {f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            float lo, hi;
            split(fma2(f2(s[64 * h + 2 * e], s[64 * h + 2 * e + 1]), scale2, base2), lo, hi);
            lo = exp2f(lo);
            hi = exp2f(hi);
            sums[e & 3] = add2(sums[e & 3], f2(lo, hi));
            const typename H::T2 h2 = H::down(lo, hi);
            w[e] = *reinterpret_cast<const uint32_t*>(&h2);
          }
          tmem_st32(t_p + 32 * h, w);
          tmem_st_wait();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&p_full[2 * t + h]);
        }
        float sum, other;
        split(add2(add2(sums[0], sums[1]), add2(sums[2], sums[3])), sum, other);
        l += sum + other;
        ++done;
        ++total;
      }
      if (ok && done > 0) {
        ok = wait(&o_full[t], (total - 1) & 1, bad);
        ok = __all_sync(0xffffffffu, ok);
        tc::fence_after_sync();
      }
      if (ok && u.row[t] < u.s.n) {
        const bool mine = u.row[t] + row < u.s.n;
        const bool none = !sees || pos < 0;
        const float inv = none ? 0.f : 1.f / l;
        float* to_lse = a.parts > 1 ? a.part_lse + static_cast<long long>(u.part) * p.heads * p.tokens : a.lse;
        if (to_lse != nullptr && mine)
          to_lse[static_cast<long long>(u.head[t]) * p.tokens + u.s.q0 + u.row[t] + row] = none ? -INFINITY : (m * p.scale_log2 + log2f(l) - Weights<H>::kBias) / kLog2e;
        const int first_row = u.s.q0 + u.row[t] + (warp & 3) * 32, rows = u.s.n - u.row[t] - (warp & 3) * 32, head = u.head[t];
        const bool odd = *reinterpret_cast<const volatile int*>(&u.odd) != 0;
#pragma unroll 1
        for (int c0 = 0; c0 < p.head_dim; c0 += 64) {
          uint32_t o[2][32] = {};
          if (done > 0) {
            tc::tmem_ld_32x32(t_o + c0, o[0]);
            tc::tmem_ld_32x32(t_o + c0 + 32, o[1]);
            tc::tmem_ld_wait();
          }
          float f[64];
#pragma unroll
          for (int e = 0; e < 64; ++e) f[e] = none ? 0.f : __uint_as_float(o[e / 32][e % 32]) * inv;
          if (odd && mine) {   // (rows behind the text are another's, or none)
            const unsigned long long marks = odd_columns<H>(p, a.v, u, blocks, pos, c0);
#pragma unroll
            for (int e = 0; e < 64; ++e) f[e] = (marks >> e) & 1 ? NAN : f[e];
          }
          if (a.parts > 1) {
            float* to = a.part_o + ((static_cast<long long>(u.part) * p.tokens + first_row + lane) * p.heads + head) * p.head_dim + c0;
#pragma unroll
            for (int e = 0; e < 64; e += 4)
              if (mine && c0 + e < p.head_dim) *reinterpret_cast<float4*>(to + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
            continue;
          }
          rows_out<H>(s_out + warp * kOut, &tm_o, f, a.o, p.heads, p.head_dim, head, first_row, rows, c0);
          if (a.o_rest != nullptr) {
#pragma unroll
            for (int e = 0; e < 64; ++e) f[e] -= H::up(H::down(f[e]));
            rows_out<H>(s_out + warp * kOut, &tm_rest, f, a.o_rest, p.heads, p.head_dim, head, first_row, rows, c0);
          }
        }
      }
      tc::fence_before_sync();   // the next unit's first product with V writes O
      plan.give_back(k);
    }
    rows_sent();
    tc::fence_before_sync();
  }
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 31);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// The parts' results joined: each counts with its share of the sum of exponentials.  Four elements of a head per thread.
template <typename H>
__global__ void __launch_bounds__(256) packed_join_kernel(const Forward a) {
  pdl_wait();
  pdl_trigger();
  const Problem& p = a.p;
  const long long rows = static_cast<long long>(p.tokens) * p.heads;
  const int lanes = p.head_dim / 4, per_block = 256 / lanes, in = threadIdx.x / lanes, c = threadIdx.x % lanes * 4;
  if (in >= per_block) return;
  for (long long r = blockIdx.x * static_cast<long long>(per_block) + in; r < rows; r += static_cast<long long>(gridDim.x) * per_block) {
    const long long t = r / p.heads;
    const int h = static_cast<int>(r - t * p.heads);
    const float* lse = a.part_lse + static_cast<long long>(h) * p.tokens + t;
    const long long part = static_cast<long long>(p.heads) * p.tokens;
    float top = -INFINITY;
    for (int i = 0; i < a.parts; ++i) top = fmaxf(top, lse[i * part]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float whole = 0.f;
    for (int i = 0; i < a.parts; ++i) {
      const float l = lse[i * part];
      // parts that saw nothing are left out; where none saw anything, and where scores were all minus infinity, theirs are the zeros and the NaN
      if (l == -INFINITY && top != -INFINITY) continue;
      const float w = top == -INFINITY ? 1.f : exp2f((l - top) * kLog2e);
      const float4 x = *reinterpret_cast<const float4*>(a.part_o + (i * part + r) * p.head_dim + c);
      sum.x = fmaf(w, x.x, sum.x), sum.y = fmaf(w, x.y, sum.y), sum.z = fmaf(w, x.z, sum.z), sum.w = fmaf(w, x.w, sum.w);
      whole += w;
    }
    const float inv = 1.f / whole;
    const float f[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
    typename H::T2 out[2] = {H::down(f[0], f[1]), H::down(f[2], f[3])};
    *reinterpret_cast<uint2*>(static_cast<typename H::T*>(a.o) + r * p.head_dim + c) = *reinterpret_cast<const uint2*>(out);
    if (a.o_rest != nullptr) {
      const float2 u = H::up(out[0]), v = H::up(out[1]);
      typename H::T2 rest[2] = {H::down(f[0] - u.x, f[1] - u.y), H::down(f[2] - v.x, f[3] - v.y)};
      *reinterpret_cast<uint2*>(static_cast<typename H::T*>(a.o_rest) + r * p.head_dim + c) = *reinterpret_cast<const uint2*>(rest);
    }
    if (a.lse != nullptr && c == 0) a.lse[static_cast<long long>(h) * p.tokens + t] = top == -INFINITY ? -INFINITY : top + logf(whole);
  }
}

constexpr int kSms = 148;
// Two heads that share keys and values make a unit, or else 256 rows of one: an odd number of heads leaves one alone, sequences of up to 128 rows the second tile
// of rows empty.  (8 texts of up to 130 rows behind up to 4096 keys, 12 heads over 4 of 64: 60 us with rows, 42 with heads.)
bool pairs_heads(const PackedAttentionArgs& a) {
  const int group = a.heads / a.kv_heads;
  return group % 2 == 0 || (group > 1 && a.tokens / a.sequences <= kRows);
}
int head_units_of(const PackedAttentionArgs& a) { return pairs_heads(a) ? a.kv_heads * ((a.heads / a.kv_heads + 1) / 2) : a.heads; }
long long units_of(const PackedAttentionArgs& a) { return slots_of(a.tokens, a.sequences, pairs_heads(a) ? kRows : 2 * kRows) * head_units_of(a); }
// How many blocks share out the keys of a unit, by what it costs in microseconds: a step of a unit 2, its beginning and end 5, results in parts 4 and 0.45 per MB (12 heads
// over 4 of 64, 8 texts of some 100 rows behind some 3000 keys: 59 / 43 / 52 / 50 us in 1 / 2 / 3 / 4 parts; 16 heads of 128, 2048 rows: 47 / 61 / 73 / 81; one row over
// 16384 keys 228 in one, 36 in 16).  The host knows no lengths: an average sequence, whose last tile is half full.
int parts_of(const PackedAttentionArgs& a) {
  const int rows = pairs_heads(a) ? kRows : 2 * kRows;
  const float slots = fminf(static_cast<float>(slots_of(a.tokens, a.sequences, rows)), static_cast<float>(a.tokens) / rows + 0.5f * (a.sequences + 1));
  const float units = slots * head_units_of(a), megabytes = static_cast<float>(a.tokens) * a.heads * a.head_dim * 4e-6f;
  if (units >= kSms) return 1;
  const float steps = fmaxf(1.f, (a.k_tokens - 0.5f * a.tokens) / a.sequences / kRows);
  int best = 1;
  float least = INFINITY;
  for (int parts = 1; parts <= 16 && parts * megabytes <= 64.f; ++parts) {
    const float cost = fmaxf(1.f, units * parts / kSms + (parts > 1 ? 0.3f : 0.f)) * (2.f * steps / parts + 5.f) + (parts > 1 ? 4.f + 0.45f * parts * megabytes : 0.f);
    if (cost < least) {
      least = cost;
      best = parts;
    }
  }
  return best;
}

template <typename H, int DP>
cudaError_t launch(const PackedAttentionArgs& args, cudaStream_t stream) {
  Forward f;
  f.p = problem_of(args);
  f.o = args.o;
  f.o_rest = args.o_rest;
  f.lse = args.lse;
  f.v = args.v;
  f.pair_heads = pairs_heads(args) ? 1 : 0;
  f.head_units = head_units_of(args);
  f.parts = args.workspace != nullptr ? parts_of(args) : 1;
  f.part_o = static_cast<float*>(args.workspace);
  f.part_lse = f.part_o + static_cast<size_t>(f.parts) * args.tokens * args.heads * args.head_dim;
  const long long units = units_of(args) * f.parts;
  if (f.p.err == nullptr || units > INT_MAX) return cudaErrorInvalidValue;
  f.units = static_cast<int>(units);
  CUtensorMap q, k, v, o, rest = {};
  if (!encode_rows(&q, args.type, args.q, args.tokens, args.heads, args.head_dim) || !encode_rows(&k, args.type, args.k, args.k_tokens, args.kv_heads, args.head_dim) ||
      !encode_rows(&v, args.type, args.v, args.k_tokens, args.kv_heads, args.head_dim) || !encode_result(&o, args.type, args.o, args.tokens, args.heads, args.head_dim) ||
      (args.o_rest != nullptr && !encode_result(&rest, args.type, args.o_rest, args.tokens, args.heads, args.head_dim)))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(packed_attention_kernel<H, DP>, smem_bytes<DP>(), allowed);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL((packed_attention_kernel<H, DP>), f.units, kThreads, smem_bytes<DP>(), stream, q, k, v, o, rest, f);
  count_launch();
  if (f.parts > 1) {
    const int per_block = 256 / (args.head_dim / 4);
    const long long blocks = (static_cast<long long>(args.tokens) * args.heads + per_block - 1) / per_block;
    MCCL_LAUNCH_PDL(packed_join_kernel<H>, static_cast<int>(blocks < 16 * kSms ? blocks : 16 * kSms), 256, 0, stream, f);
    count_launch();
  }
  return ::mccl::launch_status();
}

}  // namespace

size_t packed_attention_workspace(const PackedAttentionArgs& a) {
  if (a.tokens <= 0 || a.heads <= 0 || a.sequences <= 0) return 0;
  const int parts = parts_of(a);
  return parts == 1 ? 0 : static_cast<size_t>(parts) * a.tokens * a.heads * (a.head_dim + 1) * sizeof(float);
}

cudaError_t packed_attention(const PackedAttentionArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.heads <= 0) return cudaSuccess;
  if (a.type == Half16::bf16) return a.head_dim <= 64 ? launch<Bf16, 64>(a, stream) : launch<Bf16, 128>(a, stream);
  return a.head_dim <= 64 ? launch<Fp16, 64>(a, stream) : launch<Fp16, 128>(a, stream);
}

}  // namespace ops
}  // namespace mccl
