// Causal attention of packed sequences, forward, on the 5th-generation tensor cores.
//
// A block has two tiles of 128 queries that read the same keys and values: the same rows of two query heads that share them, or 256
// neighbouring rows of one head.  Per tile and block of 128 keys:
//   S = Q K^T (tcgen05, operands in shared memory, sums in tensor memory)
//   m' = max(m, rowmax S),  P = exp2((S - m') c),  l = l 2^((m - m') c) + sum P,  O = O 2^((m - m') c) + P V
// P goes back to the columns of S in 16 bits and is the left operand of the second product from there, so no weight passes through shared memory.
// One warpgroup per tile has a row per thread; one warp issues the products of both tiles in turn, so that the tensor cores work on one
// tile while the other's exponentials are computed; one warp brings tiles by TMA; one looks after blocks that not every row sees in whole.
#include "packed_tiles.cuh"

#include "smem_limit.hpp"

#include <climits>

namespace mccl {
namespace ops {

namespace {

using namespace packed;

constexpr int kStages = 4;                 // tiles of keys and values under way
constexpr int kThreads = 12 * 32;          // warps 0-3 and 4-7: rows of tiles 0 and 1; 8: products; 9: loads; 10: blocks seen in part; 11: nothing
// A row's scores need more registers than an even share: 256 x 208 + 128 x 80 of the launch's 384 x 168.
constexpr int kRowRegisters = 208, kOtherRegisters = 80;
constexpr int kStage = 8 * 2048;           // results on their way out, 32 rows x 64 bytes per warp

struct Forward {
  Problem p;
  void* o;
  void* o_rest;      // may be null
  float* lse;
  TokenView v;       // for values that are not finite
  int pair_heads;    // a block's tiles are two heads, otherwise two times 128 rows
  int head_units;    // blocks per slot
  int units;
};

template <int DP>
constexpr int smem_bytes() { return (2 + kStages) * (DP / 64) * kSub + kStage + 512 + 1024; }

// Weights are kept 2^kBias times larger in fp16, whose smallest normal number is 2^-14; the running maximum may be exceeded by 2^kSlack before sums are
// rescaled (exact in fp32 either way), so that the largest weight is 2^8 in bf16 and 2^15 in fp16.
template <typename H>
struct Weights {
  static constexpr float kBias = 0.f, kSlack = 8.f;
};
template <>
struct Weights<Fp16> {
  static constexpr float kBias = 11.f, kSlack = 4.f;
};

// The tiles of a unit.
struct Unit {
  Sequence s;
  int row[2], head[2];       // first row within the sequence; row >= s.n: nothing
  int first[2], last[2];     // positions of the tile's rows
  Blocks b[2], all;
  bool any;
  // Whether all rows of the unit that have block b see all of its keys.
  __device__ __forceinline__ bool whole(const Problem& p, int block) const {
    return (!b[0].has(block) || all_seen(p, block, first[0], last[0])) && (!b[1].has(block) || all_seen(p, block, first[1], last[1]));
  }
};
__device__ __forceinline__ Unit unit_of(const Forward& a, int u) {
  const Problem& p = a.p;
  const int rows = a.pair_heads ? kRows : 2 * kRows;
  const int slots = a.units / a.head_units;
  const int in = u % a.head_units, slot = slots - 1 - u / a.head_units;   // long rows first
  Unit r;
  r.any = false;
  const int s = find_sequence(p.offsets, p.sequences, p.tokens, slot, rows);
  if (s < 0) return r;
  r.s = sequence_of(p, s);
  const int row = (slot - (r.s.q0 / rows + s)) * rows;
  if (row < 0 || row >= r.s.n) return r;
  r.any = true;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (a.pair_heads) {
      r.row[t] = row;
      r.head[t] = 2 * in + t;   // an even number of heads shares keys and values
    } else {
      r.row[t] = row + t * kRows;
      r.head[t] = in;
    }
    r.first[t] = r.s.m - r.s.n + r.row[t];
    r.last[t] = min(r.first[t] + kRows, r.s.m) - 1;
    r.b[t] = r.row[t] < r.s.n ? blocks_of(p, r.first[t], r.last[t]) : Blocks{0, 0, 0};
  }
  r.all.hi = max(r.b[0].hi, r.b[1].hi);
  r.all.lo = r.b[1].hi == 0 ? r.b[0].lo : (r.b[0].hi == 0 ? r.b[1].lo : min(r.b[0].lo, r.b[1].lo));
  r.all.sink = max(r.b[0].sink, r.b[1].sink);
  if (r.all.sink >= r.all.lo) r.all.sink = r.all.lo = 0;   // one run
  return r;
}

template <typename H, int DP>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Forward a) {
  constexpr int kTile = (DP / 64) * kSub;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;                        // [2] tiles
  uint8_t* s_kv = s_q + 2 * kTile;            // [kStages] tiles
  uint8_t* s_out = s_kv + kStages * kTile;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(s_out + kStage);   // [2]
  uint64_t* kv_full = q_full + 2;             // [kStages]
  uint64_t* kv_empty = kv_full + kStages;     // [kStages]
  uint64_t* raw_full = kv_empty + kStages;    // [kStages]: values that are looked at before they are used are here, ...
  uint64_t* looked = raw_full + kStages;      // [kStages]: ... and have been
  uint64_t* s_full = looked + kStages;        // [2]
  uint64_t* p_full = s_full + 2;              // [2]
  uint64_t* o_full = p_full + 2;              // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  volatile int* bad = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* odd_values = bad + 1;
  Unit* s_unit = reinterpret_cast<Unit*>(tmem_slot + 4);

  const Problem& p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int t = 0; t < 2; ++t) {
      tc::mbar_init(&q_full[t], 1);
      tc::mbar_init(&s_full[t], 1);
      tc::mbar_init(&p_full[t], 128);
      tc::mbar_init(&o_full[t], 1);
    }
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(&kv_full[i], 1);
      tc::mbar_init(&kv_empty[i], 1);
      tc::mbar_init(&raw_full[i], 1);
      tc::mbar_init(&looked[i], 1);
    }
    *bad = 0;
    *odd_values = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) tc::tmem_alloc(tmem_slot, 512);
  pdl_wait();
  if (warp == 0) {
    const Unit found = unit_of(a, static_cast<int>(blockIdx.x));
    if (lane == 0) *s_unit = found;
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  const Unit& u = *s_unit;
  pdl_trigger();
  // tensor memory: S of tile t in columns 128 t .. 128 t + 127 (P in the first 64 of them), O in 256 + DP t ..
  const int kv = u.any ? u.head[0] / p.group : 0;

  if (u.any && warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegisters));
  if (warp == 9) {
    // ------------------------------------------------------------------------------------------- loads ----
    if (tc::elect_one()) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (u.b[t].hi > 0) {
          tc::mbar_expect_tx(&q_full[t], kTile);
          load_tile<DP>(s_q + t * kTile, &tm_q, &q_full[t], u.head[t], u.s.q0 + u.row[t]);
        }
      int n = 0;   // tiles so far
      uint32_t raw = 0, uses = 0, raw_uses = 0;   // a bit per stage: which barrier its last load is on, phases of both kinds
      bool ok = true;
      for (int b = u.all.next(-1); ok && b < u.all.hi; b = u.all.next(b)) {
        const bool look = !u.whole(p, b);
        for (int v = 0; v < 2 && ok; ++v) {
          const int st = n % kStages;
          if (n >= kStages) ok = wait(&kv_empty[st], (n / kStages - 1) & 1, bad);
          if (!ok) break;
          const bool r = look && v == 1;
          uint64_t* full = r ? &raw_full[st] : &kv_full[st];
          (r ? raw_uses : uses) ^= 1u << st;
          raw = (raw & ~(1u << st)) | (r ? 1u << st : 0u);
          tc::mbar_expect_tx(full, kTile);
          load_tile<DP>(s_kv + st * kTile, v == 0 ? &tm_k : &tm_v, full, kv, u.s.k0 + b * kRows);
          ++n;
        }
      }
      if (!ok) {   // loads that were issued must land before the block retires
        for (int t = 0; t < 2; ++t)
          if (u.b[t].hi > 0) tc::mbar_wait(&q_full[t], 0, 1u << 18);
        for (int st = 0; st < min(n, kStages); ++st) {
          const bool r = (raw >> st) & 1;
          tc::mbar_wait(r ? &raw_full[st] : &kv_full[st], (((r ? raw_uses : uses) >> st) & 1) ^ 1, 1u << 18);
        }
      }
    }
    __syncwarp();
  } else if (warp == 10) {
    // --------------------------------------------------------- blocks of keys that not every row sees ----
    // A weight of zero times a value that is not finite would be NaN in rows that do not see the value: such values become zeros, and rows that do see
    // them are put right at the end.  Rows behind the sequence are another sequence's.
    int n = 1;
    uint32_t phase = 0;   // a bit per stage
    for (int b = u.all.next(-1); b < u.all.hi; b = u.all.next(b), n += 2) {
      if (u.whole(p, b)) continue;
      const int st = n % kStages, rows = min(kRows, u.s.m - b * kRows);
      const bool ok = wait(&raw_full[st], (phase >> st) & 1, bad);
      if (!__all_sync(0xffffffffu, ok)) break;
      phase ^= 1u << st;
      uint8_t* tile = s_kv + st * kTile;
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
        if (lane == 0) *odd_values = 1;
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&looked[st]);
    }
  } else if (warp == 8) {
    // ---------------------------------------------------------------------------------------- products ----
    constexpr uint32_t idesc_s = idesc16<H>(kRows, kRows, false, false);
    const uint32_t idesc_o = idesc16<H>(kRows, (p.head_dim + 15) / 16 * 16, false, true);
    const int steps = (p.head_dim + 15) / 16;
    int n = 0, before = -1;
    bool begun[2] = {false, false}, have_q[2] = {false, false};
    uint32_t p_phase[2] = {0, 0}, full_phase = 0, looked_phase = 0;   // the last two: a bit per stage
    bool ok = true;
    auto all_wait = [&](uint64_t* bar, uint32_t parity) {
      const bool w = ok && wait(bar, parity, bad);
      ok = __all_sync(0xffffffffu, w);
      return ok;
    };
    int b = u.all.next(-1);
    while (ok && (b < u.all.hi || before >= 0)) {
      const bool more = b < u.all.hi;
      const int sk = n % kStages, sv = (n - 1 + kStages) % kStages;   // keys of b, values of `before`
      if (more) {
        if (!all_wait(&kv_full[sk], (full_phase >> sk) & 1)) break;
        full_phase ^= 1u << sk;
      }
      if (before >= 0) {
        const bool look = !u.whole(p, before);
        if (!all_wait(look ? &looked[sv] : &kv_full[sv], ((look ? looked_phase : full_phase) >> sv) & 1)) break;
        (look ? looked_phase : full_phase) ^= 1u << sv;
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (ok && before >= 0 && u.b[t].has(before) && all_wait(&p_full[t], p_phase[t])) {
          p_phase[t] ^= 1;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            mma_weights(tmem + 256 + t * DP, tmem + t * 128, s_kv + sv * kTile, idesc_o, begun[t]);
            tc::mma_commit(&o_full[t]);
          }
          __syncwarp();
          begun[t] = true;
        }
        if (ok && more && u.b[t].has(b) && (have_q[t] || all_wait(&q_full[t], 0))) {
          have_q[t] = true;
          tc::fence_after_sync();
          if (tc::elect_one()) {
            mma_rows(tmem + t * 128, s_q + t * kTile, s_kv + sk * kTile, idesc_s, steps);
            tc::mma_commit(&s_full[t]);
          }
          __syncwarp();
        }
      }
      if (tc::elect_one()) {
        if (before >= 0) tc::mma_commit(&kv_empty[sv]);
        if (more) tc::mma_commit(&kv_empty[sk]);
      }
      __syncwarp();
      before = more ? b : -1;
      if (more) b = u.all.next(b);
      n += 2;
    }
  }
  } else if (u.any) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRowRegisters));
    // ------------------------------------------------------------------------------------------ a row per thread ----
    const int t = warp >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t t_s = lane_base + t * 128, t_o = lane_base + 256 + t * DP;
    const int pos = u.first[t] + row, first = u.first[t], last = u.last[t];
    const Blocks blocks = u.b[t];
    float m = -INFINITY, l = 0.f;
    uint32_t phase = 0;   // of the next S
    int done = 0;         // blocks so far
    bool ok = true;
    for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b)) {
      ok = wait(&s_full[t], phase, bad);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      phase ^= 1;
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
      if (!all_seen(p, b, first, last)) {
        const int high = pos - b * kRows, low = high - p.window, sink = p.sinks - b * kRows;   // columns seen: c <= high and (c > low or c < sink)
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = c <= high && (c > low || c < sink) ? s[c] : -INFINITY;
      }
      float mx = fmaxf(s[0], s[1]);
#pragma unroll
      for (int c = 2; c < 128; c += 2) mx = fmaxf(mx, fmaxf(s[c], s[c + 1]));
      // a row's maximum stays until it is passed by 2^kSlack.  (Each row's own: its bits do not depend on what else is in the tile.)
      const bool raise = (mx - m) * p.scale_log2 > Weights<H>::kSlack || (m == -INFINITY && mx > m);
      if (__any_sync(0xffffffffu, raise)) {
        const float next = raise ? mx : m, f = raise ? (m == -INFINITY ? 0.f : exp2f((m - next) * p.scale_log2)) : 1.f;
        if (done > 0) {
          ok = wait(&o_full[t], (done - 1) & 1, bad);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld_32x32(t_o + 32 * c, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
            tmem_st32(t_o + 32 * c, o);
          }
        }
        l *= f;
        m = next;
      }
      const float base = (m == -INFINITY ? 0.f : m * p.scale_log2) - Weights<H>::kBias;
      float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float x = exp2f(fmaf(s[64 * c + 2 * e], p.scale_log2, -base)), y = exp2f(fmaf(s[64 * c + 2 * e + 1], p.scale_log2, -base));
          sum0 += x;
          sum1 += y;
          const typename H::T2 h = H::down(x, y);
          w[e] = *reinterpret_cast<const uint32_t*>(&h);
        }
        tmem_st32(t_s + 32 * c, w);
      }
      l += sum0 + sum1;
      tmem_st_wait();
      tc::fence_before_sync();
      tc::mbar_arrive(&p_full[t]);
      ++done;
    }
    if (ok && done > 0) {
      ok = wait(&o_full[t], (done - 1) & 1, bad);
      ok = __all_sync(0xffffffffu, ok);
      tc::fence_after_sync();
    }
    if (ok && u.row[t] < u.s.n) {
      const bool mine = u.row[t] + row < u.s.n;
      // nothing seen: no key up to the position, or none within the window and no first ones
      const bool none = pos < 0;
      const float inv = none ? 0.f : 1.f / l;
      if (a.lse != nullptr && mine)
        a.lse[static_cast<long long>(u.head[t]) * p.tokens + u.s.q0 + u.row[t] + row] = none ? -INFINITY : (m * p.scale_log2 + log2f(l) - Weights<H>::kBias) / kLog2e;
      uint8_t* stage = s_out + warp * 2048;
      const long long o_at = (static_cast<long long>(u.s.q0 + u.row[t] + (warp & 3) * 32) * p.heads + u.head[t]) * p.head_dim;
      const bool odd = *odd_values != 0;
      for (int c0 = 0; c0 < p.head_dim; c0 += 32) {
        uint32_t o[32] = {};
        if (done > 0) {
          tc::tmem_ld_32x32(t_o + c0, o);
          tc::tmem_ld_wait();
        }
        float f[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = none ? 0.f : __uint_as_float(o[e]) * inv;
        if (odd) {
          // values that are not finite in blocks that were looked at, seen by this row
          const typename H::T* v = static_cast<const typename H::T*>(a.v.p) + kv * a.v.head + static_cast<long long>(u.s.k0) * a.v.token + c0;
          for (int b = blocks.next(-1); b < blocks.hi; b = blocks.next(b)) {
            if (u.whole(p, b)) continue;
            for (int j = b * kRows; j < min(b * kRows + kRows, pos + 1); ++j) {
              if (j <= pos - p.window && j >= p.sinks) continue;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (c0 + e < p.head_dim && !(fabsf(H::up(v[j * a.v.token + e])) < INFINITY)) f[e] = NAN;
            }
          }
        }
        const long long stride = static_cast<long long>(p.heads) * p.head_dim;
        const int rows = u.s.n - u.row[t] - (warp & 3) * 32;
        rows_out<H>(stage, f, static_cast<typename H::T*>(a.o) + o_at, stride, rows, c0, p.head_dim);
        if (a.o_rest != nullptr) {
#pragma unroll
          for (int e = 0; e < 32; ++e) f[e] -= H::up(H::down(f[e]));
          rows_out<H>(stage, f, static_cast<typename H::T*>(a.o_rest) + o_at, stride, rows, c0, p.head_dim);
        }
      }
    }
    tc::fence_before_sync();
  }
  __syncthreads();
  if (*bad && tid == 0) atomicExch(p.err, 31);
  if (warp == 8) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
  zero_outside<typename H::T>(a.o, p.heads * p.head_dim, a.lse, p.heads, p.offsets, p.sequences, p.tokens);
}

template <typename H, int DP>
cudaError_t launch(const PackedAttentionArgs& args, cudaStream_t stream) {
  Forward f;
  f.p = problem_of(args);
  f.o = args.o;
  f.o_rest = args.o_rest;
  f.lse = args.lse;
  f.v = args.v;
  f.pair_heads = f.p.group % 2 == 0 ? 1 : 0;
  f.head_units = f.pair_heads ? args.heads / 2 : args.heads;
  const long long units = slots_of(args.tokens, args.sequences, f.pair_heads ? kRows : 2 * kRows) * f.head_units;
  if (f.p.err == nullptr || units > INT_MAX) return cudaErrorInvalidValue;
  f.units = static_cast<int>(units);
  CUtensorMap q, k, v;
  if (!encode_rows(&q, args.type, args.q, args.tokens, args.heads, args.head_dim) || !encode_rows(&k, args.type, args.k, args.k_tokens, args.kv_heads, args.head_dim) ||
      !encode_rows(&v, args.type, args.v, args.k_tokens, args.kv_heads, args.head_dim))
    return cudaErrorInvalidValue;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(packed_attention_kernel<H, DP>, smem_bytes<DP>(), allowed);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL((packed_attention_kernel<H, DP>), f.units, kThreads, smem_bytes<DP>(), stream, q, k, v, f);
  count_launch();
  return ::mccl::launch_status();
}

}  // namespace

cudaError_t packed_attention(const PackedAttentionArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.heads <= 0) return cudaSuccess;
  if (a.type == Half16::bf16) return a.head_dim <= 64 ? launch<Bf16, 64>(a, stream) : launch<Bf16, 128>(a, stream);
  return a.head_dim <= 64 ? launch<Fp16, 64>(a, stream) : launch<Fp16, 128>(a, stream);
}

}  // namespace ops
}  // namespace mccl
