// What the kernels of packed attention share: which tile a block works on, which keys its rows see, tiles in shared memory and tensor memory.
#pragma once

#include "../core/launch.hpp"
#include "../symm/cu_driver.hpp"
#include "half16.cuh"
#include "ops.hpp"
#include "packed.hpp"
#include "packed_keys.hpp"
#include "tcgen05.cuh"

#include <type_traits>

namespace mccl {
namespace ops {

int* gemm_error_device_ptr();

namespace packed {

constexpr int kSub = kRows * 64 * 2;       // a tile's 64 columns: rows of 128 bytes with the 128-byte swizzle, 16 KB
constexpr float kLog2e = 1.4426950408889634f;

// What all kernels know of the problem.
struct Problem {
  const int* offsets;
  const int* k_offsets;
  int tokens, k_tokens, sequences, heads, kv_heads, group, head_dim;
  int window, sinks;   // window: 2^30 without one
  float scale, scale_log2;
  int* err;
};

// A sequence's rows among the queries and among the keys.
struct Sequence {
  int q0, n, k0, m;
};
__device__ __forceinline__ int clamp(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }
__device__ __forceinline__ Sequence sequence_of(const Problem& p, int s) {
  Sequence r;
  r.q0 = clamp(p.offsets[s], 0, p.tokens);
  r.n = clamp(p.offsets[s + 1], r.q0, p.tokens) - r.q0;
  r.k0 = clamp(p.k_offsets[s], 0, p.k_tokens);
  r.m = clamp(p.k_offsets[s + 1], r.k0, p.k_tokens) - r.k0;
  return r;
}

// Slots of `rows` rows: sequence s begins at slot offsets[s] / rows + s, which leaves it enough of them (floor(a + n) - floor(a) + 1 >= ceil(n)) and needs no sums
// over the sequences before it.  Whole-warp call: the sequence whose slots `slot` belongs to (-1: none) by probing 32 places at a time.
__device__ __forceinline__ int find_sequence(const int* offsets, int sequences, int tokens, int slot, int rows) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = sequences;
  bool first = true;
  while (n > 1 || first) {
    first = false;
    const int step = (n + 31) / 32, at = lo + lane * step;
    const bool below = lane * step < n && clamp(offsets[at], 0, tokens) / rows + at <= slot;
    const int count = __popc(__ballot_sync(0xffffffffu, below));
    if (count == 0) return -1;
    lo += (count - 1) * step;
    n = min(step, n - (count - 1) * step);
  }
  return lo;
}
__host__ __device__ __forceinline__ long long slots_of(long long tokens, int sequences, int rows) { return tokens / rows + sequences; }

// Blocks of keys that a tile of queries sees: [0, sink) and [lo, hi).
struct Blocks {
  int sink, lo, hi;
  __device__ __forceinline__ bool has(int b) const { return b < sink || (b >= lo && b < hi); }
  __device__ __forceinline__ int next(int b) const {   // the next one after b
    ++b;
    return b >= sink && b < lo ? lo : b;
  }
};
// rows: positions first .. last
__device__ __forceinline__ Blocks blocks_of(const Problem& p, int first, int last) {
  Blocks r;
  r.hi = last < 0 ? 0 : last / kRows + 1;
  r.lo = min(max(0, first - p.window + 1) / kRows, r.hi);
  r.sink = min((min(p.sinks, 1 << 30) + kRows - 1) / kRows, r.lo);
  return r;
}
// Whether every one of the positions first .. last sees all keys of block b.
__device__ __forceinline__ bool all_seen(const Problem& p, int b, int first, int last) {
  const int k0 = b * kRows, k1 = k0 + kRows - 1;
  return k1 <= first && (k0 > last - p.window || k1 < p.sinks);
}

// --------------------------------------------------------------------------------------------------- memory ----
// Byte offset of 16-byte chunk c (0..7) of row r in a [rows x 64] tile as TMA stores it with the 128-byte swizzle.
__device__ __forceinline__ uint32_t sw128(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 64 columns from `col` of `head` in rows row .. row + 127; zeros behind the tensor's end and its head_dim.
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint64_t* bar, int col, int head, int row) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(tc::smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(bar)), "r"(col), "r"(head), "r"(row)
      : "memory");
}
template <int DP>
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int row) {
#pragma unroll
  for (int c = 0; c < DP / 64; ++c) load_box(dst + c * kSub, map, bar, c * 64, head, row);
}

// Instruction descriptor of 16-bit operands with fp32 sums.
template <typename H>
__host__ __device__ constexpr uint32_t idesc16(int m, int n, bool a_mn, bool b_mn) {
  constexpr uint32_t type = std::is_same<H, Bf16>::value ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (a_mn ? (1u << 15) : 0u) | (b_mn ? (1u << 16) : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}
// D[tmem] (+)= A B[smem]; issued by one thread.  A in tensor memory or (a descriptor) in shared memory.  Adding is told apart from overwriting while compiling where it can
// be: every instruction of that thread counts.
__device__ __forceinline__ void mma_add(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.u32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void mma_add(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.u32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void mma_new(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, 0, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
}
__device__ __forceinline__ void mma_either(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
               ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
               : "memory");
}
// Products over K-major tiles: D[128 x 128 keys] = A B^T over `steps` steps of 16 columns (all DP columns, where they are that many, without counting).
template <int DP>
__device__ __forceinline__ void mma_rows(uint32_t d, const uint8_t* a, const uint8_t* b, uint32_t idesc, int steps) {
  const uint64_t da = tc::smem_desc_k_sw128(a), db = tc::smem_desc_k_sw128(b);
  if (steps == DP / 16) {
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      const uint64_t off = static_cast<uint64_t>((k >> 2) * (kSub >> 4) + (k & 3) * 2);
      k == 0 ? mma_new(d, da, db, idesc) : mma_add(d, da + off, db + off, idesc);
    }
  } else {
#pragma unroll 1
    for (int k = 0; k < steps; ++k) {
      const uint64_t off = static_cast<uint64_t>((k >> 2) * (kSub >> 4) + (k & 3) * 2);
      k == 0 ? mma_new(d, da, db, idesc) : mma_add(d, da + off, db + off, idesc);
    }
  }
}
// D[128 x n] (+)= A[tmem, 128 x kKeys] B with B's rows along the sum: kKeys rows of a tile.  A's second 64 columns are `kApart` columns behind the first.
template <int kKeys, int kApart = 0>
__device__ __forceinline__ void mma_weights(uint32_t d, uint32_t a, const uint8_t* b, uint32_t idesc, bool accumulate) {
  const uint64_t db = tc::smem_desc_mn_sw128(b, kSub);
#pragma unroll
  for (int k = 0; k < kKeys / 16; ++k) {
    const uint32_t at = a + (k >> 2) * kApart + 8 * (k & 3);
    k == 0 ? mma_either(d, at, db, idesc, accumulate) : mma_add(d, at, db + 128 * k, idesc);
  }
}

// The same with A and B in halves: of each 64 columns (two times, `kApart` columns of tensor memory apart) the 32 from 32 h on.
template <int kApart>
__device__ __forceinline__ void mma_half(uint32_t d, uint32_t a, const uint8_t* b, int h, uint32_t idesc, bool accumulate) {
  const uint64_t db = tc::smem_desc_mn_sw128(b, kSub);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int w = i >> 1, k = 4 * w + 2 * h + (i & 1);
    const uint32_t at = a + w * kApart + 8 * (k & 3);
    i == 0 ? mma_either(d, at, db + 128 * k, idesc, accumulate) : mma_add(d, at, db + 128 * k, idesc);
  }
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// A warp's 32 rows (a lane's each) of 64 columns from c0 on leave through 4 KB of its own as one TMA store (rows from `row` on of `head`; columns behind head_dim are
// cut off), or, where not all of the rows are the sequence's, row by row.  f: this lane's columns.  (Stores of registers, each lane to a row of its own, and stores
// through shared memory, four lanes to a row, both took a tile of 128 columns some 5000 clocks.)
constexpr int kOut = 4096;
template <typename H>
__device__ __forceinline__ void rows_out(uint8_t* stage, const CUtensorMap* map, const float (&f)[64], void* base, int heads, int head_dim, int head, int row, int rows, int c0) {
  const int lane = threadIdx.x & 31;
  uint4 x[8];
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    typename H::T2* h = reinterpret_cast<typename H::T2*>(&x[c]);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = H::down(f[8 * c + 2 * e], f[8 * c + 2 * e + 1]);
  }
  if (rows < 32) {
    typename H::T* to = static_cast<typename H::T*>(base) + (static_cast<long long>(row + lane) * heads + head) * head_dim + c0;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (lane < rows && c0 + 8 * c < head_dim) *reinterpret_cast<uint4*>(to + 8 * c) = x[c];
    return;
  }
  if (tc::elect_one()) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // what was here before has been read
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(stage + sw128(lane, c)) = x[c];
  fence_async_smem();
  __syncwarp();
  if (tc::elect_one()) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(tc::smem_u32(stage)), "r"(c0), "r"(head),
                 "r"(row)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
  }
  __syncwarp();
}
// The thread that sent a warp's rows waits until they have been read; by the whole warp, before the block retires.
__device__ __forceinline__ void rows_sent() {
  if (tc::elect_one()) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
}

// Rows of no sequence: zeros in x [tokens, width], minus infinity in lse [heads, tokens] (may be null).  Share `share` of `shares`, by `threads` threads.
template <typename T>
__device__ __forceinline__ void zero_outside(void* x, int width, float* lse, int heads, const int* offsets, int sequences, int tokens, int share, int shares, int thread,
                                             int threads) {
  const int begin = clamp(offsets[0], 0, tokens), end = max(begin, clamp(offsets[sequences], 0, tokens)), outside = begin + tokens - end;
  for (int i = share; i < outside; i += shares) {
    const long long r = i < begin ? i : end + (i - begin);
    uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(x) + r * width);
    for (int c = thread; c < width / 8; c += threads) to[c] = make_uint4(0u, 0u, 0u, 0u);
    if (lse != nullptr)
      for (int h = thread; h < heads; h += threads) lse[static_cast<long long>(h) * tokens + r] = -INFINITY;
  }
}

// Two fp32 numbers in one register pair and instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split(F2 a, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v)); }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// A block's two words on its waits: [0] a role has given up, [1] counts what goes on: units looked for, and every 16th step of loads.
__device__ __forceinline__ void goes_on(volatile int* bad) { atomicAdd(const_cast<int*>(bad) + 1, 1); }
// A wait for another role's part of a step that gives up, and at once when another role of the block has: the first to give up says so in *bad.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* bad) {
  for (uint32_t i = 0; i < (1u << 17); ++i) {   // 0.2 s: the instruction itself waits for 1.5 us
    if (tc::mbar_try_wait(bar, parity)) return true;
    if ((i & 15) == 15 && *bad) return false;
  }
  *bad = 1;
  return false;
}
// A wait that may be for a whole unit, of any number of steps (a block of keys that a million rows of 128 heads see takes 2 s): gives up where nothing goes on for as long as above.
__device__ __forceinline__ bool wait_unit(uint64_t* bar, uint32_t parity, volatile int* bad) {
  for (int steps = bad[1];;) {
    for (uint32_t i = 0; i < (1u << 17); ++i) {
      if (tc::mbar_try_wait(bar, parity)) return true;
      if ((i & 15) == 15 && *bad) return false;
    }
    const int now = bad[1];
    if (now == steps) break;
    steps = now;
  }
  *bad = 1;
  return false;
}

inline Problem problem_of(const PackedAttentionArgs& a) {
  Problem p;
  p.offsets = a.offsets;
  p.k_offsets = a.k_offsets;
  p.tokens = a.tokens;
  p.k_tokens = a.k_tokens;
  p.sequences = a.sequences;
  p.heads = a.heads;
  p.kv_heads = a.kv_heads;
  p.group = a.heads / a.kv_heads;
  p.head_dim = a.head_dim;
  p.window = a.window > 0 && a.window < (1 << 30) ? a.window : 1 << 30;
  p.sinks = a.sinks;
  p.scale = a.scale;
  p.scale_log2 = a.scale * kLog2e;
  p.err = gemm_error_device_ptr();
  return p;
}

// ------------------------------------------------------------------------------------------------ units of work ----
// A block goes on from unit to unit: one warp plans, the others take what it describes.  The first unit is the block's own, the next ones are blocks of the grid
// that have not begun, which it asks the hardware for (the launch's order: long ones first).
struct Plan {
  uint64_t* full;        // [2]: a unit is described
  uint64_t* empty;       // [2]: all roles are done with it
  uint64_t* answer;      // of the request for the next one
  uint64_t* loads_done;  // the unit's last loads are under way: no earlier is the next one asked for, another block may be free sooner
  uint4* next;
  volatile int* bad;     // [2]
  static constexpr int kBarriers = 6;
  __device__ __forceinline__ static Plan at(uint64_t* barriers, uint4* next, volatile int* bad) { return {barriers, barriers + 2, barriers + 4, barriers + 5, next, bad}; }
  __device__ __forceinline__ void init(int roles) const {   // one thread
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], roles);
    }
    tc::mbar_init(answer, 1);
    tc::mbar_init(loads_done, 1);
  }
  // Unit k of this block is described (false: there is none).  Whole warps.
  template <typename Unit>
  __device__ __forceinline__ bool take(const Unit* units, int k) const {
    const bool ok = wait_unit(&full[k & 1], (k >> 1) & 1, bad);
    return __all_sync(0xffffffffu, ok) && !units[k & 1].end;
  }
  __device__ __forceinline__ void give_back(int k) const {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) tc::mbar_arrive(&empty[k & 1]);
  }
  // The planning warp.  find(id): the unit of block `id` (any: whether there is work for the others).
  template <typename Unit, typename Find>
  __device__ __forceinline__ void run(Unit* units, Find find) const {
    const int lane = threadIdx.x & 31;
    int id = static_cast<int>(blockIdx.x), asked = 0;
    auto free = [&](int k) { return __all_sync(0xffffffffu, k < 2 || wait(&empty[k & 1], ((k >> 1) - 1) & 1, bad)); };
    for (int k = 0;;) {
      const Unit found = find(id);
      if (lane == 0) goes_on(bad);   // (there may be many without work)
      if (found.any) {
        if (!free(k)) return;
        if (lane == 0) {
          units[k & 1] = found;
          tc::mbar_arrive(&full[k & 1]);
        }
        __syncwarp();
        const bool near = wait_unit(loads_done, k & 1, bad);
        if (!__all_sync(0xffffffffu, near)) return;
        ++k;
      }
      if (lane == 0) {
        fence_async_smem();   // the last answer has been read
        tc::mbar_expect_tx(answer, 16);
        asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(tc::smem_u32(next)), "r"(tc::smem_u32(answer))
                     : "memory");
      }
      __syncwarp();
      const bool ok = wait(answer, asked & 1, bad);
      if (!__all_sync(0xffffffffu, ok)) {
        tc::mbar_wait(answer, asked & 1, 1u << 16);   // it must land before the block retires
        return;
      }
      ++asked;
      uint32_t got, x;
      asm volatile(
          "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
          "ld.shared.b128 h, [%2];\n\t"
          "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
          "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
          "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
          : "=r"(got), "=r"(x)
          : "r"(tc::smem_u32(next))
          : "memory");
      __syncwarp();
      if (got == 0) {
        if (!free(k)) return;
        if (lane == 0) {
          units[k & 1].end = true;
          tc::mbar_arrive(&full[k & 1]);
        }
        __syncwarp();
        return;
      }
      id = static_cast<int>(x);
    }
  }
};

// [tokens, heads, head_dim] as boxes of 64 columns of `rows` rows of a head.  (The stride of a dimension of one is never used and may be anything.)
inline bool encode_rows(CUtensorMap* map, Half16 type, const TokenView& t, int tokens, int heads, int head_dim, int rows = kRows) {
  const CuDriver& cu = CuDriver::get();
  if (!cu.loaded || !cu.TensorMapEncodeTiled) return false;
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>((heads > 1 ? t.head : head_dim) * 2), static_cast<cuuint64_t>((tokens > 1 ? t.token : head_dim) * 2)};
  const cuuint32_t box[3] = {64, 1, static_cast<cuuint32_t>(rows)}, step[3] = {1, 1, 1};
  return cu.TensorMapEncodeTiled(map, type == Half16::bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(t.p), size,
                                 strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A contiguous result, as the 32 rows that a warp stores.
inline bool encode_result(CUtensorMap* map, Half16 type, const void* p, int tokens, int heads, int head_dim) {
  return encode_rows(map, type, {p, static_cast<long long>(heads) * head_dim, head_dim}, tokens, heads, head_dim, 32);
}

}  // namespace packed
}  // namespace ops
}  // namespace mccl
