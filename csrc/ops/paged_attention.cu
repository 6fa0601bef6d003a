// Attention of one new token per sequence over a paged key-value cache.
//
// The formula, for one sequence and head with query q: o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j over the visible
// positions j and m their maximum.  Sums over any split of the positions join exactly: parts (m, l, o) combine with weights exp(m_part - m).
#include "../core/launch.hpp"
#include "../symm/cu_driver.hpp"
#include "gemm_common.cuh"
#include "half16.cuh"
#include "ops.hpp"
#include "serving.hpp"
#include "tcgen05.cuh"

namespace mccl {
namespace ops {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 16;          // positions that a warp takes at a time
constexpr int kSequences = 1024;   // most sequences of a launch: their lengths and first tiles are kept in shared memory

// What a sequence's visible positions are in tiles: tile t of `tiles` is the one of positions 16 * (t + (t >= head ? skip : 0)) and on.
struct Span {
  int length, first;   // positions [first, length) and those below `sinks` are seen
  int tiles, head, skip;
};
__device__ __forceinline__ Span span_of(int length, int window, int sinks) {
  Span s;
  s.length = length;
  s.first = 0;
  s.tiles = (length + kTile - 1) / kTile;
  s.head = s.tiles;
  s.skip = 0;
  if (window > 0 && length > window) {
    s.first = length - window;
    const int head = (min(sinks, s.first) + kTile - 1) / kTile, tail = s.first / kTile;
    if (tail > head) {
      s.head = head;
      s.skip = tail - head;
      s.tiles -= s.skip;
    }
  }
  return s;
}

struct Launch {
  PagedAttentionArgs a;
  int group, blocks_of_heads;   // query heads per head of keys and values, and blocks of 16 (or 8) that they make
  int items_per_sequence;       // kv_heads * blocks_of_heads
  int page_tiles, page_shift;   // page_size / 16 where that is whole (else 0), its logarithm where that is whole (else -1)
  int whole;                    // an item is one warp's
  float scale_log2;
  long long* plan;              // tiles per warp, then the first tile of every sequence (and behind the last)
  float* part_ml;               // [warps][2][rows][2]
  float* part_o;                // [warps][2][rows][DP]
  int* err;                     // set when a wait inside the kernel ran out
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

__device__ __forceinline__ void load_matrix(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void load_matrix_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <typename H>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<Bf16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<Fp16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename H>
__device__ __forceinline__ uint32_t pair(float a, float b) {
  const typename H::T2 v = H::down(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename H>
__device__ __forceinline__ float2 unpair(uint32_t v) {
  return H::up(*reinterpret_cast<const typename H::T2*>(&v));
}

// Where a warp is: an item is a head of keys and values of a sequence (and a block of its query heads), t the tile within it.
struct Place {
  int item, t;
};

template <int DP, int WARPS, int STAGES>
struct Shape {
  static constexpr int kTileBytes = kTile * DP * 2;   // of K, and of V
  static constexpr int kRing = WARPS * STAGES * 2 * kTileBytes;
  static constexpr int kBars = WARPS * STAGES * 8, kMasks = WARPS * STAGES * 4;
  static constexpr int kSmem = kRing + kBars + (kSequences + 1) * 8 + kSequences * 4 + kMasks + 1024;   // the ring starts on 1024 bytes
};

// A tile is DP / 64 blocks of 16 rows x 128 bytes, the eight 16-byte pieces of a row in the order of the 128-byte swizzle (64: for DP = 32), so that
// the same piece of eight neighbouring rows lies in eight different groups of banks.
template <int DP>
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
  if (DP == 32) return static_cast<uint32_t>(row * 64 + (piece ^ ((row >> 1) & 3)) * 16);
  return static_cast<uint32_t>((piece >> 3) * (kTile * 128) + row * 128 + ((piece & 7) ^ (row & 7)) * 16);
}

// Box of 16 positions x 64 (32) columns of one page and head; zero fill outside the tensor, pages among it.
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, uint32_t bar, int col, int at, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(col), "r"(at), "r"(head), "r"(page)
      : "memory");
}

template <typename H, int DP, int WARPS, int STAGES, int ROWS, bool TMA>
__global__ void __launch_bounds__(WARPS * 32, 1) paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, Launch p) {
  using S = Shape<DP, WARPS, STAGES>;
  using T = typename H::T;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kRing);
  long long* first_tile = reinterpret_cast<long long*>(bars + WARPS * STAGES);
  int* length_of = reinterpret_cast<int*>(first_tile + kSequences + 1);
  uint32_t* masks = reinterpret_cast<uint32_t*>(length_of + kSequences);
  __shared__ long long warp_sum[WARPS];
  const PagedAttentionArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int room = a.table.width * a.table.page_size;
  uint64_t* bar = bars + warp * STAGES;   // one per stage: its copies have landed
  if (TMA && lane == 0) {
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(bar + i, 1);
    tc::mbar_init_fence();
  }
  __syncwarp();

  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  // ---- lengths, and the tiles in front of every sequence
  {
    constexpr int kPer = (kSequences + WARPS * 32 - 1) / (WARPS * 32);
    int mine[kPer];
    long long sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = threadIdx.x * kPer + i;
      mine[i] = 0;
      if (b < a.batch) {
        const int length = min(max(__ldg(a.lengths + b), 0), room);
        length_of[b] = length;
        mine[i] = span_of(length, a.window, a.sinks).tiles;
      }
      sum += mine[i];
    }
    long long before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += other;
    }
    if (lane == 31) warp_sum[warp] = before;
    __syncthreads();
    before -= sum;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = threadIdx.x * kPer + i;
      if (b < a.batch) first_tile[b] = before;
      before += mine[i];
      if (b == a.batch - 1) first_tile[a.batch] = before;
    }
    __syncthreads();
  }
  // sequences that see nothing
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (length_of[b] != 0) continue;
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + static_cast<long long>(b) * a.heads * a.head_dim);
    for (int i = threadIdx.x; i < a.heads * a.head_dim / 8; i += WARPS * 32) o[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int i = threadIdx.x; i < a.heads; i += WARPS * 32) a.lse[static_cast<long long>(b) * a.heads + i] = -INFINITY;
  }

  // ---- this warp's run of tiles
  const int items = a.batch * p.items_per_sequence, warps = gridDim.x * WARPS, me = blockIdx.x * WARPS + warp;
  const long long units = first_tile[a.batch] * p.items_per_sequence;
  Place begin, end;   // [begin, end)
  if (p.whole) {
    begin = {static_cast<int>(static_cast<long long>(items) * me / warps), 0};
    end = {static_cast<int>(static_cast<long long>(items) * (me + 1) / warps), 0};
  } else {
    const long long per = max((units + warps - 1) / warps, static_cast<long long>(2));
    if (blockIdx.x == 0) {
      if (threadIdx.x == 0) p.plan[0] = per;
      for (int b = threadIdx.x; b <= a.batch; b += WARPS * 32) p.plan[1 + b] = first_tile[b];
    }
    const long long u0 = min(per * me, units), u1 = min(u0 + per, units);
    if (u0 >= u1) return;
    auto find = [&](long long u) {
      const long long tile = u / p.items_per_sequence;   // the sequence is the one that this would be in if it had one item
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first_tile[mid] <= tile) lo = mid; else hi = mid - 1;
      }
      const int tiles = static_cast<int>(first_tile[lo + 1] - first_tile[lo]);
      const long long in = u - first_tile[lo] * p.items_per_sequence;
      const int k = static_cast<int>(in / tiles);
      return Place{lo * p.items_per_sequence + k, static_cast<int>(in - static_cast<long long>(k) * tiles)};
    };
    begin = find(u0);
    end = find(u1 - 1);
    ++end.t;
  }
  auto before_end = [&](const Place& at) { return at.item < end.item || (at.item == end.item && at.t < end.t); };
  auto tiles_of = [&](int item) {
    const int b = item / p.items_per_sequence;
    return item < items ? static_cast<int>(first_tile[b + 1] - first_tile[b]) : 1;
  };

  // ---- the loading side: one tile of K and V into a stage
  const uint32_t ring = tc::smem_u32(smem) + warp * (STAGES * 2 * S::kTileBytes);
  uint32_t* mask_ring = masks + warp * STAGES;
  Place load = begin;
  int load_item = -1, load_tiles = 0, load_kv = 0, load_slot = -1, load_page = 0;
  int ahead = 0;   // tiles that are loaded and not yet used
  Span span = {};
  const int* table = nullptr;
  auto settle = [&](Place& at, int& tiles) {   // past items without tiles and past the end of one
    while (at.item < items && at.t >= tiles) {
      ++at.item;
      at.t = 0;
      tiles = tiles_of(at.item);
    }
  };
  load_tiles = tiles_of(load.item);
  settle(load, load_tiles);
  auto issue = [&](int stage) {
    if (before_end(load)) {
      if (load.item != load_item) {
        load_item = load.item;
        load_slot = -1;
        const int b = load.item / p.items_per_sequence;
        load_kv = (load.item - b * p.items_per_sequence) / p.blocks_of_heads;
        span = span_of(length_of[b], a.window, a.sinks);
        table = a.table.p + b * a.table.stride;
      }
      const int tile = load.t + (load.t >= span.head ? span.skip : 0);
      const int r16 = lane & 15, j = tile * kTile + r16;
      const bool seen = j < span.length && (j >= span.first || j < a.sinks);
      const uint32_t to = ring + stage * (2 * S::kTileBytes);
      if (TMA) {   // the tile lies in one page
        const int slot = p.page_shift >= 0 ? tile >> p.page_shift : tile / p.page_tiles;
        if (slot != load_slot) {
          load_slot = slot;
          load_page = __ldg(table + slot);
          if (load_page >= a.table.pages) load_page = -1;   // outside the tensor: zeros come back
        }
        const uint32_t mask = load_page >= 0 ? __ballot_sync(0xffffffffu, seen) & 0xffffu : 0u;
        if (tc::elect_one()) {
          mask_ring[stage] = mask;
          tc::mbar_expect_tx(bar + stage, 2 * S::kTileBytes);
          const uint32_t full = tc::smem_u32(bar + stage);
          const int at = (tile - slot * p.page_tiles) * kTile;
          constexpr int kBox = DP < 64 ? DP : 64;
#pragma unroll
          for (int c = 0; c < DP / kBox; ++c) {
            load_box(to + c * (kTile * kBox * 2), &k_map, full, c * kBox, at, load_kv, load_page);
            load_box(to + S::kTileBytes + c * (kTile * kBox * 2), &v_map, full, c * kBox, at, load_kv, load_page);
          }
        }
        __syncwarp();
      } else {
        int page = -1, at = 0;
        if (seen) {
          const int slot = j / a.table.page_size;
          page = __ldg(table + slot);
          at = j - slot * a.table.page_size;
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, seen && page >= 0 && page < a.table.pages) & 0xffffu;
        if (lane == 0) mask_ring[stage] = mask;
        constexpr int kPieces = DP / 8, kRowsAtOnce = 32 / kPieces;
        const int piece = lane % kPieces, row0 = lane / kPieces;
        const T* k = static_cast<const T*>(a.k_pages.p) + load_kv * a.k_pages.head + piece * 8;
        const T* v = static_cast<const T*>(a.v_pages.p) + load_kv * a.v_pages.head + piece * 8;
        const bool column = piece * 8 < a.head_dim;
#pragma unroll
        for (int i = 0; i < kTile / kRowsAtOnce; ++i) {
          const int row = row0 + i * kRowsAtOnce;
          const int its_page = __shfl_sync(0xffffffffu, page, row), its_at = __shfl_sync(0xffffffffu, at, row);
          const bool good = column && ((mask >> row) & 1u);
          const T* from_k = good ? k + its_page * a.k_pages.page + its_at * a.k_pages.token : static_cast<const T*>(a.k_pages.p);
          const T* from_v = good ? v + its_page * a.v_pages.page + its_at * a.v_pages.token : static_cast<const T*>(a.v_pages.p);
          const uint32_t spot = to + swizzled<DP>(row, piece);
          copy16(spot, from_k, good);
          copy16(spot + S::kTileBytes, from_v, good);
        }
      }
      ++load.t;
      settle(load, load_tiles);
      ++ahead;
    }
    if (!TMA) copy_commit();
  };

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);

  // ---- the computing side
  constexpr int kSteps = DP / 16, kCols = DP / 8;
  Place at = begin;
  int tiles = tiles_of(at.item);
  settle(at, tiles);
  bool first_piece = true, ok = true;
  int stage = 0;
  uint32_t parity = 0;
  // where in a tile a lane's rows of the fragments are: of K (two groups of eight positions, two pieces) and of V (transposed); the pieces of
  // step s are the ones of step 0 with s & 3 in the address bits above
  const uint32_t k_lane = swizzled<DP>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1), v_lane = swizzled<DP>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
  while (before_end(at)) {
    // a new piece of an item: its queries
    const int item = at.item, b = item / p.items_per_sequence, hh = item - b * p.items_per_sequence;
    const int kv = hh / p.blocks_of_heads, in_group = (hh - kv * p.blocks_of_heads) * ROWS;
    const int heads = min(p.group - in_group, ROWS), head0 = kv * p.group + in_group;
    const int from = at.t;
    uint32_t q[kSteps][4];
    {
      const T* base = static_cast<const T*>(a.q.p) + b * a.q.token + head0 * a.q.head;
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = g + (i & 1) * 8, col = s * 16 + (i >> 1) * 8 + 2 * t4;
          q[s][i] = 0;
          if ((ROWS == 16 || (i & 1) == 0) && row < heads && col < a.head_dim) q[s][i] = __ldg(reinterpret_cast<const uint32_t*>(base + row * a.q.head + col));
        }
    }
    float o[kCols][4];
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    constexpr int kHalves = ROWS / 8;   // rows g, and rows g + 8
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    const int stop = item == end.item ? min(tiles, end.t) : tiles;
    for (; at.t < stop; ++at.t) {
      if (TMA) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(bar + stage, parity));
        if (!ok) break;
      } else {
        copy_wait<STAGES - 2>();
        __syncwarp();
      }
      --ahead;
      issue(stage == 0 ? STAGES - 1 : stage - 1);
      const uint32_t k_tile = ring + stage * (2 * S::kTileBytes), v_tile = k_tile + S::kTileBytes;
      const uint32_t mask = mask_ring[stage];
      // scores of 16 positions: two products side by side over two halves of the head, four chains
      float s[2][2][4] = {};
#pragma unroll
      for (int step = 0; step < kSteps; ++step) {
        uint32_t r[4];
        load_matrix(r, k_tile + (step >> 2) * (kTile * 128) + (k_lane ^ ((step & 3) << 5)));
        mma<H>(s[step & 1][0], q[step], r[0], r[1]);
        mma<H>(s[step & 1][1], q[step], r[2], r[3]);
      }
      float z[2][4];   // [row half][position: 2 t4, 2 t4 + 1, 8 + 2 t4, 9 + 2 t4]
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = (s[0][i >> 1][h * 2 + (i & 1)] + s[1][i >> 1][h * 2 + (i & 1)]) * p.scale_log2;
          z[h][i] = (mask >> ((i >> 1) * 8 + 2 * t4 + (i & 1))) & 1u ? v : -INFINITY;
        }
      float keep[2];
      bool moved = false;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        float top = fmaxf(fmaxf(z[h][0], z[h][1]), fmaxf(z[h][2], z[h][3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float now = fmaxf(m[h], top), base = now == -INFINITY ? 0.f : now;
        moved |= now != m[h];
        keep[h] = exp2f(m[h] - base);
        m[h] = now;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[h][i] = exp2f(z[h][i] - base);
          sum += z[h][i];
        }
        l[h] = l[h] * keep[h] + sum;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 2 * kHalves; ++i) o[c][i] *= keep[i >> 1];
      }
      // weights as the sum of two 16-bit values: rounded once to 16 bits they would cost the result as much as its own rounding does,
      // and the tensor cores have nothing else to do
      uint32_t hi[4] = {}, lo[4] = {};
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          hi[i * 2 + h] = pair<H>(z[h][2 * i], z[h][2 * i + 1]);
          const float2 back = unpair<H>(hi[i * 2 + h]);
          lo[i * 2 + h] = pair<H>(z[h][2 * i] - back.x, z[h][2 * i + 1] - back.y);
        }
      // values of positions that are not seen may be anything: they are cleared, for zero times anything need not be zero
      uint32_t clear[2] = {0xffffffffu, 0xffffffffu};
      if (TMA && mask != 0xffffu) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          clear[i] = ((mask >> (i * 8 + 2 * t4)) & 1u ? 0x0000ffffu : 0u) | ((mask >> (i * 8 + 2 * t4 + 1)) & 1u ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int c = 0; c < kCols; c += 2) {
        uint32_t r[4];
        load_matrix_t(r, v_tile + (c >> 3) * (kTile * 128) + (v_lane ^ (((c >> 1) & 3) << 5)));
        if (TMA) {
          r[0] &= clear[0];
          r[1] &= clear[1];
          r[2] &= clear[0];
          r[3] &= clear[1];
        }
        mma<H>(o[c], hi, r[0], r[1]);
        mma<H>(o[c + 1], hi, r[2], r[3]);
        mma<H>(o[c], lo, r[0], r[1]);
        mma<H>(o[c + 1], lo, r[2], r[3]);
      }
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
    if (TMA && !ok) break;

    // ---- the end of this piece: the result where it is the whole item, else a part for the join
    const bool complete = from == 0 && at.t == tiles;
    const size_t slot = (static_cast<size_t>(me) * 2 + (first_piece ? 0 : 1)) * ROWS;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = g + h * 8;
      if (row >= heads) continue;
      if (complete) {
        const float inv = 1.f / l[h];
        T* to = static_cast<T*>(a.o) + (static_cast<long long>(b) * a.heads + head0 + row) * a.head_dim;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int col = c * 8 + 2 * t4;
          if (col < a.head_dim) *reinterpret_cast<typename H::T2*>(to + col) = H::down(o[c][2 * h] * inv, o[c][2 * h + 1] * inv);
        }
        if (a.lse && t4 == 0) a.lse[static_cast<long long>(b) * a.heads + head0 + row] = ((m[h] == -INFINITY ? 0.f : m[h]) + log2f(l[h])) * kLn2;
      } else {
        float* to = p.part_o + (slot + row) * DP;
#pragma unroll
        for (int c = 0; c < kCols; ++c) *reinterpret_cast<float2*>(to + c * 8 + 2 * t4) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(p.part_ml + (slot + row) * 2) = make_float2(m[h], l[h]);
      }
    }
    first_piece = false;
    settle(at, tiles);
  }
  if (!TMA) copy_wait<0>();
  if (TMA && !ok) {
    if (lane == 0) atomicExch(p.err, 21);
    for (; ahead > 0; --ahead) {   // copies that were issued must land before the block retires
      tc::mbar_wait(bar + stage, parity, 1u << 20);
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
}

// One block per sequence and query head whose tiles were shared out: the parts of its warps in order.
template <typename H, int DP, int ROWS>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(Launch p) {
  using T = typename H::T;
  constexpr int kLanes = DP / 4, kGroups = 256 / kLanes;   // four columns per thread, the parts shared out over the groups
  __shared__ float weight[256];
  __shared__ float4 sums[256];
  __shared__ float red[8];
  const PagedAttentionArgs& a = p.a;
  const int b = blockIdx.y, h = blockIdx.x, kv = h / p.group, in_group = h - kv * p.group;
  const int k = kv * p.blocks_of_heads + in_group / ROWS, row = in_group % ROWS;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  const long long per = p.plan[0], first = p.plan[1 + b], tiles = p.plan[2 + b] - first;
  if (tiles <= 0) return;
  const long long s = first * p.items_per_sequence + k * tiles, e = s + tiles;
  const int w0 = static_cast<int>(s / per), w1 = static_cast<int>((e - 1) / per), parts = w1 - w0 + 1;
  if (parts == 1) return;
  auto slot = [&](int i) { return (static_cast<size_t>(w0 + i) * 2 + (i == 0 && per * w0 != s ? 1 : 0)) * ROWS + row; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < parts; i += 256) top = fmaxf(top, p.part_ml[slot(i) * 2]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  top = red[0];
  for (int i = 1; i < 8; ++i) top = fmaxf(top, red[i]);
  const float base = top == -INFINITY ? 0.f : top;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i0 = 0; i0 < parts; i0 += 256) {
    const int n = min(parts - i0, 256);
    float mine = 0.f;
    if (threadIdx.x < n) {
      const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot(i0 + threadIdx.x) * 2);
      const float w = exp2f(ml.x - base);
      weight[threadIdx.x] = w;
      mine = w * ml.y;
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();   // red is free
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mine;
    __syncthreads();
    for (int i = 0; i < 8; ++i) l += red[i];
#pragma unroll 4
    for (int i = group; i < n; i += kGroups) {
      const float w = weight[i];
      const float4 v = *reinterpret_cast<const float4*>(p.part_o + slot(i0 + i) * DP + lane * 4);
      sum.x += w * v.x;
      sum.y += w * v.y;
      sum.z += w * v.z;
      sum.w += w * v.w;
    }
    __syncthreads();
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  const long long out = static_cast<long long>(b) * a.heads + h;
  if (group == 0 && lane * 4 < a.head_dim) {
    for (int i = 1; i < kGroups; ++i) {
      const float4 v = sums[i * kLanes + lane];
      sum.x += v.x;
      sum.y += v.y;
      sum.z += v.z;
      sum.w += v.w;
    }
    const float inv = 1.f / l;
    typename H::T2* to = reinterpret_cast<typename H::T2*>(static_cast<T*>(a.o) + out * a.head_dim + lane * 4);
    to[0] = H::down(sum.x * inv, sum.y * inv);
    to[1] = H::down(sum.z * inv, sum.w * inv);
  }
  if (threadIdx.x == 0 && a.lse) a.lse[out] = (base + log2f(l)) * kLn2;
}

int sm_count() {
  static const int n = [] {
    int device = 0, sms = 148;
    if (cudaGetDevice(&device) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    return sms;
  }();
  return n;
}

int padded_dim(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : (d <= 128 ? 128 : 256)); }
int warps_of(int dp) { return dp == 256 ? 4 : 8; }
int rows_of(const PagedAttentionArgs& a) { return a.heads / a.kv_heads <= 8 ? 8 : 16; }

size_t plan_bytes() { return (kSequences + 2) * sizeof(long long); }

// Keys or values as boxes of 16 positions of one page and head.  False where the strides do not fit a tensor map.
bool encode_pages(CUtensorMap* map, const PagedTensor& t, const PagedAttentionArgs& a, int dp) {
  const CuDriver& cu = CuDriver::get();
  if (!cu.loaded || !cu.TensorMapEncodeTiled) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.table.page_size), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(a.table.pages)};
  // the stride of a dimension of one is never used and may be anything
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.token * 2), static_cast<cuuint64_t>((a.kv_heads > 1 ? t.head : 8) * 2),
                                 static_cast<cuuint64_t>((a.table.pages > 1 ? t.page : 8) * 2)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(dp < 64 ? dp : 64), kTile, 1, 1}, step[4] = {1, 1, 1, 1};
  return cu.TensorMapEncodeTiled(map, a.type == Half16::bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, t.p, dims, strides, box, step,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, dp < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename H, int DP, int WARPS, int STAGES, int ROWS, bool TMA>
cudaError_t launch(const Launch& p, const CUtensorMap (&maps)[2], cudaStream_t stream) {
  constexpr int smem = Shape<DP, WARPS, STAGES>::kSmem;
  static const cudaError_t rc = cudaFuncSetAttribute(paged_attention_kernel<H, DP, WARPS, STAGES, ROWS, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL((paged_attention_kernel<H, DP, WARPS, STAGES, ROWS, TMA>), sm_count(), WARPS * 32, smem, stream, maps[0], maps[1], p);
  count_launch();
  if (!p.whole) {
    MCCL_LAUNCH_PDL((paged_attention_join_kernel<H, DP, ROWS>), dim3(p.a.heads, p.a.batch), 256, 0, stream, p);
    count_launch();
  }
  return ::mccl::launch_status();
}

template <typename H, int ROWS, bool TMA>
cudaError_t by_dim(const Launch& p, const CUtensorMap (&maps)[2], cudaStream_t stream) {
  switch (padded_dim(p.a.head_dim)) {
    case 32: return launch<H, 32, 8, 8, ROWS, TMA>(p, maps, stream);
    case 64: return launch<H, 64, 8, 6, ROWS, TMA>(p, maps, stream);
    case 128: return launch<H, 128, 8, 3, ROWS, TMA>(p, maps, stream);
    default: return launch<H, 256, 4, 3, ROWS, TMA>(p, maps, stream);
  }
}
template <typename H>
cudaError_t by_rows(const Launch& p, int rows, bool tma, const CUtensorMap (&maps)[2], cudaStream_t stream) {
  if (tma) return rows == 8 ? by_dim<H, 8, true>(p, maps, stream) : by_dim<H, 16, true>(p, maps, stream);
  return rows == 8 ? by_dim<H, 8, false>(p, maps, stream) : by_dim<H, 16, false>(p, maps, stream);
}

}  // namespace

size_t paged_attention_workspace(const PagedAttentionArgs& a) {
  const int dp = padded_dim(a.head_dim), rows = rows_of(a);
  const size_t slots = static_cast<size_t>(sm_count()) * warps_of(dp) * 2 * rows;
  return plan_bytes() + slots * (2 + dp) * sizeof(float);
}

cudaError_t paged_attention(const PagedAttentionArgs& args, cudaStream_t stream) {
  if (args.batch <= 0 || args.heads <= 0) return cudaSuccess;
  Launch p;
  p.group = args.heads / args.kv_heads;
  const int rows = rows_of(args);
  p.blocks_of_heads = (p.group + rows - 1) / rows;
  p.items_per_sequence = args.kv_heads * p.blocks_of_heads;
  p.page_tiles = args.table.page_size % kTile == 0 ? args.table.page_size / kTile : 0;
  p.page_shift = -1;
  for (int s = 0; s < 27; ++s)
    if (p.page_tiles == 1 << s) p.page_shift = s;
  p.scale_log2 = args.scale * kLog2e;
  p.whole = static_cast<long long>(args.table.width) * args.table.page_size <= 64 ? 1 : 0;
  p.plan = static_cast<long long*>(args.workspace);
  const size_t slots = static_cast<size_t>(sm_count()) * warps_of(padded_dim(args.head_dim)) * 2 * rows;
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(args.workspace) + plan_bytes());
  p.part_o = p.part_ml + slots * 2;
  p.err = gemm_error_device_ptr();
  CUtensorMap maps[2] = {};
  const int dp = padded_dim(args.head_dim);
  const bool tma = p.page_tiles > 0 && encode_pages(&maps[0], args.k_pages, args, dp) && encode_pages(&maps[1], args.v_pages, args, dp);
  for (int b = 0; b < args.batch; b += kSequences) {
    p.a = args;
    p.a.batch = args.batch - b < kSequences ? args.batch - b : kSequences;
    p.a.lengths = args.lengths + b;
    p.a.table.p = args.table.p + b * args.table.stride;
    p.a.q.p = static_cast<const char*>(args.q.p) + b * args.q.token * 2;
    p.a.o = static_cast<char*>(args.o) + static_cast<long long>(b) * args.heads * args.head_dim * 2;
    p.a.lse = args.lse ? args.lse + static_cast<long long>(b) * args.heads : nullptr;
    const cudaError_t rc = args.type == Half16::bf16 ? by_rows<Bf16>(p, rows, tma, maps, stream) : by_rows<Fp16>(p, rows, tma, maps, stream);
    if (rc != cudaSuccess) return rc;
  }
  return cudaSuccess;
}

}  // namespace ops
}  // namespace mccl
