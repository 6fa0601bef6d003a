// Attention of one new token per sequence over a paged key-value cache.
//
// The formula, for one sequence and head with query q: o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m), s_j = scale q . k_j over the visible
// positions j and m their maximum.  Sums over any split of the positions join exactly: parts (m, l, o) combine with weights exp(m_part - m).
//
// Every key and value is read once and used for up to 16 query heads that share it (more of them: once per 16), at most 8 multiply-adds per byte: memory bounds
// it.  So all tiles of all
// sequences and heads are counted through and every warp of one block per SM streams an equal run of them, whatever the lengths are, through a ring of its
// own that no other warp waits for.  The pieces that a run leaves of an item at its two ends are joined in shared memory, what crosses a block's bounds by a
// second small kernel; everything is added in the order of the positions, so results repeat bit for bit.  Scores and weighted sums are m16n8k16 products:
// eight heads that share keys fill half of their rows, single ones an eighth, and still they run at a quarter of their rate, while the generation's own
// instruction would want 64 rows.
// Measured: 2 x 131009 positions, 32 heads over 8 of 128 (1071 MB): 165 us, 6.5 TB/s; 64 ragged sequences of up to 2048, 16 heads of 128 (540 MB): 87 us, 6.2
// TB/s (by the lengths that are drawn up to 96); 48 windows of 1024 (101 MB): 25.2 us, of which 15.6 from the first load's issue to the last tile: the rest is finding the run (1.8), joining (1.6) and the second
// kernel with its start (3.5); one sequence of 37 tokens: 5.0 us, a chain of four dependent loads.
#include "../core/launch.hpp"
#include "../symm/cu_driver.hpp"
#include "divisor.cuh"
#include "gemm_common.cuh"
#include "half16.cuh"
#include "ops.hpp"
#include "serving.hpp"
#include "smem_limit.hpp"
#include "tcgen05.cuh"

namespace mccl {
namespace ops {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kBlock = 16;         // positions of a block: a tile is one or two
constexpr int kLeast = 2;          // fewest tiles of a warp
constexpr int kSequences = 1024;   // most sequences of a launch: their lengths and first tiles are kept in shared memory

// What a sequence's visible positions are in tiles of KT: tile t of `tiles` is the one of positions KT * (t + (t >= head ? skip : 0)) and on.
struct Span {
  int length, first;   // positions [first, length) and those below `sinks` are seen
  int tiles, head, skip;
};
template <int KT>
__device__ __forceinline__ Span span_of(int length, int window, int sinks) {
  Span s;
  s.length = length;
  s.first = 0;
  s.tiles = (length + KT - 1) / KT;
  s.head = s.tiles;
  s.skip = 0;
  if (window > 0 && length > window) {
    s.first = length - window;
    const int head = (min(sinks, s.first) + KT - 1) / KT, tail = s.first / KT;
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
  int group;                    // query heads per head of keys and values
  Divisor head_blocks, items;   // blocks of 16 (or 8) that they make; items of a sequence: kv_heads * head_blocks
  Divisor page_boxes, warps;    // boxes of a page; warps of the grid
  int whole;                    // an item is one warp's
  float scale_log2;
  int2* open;                   // [blocks]: the item that begins in a block and goes on behind it (-1: none), and the block where it ends
  float* part_ml;               // [blocks][2][rows][2]
  float* part_o;                // [blocks][2][rows][DP]
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

// Weights, and with them their sums, are kept times 2^kLift: fp16 has steps of 2^-24 at its low end, and what many positions have that are far below the largest
// would be lost in the products while the sum of weights counts it.  The largest stays below fp16's limit, and bf16 needs no factor.
template <typename H>
constexpr float kLift = 0.f;
template <>
constexpr float kLift<Fp16> = 15.f;

template <typename H>
__device__ __forceinline__ uint32_t pair(float a, float b) {
  const typename H::T2 v = H::down(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename H>
__device__ __forceinline__ float2 unpair(uint32_t v) {
  return H::up(*reinterpret_cast<const typename H::T2*>(&v));
}

// A stage is a tile of K, the same of V, and the queries where the tile is the first of its piece.  A tile is KT / 16 blocks of 16 positions; a block
// is DP / 64 runs of 16 rows x 128 bytes, the eight 16-byte pieces of a row in the order of the 128-byte swizzle (DP = 32: one run of 64-byte rows with
// that swizzle), so that the same piece of eight neighbouring rows lies in eight different groups of banks.  Queries are one block of ROWS rows.
template <int DP, int KT, int WARPS, int STAGES, int ROWS>
struct Shape {
  static constexpr int kBlockBytes = kBlock * DP * 2;
  static constexpr int kTileBytes = KT * DP * 2;
  static constexpr int kQueryBytes = ROWS * DP * 2;
  static constexpr int kStageBytes = 2 * kTileBytes + kQueryBytes;
  static constexpr int kRing = WARPS * STAGES * kStageBytes;
  static constexpr int kPiece = ROWS * DP * 4;   // a piece's sums: the first of each warp has a place of its own, the last the warp's part of the ring
  static constexpr int kBars = WARPS * STAGES * 8;
  static constexpr int kSmem = kRing + WARPS * kPiece + kBars + (kSequences + 1) * 4 + kSequences * 4 + WARPS * STAGES * 4 + 8 + 1024;   // the ring starts on 1024 bytes
  static_assert(STAGES * kStageBytes >= kPiece && kStageBytes % (DP < 64 ? 512 : 1024) == 0);   // where the swizzle repeats
  static constexpr int kBoxes = DP < 64 ? 1 : DP / 64;   // TMA boxes of a block
};

template <int DP, int R>
__device__ __forceinline__ uint32_t swizzled(int row, int piece) {
  if (DP == 32) return static_cast<uint32_t>(row * 64 + (piece ^ ((row >> 1) & 3)) * 16);
  return static_cast<uint32_t>((piece >> 3) * (R * 128) + row * 128 + ((piece & 7) ^ (row & 7)) * 16);
}

// Box of BOX positions (or ROWS queries) x 64 (32) columns; zero fill outside the tensor, pages among it.
__device__ __forceinline__ void load_pages(uint32_t to, const CUtensorMap* map, uint32_t bar, int col, int at, int head, int page) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(col), "r"(at), "r"(head), "r"(page)
      : "memory");
}
__device__ __forceinline__ void load_queries(uint32_t to, const CUtensorMap* map, uint32_t bar, int col, int head, int b) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(to), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(col), "r"(head), "r"(b)
      : "memory");
}

// Sums of a split that are joined one after the other, four columns of one row.
struct Sums {
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  __device__ __forceinline__ void add(float m2, float l2, const float4& o2) {
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float a = exp2f(m - base), b = exp2f(m2 - base);
    m = top;
    l = l * a + l2 * b;
    o.x = o.x * a + o2.x * b;
    o.y = o.y * a + o2.y * b;
    o.z = o.z * a + o2.z * b;
    o.w = o.w * a + o2.w * b;
  }
};
template <typename H>
__device__ __forceinline__ float log_of_sum(float m, float l) { return ((m == -INFINITY ? 0.f : m) + (log2f(l) - kLift<H>)) * kLn2; }
template <typename H>
__device__ __forceinline__ void store_result(const PagedAttentionArgs& a, long long row, int col, const Sums& s) {
  if (col < a.head_dim) {
    const float inv = 1.f / s.l;
    typename H::T2* to = reinterpret_cast<typename H::T2*>(static_cast<typename H::T*>(a.o) + row * a.head_dim + col);
    to[0] = H::down(s.o.x * inv, s.o.y * inv);
    to[1] = H::down(s.o.z * inv, s.o.w * inv);
  }
  if (col == 0 && a.lse) a.lse[row] = log_of_sum<H>(s.m, s.l);
}

template <typename H, int DP, int KT, int WARPS, int STAGES, int ROWS, int BOX>
__global__ void __launch_bounds__(WARPS * 32, 1)
paged_attention_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap q_map, Launch p) {
  using S = Shape<DP, KT, WARPS, STAGES, ROWS>;
  using T = typename H::T;
  constexpr int kSub = KT / kBlock;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024 - (tc::smem_u32(smem_raw) & 1023)) & 1023);
  unsigned char* first_pieces = smem + S::kRing;
  uint64_t* bars = reinterpret_cast<uint64_t*>(first_pieces + WARPS * S::kPiece);
  unsigned* first_tile = reinterpret_cast<unsigned*>(bars + WARPS * STAGES);   // (a launch has fewer than 2^32 tiles of all its items)
  int* length_of = reinterpret_cast<int*>(first_tile + kSequences + 1);
  uint32_t* masks = reinterpret_cast<uint32_t*>(length_of + kSequences);
  __shared__ unsigned warp_sum[WARPS];
  __shared__ int piece_item[WARPS][2];     // -1: none
  __shared__ int piece_ends[WARPS][2];     // 1: begins its item, 2: ends it
  __shared__ float2 piece_ml[WARPS][2][ROWS];
  const PagedAttentionArgs& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t4 = lane & 3;
  const int room = a.table.width * a.table.page_size;
  uint64_t* bar = bars + warp * STAGES;   // one per stage: its copies have landed
  if (BOX > 0 && lane == 0) {
    for (int i = 0; i < STAGES; ++i) tc::mbar_init(bar + i, 1);
    tc::mbar_init_fence();
    tc::tma_prefetch_desc(&k_map);
    tc::tma_prefetch_desc(&v_map);
    tc::tma_prefetch_desc(&q_map);
  }
  if (lane < 2) piece_item[warp][lane] = -1;
  __syncwarp();

  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();

  // ---- lengths, and the tiles in front of every sequence
  {
    constexpr int kPer = (kSequences + WARPS * 32 - 1) / (WARPS * 32);
    unsigned mine[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = threadIdx.x * kPer + i;
      mine[i] = 0;
      if (b < a.batch) {
        const int length = min(max(__ldg(a.lengths + b), 0), room);
        length_of[b] = length;
        mine[i] = span_of<KT>(length, a.window, a.sinks).tiles;
      }
      sum += mine[i];
    }
    unsigned before = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned other = __shfl_up_sync(0xffffffffu, before, o);
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

  // ---- this warp's run of tiles: `left` of them from tile `begin.t` of an item on
  struct Place {
    int item, t;   // an item is a head of keys and values of a sequence (and a block of its query heads), t the tile within it
  };
  const unsigned per_sequence = p.items.d, items = a.batch * per_sequence, me = blockIdx.x * WARPS + warp;
  const unsigned units = first_tile[a.batch] * per_sequence;
  Place begin = {0, 0};
  int left = 0;
  unsigned per = 0;
  if (p.whole) {
    auto unit = [&](unsigned item) {
      const unsigned b = p.items.of(item);
      return b >= a.batch ? units : first_tile[b] * per_sequence + (item - b * per_sequence) * (first_tile[b + 1] - first_tile[b]);
    };
    const unsigned each = p.warps.of(items), more = items - each * p.warps.d;   // the first `more` warps have one more
    begin.item = me * each + min(me, more);
    left = static_cast<int>(unit(begin.item + each + (me < more ? 1 : 0)) - unit(begin.item));
  } else {
    per = max(p.warps.of(units + p.warps.d - 1), static_cast<unsigned>(kLeast));
    const unsigned u = per * me;
    if (u < units) {
      const unsigned tile = p.items.of(u);   // the sequence is the last that begins at or before this tile
      left = static_cast<int>(min(per, units - u));
      static_assert(kSequences <= 32 * 32);
      const int group = __popc(__ballot_sync(0xffffffffu, lane * 32 < a.batch && first_tile[lane * 32] <= tile)) - 1;
      const int b = group * 32 + __popc(__ballot_sync(0xffffffffu, group * 32 + lane < a.batch && first_tile[group * 32 + lane] <= tile)) - 1;
      const unsigned tiles = first_tile[b + 1] - first_tile[b], in = u - first_tile[b] * per_sequence, k = in / tiles;
      begin = {static_cast<int>(b * per_sequence + k), static_cast<int>(in - k * tiles)};
    }
  }
  auto tiles_of = [&](int item) {
    const int b = p.items.of(item);
    return static_cast<unsigned>(item) < items ? static_cast<int>(first_tile[b + 1] - first_tile[b]) : 1;
  };
  auto settle = [&](Place& at, int& tiles) {   // past items without tiles and past the end of one
    while (static_cast<unsigned>(at.item) < items && at.t >= tiles) {
      ++at.item;
      at.t = 0;
      tiles = tiles_of(at.item);
    }
  };

  // ---- the loading side: a tile of K and V into a stage
  const uint32_t ring = tc::smem_u32(smem) + warp * (STAGES * S::kStageBytes);
  uint32_t* mask_ring = masks + warp * STAGES;
  Place load = begin;
  int to_load = left, load_item = -1, load_tiles = tiles_of(load.item), load_b = 0, load_kv = 0, load_group = 0, load_slot = -1, load_page = 0;
  int ahead = 0;   // tiles that are loaded and not yet used
  Span span = {};
  const int* table = nullptr;
  if (left > 0) settle(load, load_tiles);
  auto issue = [&](int stage) {
    if (to_load > 0) {
      const bool fresh = load.item != load_item;
      if (fresh) {
        load_item = load.item;
        load_slot = -1;
        load_b = p.items.of(load.item);
        const int hh = load.item - load_b * per_sequence;
        load_kv = p.head_blocks.of(hh);
        load_group = (hh - load_kv * p.head_blocks.d) * ROWS;
        span = span_of<KT>(length_of[load_b], a.window, a.sinks);
        table = a.table.p + load_b * a.table.stride;
      }
      const int head0 = load_kv * p.group + load_group;
      const int tile = load.t + (load.t >= span.head ? span.skip : 0);
      const uint32_t to = ring + stage * S::kStageBytes;
      if (BOX > 0) {   // every box of positions lies in one page
        const int j = tile * KT + lane;
        uint32_t mask = __ballot_sync(0xffffffffu, j < span.length && (j >= span.first || j < a.sinks));
        if (KT < 32) mask &= 0xffffu;
        constexpr int kBoxes = KT / (BOX > 0 ? BOX : KT);
        int page[kBoxes], at[kBoxes];
#pragma unroll
        for (int i = 0; i < kBoxes; ++i) {
          const int box = tile * kBoxes + i, slot = p.page_boxes.of(box);
          if (slot != load_slot && (i == 0 || box * BOX < span.length)) {
            load_slot = slot;
            load_page = __ldg(table + slot);
            if (load_page >= a.table.pages) load_page = -1;   // outside the tensor: zeros come back
          }
          page[i] = slot == load_slot ? load_page : -1;
          at[i] = (box - slot * p.page_boxes.d) * BOX;
          if (page[i] < 0) mask &= ~(((BOX == 32 ? 0u : 1u << (BOX & 31)) - 1u) << (i * BOX));
        }
        if (tc::elect_one()) {
          mask_ring[stage] = mask;
          tc::mbar_expect_tx(bar + stage, 2 * S::kTileBytes + (fresh ? S::kQueryBytes : 0));
          const uint32_t full = tc::smem_u32(bar + stage);
          constexpr int kBox = DP / S::kBoxes;
          if (fresh) {
#pragma unroll
            for (int c = 0; c < S::kBoxes; ++c) load_queries(to + 2 * S::kTileBytes + c * (ROWS * kBox * 2), &q_map, full, c * kBox, head0, load_b);
          }
#pragma unroll
          for (int i = 0; i < kBoxes; ++i)
#pragma unroll
            for (int c = 0; c < S::kBoxes; ++c) {
              const int row = i * BOX;
              const uint32_t spot = to + row / kBlock * S::kBlockBytes + c * (kBlock * kBox * 2) + row % kBlock * (kBox * 2);
              load_pages(spot, &k_map, full, c * kBox, at[i], load_kv, page[i]);
              load_pages(spot + S::kTileBytes, &v_map, full, c * kBox, at[i], load_kv, page[i]);
            }
        }
        __syncwarp();
      } else {
        const int j = tile * KT + lane % KT;
        const bool seen = j < span.length && (j >= span.first || j < a.sinks);
        int page = -1, at = 0;
        if (seen) {
          const int slot = j / a.table.page_size;
          page = __ldg(table + slot);
          at = j - slot * a.table.page_size;
        }
        uint32_t mask = __ballot_sync(0xffffffffu, seen && page >= 0 && page < a.table.pages);
        if (KT < 32) mask &= 0xffffu;
        if (lane == 0) mask_ring[stage] = mask;
        constexpr int kPieces = DP / 8, kRowsAtOnce = 32 / kPieces;
        const int piece = lane % kPieces, row0 = lane / kPieces;
        const T* k = static_cast<const T*>(a.k_pages.p) + load_kv * a.k_pages.head + piece * 8;
        const T* v = static_cast<const T*>(a.v_pages.p) + load_kv * a.v_pages.head + piece * 8;
        const bool column = piece * 8 < a.head_dim;
#pragma unroll
        for (int i = 0; i < KT / kRowsAtOnce; ++i) {
          const int row = row0 + i * kRowsAtOnce;
          const int its_page = __shfl_sync(0xffffffffu, page, row), its_at = __shfl_sync(0xffffffffu, at, row);
          const bool good = column && ((mask >> row) & 1u);
          const T* from_k = good ? k + its_page * a.k_pages.page + its_at * a.k_pages.token : static_cast<const T*>(a.k_pages.p);
          const T* from_v = good ? v + its_page * a.v_pages.page + its_at * a.v_pages.token : static_cast<const T*>(a.v_pages.p);
          const uint32_t spot = to + (row / kBlock) * S::kBlockBytes + swizzled<DP, kBlock>(row % kBlock, piece);
          copy16(spot, from_k, good);
          copy16(spot + S::kTileBytes, from_v, good);
        }
        if (fresh) {
          const T* q = static_cast<const T*>(a.q.p) + load_b * a.q.token + piece * 8;
          for (int row = row0; row < ROWS; row += kRowsAtOnce) {
            const bool good = column && load_group + row < p.group;
            copy16(to + 2 * S::kTileBytes + swizzled<DP, ROWS>(row, piece), good ? q + (head0 + row) * a.q.head : static_cast<const T*>(a.q.p), good);
          }
        }
      }
      ++load.t;
      if (--to_load > 0) settle(load, load_tiles);
      ++ahead;
    }
    if (BOX == 0) copy_commit();
  };

#pragma unroll
  for (int s = 0; s < STAGES; ++s) issue(s);

  // sequences that see nothing
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (length_of[b] != 0) continue;
    uint4* o = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + static_cast<long long>(b) * a.heads * a.head_dim);
    for (int i = threadIdx.x; i < a.heads * a.head_dim / 8; i += WARPS * 32) o[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int i = threadIdx.x; i < a.heads; i += WARPS * 32) a.lse[static_cast<long long>(b) * a.heads + i] = -INFINITY;
  }

  // ---- the computing side
  constexpr int kSteps = DP / 16, kCols = DP / 8, kHalves = ROWS / 8;   // halves: rows g, and rows g + 8
  constexpr int kChains = KT == 16 ? 2 : 1;
  Place at = begin;
  int tiles = tiles_of(at.item);
  if (left > 0) settle(at, tiles);
  bool first_piece = true, ok = true;
  int stage = 0;
  uint32_t parity = 0;
  // where in a block a lane's rows of the fragments are: of K (two groups of eight positions, two pieces), of V (transposed) and of the queries; the
  // pieces of a later step are the ones of the first with the step in the address bits above
  const uint32_t k_lane = swizzled<DP, kBlock>((lane >> 4) * 8 + (lane & 7), (lane >> 3) & 1), v_lane = swizzled<DP, kBlock>(((lane >> 3) & 1) * 8 + (lane & 7), lane >> 4);
  while (left > 0) {
    const int item = at.item, from = at.t, stop = min(tiles, from + left);
    left -= stop - from;
    uint32_t q[kSteps][4];
    float o[kCols][4];
#pragma unroll
    for (int c = 0; c < kCols; ++c) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (; at.t < stop; ++at.t) {
      if (BOX > 0) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(bar + stage, parity));
        if (!ok) break;
      } else {
        copy_wait<STAGES - 1>();
        __syncwarp();
      }
      --ahead;
      const uint32_t k_tile = ring + stage * S::kStageBytes, v_tile = k_tile + S::kTileBytes;
      const uint32_t mask = mask_ring[stage];
      if (at.t == from) {   // a new piece: its queries
        const uint32_t q_tile = v_tile + S::kTileBytes;
#pragma unroll
        for (int s = 0; s < kSteps; s += 2 / kHalves) {
          uint32_t r[4];
          if (ROWS == 8) {
            load_matrix(r, q_tile + swizzled<DP, ROWS>(lane & 7, 2 * s + (lane >> 3)));
            q[s][0] = r[0], q[s][1] = 0, q[s][2] = r[1], q[s][3] = 0;
            q[s + 1][0] = r[2], q[s + 1][1] = 0, q[s + 1][2] = r[3], q[s + 1][3] = 0;
          } else {
            load_matrix(q[s], q_tile + swizzled<DP, ROWS>(((lane >> 3) & 1) * 8 + (lane & 7), 2 * s + (lane >> 4)));
          }
        }
      }
      // scores: per 16 positions two products side by side
      float s[kChains][2 * kSub][4] = {};
#pragma unroll
      for (int step = 0; step < kSteps; ++step)
#pragma unroll
        for (int i = 0; i < kSub; ++i) {
          uint32_t r[4];
          load_matrix(r, k_tile + i * S::kBlockBytes + (step >> 2) * (kBlock * 128) + (k_lane ^ ((step & 3) << 5)));
          mma<H>(s[step % kChains][2 * i], q[step], r[0], r[1]);
          mma<H>(s[step % kChains][2 * i + 1], q[step], r[2], r[3]);
        }
      float z[2][4 * kSub];   // [row half][8 i + 2 t4, 8 i + 2 t4 + 1 for each i]
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < 4 * kSub; ++i) {
          float v = s[0][i >> 1][h * 2 + (i & 1)];
          if (kChains == 2) v += s[kChains - 1][i >> 1][h * 2 + (i & 1)];
          z[h][i] = (mask >> ((i >> 1) * 8 + 2 * t4 + (i & 1))) & 1u ? v * p.scale_log2 : -INFINITY;
        }
      float keep[2];
      bool moved = false;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        float top = fmaxf(z[h][0], z[h][1]);
#pragma unroll
        for (int i = 2; i < 4 * kSub; ++i) top = fmaxf(top, z[h][i]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float now = fmaxf(m[h], top), base = now == -INFINITY ? 0.f : now;
        moved |= now != m[h];
        keep[h] = exp2f(m[h] - base);
        m[h] = now;
        float sum = 0.f;
        const float lifted = base - kLift<H>;
#pragma unroll
        for (int i = 0; i < 4 * kSub; ++i) {
          z[h][i] = exp2f(z[h][i] - lifted);
          sum += z[h][i];
        }
        l[h] = l[h] * keep[h] + sum;
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int c = 0; c < kCols; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[c][i] *= keep[ROWS == 8 ? 0 : i >> 1];
      }
#pragma unroll
      for (int i = 0; i < kSub; ++i) {
        // weights as the sum of two 16-bit values: rounded once to 16 bits they would cost the result as much as its own rounding does.  With
        // eight queries the rest goes into the eight rows of the product that have none.
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float w0 = z[h][4 * i + 2 * e], w1 = z[h][4 * i + 2 * e + 1];
            hi[e * 2 + h] = pair<H>(w0, w1);
            const float2 back = unpair<H>(hi[e * 2 + h]);
            const uint32_t rest = pair<H>(w0 - back.x, w1 - back.y);
            if (ROWS == 8) hi[e * 2 + 1] = rest; else lo[e * 2 + h] = rest;
          }
        // values of positions that are not seen may be anything: they are cleared, for zero times anything need not be zero
        uint32_t clear[2] = {0xffffffffu, 0xffffffffu};
        if (BOX > 0 && ((mask >> (16 * i)) & 0xffffu) != 0xffffu) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            clear[e] = ((mask >> (16 * i + e * 8 + 2 * t4)) & 1u ? 0x0000ffffu : 0u) | ((mask >> (16 * i + e * 8 + 2 * t4 + 1)) & 1u ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int c = 0; c < kCols; c += 2) {
          uint32_t r[4];
          load_matrix_t(r, v_tile + i * S::kBlockBytes + (c >> 3) * (kBlock * 128) + (v_lane ^ (((c >> 1) & 3) << 5)));
          if (BOX > 0) {
            r[0] &= clear[0];
            r[1] &= clear[1];
            r[2] &= clear[0];
            r[3] &= clear[1];
          }
          mma<H>(o[c], hi, r[0], r[1]);
          mma<H>(o[c + 1], hi, r[2], r[3]);
          if (ROWS == 16) {
            mma<H>(o[c], lo, r[0], r[1]);
            mma<H>(o[c + 1], lo, r[2], r[3]);
          }
        }
      }
      __syncwarp();   // every lane has read its fragments
      issue(stage);
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
    if (BOX > 0 && !ok) break;

    // ---- the end of this piece: the result where it is the whole item, else its sums for the block
    const bool complete = from == 0 && at.t == tiles;
    const int b = p.items.of(item), hh = item - b * per_sequence;
    const int kv = p.head_blocks.of(hh), in_group = (hh - kv * p.head_blocks.d) * ROWS;
    const int heads = min(p.group - in_group, ROWS), head0 = kv * p.group + in_group;
    const int which = first_piece ? 0 : 1;
    unsigned char* sums = first_piece ? first_pieces + warp * S::kPiece : smem + warp * (STAGES * S::kStageBytes);
    if (ROWS == 8) {
#pragma unroll
      for (int c = 0; c < kCols; ++c) o[c][0] += o[c][2], o[c][1] += o[c][3];
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      const int row = g + h * 8;
      if (row >= heads) continue;
      if (complete) {
        const float inv = 1.f / l[h];
        const long long out = static_cast<long long>(b) * a.heads + head0 + row;
        T* to = static_cast<T*>(a.o) + out * a.head_dim;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
          const int col = c * 8 + 2 * t4;
          if (col < a.head_dim) *reinterpret_cast<typename H::T2*>(to + col) = H::down(o[c][2 * h] * inv, o[c][2 * h + 1] * inv);
        }
        if (a.lse && t4 == 0) a.lse[out] = log_of_sum<H>(m[h], l[h]);
      } else {
        float* to = reinterpret_cast<float*>(sums) + row * DP;
#pragma unroll
        for (int c = 0; c < kCols; ++c) *reinterpret_cast<float2*>(to + c * 8 + 2 * t4) = make_float2(o[c][2 * h], o[c][2 * h + 1]);
        if (t4 == 0) piece_ml[warp][which][row] = make_float2(m[h], l[h]);
      }
    }
    if (!complete && lane == 0) {
      piece_item[warp][which] = item;
      piece_ends[warp][which] = (from == 0 ? 1 : 0) | (at.t == tiles ? 2 : 0);
    }
    first_piece = false;
    if (left > 0) settle(at, tiles);
  }
  if (BOX == 0) copy_wait<0>();
  if (BOX > 0 && !ok) {
    if (lane == 0) atomicExch(p.err, 21);
    for (; ahead > 0; --ahead) {   // copies that were issued must land before the block retires
      tc::mbar_wait(bar + stage, parity, 1u << 20);
      if (++stage == STAGES) {
        stage = 0;
        parity ^= 1;
      }
    }
  }
  if (p.whole) return;

  // ---- pieces of one item, a run, are joined in the order of their positions, four columns of a row per lane.  What lies within the block is a result;
  // what came from the block before, or goes on in the next, is left for the join.  The warps take runs (and 32 lanes' worth of a run) in turn: one run
  // after the other took 2.5 us where every warp ended one and began another.
  __syncthreads();
  const int their_item = lane < 2 * WARPS ? piece_item[lane >> 1][lane & 1] : -1, their_ends = lane < 2 * WARPS ? piece_ends[lane >> 1][lane & 1] : 0;
  const unsigned pieces = __ballot_sync(0xffffffffu, their_item >= 0), below = pieces & ((1u << lane) - 1u);
  const int before = __shfl_sync(0xffffffffu, their_item, below != 0 ? 31 - __clz(below) : 0);
  const unsigned starts = __ballot_sync(0xffffffffu, their_item >= 0 && (below == 0 || before != their_item));
  const int parts = (min(p.group, ROWS) * (DP / 4) + 31) / 32;   // of a run
  for (int n = warp; n < __popc(starts) * parts; n += WARPS) {
    const int which = n / parts;
    unsigned rest = starts;
    for (int i = 0; i < which; ++i) rest &= rest - 1;
    const int first = __ffs(rest) - 1, item = __shfl_sync(0xffffffffu, their_item, first);
    const unsigned run = __ballot_sync(0xffffffffu, their_item == item) & pieces;
    const int begun = __shfl_sync(0xffffffffu, their_ends, first) & 1, ended = __shfl_sync(0xffffffffu, their_ends, 31 - __clz(run)) & 2;
    const int b = p.items.of(item), hh = item - b * per_sequence;
    const int kv = p.head_blocks.of(hh), in_group = (hh - kv * p.head_blocks.d) * ROWS;
    const int u = (n - which * parts) * 32 + lane;
    if (u < min(p.group - in_group, ROWS) * (DP / 4)) {
      const int row = u / (DP / 4), col = u % (DP / 4) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2 * WARPS; ++i)
        if ((run >> i) & 1u) top = fmaxf(top, piece_ml[i >> 1][i & 1][row].x);
      Sums sum;
      sum.m = top;
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int i = 0; i < 2 * WARPS; ++i) {
        if (!((run >> i) & 1u)) continue;
        const float2 ml = piece_ml[i >> 1][i & 1][row];
        const float weight = exp2f(ml.x - base);
        const float4 o = *reinterpret_cast<const float4*>((i & 1 ? smem + (i >> 1) * (STAGES * S::kStageBytes) : first_pieces + (i >> 1) * S::kPiece) + (row * DP + col) * 4);
        sum.l += weight * ml.y;
        sum.o.x += weight * o.x;
        sum.o.y += weight * o.y;
        sum.o.z += weight * o.z;
        sum.o.w += weight * o.w;
      }
      if (begun && ended) {
        store_result<H>(a, static_cast<long long>(b) * a.heads + kv * p.group + in_group + row, col, sum);
      } else {
        const size_t slot = (static_cast<size_t>(blockIdx.x) * 2 + begun) * ROWS + row;
        *reinterpret_cast<float4*>(p.part_o + slot * DP + col) = sum.o;
        if (col == 0) *reinterpret_cast<float2*>(p.part_ml + slot * 2) = make_float2(sum.m, sum.l);
      }
    }
    __syncwarp();
  }
  if (warp == 0) {   // whether the last run goes on, and to where
    int2 open = make_int2(-1, 0);
    if (pieces != 0) {
      const int item = __shfl_sync(0xffffffffu, their_item, 31 - __clz(pieces));
      const int begun = __shfl_sync(0xffffffffu, their_ends, 31 - __clz(starts)) & 1, ended = __shfl_sync(0xffffffffu, their_ends, 31 - __clz(pieces)) & 2;
      const int b = p.items.of(item), hh = item - b * per_sequence;
      if (begun && !ended) open = make_int2(item, (first_tile[b] * per_sequence + (hh + 1) * (first_tile[b + 1] - first_tile[b]) - 1) / (per * WARPS));
    }
    if (lane == 0) p.open[blockIdx.x] = open;
  }
}

// Block (c, row): the item that begins in block c and goes on behind it, if there is one, and one of its queries: its parts in order.
template <typename H, int DP, int ROWS>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(Launch p) {
  constexpr int kLanes = DP / 4, kGroups = 128 / kLanes;   // four columns per thread, the parts shared out over the groups
  __shared__ __align__(16) unsigned char raw[128 * sizeof(Sums)];
  Sums* sums = reinterpret_cast<Sums*>(raw);
  const PagedAttentionArgs& a = p.a;
  const int lane = threadIdx.x % kLanes, group = threadIdx.x / kLanes, c0 = blockIdx.x, row = blockIdx.y;
  ::mccl::pdl_wait();
  ::mccl::pdl_trigger();
  // a thread's first part is on its way before it is known whether there is one (there is room for it)
  const size_t first = (static_cast<size_t>(min(c0 + group, static_cast<int>(gridDim.x) - 1)) * 2 + (group == 0)) * ROWS + row;
  const float2 first_ml = *reinterpret_cast<const float2*>(p.part_ml + first * 2);
  const float4 first_o = *reinterpret_cast<const float4*>(p.part_o + first * DP + lane * 4);
  const int2 open = p.open[c0];
  if (open.x < 0) return;
  const int b = p.items.of(open.x), hh = open.x - b * p.items.d, kv = p.head_blocks.of(hh), in_group = (hh - kv * p.head_blocks.d) * ROWS;
  if (in_group + row >= p.group) return;
  Sums sum;
  if (c0 + group <= open.y) sum.add(first_ml.x, first_ml.y, first_o);
#pragma unroll 4
  for (int c = c0 + group + kGroups; c <= open.y; c += kGroups) {
    const size_t slot = static_cast<size_t>(c) * 2 * ROWS + row;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
    sum.add(ml.x, ml.y, *reinterpret_cast<const float4*>(p.part_o + slot * DP + lane * 4));
  }
  sums[threadIdx.x] = sum;
  __syncthreads();
  if (group == 0) {
    for (int i = 1; i < kGroups; ++i) {
      const Sums& other = sums[i * kLanes + lane];
      sum.add(other.m, other.l, other.o);
    }
    store_result<H>(a, static_cast<long long>(b) * a.heads + kv * p.group + in_group + row, lane * 4, sum);
  }
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
int rows_of(const PagedAttentionArgs& a) { return a.heads / a.kv_heads <= 8 ? 8 : 16; }
size_t open_bytes() { return (static_cast<size_t>(sm_count()) * sizeof(int2) + 15) / 16 * 16; }
// Whether every item is one warp's: so short that a split would not pay for the join, a launch of its own.  Longest sequences that the table has room for, 64
// limit / 128 / 256: 16 x 8 heads of 64 up to 128 positions 9.2 / 7.7 / 7.6 us, 32 x 8 up to 256 9.3 / 9.3 / 12.2, 256 x 12 up to 256 28.7 / 28.5 / 33.5.
bool whole(const PagedAttentionArgs& a) { return static_cast<long long>(a.table.width) * a.table.page_size <= 128; }

bool encode(CUtensorMap* map, Half16 type, int dims, const void* base, const cuuint64_t* size, const cuuint64_t* strides, const cuuint32_t* box) {
  const CuDriver& cu = CuDriver::get();
  if (!cu.loaded || !cu.TensorMapEncodeTiled) return false;
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return cu.TensorMapEncodeTiled(map, type == Half16::bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, dims, const_cast<void*>(base), size, strides,
                                 box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, box[0] < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Keys or values as boxes of positions of one page and head, queries as boxes of `rows` heads.  False where the strides do not fit a tensor
// map.  (The stride of a dimension of one is never used and may be anything.)
bool encode_pages(CUtensorMap* map, const PagedTensor& t, const PagedAttentionArgs& a, int dp, int positions) {
  const cuuint64_t size[4] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.table.page_size), static_cast<cuuint64_t>(a.kv_heads),
                              static_cast<cuuint64_t>(a.table.pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(t.token * 2), static_cast<cuuint64_t>((a.kv_heads > 1 ? t.head : 8) * 2),
                                 static_cast<cuuint64_t>((a.table.pages > 1 ? t.page : 8) * 2)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(dp < 64 ? dp : 64), static_cast<cuuint32_t>(positions), 1, 1};
  return encode(map, a.type, 4, t.p, size, strides, box);
}
bool encode_queries(CUtensorMap* map, const PagedAttentionArgs& a, int dp, int rows) {
  const cuuint64_t size[3] = {static_cast<cuuint64_t>(a.head_dim), static_cast<cuuint64_t>(a.heads), static_cast<cuuint64_t>(a.batch)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>((a.heads > 1 ? a.q.head : 8) * 2), static_cast<cuuint64_t>((a.batch > 1 ? a.q.token : 8) * 2)};
  const cuuint32_t box[3] = {static_cast<cuuint32_t>(dp < 64 ? dp : 64), static_cast<cuuint32_t>(rows), 1};
  return encode(map, a.type, 3, a.q.p, size, strides, box);
}

template <typename H, int DP, int KT, int WARPS, int STAGES, int ROWS, int BOX>
cudaError_t launch(Launch& p, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  constexpr int smem = Shape<DP, KT, WARPS, STAGES, ROWS>::kSmem;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(paged_attention_kernel<H, DP, KT, WARPS, STAGES, ROWS, BOX>, smem, allowed);
  if (rc != cudaSuccess) return rc;
  p.warps = Divisor(sm_count() * WARPS);
  MCCL_LAUNCH_PDL((paged_attention_kernel<H, DP, KT, WARPS, STAGES, ROWS, BOX>), sm_count(), WARPS * 32, smem, stream, maps[0], maps[1], maps[2], p);
  count_launch();
  if (!p.whole) {
    MCCL_LAUNCH_PDL((paged_attention_join_kernel<H, DP, ROWS>), dim3(sm_count(), p.group < ROWS ? p.group : ROWS), 128, 0, stream, p);
    count_launch();
  }
  return ::mccl::launch_status();
}

// Sizes of tile and ring: as many warps as hide the latency of a tile's chain (scores, maximum, weights, products), two stages of 8 KB each.  More bytes in
// flight are slower (2 x 131009 positions: three stages 181 us, two 172), fewer warps too (4 x 4 stages 191, 6 x 2 182).
template <typename H, int BOX>
cudaError_t by_size(Launch& p, int rows, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  const int dp = padded_dim(p.a.head_dim);
  if (rows == 8) {
    if (dp == 32) return launch<H, 32, 32, 8, 4, 8, BOX>(p, maps, stream);
    if (dp == 64) return launch<H, 64, 32, 8, 2, 8, BOX>(p, maps, stream);
    if (dp == 128) return launch<H, 128, 16, 8, 2, 8, BOX>(p, maps, stream);
    return launch<H, 256, 16, 4, 2, 8, BOX>(p, maps, stream);
  }
  if (dp == 32) return launch<H, 32, 32, 8, 4, 16, BOX>(p, maps, stream);
  if (dp == 64) return launch<H, 64, 32, 8, 2, 16, BOX>(p, maps, stream);
  if (dp == 128) return launch<H, 128, 16, 6, 2, 16, BOX>(p, maps, stream);
  return launch<H, 256, 16, 3, 2, 16, BOX>(p, maps, stream);
}

template <typename H>
cudaError_t by_box(Launch& p, int box, int rows, const CUtensorMap (&maps)[3], cudaStream_t stream) {
  return box == 16 ? by_size<H, 16>(p, rows, maps, stream) : (box == 8 ? by_size<H, 8>(p, rows, maps, stream) : by_size<H, 0>(p, rows, maps, stream));
}

}  // namespace

size_t paged_attention_workspace(const PagedAttentionArgs& a) {
  if (whole(a)) return 0;
  return open_bytes() + static_cast<size_t>(sm_count()) * 2 * rows_of(a) * (2 + padded_dim(a.head_dim)) * sizeof(float);
}

cudaError_t paged_attention(const PagedAttentionArgs& args, cudaStream_t stream) {
  if (args.batch <= 0 || args.heads <= 0) return cudaSuccess;
  Launch p;
  p.group = args.heads / args.kv_heads;
  const int rows = rows_of(args), dp = padded_dim(args.head_dim);
  p.head_blocks = Divisor((p.group + rows - 1) / rows);
  p.items = Divisor(args.kv_heads * p.head_blocks.d);
  // positions that are certain to lie in one page: what a TMA box may hold.  Pages of any other size come by 16-byte copies, whose addresses cost a warp some 500
  // instructions per tile (16 ragged sequences, pages of 24: 47 us so, 38 in boxes of 8).
  const int box = args.table.page_size % 16 == 0 ? 16 : (args.table.page_size % 8 == 0 ? 8 : 0);
  p.page_boxes = Divisor(box > 0 ? args.table.page_size / box : 1);
  p.scale_log2 = args.scale * kLog2e;
  p.whole = whole(args) ? 1 : 0;
  p.open = static_cast<int2*>(args.workspace);
  p.part_ml = reinterpret_cast<float*>(static_cast<char*>(args.workspace) + open_bytes());
  p.part_o = p.part_ml + static_cast<size_t>(sm_count()) * 2 * rows * 2;
  p.err = gemm_error_device_ptr();
  CUtensorMap maps[3] = {};
  const bool paged = box > 0 && encode_pages(&maps[0], args.k_pages, args, dp, box) && encode_pages(&maps[1], args.v_pages, args, dp, box);
  // tiles of a launch are counted in 32 bits: as many sequences as cannot have more (a product with the blocks' number is among the sums)
  const long long most = (static_cast<long long>(args.table.width) * args.table.page_size / kBlock + 1) * p.items.d, room = 0x7f000000ll / most;
  if (room < 1) return cudaErrorInvalidValue;
  const int step = room < kSequences ? static_cast<int>(room) : kSequences;
  for (int b = 0; b < args.batch; b += step) {
    p.a = args;
    p.a.batch = args.batch - b < step ? args.batch - b : step;
    p.a.lengths = args.lengths + b;
    p.a.table.p = args.table.p + b * args.table.stride;
    p.a.q.p = static_cast<const char*>(args.q.p) + b * args.q.token * 2;
    p.a.o = static_cast<char*>(args.o) + static_cast<long long>(b) * args.heads * args.head_dim * 2;
    p.a.lse = args.lse ? args.lse + static_cast<long long>(b) * args.heads : nullptr;
    const bool tma = paged && encode_queries(&maps[2], p.a, dp, rows);
    const cudaError_t rc = args.type == Half16::bf16 ? by_box<Bf16>(p, tma ? box : 0, rows, maps, stream) : by_box<Fp16>(p, tma ? box : 0, rows, maps, stream);
    if (rc != cudaSuccess) return rc;
  }
  return cudaSuccess;
}

}  // namespace ops
}  // namespace mccl
