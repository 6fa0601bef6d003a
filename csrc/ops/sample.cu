// The choice of a token per row of logits from a given random number, under temperature, top-k, top-p and min-p.
//
// Nothing is sorted.  What is kept is a beginning of the tokens in the order (likeliest first, lowest number among equals), so one border says it all:
// tokens up to it are kept.  A row belongs to a cluster of 1 to 8 blocks whose warps have neighbouring parts of it:
//   1. maximum (and whether anything is not finite)
//   2. where there is a top-k or top-p: counts and sums of weights over 2048 equal steps of the logit; the border's step is found from their running sums,
//      and the few tokens in it are brought together and sorted (a step with too many is divided again, by logit and number, until it has few enough)
//   3. sums of the kept weights per warp; the warp in whose part the random number falls goes through it once more
// Where all tokens that min-p keeps do not fill the share of top-p, none of them lies behind its border: then the sums come with the counts, and nothing is searched
// (64 x 128000 fp32 with settings per row: 69 -> 47 us, 52 with the weights as exact as they are now).
// Weights are whole numbers, exp((l - max) / T) 2^43 rounded, and their sums are exact: nothing depends on the order in which they are added, and the running
// sum of 100000 tokens is off by 1e-11 of itself where sums of fp32 would be off by more than a token's weight.
//
// What bounds it: for one row the chain of passes and barriers (32000 tokens under top-k 50 and top-p 0.9: 11.6 us; maximum 1.1, barrier 0.6, counts 2.1, their sum over 8
// blocks 1.5, border 0.9, list 1.7, the choice among 50 3), for many the instructions: some 125 per token in all passes (64 x 128000 under top-p 0.95 and min-p
// 0.01), at 58 % of the issue slots; 10 us of them for a pass itself, 13 for the weights, 6 for the additions in shared memory.
#include "../core/launch.hpp"
#include "half16.cuh"
#include "ops.hpp"
#include "packed.hpp"
#include "smem_limit.hpp"

#include <cooperative_groups.h>

#include <climits>

namespace mccl {
namespace ops {

namespace {

namespace cg = cooperative_groups;
using u64 = unsigned long long;

constexpr int kThreads = 512, kWarps = kThreads / 32, kMost = 8;   // blocks per row at most
constexpr int kBins = 2048, kList = 1024;
constexpr int kOne = 43;             // a weight of one is 2^43: the sum of 2^20 of them stays below 2^63
constexpr float kReach = 30.6f;      // exp(-30.6) 2^43 is below one half (44 powers of two are 30.5)
constexpr double kLog2e = 1.4426950408889634;

struct Histogram {
  unsigned count[kBins];
  u64 sum[kBins];
};
// A block's own: sums in three parts of 15 bits, whose 32-bit words hold those of 2^17 weights (one 64-bit addition in shared memory is a loop of exchanges).
constexpr int kPart = 15, kBlockTokens = 1 << 17;
struct Parts {
  unsigned count[kBins];
  unsigned sum[3][kBins];
};
// Where a border lies: the interval, what is in front of it, how many are in it.
struct Border {
  u64 lo, hi;      // of composite keys (levels behind the first)
  u64 sum;         // weights in front
  int bin, count, inside;
  int found;
};
struct Shared {
  Parts mine;
  Histogram merged;                    // in the first block: over the whole row
  u64 list[kList];
  u64 weights[kList];
  u64 best[kMost];                     // per block: the likeliest (composite key)
  int strange[kMost];
  u64 low[kMost], high[kMost];
  u64 total[kMost];
  u64 strong[kMost];                   // per block: the sum of weights of min_p and more, ...
  u64 warp_strong[kWarps];             // ... and per warp
  u64 scan[kWarps];
  unsigned scan_count[kWarps];
  u64 warp_sum[kWarps];
  Border border;
  u64 result;
  int place;
  unsigned listed;
  double enough;                       // in the first block: the sum of weights that top-p asks for
  u64 power[64];                       // 2^(j / 64) 2^43
};

template <typename T>
__device__ __forceinline__ float value_of(T x);
template <>
__device__ __forceinline__ float value_of(float x) { return x; }
template <>
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }

// A number whose order is that of values.  (-0 counts as +0; below that of -inf and above that of +inf are NaNs.)
__device__ __forceinline__ unsigned rising(float x) {
  unsigned b = __float_as_uint(x);
  if (b == 0x80000000u) b = 0;
  return b ^ (static_cast<unsigned>(static_cast<int>(b) >> 31) | 0x80000000u);
}
constexpr unsigned kPlusInfinity = 0xff800000u, kMinusInfinity = 0x007fffffu;
// Ascending order of this number is descending order of values, then ascending of token numbers.
__device__ __forceinline__ u64 composite(float x, int i) { return (static_cast<u64>(~rising(x)) << 32) | static_cast<unsigned>(i); }
__device__ __forceinline__ float value_of_key(u64 c) {
  const unsigned up = ~static_cast<unsigned>(c >> 32);
  return __uint_as_float((up & 0x80000000u) ? (up & 0x7fffffffu) : ~up);
}

// Weights of a row, 2^(t / 64) 2^43 rounded for t = (x - max) 64 / (T ln 2), in 32-bit arithmetic (in fp64 a pass over 64 x 128000 logits took 82 us): a table of 64 powers and a
// Taylor series for what is left, from whose first term on everything is carried in two parts.  Before its last rounding a weight is off by less than 2^-36 of itself.  (In one part of
// 30 bits it was 2^-29.1, and 64 x 128000 logits under top-p and min-p took 47 us where they take 52.)
struct Scale {
  float max, per, per_low;    // the factor in two parts
  const u64* power;           // 2^(j / 64) 2^43, 64 of them
  __device__ __forceinline__ bool some(float x) const { return __fmul_rn(__fsub_rn(x, max), per) > -64.f * 44.f; }
  // x for which some() holds
  __device__ __forceinline__ u64 weight(float x) const {
    constexpr double kStep = 0.6931471805599453 / 64.0;
    constexpr float kHigh = static_cast<float>(kStep), kLow = static_cast<float>(kStep - static_cast<double>(kHigh));
    // x - max and its product with the factor, each with what rounding leaves: t and t_low are off by less than 2^-36 together
    const float d = __fsub_rn(x, max), back = __fsub_rn(d, x);
    const float d_low = __fsub_rn(__fsub_rn(x, __fsub_rn(d, back)), __fadd_rn(max, back));
    const float t = __fmul_rn(d, per);
    const float t_low = fmaf(d_low, per, fmaf(d, per_low, fmaf(d, per, -t)));
    // t = 64 n + j + f with |f| <= 1/2, and t_low
    const float r = __fadd_rn(t, 12582912.f);   // 1.5 2^23: the sum's last bit is worth one
    const int whole = __float_as_int(r) - 0x4b400000;
    const float f = __fsub_rn(t, __fsub_rn(r, 12582912.f));
    // 2^((f + t_low) / 64) - 1 = z + z^2 / 2 + z^3 / 6 + z^4 / 24 (the next term is below 2^-44), as a whole number of 2^-38: |z| < 2^-7.5, and what follows its first part is below 2^-15
    const float high = __fmul_rn(f, kHigh);
    const float low = fmaf(t_low, kHigh, fmaf(f, kLow, fmaf(f, kHigh, -high)));
    const float z = __fadd_rn(high, low);
    const float rest = fmaf(__fmul_rn(z, z), fmaf(z, fmaf(z, 1.f / 24.f, 1.f / 6.f), 0.5f), low);
    const int more = __float2int_rn(high * 274877906944.f) + __float2int_rn(rest * 274877906944.f);
    const u64 p = power[whole & 63];
    const u64 w = p + static_cast<u64>((static_cast<long long>(static_cast<int>(p >> 13)) * more) >> (38 + 30 - kOne));
    // w 2^n, rounded
    return ((w << 1 >> -(whole >> 6)) + 1) >> 1;
  }
};

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) v += __shfl_xor_sync(0xffffffffu, v, s);
  return v;
}
__device__ __forceinline__ u64 warp_min(u64 v) {
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) v = min(v, __shfl_xor_sync(0xffffffffu, v, s));
  return v;
}

// A warp's part [lo, hi) of the row, in order: f(value, number, valid) by whole warps, V neighbouring tokens per lane and step.  Several steps' loads are under
// way together (one at a time 17 us for the maximum of 64 x 128000).
template <typename T, int V, typename F>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, F f) {
  constexpr int kSteps = V == 1 ? 4 : 16 / V;
  const int lane = threadIdx.x & 31;
  for (int base = lo; base < hi; base += 32 * V * kSteps) {
    const int i0 = base + lane * V;
    if constexpr (V == 1) {
      T x[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k)
        if (i0 + 32 * k < hi) x[k] = row[i0 + 32 * k];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) f(value_of<T>(x[k]), i0 + 32 * k, i0 + 32 * k < hi);
    } else {
      uint4 raw[kSteps];
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int i = i0 + 32 * V * k;
        if (i + V <= hi) {
          raw[k] = *reinterpret_cast<const uint4*>(row + i);
        } else {
          raw[k] = make_uint4(0u, 0u, 0u, 0u);
          T* x = reinterpret_cast<T*>(&raw[k]);
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (i + e < hi) x[e] = row[i + e];
        }
      }
#pragma unroll
      for (int k = 0; k < kSteps; ++k) {
        const int i = i0 + 32 * V * k;
        const T* x = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) f(value_of<T>(x[e]), i + e, i + e < hi);
      }
    }
  }
}

template <bool WEIGHTS>
__device__ __forceinline__ void add(Parts& h, int bin, u64 w) {
  atomicAdd(&h.count[bin], 1u);
  if (WEIGHTS) {
    atomicAdd(&h.sum[0][bin], static_cast<unsigned>(w) & ((1u << kPart) - 1));
    atomicAdd(&h.sum[1][bin], static_cast<unsigned>(w >> kPart) & ((1u << kPart) - 1));
    if (w >> 2 * kPart) atomicAdd(&h.sum[2][bin], static_cast<unsigned>(w >> 2 * kPart));   // (seldom: 1e-4 of the likeliest token's weight and more)
  }
}
template <bool WEIGHTS>
__device__ __forceinline__ void clear(Parts& h) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    h.count[b] = 0;
    if (WEIGHTS) h.sum[0][b] = h.sum[1][b] = h.sum[2][b] = 0;
  }
}

// list[0 .. n) of different numbers in ascending order; by a block.  Up to kThreads numbers each thread counts how many are smaller than its own (n steps without a barrier:
// 50 numbers 0.4 us, 2.4 in a network), more go through a bitonic network, with the highest number behind them.
__device__ __forceinline__ void sort(u64* list, int n) {
  const int tid = static_cast<int>(threadIdx.x);
  if (n <= kThreads) {
    const u64 x = tid < n ? list[tid] : 0;
    int rank = 0;
    if (tid < n) {
#pragma unroll 8
      for (int j = 0; j < n; ++j) rank += list[j] < x ? 1 : 0;
    }
    __syncthreads();
    if (tid < n) list[rank] = x;
    __syncthreads();
    return;
  }
  for (int i = n + tid; i < kList; i += kThreads) list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= kList; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < kList / 2; i += kThreads) {
        const int a = 2 * i - (i & (j - 1)), o = a + j;
        const u64 x = list[a], y = list[o];
        if ((x > y) == ((a & k) == 0)) {
          list[a] = y;
          list[o] = x;
        }
      }
      __syncthreads();
    }
  }
}

// The first i < n whose running sum of w[0 .. i] is `aim` or more (n without one); by a block, and the whole sum.
__device__ __forceinline__ int first_at(Shared& s, const u64* w, int n, u64 aim, u64& whole) {
  constexpr int kEach = kList / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, base = static_cast<int>(threadIdx.x) * kEach;
  u64 v[kEach], in = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) in += v[e] = base + e < n ? w[base + e] : 0;
  const u64 mine = in;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += x;
  }
  if (lane == 31) s.scan[warp] = in;
  if (threadIdx.x == 0) s.place = n;
  __syncthreads();
  u64 before = in - mine;
  whole = 0;
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += s.scan[i];
    whole += s.scan[i];
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (base + e < n && before < aim && before + v[e] >= aim) s.place = base + e;   // one thread's
    before += v[e];
  }
  __syncthreads();
  const int at = s.place;
  __syncthreads();
  return at;
}

// The blocks' bins added up in the first block's `merged`.  Begins and ends with a barrier of the cluster.
template <bool WEIGHTS>
__device__ __forceinline__ void merge(cg::cluster_group& cluster, Shared& s) {
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  cluster.sync();
  Shared* first = cluster.map_shared_rank(&s, 0);
  const int share = kBins / blocks;
  for (int b = rank * share + threadIdx.x; b < (rank + 1) * share; b += kThreads) {
    unsigned count = 0;
    u64 sum = 0;
#pragma unroll
    for (int r = 0; r < kMost; ++r) {   // (all loads under way together)
      if (r >= blocks) continue;
      const Shared* other = cluster.map_shared_rank(&s, r);
      count += other->mine.count[b];
      if (WEIGHTS) sum += other->mine.sum[0][b] + (static_cast<u64>(other->mine.sum[1][b]) << kPart) + (static_cast<u64>(other->mine.sum[2][b]) << 2 * kPart);
    }
    first->merged.count[b] = count;
    if (WEIGHTS) first->merged.sum[b] = sum;
  }
  cluster.sync();
}

template <typename T, int V>
struct Row {
  const T* row;
  int lo, hi;   // this warp's part
  Scale scale;
  float steps, most;   // bins of the first level per unit of logit, and the maximum
  float temperature;
  int vocab;
  u64 least;           // min_p as a weight (0: none)

  __device__ __forceinline__ int bin(float x) const {
    const int b = static_cast<int>((most - x) * steps);   // both grow together: rounding keeps the order
    return b < 0 ? 0 : (b < kBins ? b : kBins - 1);
  }

  // A logit from which on all weights are (1 - share) / 2 / vocab or more (rounded down: it may lie below).
  __device__ __forceinline__ float deep_below(float share) const {
    return __fsub_rd(most, __fmul_ru(temperature, logf(2.f * static_cast<float>(vocab) / (1.f - share))));
  }

  // First block only, all threads: the first bin at whose end `need` tokens (with WEIGHTS: share of all blocks' weights, or s.enough of them) have been passed, behind
  // count0 tokens and weights of sum0; s.border has it, or found = 0.
  template <bool WEIGHTS>
  __device__ __forceinline__ static void find_bin(Shared& s, int blocks, int count0, u64 sum0, unsigned need, float share) {
    constexpr int kEach = kBins / kThreads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned c[kEach], count = 0;
    u64 w[kEach], sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      c[e] = s.merged.count[threadIdx.x * kEach + e];
      w[e] = WEIGHTS ? s.merged.sum[threadIdx.x * kEach + e] : 0;
      count += c[e];
      sum += w[e];
    }
    unsigned in_count = count;
    u64 in_sum = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned a = __shfl_up_sync(0xffffffffu, in_count, o);
      const u64 b = WEIGHTS ? __shfl_up_sync(0xffffffffu, in_sum, o) : 0;
      if (lane >= o) {
        in_count += a;
        in_sum += b;
      }
    }
    if (lane == 31) {
      s.scan_count[warp] = in_count;
      s.scan[warp] = in_sum;
    }
    if (threadIdx.x == 0) s.border.found = 0;
    __syncthreads();
    if (WEIGHTS && share >= 0.f) {   // a token is kept while the weights in front of it are below the share of all: the border is where they are reached
      u64 all = 0;
      for (int i = 0; i < blocks; ++i) all += s.total[i];
      if (threadIdx.x == 0) s.enough = static_cast<double>(share) * static_cast<double>(all);
      __syncthreads();
    }
    unsigned before = static_cast<unsigned>(count0) + in_count - count;
    u64 before_sum = sum0 + in_sum - sum;
    for (int i = 0; i < warp; ++i) {
      before += s.scan_count[i];
      before_sum += s.scan[i];
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      if (c[e] > 0 && !reached<WEIGHTS>(s, before, before_sum, need) && reached<WEIGHTS>(s, before + c[e], before_sum + w[e], need)) {   // one thread's at most: both grow
        s.border.bin = threadIdx.x * kEach + e;
        s.border.count = static_cast<int>(before);
        s.border.sum = before_sum;
        s.border.inside = static_cast<int>(c[e]);
        s.border.found = 1;
      }
      before += c[e];
      before_sum += w[e];
    }
    __syncthreads();
  }
  template <bool WEIGHTS>
  __device__ __forceinline__ static bool reached(const Shared& s, unsigned count, u64 sum, unsigned need) {
    return WEIGHTS ? count > 0 && static_cast<double>(sum) >= s.enough : count >= need;
  }

  // The first block has all candidates in its list: the choice among them.  need: top-k (0: none); share: top-p of the sum of these (1: none, below 0: s.enough);
  // weights below `least` do not count.
  __device__ long long choose(Shared& s, int n, unsigned need, float share, u64 least, double u) const {
    sort(s.list, n);
    int kept = need > 0 ? min(n, static_cast<int>(need)) : n;
    for (int i = threadIdx.x; i < kept; i += kThreads) s.weights[i] = scale.weight(value_of_key(s.list[i]));
    __syncthreads();
    u64 whole;
    if (share < 1.f) {
      double enough = s.enough;
      if (share >= 0.f) {
        first_at(s, s.weights, kept, 0, whole);
        enough = static_cast<double>(share) * static_cast<double>(whole);
      }
      // the first that reaches it stays, whatever it asks for
      kept = min(kept, first_at(s, s.weights, kept, static_cast<u64>(max(1ll, static_cast<long long>(ceil(enough)))), whole) + 1);
    }
    // by number
    for (int i = threadIdx.x; i < kept; i += kThreads) s.list[i] = (s.list[i] << 32) | static_cast<unsigned>(i);
    __syncthreads();
    sort(s.list, kept);
    u64 mine[kList / kThreads];
#pragma unroll
    for (int e = 0; e < kList / kThreads; ++e) {
      const int i = static_cast<int>(threadIdx.x) + e * kThreads;
      mine[e] = i < kept ? s.weights[s.list[i] & 0xffffffffu] : 0;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kList / kThreads; ++e) s.weights[threadIdx.x + e * kThreads] = mine[e] < least ? 0 : mine[e];
    __syncthreads();
    first_at(s, s.weights, kept, 0, whole);
    const double at = u * static_cast<double>(whole);
    const u64 aim = at > 0.0 ? min(static_cast<u64>(at), whole - 1) : 0;
    return static_cast<long long>(s.list[first_at(s, s.weights, kept, aim + 1, whole)] >> 32);
  }

  // The composite key of the last token kept: the need-th (fewer tokens: none, ~0), or with WEIGHTS the one that reaches `share` of the weights, among those
  // up to `limit`.  The same in all blocks.  `few` is called instead, in all blocks, where the first one can have all candidates up to it in its list; it has
  // then been told how many there are.  summed: min_p keeps no token that top-p would not, and s.warp_sum has the warps' sums of what is kept.
  template <bool WEIGHTS, typename F>
  __device__ u64 find(cg::cluster_group& cluster, Shared& s, u64 limit, unsigned need, float share, bool& done, bool& summed, F few) const {
    const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Shared* first = cluster.map_shared_rank(&s, 0);
    auto tell = [&] {   // the first block's border to all
      if (rank == 0 && static_cast<int>(threadIdx.x) < blocks && threadIdx.x > 0) cluster.map_shared_rank(&s, threadIdx.x)->border = s.border;
      if (rank == 0 && threadIdx.x == 0) s.listed = 0;
      cluster.sync();
    };
    const bool limited = limit != ~0ull;
    clear<WEIGHTS>(s.mine);
    __syncthreads();
    // All tokens with weights below (1 - share) / 2 / vocab together are less than half of what lies behind the border: they count in the sum of all, but it is not
    // among them, and they are not counted in their bins.
    const int deep = WEIGHTS ? bin(deep_below(share)) : kBins - 1;   // (whole bins: what is counted is what is found again)
    u64 all = 0, strong = 0;
    walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
      if (valid && scale.some(x) && (!limited || composite(x, i) <= limit)) {
        const u64 w = WEIGHTS ? scale.weight(x) : 0;
        if (WEIGHTS) all += w;
        if (WEIGHTS && w >= least) strong += w;
        const int at = bin(x);
        if (at <= deep) add<WEIGHTS>(s.mine, at, w);
      }
    });
    if (WEIGHTS) {
      all = warp_sum(all);
      strong = warp_sum(strong);
      if (lane == 0) {
        s.warp_sum[warp] = all;
        s.warp_strong[warp] = strong;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int i = 1; i < kWarps; ++i) {
          all += s.warp_sum[i];
          strong += s.warp_strong[i];
        }
        first->total[rank] = all;
        first->strong[rank] = strong;
      }
    }
    merge<WEIGHTS>(cluster, s);
    if (rank == 0) {
      find_bin<WEIGHTS>(s, blocks, 0, 0, need, share);
      if (WEIGHTS && threadIdx.x == 0 && least > 0) {   // all tokens that min_p keeps do not fill the share: the border lies behind them (with room for these roundings)
        u64 kept = 0;
        for (int i = 0; i < blocks; ++i) kept += s.strong[i];
        if (static_cast<double>(kept) * (1.0 + 1e-15) <= s.enough) s.border.found = 2;
      }
      __syncthreads();
    }
    tell();
    if (!s.border.found) return ~0ull;
    if (s.border.found == 2) {
      if (threadIdx.x < kWarps) s.warp_sum[threadIdx.x] = s.warp_strong[threadIdx.x];
      summed = true;
      return limit;
    }
    bool level = true;   // still the first
    Border b = s.border;
    if (!limited && b.count + b.inside <= kList) {
      walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
        if (valid && scale.some(x) && bin(x) <= b.bin) {
          const unsigned at = atomicAdd(&first->listed, 1u);
          if (at < kList) first->list[at] = composite(x, i);
        }
      });
      cluster.sync();
      if (rank == 0) few(b.count + b.inside);
      done = true;
      return 0;
    }
    auto member = [&](float x, int i, u64& c) {
      c = composite(x, i);
      return level ? scale.some(x) && bin(x) == b.bin && c <= limit : c >= b.lo && c <= b.hi;
    };
    while (b.inside > kList) {
      u64 low = ~0ull, high = 0;
      walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
        u64 c;
        if (valid && member(x, i, c)) {
          low = min(low, c);
          high = max(high, c);
        }
      });
      low = warp_min(low);
      high = ~warp_min(~high);
      if (lane == 0) {
        s.scan[warp] = low;
        s.warp_sum[warp] = high;
      }
      clear<WEIGHTS>(s.mine);
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < blocks) {
        u64 l = ~0ull, h = 0;
        for (int i = 0; i < kWarps; ++i) {
          l = min(l, s.scan[i]);
          h = max(h, s.warp_sum[i]);
        }
        Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
        other->low[rank] = l;
        other->high[rank] = h;
      }
      cluster.sync();
      low = s.low[0];
      high = s.high[0];
      for (int i = 1; i < blocks; ++i) {
        low = min(low, s.low[i]);
        high = max(high, s.high[i]);
      }
      int shift = 0;
      while (((high - low) >> shift) >= kBins) ++shift;
      walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
        u64 c;
        if (valid && member(x, i, c)) add<WEIGHTS>(s.mine, static_cast<int>((c - low) >> shift), WEIGHTS ? scale.weight(x) : 0);
      });
      merge<WEIGHTS>(cluster, s);
      if (rank == 0) {
        find_bin<WEIGHTS>(s, blocks, b.count, b.sum, need, -1.f);
        if (threadIdx.x == 0) {
          s.border.lo = low + (static_cast<u64>(s.border.bin) << shift);
          s.border.hi = min(high, s.border.lo + ((1ull << shift) - 1));
        }
        __syncthreads();
      }
      tell();
      level = false;
      b = s.border;
    }
    walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
      u64 c;
      if (valid && member(x, i, c)) {
        const unsigned at = atomicAdd(&first->listed, 1u);
        if (at < kList) first->list[at] = c;
      }
    });
    cluster.sync();
    if (rank == 0) {
      sort(s.list, b.inside);
      if (threadIdx.x < 32) {
        u64 sum = b.sum;
        for (int base = 0; base < b.inside; base += 32) {
          const int i = base + lane;
          u64 in = WEIGHTS && i < b.inside ? scale.weight(value_of_key(s.list[i])) : 0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += x;
          }
          const unsigned there = __ballot_sync(0xffffffffu, i < b.inside && reached<WEIGHTS>(s, static_cast<unsigned>(b.count + i + 1), sum + in, need));
          if (there) {
            if (lane < blocks) cluster.map_shared_rank(&s, lane)->result = s.list[base + __ffs(there) - 1];
            break;
          }
          sum += __shfl_sync(0xffffffffu, in, 31);
        }
      }
    }
    cluster.sync();
    return s.result;
  }
};

template <typename T>
__device__ __forceinline__ T setting(const RowSetting<T>& s, int row) { return s.each != nullptr ? s.each[row] : s.all; }

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(gridDim.z), rank = static_cast<int>(blockIdx.z), line = static_cast<int>(blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 64) s.power[threadIdx.x] = static_cast<u64>(__double2ll_rn(exp2(static_cast<double>(threadIdx.x) / 64.0) * static_cast<double>(1ull << kOne)));
  cluster.sync();   // all blocks are there: their memory may be written
  pdl_wait();
  pdl_trigger();
  const int warps = blocks * kWarps, part = ((a.vocab + warps - 1) / warps + 7) / 8 * 8;
  Row<T, V> r;
  r.row = static_cast<const T*>(a.logits) + line * a.stride;
  r.lo = min(a.vocab, (rank * kWarps + warp) * part);
  r.hi = min(a.vocab, r.lo + part);

  // ---- the likeliest, and the range
  unsigned top = 0, bottom = ~0u;
  int top_at = 0;
  walk<T, V>(r.row, r.lo, r.hi, [&](float x, int i, bool valid) {
    if (!valid) return;
    const unsigned up = rising(x);
    bottom = min(bottom, up);
    if (up > top) {   // a lane's numbers ascend: the first of equals stays
      top = up;
      top_at = i;
    }
  });
  u64 best = (static_cast<u64>(~top) << 32) | static_cast<unsigned>(top_at);   // (a warp without tokens: a NaN's, behind all values)
  bool strange = top >= kPlusInfinity || bottom < kMinusInfinity;
  best = warp_min(best);
  strange = __any_sync(0xffffffffu, strange);
  if (lane == 0) {
    s.scan[warp] = best;
    s.scan_count[warp] = strange ? 1 : 0;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < blocks) {
    int odd = 0;
    for (int i = 0; i < kWarps; ++i) {
      best = min(i == 0 ? ~0ull : best, s.scan[i]);
      odd |= static_cast<int>(s.scan_count[i]);
    }
    Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
    other->best[rank] = best;
    other->strange[rank] = odd;
  }
  cluster.sync();
  best = s.best[0];
  int odd = s.strange[0];
  for (int i = 1; i < blocks; ++i) {
    best = min(best, s.best[i]);
    odd |= s.strange[i];
  }
  const float temperature = setting(a.temperature, line), most = value_of_key(best);
  // (nothing reads another block's memory from here on unless it has passed another barrier: a block may leave)
  if (odd || __float_as_uint(most) == 0xff800000u || !(temperature >= 0.f)) {
    if (rank == 0 && threadIdx.x == 0) a.tokens[line] = -1;
    return;
  }
  if (temperature < 1e-36f) {   // zero, or so small that the factor of the logits is no number of 32 bits (from 2.7e-37 down)
    if (rank == 0 && threadIdx.x == 0) a.tokens[line] = static_cast<long long>(best & 0xffffffffu);
    return;
  }
  r.most = most;
  r.temperature = temperature;
  r.vocab = a.vocab;
  const double per = 64.0 * kLog2e / static_cast<double>(temperature);
  r.scale = {most, static_cast<float>(per), static_cast<float>(per - static_cast<double>(static_cast<float>(per))), s.power};
  r.steps = static_cast<float>(kBins) / (kReach * temperature);

  // ---- the border
  const int k = setting(a.top_k, line);
  const float top_p = setting(a.top_p, line);
  const float min_p = setting(a.min_p, line);
  const u64 least = min_p > 0.f ? static_cast<u64>(ceil(static_cast<double>(min(min_p, 1.f)) * static_cast<double>(1ull << kOne))) : 0;
  const double u = a.uniform64 ? static_cast<const double*>(a.uniform)[line] : static_cast<double>(static_cast<const float*>(a.uniform)[line]);
  u64 border = ~0ull;
  r.least = least;
  bool done = false, summed = false;
  if (k > 0 && k < a.vocab) {
    border = r.template find<false>(cluster, s, border, static_cast<unsigned>(k), 0.f, done, summed, [&](int n) {
      const long long token = r.choose(s, n, static_cast<unsigned>(k), top_p < 1.f ? fmaxf(top_p, 0.f) : 1.f, least, u);
      if (threadIdx.x == 0) a.tokens[line] = token;
    });
  }
  if (top_p < 1.f && !done) {
    const u64 limit = border;
    border = min(limit, r.template find<true>(cluster, s, limit, 0, fmaxf(top_p, 0.f), done, summed, [&](int n) {
      const long long token = r.choose(s, n, 0, -1.f, least, u);
      if (threadIdx.x == 0) a.tokens[line] = token;
    }));
  }
  if (done) return;

  // ---- the choice
  const bool limited = border != ~0ull;
  // logits below this are none of the kept ones: the border's, or half of min_p (which the weights below decide on)
  const float low = fmaxf(limited ? value_of_key(border) : -INFINITY, min_p > 0.f ? __fadd_rd(most, __fmul_rd(temperature, logf(0.5f * fminf(min_p, 1.f)))) : -INFINITY);
  auto kept = [&](float x, int i) -> u64 {
    if (!(x >= low) || !r.scale.some(x) || (limited && composite(x, i) > border)) return 0;
    const u64 w = r.scale.weight(x);
    return w < least ? 0 : w;
  };
  if (!summed) {
    u64 sum = 0;
    walk<T, V>(r.row, r.lo, r.hi, [&](float x, int i, bool valid) { sum += valid ? kept(x, i) : 0; });
    sum = warp_sum(sum);
    if (lane == 0) s.warp_sum[warp] = sum;
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < blocks) {
    u64 all = 0;
    for (int i = 0; i < kWarps; ++i) all += s.warp_sum[i];
    cluster.map_shared_rank(&s, threadIdx.x)->total[rank] = all;
  }
  cluster.sync();
  u64 total = 0, before = 0;
  for (int i = 0; i < blocks; ++i) {
    if (i < rank) before += s.total[i];
    total += s.total[i];
  }
  // the first token at whose end the running sum is above this
  const double at = u * static_cast<double>(total);
  const u64 aim = at > 0.0 ? min(static_cast<u64>(at), total - 1) : 0;
  if (!(aim >= before && aim < before + s.total[rank])) return;   // whole blocks
  // the warp whose part it falls into; all threads take a few neighbouring tokens of that part
  int owner = 0;
  while (aim >= before + s.warp_sum[owner]) before += s.warp_sum[owner++];
  const int begin = min(a.vocab, (rank * kWarps + owner) * part), end = min(a.vocab, begin + part), each = (end - begin + kThreads - 1) / kThreads;
  const int lo = min(end, begin + static_cast<int>(threadIdx.x) * each), hi = min(end, lo + each);
  u64 mine = 0;
  for (int i = lo; i < hi; ++i) mine += kept(value_of<T>(r.row[i]), i);
  u64 in = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += x;
  }
  if (lane == 31) s.scan[warp] = in;
  __syncthreads();
  before += in - mine;
  for (int i = 0; i < warp; ++i) before += s.scan[i];
  if (aim >= before && aim < before + mine) {
    int i = lo;
    for (;; ++i) {
      before += kept(value_of<T>(r.row[i]), i);
      if (before > aim) break;
    }
    a.tokens[line] = i;
  }
}

template <typename T, int V>
cudaError_t launch(const SampleArgs& a, cudaStream_t stream) {
  // blocks per row: as many as leave no SM idle, with some 2000 tokens each and no more than a block may add up
  int blocks = 1;
  while (a.vocab > blocks * kBlockTokens) blocks *= 2;
  while (blocks < kMost && static_cast<long long>(a.rows) * blocks * 2 <= 2 * 148 && a.vocab / blocks > 4096) blocks *= 2;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t rc = raise_smem_limit(sample_kernel<T, V>, sizeof(Shared), allowed);
  if (rc != cudaSuccess) return rc;
  MCCL_LAUNCH_PDL_CLUSTER((sample_kernel<T, V>), dim3(a.rows, 1, blocks), kThreads, sizeof(Shared), stream, blocks, a);
  count_launch();
  return ::mccl::launch_status();
}

template <typename T>
cudaError_t by_alignment(const SampleArgs& a, cudaStream_t stream) {
  constexpr int kVector = 16 / sizeof(T);
  const bool aligned = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && (a.rows <= 1 || a.stride % kVector == 0);
  return aligned ? launch<T, kVector>(a, stream) : launch<T, 1>(a, stream);
}

}  // namespace

cudaError_t sample(const SampleArgs& a, cudaStream_t stream) {
  if (a.rows <= 0) return cudaSuccess;
  if (a.vocab <= 0 || a.vocab > (1 << 20)) return cudaErrorInvalidValue;
  switch (a.type) {
    case Logits::bf16: return by_alignment<__nv_bfloat16>(a, stream);
    case Logits::fp16: return by_alignment<__half>(a, stream);
    default: return by_alignment<float>(a, stream);
  }
}

}  // namespace ops
}  // namespace mccl
