// The choice of a token per row of logits from a given random number, under temperature, top-k, top-p and min-p.
//
// Nothing is sorted.  What is kept is a beginning of the tokens in the order (likeliest first, lowest number among equals), so one border says it all:
// tokens up to it are kept.  A row belongs to a cluster of 1 to 8 blocks whose warps have neighbouring parts of it:
//   1. maximum (and whether anything is not finite)
//   2. where there is a top-k or top-p: counts and sums of weights over 2048 equal steps of the logit; the border's step is found from their running sums,
//      and the few tokens in it are brought together and sorted (a step with too many is divided again, by logit and number, until it has few enough)
//   3. sums of the kept weights per warp; the warp in whose part the random number falls goes through it once more
// Weights are whole numbers, exp((l - max) / T) 2^43 rounded, and their sums are exact: nothing depends on the order in which they are added, and the running
// sum of 100000 tokens is off by 1e-11 of itself where sums of fp32 would be off by more than a token's weight.
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
constexpr float kReach = 30.6f;      // exp(-30.6) 2^43 is below one half
constexpr double kLog2e = 1.4426950408889634;

struct Histogram {
  unsigned count[kBins];
  u64 sum[kBins];
};
// Where a border lies: the interval, what is in front of it, how many are in it.
struct Border {
  u64 lo, hi;      // of composite keys (levels behind the first)
  u64 sum;         // weights in front
  int bin, count, inside;
  int found;
};
struct Shared {
  Histogram mine, merged;              // merged: in the first block, sums over the row; of the first level
  Histogram deeper;                    // ... and of the others
  u64 list[kList];
  u64 weights[kList];
  u64 best[kMost];                     // per block: the likeliest (composite key)
  float least[kMost];
  int strange[kMost];
  u64 low[kMost], high[kMost];
  u64 total[kMost];
  u64 scan[kWarps];
  unsigned scan_count[kWarps];
  u64 warp_sum[kWarps];
  Border border;
  u64 result, result_sum;
  unsigned listed;
  double power[64];                    // 2^(j / 64)
};

template <typename T>
__device__ __forceinline__ float value_of(T x);
template <>
__device__ __forceinline__ float value_of(float x) { return x; }
template <>
__device__ __forceinline__ float value_of(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float value_of(__half x) { return __half2float(x); }

// Ascending order of this number is descending order of values, then ascending of token numbers.  (-0 counts as +0.)
__device__ __forceinline__ u64 composite(float x, int i) {
  unsigned b = __float_as_uint(x);
  if (b == 0x80000000u) b = 0;
  const unsigned up = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<u64>(~up) << 32) | static_cast<unsigned>(i);
}
__device__ __forceinline__ float value_of_key(u64 c) {
  const unsigned up = ~static_cast<unsigned>(c >> 32);
  return __uint_as_float((up & 0x80000000u) ? (up & 0x7fffffffu) : ~up);
}

// Weights of a row.
struct Scale {
  double max, per;   // 64 / (T ln 2)
  const double* power;
  // 2^(t / 64) 2^43 for t = (x - max) per, rounded: t = 64 n + j + f with |f| <= 1/2, 2^(f / 64) by its series up to the fourth power (the next term is 2^-47)
  __device__ __forceinline__ u64 weight(float x) const {
    const double t = (static_cast<double>(x) - max) * per;
    if (!(t > -64.0 * 44.5)) return 0;
    const double round = 6755399441055744.0;   // 1.5 2^52: the sum's last bit is worth one
    const double r = t + round;
    const int whole = __double2loint(r);
    const double z = (t - (r - round)) * (0.6931471805599453 / 64.0);
    const double q = z * (1.0 + z * (0.5 + z * (1.0 / 6.0 + z * (1.0 / 24.0))));
    double p = power[whole & 63];
    p = p + p * q;
    return __double2ull_rn(__hiloint2double(__double2hiint(p) + (((whole >> 6) + kOne) << 20), __double2loint(p)));
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

// A warp's part [lo, hi) of the row, in order: f(value, number, valid) by whole warps, V neighbouring tokens per lane and step.
template <typename T, int V, typename F>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, F f) {
  const int lane = threadIdx.x & 31;
  for (int base = lo; base < hi; base += 32 * V) {
    const int i = base + lane * V;
    if constexpr (V == 1) {
      f(i < hi ? value_of<T>(row[i]) : 0.f, i, i < hi);
    } else {
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      T* x = reinterpret_cast<T*>(&raw);
      if (i + V <= hi) {
        raw = *reinterpret_cast<const uint4*>(row + i);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (i + e < hi) x[e] = row[i + e];
      }
#pragma unroll
      for (int e = 0; e < V; ++e) f(value_of<T>(x[e]), i + e, i + e < hi);
    }
  }
}

// Adds a warp's weights to bins: at once where all lanes have the same bin (rows of equal logits).  bin < 0: nothing.
__device__ __forceinline__ void add(Histogram& h, int bin, u64 w) {
  int same = 0;
  __match_all_sync(0xffffffffu, bin, &same);
  if (same) {
    if (bin < 0) return;
    const u64 sum = warp_sum(w);
    if ((threadIdx.x & 31) == 0) {
      atomicAdd(&h.count[bin], 32u);
      atomicAdd(&h.sum[bin], sum);
    }
  } else if (bin >= 0) {
    atomicAdd(&h.count[bin], 1u);
    atomicAdd(&h.sum[bin], w);
  }
}

__device__ __forceinline__ void clear(Histogram& h) {
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    h.count[b] = 0;
    h.sum[b] = 0;
  }
}

// The blocks' bins added up in the first block's `to`.  Ends with a barrier of the cluster.
__device__ __forceinline__ void merge(cg::cluster_group& cluster, Shared& s, Histogram Shared::*to) {
  const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  cluster.sync();
  Shared* first = cluster.map_shared_rank(&s, 0);
  const int share = kBins / blocks;
  for (int b = rank * share + threadIdx.x; b < (rank + 1) * share; b += kThreads) {
    unsigned count = 0;
    u64 sum = 0;
    for (int r = 0; r < blocks; ++r) {
      const Shared* other = cluster.map_shared_rank(&s, r);
      count += other->mine.count[b];
      sum += other->mine.sum[b];
    }
    (first->*to).count[b] = count;
    (first->*to).sum[b] = sum;
  }
  cluster.sync();
}

// First block only, all threads: the first bin at whose end `reached` is true of (tokens, weights) up to there; s.border has it, or found = 0.
template <typename F>
__device__ __forceinline__ void find_bin(Shared& s, const Histogram& h, int count0, u64 sum0, F reached) {
  constexpr int kEach = kBins / kThreads;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned c[kEach], count = 0;
  u64 w[kEach], sum = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    c[e] = h.count[threadIdx.x * kEach + e];
    w[e] = h.sum[threadIdx.x * kEach + e];
    count += c[e];
    sum += w[e];
  }
  unsigned in_count = count;
  u64 in_sum = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned a = __shfl_up_sync(0xffffffffu, in_count, o);
    const u64 b = __shfl_up_sync(0xffffffffu, in_sum, o);
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
  unsigned before = static_cast<unsigned>(count0) + in_count - count;
  u64 before_sum = sum0 + in_sum - sum;
  for (int i = 0; i < warp; ++i) {
    before += s.scan_count[i];
    before_sum += s.scan[i];
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (c[e] > 0 && !reached(before, before_sum) && reached(before + c[e], before_sum + w[e])) {   // one thread's at most: both grow
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

template <typename T, int V>
struct Row {
  const T* row;
  int lo, hi;   // this warp's part
  Scale scale;
  float steps, most;   // bins of the first level per unit of logit, and the maximum

  __device__ __forceinline__ int bin(float x) const {
    const int b = static_cast<int>((most - x) * steps);   // both grow together: rounding keeps the order
    return b < 0 ? 0 : (b < kBins ? b : kBins - 1);
  }

  // The composite key of the border token and the sum of weights up to and with it, for all blocks.  Called with s.border of the first block (found) from
  // the first level; `reached` as in find_bin.
  template <typename F>
  __device__ void resolve(cg::cluster_group& cluster, Shared& s, F reached, u64& key, u64& sum) const {
    const int blocks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Shared* first = cluster.map_shared_rank(&s, 0);
    auto tell = [&] {   // the first block's border to all
      if (rank == 0 && static_cast<int>(threadIdx.x) < blocks && threadIdx.x > 0) cluster.map_shared_rank(&s, threadIdx.x)->border = s.border;
      if (rank == 0 && threadIdx.x == 0) s.listed = 0;
      cluster.sync();
    };
    tell();
    bool level = true;   // still the first
    while (s.border.inside > kList) {
      const Border b = s.border;
      auto member = [&](float x, int i, u64& c) {
        c = composite(x, i);
        return level ? (bin(x) == b.bin && scale.weight(x) > 0) : (c >= b.lo && c <= b.hi);
      };
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
      clear(s.mine);
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
      for (int i = 0; i < blocks; ++i) {
        low = min(i == 0 ? ~0ull : low, s.low[i]);
        high = max(i == 0 ? 0ull : high, s.high[i]);
      }
      int shift = 0;
      while (((high - low) >> shift) >= kBins) ++shift;
      walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
        u64 c = 0;
        const bool in = valid && member(x, i, c);
        add(s.mine, in ? static_cast<int>((c - low) >> shift) : -1, in ? scale.weight(x) : 0);
      });
      merge(cluster, s, &Shared::deeper);
      if (rank == 0) {
        find_bin(s, s.deeper, b.count, b.sum, reached);
        if (threadIdx.x == 0) {
          s.border.lo = low + (static_cast<u64>(s.border.bin) << shift);
          s.border.hi = min(high, s.border.lo + ((1ull << shift) - 1));
        }
        __syncthreads();
      }
      level = false;
      tell();
    }
    const Border b = s.border;
    walk<T, V>(row, lo, hi, [&](float x, int i, bool valid) {
      if (!valid) return;
      const u64 c = composite(x, i);
      if (level ? (bin(x) == b.bin && scale.weight(x) > 0) : (c >= b.lo && c <= b.hi)) {
        const unsigned at = atomicAdd(&first->listed, 1u);
        if (at < kList) first->list[at] = c;
      }
    });
    cluster.sync();
    if (rank == 0) {
      int n = 32;
      while (n < b.inside) n <<= 1;
      for (int i = b.inside + threadIdx.x; i < n; i += kThreads) s.list[i] = ~0ull;
      __syncthreads();
      for (int k = 2; k <= n; k <<= 1) {   // bitonic
        for (int j = k >> 1; j > 0; j >>= 1) {
          for (int i = threadIdx.x; i < n / 2; i += kThreads) {
            const int a = 2 * i - (i & (j - 1)), o = a + j;
            const u64 x = s.list[a], y = s.list[o];
            if ((x > y) == ((a & k) == 0)) {
              s.list[a] = y;
              s.list[o] = x;
            }
          }
          __syncthreads();
        }
      }
      for (int i = threadIdx.x; i < b.inside; i += kThreads) s.weights[i] = scale.weight(value_of_key(s.list[i]));
      __syncthreads();
      if (threadIdx.x < 32) {
        u64 sum = b.sum;
        for (int base = 0; base < b.inside; base += 32) {
          const int i = base + lane;
          u64 in = i < b.inside ? s.weights[i] : 0;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const u64 x = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += x;
          }
          const unsigned there = __ballot_sync(0xffffffffu, i < b.inside && reached(static_cast<unsigned>(b.count + i + 1), sum + in));
          if (there) {
            const int at = __ffs(there) - 1;
            if (lane == at) {
              s.result = s.list[i];
              s.result_sum = sum + in;
            }
            break;
          }
          sum += __shfl_sync(0xffffffffu, in, 31);
        }
      }
      __syncthreads();
      if (threadIdx.x > 0 && static_cast<int>(threadIdx.x) < blocks) {
        Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
        other->result = s.result;
        other->result_sum = s.result_sum;
      }
    }
    cluster.sync();
    key = s.result;
    sum = s.result_sum;
  }
};

template <typename T>
__device__ __forceinline__ T setting(const RowSetting<T>& s, int row) { return s.each != nullptr ? s.each[row] : s.all; }

template <typename T, int V>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const SampleArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(gridDim.z), rank = static_cast<int>(blockIdx.z), line = static_cast<int>(blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < 64) s.power[threadIdx.x] = exp2(static_cast<double>(threadIdx.x) / 64.0);
  cluster.sync();   // all blocks are there: their memory may be written
  pdl_wait();
  pdl_trigger();
  const int warps = blocks * kWarps, part = ((a.vocab + warps - 1) / warps + 7) / 8 * 8;
  Row<T, V> r;
  r.row = static_cast<const T*>(a.logits) + line * a.stride;
  r.lo = min(a.vocab, (rank * kWarps + warp) * part);
  r.hi = min(a.vocab, r.lo + part);

  // ---- the likeliest, and the range
  u64 best = ~0ull;
  bool strange = false;
  walk<T, V>(r.row, r.lo, r.hi, [&](float x, int i, bool valid) {
    if (!valid) return;
    best = min(best, composite(x, i));
    const unsigned b = __float_as_uint(x);
    strange |= (b & 0x7fffffffu) > 0x7f800000u || b == 0x7f800000u;
  });
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
  if (temperature < 1.2e-38f) {   // zero, or too small to divide by
    if (rank == 0 && threadIdx.x == 0) a.tokens[line] = static_cast<long long>(best & 0xffffffffu);
    return;
  }
  r.most = most;
  r.scale = {static_cast<double>(most), 64.0 * kLog2e / static_cast<double>(temperature), s.power};
  r.steps = static_cast<float>(kBins) / (kReach * temperature);

  // ---- the border
  const int k = setting(a.top_k, line);
  const float top_p = setting(a.top_p, line);
  u64 border = ~0ull;
  const bool some_k = k > 0 && k < a.vocab, some_p = top_p < 1.f;
  if (some_k || some_p) {
    clear(s.mine);
    __syncthreads();
    walk<T, V>(r.row, r.lo, r.hi, [&](float x, int i, bool valid) {
      const u64 w = valid ? r.scale.weight(x) : 0;
      add(s.mine, w > 0 ? r.bin(x) : -1, w);
    });
    merge(cluster, s, &Shared::merged);
    u64 sum = 0;
    bool limited = false;
    if (some_k) {
      auto reached = [&](unsigned count, u64) { return count >= static_cast<unsigned>(k); };
      if (rank == 0) {
        find_bin(s, s.merged, 0, 0, reached);
        if (static_cast<int>(threadIdx.x) < blocks && threadIdx.x > 0) cluster.map_shared_rank(&s, threadIdx.x)->border.found = s.border.found;
      }
      cluster.sync();
      limited = s.border.found != 0;   // otherwise fewer than k have a weight at all
      if (limited) r.resolve(cluster, s, reached, border, sum);
    }
    if (some_p) {
      if (!limited) {   // all weights
        if (rank == 0) {
          find_bin(s, s.merged, 0, 0, [](unsigned, u64) { return false; });
          if (threadIdx.x == 0) {
            u64 all = 0;
            for (int i = 0; i < kWarps; ++i) all += s.scan[i];
            s.result_sum = all;
          }
          __syncthreads();
        }
      }
      // a token is kept while the weights in front of it are below top_p times the sum: the border is where they are reached
      const double enough = static_cast<double>(top_p) * static_cast<double>(rank == 0 ? s.result_sum : 0);
      auto reached = [&](unsigned count, u64 w) { return count > 0 && static_cast<double>(w) >= enough; };
      if (rank == 0) find_bin(s, s.merged, 0, 0, reached);
      u64 key, ignored;
      r.resolve(cluster, s, reached, key, ignored);
      border = min(border, key);
    }
  }

  // ---- the choice
  const float min_p = setting(a.min_p, line);
  const double least = static_cast<double>(min(min_p, 1.f)) * static_cast<double>(1ull << kOne);
  auto kept = [&](float x, int i) -> u64 {
    if (composite(x, i) > border) return 0;
    const u64 w = r.scale.weight(x);
    return min_p > 0.f && static_cast<double>(w) < least ? 0 : w;
  };
  u64 sum = 0;
  walk<T, V>(r.row, r.lo, r.hi, [&](float x, int i, bool valid) { sum += valid ? kept(x, i) : 0; });
  sum = warp_sum(sum);
  if (lane == 0) s.warp_sum[warp] = sum;
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
  const double u = a.uniform64 ? static_cast<const double*>(a.uniform)[line] : static_cast<double>(static_cast<const float*>(a.uniform)[line]);
  // the first token at whose end the running sum is above this
  const double at = u * static_cast<double>(total);
  const u64 aim = at > 0.0 ? min(static_cast<u64>(at), total - 1) : 0;
  for (int i = 0; i < warp; ++i) before += s.warp_sum[i];
  if (!(aim >= before && aim < before + s.warp_sum[warp])) return;   // whole warps
  int token = -1;
  for (int base = r.lo; base < r.hi && token < 0; base += 32) {
    const int i = base + lane;
    const u64 w = i < r.hi ? kept(value_of<T>(r.row[i]), i) : 0;
    u64 in = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += x;
    }
    const unsigned there = __ballot_sync(0xffffffffu, before + in > aim);
    if (there) token = base + __ffs(there) - 1;
    before += __shfl_sync(0xffffffffu, in, 31);
  }
  if (lane == 0) a.tokens[line] = token;
}

template <typename T, int V>
cudaError_t launch(const SampleArgs& a, cudaStream_t stream) {
  // blocks per row: as many as leave no SM idle, with some 2000 tokens each
  int blocks = 1;
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
