// Rotary positions of queries and keys: (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of a head's first elements, the rest copied.
//
// Bound by memory: every element is read and written once.  A thread holds the cosines and sines of one place within the head and goes over several heads of
// its token with them, so that the tables cost a fraction of the rest.  Pairs are neighbours within 16 bytes, or half a turned part apart: two accesses of 16
// bytes then (8 where the half is an odd number of 4).  Products and sums are fp32, rounded once.
#include "../core/launch.hpp"
#include "divisor.cuh"
#include "half16.cuh"
#include "ops.hpp"
#include "packed.hpp"

#include <climits>

namespace mccl {
namespace ops {

namespace {

constexpr int kThreads = 256;

struct Rotary {
  RotaryArgs a;
  Divisor places, groups;   // places within a head that a thread may have; threads that share out a token's heads
  int turned;               // the first of them turn pairs
};

template <typename H, int N>
struct Vector;
template <typename H>
struct Vector<H, 8> {
  uint4 raw;
  __device__ __forceinline__ void up(float (&f)[8]) const { unpack8_as<H>(raw, f); }
  __device__ __forceinline__ void down(const float (&f)[8]) { raw = pack8_as<H>(f); }
};
template <typename H>
struct Vector<H, 4> {
  uint2 raw;
  __device__ __forceinline__ void up(float (&f)[4]) const {
    const typename H::T2* h = reinterpret_cast<const typename H::T2*>(&raw);
    const float2 a = H::up(h[0]), b = H::up(h[1]);
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  }
  __device__ __forceinline__ void down(const float (&f)[4]) {
    typename H::T2* h = reinterpret_cast<typename H::T2*>(&raw);
    h[0] = H::down(f[0], f[1]);
    h[1] = H::down(f[2], f[3]);
  }
};

// HALVES: N elements and the N of the other half per place; otherwise 8 elements, four pairs.  Behind the turned places 8 elements each are copied.
template <typename H, bool HALVES, int N>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r, int total) {
  using T = typename H::T;
  const RotaryArgs& a = r.a;
  pdl_wait();
  pdl_trigger();
  const int i = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  if (i >= total) return;
  const int rest = r.places.of(i), place = i - rest * r.places.d, t = r.groups.of(rest), group = rest - t * r.groups.d;
  const int pos = a.positions != nullptr ? __ldg(a.positions + t) : t;
  const bool inside = pos >= 0 && pos < a.rope_rows, turn = place < r.turned;
  constexpr int kPairs = HALVES ? N : 4;
  float c[kPairs], s[kPairs];
  if (turn && inside) {
    const float* at_c = a.cos + static_cast<long long>(pos) * a.width + place * kPairs;
    const float* at_s = a.sin + static_cast<long long>(pos) * a.width + place * kPairs;
#pragma unroll
    for (int e = 0; e < kPairs; e += 4) {
      const float4 x = __ldg(reinterpret_cast<const float4*>(at_c + e)), y = __ldg(reinterpret_cast<const float4*>(at_s + e));
      c[e] = x.x, c[e + 1] = x.y, c[e + 2] = x.z, c[e + 3] = x.w;
      s[e] = y.x, s[e + 1] = y.y, s[e + 2] = y.z, s[e + 3] = y.w;
    }
    if (a.inverse) {
#pragma unroll
      for (int e = 0; e < kPairs; ++e) s[e] = -s[e];
    }
  }
  const int column = turn ? place * (HALVES ? N : 8) : 2 * a.width + (place - r.turned) * 8;
#pragma unroll 4
  for (int h = group; h < a.q.heads + a.k.heads; h += r.groups.d) {
    const bool is_q = h < a.q.heads;
    const RotaryPart& part = is_q ? a.q : a.k;
    const int hh = is_q ? h : h - a.q.heads;
    const T* x = static_cast<const T*>(part.x.p) + t * part.x.token + hh * part.x.head + column;
    T* y = static_cast<T*>(part.out) + (static_cast<long long>(t) * part.heads + hh) * a.head_dim + column;
    if (!turn) {
      *reinterpret_cast<uint4*>(y) = inside ? __ldg(reinterpret_cast<const uint4*>(x)) : make_uint4(0u, 0u, 0u, 0u);
    } else if constexpr (HALVES) {
      using V = decltype(Vector<H, N>::raw);
      Vector<H, N> lo{}, hi{};
      if (inside) {
        lo.raw = __ldg(reinterpret_cast<const V*>(x));
        hi.raw = __ldg(reinterpret_cast<const V*>(x + a.width));
        float f[N], g[N];
        lo.up(f);
        hi.up(g);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const float u = f[e], v = g[e];
          f[e] = u * c[e] - v * s[e];
          g[e] = u * s[e] + v * c[e];
        }
        lo.down(f);
        hi.down(g);
      }
      *reinterpret_cast<V*>(y) = lo.raw;
      *reinterpret_cast<V*>(y + a.width) = hi.raw;
    } else {
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      if (inside) {
        float f[8];
        unpack8_as<H>(__ldg(reinterpret_cast<const uint4*>(x)), f);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = f[2 * e], v = f[2 * e + 1];
          f[2 * e] = u * c[e] - v * s[e];
          f[2 * e + 1] = u * s[e] + v * c[e];
        }
        raw = pack8_as<H>(f);
      }
      *reinterpret_cast<uint4*>(y) = raw;
    }
  }
}

template <typename H>
cudaError_t launch(const RotaryArgs& args, cudaStream_t stream) {
  const int wide = args.halves && args.width % 8 != 0 ? 4 : 8;
  const int turned = args.halves ? args.width / wide : args.width / 4, heads = args.q.heads + args.k.heads;
  const int places = turned + (args.head_dim - 2 * args.width) / 8;
  // a thread takes as many heads as leave every SM its threads, up to 4: more of them share what it holds
  const long long one = static_cast<long long>(args.tokens) * places * heads;
  int per_thread = static_cast<int>(one / (148ll * 2048));
  per_thread = per_thread < 1 ? 1 : (per_thread > 4 ? 4 : per_thread);
  const int groups = (heads + per_thread - 1) / per_thread;
  const long long per_token = static_cast<long long>(groups) * places;
  if (per_token > INT_MAX / 2) return cudaErrorInvalidValue;
  // indices are counted in 32 bits: as many tokens at a time as they reach
  const int step = static_cast<int>((INT_MAX - kThreads) / per_token);
  for (long long t0 = 0; t0 < args.tokens; t0 += step) {
    Rotary r;
    r.a = args;
    const int tokens = static_cast<int>(args.tokens - t0 < step ? args.tokens - t0 : step);
    for (RotaryPart* part : {&r.a.q, &r.a.k}) {
      if (part->heads == 0) continue;
      part->x.p = static_cast<const char*>(part->x.p) + t0 * part->x.token * 2;
      part->out = static_cast<char*>(part->out) + t0 * part->heads * args.head_dim * 2;
    }
    if (args.positions != nullptr) {
      r.a.positions = args.positions + t0;
    } else if (t0 > 0) {   // token t0 stands at position t0
      r.a.cos = args.cos + t0 * args.width;
      r.a.sin = args.sin + t0 * args.width;
      r.a.rope_rows = args.rope_rows > t0 ? static_cast<int>(args.rope_rows - t0) : 0;
    }
    r.places = Divisor(places);
    r.groups = Divisor(groups);
    r.turned = turned;
    const int total = static_cast<int>(tokens * per_token);
    const int blocks = (total + kThreads - 1) / kThreads;
    if (!args.halves) {
      MCCL_LAUNCH_PDL((rotary_kernel<H, false, 8>), blocks, kThreads, 0, stream, r, total);
    } else if (wide == 8) {
      MCCL_LAUNCH_PDL((rotary_kernel<H, true, 8>), blocks, kThreads, 0, stream, r, total);
    } else {
      MCCL_LAUNCH_PDL((rotary_kernel<H, true, 4>), blocks, kThreads, 0, stream, r, total);
    }
    count_launch();
  }
  return ::mccl::launch_status();
}

}  // namespace

cudaError_t rotary(const RotaryArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0 || a.q.heads + a.k.heads <= 0) return cudaSuccess;
  return a.type == Half16::bf16 ? launch<Bf16>(a, stream) : launch<Fp16>(a, stream);
}

}  // namespace ops
}  // namespace mccl
