// Rotary positions of queries and keys: (a, b) -> (a cos - b sin, a sin + b cos) for the pairs of a head's first elements, the rest copied.
//
// Bound by memory: every element is read and written once (16384 tokens of 32 + 8 heads of 128: 51 us, 6.6 TB/s; a device-to-device copy of as much takes 58).  A thread holds the cosines and sines of one place within the head and goes over several heads of
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
  int turned;               // the first of them turn pairs, ...
  int apart, lone;          // ... the others copy N elements and, with halves, the N `apart` behind them; place `lone` has no second ones
};

// N values of one access.
template <int N>
struct Access;
template <>
struct Access<8> {
  using V = uint4;
};
template <>
struct Access<4> {
  using V = uint2;
};
template <typename H, int N>
__device__ __forceinline__ void up(const typename Access<N>::V& raw, float (&f)[N]) {
  const typename H::T2* h = reinterpret_cast<const typename H::T2*>(&raw);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) {
    const float2 t = H::up(h[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename H, int N>
__device__ __forceinline__ typename Access<N>::V down(const float (&f)[N]) {
  typename Access<N>::V raw;
  typename H::T2* h = reinterpret_cast<typename H::T2*>(&raw);
#pragma unroll
  for (int i = 0; i < N / 2; ++i) h[i] = H::down(f[2 * i], f[2 * i + 1]);
  return raw;
}

// HALVES: N elements and the N of the other half per place; otherwise 8 elements, four pairs.  Behind the turned places as many elements per place are copied, in
// the same accesses (with a way of their own for copies, halves of 64 of 128 elements took 71 us where they take 51, of 16384 tokens with 32 + 8 heads).  HEADS heads per thread, all of whose loads are
// under way together.
template <typename H, bool HALVES, int N, int HEADS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const Rotary r, int total) {
  using T = typename H::T;
  using V = typename Access<N>::V;
  const RotaryArgs& a = r.a;
  pdl_wait();
  pdl_trigger();
  const int i = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  if (i >= total) return;
  const int rest = r.places.of(i), place = i - rest * r.places.d, t = r.groups.of(rest), group = rest - t * r.groups.d;
  const int pos = a.positions != nullptr ? __ldg(a.positions + t) : t;
  const bool inside = pos >= 0 && pos < a.rope_rows, turn = place < r.turned;
  const int second = turn ? a.width : r.apart;
  const bool two = HALVES && place != r.lone;
  const int column = turn ? place * N : 2 * a.width + (place - r.turned) * N;
  const T* from[HEADS];
  T* to[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    const int h = group + j * r.groups.d;
    const bool is_q = h < a.q.heads, any = h < a.q.heads + a.k.heads;
    const RotaryPart& part = is_q ? a.q : a.k;
    const int hh = is_q ? h : h - a.q.heads;
    from[j] = any && inside ? static_cast<const T*>(part.x.p) + t * part.x.token + hh * part.x.head + column : nullptr;
    to[j] = any ? static_cast<T*>(part.out) + (static_cast<long long>(t) * part.heads + hh) * a.head_dim + column : nullptr;
  }
  constexpr int kPairs = HALVES ? N : 4;
  V lo[HEADS], hi[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    lo[j] = hi[j] = V{};
    if (from[j] != nullptr) {
      lo[j] = __ldg(reinterpret_cast<const V*>(from[j]));
      if (two) hi[j] = __ldg(reinterpret_cast<const V*>(from[j] + second));
    }
  }
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; e += 4) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    if (inside && turn) {
      x = __ldg(reinterpret_cast<const float4*>(a.cos + static_cast<long long>(pos) * a.width + place * kPairs + e));
      y = __ldg(reinterpret_cast<const float4*>(a.sin + static_cast<long long>(pos) * a.width + place * kPairs + e));
    }
    c[e] = x.x, c[e + 1] = x.y, c[e + 2] = x.z, c[e + 3] = x.w;
    s[e] = y.x, s[e + 1] = y.y, s[e + 2] = y.z, s[e + 3] = y.w;
  }
  if (a.inverse) {
#pragma unroll
    for (int e = 0; e < kPairs; ++e) s[e] = -s[e];
  }
#pragma unroll
  for (int j = 0; j < HEADS; ++j) {
    if (to[j] == nullptr) continue;
    if (!turn) {
      *reinterpret_cast<V*>(to[j]) = lo[j];
      if (two) *reinterpret_cast<V*>(to[j] + second) = hi[j];
      continue;
    }
    float f[N];
    up<H, N>(lo[j], f);
    if constexpr (HALVES) {
      float g[N];
      up<H, N>(hi[j], g);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float u = f[e], v = g[e];
        f[e] = u * c[e] - v * s[e];
        g[e] = u * s[e] + v * c[e];
      }
      *reinterpret_cast<V*>(to[j]) = down<H, N>(f);
      *reinterpret_cast<V*>(to[j] + a.width) = down<H, N>(g);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float u = f[2 * e], v = f[2 * e + 1];
        f[2 * e] = u * c[e] - v * s[e];
        f[2 * e + 1] = u * s[e] + v * c[e];
      }
      *reinterpret_cast<V*>(to[j]) = down<H, N>(f);
    }
  }
}

template <typename H, bool HALVES, int N>
void enqueue(const Rotary& r, int total, int per_thread, cudaStream_t stream) {
  const int blocks = (total + kThreads - 1) / kThreads;
  if (per_thread == 1) MCCL_LAUNCH_PDL((rotary_kernel<H, HALVES, N, 1>), blocks, kThreads, 0, stream, r, total);
  else MCCL_LAUNCH_PDL((rotary_kernel<H, HALVES, N, 2>), blocks, kThreads, 0, stream, r, total);
}

template <typename H>
cudaError_t launch(const RotaryArgs& args, cudaStream_t stream) {
  const int wide = args.halves && args.width % 8 != 0 ? 4 : 8;
  const int turned = args.halves ? args.width / wide : args.width / 4, heads = args.q.heads + args.k.heads;
  const int copied = (args.head_dim - 2 * args.width) / wide, pieces = args.halves ? 2 : 1, places = turned + (copied + pieces - 1) / pieces;
  // a thread takes two heads where that leaves every SM its threads (16384 tokens of 32 + 8 heads: 51.1 us with two, 52.3 with four)
  const long long one = static_cast<long long>(args.tokens) * places * heads;
  const int per_thread = one / 2 < 148ll * 2048 ? 1 : 2;
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
    r.apart = (copied + 1) / 2 * wide;
    r.lone = args.halves && copied % 2 != 0 ? places - 1 : -1;
    const int total = static_cast<int>(tokens * per_token);
    if (!args.halves) enqueue<H, false, 8>(r, total, per_thread, stream);
    else if (wide == 8) enqueue<H, true, 8>(r, total, per_thread, stream);
    else enqueue<H, true, 4>(r, total, per_thread, stream);
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
