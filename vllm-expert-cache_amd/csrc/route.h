// expert_cache_route on gfx950: gate logits to routing weights and expert ids.
//
// A wave takes a token and holds its row in registers, V values a lane. Selection is k rounds
// of a wave minimum over keys that order the candidates best first, each followed by a ballot
// for the lowest expert that has it: no sort, since k is a handful.
//
// Keys. Without a bias the order of the scores is that of the logits, so the key is the logit's
// own 32 bits, and equal logits are equal scores. With one, score + bias is rounded, and two
// orders of the same operations in 32 bits disagree about which of two near experts comes
// first; in 64 bits the difference is far below what inputs of 32 bits can be apart, so that
// key is a double. The weights of the few selected experts are computed in 64 bits too.
// A token is a few hundred bytes, so a call is bound by one wave's chain of latencies: the row's
// load, then k minima over the wave by DPP. One token of 128 experts, top-8 takes
// 3.5 us in a graph where an empty launch takes 1.9; 60 tokens of 256 with groups and a bias 7.8,
// for its keys of 64 bits and the groups' own rounds; 8192 tokens of 128 7.0.
#pragma once
#include "mfma.h"
#include "wave.h"

namespace ec {

constexpr int kRouteWaves = 4;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 64;
constexpr int kRouteMaxGroups = 64;

struct RouteArgs {
  const void* logits;
  long long row_stride;  // elements
  const float* bias;
  int T, E, k, groups, topk_groups;
  bool sigmoid, renormalize, wide;
  float scale;
  float* weights;
  void* ids;
};

// Keys ascend from the best candidate; kNone is none at all.
struct LogitKey {
  using Key = unsigned;
  static constexpr Key kNone = 0xFFFFFFFFu;
  static __device__ __forceinline__ Key of(float x) {
    const unsigned b = bits_as<unsigned>(x + 0.f);  // -0 becomes +0: they tie
    return ~(b & 0x80000000u ? ~b : b | 0x80000000u);
  }
  static __device__ __forceinline__ Key min_of(Key v) { return wave_min_u32(v); }
  // of lane (own lane xor X), of lane l
  template <int X>
  static __device__ __forceinline__ Key from(Key v) {
    return lane_xor<X>(v);
  }
  static __device__ __forceinline__ Key at(Key v, int l) {
    return (Key)__builtin_amdgcn_readlane((int)v, l);
  }
};
struct ScoreKey {
  using Key = unsigned long long;
  static constexpr Key kNone = ~0ull;
  static __device__ __forceinline__ Key of(double x) {
    const Key b = bits_as<Key>(x + 0.0);
    return ~(b >> 63 ? ~b : b | 1ull << 63);
  }
  static __device__ __forceinline__ double value(Key k) {
    const Key b = ~k;
    return bits_as<double>(b >> 63 ? b & ~(1ull << 63) : ~b);
  }
  static __device__ __forceinline__ Key min_of(Key v) {
    const unsigned hi = wave_min_u32((unsigned)(v >> 32));
    const unsigned lo = wave_min_u32((unsigned)(v >> 32) == hi ? (unsigned)v : 0xFFFFFFFFu);
    return (Key)hi << 32 | lo;
  }
  template <int X>
  static __device__ __forceinline__ Key from(Key v) {
    return (Key)lane_xor<X>((unsigned)(v >> 32)) << 32 | lane_xor<X>((unsigned)v);
  }
  static __device__ __forceinline__ Key at(Key v, int l) {
    return (Key)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 |
           (unsigned)__builtin_amdgcn_readlane((int)v, l);
  }
};

__device__ __forceinline__ bool is_candidate(float x) { return x > -__builtin_inff(); }

__device__ __forceinline__ float wave_max_f32(float v) {
  const auto step = [&](unsigned o) { v = fmaxf(v, bits_as<float>(o)); };
  step(lane_xor<1>(bits_as<unsigned>(v)));
  step(lane_xor<2>(bits_as<unsigned>(v)));
  step(lane_xor<4>(bits_as<unsigned>(v)));
  step(lane_xor<8>(bits_as<unsigned>(v)));
  step(lane_xor<16>(bits_as<unsigned>(v)));
  step(lane_xor<32>(bits_as<unsigned>(v)));
  return v;
}
template <int X, class T>
__device__ __forceinline__ T lane_xor_64(T v) {
  const unsigned long long b = bits_as<unsigned long long>(v);
  return bits_as<T>((unsigned long long)lane_xor<X>((unsigned)(b >> 32)) << 32 |
                    lane_xor<X>((unsigned)b));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += lane_xor_64<1>(v);
  v += lane_xor_64<2>(v);
  v += lane_xor_64<4>(v);
  v += lane_xor_64<8>(v);
  v += lane_xor_64<16>(v);
  return v + lane_xor_64<32>(v);
}

// exp(x - m) with m the largest: where that is +infinity its holders share the whole weight.
__device__ __forceinline__ double softmax_term(float x, float m) {
  return x == m ? 1.0 : exp((double)x - (double)m);
}

// The groups that stay, a bit each: of every group the best key, or with a bias the sum of
// its two best, and of those the topk_groups best, the lower group first where they tie.
// P lanes share a group and walk its keys, which the wave has put into LDS.
template <class K, bool BIAS>
__device__ unsigned long long keep_groups(const typename K::Key* keys, const RouteArgs& a) {
  using Key = typename K::Key;
  const int lane = __lane_id(), n = a.E / a.groups;
  int P = 1;
  while (2 * P * a.groups <= kWave) P *= 2;
  const int g = lane / P;
  Key b0 = K::kNone, b1 = K::kNone;
  if (g < a.groups) {
    for (int i = lane & (P - 1); i < n; i += P) {
      const Key v = keys[g * n + i];
      b1 = min(b1, max(b0, v));
      b0 = min(b0, v);
    }
  }
  const auto join = [&](Key o0, Key o1) {
    b1 = min(max(b0, o0), min(b1, o1));
    b0 = min(b0, o0);
  };
  if (P > 1) join(K::template from<1>(b0), K::template from<1>(b1));
  if (P > 2) join(K::template from<2>(b0), K::template from<2>(b1));
  if (P > 4) join(K::template from<4>(b0), K::template from<4>(b1));
  if (P > 8) join(K::template from<8>(b0), K::template from<8>(b1));
  if (P > 16) join(K::template from<16>(b0), K::template from<16>(b1));
  if constexpr (BIAS) {
    if (b1 != K::kNone) b0 = K::of(K::value(b0) + K::value(b1));
  }
  int better = 0;
  for (int o = 0; o < a.groups; ++o) {
    const Key v = K::at(b0, o * P);
    better += v < b0 || (v == b0 && o < g);
  }
  const bool keep = g < a.groups && (lane & (P - 1)) == 0 && better < a.topk_groups;
  const unsigned long long lanes = ballot(keep);
  unsigned long long kept = 0;
  for (int o = 0; o < a.groups; ++o) kept |= (lanes >> (o * P) & 1ull) << o;
  return kept;
}

template <class X, int V, bool BIAS>
__global__ __launch_bounds__(kRouteWaves* kWave) void route_k(RouteArgs a) {
  using K = std::conditional_t<BIAS, ScoreKey, LogitKey>;
  using Key = typename K::Key;
  __shared__ Key row[kRouteWaves][V * kWave];
  const int lane = __lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const long long t = (long long)blockIdx.x * kRouteWaves + wave;
  const bool live = t < a.T;
  const X* in = static_cast<const X*>(a.logits) + (live ? t : 0) * a.row_stride;

  float x[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * kWave + lane;
    x[i] = live && e < a.E ? to_f32(in[e]) : -__builtin_inff();
  }
  float top = -__builtin_inff();
  double total = 0;
  if (!a.sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) top = fmaxf(top, x[i]);
    top = wave_max_f32(top);
    if (BIAS || !a.renormalize) {  // otherwise the scores' sum cancels
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (is_candidate(x[i])) total += softmax_term(x[i], top);
      total = wave_sum_f64(total);
    }
  }
  const auto score = [&](float v) {
    return a.sigmoid ? 1.0 / (1.0 + exp(-(double)v)) : softmax_term(v, top) / total;
  };

  Key key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = i * kWave + lane;
    key[i] = K::kNone;
    if (is_candidate(x[i])) {
      if constexpr (BIAS) {
        const float b = a.bias[e];
        if (is_candidate(b)) key[i] = K::of(score(x[i]) + (double)b);
      } else {
        key[i] = K::of(x[i]);
      }
    }
  }
  if (a.groups > 1) {
#pragma unroll
    for (int i = 0; i < V; ++i) row[wave][i * kWave + lane] = key[i];
    lds_sync();
    const unsigned long long kept = keep_groups<K, BIAS>(row[wave], a);
    const int n = a.E / a.groups;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (!(kept >> min((i * kWave + lane) / n, 63) & 1)) key[i] = K::kNone;
  }

  // lane j ends with the j-th selected expert and its logit
  int id = -1;
  float mine = 0;
  for (int j = 0; j < a.k; ++j) {
    Key best = key[0];
#pragma unroll
    for (int i = 1; i < V; ++i) best = min(best, key[i]);
    best = K::min_of(best);
    if (best == K::kNone) break;
    bool found = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const unsigned long long at = found ? 0 : ballot(key[i] == best);
      if (at) {
        found = true;
        const int l = __builtin_ctzll(at);
        const float v = bits_as<float>(__builtin_amdgcn_readlane(bits_as<int>(x[i]), l));
        if (lane == l) key[i] = K::kNone;
        if (lane == j) {
          id = i * kWave + l;
          mine = v;
        }
      }
    }
  }
  double w = id < 0 ? 0.0 : a.sigmoid || !a.renormalize ? score(mine) : softmax_term(mine, top);
  if (a.renormalize) {
    const double sum = wave_sum_f64(w);
    w = sum > 0 ? w / sum : 0.0;
  }
  if (!live || lane >= a.k) return;
  a.weights[t * a.k + lane] = (float)(w * (double)a.scale);
  if (a.wide)
    static_cast<long long*>(a.ids)[t * a.k + lane] = id;
  else
    static_cast<int*>(a.ids)[t * a.k + lane] = id;
}

}  // namespace ec
