// expert_cache_experts on gfx950: a whole MoE layer for a few tokens over slot-resident experts.
//
//   y_t = sum_j p_tj W2_s (silu(Wg_s x_t) * (Wu_s x_t)),   s = slot id j of token t
//
// Three launches: experts_up_k (gate and up projection, SiLU product, routing weight),
// experts_down_k (down projection of every token-expert pair) and experts_sum_k.
//
// A few tokens read every weight of their experts once and do 2-32 operations on it, so the
// step is bound by the slots' bytes; a workgroup takes 16 rows of one expert for all of that
// expert's tokens, its waves split the rows' length between them, and LDS joins them. Pairs
// that name the same slot are found by every workgroup for itself: the step has at most 1024.
#pragma once
#include "mfma.h"
#include "wave.h"

namespace ec {

constexpr int kExpertsMaxPairs = 1024;
constexpr int kExpertsMaxK = 64;
constexpr int kUnit = 128;  // values of k a wave takes at a time: one block of e4m3 scales

struct ExpertsArgs {
  const void* x;
  long long x_stride;  // elements
  const void* w13;
  const void* w2;
  const float* s13;
  const float* s2;
  const float* probs;
  const void* ids;
  int n, k, S, H, I;
  bool wide, by_slot;
  Bf16* hi;  // [n][I] hidden values times routing weight, as two bfloat16
  Bf16* lo;
  float* part;  // [n][H]
  void* out;
  long long out_stride;  // elements
};

// Which of a lane's 16-byte loads of a unit starts at which k, and which operand of eight
// values (f of 4) does.
template <class W>
__device__ __forceinline__ int load_at(int l, int quarter) {
  return sizeof(W) == 2 ? l * 32 + quarter * 8 : l * 64 + quarter * 16;
}
template <class W>
__device__ __forceinline__ int operand_at(int f, int quarter) {
  return sizeof(W) == 2 ? f * 32 + quarter * 8 : (f >> 1) * 64 + quarter * 16 + (f & 1) * 8;
}

// The pairs of the workgroup's slot, in order, into LDS; their number, or 0 where the slot is
// another workgroup's. A workgroup belongs to pair `p` (and works if p is the first of its
// slot), or, where there are more pairs than slots, to slot `p`. A pair whose weight is zero
// or whose id names no slot is left out. Every wave builds the whole list.
__device__ __forceinline__ int list_pairs(const ExpertsArgs& a, int p, int& slot,
                                          unsigned short* list) {
  const int lane = __lane_id();
  slot = a.by_slot ? p : __builtin_amdgcn_readfirstlane(load_id(a.ids, p, a.wide, a.S));
  if (slot < 0) return 0;
  int count = 0;
  for (int base = 0; base < a.n; base += kWave) {
    const int j = base + lane;
    const int at = min(j, a.n - 1);
    const bool mine = load_id(a.ids, at, a.wide, a.S) == slot && a.probs[at] != 0.f && j < a.n;
    const unsigned long long m = ballot(mine);
    if (count == 0 && m != 0 && !a.by_slot && base + __builtin_ctzll(m) != p) return 0;
    if (mine) list[count + __builtin_popcountll(m & lanes_below())] = (unsigned short)j;
    count += __builtin_popcountll(m);
  }
  lds_sync();
  return count;
}

__device__ __forceinline__ u32x4 keep(bool c, u32x4 v) {
  return u32x4{c ? v[0] : 0, c ? v[1] : 0, c ? v[2] : 0, c ? v[3] : 0};
}

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

// A lane's share of one unit: R rows of weights, NB operands of tokens, and a scale a row set.
template <class W, int R, int NB>
struct Unit {
  static constexpr int kLoads = sizeof(W) == 2 ? 4 : 2;
  u32x4 w[R][kLoads];
  u32x4 b[NB][4];
  float s[R];

  __device__ __forceinline__ void load(const W* const (&rows)[R], const void* const (&cols)[NB],
                                       const float* const (&scale)[R], int u, int K, int quarter) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      int at = u * kUnit + load_at<W>(l, quarter);
      at = at < K ? at : 0;
#pragma unroll
      for (int r = 0; r < R; ++r) w[r][l] = load16(rows[r] + at);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      int at = u * kUnit + operand_at<W>(f, quarter);
      at = at < K ? at : 0;
#pragma unroll
      for (int c = 0; c < NB; ++c)
        b[c][f] = load16(static_cast<const unsigned short*>(cols[c]) + at);
    }
    if constexpr (__is_same(W, E4m3)) {
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] = scale[r][u];
    }
  }
  // Past the end of k both operands are zero (a weight read there may be no number).
  __device__ __forceinline__ void cut(int u, int K, int quarter) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const bool in = u * kUnit + load_at<W>(l, quarter) < K;
#pragma unroll
      for (int r = 0; r < R; ++r) w[r][l] = keep(in, w[r][l]);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const bool in = u * kUnit + operand_at<W>(f, quarter) < K;
#pragma unroll
      for (int c = 0; c < NB; ++c) b[c][f] = keep(in, b[c][f]);
    }
  }
  // acc[r] += rows times columns: NB = 1 columns of X, NB = 2 columns as two bfloat16
  template <class X>
  __device__ __forceinline__ void add(f32x4 (&acc)[R]) const {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      f32x4 c = __is_same(W, E4m3) ? f32x4{0, 0, 0, 0} : acc[r];
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const u32x4 v = w[r][sizeof(W) == 2 ? f : f >> 1];
        if constexpr (NB == 1)
          c = Frag<X>::mfma(operand<X, W>(v, f & 1), b[0][f], c);
        else
          c = mfma_split<W>(v, f & 1, b[0][f], b[1][f], c);
      }
      if constexpr (__is_same(W, E4m3)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][i] = fmaf(s[r], c[i], acc[r][i]);
      } else {
        acc[r] = c;
      }
    }
  }
};

// The wave's share of K in steps of `stride` units from `first`, D units in flight.
template <class X, class W, int R, int NB, int D>
__device__ __forceinline__ void product(const W* const (&rows)[R], const void* const (&cols)[NB],
                                        const float* const (&scale)[R], int first, int stride,
                                        int K, f32x4 (&acc)[R]) {
  const int quarter = __lane_id() >> 4, units = (K + kUnit - 1) / kUnit;
  Unit<W, R, NB> buf[D];
#pragma unroll
  for (int d = 0; d < D; ++d)
    buf[d].load(rows, cols, scale, min(first + d * stride, units - 1), K, quarter);
  for (int u = first; u < units; u += D * stride) {
#pragma unroll
    for (int d = 0; d < D; ++d) {
      const int at = u + d * stride;
      if (at < units) {
        if ((at + 1) * kUnit > K) buf[d].cut(at, K, quarter);
        buf[d].template add<X>(acc);
      }
      buf[d].load(rows, cols, scale, min(at + D * stride, units - 1), K, quarter);
    }
  }
}

// Gate and up projection of 16 rows of one expert, SiLU product and routing weight.
template <class X, class W, int WAVES, int D>
__global__ __launch_bounds__(WAVES* kWave) void experts_up_k(ExpertsArgs a) {
  static_assert(WAVES * kWave >= 256);
  __shared__ unsigned short list[kExpertsMaxPairs];
  __shared__ float red[WAVES][2][4][kWave];
  const int lane = __lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int slot;
  const int count = list_pairs(a, blockIdx.y, slot, list);
  const int row0 = blockIdx.x * 16;
  const W* w13 = static_cast<const W*>(a.w13) + (long long)slot * 2 * a.I * a.H;
  const W* gate = w13 + (long long)min(row0 + (lane & 15), a.I - 1) * a.H;
  const W* const rows[2] = {gate, gate + (long long)a.I * a.H};
  const float* scale[2] = {nullptr, nullptr};
  if constexpr (__is_same(W, E4m3)) {
    const int kb = (a.H + kUnit - 1) / kUnit, rb = (2 * a.I + kUnit - 1) / kUnit;
    const float* s13 = a.s13 + (long long)slot * rb * kb;
    scale[0] = s13 + (long long)(row0 / kUnit) * kb;
    scale[1] = s13 + (long long)((a.I + row0) / kUnit) * kb;
  }
  for (int c0 = 0; c0 < count; c0 += 16) {
    const int token = list[min(c0 + (lane & 15), count - 1)] / a.k;
    const void* const cols[1] = {static_cast<const X*>(a.x) + token * a.x_stride};
    f32x4 acc[2] = {};
    const float* const sc[2] = {scale[0], scale[1]};
    product<X, W, 2, 1, D>(rows, cols, sc, wave, WAVES, a.H, acc);
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[wave][r][i][lane] = acc[r][i];
    lds_sync();
    const int row = row0 + (threadIdx.x & 15), col = threadIdx.x >> 4;
    if (threadIdx.x < 256 && row < a.I && c0 + col < count) {
      const int from = (threadIdx.x & 15) / 4 * 16 + col, i = threadIdx.x & 3;
      float g = 0, u = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        g += red[w][0][i][from];
        u += red[w][1][i][from];
      }
      if constexpr (__is_same(W, int8_t)) {
        const float* s13 = a.s13 + (long long)slot * 2 * a.I;
        g *= s13[row];
        u *= s13[a.I + row];
      }
      const int pair = list[c0 + col];
      Bf16 h, l;
      split_f32(silu(g) * u * a.probs[pair], h, l);
      a.hi[(long long)pair * a.I + row] = h;
      a.lo[(long long)pair * a.I + row] = l;
    }
    lds_sync();
  }
}

// Down projection of 16 rows of one expert for its pairs.
template <class W, int WAVES, int D>
__global__ __launch_bounds__(WAVES* kWave) void experts_down_k(ExpertsArgs a) {
  static_assert(WAVES * kWave >= 256);
  __shared__ unsigned short list[kExpertsMaxPairs];
  __shared__ float red[WAVES][4][kWave];
  const int lane = __lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int slot;
  const int count = list_pairs(a, blockIdx.y, slot, list);
  const int row0 = blockIdx.x * 16;
  const W* const rows[1] = {static_cast<const W*>(a.w2) +
                            ((long long)slot * a.H + min(row0 + (lane & 15), a.H - 1)) * a.I};
  const float* scale[1] = {nullptr};
  if constexpr (__is_same(W, E4m3)) {
    const int kb = (a.I + kUnit - 1) / kUnit, rb = (a.H + kUnit - 1) / kUnit;
    scale[0] = a.s2 + ((long long)slot * rb + row0 / kUnit) * kb;
  }
  for (int c0 = 0; c0 < count; c0 += 16) {
    const long long at = (long long)list[min(c0 + (lane & 15), count - 1)] * a.I;
    const void* const cols[2] = {a.hi + at, a.lo + at};
    f32x4 acc[1] = {};
    const float* const sc[1] = {scale[0]};
    product<Bf16, W, 1, 2, D>(rows, cols, sc, wave, WAVES, a.I, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][i][lane] = acc[0][i];
    lds_sync();
    const int row = row0 + (threadIdx.x & 15), col = threadIdx.x >> 4;
    if (threadIdx.x < 256 && row < a.H && c0 + col < count) {
      const int from = (threadIdx.x & 15) / 4 * 16 + col, i = threadIdx.x & 3;
      float y = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) y += red[w][i][from];
      if constexpr (__is_same(W, int8_t)) y *= a.s2[(long long)slot * a.H + row];
      a.part[(long long)list[c0 + col] * a.H + row] = y;
    }
    lds_sync();
  }
}

// A token's pairs added up in order; tokens without any become zero.
template <class X>
__global__ __launch_bounds__(256) void experts_sum_k(ExpertsArgs a) {
  const int t = blockIdx.y, lane = __lane_id();
  const int at = t * a.k + min(lane, a.k - 1);
  unsigned long long used =
      ballot(lane < a.k && load_id(a.ids, at, a.wide, a.S) >= 0 && a.probs[at] != 0.f);
  const int r = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (r >= a.H) return;
  f32x4 y = {0, 0, 0, 0};
  for (; used; used &= used - 1) {
    const long long pair = (long long)t * a.k + __builtin_ctzll(used);
    y += *reinterpret_cast<const f32x4*>(a.part + pair * a.H + r);
  }
  X* out = static_cast<X*>(a.out) + t * a.out_stride + r;
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = from_f32<X>(y[i]);
}

}  // namespace ec
