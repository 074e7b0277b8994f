// expert_cache_adapters on gfx950: low-rank adapters of many requests, one slot a token, added
// to the output of a projection that all tokens share.
//
//   out_t = base_t + scale_s * B_s (A_s x_t),   s = slot id of token t
//
// Two launches: adapters_shrink_k makes A_s x_t in 32 bits, the hidden length split over
// workgroups where tokens are few, and adapters_expand_k joins the parts in a fixed order and
// adds B's product to the base. Tokens come in tiles of 16, the columns of the matrix
// instruction; a tile whose tokens have several adapters runs each of them over the whole tile
// and takes from each product the columns that are its own.
#pragma once
#include "experts.h"
#include "mfma.h"
#include "wave.h"

namespace ec {

constexpr int kAdapterTile = 16;
constexpr int kAdapterMaxRank = 256;

struct AdaptersArgs {
  const void* x;
  long long x_stride;  // elements, like the strides below
  const void* a;
  const void* b;
  const float* scales;  // [S], or null: 1
  const void* ids;
  const void* base;
  long long base_stride;
  void* out;
  long long out_stride;
  int T, S, H, O, R, splits;
  bool wide;
  float* v;  // [splits][T][R]
};

// Slot of the tile's token (lane & 15), or -1.
__device__ __forceinline__ int tile_slot(const AdaptersArgs& a, int t0) {
  const int t = t0 + (__lane_id() & 15);
  const int id = load_id(a.ids, min(t, a.T - 1), a.wide, a.S);
  return t < a.T ? id : -1;
}

// A's product for one tile and one of its adapters over one split of the hidden length.
template <class X, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_shrink_k(AdaptersArgs a) {
  __shared__ float red[WAVES][4][kWave];
  const int lane = __lane_id();
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kAdapterTile, which = blockIdx.y;
  const int id = tile_slot(a, t0);
  const int slot = __builtin_amdgcn_readlane(id, which);
  const unsigned own = (unsigned)ballot(id == slot) & 0xFFFFu;
  if (slot < 0 || __builtin_ctz(own) != which) return;
  const int token = min(t0 + (lane & 15), a.T - 1);
  const unsigned short* x = static_cast<const unsigned short*>(a.x) + token * a.x_stride;
  const int units = (a.H + kUnit - 1) / kUnit, quarter = lane >> 4;
  const int per = (units + a.splits - 1) / a.splits;
  const int first = blockIdx.z * per, last = min(units, first + per);
  for (int r0 = 0; r0 < a.R; r0 += 16) {
    const X* from = static_cast<const X*>(a.a) + ((long long)slot * a.R + r0) * a.H;
    const unsigned row = row_bytes<X>(r0 + (lane & 15), r0, a.R, a.H);
    f32x4 acc = {0, 0, 0, 0};
    constexpr int D = 2;
    Rows<X> w[D];
    u32x4 b[D][4];
    pipeline<D>(
        (last - first - wave + WAVES - 1) / WAVES,
        [&](auto d, int i) EC_INLINE {
          const int u = first + wave + i * WAVES;
          w[d].load(from, row, nullptr, u, a.H, quarter);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const int k = u * kUnit + operand_at<X>(f, quarter);
            b[d][f] = load16(x + (k < a.H ? k : 0));
          }
        },
        [&](auto d, int i) EC_INLINE {
          const int u = first + wave + i * WAVES;
          if ((u + 1) * kUnit > a.H) {
            w[d].cut(u, a.H, quarter);
#pragma unroll
            for (int f = 0; f < 4; ++f)
              b[d][f] = keep(u * kUnit + operand_at<X>(f, quarter) < a.H, b[d][f]);
          }
          add_whole<X, X>(w[d], b[d], acc);
        });
#pragma unroll
    for (int i = 0; i < 4; ++i) red[wave][i][lane] = acc[i];
    lds_sync();
    for (int j = threadIdx.x; j < 256; j += WAVES * kWave) {
      const int row = r0 + (j & 15), col = j >> 4;
      if (row < a.R && own >> col & 1) {
        float y = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) y += red[w][j & 3][(j & 15) / 4 * 16 + col];
        a.v[((long long)blockIdx.z * a.T + t0 + col) * a.R + row] = y;
      }
    }
    lds_sync();
  }
}

// B's product and the sum with the base, 16 outputs a wave for one tile.
template <class X, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_expand_k(AdaptersArgs a) {
  const int lane = __lane_id(), quarter = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kAdapterTile;
  const int row0 = (blockIdx.y * WAVES + wave) * 16;
  if (row0 >= a.O) return;
  const int id = tile_slot(a, t0);
  const int token = t0 + (lane & 15);
  const int brow = min(row0 + (lane & 15), a.O - 1);
  f32x4 total = {0, 0, 0, 0};
  if (ballot(id >= 0)) {
    const float scale = id < 0 ? 0.f : a.scales ? a.scales[id] : 1.f;
    for (int k0 = 0; k0 < a.R; k0 += 32) {
      const int k = k0 + quarter * 8;
      u32x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
      if (id >= 0 && k < a.R) {
        float v[8] = {};
        for (int s = 0; s < a.splits; ++s) {
          const float* from = a.v + ((long long)s * a.T + token) * a.R + k;
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] += from[i];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          Bf16 h0, l0, h1, l1;
          split_f32(v[2 * i] * scale, h0, l0);
          split_f32(v[2 * i + 1] * scale, h1, l1);
          hi[i] = h0.v | (unsigned)h1.v << 16;
          lo[i] = l0.v | (unsigned)l1.v << 16;
        }
      }
      unsigned long long left = ballot(id >= 0) & 0xFFFFu;
      while (left) {
        const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        left &= ~ballot(id == slot);
        u32x4 w = load16(static_cast<const X*>(a.b) + ((long long)slot * a.O + brow) * a.R +
                         min(k, a.R - 8));
        w = keep(k < a.R, w);
        const f32x4 c = mfma_split<X>(w, 0, hi, lo, f32x4{0, 0, 0, 0});
#pragma unroll
        for (int i = 0; i < 4; ++i) total[i] += id == slot ? c[i] : 0.f;
      }
    }
  }
  if (token >= a.T || (id < 0 && a.base == a.out)) return;
  const X* base = static_cast<const X*>(a.base) + token * a.base_stride;
  X* out = static_cast<X*>(a.out) + token * a.out_stride;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int o = row0 + quarter * 4 + i;
    if (o < a.O) out[o] = id < 0 ? base[o] : from_f32<X>(to_f32(base[o]) + total[i]);
  }
}

}  // namespace ec
