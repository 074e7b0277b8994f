// expert_cache_adapt on gfx950: low-rank adapters of many requests, one slot a token, added to
// the output of a projection that all tokens share.
//
//   out_t = base_t + scale_s * B_s (A_s x_t),   s = slot id of token t
//
// Two launches: a shrink kernel makes A_s x_t in 32 bits, the hidden length split over workgroups,
// and an expand kernel joins the parts in a fixed order and adds B's product to the base. Tokens
// come in tiles of 16, the columns of the matrix instruction; where a tile's tokens have several
// adapters, each of them runs over the whole tile and the columns that are its own are taken from
// its product. A few tokens (adapters_shrink_k, adapters_expand_k) have as many adapters, so each
// adapter of a tile has workgroups of its own; of many tokens (.._many_k) neighbours share theirs,
// so a workgroup takes 64 and reads the adapter once for them.
#pragma once
#include "experts.h"
#include "mfma.h"
#include "wave.h"

namespace ec {

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
  bool aligned;  // rows of base and out are 16-byte aligned
  float* v;      // [splits][T][R]
};

// Slot of the tile's token (lane & 15), or -1.
__device__ __forceinline__ int tile_slot(const AdaptersArgs& a, int t0) {
  const int t = t0 + (__lane_id() & 15);
  const int id = load_id(a.ids, min(t, a.T - 1), a.wide, a.S);
  return t < a.T ? id : -1;
}

// A's product for one tile and the adapters blockIdx.y, blockIdx.y + gridDim.y, ... of its
// tokens that are an adapter's first, over one split of the hidden length: 16 * TILES ranks at
// a time, which share what is loaded of the tokens.
template <class X, int WAVES, int TILES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_shrink_k(AdaptersArgs a) {
  constexpr int kRows = TILES * kTile, D = 2;
  __shared__ float red[WAVES][TILES][4][kWave];
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kTile;
  const int id = tile_slot(a, t0);
  const int units = (a.H + kUnit - 1) / kUnit, per = (units + a.splits - 1) / a.splits;
  const int first = blockIdx.z * per, count = min(units - first, per);
  for (int which = blockIdx.y; which < kTile; which += gridDim.y) {
    const int slot = __builtin_amdgcn_readlane(id, which);
    const unsigned own = (unsigned)ballot(id == slot) & 0xFFFFu;
    if (slot < 0 || __builtin_ctz(own) != which) continue;
    // the columns of other adapters read what this one's first token has
    const int token = t0 + (own >> column & 1 ? column : which);
    const unsigned short* x = static_cast<const unsigned short*>(a.x) + token * a.x_stride;
    for (int r0 = 0; r0 < a.R; r0 += kRows) {
      const X* from = static_cast<const X*>(a.a) + ((long long)slot * a.R + r0) * a.H;
      unsigned rows[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        rows[t] = row_bytes<X>(r0 + t * kTile + column, r0, a.R, a.H);
      f32x4 acc[TILES];
#pragma unroll
      for (int t = 0; t < TILES; ++t) acc[t] = f32x4{0, 0, 0, 0};
      Rows<X> w[D][TILES];
      u32x4 b[D][4];
      pipeline<D>(
          (count - wave + WAVES - 1) / WAVES,
          [&](auto d, int i) EC_INLINE {
            const int u = first + wave + i * WAVES;
            each<TILES>([&](auto t) EC_INLINE {
              w[d][t].load(from, rows[t], nullptr, u, a.H, quarter);
            });
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              const int k = u * kUnit + operand_at<X>(f, quarter);
              b[d][f] = load16(x + (k < a.H ? k : 0));
            }
          },
          [&](auto d, int i) EC_INLINE {
            const int u = first + wave + i * WAVES;
            if ((u + 1) * kUnit > a.H) {
              each<TILES>([&](auto t) EC_INLINE { w[d][t].cut(u, a.H, quarter); });
#pragma unroll
              for (int f = 0; f < 4; ++f)
                b[d][f] = keep(u * kUnit + operand_at<X>(f, quarter) < a.H, b[d][f]);
            }
            each<TILES>([&](auto t) EC_INLINE { add_whole<X, X>(w[d][t], b[d], acc[t]); });
          });
      each<TILES>([&](auto t) EC_INLINE {
#pragma unroll
        for (int i = 0; i < 4; ++i) red[wave][t][i][lane] = acc[t][i];
      });
      lds_sync();
      for (int j = threadIdx.x; j < kRows * kTile; j += WAVES * kWave) {
        const int r = j % kRows, col = j / kRows;
        if (r0 + r < a.R && own >> col & 1) {
          float y = 0;
#pragma unroll
          for (int w = 0; w < WAVES; ++w) y += red[w][r / kTile][r & 3][r % kTile / 4 * 16 + col];
          a.v[((long long)blockIdx.z * a.T + t0 + col) * a.R + r0 + r] = y;
        }
      }
      lds_sync();
    }
  }
}

// B's product and the sum with the base for one tile, 16 * TILES outputs a wave. The rows of
// the TILES instructions are interleaved so that a lane ends with 4 * TILES neighbouring ones.
// AHEAD adapters of a tile are loaded at a time.
template <class X, int WAVES, int TILES, int AHEAD>
__global__ __launch_bounds__(WAVES* kWave) void adapters_expand_k(AdaptersArgs a) {
  constexpr int kRun = 4 * TILES;
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kTile, token = t0 + column;
  const int row0 = (blockIdx.y * WAVES + wave) * (16 * TILES);
  if (row0 >= a.O) return;
  const int id = tile_slot(a, t0);
  const bool fast = a.aligned && row0 + 16 * TILES <= a.O;
  const bool write = token < a.T && !(id < 0 && a.base == a.out);
  const int o0 = row0 + quarter * kRun;
  const unsigned short* base = static_cast<const unsigned short*>(a.base) +
                               min(token, a.T - 1) * a.base_stride + o0;
  unsigned short in[kRun];
  if (fast) {
    __builtin_memcpy(in, __builtin_assume_aligned(base, 8 * (TILES > 1 ? 2 : 1)), sizeof in);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i) in[i] = o0 + i < a.O ? base[i] : 0;
  }
  f32x4 total[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) total[t] = f32x4{0, 0, 0, 0};
  if (ballot(id >= 0)) {
    unsigned rows[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
      rows[t] = row_bytes<X>(row0 + (column >> 2) * kRun + t * 4 + (column & 3), row0, a.O, a.R);
    const float scale = id < 0 ? 0.f : a.scales ? a.scales[id] : 1.f;
    for (int k0 = 0; k0 < a.R; k0 += 32) {
      const int k = k0 + quarter * 8;
      const bool live = id >= 0 && k < a.R;
      f32x4 v0 = {0, 0, 0, 0}, v1 = v0;
      if (live) {
        const float* from = a.v + (long long)token * a.R + k;
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s) {
          v0 += *reinterpret_cast<const f32x4*>(from + (long long)s * a.T * a.R);
          v1 += *reinterpret_cast<const f32x4*>(from + (long long)s * a.T * a.R + 4);
        }
      }
      u32x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        Bf16 h0, l0, h1, l1;
        split_f32((i < 2 ? v0[2 * i] : v1[2 * i - 4]) * scale, h0, l0);
        split_f32((i < 2 ? v0[2 * i + 1] : v1[2 * i - 3]) * scale, h1, l1);
        hi[i] = h0.v | (unsigned)h1.v << 16;
        lo[i] = l0.v | (unsigned)l1.v << 16;
      }
      const unsigned at = (k < a.R ? k : 0) * 2u;
      unsigned long long left = ballot(id >= 0) & 0xFFFFu;
      while (left) {
        int slot[AHEAD];
        u32x4 w[AHEAD][TILES];
        each<AHEAD>([&](auto n) EC_INLINE {
          // (past the last adapter: the one before once more, for no column)
          const bool more = n == 0 || left != 0;
          const int s = more ? __builtin_amdgcn_readlane(id, __builtin_ctzll(left | 1ull << 32))
                             : slot[n > 0 ? n - 1 : 0];
          const int read = s < 0 ? 0 : s;
          left &= ~ballot(id == s);
          slot[n] = more ? s : -2;
          const char* from = static_cast<const char*>(a.b) +
                             ((long long)read * a.O + row0) * (2LL * a.R);
          each<TILES>([&](auto t) EC_INLINE { w[n][t] = load16(from + (rows[t] + at)); });
        });
        each<AHEAD>([&](auto n) EC_INLINE {
          each<TILES>([&](auto t) EC_INLINE {
            const f32x4 c = mfma_split<X>(keep(k < a.R, w[n][t]), 0, hi, lo, f32x4{0, 0, 0, 0});
#pragma unroll
            for (int i = 0; i < 4; ++i) total[t][i] += id == slot[n] ? c[i] : 0.f;
          });
        });
      }
    }
  }
  if (!write) return;
  unsigned short* out = static_cast<unsigned short*>(a.out) + token * a.out_stride + o0;
  if (id >= 0) {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      in[i] = from_f32<X>(to_f32(X{in[i]}) + total[i / 4][i & 3]).v;
  }
  if (fast) {
    __builtin_memcpy(__builtin_assume_aligned(out, 8 * (TILES > 1 ? 2 : 1)), in, sizeof in);
  } else {
#pragma unroll
    for (int i = 0; i < kRun; ++i)
      if (o0 + i < a.O) out[i] = in[i];
  }
}

constexpr int kManyTokens = 64;  // of a workgroup of the kernels below: a lane each
constexpr int kManyTiles = kManyTokens / kTile;

// A's product for 64 tokens over one split of the hidden length, 64 ranks at a time.
template <class X, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_shrink_many_k(AdaptersArgs a) {
  constexpr int T = kManyTiles, N = 4, kRows = N * kTile;
  __shared__ float red[WAVES][N][4][kWave];
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kManyTokens;
  int id = load_id(a.ids, min(t0 + lane, a.T - 1), a.wide, a.S);
  if (t0 + lane >= a.T) id = -1;
  const int units = (a.H + kUnit - 1) / kUnit, per = (units + a.splits - 1) / a.splits;
  const int first = blockIdx.y * per, count = min(units - first, per);
  for (unsigned long long left = ballot(id >= 0); left;) {
    const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const unsigned long long own = ballot(id == slot);
    left &= ~own;
    // columns of other adapters read what this one's first token has
    const unsigned short* x[T];
#pragma unroll
    for (int c = 0; c < T; ++c) {
      const int t = c * kTile + column;
      x[c] = static_cast<const unsigned short*>(a.x) +
             (t0 + (own >> t & 1 ? t : __builtin_ctzll(own))) * a.x_stride;
    }
    const auto has = [&](int c) EC_INLINE { return (own >> c * kTile & 0xFFFF) != 0; };
    for (int r0 = 0; r0 < a.R; r0 += kRows) {
      const X* from = static_cast<const X*>(a.a) + ((long long)slot * a.R + r0) * a.H;
      unsigned rows[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
        rows[n] = row_bytes<X>(r0 + n * kTile + column, r0, a.R, a.H);
      f32x4 acc[T][N];
#pragma unroll
      for (int c = 0; c < T; ++c)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[c][n] = f32x4{0, 0, 0, 0};
      for (int i = wave; i < count; i += WAVES) {
        const int u = first + i;
        Rows<X> w[N];
        u32x4 b[T][4];
        each<N>([&](auto n) EC_INLINE { w[n].load(from, rows[n], nullptr, u, a.H, quarter); });
        each<T>([&](auto c) EC_INLINE {
          if (has(c)) {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              const int k = u * kUnit + operand_at<X>(f, quarter);
              b[c][f] = load16(x[c] + (k < a.H ? k : 0));
            }
          }
        });
        if ((u + 1) * kUnit > a.H) {
          each<N>([&](auto n) EC_INLINE { w[n].cut(u, a.H, quarter); });
          each<T>([&](auto c) EC_INLINE {
#pragma unroll
            for (int f = 0; f < 4; ++f)
              b[c][f] = keep(u * kUnit + operand_at<X>(f, quarter) < a.H, b[c][f]);
          });
        }
        each<T>([&](auto c) EC_INLINE {
          if (has(c))
            each<N>([&](auto n) EC_INLINE { add_whole<X, X>(w[n], b[c], acc[c][n]); });
        });
      }
      each<T>([&](auto c) EC_INLINE {
        if (!has(c)) return;
        lds_sync();
        each<N>([&](auto n) EC_INLINE {
#pragma unroll
          for (int i = 0; i < 4; ++i) red[wave][n][i][lane] = acc[c][n][i];
        });
        lds_sync();
        for (int j = threadIdx.x; j < kRows * kTile; j += WAVES * kWave) {
          const int r = j % kRows, t = c * kTile + j / kRows;
          if (r0 + r < a.R && own >> t & 1) {
            float y = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w)
              y += red[w][r / kTile][r & 3][r % kTile / 4 * 16 + j / kRows];
            a.v[((long long)blockIdx.y * a.T + t0 + t) * a.R + r0 + r] = y;
          }
        }
      });
    }
  }
}

// B's product and the sum with the base for 64 tokens, 64 outputs a wave: the tokens' low-rank
// values are joined, scaled and split into two bfloat16 once for the workgroup, in LDS.
template <class X, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_expand_many_k(AdaptersArgs a) {
  constexpr int T = kManyTiles, N = 4, kRun = 4 * N, kRanks = 64;
  __shared__ __attribute__((aligned(16))) Bf16 low[2][kManyTokens][kRanks + 8];
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kManyTokens;
  const int row0 = (blockIdx.y * WAVES + wave) * (16 * N);
  const bool some = row0 < a.O;
  const int o0 = row0 + quarter * kRun;
  const bool fast = a.aligned && row0 + 16 * N <= a.O;
  u32x4 in[T][2];
#pragma unroll
  for (int c = 0; c < T; ++c) {
    const long long token = min(t0 + c * kTile + column, a.T - 1);
    const unsigned short* base =
        static_cast<const unsigned short*>(a.base) + token * a.base_stride + o0;
    if (fast) {
      in[c][0] = load16(base);
      in[c][1] = load16(base + 8);
    } else {
#pragma unroll
      for (int i = 0; i < kRun / 2; ++i) {
        const unsigned lo = o0 + 2 * i < a.O ? base[2 * i] : 0;
        const unsigned hi = o0 + 2 * i + 1 < a.O ? base[2 * i + 1] : 0;
        in[c][i / 4][i % 4] = lo | hi << 16;
      }
    }
  }
  int id = load_id(a.ids, min(t0 + lane, a.T - 1), a.wide, a.S);
  if (t0 + lane >= a.T) id = -1;
  const unsigned long long with = ballot(id >= 0);
  f32x4 total[T][N];
#pragma unroll
  for (int c = 0; c < T; ++c)
#pragma unroll
    for (int n = 0; n < N; ++n) total[c][n] = f32x4{0, 0, 0, 0};
  unsigned rows[N];
#pragma unroll
  for (int n = 0; n < N; ++n)
    rows[n] = row_bytes<X>(min(row0, a.O - 1) + (column >> 2) * kRun + n * 4 + (column & 3),
                           min(row0, a.O - 1), a.O, a.R);
  for (int r0 = 0; with && r0 < a.R; r0 += kRanks) {
    lds_sync();
    for (int j = threadIdx.x; j < kManyTokens * (kRanks / 4); j += WAVES * kWave) {
      const int t = j / (kRanks / 4), r = j % (kRanks / 4) * 4;
      const int slot = __shfl(id, t);
      f32x4 v = {0, 0, 0, 0};
      if (slot >= 0 && r0 + r < a.R) {
        const float* from = a.v + (long long)(t0 + t) * a.R + r0 + r;
#pragma unroll 4
        for (int s = 0; s < a.splits; ++s)
          v += *reinterpret_cast<const f32x4*>(from + (long long)s * a.T * a.R);
        v *= a.scales ? a.scales[slot] : 1.f;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) split_f32(v[i], low[0][t][r + i], low[1][t][r + i]);
    }
    lds_sync();
    for (unsigned long long left = some ? with : 0; left;) {
      const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      const unsigned long long own = ballot(id == slot);
      left &= ~own;
      const char* from =
          static_cast<const char*>(a.b) + ((long long)slot * a.O + row0) * (2LL * a.R);
      u32x4 w[2][N];
      each<2>([&](auto h) EC_INLINE {
        const int k = r0 + h * 32 + quarter * 8;
        each<N>([&](auto n) EC_INLINE {
          w[h][n] = load16(from + (rows[n] + (k < a.R ? k : 0) * 2u));
        });
      });
      if (r0 + kRanks > a.R) {
        each<2>([&](auto h) EC_INLINE {
          const bool live = r0 + h * 32 + quarter * 8 < a.R;
          each<N>([&](auto n) EC_INLINE { w[h][n] = keep(live, w[h][n]); });
        });
      }
      each<T>([&](auto c) EC_INLINE {
        if ((own >> c * kTile & 0xFFFF) == 0) return;
        f32x4 sum[N];
        each<N>([&](auto n) EC_INLINE { sum[n] = f32x4{0, 0, 0, 0}; });
        each<2>([&](auto h) EC_INLINE {
          const int t = c * kTile + column, k = h * 32 + quarter * 8;
          const u32x4 hi = load16(&low[0][t][k]), lo = load16(&low[1][t][k]);
          each<N>([&](auto n) EC_INLINE { sum[n] = mfma_split<X>(w[h][n], 0, hi, lo, sum[n]); });
        });
        const bool mine = own >> (c * kTile + column) & 1;
        each<N>([&](auto n) EC_INLINE {
#pragma unroll
          for (int i = 0; i < 4; ++i) total[c][n][i] += mine ? sum[n][i] : 0.f;
        });
      });
    }
  }
  if (!some) return;
  each<T>([&](auto c) EC_INLINE {
    const int t = c * kTile + column;
    const bool adapted = with >> t & 1;
    if (t0 + t >= a.T || (!adapted && a.base == a.out)) return;
    unsigned short* out = static_cast<unsigned short*>(a.out) + (t0 + t) * a.out_stride + o0;
    if (adapted) {
#pragma unroll
      for (int i = 0; i < kRun / 2; ++i) {
        const unsigned v = in[c][i / 4][i % 4];
        const X lo{(unsigned short)v}, hi{(unsigned short)(v >> 16)};
        in[c][i / 4][i % 4] =
            from_f32<X>(to_f32(lo) + total[c][i / 2][2 * i & 3]).v |
            (unsigned)from_f32<X>(to_f32(hi) + total[c][i / 2][(2 * i + 1) & 3]).v << 16;
      }
    }
    if (fast) {
      *reinterpret_cast<u32x4*>(out) = in[c][0];
      *reinterpret_cast<u32x4*>(out + 8) = in[c][1];
    } else {
#pragma unroll
      for (int i = 0; i < kRun; ++i)
        if (o0 + i < a.O) out[i] = (unsigned short)(in[c][i / 8][i / 2 % 4] >> (i & 1) * 16);
    }
  });
}

}  // namespace ec
