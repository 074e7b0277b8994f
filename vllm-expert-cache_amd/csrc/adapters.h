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

// A's product for one tile and the adapter of its token blockIdx.y, if that is the adapter's
// first, over one split of the hidden length and 16 * TILES ranks, which share what is loaded of
// the tokens. 33 tokens with an adapter each, rank 32, H 4096: 6.8 us for 7.6 MB, of which the
// launch and one chain of loads are most.
template <class X, int WAVES, int TILES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_shrink_k(AdaptersArgs a) {
  constexpr int kRows = TILES * kTile, D = 2;
  __shared__ float red[WAVES][TILES][4][kWave];
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kTile, which = blockIdx.y;
  const int id = tile_slot(a, t0);
  const int slot = __builtin_amdgcn_readlane(id, which);
  const unsigned own = (unsigned)ballot(id == slot) & 0xFFFFu;
  if (slot < 0 || __builtin_ctz(own) != which) return;
  const int split = blockIdx.z % a.splits, r0 = blockIdx.z / a.splits * kRows;
  const int units = (a.H + kUnit - 1) / kUnit, per = (units + a.splits - 1) / a.splits;
  const int first = split * per, count = min(units - first, per);
  // the columns of other adapters read what this one's first token has
  const int token = t0 + (own >> column & 1 ? column : which);
  const unsigned short* x = static_cast<const unsigned short*>(a.x) + token * a.x_stride;
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
  products_done();
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
      a.v[((long long)split * a.T + t0 + col) * a.R + r0 + r] = y;
    }
  }
}

// B's product and the sum with the base for one tile, 16 outputs a wave: few, so that a tile has
// many waves. Of the tile's adapters a workgroup takes every gridDim.z-th and writes the rows of
// their tokens; the first one writes those without an adapter as well. AHEAD adapters are loaded
// at a time: 33 tokens, rank 64, H and O 4096, an adapter each, all of a tile's in one workgroup,
// take 27.1 us a call one by one and 23.4 us four by four. With rank 32 and four workgroups the
// kernel takes 5.6 us: two chains of loads (ids, then values and B) and the launch.
template <class X, int WAVES, int AHEAD>
__global__ __launch_bounds__(WAVES* kWave) void adapters_expand_k(AdaptersArgs a) {
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.x * kTile, token = t0 + column;
  const int row0 = (blockIdx.y * WAVES + wave) * kTile;
  if (row0 >= a.O) return;
  int id = tile_slot(a, t0);
  bool mine = id < 0 && blockIdx.z == 0 && a.base != a.out;
  int which = 0;
  for (unsigned left = (unsigned)ballot(id >= 0) & 0xFFFFu; left; ++which) {
    const bool same = id == __builtin_amdgcn_readlane(id, __builtin_ctz(left));
    left &= ~(unsigned)ballot(same);
    if (which % gridDim.z == blockIdx.z) mine |= same;
  }
  const bool write = token < a.T && mine;
  if (ballot(write) == 0) return;
  if (!mine) id = -1;  // another workgroup's
  const bool fast = a.aligned && row0 + kTile <= a.O;
  const int o0 = row0 + quarter * 4;
  const unsigned short* base = static_cast<const unsigned short*>(a.base) +
                               min(token, a.T - 1) * a.base_stride + o0;
  unsigned short in[4] = {};
  if (write && fast) {
    __builtin_memcpy(in, __builtin_assume_aligned(base, 8), sizeof in);
  } else if (write) {
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = o0 + i < a.O ? base[i] : 0;
  }
  f32x4 total = {0, 0, 0, 0};
  if (ballot(id >= 0)) {
    const unsigned row = row_bytes<X>(row0 + column, row0, a.O, a.R);
    const float scale = id < 0 ? 0.f : a.scales ? a.scales[id] : 1.f;
    for (int k0 = 0; k0 < a.R; k0 += 32) {
      const int k = k0 + quarter * 8;
      const unsigned at = (k < a.R ? k : 0) * 2u;
      unsigned left = (unsigned)ballot(id >= 0) & 0xFFFFu;
      int slot[AHEAD];
      u32x4 w[AHEAD];
      const auto load = [&]() EC_INLINE {
        each<AHEAD>([&](auto n) EC_INLINE {
          // (past the last adapter: the one before once more, for no column)
          const bool more = n == 0 || left != 0;
          const int s = more ? __builtin_amdgcn_readlane(id, __builtin_ctz(left | 1u << 31))
                             : slot[n > 0 ? n - 1 : 0];
          const int read = s < 0 ? 0 : s;
          left &= ~(unsigned)ballot(id == s);
          slot[n] = more ? s : -2;
          w[n] = load16(static_cast<const char*>(a.b) +
                        ((long long)read * a.O + row0) * (2LL * a.R) + (row + at));
        });
      };
      load();  // under way while the tokens' values are joined
      f32x4 v0 = {0, 0, 0, 0}, v1 = v0;
      if (id >= 0 && k < a.R) {
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
      for (;;) {
        each<AHEAD>([&](auto n) EC_INLINE {
          const f32x4 c = mfma_split<X>(keep(k < a.R, w[n]), 0, hi, lo, f32x4{0, 0, 0, 0});
#pragma unroll
          for (int i = 0; i < 4; ++i) total[i] += id == slot[n] ? c[i] : 0.f;
        });
        settled(total);
        if (left == 0) break;
        load();
      }
    }
  }
  if (!write) return;
  unsigned short* out = static_cast<unsigned short*>(a.out) + token * a.out_stride + o0;
  if (id >= 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) in[i] = from_f32<X>(to_f32(X{in[i]}) + total[i]).v;
  }
  if (fast) {
    __builtin_memcpy(__builtin_assume_aligned(out, 8), in, sizeof in);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (o0 + i < a.O) out[i] = in[i];
  }
}

constexpr int kManyTokens = 64;  // of a workgroup of the kernels below: a lane each
constexpr int kManyTiles = kManyTokens / kTile;

// A's product for 64 tokens over one split of the hidden length, 64 ranks at a time. A unit of
// the tokens and of A goes through LDS: from the L1 each wave would take the rows it shares with
// the others for itself, and what a compute unit gets from its L1 (56 bytes/ns) is the bound
// then. A wave has 32 of the ranks, 32 of the tokens and a part of each unit. 4096 tokens, H
// 4096, rank 64, 7 adapters: 18.6 us for 33.5 MB of tokens, one workgroup a compute unit (170
// registers), bound by the barriers of a unit and by workgroups whose tokens have two adapters.
// 32 ranks at a time for short ranks gain nothing (rank 16 18.9 / 18.7, rank 32 35.6 / 36.3 us a
// call).
template <class X>
__global__ __launch_bounds__(8 * kWave, 2) void adapters_shrink_many_k(AdaptersArgs a) {
  constexpr int kRows = 64, D = 4;
  constexpr int kPitch = 2 * kUnit + 16;  // bytes of a row: 16 rows start in different banks
  constexpr int kLine = 2 * kUnit / 16;   // lanes that read a row's unit
  constexpr int kEach = 8 * kWave / kLine;  // rows that the workgroup reads at once
  __shared__ __attribute__((aligned(16))) union {
    char unit[2][kRows + kManyTokens][kPitch];
    f32x4 parts[4][2][2][kWave];
  } lds;
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int half = wave & 1, group = wave / 2 % 2, part = wave / 4;
  const int t0 = blockIdx.x * kManyTokens;
  int id = load_id(a.ids, min(t0 + lane, a.T - 1), a.wide, a.S);
  if (t0 + lane >= a.T) id = -1;
  // a split has every a.splits-th unit, and each workgroup starts at another of them
  const int units = (a.H + kUnit - 1) / kUnit;
  const int count = (units - (int)blockIdx.y + a.splits - 1) / a.splits;
  const int start = first_unit(blockIdx.x, count);
  const int my_row = threadIdx.x / kLine, my_k = threadIdx.x % kLine * 8;
  for (unsigned long long left = ballot(id >= 0); left;) {
    const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
    const unsigned long long own = ballot(id == slot);
    left &= ~own;
    const bool any = (unsigned)(own >> half * 32) != 0;
    // tokens of other adapters read what this one's first token has
    const unsigned short* x[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int t = my_row + j * kEach;
      x[j] = static_cast<const unsigned short*>(a.x) +
             (t0 + (own >> t & 1 ? t : __builtin_ctzll(own))) * a.x_stride;
    }
    for (int r0 = 0; r0 < a.R; r0 += kRows) {
      const char* from = static_cast<const char*>(a.a) + ((long long)slot * a.R + r0) * (2LL * a.H);
      unsigned rows[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) rows[j] = row_bytes<X>(r0 + my_row + j * kEach, r0, a.R, a.H);
      f32x4 acc[2][2];
      each<2>([&](auto r) EC_INLINE {
        each<2>([&](auto c) EC_INLINE { acc[r][c] = f32x4{0, 0, 0, 0}; });
      });
      u32x4 w[D][2], b[D][2];
      const auto unit = [&](int i) EC_INLINE {
        return (int)blockIdx.y + a.splits * wrap(i + start, count);
      };
      lds_sync();  // the parts of the ranks before have been read
      pipeline<D>(
          count,
          [&](auto d, int i) EC_INLINE {
            const int k = unit(i) * kUnit + my_k;
            const unsigned at = k < a.H ? 2u * k : 0u;
            each<2>([&](auto j) EC_INLINE { w[d][j] = load16(from + (rows[j] + at)); });
            each<2>([&](auto j) EC_INLINE { b[d][j] = load16(x[j] + at / 2); });
          },
          [&](auto d, int i) EC_INLINE {
            char(*to)[kPitch] = lds.unit[i & 1];
            const bool in = unit(i) * kUnit + my_k < a.H;
            each<2>([&](auto j) EC_INLINE {
              *reinterpret_cast<u32x4*>(&to[my_row + j * kEach][2 * my_k]) = keep(in, w[d][j]);
            });
            each<2>([&](auto j) EC_INLINE {
              *reinterpret_cast<u32x4*>(&to[kRows + my_row + j * kEach][2 * my_k]) =
                  keep(in, b[d][j]);
            });
            lds_sync();  // two units in turn: the other is free once all have come here
            if (!any) return;
            each<2>([&](auto s) EC_INLINE {  // 32 values of k at a time, of the unit's four
              const int k = (part * 2 + s) * 64 + quarter * 16;
              u32x4 rw[2], cl[2];
              each<2>([&](auto n) EC_INLINE {
                rw[n] = load16(&to[group * 32 + n * 16 + column][k]);
                cl[n] = load16(&to[kRows + half * 32 + n * 16 + column][k]);
              });
              each<2>([&](auto r) EC_INLINE {
                each<2>([&](auto c) EC_INLINE {
                  acc[r][c] = Frag<X>::mfma(rw[r], cl[c], acc[r][c]);
                });
              });
            });
          });
      products_done();
      lds_sync();
      if (part) {
        each<2>([&](auto r) EC_INLINE {
          each<2>([&](auto c) EC_INLINE {
            lds.parts[wave - 4][r][c][lane] = acc[r][c];
          });
        });
      }
      lds_sync();
      if (!part) {
        each<2>([&](auto r) EC_INLINE {
          each<2>([&](auto c) EC_INLINE {
            const int t = half * 32 + c * 16 + column;
            const int row = r0 + group * 32 + r * 16 + quarter * 4;
            const f32x4 y = acc[r][c] + lds.parts[wave][r][c][lane];
            if (own >> t & 1 && row < a.R)
              *reinterpret_cast<f32x4*>(
                  a.v + ((long long)blockIdx.y * a.T + t0 + t) * a.R + row) = y;
          });
        });
      }
    }
  }
}

// B's product and the sum with the base for 64 tokens: the tokens' low-rank values are joined,
// scaled and split into two bfloat16 once for the workgroup, in LDS. A wave has 64 outputs; the
// rows of its instructions are interleaved so that a lane ends with two runs of eight neighbouring
// outputs and the wave reads and writes 64 bytes of a token at a time. 4096 tokens, rank 64, O
// 4096: 28.0 us for 67 MB read and written (2.4 TB/s), bound by the chain from ids over values and
// split to the products: at 212 registers a compute unit holds one workgroup, so the 512 of them
// run in two rounds with nothing beside a chain. Float16 takes all 256 registers and 100 bytes of
// scratch a lane, for weights in halves; the whole call takes 58 us and not 49.
template <class X, int WAVES>
__global__ __launch_bounds__(WAVES* kWave) void adapters_expand_many_k(AdaptersArgs a) {
  constexpr int T = kManyTiles, N = 4, kRanks = 64;
  __shared__ __attribute__((aligned(16))) Bf16 low[2][kManyTokens][kRanks + 8];
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t0 = blockIdx.y * kManyTokens;
  const int row0 = (blockIdx.x * WAVES + wave) * (16 * N);
  const bool some = row0 < a.O;
  const int o0 = row0 + quarter * 8;  // eight outputs from here, and eight from 32 after it
  const bool fast = a.aligned && row0 + 16 * N <= a.O;
  int id = load_id(a.ids, min(t0 + lane, a.T - 1), a.wide, a.S);
  u32x4 in[T][2];
#pragma unroll
  for (int c = 0; c < T; ++c) {
    const long long token = min(t0 + c * kTile + column, a.T - 1);
    const unsigned short* base =
        static_cast<const unsigned short*>(a.base) + token * a.base_stride + o0;
    if (fast) {
      in[c][0] = load16(base);
      in[c][1] = load16(base + 32);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int at = i / 4 * 32 + i % 4 * 2;
        const unsigned lo = o0 + at < a.O ? base[at] : 0;
        const unsigned hi = o0 + at + 1 < a.O ? base[at + 1] : 0;
        in[c][i / 4][i % 4] = lo | hi << 16;
      }
    }
  }
  if (t0 + lane >= a.T) id = -1;
  const unsigned long long with = ballot(id >= 0);
  const float scale = id < 0 ? 0.f : a.scales ? a.scales[id] : 1.f;
  f32x4 total[T][N];
#pragma unroll
  for (int c = 0; c < T; ++c)
#pragma unroll
    for (int n = 0; n < N; ++n) total[c][n] = f32x4{0, 0, 0, 0};
  unsigned rows[N];
  const int from0 = min(row0, a.O - 1);
#pragma unroll
  for (int n = 0; n < N; ++n)
    rows[n] = row_bytes<X>(from0 + n / 2 * 32 + (column >> 2) * 8 + n % 2 * 4 + (column & 3),
                           from0, a.O, a.R);
  u32x4 w[2][N];
  // 64 ranks of an adapter's rows
  const auto load_rows = [&](int slot, int r0) EC_INLINE {
    const char* from = static_cast<const char*>(a.b) +
                       ((long long)slot * a.O + from0) * (2LL * a.R);
    each<2>([&](auto h) EC_INLINE {
      const int k = r0 + h * 32 + quarter * 8;
      each<N>([&](auto n) EC_INLINE {
        w[h][n] = load16(from + (rows[n] + (k < a.R ? k : 0) * 2u));
      });
    });
  };
  for (int r0 = 0; with && r0 < a.R; r0 += kRanks) {
    // the first adapter's rows come while the tokens' values are joined
    load_rows(__builtin_amdgcn_readlane(id, __builtin_ctzll(with)), r0);
    lds_sync();
    constexpr int kEach = kManyTokens * (kRanks / 4) / (WAVES * kWave);
    const int t = threadIdx.x / (kRanks / 4), r = threadIdx.x % (kRanks / 4) * 4;
    constexpr int kStep = kManyTokens / kEach;  // tokens between a thread's values
    f32x4 v[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) v[j] = f32x4{0, 0, 0, 0};
#pragma unroll 2
    for (int s = 0; s < a.splits; ++s)
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        v[j] += *reinterpret_cast<const f32x4*>(
            a.v + ((long long)s * a.T + min(t0 + t + j * kStep, a.T - 1)) * a.R +
            min(r0 + r, a.R - 4));
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int at = t + j * kStep;
      v[j] *= __shfl(scale, at);
      const bool live = r0 + r < a.R && (with >> at & 1);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        split_f32(live ? v[j][i] : 0.f, low[0][at][r + i], low[1][at][r + i]);
    }
    lds_sync();
    bool loaded = true;
    for (unsigned long long left = some ? with : 0; left;) {
      const int slot = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
      const unsigned long long own = ballot(id == slot);
      left &= ~own;
      if (!loaded) load_rows(slot, r0);
      loaded = false;
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
          settled(total[c][n]);
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
      for (int i = 0; i < 8; ++i) {
        const unsigned v = in[c][i / 4][i % 4];
        const X lo{(unsigned short)v}, hi{(unsigned short)(v >> 16)};
        in[c][i / 4][i % 4] =
            from_f32<X>(to_f32(lo) + total[c][i / 2][2 * i & 3]).v |
            (unsigned)from_f32<X>(to_f32(hi) + total[c][i / 2][(2 * i + 1) & 3]).v << 16;
      }
    }
    if (fast) {
      *reinterpret_cast<u32x4*>(out) = in[c][0];
      *reinterpret_cast<u32x4*>(out + 32) = in[c][1];
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int at = i / 8 * 32 + i % 8;
        if (o0 + at < a.O) out[at] = (unsigned short)(in[c][i / 8][i / 2 % 4] >> (i & 1) * 16);
      }
    }
  });
}

}  // namespace ec
