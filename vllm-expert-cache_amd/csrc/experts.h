// expert_cache_moe on gfx950: a whole MoE layer for a few tokens over slot-resident experts.
//
//   y_t = sum_j p_tj W2_s (silu(Wg_s x_t) * (Wu_s x_t)),   s = slot id j of token t
//
// experts_up_k makes gate and up projection, SiLU product and routing weight; up to 16 tokens
// experts_down_k makes the down projection and the sum over a token's experts, above that
// experts_pairs_k the down projection of every pair and experts_sum_k the sum.
//
// A few tokens read every weight of their experts once and do 2-32 operations on it, so the
// step is bound by the slots' bytes. A workgroup takes 16 rows of one expert for all of that
// expert's tokens, its waves split the rows' length between them, and LDS joins them. Pairs
// that name the same slot are found by every workgroup for itself: the step has at most 1024.
#pragma once
#include "mfma.h"
#include "wave.h"

#include <utility>

#define EC_INLINE __attribute__((always_inline))

namespace ec {

constexpr int kExpertsMaxPairs = 1024;
constexpr int kExpertsMaxK = 64;
constexpr int kUnit = 128;  // values of k a wave takes at a time: one block of e4m3 scales
constexpr int kTile = 16;   // rows, and columns of tokens, of one matrix instruction
constexpr int kFewTokens = 16;  // most tokens of experts_down_k

// What experts_up_k leaves of one slot (or pair) for experts_down_k: the slot, how many tokens
// are its, and their pairs.
struct alignas(16) ExpertsMeta {
  unsigned slot, count;
  unsigned pairs[kFewTokens / 2];  // two each
  unsigned unused[2];
};

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
  bool few;     // experts_down_k makes the down projection
  Bf16* hi;  // [n][I] hidden values times routing weight, as two bfloat16
  Bf16* lo;
  float* part;        // [n][H]; few: [tiles of H][splits][16][16], where splits > 1
  ExpertsMeta* meta;  // few: [n or S]
  int* arrived;       // few: [down_groups] workgroups that have left their part
  int down_groups, splits;
  int k_waves;  // not few: waves that share a row's length
  void* out;
  long long out_stride;  // elements
};

// f(0), f(1), ... f(N - 1) with compile-time arguments: arrays that they index stay in registers.
template <class F, int... I>
__device__ __forceinline__ void each(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __forceinline__ void each(F&& f) {
  each(f, std::make_integer_sequence<int, N>());
}

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

struct Pairs {
  unsigned short pair[kExpertsMaxPairs];
  float weight[kExpertsMaxPairs];
};

// The pairs of the workgroup's slot with their weights, in order of tokens, into LDS; their
// number, or 0 where there are none or they are another workgroup's. A workgroup belongs to pair
// `p` (and its slot, if p is the first pair that names it), or, where there are more pairs than
// slots, to slot `p`. A pair whose weight is zero is left out; a token that names the slot twice
// has one pair with both weights. Every wave goes through the ids, the first one writes.
__device__ __forceinline__ int list_pairs(const ExpertsArgs& a, int p, int& slot, Pairs& list) {
  const int lane = __lane_id();
  const bool writer = threadIdx.x < kWave;
  int at = min(lane, a.n - 1);
  RawId own = raw_id(a.ids, min(p, a.n - 1), a.wide), raw = raw_id(a.ids, at, a.wide);
  float w = a.probs[at];
  together(own, raw, w);
  int id = id_of(raw, a.wide, a.S);
  slot = a.by_slot ? p : __builtin_amdgcn_readfirstlane(id_of(own, a.wide, a.S));
  if (slot < 0) return 0;
  int count = 0, last = -1;  // last token seen
  // 64 pairs from `base`; false if the slot is another workgroup's
  const auto take = [&](int base, int at, int id, float w) EC_INLINE {
    const bool mine = id == slot && w != 0.f && base + lane < a.n;
    const unsigned long long m = ballot(mine);
    if (m == 0) return true;
    if (count == 0 && !a.by_slot && base + __builtin_ctzll(m) != p) return false;
    const int token = at / a.k;
    const unsigned long long before = m & lanes_below();
    const int prev = __shfl(token, before ? 63 - __builtin_clzll(before) : 0);
    const bool again = mine && token == (before ? prev : last);
    const unsigned long long firsts = ballot(mine && !again);
    const int pos = count + __builtin_popcountll(firsts & lanes_below()) - (again ? 1 : 0);
    if (writer) {
      if (mine && !again) {
        list.pair[pos] = (unsigned short)at;
        list.weight[pos] = w;
      }
      for (unsigned long long r = m & ~firsts; r; r &= r - 1)
        if (lane == __builtin_ctzll(r)) list.weight[pos] += w;
    }
    count += __builtin_popcountll(firsts);
    last = __shfl(token, 63 - __builtin_clzll(m));
    return true;
  };
  if (!take(0, at, id, w)) return 0;
  // Loads of four lots are under way at once: one lot at a time, 128 tokens, top-8, 2048 x 256
  // take 123 us and not 111.
  constexpr int kAhead = 4;
  for (int base = kWave; base < a.n; base += kAhead * kWave) {
    RawId raws[kAhead];
    float ws[kAhead];
    each<kAhead>([&](auto j) EC_INLINE {
      at = min(base + j * kWave + lane, a.n - 1);
      raws[j] = raw_id(a.ids, at, a.wide);
      ws[j] = a.probs[at];
    });
    bool own_slot = true;
    each<kAhead>([&](auto j) EC_INLINE {
      const int from = base + j * kWave;
      if (own_slot && from < a.n)
        own_slot = take(from, min(from + lane, a.n - 1), id_of(raws[j], a.wide, a.S), ws[j]);
    });
    if (!own_slot) return 0;
  }
  return count;
}

__device__ __forceinline__ u32x4 keep(bool c, u32x4 v) {
  return u32x4{c ? v[0] : 0, c ? v[1] : 0, c ? v[2] : 0, c ? v[3] : 0};
}

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

template <class W>
struct Rows {
  static constexpr int kLoads = sizeof(W) == 2 ? 4 : 2;
  u32x4 w[kLoads];
  float s;  // e4m3: the scale of the unit's block

  // `base`: the tile's first row (the same in all lanes); `row`: bytes from there to the lane's.
  __device__ __forceinline__ void load(const W* base, unsigned row, const float* scale, int u,
                                       int K, int quarter) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l) {
      const unsigned at = u * kUnit + load_at<W>(l, quarter);
      w[l] = load16(reinterpret_cast<const char*>(base) +
                    (row + (at < (unsigned)K ? at * (unsigned)sizeof(W) : 0u)));
    }
    if constexpr (__is_same(W, E4m3)) s = load_uniform(scale + u);
  }
  // Past the end of k weights and columns are zero (a weight read there may be no number).
  __device__ __forceinline__ void cut(int u, int K, int quarter) {
#pragma unroll
    for (int l = 0; l < kLoads; ++l)
      w[l] = keep(u * kUnit + load_at<W>(l, quarter) < K, w[l]);
  }
  __device__ __forceinline__ u32x4 at(int f) const { return w[sizeof(W) == 2 ? f : f >> 1]; }
};

// 8 * G rows times packed columns. A wave that has few tokens lets the 16 columns of the operand be
// pieces of the unit: its four operands of eight values (times two where a value is two
// bfloat16) of up to four (two) tokens, all in one load, where whole columns take four (eight)
// loads. A load costs a compute unit the same whether one lane in four or each has something
// to read. The weights' rows are pieces as well: of the 16 rows of an instruction the first
// eight are the first 64 bytes of eight rows and the others their next 64, so that a load takes
// 128 bytes of a row at once (which loads past the caches need to be fast). Of a product only
// the columns whose piece goes with the weights mean anything: row m's half m / 8 and the
// instruction x of two have piece 2 * (m / 8) + x. The sums of the two instructions and of the
// rows' two groups are kept apart; in the end a lane takes what is its column's, if anything,
// and a token's columns and halves are added up.
template <class W, int G>
struct Packed {
  static constexpr int kWide = sizeof(W) == 2 ? 2 : 1;  // loads along k of a row group
  u32x4 w[G][kWide];
  u32x4 b;
  float s;  // e4m3: the scale of the unit's block

  // Where the lane's loads and its piece of the columns start in a unit.
  static __device__ __forceinline__ int row_at() {
    const int m = __lane_id() & 15, quarter = __lane_id() >> 4;
    return (m >> 3) * (64 / sizeof(W)) + quarter * (16 / sizeof(W));
  }
  static __device__ __forceinline__ int piece_at() {
    const int f = __lane_id() & 3, quarter = __lane_id() >> 4;
    return sizeof(W) == 2 ? (2 * (f & 1) + (f >> 1)) * 32 + quarter * 8
                          : (f >> 1) * 64 + quarter * 16 + (f & 1) * 8;
  }
  // `base`: the tile's first row (the same in all lanes); `row`: bytes from there to the lane's
  // row of each group; `col`: its column.
  template <bool ONCE>
  __device__ __forceinline__ void load(const W* base, const unsigned (&row)[G],
                                       const float* scale, int u, int K) {
#pragma unroll
    for (int l = 0; l < kWide; ++l) {
      unsigned at = u * kUnit + row_at() + l * 64;
      at = at < (unsigned)K ? at * (unsigned)sizeof(W) : 0u;
#pragma unroll
      for (int g = 0; g < G; ++g)
        w[g][l] = load16_of<ONCE>(reinterpret_cast<const char*>(base) + (row[g] + at));
    }
    if constexpr (__is_same(W, E4m3)) s = load_uniform(scale + u);
  }
  __device__ __forceinline__ void load_cols(const void* col, int u, int K) {
    const int at = u * kUnit + piece_at();
    b = load16(static_cast<const unsigned short*>(col) + (at < K ? at : 0));
  }
  // Past the end of k weights and columns are zero.
  __device__ __forceinline__ void cut(int u, int K) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int l = 0; l < kWide; ++l)
        w[g][l] = keep(u * kUnit + row_at() + l * 64 < K, w[g][l]);
    b = keep(u * kUnit + piece_at() < K, b);
  }
};

template <class W, int G>
struct PackedSum {
  static constexpr int kApart = __is_same(W, E4m3) ? 1 : 2;  // scales need the lane's own at once
  f32x4 c[G][kApart];

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int x = 0; x < kApart; ++x) c[g][x] = f32x4{0, 0, 0, 0};
  }
  static __device__ __forceinline__ f32x4 pick(f32x4 even, f32x4 odd) {
    const bool o = __lane_id() & 1;
    return f32x4{o ? odd[0] : even[0], o ? odd[1] : even[1], o ? odd[2] : even[2],
                 o ? odd[3] : even[3]};
  }
  // Columns of X, values of which are the weights' operand.
  template <class X>
  __device__ __forceinline__ void add(const Packed<W, G>& r) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      f32x4 t[2];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        t[x] = __is_same(W, E4m3) ? f32x4{0, 0, 0, 0} : c[g][x % kApart];
        if constexpr (__is_same(X, Bf16) && __is_same(W, F16)) {
          u32x4 hi, lo;
          split_f16(r.w[g][x], hi, lo);
          t[x] = Frag<Bf16>::mfma(lo, r.b, t[x]);
          t[x] = Frag<Bf16>::mfma(hi, r.b, t[x]);
        } else {
          const u32x4 v = r.w[g][x % Packed<W, G>::kWide];
          t[x] = Frag<X>::mfma(operand<X, W>(v, x), r.b, t[x]);
        }
      }
      if constexpr (__is_same(W, E4m3)) {
        const f32x4 v = pick(t[0], t[1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[g][0][i] = fmaf(r.s, v[i], c[g][0][i]);
        settled(c[g][0]);
      } else {
        c[g][0] = t[0];
        c[g][1 % kApart] = t[1];
      }
    }
  }
  // The sums of token (column / COLUMNS), rows 8 * g + 4 * (quarter & 1) + 0..3, in every lane.
  template <int COLUMNS>
  __device__ __forceinline__ f32x4 total(int g) const {
    const int lane = __lane_id();
    f32x4 v = c[g][0];
    if constexpr (kApart == 2) v = pick(c[g][0], c[g][1]);
    const bool mine = (lane >> 1 & 1) == lane >> 5;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f = mine ? v[i] : 0.f;
      f += bits_as<float>(lane_xor<1>(bits_as<unsigned>(f)));
      f += bits_as<float>(lane_xor<2>(bits_as<unsigned>(f)));
      if constexpr (COLUMNS == 8) f += bits_as<float>(lane_xor<4>(bits_as<unsigned>(f)));
      v[i] = f + bits_as<float>(lane_xor<32>(bits_as<unsigned>(f)));
    }
    return v;
  }
};

// Sums of whole columns, a token each.
template <class W, class X>
__device__ __forceinline__ void add_whole(const Rows<W>& r, const u32x4 (&cols)[4], f32x4& acc) {
  f32x4 c = __is_same(W, E4m3) ? f32x4{0, 0, 0, 0} : acc;
#pragma unroll
  for (int f = 0; f < 4; ++f) c = Frag<X>::mfma(operand<X, W>(r.at(f), f & 1), cols[f], c);
  if constexpr (__is_same(W, E4m3)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(r.s, c[i], acc[i]);
    settled(acc);
  } else {
    acc = c;
  }
}
template <class W>
__device__ __forceinline__ void add_whole_split(const Rows<W>& r, const u32x4 (&cols)[8],
                                                f32x4& acc) {
  f32x4 c = __is_same(W, E4m3) ? f32x4{0, 0, 0, 0} : acc;
#pragma unroll
  for (int f = 0; f < 4; ++f) c = mfma_split<W>(r.at(f), f & 1, cols[f], cols[4 + f], c);
  if constexpr (__is_same(W, E4m3)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = fmaf(r.s, c[i], acc[i]);
    settled(acc);
  } else {
    acc = c;
  }
}

// n units through D stages, D loads ahead of the computing. The loop's loads are unconditional,
// so that the wait before each unit leaves the later ones in flight.
template <int D, class Load, class Compute>
__device__ __forceinline__ void pipeline(int n, Load&& load, Compute&& compute) {
  if (n <= 0) return;
  each<D>([&](auto d) EC_INLINE { load(d, min((int)d, n - 1)); });
  int i = 0;
  for (; i + 2 * D <= n; i += D) {
    each<D>([&](auto d) EC_INLINE {
      compute(d, i + d);
      load(d, i + D + d);
    });
  }
  each<D>([&](auto d) EC_INLINE {
    if (i + d < n) compute(d, i + d);
    if (i + D + d < n) load(d, i + D + d);
  });
  each<D>([&](auto d) EC_INLINE {
    if (i + D + d < n) compute(d, i + D + d);
  });
}

// Bytes from row `row0` of a matrix to row `row`, or to its last one.
template <class W>
__device__ __forceinline__ unsigned row_bytes(int row, int row0, int rows, int K) {
  return (unsigned)(min(row, rows - 1) - row0) * (unsigned)(K * sizeof(W));
}

// Where along k a workgroup starts: rows whose length is a multiple of a few KB put the same k
// of all rows on the same few memory channels, and workgroups that start alike stay together.
__device__ __forceinline__ int first_unit(unsigned seed, int units) {
  return (int)((seed * 2654435761u >> 8) % (unsigned)units);
}
__device__ __forceinline__ int wrap(int u, int units) { return u < units ? u : u - units; }

// Gate and up projection of 16 rows of one expert, SiLU product and routing weight. Bound by the
// weights' bytes where a call has many: one token on 2 bf16 experts, 470 MB here, takes 68.8 us
// (6.8 TB/s; a bare read of as much gets 6.6); by latency where it has few: 8 int8 experts of
// 2048 x 768, 25 MB, take 9.0 us, a bare read 4.9. Two units ahead / one: 14.1 / 14.7 us for that
// whole call, 8 fp8 experts of 44 MB 64 / 67; 1024 pairs of 2048 x 256 111 / 106.
template <class X, class W, bool ONCE, int WAVES, int D>
__global__ __launch_bounds__(WAVES* kWave) void experts_up_k(ExpertsArgs a) {
  static_assert(WAVES * kWave >= 256);
  __shared__ Pairs list;
  __shared__ __attribute__((aligned(16))) union {
    float packed[WAVES][2][4][kTile];  // token, row
    float whole[WAVES][2][4][kWave];
  } red;
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (a.few && blockIdx.y == 0)
    for (int i = blockIdx.x * WAVES * kWave + threadIdx.x; i < a.down_groups;
         i += gridDim.x * WAVES * kWave)
      a.arrived[i] = 0;
  int slot;
  const int count = list_pairs(a, blockIdx.y, slot, list);
  if (count == 0) {
    if (a.few && blockIdx.x == 0 && threadIdx.x == 0) a.meta[blockIdx.y].count = 0;
    return;
  }
  const int row0 = blockIdx.x * kTile;
  const W* gate = static_cast<const W*>(a.w13) + ((long long)slot * 2 * a.I + row0) * a.H;
  const W* up = gate + (long long)a.I * a.H;
  const float *gscale = nullptr, *uscale = nullptr;
  if constexpr (__is_same(W, E4m3)) {
    const int kb = (a.H + kUnit - 1) / kUnit, rb = (2 * a.I + kUnit - 1) / kUnit;
    const float* s13 = a.s13 + (long long)slot * rb * kb;
    gscale = s13 + (long long)(row0 / kUnit) * kb;
    uscale = s13 + (long long)((a.I + row0) / kUnit) * kb;
  }
  const int row = row0 + (threadIdx.x & 15), col = threadIdx.x >> 4;
  float sg = 1.f, su = 1.f;
  if constexpr (__is_same(W, int8_t)) {
    const float* s13 = a.s13 + (long long)slot * 2 * a.I + min(row, a.I - 1);
    sg = s13[0];
    su = s13[a.I];
  }
  lds_sync();
  if (a.few && blockIdx.x == 0 && 2 * threadIdx.x < count) {
    const int i = 2 * threadIdx.x;
    ExpertsMeta& m = a.meta[blockIdx.y];
    m.pairs[threadIdx.x] = list.pair[i] | (i + 1 < count ? list.pair[i + 1] : 0xFFFFu) << 16;
    if (i == 0) {
      m.slot = slot;
      m.count = count;
    }
  }
  const int units = (a.H + kUnit - 1) / kUnit, mine = (units - wave + WAVES - 1) / WAVES;
  const int start = first_unit(blockIdx.y * gridDim.x + blockIdx.x, units);
  const auto unit = [&](int i) EC_INLINE { return wrap(wave + i * WAVES + start, units); };
  const auto store = [&](int c, float vg, float vu) EC_INLINE {
    const long long at = (long long)list.pair[c] * a.I + row;
    Bf16 h, l;
    split_f32(silu(vg * sg) * (vu * su) * list.weight[c], h, l);
    a.hi[at] = h;
    a.lo[at] = l;
  };
  if (count <= 4) {
    using P = Packed<W, 2>;
    const int token = list.pair[min(column >> 2, count - 1)] / a.k;
    const unsigned short* x = static_cast<const unsigned short*>(a.x) + token * a.x_stride;
    const unsigned rows[2] = {row_bytes<W>(row0 + (column & 7), row0, a.I, a.H),
                              row_bytes<W>(row0 + 8 + (column & 7), row0, a.I, a.H)};
    P g[D], u[D];
    PackedSum<W, 2> pg, pu;
    pg.clear();
    pu.clear();
    pipeline<D>(
        mine,
        [&](auto d, int i) EC_INLINE {
          const int at = unit(i);
          g[d].template load<ONCE>(gate, rows, gscale, at, a.H);
          u[d].template load<ONCE>(up, rows, uscale, at, a.H);
          g[d].load_cols(x, at, a.H);
        },
        [&](auto d, int i) EC_INLINE {
          const int at = unit(i);
          u[d].b = g[d].b;
          if ((at + 1) * kUnit > a.H) {
            g[d].cut(at, a.H);
            u[d].cut(at, a.H);
          }
          pg.template add<X>(g[d]);
          pu.template add<X>(u[d]);
        });
    products_done();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f32x4 vg = pg.template total<4>(t), vu = pu.template total<4>(t);
      if ((column & 3) == 0 && quarter < 2) {
        *reinterpret_cast<f32x4*>(&red.packed[wave][0][column >> 2][t * 8 + quarter * 4]) = vg;
        *reinterpret_cast<f32x4*>(&red.packed[wave][1][column >> 2][t * 8 + quarter * 4]) = vu;
      }
    }
    lds_sync();
    if (col < count && row < a.I) {
      float vg = 0, vu = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        vg += red.packed[w][0][col][threadIdx.x & 15];
        vu += red.packed[w][1][col][threadIdx.x & 15];
      }
      store(col, vg, vu);
    }
    return;
  }
  const unsigned rows = row_bytes<W>(row0 + column, row0, a.I, a.H);
  for (int c0 = 0; c0 < count; c0 += kTile) {
    f32x4 vg = {0, 0, 0, 0}, vu = {0, 0, 0, 0};
    const int token = list.pair[min(c0 + column, count - 1)] / a.k;
    const unsigned short* x = static_cast<const unsigned short*>(a.x) + token * a.x_stride;
    Rows<W> g[1], u[1];
    u32x4 b[1][4];
    pipeline<1>(
        mine,
        [&](auto d, int i) EC_INLINE {
          const int at = unit(i);
          g[d].load(gate, rows, gscale, at, a.H, quarter);
          u[d].load(up, rows, uscale, at, a.H, quarter);
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            const int k = at * kUnit + operand_at<W>(f, quarter);
            b[d][f] = load16(x + (k < a.H ? k : 0));
          }
        },
        [&](auto d, int i) EC_INLINE {
          const int at = unit(i);
          if ((at + 1) * kUnit > a.H) {
            g[d].cut(at, a.H, quarter);
            u[d].cut(at, a.H, quarter);
#pragma unroll
            for (int f = 0; f < 4; ++f)
              b[d][f] = keep(at * kUnit + operand_at<W>(f, quarter) < a.H, b[d][f]);
          }
          add_whole<W, X>(g[d], b[d], vg);
          add_whole<W, X>(u[d], b[d], vu);
        });
    products_done();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      red.whole[wave][0][i][lane] = vg[i];
      red.whole[wave][1][i][lane] = vu[i];
    }
    lds_sync();
    if (threadIdx.x < 256 && row < a.I && c0 + col < count) {
      const int from = (threadIdx.x & 15) / 4 * 16 + col, i = threadIdx.x & 3;
      float vg = 0, vu = 0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        vg += red.whole[w][0][i][from];
        vu += red.whole[w][1][i][from];
      }
      store(c0 + col, vg, vu);
    }
    lds_sync();
  }
}

// The value of one of a workgroup's parts for the one that adds them up, and back: device scope,
// past the caches of one die. A part is in memory once its store has completed (mem_sync),
// before the workgroup counts itself in.
__device__ __forceinline__ void store_part(float* p, float v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_part(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Counts the workgroup in after its stores; whether it is the last of `all`.
__device__ __forceinline__ bool arrive(int* counter, int all, int* flag) {
  mem_sync();
  if (threadIdx.x == 0)
    *flag = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
            all - 1;
  lds_sync();
  return *flag;
}

// A few tokens: 8 * G rows of the result. The step's experts lie one after another, once for every
// two of their tokens; the workgroups of the rows and their waves take a run of the units each,
// and a wave that comes to another expert adds what it has of the last one to the sums of that
// one's tokens. The last workgroup of the rows to arrive adds up the parts, in order. 2 bf16
// experts, 235 MB here, take 36.8 us (6.4 TB/s), 8 int8 experts, 12.6 MB, 5.3 us (a bare read
// 3.0-3.7). Three units ahead / two: 4 tokens on fp8 experts of 2048 x 768 31.8 / 33.4 us a call,
// one token on experts of 1024 x 512 13.0 / 12.6.
template <class X, class W, bool ONCE, int G, int WAVES, int D>
__global__ __launch_bounds__(WAVES* kWave) void experts_down_k(ExpertsArgs a) {
  constexpr int kRows = 8 * G;
  static_assert(WAVES * kWave >= kFewTokens * kRows);
  __shared__ int slots[kExpertsMaxPairs];
  __shared__ unsigned pairs[kExpertsMaxPairs];  // two, the second 0xFFFF where there is one
  __shared__ __attribute__((aligned(16))) float sums[WAVES][kFewTokens][kRows];  // token, row
  __shared__ int last;
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row0 = blockIdx.x * kRows;
  const int all = a.by_slot ? a.S : a.n;
  int live = 0;
  for (int base = 0; base < all; base += kWave) {
    const u32x4* m = reinterpret_cast<const u32x4*>(a.meta + min(base + lane, all - 1));
    const u32x4 head = m[0], mid = m[1], tail = m[2];
    const unsigned two[kFewTokens / 2] = {head[2], head[3], mid[0],  mid[1],
                                          mid[2],  mid[3],  tail[0], tail[1]};
    const int twos = base + lane < all ? (int)(head[1] + 1) / 2 : 0;
    const int upto = wave_incl_scan(twos);
    if (wave == 0) {
#pragma unroll
      for (int i = 0; i < kFewTokens / 2; ++i)
        if (i < twos) {
          slots[live + upto - twos + i] = (int)head[0];
          pairs[live + upto - twos + i] = two[i];
        }
    }
    live += __builtin_amdgcn_readlane(upto, 63);
  }
  for (int i = lane; i < kFewTokens * kRows; i += kWave) sums[wave][i / kRows][i % kRows] = 0.f;
  lds_sync();

  const int units = (a.I + kUnit - 1) / kUnit, total = live * units;
  const int share = blockIdx.y * WAVES + wave, shares = a.splits * WAVES;
  const int first = (int)((long long)total * share / shares);
  const int end = (int)((long long)total * (share + 1) / shares);
  const int rb = (a.H + kUnit - 1) / kUnit;

  if (first < end) {
    Packed<W, G> w[D];
    // the next unit to load: expert and unit within it, and where this lane reads both
    int le = first / units, lu = first - le * units, left = end - first;
    const W* base = nullptr;
    unsigned rows[G];
#pragma unroll
    for (int g = 0; g < G; ++g)
      rows[g] = row_bytes<W>(row0 + g * 8 + (column & 7), row0, a.H, a.I);
    const float* scale = nullptr;
    const Bf16* cols = nullptr;
    const int start = first_unit(blockIdx.x, units);  // of every share of the rows' units
    const auto enter = [&](int e) EC_INLINE {
      const int slot = __builtin_amdgcn_readfirstlane(slots[e]);
      base = static_cast<const W*>(a.w2) + ((long long)slot * a.H + row0) * a.I;
      // columns 0-7 are the first token's, 8-15 the second's, or the first's again
      const unsigned p = pairs[e];
      const unsigned pair = column < 8 || p >> 16 == 0xFFFFu ? p & 0xFFFFu : p >> 16;
      cols = (column & 4 ? a.lo : a.hi) + (long long)pair * a.I;
      if constexpr (__is_same(W, E4m3))
        scale = a.s2 + ((long long)slot * rb + row0 / kUnit) * units;
    };
    enter(le);
    int ce = le, cu = lu;  // the unit to compute
    PackedSum<W, G> acc;
    acc.clear();
    pipeline<D>(
        end - first,
        [&](auto d, int) EC_INLINE {
          const int at = wrap(lu + start, units);
          w[d].template load<ONCE>(base, rows, scale, at, a.I);
          w[d].load_cols(cols, at, a.I);
          if (--left > 0 && ++lu == units) {
            lu = 0;
            enter(++le);
          }
        },
        [&](auto d, int i) EC_INLINE {
          const int at = wrap(cu + start, units);
          if ((at + 1) * kUnit > a.I) w[d].cut(at, a.I);
          acc.template add<Bf16>(w[d]);
          if (++cu == units || i + 1 == end - first) {
            const unsigned p = pairs[ce], pair = column == 0 ? p & 0xFFFFu : p >> 16;
            const bool here = (column & 7) == 0 && quarter < 2 && pair != 0xFFFFu;
            products_done();
#pragma unroll
            for (int g = 0; g < G; ++g) {
              f32x4 v = acc.template total<8>(g);
              if constexpr (__is_same(W, int8_t)) {
                const long long at = (long long)__builtin_amdgcn_readfirstlane(slots[ce]) * a.H;
                const f32x4* s2 = reinterpret_cast<const f32x4*>(a.s2 + at + row0 + g * 8);
                const f32x4 low = load_uniform(s2), high = load_uniform(s2 + 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] *= quarter & 1 ? high[i] : low[i];
              }
              if (here)
                *reinterpret_cast<f32x4*>(&sums[wave][pair / a.k][g * 8 + quarter * 4]) += v;
            }
            acc.clear();
            cu = 0;
            ++ce;
          }
        });
  }
  lds_sync();
  const int t = threadIdx.x / kRows, r = row0 + threadIdx.x % kRows;
  const bool one = t < kFewTokens && r < a.H && t * a.k < a.n;
  float y = 0;
  if (one) {
#pragma unroll
    for (int w = 0; w < WAVES; ++w) y += sums[w][t][threadIdx.x % kRows];
  }
  if (a.splits > 1) {
    float* part = a.part + (long long)blockIdx.x * a.splits * kFewTokens * kRows + threadIdx.x;
    if (one) store_part(part + blockIdx.y * kFewTokens * kRows, y);
    if (!arrive(a.arrived + blockIdx.x, a.splits, &last)) return;
    y = 0;
    if (one)
      for (int s = 0; s < a.splits; ++s) y += load_part(part + s * kFewTokens * kRows);
  }
  if (one) static_cast<X*>(a.out)[t * a.out_stride + r] = from_f32<X>(y);
}

// More tokens: down projection of one expert for its pairs, 16 * TILES rows a wave, which share
// what it loads of the columns. a.k_waves of the waves split the length of the same rows. At least
// two workgroups a compute unit (168 to 254 registers): held to three the compiler spills (32
// tokens, top-8 of 128, 2048 x 768 bf16 211 us, not 181). 16 tokens on fp8 experts of 44 MB: 800 MB
// here in 143 us (5.6 TB/s), bound by the latency of the one unit that a wave has under way.
template <class W, bool ONCE, int WAVES, int TILES, int D>
__global__ __launch_bounds__(WAVES* kWave, 2) void experts_pairs_k(ExpertsArgs a) {
  constexpr int kThreads = WAVES * kWave, kRows = TILES * kTile;  // rows of a wave
  __shared__ Pairs list;
  __shared__ __attribute__((aligned(16))) union {
    float packed[WAVES][2][kRows];  // token, row
    float whole[WAVES][TILES][4][kWave];
  } red;
  const int lane = __lane_id(), quarter = lane >> 4, column = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  int slot;
  const int count = list_pairs(a, blockIdx.y, slot, list);
  const int k_wave = wave % a.k_waves, group = wave / a.k_waves;
  const int all_rows = WAVES / a.k_waves * kRows;
  const int first_row = blockIdx.x * all_rows;
  const int row0 = min(first_row + group * kRows, (a.H - 1) / kRows * kRows);
  const int units = (a.I + kUnit - 1) / kUnit;
  const int mine = (units - k_wave + a.k_waves - 1) / a.k_waves;
  lds_sync();
  if (count > 0) {
    const W* base = static_cast<const W*>(a.w2) + ((long long)slot * a.H + row0) * a.I;
    const float* scale = nullptr;
    if constexpr (__is_same(W, E4m3)) {
      static_assert(kUnit % kRows == 0);  // one block of scales for all of the rows
      const int rb = (a.H + kUnit - 1) / kUnit;
      scale = a.s2 + ((long long)slot * rb + row0 / kUnit) * units;
    }
    const int start = first_unit(blockIdx.y * gridDim.x + blockIdx.x, units);
    const auto unit = [&](int i) EC_INLINE { return wrap(k_wave + i * a.k_waves + start, units); };
    const bool packed = count <= 2;
    for (int c0 = 0; c0 < count; c0 += kTile) {
      if (packed) {
        const Bf16* cols = (column & 4 ? a.lo : a.hi) +
                           (long long)list.pair[min(column >> 3, count - 1)] * a.I;
        unsigned rows[TILES][2];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
          for (int g = 0; g < 2; ++g)
            rows[t][g] = row_bytes<W>(row0 + t * kTile + g * 8 + (column & 7), row0, a.H, a.I);
        Packed<W, 2> w[D][TILES];
        PackedSum<W, 2> acc[TILES];
        each<TILES>([&](auto t) EC_INLINE { acc[t].clear(); });
        pipeline<D>(
            mine,
            [&](auto d, int i) EC_INLINE {
              const int u = unit(i);
              each<TILES>([&](auto t) EC_INLINE {
                w[d][t].template load<ONCE>(base, rows[t], scale, u, a.I);
              });
              w[d][0].load_cols(cols, u, a.I);
            },
            [&](auto d, int i) EC_INLINE {
              const int u = unit(i);
              each<TILES>([&](auto t) EC_INLINE { w[d][t].b = w[d][0].b; });
              // (all cuts before the first sum, so that no branch is between two tiles' sums)
              if ((u + 1) * kUnit > a.I)
                each<TILES>([&](auto t) EC_INLINE { w[d][t].cut(u, a.I); });
              each<TILES>([&](auto t) EC_INLINE { acc[t].template add<Bf16>(w[d][t]); });
            });
        products_done();
        each<TILES>([&](auto t) EC_INLINE {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const f32x4 v = acc[t].template total<8>(g);
            if ((column & 7) == 0 && quarter < 2)
              *reinterpret_cast<f32x4*>(
                  &red.packed[wave][column >> 3][t * kTile + g * 8 + quarter * 4]) = v;
          }
        });
      } else {
        f32x4 v[TILES];
        unsigned rows[TILES];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          rows[t] = row_bytes<W>(row0 + t * kTile + column, row0, a.H, a.I);
        Rows<W> w[1][TILES];
        const long long at = (long long)list.pair[min(c0 + column, count - 1)] * a.I;
        u32x4 b[1][8];
        each<TILES>([&](auto t) EC_INLINE { v[t] = f32x4{0, 0, 0, 0}; });
        pipeline<1>(
            mine,
            [&](auto d, int i) EC_INLINE {
              const int u = unit(i);
              each<TILES>([&](auto t) EC_INLINE {
                w[d][t].load(base, rows[t], scale, u, a.I, quarter);
              });
#pragma unroll
              for (int f = 0; f < 4; ++f) {
                const int k = u * kUnit + operand_at<W>(f, quarter);
                b[d][f] = load16(a.hi + at + (k < a.I ? k : 0));
                b[d][4 + f] = load16(a.lo + at + (k < a.I ? k : 0));
              }
            },
            [&](auto d, int i) EC_INLINE {
              const int u = unit(i);
              if ((u + 1) * kUnit > a.I) {
                each<TILES>([&](auto t) EC_INLINE { w[d][t].cut(u, a.I, quarter); });
#pragma unroll
                for (int f = 0; f < 8; ++f)
                  b[d][f] = keep(u * kUnit + operand_at<W>(f & 3, quarter) < a.I, b[d][f]);
              }
              each<TILES>([&](auto t) EC_INLINE { add_whole_split<W>(w[d][t], b[d], v[t]); });
            });
        products_done();
        each<TILES>([&](auto t) EC_INLINE {
#pragma unroll
          for (int i = 0; i < 4; ++i) red.whole[wave][t][i][lane] = v[t][i];
        });
      }
      lds_sync();
      const int here = min(count - c0, kTile);
      for (int j = threadIdx.x; j < all_rows * here; j += kThreads) {
        const int r = j % all_rows, col = j / all_rows, row = first_row + r;
        if (row >= a.H) continue;
        const int wave0 = r / kRows * a.k_waves, tile = r % kRows / kTile;
        const int from = r % kTile / 4 * 16 + col;
        float y = 0;
        for (int w = wave0; w < wave0 + a.k_waves; ++w)
          y += packed ? red.packed[w][col & 1][r % kRows]
                      : red.whole[w][tile][r & 3][from];
        if constexpr (__is_same(W, int8_t)) y *= a.s2[(long long)slot * a.H + row];
        a.part[(long long)list.pair[c0 + col] * a.H + row] = y;
      }
      lds_sync();
    }
  }
}

// A token's pairs added up in order; tokens without any become zero. 16 tokens of top-8, H 7168:
// 4.1 us, mostly its launch.
template <class X>
__global__ __launch_bounds__(256) void experts_sum_k(ExpertsArgs a) {
  const int t = blockIdx.y, lane = __lane_id();
  const int at = t * a.k + min(lane, a.k - 1);
  const int id = load_id(a.ids, at, a.wide, a.S);
  unsigned long long used = ballot(lane < a.k && id >= 0 && a.probs[at] != 0.f);
  for (unsigned long long r = used; r; r &= r - 1) {  // a slot's first pair has the rest of it
    const int j = __builtin_ctzll(r);
    const unsigned long long same = ballot(id == __builtin_amdgcn_readlane(id, j)) & used;
    used &= ~(same & (same - 1));
    r &= used;
  }
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
