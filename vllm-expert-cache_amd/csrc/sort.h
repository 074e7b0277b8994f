// Pairs of token and slot sorted by slot and back on gfx950: expert_cache_sort,
// expert_cache_dispatch, expert_cache_combine, expert_cache_combine_grad.
//
// Sorting is a stable counting sort of n = T * k pairs by S + 1 keys, the last for pairs that have
// no slot. Waves take 64 pairs at a time. A lane finds the lanes with its key by a ballot for every
// bit of the key, so its rank among the wave's equal keys is a count of lower lanes and the wave's
// own counter in LDS: no place depends on the order of atomics. Sums of the counters over lower keys
// and earlier waves give the places. Up to 4096 pairs are one workgroup's, their keys and ranks in
// registers; more take a launch before that which counts every workgroup's keys.
//
// The rows move as they lie: `dispatch` reads a token's row once and writes it to its k places,
// `combine` reads the k rows and sums them in 32 bits in the order of j, and `combine_grad` is a
// wave for every pair, which has the pair's gradient row and its dot product from one pass.
#pragma once
#include "mfma.h"
#include "wave.h"

namespace ec {

constexpr int kSortMaxSlots = 1024;
constexpr int kSortMaxPairs = 1 << 24;
constexpr int kSortOne = 4096;      // pairs that one workgroup sorts
constexpr int kSortLot = 1024;      // pairs that a workgroup of many takes at a time
constexpr int kSortMaxBlocks = 256;
constexpr int kMoveWaves = 4;       // waves of a workgroup that moves rows

struct SortArgs {
  const void* ids;
  const float* probs;  // of Experts8: pairs of weight 0 have no slot
  int n, S, chunk;     // pairs, slots, pairs a workgroup
  bool wide;
  int* offsets;
  int* rows;
  int* places;
  int* counts;         // [blocks, S + 1]
  int2* tiles;         // of Experts8: slot and first row of every tile, and their number
  int* n_tiles;
  int tile_rows;
};

__device__ __forceinline__ int sort_key(const SortArgs& a, int i) {
  int id = load_id(a.ids, i, a.wide, a.S);
  if (a.probs != nullptr && a.probs[i] == 0.f) id = -1;
  return id < 0 ? a.S : id;
}

__global__ __launch_bounds__(1024) void sort_count_k(SortArgs a) {
  __shared__ int count[kSortMaxSlots + 1];
  for (int e = threadIdx.x; e <= a.S; e += blockDim.x) count[e] = 0;
  lds_sync();
  const int first = blockIdx.x * a.chunk, end = min(a.n, first + a.chunk);
#pragma unroll 4
  for (int i = first + threadIdx.x; i < end; i += blockDim.x) atomicAdd(&count[sort_key(a, i)], 1);
  lds_sync();
  for (int e = threadIdx.x; e <= a.S; e += blockDim.x)
    a.counts[(long long)blockIdx.x * (a.S + 1) + e] = count[e];
}

// Sum of v over lower threads of a workgroup of W waves, and over all of them; `word` is W ints.
template <int W>
__device__ __forceinline__ int before_me(int v, int* word, int& all) {
  const int wave = threadIdx.x / kWave, scan = wave_incl_scan(v);
  lds_sync();  // word's last use
  if (__lane_id() == kWave - 1) word[wave] = scan;
  lds_sync();
  int before;
  wave_sums<W>(word, wave, before, all);
  return before + scan - v;
}

// W waves take R x 64 W pairs at a time, wave w the w-th R x 64 of them. A pair's place is its key's
// first place, plus the key's pairs in earlier lots, in earlier waves, in this wave's earlier
// groups of 64, and in lower lanes.
template <int W, int R, bool MANY>
__global__ __launch_bounds__(W* kWave) void sort_place_k(SortArgs a) {
  constexpr int kThreads = W * kWave, kLot = kThreads * R, kKeys = kSortMaxSlots + 1;
  constexpr int kPer = (kSortMaxSlots + kThreads - 1) / kThreads;  // keys a thread
  __shared__ int start[kKeys], of_wave[W * kKeys], word[W];
  const int keys = a.S + 1, wave = threadIdx.x / kWave, lane = __lane_id();
  const int lo = blockIdx.x * a.chunk, hi = min(a.n, lo + a.chunk);
  const int bits = 32 - __builtin_clz(a.S);
  volatile int* const mine = of_wave + wave * keys;
  int key[R], rank[R];
  const auto take = [&](int lot) {  // keys of this wave's groups, and their ranks in the wave
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = lot + (wave * R + r) * kWave + lane;
      key[r] = i < hi ? sort_key(a, i) : -1;
    }
    for (int e = lane; e < keys; e += kWave) mine[e] = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned long long same = wave_match(key[r], bits);
      if (key[r] >= 0) {
        rank[r] = mine[key[r]] + __popcll(same & lanes_below());
        __builtin_amdgcn_wave_barrier();
        // the last of the equal ones counts them all
        if ((same >> lane) == 1) mine[key[r]] = rank[r] + 1;
      }
      __builtin_amdgcn_wave_barrier();
    }
  };
  // of_wave to the key's pairs in earlier waves; the key's sum
  const auto add_waves = [&](int e) {
    int c[W], sum = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) c[w] = of_wave[w * keys + e];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      of_wave[w * keys + e] = sum;
      sum += c[w];
    }
    return sum;
  };

  take(lo);
  lds_sync();
  // thread t has keys t * kPer and on, the last one also that of pairs without a slot; `own` are
  // a lot's pairs, `all` those of all workgroups, `first` those of lower keys of the thread and
  // of earlier workgroups
  int own[kPer], all[kPer], first[kPer], sum = 0, own_none = 0, none = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = threadIdx.x * kPer + j;
    own[j] = all[j] = first[j] = 0;
    if (e < a.S) {
      own[j] = all[j] = add_waves(e);
      if constexpr (MANY) {
        all[j] = 0;
#pragma unroll 8
        for (int b = 0; b < (int)gridDim.x; ++b) {
          const int c = a.counts[(long long)b * keys + e];
          first[j] += b < (int)blockIdx.x ? c : 0;
          all[j] += c;
        }
      }
    }
    first[j] += sum;
    sum += all[j];
  }
  const bool last = threadIdx.x == kThreads - 1;
  if (last) {
    own_none = add_waves(a.S);
    if constexpr (MANY) {
#pragma unroll 8
      for (int b = 0; b < (int)blockIdx.x; ++b) none += a.counts[(long long)b * keys + a.S];
    }
  }
  int live;
  const int ahead = before_me<W>(sum, word, live);
#pragma unroll
  for (int j = 0; j < kPer; ++j)
    if (threadIdx.x * kPer + j < a.S) start[threadIdx.x * kPer + j] = ahead + first[j];
  if (last) start[a.S] = live + none;
  if (blockIdx.x == 0) {
    int tiles = 0, n_tiles;
#pragma unroll
    for (int j = 0, at = ahead; j < kPer; at += all[j++]) {
      if (threadIdx.x * kPer + j < a.S) a.offsets[threadIdx.x * kPer + j] = at;
      if (a.tiles) tiles += (all[j] + a.tile_rows - 1) / a.tile_rows;
    }
    if (last) a.offsets[a.S] = live;
    if (a.tiles) {
      int t = before_me<W>(tiles, word, n_tiles);
#pragma unroll
      for (int j = 0, at = ahead; j < kPer; at += all[j++])
        for (int row = 0; row < all[j]; row += a.tile_rows)
          a.tiles[t++] = make_int2(threadIdx.x * kPer + j, at + row);
      if (last) *a.n_tiles = n_tiles;
    }
  }
  for (int lot = lo;;) {
    lds_sync();
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (key[r] < 0) continue;
      const int i = lot + (wave * R + r) * kWave + lane;
      const int p = start[key[r]] + mine[key[r]] + rank[r];
      const bool has = key[r] < a.S;
      a.rows[p] = has ? i : -1;
      a.places[i] = has ? p : -1;
    }
    lot += kLot;
    if (!MANY || lot >= hi) break;
    lds_sync();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (threadIdx.x * kPer + j < a.S) start[threadIdx.x * kPer + j] += own[j];
    if (last) start[a.S] += own_none;
    take(lot);
    lds_sync();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (threadIdx.x * kPer + j < a.S) own[j] = add_waves(threadIdx.x * kPer + j);
    if (last) own_none = add_waves(a.S);
  }
}

// ---- rows ---------------------------------------------------------------------------------

// 16 bytes of elements of type X from an address that is aligned to X; where fewer than 16 bytes
// are left of a row, those alone.
template <class X>
struct Piece {
  static constexpr int kN = 16 / sizeof(X);
  X v[kN];
};

template <class X>
__device__ __forceinline__ Piece<X> load_piece(const X* p, long long left) {
  Piece<X> r{};
  if (left >= Piece<X>::kN) {
    __builtin_memcpy(&r, p, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<X>::kN; ++i)
      if (i < left) r.v[i] = p[i];
  }
  return r;
}
template <class X>
__device__ __forceinline__ void store_piece(X* p, const Piece<X>& r, long long left) {
  if (left >= Piece<X>::kN) {
    __builtin_memcpy(p, &r, 16);
  } else {
#pragma unroll
    for (int i = 0; i < Piece<X>::kN; ++i)
      if (i < left) p[i] = r.v[i];
  }
}

template <>
__device__ __forceinline__ float from_f32<float>(float f) {
  return f;
}

struct MoveArgs {
  const void* x;        // rows that are read
  const void* y;        // of combine_grad: the rows that were combined
  const float* weights;
  const int* places;
  const int* offsets;
  void* out;
  float* dweights;
  long long x_stride, y_stride, out_stride;  // elements
  int T, k, S, H, n, chunks;                 // n = T * k; chunks a row
};

// Rows of the same address pattern: out[p] = x[token] at the token's k places, zeros behind the
// last place. A wave takes 4 KB of a token's row.
template <class X>
__global__ __launch_bounds__(kMoveWaves* kWave) void dispatch_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN, kPieces = 4;
  const long long w = (long long)blockIdx.x * kMoveWaves + threadIdx.x / kWave;
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.chunks));
  if (t >= a.T) return;
  const int first = (int)(w - (long long)t * a.chunks) * (kPieces * kWave * kN) +
                    (int)__lane_id() * kN;
  const X* const x = static_cast<const X*>(a.x) + t * a.x_stride;
  Piece<X> r[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int h = first + i * kWave * kN;
    if (h < a.H) r[i] = load_piece(x + h, a.H - h);
  }
  const auto put = [&](int p) {
    X* const to = static_cast<X*>(a.out) + (long long)p * a.out_stride;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int h = first + i * kWave * kN;
      if (h < a.H) store_piece(to + h, r[i], a.H - h);
    }
  };
  for (int j = 0; j < a.k; ++j) {
    const int p = a.places[(long long)t * a.k + j];
    if ((unsigned)p < (unsigned)a.n) put(p);
  }
  const int live = a.offsets[a.S];
  if (live >= a.n || live < 0) return;
#pragma unroll
  for (int i = 0; i < kPieces; ++i) r[i] = Piece<X>{};
  for (int p = live + t; p < a.n; p += a.T) put(p);
}

// out[t] = sum_j weights[t, j] x[places[t, j]]: a wave takes 1 KB of a token's row.
template <class X, class OUT = X>
__global__ __launch_bounds__(kMoveWaves* kWave) void combine_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN;
  const long long w = (long long)blockIdx.x * kMoveWaves + threadIdx.x / kWave;
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.chunks));
  if (t >= a.T) return;
  const int h = (int)(w - (long long)t * a.chunks) * (kWave * kN) + (int)__lane_id() * kN;
  float sum[kN] = {};
  for (int j = 0; j < a.k; ++j) {
    const long long pair = (long long)t * a.k + j;
    const int p = a.places[pair];
    const float weight = a.weights ? a.weights[pair] : 1.f;
    if ((unsigned)p >= (unsigned)a.n || weight == 0.f || h >= a.H) continue;
    const Piece<X> r =
        load_piece(static_cast<const X*>(a.x) + (long long)p * a.x_stride + h, a.H - h);
#pragma unroll
    for (int i = 0; i < kN; ++i) sum[i] = fmaf(weight, to_f32(r.v[i]), sum[i]);
  }
  if (h >= a.H) return;
  OUT* const to = static_cast<OUT*>(a.out) + t * a.out_stride + h;
  struct {
    OUT v[kN];
  } o;
#pragma unroll
  for (int i = 0; i < kN; ++i) o.v[i] = from_f32<OUT>(sum[i]);
  if (h + kN <= a.H) {
    __builtin_memcpy(to, &o, sizeof o);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (h + i < a.H) to[i] = o.v[i];
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// For every pair (t, j): out[p] = weights[t, j] x[t] (x is the gradient of combine's result) and
// dweights[t, j] = <x[t], y[p]>, p its place. Rows behind the last place become zeros.
template <class X>
__global__ __launch_bounds__(kMoveWaves* kWave) void combine_grad_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN;
  const int pair =
      __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kMoveWaves + threadIdx.x / kWave));
  if (pair >= a.n) return;
  const int p = a.places[pair];
  const bool live = (unsigned)p < (unsigned)a.n;
  const float weight = a.weights ? a.weights[pair] : 1.f;
  const X* const g = static_cast<const X*>(a.x) + (long long)(pair / a.k) * a.x_stride;
  float dot = 0.f;
  if (live) {
    const X* const y = static_cast<const X*>(a.y) + (long long)p * a.y_stride;
    X* const to = static_cast<X*>(a.out) + (long long)p * a.out_stride;
    for (int h = (int)__lane_id() * kN; h < a.H; h += kWave * kN) {
      const Piece<X> r = load_piece(g + h, a.H - h);
      if (a.dweights) {
        const Piece<X> v = load_piece(y + h, a.H - h);
#pragma unroll
        for (int i = 0; i < kN; ++i) dot = fmaf(to_f32(r.v[i]), to_f32(v.v[i]), dot);
      }
      if (a.out) {
        Piece<X> o;
#pragma unroll
        for (int i = 0; i < kN; ++i) o.v[i] = from_f32<X>(weight * to_f32(r.v[i]));
        store_piece(to + h, o, a.H - h);
      }
    }
  }
  if (a.dweights) {
    dot = wave_sum(dot);
    if (__lane_id() == 0) a.dweights[pair] = live ? dot : 0.f;
  }
  const int behind = a.offsets[a.S];
  if (a.out && behind >= 0 && pair < a.n - behind) {
    X* const to = static_cast<X*>(a.out) + (long long)(behind + pair) * a.out_stride;
    for (int h = (int)__lane_id() * kN; h < a.H; h += kWave * kN)
      store_piece(to + h, Piece<X>{}, a.H - h);
  }
}

}  // namespace ec
