// Pairs of token and slot sorted by slot and back on gfx950: expert_cache_sort,
// expert_cache_dispatch, expert_cache_combine, expert_cache_combine_grad.
//
// Sorting is a stable counting sort of n = T * k pairs by S + 1 keys, the last for pairs that have
// no slot. Waves take 64 pairs at a time. A lane finds the lanes with its key by a ballot for every
// bit of the key, so its rank among the wave's equal keys is a count of lower lanes and the wave's
// own counter in LDS: no place depends on the order of atomics. Sums of the counters over lower keys
// and earlier waves give the places. Up to 4096 pairs are one workgroup's, their keys and ranks in
// registers; more take a launch before that which counts every workgroup's keys. 8 pairs take 3.0 us of
// kernel, 1551 5.0, 32768 of 128 slots 2.8 and 5.5: a chain of loads, barriers and ballots, not bytes.
//
// The rows move as they lie: `dispatch` reads a token's row once and writes it to its k places,
// `combine` reads the k rows and sums them in 32 bits in the order of j, and `combine_grad` is a wave
// for every pair, which has the pair's gradient row and its dot product from one pass.
#pragma once
#include "mfma.h"
#include "wave.h"

namespace ec {

constexpr int kSortMaxSlots = 1024;
constexpr int kSortMaxPairs = 1 << 24;
constexpr int kSortOne = 4096;      // pairs that one workgroup sorts
constexpr int kSortLot = 1024;      // pairs that a workgroup of many takes at a time
// Workgroups at most, since each reads the counts of all: 2^20 pairs of 128 slots take 26 us, with up to
// 128 of them 27 and with 512 35; 2^24 pairs 164, 294 and 134.
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
  int4* tiles;         // of Experts8: slot, first row and end of every tile, and their number
  int* n_tiles;
  int tile_rows;
};

__device__ __forceinline__ int sort_key(const SortArgs& a, int i) {
  int id = load_id(a.ids, i, a.wide, a.S);
  if (a.probs != nullptr && a.probs[i] == 0.f) id = -1;
  return id < 0 ? a.S : id;
}

// The keys of a workgroup's pairs counted.
__device__ __forceinline__ void sort_count(const SortArgs& a) {
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
__device__ __forceinline__ void sort_place(const SortArgs& a) {
  constexpr int kThreads = W * kWave, kLot = kThreads * R, kKeys = kSortMaxSlots + 1;
  constexpr int kPer = (kSortMaxSlots + kThreads - 1) / kThreads;  // keys a thread
  __shared__ int start[kKeys], of_wave[W * kKeys], word[W];
  const int keys = a.S + 1, wave = threadIdx.x / kWave, lane = __lane_id();
  const int blocks = MANY ? (a.n - 1) / a.chunk + 1 : 1;
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
        for (int b = 0; b < blocks; ++b) {
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
#pragma unroll
    for (int j = 0, at = ahead; j < kPer; at += all[j++]) {
      if (threadIdx.x * kPer + j < a.S) a.offsets[threadIdx.x * kPer + j] = at;
    }
    if (last) a.offsets[a.S] = live;
    if (a.tiles) {
      // Slot by slot: with tiles of half their rows or fewer behind all others 2048 tokens, 2 of 8 slots
      // of 4096 x 14336, took 900 us and not 891, and 4096, 4 of 16 of 2048 x 4096, 592 and not 582.
      int tile = 0, tiles;
#pragma unroll
      for (int j = 0; j < kPer; ++j) tile += (all[j] + a.tile_rows - 1) / a.tile_rows;
      tile = before_me<W>(tile, word, tiles);
#pragma unroll
      for (int j = 0, at = ahead; j < kPer; at += all[j++])
        for (int row = 0; row < all[j]; row += a.tile_rows)
          a.tiles[tile++] =
              make_int4(threadIdx.x * kPer + j, at + row, at + min(all[j], row + a.tile_rows), 0);
      if (last) *a.n_tiles = tiles;
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

__global__ __launch_bounds__(1024) void sort_count_k(SortArgs a) { sort_count(a); }

template <int W, int R, bool MANY>
__global__ __launch_bounds__(W* kWave) void sort_place_k(SortArgs a) {
  sort_place<W, R, MANY>(a);
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
  const int* rows;
  void* out;
  float* dweights;
  long long x_stride, y_stride, out_stride;  // elements
  int T, k, H, n, chunks;                    // n = T * k; chunks a row
};

constexpr int kMovePieces = 4;  // a lane and row

// How rows are loaded and stored: as whole, aligned pieces of 16 bytes, past the caches where they
// would not stay there anyway; as pieces at any element, the last of a row moved forward to its end;
// element by element (rows shorter than a piece).
enum class Move { kWhole, kOnce, kAnywhere, kElements };

// Where a lane's piece begins that would begin at h, and how many of its elements are the piece's
// before it.
template <class X, Move MOVE>
struct Place {
  int h, skip;
  bool in;
  __device__ __forceinline__ Place(int at, int H) : h(at), skip(0), in(at < H) {
    if (MOVE == Move::kAnywhere && at > H - Piece<X>::kN) {
      h = H - Piece<X>::kN;
      skip = at - h;
    }
  }
};

template <Move MOVE, class X>
__device__ __forceinline__ Piece<X> get(const X* row, int h, int H) {
  using Loose = u32x4 __attribute__((aligned(sizeof(X))));
  if constexpr (MOVE == Move::kElements) return load_piece(row + h, H - h);
  if constexpr (MOVE == Move::kAnywhere)
    return bits_as<Piece<X>>((u32x4) * reinterpret_cast<const Loose*>(row + h));
  return bits_as<Piece<X>>(load16_of<MOVE == Move::kOnce>(row + h));
}
template <Move MOVE, class X>
__device__ __forceinline__ void put(X* row, int h, int H, const Piece<X>& r) {
  using Loose = u32x4 __attribute__((aligned(sizeof(X))));
  const u32x4 v = bits_as<u32x4>(r);
  if constexpr (MOVE == Move::kElements) {
    store_piece(row + h, r, H - h);
  } else if constexpr (MOVE == Move::kAnywhere) {
    *reinterpret_cast<Loose*>(row + h) = v;
  } else if constexpr (MOVE == Move::kOnce) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(row + h));
  } else {
    *reinterpret_cast<u32x4*>(row + h) = v;
  }
}

// Zeros in row p: from a wave's lanes, `from` on.
template <class X, Move MOVE>
__device__ __forceinline__ void clear_row(const MoveArgs& a, int p, int from) {
#pragma unroll
  for (int i = 0; i < kMovePieces; ++i) {
    const Place<X, MOVE> at(from + i * kWave * Piece<X>::kN, a.H);
    if (at.in) put<MOVE>(static_cast<X*>(a.out) + (long long)p * a.out_stride, at.h, a.H, Piece<X>{});
  }
}

// out[places[t, j]] = x[t], and zeros in rows without a pair. A wave takes 4 KB of a token's row, reads
// it once and writes it to its k places, and looks after the rows t k to t k + k - 1 if they have no
// pair. Front to back over the rows, 134 MB of them took 38 us and not 28.
template <class X, Move MOVE>
__global__ __launch_bounds__(kMoveWaves* kWave) void dispatch_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN;
  const long long w = (long long)blockIdx.x * kMoveWaves + threadIdx.x / kWave;
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.chunks)), lane = __lane_id();
  if (t >= a.T) return;
  const int first = (int)(w - (long long)t * a.chunks) * (kMovePieces * kWave * kN) + lane * kN;
  const X* const x = static_cast<const X*>(a.x) + t * a.x_stride;
  const long long pair = (long long)t * a.k + min(lane, a.k - 1);
  const int place = a.places[pair], row = a.rows[pair];
  Piece<X> r[kMovePieces];
#pragma unroll
  for (int i = 0; i < kMovePieces; ++i) {
    const Place<X, MOVE> at(first + i * kWave * kN, a.H);
    if (at.in) r[i] = get<MOVE == Move::kOnce ? Move::kWhole : MOVE>(x, at.h, a.H);
  }
  for (unsigned long long left = ballot(lane < a.k && (unsigned)place < (unsigned)a.n); left;
       left &= left - 1) {
    const int p = __builtin_amdgcn_readlane(place, __builtin_ctzll(left));
    X* const to = static_cast<X*>(a.out) + (long long)p * a.out_stride;
#pragma unroll
    for (int i = 0; i < kMovePieces; ++i) {
      const Place<X, MOVE> at(first + i * kWave * kN, a.H);
      if (at.in) put<MOVE>(to, at.h, a.H, r[i]);
    }
  }
  for (unsigned long long left = ballot(lane < a.k && (unsigned)row >= (unsigned)a.n); left;
       left &= left - 1)
    clear_row<X, MOVE>(a, t * a.k + __builtin_ctzll(left), first);
}

// out[t] = sum_j weights[t, j] x[places[t, j]], in the order of j: a wave takes 1 KB of a token's
// row. Lane j looks up pair j, so that the rows' loads wait for one load and not for one each, and
// eight of them are under way. 8192 tokens of 8 rows of 2048 bf16 take 50 us, 6.0 TB/s.
template <class X, Move MOVE, class OUT = X>
__global__ __launch_bounds__(kMoveWaves* kWave) void combine_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN, kAhead = 8;
  const long long w = (long long)blockIdx.x * kMoveWaves + threadIdx.x / kWave;
  const int t = __builtin_amdgcn_readfirstlane((int)(w / a.chunks)), lane = __lane_id();
  if (t >= a.T) return;
  const Place<X, MOVE> at((int)(w - (long long)t * a.chunks) * (kWave * kN) + lane * kN, a.H);
  const long long pair = (long long)t * a.k + min(lane, a.k - 1);
  const int place = a.places[pair];
  const float weight = a.weights ? a.weights[pair] : 1.f;
  unsigned long long left =
      ballot(lane < a.k && (unsigned)place < (unsigned)a.n && weight != 0.f);
  // lanes behind a row's end stay, since their places and weights are read, and load its first piece
  const int h = at.in ? at.h : 0;
  float sum[kN] = {};
  while (left) {
    Piece<X> r[kAhead];
    float f[kAhead];
    int taken = 0;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (left == 0) break;
      const int j = __builtin_ctzll(left);
      left &= left - 1;
      const int p = __builtin_amdgcn_readlane(place, j);
      f[u] = bits_as<float>(__builtin_amdgcn_readlane(bits_as<int>(weight), j));
      r[u] = get<MOVE>(static_cast<const X*>(a.x) + (long long)p * a.x_stride, h, a.H);
      ++taken;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (u < taken)
#pragma unroll
        for (int i = 0; i < kN; ++i) sum[i] = fmaf(f[u], to_f32(r[u].v[i]), sum[i]);
  }
  if (!at.in) return;
  OUT* const to = static_cast<OUT*>(a.out) + t * a.out_stride + at.h;
  struct Results {
    OUT v[kN];
  } o;
#pragma unroll
  for (int i = 0; i < kN; ++i) o.v[i] = from_f32<OUT>(sum[i]);
  if constexpr (MOVE == Move::kElements) {
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (at.h + i < a.H) to[i] = o.v[i];
  } else if constexpr (sizeof(OUT) == sizeof(X)) {
    put<MOVE == Move::kOnce ? Move::kWhole : MOVE>(to - at.h, at.h, a.H, bits_as<Piece<OUT>>(o));
  } else {
    __builtin_memcpy(to, &o, sizeof o);  // Experts8's rows, of any place
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// For the pair (t, j) at place p: out[p] = weights[t, j] x[t] (x is the gradient of combine's result)
// and dweights[t, j] = <x[t], y[p]>. A wave a pair, neighbours sharing x's row; it also clears the row
// of its own number if that has no pair. 65536 pairs of 2048 bf16 values 109 us, 5.2 TB/s; by places
// and through the caches a sixth more.
template <class X, Move MOVE>
__global__ __launch_bounds__(kMoveWaves* kWave) void combine_grad_k(MoveArgs a) {
  constexpr int kN = Piece<X>::kN, kStep = kMovePieces * kWave * kN;
  const int pair =
      __builtin_amdgcn_readfirstlane((int)(blockIdx.x * kMoveWaves + threadIdx.x / kWave));
  if (pair >= a.n) return;
  const int p = load_uniform(a.places + pair), row = load_uniform(a.rows + pair);
  const float weight = a.weights ? load_uniform(a.weights + pair) : 1.f;
  const int lane_at = (int)__lane_id() * kN;
  float dot = 0.f;
  if ((unsigned)p < (unsigned)a.n) {
    const X* const g = static_cast<const X*>(a.x) + (long long)(pair / a.k) * a.x_stride;
    const X* const y = static_cast<const X*>(a.y) + (long long)p * a.y_stride;
    X* const to = static_cast<X*>(a.out) + (long long)p * a.out_stride;
    for (int from = lane_at; from < a.H; from += kStep) {
      Piece<X> r[kMovePieces], v[kMovePieces];
#pragma unroll
      for (int i = 0; i < kMovePieces; ++i) {
        const Place<X, MOVE> at(from + i * kWave * kN, a.H);
        if (!at.in) continue;
        if (a.dweights) v[i] = get<MOVE>(y, at.h, a.H);
        r[i] = get<MOVE == Move::kOnce ? Move::kWhole : MOVE>(g, at.h, a.H);
      }
#pragma unroll
      for (int i = 0; i < kMovePieces; ++i) {
        const Place<X, MOVE> at(from + i * kWave * kN, a.H);
        if (!at.in) continue;
        Piece<X> o;
#pragma unroll
        for (int e = 0; e < kN; ++e) {
          const float x = to_f32(r[i].v[e]);
          if (a.dweights && (MOVE != Move::kAnywhere || e >= at.skip))
            dot = fmaf(x, to_f32(v[i].v[e]), dot);
          o.v[e] = from_f32<X>(weight * x);
        }
        if (a.out) put<MOVE>(to, at.h, a.H, o);
      }
    }
  }
  if (a.dweights) {
    dot = wave_sum(dot);
    if (__lane_id() == 0) a.dweights[pair] = dot;
  }
  if (a.out && (unsigned)row >= (unsigned)a.n)
    for (int from = lane_at; from < a.H; from += kStep) clear_row<X, MOVE>(a, pair, from);
}

}  // namespace ec
