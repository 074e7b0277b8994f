// Pairs of token and slot sorted by slot and back on gfx950: expert_cache_sort,
// expert_cache_dispatch, expert_cache_combine, expert_cache_combine_grad.
//
// Sorting is a stable counting sort of n = T * k pairs by S + 1 keys, the last for pairs that have
// no slot. A workgroup cuts its pairs into one run a wave, counts each run's keys in LDS, and from
// the sums over lower keys and earlier runs every wave then knows where its first pair of every key
// goes. Within 64 pairs a lane's place is the number of equal keys in lower lanes (ballots), so no
// place depends on the order of atomics. Many pairs take two launches: the workgroups' counts, then
// the same with the counts of earlier workgroups added.
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
constexpr int kSortOne = 16384;     // pairs that one workgroup sorts
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
  for (int i = first + threadIdx.x; i < end; i += blockDim.x) atomicAdd(&count[sort_key(a, i)], 1);
  lds_sync();
  for (int e = threadIdx.x; e <= a.S; e += blockDim.x)
    a.counts[(long long)blockIdx.x * (a.S + 1) + e] = count[e];
}

// Exclusive prefix sums of v[0..m) in place by the first wave; v[m] becomes the sum.
__device__ __forceinline__ void sort_scan(int* v, int m) {
  if (threadIdx.x < kWave) {
    const int lane = threadIdx.x, per = (m + kWave - 1) / kWave;
    const int lo = min(m, lane * per), hi = min(m, lo + per);
    int sum = 0;
    for (int i = lo; i < hi; ++i) sum += v[i];
    int at = wave_incl_scan(sum) - sum;
    for (int i = lo; i < hi; ++i) {
      const int c = v[i];
      v[i] = at;
      at += c;
    }
    if (lane == kWave - 1) v[m] = at;
  }
}

template <bool MANY>
__global__ __launch_bounds__(1024) void sort_place_k(SortArgs a) {
  extern __shared__ int sort_lds[];
  const int keys = a.S + 1, waves = blockDim.x / kWave;
  int* const start = sort_lds;              // [keys + 1] first place of every key
  int* const tile = start + keys + 1;       // [keys] tiles before every key's
  int* const of_wave = tile + keys;         // [waves, keys]
  for (int i = threadIdx.x; i < waves * keys; i += blockDim.x) of_wave[i] = 0;
  lds_sync();
  const int wave = threadIdx.x / kWave;
  const int lo = blockIdx.x * a.chunk, hi = min(a.n, lo + a.chunk);
  const int run = ((hi - lo + waves - 1) / waves + kWave - 1) / kWave * kWave;
  const int first = min(hi, lo + wave * run), end = min(hi, first + run);
  int* const mine = of_wave + wave * keys;
  for (int i = first + (int)__lane_id(); i < end; i += kWave) atomicAdd(&mine[sort_key(a, i)], 1);
  lds_sync();
  // every wave's counts to those of the waves before it, from what earlier workgroups have
  for (int e = threadIdx.x; e < keys; e += blockDim.x) {
    int before = 0, all = 0;
    if constexpr (MANY) {
#pragma unroll 8
      for (int b = 0; b < (int)gridDim.x; ++b) {
        const int c = a.counts[(long long)b * keys + e];
        before += b < (int)blockIdx.x ? c : 0;
        all += c;
      }
    }
    for (int w = 0; w < waves; ++w) {
      const int c = of_wave[w * keys + e];
      of_wave[w * keys + e] = before;
      before += c;
    }
    start[e] = MANY ? all : before;
    tile[e] = a.tiles && e < a.S ? (start[e] + a.tile_rows - 1) / a.tile_rows : 0;
  }
  lds_sync();
  sort_scan(start, keys);
  lds_sync();
  if (blockIdx.x == 0) {
    for (int e = threadIdx.x; e < keys; e += blockDim.x) a.offsets[e] = start[e];
    if (a.tiles) {
      sort_scan(tile, a.S);  // tile[S] is the last key's, whose own is 0
      lds_sync();
      const int n = tile[a.S];
      for (int t = threadIdx.x; t < n; t += blockDim.x) {
        int e = 0, top = a.S - 1;  // the last slot whose tiles begin at or before t
        while (e < top) {
          const int mid = (e + top + 1) / 2;
          if (tile[mid] <= t) e = mid;
          else top = mid - 1;
        }
        a.tiles[t] = make_int2(e, start[e] + (t - tile[e]) * a.tile_rows);
      }
      if (threadIdx.x == 0) *a.n_tiles = n;
    }
  }
  const int bits = 32 - __builtin_clz(a.S);
  volatile int* const at = mine;
  for (int base = first; base < end; base += kWave) {
    const int i = base + (int)__lane_id();
    const int key = i < end ? sort_key(a, i) : -1;
    const unsigned long long same = wave_match(key, bits);
    if (key >= 0) {
      const int rank = __popcll(same & lanes_below());
      const int in_key = at[key] + rank, p = start[key] + in_key;
      __builtin_amdgcn_wave_barrier();
      // the last of the equal ones counts them all
      if ((same >> __lane_id()) == 1) at[key] = in_key + 1;
      a.rows[p] = key < a.S ? i : -1;
      a.places[i] = key < a.S ? p : -1;
    }
    __builtin_amdgcn_wave_barrier();
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
  Piece<X> r;
  if (left >= Piece<X>::kN) {
    __builtin_memcpy(&r, p, 16);
  } else {
    r = Piece<X>{};
    for (int i = 0; i < left; ++i) r.v[i] = p[i];
  }
  return r;
}
template <class X>
__device__ __forceinline__ void store_piece(X* p, const Piece<X>& r, long long left) {
  if (left >= Piece<X>::kN) {
    __builtin_memcpy(p, &r, 16);
  } else {
    for (int i = 0; i < left; ++i) p[i] = r.v[i];
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
    for (int i = 0; i < a.H - h; ++i) to[i] = o.v[i];
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
