// Products in 8-bit integers on gfx950: expert_cache_quantize, expert_cache_linear8,
// expert_cache_moe8.
//
// y[t, o] = scale[t] * wscale[o] * sum_k q[t, k] w[o, k]. Sums of 8-bit products are exact in 32
// bits up to a length of 131071, in any order, so no order has to be kept for results to repeat.
// Weights are the first operand of v_mfma_i32_16x16x64_i8: a lane holds of the weights row
// (lane & 15) and of the tokens column (lane & 15), 16 bytes each at its quarter of 64 along k;
// of the product it holds column (lane & 15), rows 4 * (lane >> 4) + 0..3: four neighbouring
// outputs of one token.
//
// Tiles of TM tokens and TN outputs go through LDS in steps of 128 bytes along k, straight from
// memory (buffer loads to LDS), later steps' under way while one is computed. A wave's load is
// 8 rows of 128 bytes; chunk c (16 bytes) of row r lies at place c ^ (r & 7), so that the lanes of
// a 16-row operand read from all banks. Loads past an array's end are the buffer descriptor's to
// answer with zeros: rows behind the last, and what is behind a row's end in the last step.
//
// What bounds them (sizes as tokens, length x outputs). 4096 of 14336 x 4096, a tile of 256 x 256 for
// every compute unit, takes 174 to 195 us by the card's clock, 2.5 to 2.8 POP/s; a step of such a tile
// is 2048 clocks of matrix instructions and as many of LDS (192 KB of operands and 64 KB of loads at
// 128 bytes a clock) and takes 2700, at the 1.9 GHz to which the card goes under such loads. Each tile
// has about 10 us besides: its first loads, and 128 KB of results, which all compute units store at the
// same time. So 4096 of 4096 x 14336 takes 215 to 230 us, 2.1 POP/s. A workgroup for several tiles that
// loads the next one's first steps before it stores was no faster (247 us for four tiles each of 4096
// of 4096 x 16384, where a workgroup for each takes 229), and steps of 64 bytes and stores past the
// caches weren't either.
#pragma once
#include "mfma.h"
#include "sort.h"
#include "wave.h"

namespace ec {

using i32x4 = __attribute__((ext_vector_type(4))) int;
using f32x2 = __attribute__((ext_vector_type(2))) float;

constexpr unsigned kFarOffset = 0x78000000u;  // behind the end of every descriptor
constexpr unsigned kMaxRange = 0x70000000u;
constexpr int kMaxLength8 = 131056;        // 16 K at most: sums stay below 2^31

// ---- rows to 8 bits -------------------------------------------------------------------------

struct QuantizeArgs {
  const void* x;
  long long x_stride;    // elements
  int rows, H;
  const int* live;       // rows that there are, if fewer than `rows`
  int8_t* q;
  long long q_stride;
  float* scales;
};

constexpr int kQuantizeThreads = 256;  // of a workgroup

// q = rint(127 x / m), m the row's largest magnitude. Rows below 2^-119 count as zeros; one with an
// infinity or NaN gets a scale of NaN and zeros, so that whatever it is multiplied with shows it.
// 16-bit values are often half way between two whole numbers (m / 2 is 63.5). With v = 127 x / m,
// x = a 2^p and m = b 2^q (a, b whole and at most 2047), v is half way or at least v / (254 max(a,
// b)) > 2^-19 v away from that, since 2 v times b, or b 2^(q-p), is whole. v in 32 bits as
// x * (127 / m) is within 2 units of its last place, so it is rounded to 8 of them first: what is
// half way gets there, and nothing else does.
template <class X>
struct Quantizer {
  float inverse, scale;
  bool zero;
  __device__ __forceinline__ explicit Quantizer(unsigned largest) {
    const float m = bits_as<float>(largest);
    const bool finite = largest < 0x7F800000u;
    zero = !finite || m < 0x1p-119f;
    inverse = 127.f / (zero ? 1.f : m);
    scale = finite ? (m < 0x1p-119f ? 0.f : m / 127.f) : __builtin_nanf("");
  }
  __device__ __forceinline__ unsigned of(float x) const {
    float p = x * inverse;
    if constexpr (sizeof(X) == 2) p = bits_as<float>((bits_as<unsigned>(p) + 4) & ~7u);
    return zero ? 0u : (unsigned)(int)__builtin_rintf(p) & 0xFFu;
  }
};

// A row for every THREADS of a workgroup of GROUPS as many, all of which come here; KEPT pieces a thread
// stay in registers between the maximum and the rounding.
template <int THREADS, int GROUPS, int KEPT, class X>
__device__ __forceinline__ void quantize_row(const QuantizeArgs& a, int row) {
  constexpr int kN = Piece<X>::kN, kKept = KEPT, kStride = THREADS * kN;
  const int thread = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
  const bool in = row < a.rows;
  const X* const x = static_cast<const X*>(a.x) + (in ? row : 0) * a.x_stride;
  Piece<X> kept[kKept];
  unsigned largest = 0;
  const int first = thread * kN;
  const auto look = [&](const Piece<X>& r) {
#pragma unroll
    for (int j = 0; j < kN; ++j)
      largest = max(largest, bits_as<unsigned>(to_f32(r.v[j])) & 0x7FFFFFFFu);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    const int h = first + i * kStride;
    kept[i] = h < a.H ? load_piece(x + h, a.H - h) : Piece<X>{};
  }
#pragma unroll
  for (int i = 0; i < kKept; ++i) look(kept[i]);
  for (int h = first + kKept * kStride; h < a.H; h += kStride) look(load_piece(x + h, a.H - h));
  largest = ~wave_min_u32(~largest);
  constexpr int kWaves = THREADS / kWave;
  if constexpr (kWaves > 1) {
    __shared__ unsigned of_wave[GROUPS][kWaves];
    if (__lane_id() == 0) of_wave[group][thread / kWave] = largest;
    lds_sync();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) largest = max(largest, of_wave[group][w]);
  }
  if (!in) return;
  const Quantizer<X> quantizer(largest);
  int8_t* const q = a.q + (long long)row * a.q_stride;
  const int padded = (a.H + 15) & ~15;
  const auto write = [&](int h, const Piece<X>& r) {
    unsigned packed[kN / 4] = {};
#pragma unroll
    for (int j = 0; j < kN; ++j) packed[j / 4] |= quantizer.of(to_f32(r.v[j])) << 8 * (j % 4);
    __builtin_memcpy(q + h, packed, kN);
  };
#pragma unroll
  for (int i = 0; i < kKept; ++i)
    if (first + i * kStride < padded) write(first + i * kStride, kept[i]);
  for (int h = first + kKept * kStride; h < padded; h += kStride)
    write(h, h < a.H ? load_piece(x + h, a.H - h) : Piece<X>{});
  if (thread == 0) a.scales[row] = quantizer.scale;
}

template <int THREADS, int KEPT, class X>
__global__ __launch_bounds__(kQuantizeThreads) void quantize_k(QuantizeArgs a) {
  constexpr int kRows = kQuantizeThreads / THREADS;
  if (a.live != nullptr) a.rows = min(a.rows, load_uniform(a.live));
  if ((int)blockIdx.x * kRows >= a.rows) return;
  quantize_row<THREADS, kRows, KEPT, X>(a, blockIdx.x * kRows + threadIdx.x / THREADS);
}

// What a layer begins with, in one launch: the pairs sorted (up to 1024 R) or their keys counted, by
// the first workgroups, and the tokens quantised by the others, four rows each.
template <int R, class X, bool MANY>
__global__ __launch_bounds__(1024) void begin8_k(SortArgs s, int sorting, QuantizeArgs q) {
  if ((int)blockIdx.x >= sorting)
    quantize_row<256, 4, 2, X>(q, (blockIdx.x - sorting) * 4 + threadIdx.x / 256);
  else if constexpr (MANY)
    sort_count(s);
  else
    sort_place<16, R, false>(s);
}

constexpr int kDieUnits = 32;  // compute units of a die

// ---- tiles ----------------------------------------------------------------------------------

// A dense product; sums of a part of its length as they are; an expert's gate and up projections with
// the product of both; its down projection.
enum class Form { kDense, kPart, kGateUp, kDown };

struct Product8Args {
  const int8_t* a;       // tokens [rows, K], a_stride bytes apart
  const int8_t* w;       // weights [S or 1][N, K], w_stride bytes apart
  const float* a_scale;  // a row
  const float* w_scale;  // an output
  const float* bias;
  long long a_stride, w_stride, a_bytes, slab_bytes;
  int rows, N, K;        // of dense products: rows; of Experts8's: pairs
  int splits;            // of the length, with Form::kPart
  int out_tiles;         // tiles along N
  // Experts8: tiles of the sorted rows
  const int4* tiles;     // slot, first row, end
  const int* n_tiles;
  const int* pairs;      // the pair at every sorted row; its token is pair / k
  int k;
  void* out;
  long long out_stride;  // elements
  int scale_rows;        // of a_scale
  bool whole_stores;     // results can be stored 16 bytes at a time
};

constexpr int kStepBytes = 128;  // of a row in a step: two products' lengths

__device__ __forceinline__ void load_word_to_lds(__amdgpu_buffer_rsrc_t from, char* to,
                                                 unsigned offset) {
  using Lds = __attribute__((address_space(3))) void*;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Lds)to, 4, offset, 0, 0, 0);
}

template <class X>
__device__ __forceinline__ unsigned two_of(float a, float b) {
  using V = typename Frag<X>::V;
  using Two = __attribute__((ext_vector_type(2))) __typeof__(V{}[0] + V{}[0]);
  return bits_as<unsigned>(__builtin_convertvector(f32x2{a, b}, Two));
}

// Four words of every lane, its row of 16 lanes q has words 0..3 of its own: afterwards it has word q
// of rows 0..3.
__device__ __forceinline__ void exchange_quads(unsigned& w0, unsigned& w1, unsigned& w2,
                                               unsigned& w3) {
  const auto a = __builtin_amdgcn_permlane32_swap(w0, w2, false, false);
  const auto b = __builtin_amdgcn_permlane32_swap(w1, w3, false, false);
  const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  w0 = c[0];
  w1 = c[1];
  w2 = d[0];
  w3 = d[1];
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t range_of(const void* p, long long bytes) {
  const unsigned n = bytes < (long long)kMaxRange ? (unsigned)bytes : kMaxRange;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00027000);
}

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, char* to, unsigned offset,
                                            int step) {
  using Lds = __attribute__((address_space(3))) void*;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Lds)to, 16, offset, step, 0, 0);
}

// Waits until at most LEFT of the wave's loads and stores are under way (they finish in order) and
// its reads of LDS are done, then for the workgroup's other waves.
template <int LEFT>
__device__ __forceinline__ void landed() {
  static_assert(LEFT < 64);
  __builtin_amdgcn_s_waitcnt((LEFT & 15) | (LEFT >> 4) << 14 | 7 << 4);
  lds_sync();
}

// A workgroup takes a tile of up to TM tokens and TN outputs. Waves form WM x WN; wave row wm has the
// 16-token operands wm, wm + WM, ..., so that a tile with fewer tokens (MI rounds of WM operands, at
// most TM / 16 / WM) gives every wave less to do. A gate-up tile's weights are TN / 2 rows of the gate
// and the same of the up projection, so that a lane holds both of a hidden value. Hidden values and an
// expert's outputs go on in 32 bits: rounding hidden values to bf16 before they are quantised would
// move about one in forty to the neighbouring whole number (2^-9 of a value, of up to 127 steps). SiLU's
// exponential is the instruction's, off by up to (2 |gate| + 4) 2^-24 of itself: a hidden value that is
// nearer than 32-bit arithmetic to half way between two whole numbers may go to either, which moves
// results of 2048 tokens by 1.0e-4 to 1.6e-4 of their size from another 32-bit form's, both 0.0017 off
// the formula in 64 bits by their rounding to bf16. The library's own exponential takes 1 to 2 % longer:
// 2048 tokens, 2 of 8 slots of 4096 x 14336, 917 us and 903.
template <int TM, int TN, int WM, int WN, int ST, Form FORM, class OUT>
struct Product8 {
  static constexpr int kWaves = WM * WN;
  static constexpr int kMost = TM / WM / 16;                      // rounds
  static constexpr int kA = (TM / 8 + kWaves - 1) / kWaves;       // loads a wave and step
  static constexpr int kB = (TN / 8 + kWaves - 1) / kWaves;
  static constexpr int kN = TN / WN / 16;                         // operands a wave
  static constexpr bool kGated = FORM == Form::kGateUp, kGrouped = kGated || FORM == Form::kDown;
  static constexpr int kOut = kGated ? kN / 2 : kN;               // of them with a result
  static constexpr int kScaleLoads = TN / kWave + (TM + kWave - 1) / kWave;  // 64 scales each
  // A stage holds a step of a tile of MI rounds. Tiles of fewer rounds take more stages, as many as
  // there is room for: they have less to do while loads are under way.
  static constexpr int stage_bytes(int mi) { return (mi * WM * 16 + TN) * kStepBytes; }
  static constexpr int kRoom = TM + TN == 512 ? 155648 : ST * stage_bytes(kMost);
  static constexpr int stages(int mi) {
    const int n = kRoom / stage_bytes(mi);
    return mi == kMost ? ST : n > 4 ? 4 : n;
  }
  // behind them the scales of the tile's outputs and of its tokens
  static constexpr int kLds = kRoom + kScaleLoads * 256;
  static constexpr bool kCut = kMost >= 4;
  static_assert(kN * WN * 16 == TN && kMost * WM * 16 == TM && TN % 8 == 0 && kLds <= 163840);
  static_assert(ST >= 2 && ST * stage_bytes(kMost) <= kRoom);
  static_assert(TM % 32 == 0 && TN % kWave == 0);

  const Product8Args& a;
  char* const lds;
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN, col = lane & 15, quad = lane >> 4;
  const int chunk = (lane & 7) ^ (lane >> 3);
  const int steps = (a.K + kStepBytes - 1) / kStepBytes;
  const int width = kGated ? a.N / 2 : a.N;

  struct Tile {
    int slot, m0, m_end, n0;
    __device__ __forceinline__ int rounds() const {
      return (m_end - m0 + WM * 16 - 1) / (WM * 16);
    }
  };
  unsigned a_at[kA], b_at[kB];  // a lane's bytes from a tile's first

  __device__ __forceinline__ Product8(const Product8Args& args, char* to) : a(args), lds(to) {
#pragma unroll
    for (int i = 0; i < kA; ++i)
      a_at[i] = (unsigned)(((i * kWaves + wave) * 8 + (lane >> 3)) * a.a_stride) + 16 * chunk;
#pragma unroll
    for (int i = 0; i < kB; ++i) {
      const int r = (i * kWaves + wave) * 8 + (lane >> 3);
      b_at[i] = (unsigned)((kGated && r >= TN / 2 ? width + r - TN / 2 : r) * a.w_stride) +
                16 * chunk;
    }
  }

  __device__ __forceinline__ int a_row(int i) const { return (i * WM + wm) * 16; }
  __device__ __forceinline__ int b_row(int j) const {
    if constexpr (kGated)
      return (j < kOut ? 0 : TN / 2) + wn * kOut * 16 + (j % kOut) * 16;
    else
      return wn * kN * 16 + j * 16;
  }

  // A tile, or its part `part` of 2^cut.
  __device__ __forceinline__ Tile tile_of(int m_tile, int n_tile, int part, int cut) const {
    Tile t = {0, m_tile * TM, a.rows, n_tile * (kGated ? TN / 2 : TN)};
    if constexpr (kGrouped) {
      const u32x4 of = load_uniform(reinterpret_cast<const u32x4*>(a.tiles) + m_tile);
      t.slot = (int)of[0];
      t.m0 = (int)of[1];
      t.m_end = (int)of[2];
    }
    t.m_end = min(t.m_end, t.m0 + TM);
    if (cut) {
      t.m0 += part * (TM >> cut);
      t.m_end = max(t.m0, min(t.m_end, t.m0 + (TM >> cut)));
    }
    return t;
  }
  // The token of a row of the tile; that of its last row for those behind it.
  __device__ __forceinline__ int token(const Tile& t, int r) const {
    const int m = max(0, min(t.m0 + r, t.m_end - 1));
    return kGated ? a.pairs[m] / a.k : m;
  }

  template <int MI>
  __device__ __forceinline__ void load(const Tile& t, int step) const {
    char* const to = lds + step % stages(MI) * stage_bytes(MI);
    // all rows of MI rounds, though the tile may have fewer: a wave's loads are counted
    constexpr int kRows = MI * WM * 16;
    // the step's own offset is added behind the descriptor's check, so what is behind a row's end is
    // sent behind the array's
    const bool behind = step * kStepBytes + 16 * chunk >= a.K;
    const long long skipped = kGated ? 0 : t.m0 * a.a_stride;
    const __amdgpu_buffer_rsrc_t a_range = range_of(a.a + skipped, max(0ll, a.a_bytes - skipped));
#pragma unroll
    for (int i = 0; i < kA; ++i)
      if ((i + 1) * kWaves * 8 <= kRows || (i * kWaves + wave) * 8 < kRows)
        load_to_lds(a_range, to + (i * kWaves + wave) * 1024, behind ? kFarOffset : a_at[i],
                    step * kStepBytes);
    const long long ahead = t.n0 * a.w_stride;
    const __amdgpu_buffer_rsrc_t b_range =
        range_of(a.w + t.slot * a.slab_bytes + ahead, max(0ll, a.slab_bytes - ahead));
#pragma unroll
    for (int i = 0; i < kB; ++i)
      if ((i + 1) * kWaves * 8 <= TN || (i * kWaves + wave) * 8 < TN)
        load_to_lds(b_range, to + MI * WM * 16 * kStepBytes + (i * kWaves + wave) * 1024,
                    behind ? kFarOffset : b_at[i], step * kStepBytes);
  }
  // A tile's scales and its first steps.
  template <int MI>
  __device__ __forceinline__ void load_first(const Tile& t) {
    if constexpr (kGated)
#pragma unroll
      for (int i = 0; i < kA; ++i)
        a_at[i] = (unsigned)(token(t, (i * kWaves + wave) * 8 + (lane >> 3)) * a.a_stride) +
                  16 * chunk;
    if constexpr (FORM != Form::kPart) {  // whose N goes to whole cells, behind the scales' end
      char* const to = lds + kRoom;
      const __amdgpu_buffer_rsrc_t w_scales =
          range_of(a.w_scale + (long long)t.slot * a.N, 4ll * a.N);
      const __amdgpu_buffer_rsrc_t a_scales = range_of(a.a_scale, 4ll * a.scale_rows);
#pragma unroll
      for (int i = 0; i < (kScaleLoads + kWaves - 1) / kWaves; ++i) {
        const int part = i * kWaves + wave, r = part * kWave + lane;
        if (part < TN / kWave) {
          const int o = t.n0 + (kGated && r >= TN / 2 ? width + r - TN / 2 : r);
          load_word_to_lds(w_scales, to + part * 256, 4 * o);
        } else if (part < kScaleLoads) {
          load_word_to_lds(a_scales, to + part * 256, 4 * token(t, r - TN));
        }
      }
    }
#pragma unroll
    for (int s = 0; s < stages(MI); ++s) load<MI>(t, s);
  }

  // The tile's product, MI rounds of it, and its results.
  template <int MI>
  __device__ __forceinline__ void run(const Tile& t) {
    struct Operands {
      i32x4 a[MI], b[kN];
    };
    constexpr int kStages = stages(MI);
    i32x4 acc[MI][kN] = {};
    const auto read = [&](Operands& o, int step, int half) {
      const char* const from = lds + step % kStages * stage_bytes(MI) + col * kStepBytes +
                               16 * ((half * 4 + quad) ^ (col & 7));
#pragma unroll
      for (int j = 0; j < kN; ++j)
        o.b[j] = *(const i32x4*)(from + (MI * WM * 16 + b_row(j)) * kStepBytes);
#pragma unroll
      for (int i = 0; i < MI; ++i) o.a[i] = *(const i32x4*)(from + a_row(i) * kStepBytes);
    };
    const auto multiply = [&](const Operands& o) {
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.b[j], o.a[i], acc[i][j], 0, 0, 0);
    };
    // Operands of a half step are read from LDS while the half before is multiplied. In the middle
    // of a step its last operands have been read and the next step's loads have landed, so that
    // behind the barrier there a later step can be loaded over it. Steps past the last load nothing,
    // but are counted.
    Operands even, odd;
    load_first<MI>(t);
    // at least so many loads a step: with as many left, all before them have landed
    constexpr int kLoads = MI * WM * 16 / 8 / kWaves + TN / 8 / kWaves;
    landed<(kStages - 1) * kLoads>();
    read(even, 0, 0);
    for (int step = 0; step < steps; ++step) {
      read(odd, step, 1);
      multiply(even);
      landed<(kStages - 2) * kLoads>();
      if (kStages > 2 || step + kStages < steps) load<MI>(t, step + kStages);
      read(even, step + 1, 0);
      multiply(odd);
    }
    landed<0>();  // LDS is the next workgroup's when this one ends
    products_done();

    const char* const scales = lds + kRoom;
    f32x4 scale[kN];
    float row_scale[MI];
#pragma unroll
    for (int j = 0; j < kN; ++j)
      scale[j] = *(const f32x4*)(scales + 4 * (b_row(j) + quad * 4));
#pragma unroll
    for (int i = 0; i < MI; ++i) row_scale[i] = *(const float*)(scales + 4 * (TN + a_row(i) + col));

    // A tile's results by a descriptor that ends behind its last row. 16-bit results of a lane, four
    // of every 16 outputs, are exchanged in the wave so that a lane has the 16 of one operand.
    constexpr bool kShort = sizeof(OUT) == 2;
    constexpr int kCells = kShort ? 8 : 4;           // results a store
    constexpr int kEach = kOut * 4 / kCells;         // stores a row
    static_assert(!kShort || kOut == 4);
    OUT* const out = static_cast<OUT*>(a.out) + t.m0 * a.out_stride;
    const long long stride = a.out_stride * (long long)sizeof(OUT);
    const __amdgpu_buffer_rsrc_t range =
        range_of(out, (t.m_end - t.m0 - 1) * stride + width * (int)sizeof(OUT));
    int o[kEach];
    unsigned at[kEach];
#pragma unroll
    for (int c = 0; c < kEach; ++c) {
      o[c] = t.n0 + (kShort ? b_row(0) + quad * 16 + c * 8 : b_row(c) + quad * 4);
      at[c] = t.m0 < t.m_end && o[c] < width
                  ? (unsigned)((wm * 16 + col) * stride) + o[c] * (unsigned)sizeof(OUT)
                  : kFarOffset;
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      u32x4 cell[kEach];
      unsigned pair[kOut][2];
#pragma unroll
      for (int j = 0; j < kOut; ++j) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (FORM == Form::kPart) {
            y[e] = bits_as<float>(acc[i][j][e]);
            continue;
          }
          y[e] = (float)acc[i][j][e] * row_scale[i] * scale[j][e];
          if constexpr (kGated) {
            const float u = (float)acc[i][j + kOut][e] * row_scale[i] * scale[j + kOut][e];
            y[e] = y[e] / (1.f + __expf(-y[e])) * u;
          }
        }
        if constexpr (FORM == Form::kDense)
          if (a.bias) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              y[e] += a.bias[min(t.n0 + b_row(j) + quad * 4 + e, width - 1)];
          }
        if constexpr (kShort) {
          pair[j][0] = two_of<OUT>(y[0], y[1]);
          pair[j][1] = two_of<OUT>(y[2], y[3]);
        } else {
          cell[j] = bits_as<u32x4>(y);
        }
      }
      if constexpr (kShort) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          exchange_quads(pair[0][h], pair[1][h], pair[2][h], pair[3][h]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          cell[c] = u32x4{pair[2 * c][0], pair[2 * c][1], pair[2 * c + 1][0], pair[2 * c + 1][1]};
      }
#pragma unroll
      for (int c = 0; c < kEach; ++c) {
        if (a.whole_stores) {
          __builtin_amdgcn_raw_buffer_store_b128(cell[c], range,
                                                 at[c] + (unsigned)(i * WM * 16 * stride), 0, 0);
        } else if (t.m0 + a_row(i) + col < t.m_end && o[c] < width) {
          store_piece(out + (a_row(i) + col) * a.out_stride + o[c], bits_as<Piece<OUT>>(cell[c]),
                      width - o[c]);
        }
      }
    }
  }
};

template <int TM, int TN, int WM, int WN, int ST, Form FORM, class OUT>
__global__ __launch_bounds__(WM* WN* kWave) void product8_k(Product8Args a) {
  using P = Product8<TM, TN, WM, WN, ST, FORM, OUT>;
  __shared__ __attribute__((aligned(1024))) char lds[P::kLds];
  // Consecutive workgroups go to the eight dies in turn: each die gets a run of tiles, so that
  // its second-level cache holds what they share. Of its last tiles, fewer than it has compute units,
  // each is cut in two or four where that many parts fit beside each other: 4096 tokens of 4096 x 14336
  // (3.5 tiles a compute unit) 223 us, uncut 240; 2048, 8 of 128 slots of 2048 x 768, 269 and 273.
  const int m_tiles = P::kGrouped ? load_uniform(a.n_tiles) : (a.rows + TM - 1) / TM;
  const int splits = FORM == Form::kPart ? a.splits : 1;
  const int n = m_tiles * a.out_tiles * splits, per = (n + 7) / 8, from = (blockIdx.x & 7) * per;
  const int here = min(per, n - from), at = blockIdx.x >> 3;
  if (here <= 0) return;
  const int whole = here / kDieUnits * kDieUnits, rest = here - whole;
  const int cut = !P::kCut ? 0 : rest * 4 <= kDieUnits ? 2 : rest * 2 <= kDieUnits ? 1 : 0;
  if (at >= whole + (rest << cut)) return;
  const bool part = at >= whole;
  int tile = from + (part ? whole + ((at - whole) >> cut) : at);
  if constexpr (FORM == Form::kPart) {
    // neighbours have the same part of the length; whole steps, as many each but for the last, which has
    // one at least, since dense_plan makes at most eight parts of eight steps or more. The bound at zero
    // below is never met; without it this compiler waits a state too few at the loop's end for sums that
    // it moves there, as the test of the built code shows.
    const int split = __builtin_amdgcn_readfirstlane(tile / (m_tiles * a.out_tiles));
    tile -= split * m_tiles * a.out_tiles;
    const int steps = (a.K + kStepBytes - 1) / kStepBytes;
    const int from_k = (steps + splits - 1) / splits * split * kStepBytes;
    a.a += from_k;
    a.w += from_k;
    a.a_bytes -= from_k;
    a.slab_bytes -= from_k;
    a.K = max(0, min(a.K - from_k, (steps + splits - 1) / splits * kStepBytes));
    a.out = static_cast<OUT*>(a.out) + (long long)split * a.rows * a.out_stride;
  }
  P p(a, lds);
  // Where a column of tiles is less than a die takes at once, it takes several side by side, so that
  // small tiles, the last of a column, come behind the large ones of all.
  const int side = min(a.out_tiles, (kDieUnits + m_tiles - 1) / m_tiles);
  const int group = __builtin_amdgcn_readfirstlane(tile / (side * m_tiles));
  const int columns = min(side, a.out_tiles - group * side);
  const int in_group = tile - group * side * m_tiles;
  const int m_tile = __builtin_amdgcn_readfirstlane(in_group / columns);
  const auto t = p.tile_of(m_tile, group * side + in_group - m_tile * columns,
                           (at - whole) & ((1 << cut) - 1), part ? cut : 0);
  // a round more than a tile needs costs no more than one that it needs: variants for all of eight
  // would double the code for a sixteenth of a tile
  const int rounds = t.rounds();
  if (rounds <= 0) return;
  if (P::kMost >= 8 && rounds > 6)
    p.template run<P::kMost < 8 ? 1 : 8>(t);
  else if (P::kMost >= 6 && rounds > 4)
    p.template run<P::kMost < 6 ? 1 : 6>(t);
  else if (P::kMost >= 4 && rounds > 2)
    p.template run<P::kMost < 4 ? 1 : 4>(t);
  else if (P::kMost >= 2 && rounds > 1)
    p.template run<P::kMost < 2 ? 1 : 2>(t);
  else
    p.template run<1>(t);
}

// Sums of parts of the length to results: four outputs a thread.
struct JoinArgs {
  const int* part;       // [splits, rows, stride]
  const float* a_scale;
  const float* w_scale;
  const float* bias;
  void* out;
  long long out_stride;
  int splits, rows, N, stride;
};
constexpr int kJoinThreads = 256;

template <class OUT>
__global__ __launch_bounds__(kJoinThreads) void join8_k(JoinArgs a) {
  const int cells = a.stride / 4;
  const long long i = (long long)blockIdx.x * kJoinThreads + threadIdx.x;
  const int m = (int)(i / cells), o = (int)(i - (long long)m * cells) * 4;
  if (m >= a.rows) return;
  i32x4 sum = {};
  for (int s = 0; s < a.splits; ++s)
    sum += *(const i32x4*)(a.part + ((long long)s * a.rows + m) * a.stride + o);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (o + e >= a.N) continue;
    float y = (float)sum[e] * a.a_scale[m] * a.w_scale[o + e];
    if (a.bias) y += a.bias[o + e];
    static_cast<OUT*>(a.out)[m * a.out_stride + o + e] = from_f32<OUT>(y);
  }
}

// ---- few tokens -----------------------------------------------------------------------------
//
// One token of 2048 x 4096 takes 4.8 us in a graph, and 10 eager, which is the time of the call in
// Python; 16 tokens take 9.2, their quantising in a launch of its own included.

// Up to 16 MI tokens: a workgroup takes 16 outputs, its waves a run of the length each, and their
// sums meet in LDS. Weights go from memory to operands and are read once, and so do tokens in 8 bits.
// Tokens of a 16-bit type X are quantised by every workgroup for itself into LDS: for a few thousand
// values a second launch costs more than reading again what all others read.
constexpr int kFewWaves = 8;
constexpr int kFewValues = 16384;  // 16-bit values that a workgroup quantises, at most
constexpr int kFewPieces = 8;      // of 8 values, a lane

// Waves that share a row of T tokens.
__host__ __device__ constexpr int few_row_waves(int T) {
  return T <= 1 ? 8 : T <= 2 ? 4 : T <= 4 ? 2 : 1;
}
__host__ __device__ constexpr int few_longest(int T) {
  return few_row_waves(T) * kFewPieces * kWave * 8;
}

template <int MI, class X, class OUT>
__global__ __launch_bounds__(kFewWaves* kWave) void few8_k(Product8Args a, const X* x,
                                                           long long x_stride, int H) {
  constexpr bool kWhole = sizeof(X) == 1;
  static_assert(kWhole || MI == 1);
  constexpr int kSums = kFewWaves * MI * kWave * 4;
  // rows 16 bytes further apart than their length: 16 of them start at other banks
  constexpr int kTokens = kWhole ? 16 : kFewValues + 16 * 32;
  __shared__ __attribute__((aligned(16))) char lds[kSums * 4 > kTokens ? kSums * 4 : kTokens];
  __shared__ unsigned of_wave[kFewWaves];
  __shared__ float token_scale[16];
  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int col = lane & 15, quad = lane >> 4, n0 = blockIdx.x * 16;
  // a wave's units of 64 along k, two at least where there are enough: whole lines
  const int units = (a.K + 63) / 64;
  int per = (units + kFewWaves - 1) / kFewWaves;
  per += per & (per > 1);
  const int first = wave * per, end = min(units, first + per);

  const int8_t* const w = a.w + min(n0 + col, a.N - 1) * a.w_stride;
  constexpr int kAhead = MI > 2 ? 2 : 4;  // units under way
  i32x4 wv[kAhead], tv[kAhead][MI];
  const auto load_weights = [&](int u) {
#pragma unroll
    for (int g = 0; g < kAhead; ++g) {
      const int k = max(0, min(u + g, end - 1)) * 64 + quad * 16;
      wv[g] = *(const i32x4*)(w + (k < a.K ? k : 0));
    }
  };
  load_weights(first);

  const int pitch = a.K + 16;
  if constexpr (!kWhole) {
    const int share = few_row_waves(a.rows), in_row = wave % share;
    // as often in every wave, also in those that have no row
    for (int from = 0; from < a.rows; from += kFewWaves / share) {
      const int row = from + wave / share;
      const X* const t = x + min(row, a.rows - 1) * x_stride;
      Piece<X> kept[kFewPieces];
      unsigned largest = 0;
#pragma unroll
      for (int p = 0; p < kFewPieces; ++p) {
        const int k = ((p * share + in_row) * kWave + lane) * 8;
        kept[p] = k < H ? load_piece(t + k, H - k) : Piece<X>{};
      }
#pragma unroll
      for (int p = 0; p < kFewPieces; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          largest = max(largest, bits_as<unsigned>(to_f32(kept[p].v[e])) & 0x7FFFFFFFu);
      largest = ~wave_min_u32(~largest);
      if (share > 1) {
        if (lane == 0) of_wave[wave] = largest;
        lds_sync();
        for (int v = 0; v < share; ++v) largest = max(largest, of_wave[wave - in_row + v]);
      }
      if (row >= a.rows) continue;
      const Quantizer<X> quantizer(largest);
      if (lane == 0 && in_row == 0) token_scale[row] = quantizer.scale;
#pragma unroll
      for (int p = 0; p < kFewPieces; ++p) {
        const int k = ((p * share + in_row) * kWave + lane) * 8;
        if (k >= a.K) continue;
        unsigned q[2] = {};
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e / 4] |= quantizer.of(to_f32(kept[p].v[e])) << 8 * (e % 4);
        *(u32x2*)(lds + row * pitch + k) = u32x2{q[0], q[1]};
      }
    }
    lds_sync();
  }
  const int8_t* t[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int row = min(i * 16 + col, a.rows - 1);
    t[i] = kWhole ? a.a + row * a.a_stride : (const int8_t*)lds + row * pitch;
  }

  i32x4 acc[MI] = {};
  for (int u = first; u < end; u += kAhead) {
#pragma unroll
    for (int g = 0; g < kAhead; ++g) {
      const int k = min(u + g, end - 1) * 64 + quad * 16;
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        tv[g][i] = *(const i32x4*)(t[i] + (k < a.K ? k : 0));
        if (u + g >= end || k >= a.K) tv[g][i] = i32x4{};
      }
    }
    if (u > first) load_weights(u);
#pragma unroll
    for (int g = 0; g < kAhead; ++g)
#pragma unroll
      for (int i = 0; i < MI; ++i)
        acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[g], tv[g][i], acc[i], 0, 0, 0);
  }
  products_done();
  if constexpr (!kWhole) lds_sync();  // the sums go where the tokens were
  int* const part = reinterpret_cast<int*>(lds);
#pragma unroll
  for (int i = 0; i < MI; ++i)
    *(i32x4*)(part + (wave * MI + i) * 256 + lane * 4) = acc[i];
  lds_sync();
  // consecutive threads have consecutive outputs of a token
  for (int i = threadIdx.x; i < MI * 256; i += kFewWaves * kWave) {
    const int o = i % 16, m = i / 16;
    const int at = (m >> 4) * 256 + ((o >> 2) * 16 + (m & 15)) * 4 + (o & 3);
    if (m >= a.rows || n0 + o >= a.N) continue;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) sum += part[v * MI * 256 + at];
    float y = (float)sum * (kWhole ? a.a_scale[m] : token_scale[m]) * a.w_scale[n0 + o];
    if (a.bias) y += a.bias[n0 + o];
    static_cast<OUT*>(a.out)[m * a.out_stride + n0 + o] = from_f32<OUT>(y);
  }
}

}  // namespace ec
