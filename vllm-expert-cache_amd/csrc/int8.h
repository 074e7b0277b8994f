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
// memory (buffer loads to LDS), the next step's under way while one is computed. A wave's load is
// 8 rows of 128 bytes; chunk c (16 bytes) of row r lies at place c ^ (r & 7), so that the lanes of
// a 16-row operand read from all banks. Loads past an array's end are the buffer descriptor's to
// answer with zeros: rows behind the last, and what is behind a row's end in the last step.
#pragma once
#include "mfma.h"
#include "sort.h"
#include "wave.h"

namespace ec {

using i32x4 = __attribute__((ext_vector_type(4))) int;
using f32x2 = __attribute__((ext_vector_type(2))) float;

constexpr int kStepBytes = 128;            // of a row in a step
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

constexpr int kQuantizeThreads = 256;

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

// A row a workgroup; what fits stays in registers between the maximum and the rounding.
template <class X>
__global__ __launch_bounds__(kQuantizeThreads) void quantize_k(QuantizeArgs a) {
  constexpr int kN = Piece<X>::kN, kKept = 4, kStride = kQuantizeThreads * kN;
  const int row = blockIdx.x;
  if (a.live != nullptr && row >= *a.live) return;
  const X* const x = static_cast<const X*>(a.x) + (long long)row * a.x_stride;
  Piece<X> kept[kKept];
  unsigned largest = 0;
  const int first = threadIdx.x * kN;
  for (int i = 0, h = first; h < a.H; ++i, h += kStride) {
    const Piece<X> r = load_piece(x + h, a.H - h);
#pragma unroll
    for (int j = 0; j < kN; ++j)
      largest = max(largest, bits_as<unsigned>(to_f32(r.v[j])) & 0x7FFFFFFFu);
    if (i < kKept) {
#pragma unroll
      for (int m = 0; m < kKept; ++m)
        if (m == i) kept[m] = r;
    }
  }
  largest = ~wave_min_u32(~largest);
  __shared__ unsigned of_wave[kQuantizeThreads / kWave];
  if (__lane_id() == 0) of_wave[threadIdx.x / kWave] = largest;
  lds_sync();
#pragma unroll
  for (int w = 0; w < kQuantizeThreads / kWave; ++w) largest = max(largest, of_wave[w]);
  const Quantizer<X> quantizer(largest);
  int8_t* const q = a.q + (long long)row * a.q_stride;
  const int padded = (a.H + 15) & ~15;
  for (int i = 0, h = first; h < padded; ++i, h += kStride) {
    Piece<X> r{};
    if (i < kKept) {
#pragma unroll
      for (int m = 0; m < kKept; ++m)
        if (m == i && h < a.H) r = kept[m];
    } else if (h < a.H) {
      r = load_piece(x + h, a.H - h);
    }
    unsigned packed[kN / 4] = {};
#pragma unroll
    for (int j = 0; j < kN; ++j) packed[j / 4] |= quantizer.of(to_f32(r.v[j])) << 8 * (j % 4);
    __builtin_memcpy(q + h, packed, kN);
  }
  if (threadIdx.x == 0) a.scales[row] = quantizer.scale;
}

// ---- tiles ----------------------------------------------------------------------------------

struct Product8Args {
  const int8_t* a;       // tokens [rows, K], a_stride bytes apart
  const int8_t* w;       // weights [S or 1][N, K], w_stride bytes apart
  const float* a_scale;  // a row
  const float* w_scale;  // an output
  const float* bias;
  long long a_stride, w_stride, a_bytes, slab_bytes;
  int rows, N, K;        // of dense products: rows; of Experts8's: pairs
  int out_tiles;         // tiles along N
  // Experts8: tiles of the sorted rows
  const int2* tiles;
  const int* n_tiles;
  const int* offsets;
  const int* pairs;      // the pair at every sorted row; its token is pair / k
  int k;
  void* out;
  long long out_stride;  // elements
  bool wide_stores;
};

enum class Form { kDense, kGateUp, kDown };

__device__ __forceinline__ __amdgpu_buffer_rsrc_t range_of(const void* p, long long bytes) {
  const unsigned n = bytes < (long long)kMaxRange ? (unsigned)bytes : kMaxRange;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, (int)n, 0x00027000);
}

__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, char* to, unsigned offset,
                                            int step) {
  using Lds = __attribute__((address_space(3))) void*;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (Lds)to, 16, offset, step, 0, 0);
}

// One tile a workgroup. Waves form WM x WN; the weights' rows of a gate-up tile are TN / 2 of the
// gate and the same of the up projection, so that a lane holds both of a hidden value.
template <int TM, int TN, int WM, int WN, Form FORM, class OUT>
__global__ __launch_bounds__(WM* WN* kWave) void product8_k(Product8Args a) {
  constexpr int kWaves = WM * WN;
  constexpr int kStage = (TM + TN) * kStepBytes;
  constexpr int kA = TM / 8 / kWaves, kB = TN / 8 / kWaves;  // loads a wave and step
  constexpr int kM = TM / WM / 16, kN = TN / WN / 16;        // operands a wave
  static_assert(kA * 8 * kWaves == TM && kB * 8 * kWaves == TN);
  constexpr bool kGrouped = FORM != Form::kDense, kGated = FORM == Form::kGateUp;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];

  // consecutive workgroups go to the eight dies in turn: each die gets a run of tiles, so that
  // its second-level cache holds what they share
  const int m_tiles = kGrouped ? *a.n_tiles : (a.rows + TM - 1) / TM;
  const long long n = (long long)m_tiles * a.out_tiles, per = (n + 7) / 8;
  const long long in_die = blockIdx.x / 8, at = (blockIdx.x % 8) * per + in_die;
  if (in_die >= per || at >= n) return;
  const int n_tile = (int)(at / m_tiles), m_tile = (int)(at - (long long)n_tile * m_tiles);
  int slot = 0, m0 = m_tile * TM, m_end = a.rows;
  if constexpr (kGrouped) {
    const int2 t = a.tiles[m_tile];
    slot = t.x;
    m0 = t.y;
    m_end = a.offsets[slot + 1];
  }
  const int n0 = n_tile * (kGated ? TN / 2 : TN);

  const int lane = __lane_id(), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row_in = lane >> 3, chunk = (lane & 7) ^ row_in;
  unsigned a_at[kA], b_at[kB];
  const int8_t* a_base = a.a;
  long long a_bytes = a.a_bytes;
  if constexpr (!kGated) {
    a_base += (long long)m0 * a.a_stride;
    a_bytes -= (long long)m0 * a.a_stride;
  }
#pragma unroll
  for (int i = 0; i < kA; ++i) {
    int r = (i * kWaves + wave) * 8 + row_in;
    if constexpr (kGated) {
      const int p = m0 + r;
      r = (p < m_end ? a.pairs[p] : a.pairs[m0]) / a.k;
    }
    a_at[i] = (unsigned)(r * a.a_stride) + 16 * chunk;
  }
  const int8_t* const slab = a.w + slot * a.slab_bytes;
  const int8_t* const b_base = slab + (kGated ? 0 : n0 * a.w_stride);
  const long long b_bytes = a.slab_bytes - (b_base - slab);
#pragma unroll
  for (int i = 0; i < kB; ++i) {
    int r = (i * kWaves + wave) * 8 + row_in;
    if constexpr (kGated) {
      const int half = a.N / 2, of = n0 + (r & (TN / 2 - 1));
      r = r < TN / 2 ? min(of, half - 1) : half + min(of, half - 1);
    }
    b_at[i] = (unsigned)(r * a.w_stride) + 16 * chunk;
  }
  const __amdgpu_buffer_rsrc_t a_range = range_of(a_base, a_bytes);
  const __amdgpu_buffer_rsrc_t b_range = range_of(b_base, b_bytes);

  const int steps = (a.K + kStepBytes - 1) / kStepBytes;
  const auto load = [&](int step) {
    char* const to = lds + (step & 1) * kStage;
    const bool behind = step * kStepBytes + 16 * chunk >= a.K;
#pragma unroll
    for (int i = 0; i < kA; ++i)
      load_to_lds(a_range, to + (i * kWaves + wave) * 1024, behind ? kFarOffset : a_at[i],
                  step * kStepBytes);
#pragma unroll
    for (int i = 0; i < kB; ++i)
      load_to_lds(b_range, to + TM * kStepBytes + (i * kWaves + wave) * 1024, b_at[i],
                  step * kStepBytes);
  };

  const int wm = wave / WN, wn = wave % WN, col = lane & 15, quad = lane >> 4;
  // a wave's outputs: kN operands of 16, of a gate-up tile half of them gate and half up
  const auto b_row = [&](int j) {
    if constexpr (kGated)
      return (j < kN / 2 ? 0 : TN / 2) + wn * (kN / 2) * 16 + (j % (kN / 2)) * 16;
    else
      return wn * kN * 16 + j * 16;
  };
  i32x4 acc[kM][kN] = {};
  load(0);
  for (int step = 0; step < steps; ++step) {
    mem_sync();
    if (step + 1 < steps) load(step + 1);
    const char* const from = lds + (step & 1) * kStage;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int place = 16 * ((half * 4 + quad) ^ (col & 7));
      i32x4 av[kM], bv[kN];
#pragma unroll
      for (int i = 0; i < kM; ++i)
        av[i] = *(const i32x4*)(from + (wm * kM * 16 + i * 16 + col) * kStepBytes + place);
#pragma unroll
      for (int j = 0; j < kN; ++j)
        bv[j] = *(const i32x4*)(from + (TM + b_row(j) + col) * kStepBytes + place);
#pragma unroll
      for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int j = 0; j < kN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bv[j], av[i], acc[i][j], 0, 0, 0);
    }
  }
  products_done();

#pragma unroll
  for (int i = 0; i < kM; ++i) {
    const int m = m0 + wm * kM * 16 + i * 16 + col;
    if (m >= m_end) continue;
    const float row_scale = a.a_scale[kGated ? a.pairs[m] / a.k : m];
    OUT* const out = static_cast<OUT*>(a.out) + m * a.out_stride;
    if constexpr (kGated) {
#pragma unroll
      for (int j = 0; j < kN / 2; ++j) {
        const int o = n0 + b_row(j) + quad * 4, half = a.N / 2;
        if (o >= half) continue;  // half is a multiple of 16
        const float* const gs = a.w_scale + (long long)slot * a.N + o;
        f32x4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = (float)acc[i][j][e] * row_scale * gs[e];
          const float u = (float)acc[i][j + kN / 2][e] * row_scale * gs[half + e];
          h[e] = g / (1.f + __expf(-g)) * u;
        }
        __builtin_memcpy(out + o, &h, 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        const int o = n0 + b_row(j) + quad * 4;
        const float* const ws = a.w_scale + (long long)slot * a.N;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (o + e >= a.N) continue;
          float y = (float)acc[i][j][e] * row_scale * ws[o + e];
          if (a.bias) y += a.bias[o + e];
          out[o + e] = from_f32<OUT>(y);
        }
      }
    }
  }
}

}  // namespace ec
