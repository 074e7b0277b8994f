// libexpertcache.so: entry points of the operators for many tokens (declared in
// include/expert_cache.h): pairs sorted by slot and back, products in 8-bit integers.
//
// Argument checks run on the host before any HIP call and return -1; otherwise each entry point
// launches its kernels on the caller's stream and returns hipGetLastError(). The library keeps no
// state and allocates nothing.
#include <hip/hip_runtime.h>

#include "../../include/expert_cache.h"
#include "host.h"
#include "int8.h"
#include "sort.h"

namespace ec {
namespace {

constexpr int kMaxTopK = 64;
constexpr int kMaxRow = 1 << 20;        // elements of a row that is moved
constexpr long long kMaxGrid = 0x7FFFFFFFll;

bool type_bad(int type) { return type < EXPERT_CACHE_F32 || type > EXPERT_CACHE_F16; }
int size_of(int type) { return type == EXPERT_CACHE_F32 ? 4 : type == EXPERT_CACHE_INT8 ? 1 : 2; }

bool pairs_bad(int T, int k) {
  return T < 0 || k <= 0 || k > kMaxTopK || (long long)T * k > kSortMaxPairs;
}

// bytes from a matrix's first to its last element
long long span(long long rows, long long stride, long long length, int size) {
  return rows > 0 ? ((rows - 1) * stride + length) * size : 0;
}

// ---- sorting ------------------------------------------------------------------------------

int sort_blocks(int n) {
  if (n <= kSortOne) return 1;
  const int want = (n + 4095) / 4096;
  return want < kSortMaxBlocks ? want : kSortMaxBlocks;
}

long sort_bytes(int n, int S) {
  const int blocks = sort_blocks(n);
  return blocks > 1 ? 4L * blocks * (S + 1) : 0;
}

int launch_sort(SortArgs a, hipStream_t stream) {
  const int blocks = sort_blocks(a.n);
  a.chunk = (a.n + blocks - 1) / blocks;
  // a run of 64 pairs or more a wave, and 64 KB of counts at most
  int waves = 1;
  while (waves < 16 && waves * kWave < a.chunk) waves *= 2;
  const int keys = a.S + 1;
  while ((2 + waves) * keys * 4 + 4 > 65536) waves /= 2;
  const size_t lds = (size_t)(2 + waves) * keys * 4 + 4;
  if (blocks > 1) {
    hipLaunchKernelGGL(sort_count_k, dim3(blocks), dim3(1024), 0, stream, a);
    hipLaunchKernelGGL(sort_place_k<true>, dim3(blocks), dim3(waves * kWave), lds, stream, a);
  } else {
    hipLaunchKernelGGL(sort_place_k<false>, dim3(1), dim3(waves * kWave), lds, stream, a);
  }
  return (int)hipGetLastError();
}

// ---- rows ---------------------------------------------------------------------------------

template <class F>
int with_type(int type, F&& f) {
  switch (type) {
    case EXPERT_CACHE_F32: f(float{}); break;
    case EXPERT_CACHE_BF16: f(Bf16{}); break;
    default: f(F16{}); break;
  }
  return (int)hipGetLastError();
}

bool rows_bad(long rows, const void* x, long stride, int H) {
  return x == nullptr || (rows > 1 && stride < H);
}

// ---- 8-bit integers -----------------------------------------------------------------------

template <class X>
int launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(quantize_k<X>, dim3(a.rows), dim3(kQuantizeThreads), 0, stream, a);
  return (int)hipGetLastError();
}

template <int TM, int TN, int WM, int WN, Form FORM, class OUT>
int launch_product(const Product8Args& a, long long m_tiles, hipStream_t stream) {
  const long long blocks = (m_tiles * a.out_tiles + 7) / 8 * 8;
  if (blocks > kMaxGrid) return -1;
  hipLaunchKernelGGL((product8_k<TM, TN, WM, WN, FORM, OUT>), dim3((unsigned)blocks),
                     dim3(WM * WN * kWave), 0, stream, a);
  return (int)hipGetLastError();
}

template <class OUT>
int launch_dense(Product8Args& a, hipStream_t stream) {
  a.out_tiles = (a.N + 127) / 128;
  if (a.rows <= 32)
    return launch_product<32, 128, 1, 4, Form::kDense, OUT>(a, (a.rows + 31) / 32, stream);
  return launch_product<128, 128, 2, 2, Form::kDense, OUT>(a, (a.rows + 127) / 128, stream);
}

bool linear_bad(const expert_cache_linear* l, int type, int T) {
  if (l == nullptr || l->O <= 0 || l->H <= 0 || l->H > kMaxLength8) return true;
  if (l->w_stride % 16 || l->w_stride < l->H || l->w_stride > (1 << 22)) return true;
  if (type != EXPERT_CACHE_BF16 && type != EXPERT_CACHE_F16 && type != EXPERT_CACHE_INT8)
    return true;
  return T < 0 || T > (1 << 24) || l->O > (1 << 24);
}

long up(long v, long to) { return (v + to - 1) / to * to; }

struct Moe8Plan {
  long offsets, rows, places, counts, tiles, n_tiles, q, q_scale, h, h8, h_scale, bytes;
  long max_tiles;
  int tile_rows;
};

Moe8Plan moe8_plan(const expert_cache_experts* e, long T, long k) {
  Moe8Plan p;
  const long n = T * k;
  p.tile_rows = n > 32L * e->S ? 128 : 32;
  p.max_tiles = n / p.tile_rows + (e->S < n ? e->S : n);
  long at = 0;
  const auto take = [&](long bytes) {
    const long from = at;
    at += up(bytes, 256);
    return from;
  };
  p.offsets = take(4L * (e->S + 1));
  p.rows = take(4 * n);
  p.places = take(4 * n);
  p.counts = take(sort_bytes((int)n, e->S));
  p.tiles = take(8 * p.max_tiles);
  p.n_tiles = take(4);
  p.q = take(T * e->H);
  p.q_scale = take(4 * T);
  p.h = take(4 * n * (e->H > e->I ? e->H : e->I));  // hidden values, then the experts' outputs
  p.h8 = take(n * e->I);
  p.h_scale = take(4 * n);
  p.bytes = at;
  return p;
}

bool moe8_bad(const expert_cache_experts* e, int T, int k) {
  if (e == nullptr || e->S <= 0 || e->S > kSortMaxSlots || e->H <= 0 || e->I <= 0) return true;
  if (e->type != EXPERT_CACHE_BF16 && e->type != EXPERT_CACHE_F16) return true;
  if (e->weights != EXPERT_CACHE_INT8 || e->H % 16 || e->I % 16) return true;
  if (e->H > kMaxLength8 || e->I > kMaxLength8) return true;
  if (2LL * e->I * e->H > (long long)kMaxRange) return true;
  return pairs_bad(T, k) || (long long)T * e->H > (long long)kMaxRange;
}

template <Form FORM>
int launch_grouped(const Product8Args& a, const Moe8Plan& p, hipStream_t stream) {
  if (p.tile_rows == 32) return launch_product<32, 128, 1, 4, FORM, float>(a, p.max_tiles, stream);
  return launch_product<128, 128, 2, 2, FORM, float>(a, p.max_tiles, stream);
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int expert_cache_sort_workspace(int T, int top_k, int S, long* bytes) {
  if (bytes == nullptr || pairs_bad(T, top_k) || S <= 0 || S > kSortMaxSlots) return -1;
  *bytes = sort_bytes(T * top_k, S);
  return 0;
}

int expert_cache_sort(const void* ids, int id_bytes, int T, int top_k, int S, int* offsets,
                      int* rows, int* places, void* workspace, hipStream_t stream) {
  if (pairs_bad(T, top_k) || S <= 0 || S > kSortMaxSlots) return -1;
  if (id_bytes != 4 && id_bytes != 8) return -1;
  if (offsets == nullptr) return -1;
  const long long n = (long long)T * top_k, part = sort_bytes((int)n, S);
  if (n > 0 && (ids == nullptr || rows == nullptr || places == nullptr)) return -1;
  if (part > 0 && (workspace == nullptr || !aligned16(workspace))) return -1;
  const void* const of[] = {ids, offsets, rows, places};
  const long long size[] = {n * id_bytes, 4LL * (S + 1), 4 * n, 4 * n};
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < i; ++j)
      if (ranges_meet(of[i], size[i], of[j], size[j])) return -1;
  SortArgs a = {};
  a.ids = ids;
  a.n = (int)n;
  a.S = S;
  a.wide = id_bytes == 8;
  a.offsets = offsets;
  a.rows = rows;
  a.places = places;
  a.counts = static_cast<int*>(workspace);
  return launch_sort(a, stream);
}

int expert_cache_dispatch(const void* x, int type, long x_stride, const int* places,
                          const int* offsets, int T, int top_k, int S, int H, void* out,
                          long out_stride, hipStream_t stream) {
  if (pairs_bad(T, top_k) || type_bad(type) || S <= 0 || S > kSortMaxSlots) return -1;
  if (H <= 0 || H > kMaxRow) return -1;
  if (T == 0) return 0;
  const long long n = (long long)T * top_k;
  if (rows_bad(T, x, x_stride, H) || rows_bad(n, out, out_stride, H)) return -1;
  if (places == nullptr || offsets == nullptr) return -1;
  const long long out_bytes = span(n, out_stride, H, size_of(type));
  if (ranges_meet(x, span(T, x_stride, H, size_of(type)), out, out_bytes) ||
      ranges_meet(places, 4 * n, out, out_bytes) ||
      ranges_meet(offsets, 4LL * (S + 1), out, out_bytes))
    return -1;
  MoveArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.places = places;
  a.offsets = offsets;
  a.out = out;
  a.out_stride = out_stride;
  a.T = T;
  a.k = top_k;
  a.S = S;
  a.H = H;
  a.n = (int)n;
  const int per = 4096 / size_of(type);
  a.chunks = (H + per - 1) / per;
  const long long blocks = ((long long)T * a.chunks + kMoveWaves - 1) / kMoveWaves;
  if (blocks > kMaxGrid) return -1;
  return with_type(type, [&](auto v) {
    hipLaunchKernelGGL(dispatch_k<decltype(v)>, dim3((unsigned)blocks), dim3(kMoveWaves * kWave),
                       0, stream, a);
  });
}

int expert_cache_combine(const void* y, int type, long y_stride, const float* weights,
                         const int* places, int T, int top_k, int H, void* out, long out_stride,
                         hipStream_t stream) {
  if (pairs_bad(T, top_k) || type_bad(type) || H <= 0 || H > kMaxRow) return -1;
  if (T == 0) return 0;
  const long long n = (long long)T * top_k;
  if (rows_bad(n, y, y_stride, H) || rows_bad(T, out, out_stride, H) || places == nullptr)
    return -1;
  const long long out_bytes = span(T, out_stride, H, size_of(type));
  if (ranges_meet(y, span(n, y_stride, H, size_of(type)), out, out_bytes) ||
      ranges_meet(places, 4 * n, out, out_bytes) ||
      (weights && ranges_meet(weights, 4 * n, out, out_bytes)))
    return -1;
  MoveArgs a = {};
  a.x = y;
  a.x_stride = y_stride;
  a.weights = weights;
  a.places = places;
  a.out = out;
  a.out_stride = out_stride;
  a.T = T;
  a.k = top_k;
  a.H = H;
  a.n = (int)n;
  const int per = 1024 / size_of(type);
  a.chunks = (H + per - 1) / per;
  const long long blocks = ((long long)T * a.chunks + kMoveWaves - 1) / kMoveWaves;
  if (blocks > kMaxGrid) return -1;
  return with_type(type, [&](auto v) {
    hipLaunchKernelGGL(combine_k<decltype(v)>, dim3((unsigned)blocks), dim3(kMoveWaves * kWave),
                       0, stream, a);
  });
}

int expert_cache_combine_grad(const void* grad, int type, long grad_stride, const void* y,
                              long y_stride, const float* weights, const int* places,
                              const int* offsets, int T, int top_k, int S, int H, void* dy,
                              long dy_stride, float* dweights, hipStream_t stream) {
  if (pairs_bad(T, top_k) || type_bad(type) || S <= 0 || S > kSortMaxSlots) return -1;
  if (H <= 0 || H > kMaxRow || (dy == nullptr && dweights == nullptr)) return -1;
  if (T == 0) return 0;
  const long long n = (long long)T * top_k;
  if (rows_bad(T, grad, grad_stride, H) || places == nullptr || offsets == nullptr) return -1;
  if (dweights && rows_bad(n, y, y_stride, H)) return -1;
  if (dy && rows_bad(n, dy, dy_stride, H)) return -1;
  const int size = size_of(type);
  const void* const in[] = {grad, dweights ? y : nullptr, weights, places, offsets};
  const long long in_bytes[] = {span(T, grad_stride, H, size),
                                dweights ? span(n, y_stride, H, size) : 0,
                                weights ? 4 * n : 0, 4 * n, 4LL * (S + 1)};
  const long long dy_bytes = dy ? span(n, dy_stride, H, size) : 0;
  const long long dw_bytes = dweights ? 4 * n : 0;
  for (int i = 0; i < 5; ++i)
    if (ranges_meet(in[i], in_bytes[i], dy, dy_bytes) ||
        ranges_meet(in[i], in_bytes[i], dweights, dw_bytes))
      return -1;
  if (ranges_meet(dy, dy_bytes, dweights, dw_bytes)) return -1;
  MoveArgs a = {};
  a.x = grad;
  a.x_stride = grad_stride;
  a.y = y;
  a.y_stride = y_stride;
  a.weights = weights;
  a.places = places;
  a.offsets = offsets;
  a.out = dy;
  a.out_stride = dy_stride;
  a.dweights = dweights;
  a.T = T;
  a.k = top_k;
  a.S = S;
  a.H = H;
  a.n = (int)n;
  const unsigned blocks = (unsigned)((n + kMoveWaves - 1) / kMoveWaves);
  return with_type(type, [&](auto v) {
    hipLaunchKernelGGL(combine_grad_k<decltype(v)>, dim3(blocks), dim3(kMoveWaves * kWave), 0,
                       stream, a);
  });
}

int expert_cache_quantize(const void* x, int type, long x_stride, int T, int H, void* q,
                          long q_stride, float* scales, hipStream_t stream) {
  if (type != EXPERT_CACHE_BF16 && type != EXPERT_CACHE_F16) return -1;
  if (T < 0 || T > (1 << 24) || H <= 0 || H > kMaxRow) return -1;
  if (T == 0) return 0;
  const long padded = up(H, 16);
  if (rows_bad(T, x, x_stride, H) || rows_bad(T, q, q_stride, (int)padded)) return -1;
  if (!aligned16(q) || (T > 1 && q_stride % 16) || scales == nullptr) return -1;
  const long long q_bytes = span(T, q_stride, padded, 1), x_bytes = span(T, x_stride, H, 2);
  if (ranges_meet(x, x_bytes, q, q_bytes) || ranges_meet(x, x_bytes, scales, 4LL * T) ||
      ranges_meet(q, q_bytes, scales, 4LL * T))
    return -1;
  const QuantizeArgs a = {x, x_stride, T, H, nullptr, static_cast<int8_t*>(q), q_stride, scales};
  return type == EXPERT_CACHE_BF16 ? launch_quantize<Bf16>(a, stream)
                                   : launch_quantize<F16>(a, stream);
}

int expert_cache_linear8_workspace(const expert_cache_linear* l, int type, int T, long* bytes) {
  if (bytes == nullptr || linear_bad(l, type, T)) return -1;
  *bytes = type == EXPERT_CACHE_INT8 ? 0 : up(T * up(l->H, 16), 256) + 4L * T;
  return 0;
}

int expert_cache_linear8(const expert_cache_linear* l, const void* x, int type, long x_stride,
                         const float* x_scales, int T, void* out, int out_type, long out_stride,
                         void* workspace, hipStream_t stream) {
  if (linear_bad(l, type, T) || type_bad(out_type)) return -1;
  if (T == 0) return 0;
  if (l->w == nullptr || !aligned16(l->w) || l->scale == nullptr) return -1;
  const bool whole = type == EXPERT_CACHE_INT8;
  const long K = up(l->H, 16);
  if (rows_bad(T, x, x_stride, whole ? (int)K : l->H) || rows_bad(T, out, out_stride, l->O))
    return -1;
  if (whole && (!aligned16(x) || (T > 1 && (x_stride % 16 || x_stride > (1 << 22))) ||
                x_scales == nullptr))
    return -1;
  if (!whole && (workspace == nullptr || !aligned16(workspace))) return -1;
  const long long x_bytes = span(T, x_stride, whole ? K : l->H, size_of(type));
  const long long out_bytes = span(T, out_stride, l->O, size_of(out_type));
  if (ranges_meet(x, x_bytes, out, out_bytes) ||
      (whole && ranges_meet(x_scales, 4LL * T, out, out_bytes)))
    return -1;
  Product8Args a = {};
  a.a = static_cast<const int8_t*>(x);
  a.a_stride = x_stride;
  a.a_scale = x_scales;
  if (!whole) {
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scales = reinterpret_cast<float*>(q + up(T * K, 256));
    const QuantizeArgs z = {x, x_stride, T, l->H, nullptr, q, K, scales};
    const int rc = type == EXPERT_CACHE_BF16 ? launch_quantize<Bf16>(z, stream)
                                             : launch_quantize<F16>(z, stream);
    if (rc) return rc;
    a.a = q;
    a.a_stride = K;
    a.a_scale = scales;
  }
  a.w = static_cast<const int8_t*>(l->w);
  a.w_stride = l->w_stride;
  a.w_scale = l->scale;
  a.bias = l->bias;
  a.a_bytes = span(T, a.a_stride, K, 1);
  a.slab_bytes = span(l->O, l->w_stride, K, 1);
  a.rows = T;
  a.N = l->O;
  a.K = (int)K;
  a.out = out;
  a.out_stride = out_stride;
  if (out_type == EXPERT_CACHE_F32) return launch_dense<float>(a, stream);
  return out_type == EXPERT_CACHE_BF16 ? launch_dense<Bf16>(a, stream)
                                       : launch_dense<F16>(a, stream);
}

int expert_cache_moe8_workspace(const expert_cache_experts* e, int T, int top_k, long* bytes) {
  if (bytes == nullptr || moe8_bad(e, T, top_k)) return -1;
  *bytes = moe8_plan(e, T, top_k).bytes;
  return 0;
}

int expert_cache_moe8(const expert_cache_experts* e, const void* x, long x_stride,
                      const float* topk_weights, const void* ids, int id_bytes, int T, int top_k,
                      void* out, long out_stride, void* workspace, hipStream_t stream) {
  if (moe8_bad(e, T, top_k) || (id_bytes != 4 && id_bytes != 8)) return -1;
  if (T == 0) return 0;
  if (e->w13 == nullptr || e->w2 == nullptr || !aligned16(e->w13) || !aligned16(e->w2)) return -1;
  if (e->s13 == nullptr || e->s2 == nullptr) return -1;
  if (rows_bad(T, x, x_stride, e->H) || rows_bad(T, out, out_stride, e->H)) return -1;
  if (topk_weights == nullptr || ids == nullptr) return -1;
  if (workspace == nullptr || !aligned16(workspace)) return -1;
  const long long out_bytes = span(T, out_stride, e->H, 2), n = (long long)T * top_k;
  if (ranges_meet(x, span(T, x_stride, e->H, 2), out, out_bytes) ||
      ranges_meet(ids, n * id_bytes, out, out_bytes) ||
      ranges_meet(topk_weights, 4 * n, out, out_bytes))
    return -1;
  const Moe8Plan p = moe8_plan(e, T, top_k);
  char* const at = static_cast<char*>(workspace);
  const auto ints = [&](long offset) { return reinterpret_cast<int*>(at + offset); };
  const auto floats = [&](long offset) { return reinterpret_cast<float*>(at + offset); };
  const auto bytes = [&](long offset) { return reinterpret_cast<int8_t*>(at + offset); };

  SortArgs s = {};
  s.ids = ids;
  s.probs = topk_weights;
  s.n = (int)n;
  s.S = e->S;
  s.wide = id_bytes == 8;
  s.offsets = ints(p.offsets);
  s.rows = ints(p.rows);
  s.places = ints(p.places);
  s.counts = ints(p.counts);
  s.tiles = reinterpret_cast<int2*>(at + p.tiles);
  s.n_tiles = ints(p.n_tiles);
  s.tile_rows = p.tile_rows;
  int rc = launch_sort(s, stream);
  if (rc) return rc;

  QuantizeArgs z = {x, x_stride, T, e->H, nullptr, bytes(p.q), e->H, floats(p.q_scale)};
  rc = e->type == EXPERT_CACHE_BF16 ? launch_quantize<Bf16>(z, stream)
                                    : launch_quantize<F16>(z, stream);
  if (rc) return rc;

  Product8Args a = {};
  a.a = z.q;
  a.a_stride = e->H;
  a.a_scale = z.scales;
  a.a_bytes = (long long)T * e->H;
  a.w = static_cast<const int8_t*>(e->w13);
  a.w_stride = e->H;
  a.w_scale = e->s13;
  a.slab_bytes = 2LL * e->I * e->H;
  a.rows = (int)n;
  a.N = 2 * e->I;
  a.K = e->H;
  a.out_tiles = (e->I + 63) / 64;
  a.tiles = s.tiles;
  a.n_tiles = s.n_tiles;
  a.offsets = s.offsets;
  a.pairs = s.rows;
  a.k = top_k;
  a.out = floats(p.h);
  a.out_stride = e->I;
  rc = launch_grouped<Form::kGateUp>(a, p, stream);
  if (rc) return rc;

  z = {a.out, e->I, (int)n, e->I, s.offsets + e->S, bytes(p.h8), e->I, floats(p.h_scale)};
  rc = launch_quantize<float>(z, stream);
  if (rc) return rc;

  a.a = z.q;
  a.a_stride = e->I;
  a.a_scale = z.scales;
  a.a_bytes = n * e->I;
  a.w = static_cast<const int8_t*>(e->w2);
  a.w_stride = e->I;
  a.w_scale = e->s2;
  a.slab_bytes = (long long)e->H * e->I;
  a.N = e->H;
  a.K = e->I;
  a.out_tiles = (e->H + 127) / 128;
  a.out_stride = e->H;
  rc = launch_grouped<Form::kDown>(a, p, stream);
  if (rc) return rc;

  MoveArgs m = {};
  m.x = a.out;
  m.x_stride = e->H;
  m.weights = topk_weights;
  m.places = s.places;
  m.out = out;
  m.out_stride = out_stride;
  m.T = T;
  m.k = top_k;
  m.H = e->H;
  m.n = (int)n;
  m.chunks = (e->H + 255) / 256;
  const long long blocks = ((long long)T * m.chunks + kMoveWaves - 1) / kMoveWaves;
  if (e->type == EXPERT_CACHE_BF16)
    hipLaunchKernelGGL((combine_k<float, Bf16>), dim3((unsigned)blocks), dim3(kMoveWaves * kWave),
                       0, stream, m);
  else
    hipLaunchKernelGGL((combine_k<float, F16>), dim3((unsigned)blocks), dim3(kMoveWaves * kWave),
                       0, stream, m);
  return (int)hipGetLastError();
}

}  // extern "C"
