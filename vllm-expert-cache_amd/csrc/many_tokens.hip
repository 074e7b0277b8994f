// libexpertcache.so: entry points of the operators for many tokens (declared in
// include/expert_cache.h): pairs sorted by slot and back, products in 8-bit integers.
//
// Argument checks run on the host before any HIP call and return -1; otherwise each entry point
// launches its kernels on the caller's stream and returns hipGetLastError(). The library keeps no
// state and allocates nothing.
#include <hip/hip_runtime.h>

#include <initializer_list>
#include <type_traits>

#include "../../include/expert_cache.h"
#include "host.h"
#include "int8.h"
#include "sort.h"

namespace ec {
namespace {

constexpr int kMaxTopK = 64;
constexpr int kMaxRow = 1 << 20;        // elements of a row that is moved
// A launch has less than 2^32 threads, and these keep every one's below that:
constexpr long long kMaxMoved = 1ll << 35;   // bytes of the tokens' rows that are moved (a wave takes
                                             // 1 KB of a row, and there are up to 2^24 tokens)
constexpr int kMaxTokens8 = 1 << 23;         // rows that are quantised, at most a workgroup of 256 each
constexpr long long kMaxValues8 = 1ll << 36; // hidden values and experts' outputs (tiles of 512
                                             // threads for 2^15 of them, and one a slot)
constexpr long long kMaxResults8 = 1ll << 38;

long up(long v, long to) { return (v + to - 1) / to * to; }
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
  const int want = (n + kSortLot - 1) / kSortLot;
  return want < kSortMaxBlocks ? want : kSortMaxBlocks;
}

long sort_bytes(int n, int S) {
  const int blocks = sort_blocks(n);
  return blocks > 1 ? 4L * blocks * (S + 1) : 0;
}

template <int W, int R, bool MANY>
void launch_place(const SortArgs& a, int blocks, hipStream_t stream) {
  hipLaunchKernelGGL((sort_place_k<W, R, MANY>), dim3(blocks), dim3(W * kWave), 0, stream, a);
}

// Pairs a workgroup: whole lots, so that none but the last is short.
int sort_chunk(int n) {
  const int blocks = sort_blocks(n);
  return blocks > 1 ? ((n - 1) / blocks / kSortLot + 1) * kSortLot : n;
}

int launch_sort(SortArgs a, hipStream_t stream) {
  a.chunk = sort_chunk(a.n);
  const int blocks = a.n <= kSortOne ? 1 : (a.n - 1) / a.chunk + 1;
  if (blocks > 1) {
    hipLaunchKernelGGL(sort_count_k, dim3(blocks), dim3(1024), 0, stream, a);
    launch_place<16, 1, true>(a, blocks, stream);
  } else if (a.n <= 64) {
    launch_place<1, 1, false>(a, 1, stream);
  } else if (a.n <= 256) {
    launch_place<4, 1, false>(a, 1, stream);
  } else if (a.n <= 1024) {
    launch_place<16, 1, false>(a, 1, stream);
  } else {
    launch_place<16, 4, false>(a, 1, stream);
  }
  return (int)hipGetLastError();
}

// ---- rows ---------------------------------------------------------------------------------

// Rows of more bytes than this are moved past the caches: 512 tokens' 8 rows of 2048 bf16 (17 MB) 7.5
// us through them and 8.1 past them (combine_grad), 4096 tokens' (134 MB) 57.7 and 53.6.
constexpr long long kOnceBytes = 64ll << 20;

// Calls f with the type of the values and how their rows can be moved: those of `rows` matrices that
// begin at p[i], stride[i] elements apart.
template <class F>
int with_rows(int type, int H, long long moved, std::initializer_list<const void*> p,
              std::initializer_list<long> stride, F&& f) {
  const int size = size_of(type), piece = 16 / size;
  bool whole = H % piece == 0;
  for (const void* q : p) whole = whole && aligned16(q);
  for (long n : stride) whole = whole && n % piece == 0;
  const auto of = [&](auto x) {
    using std::integral_constant;
    if (H < piece) f(x, integral_constant<Move, Move::kElements>());
    else if (!whole) f(x, integral_constant<Move, Move::kAnywhere>());
    else if (moved >= kOnceBytes) f(x, integral_constant<Move, Move::kOnce>());
    else f(x, integral_constant<Move, Move::kWhole>());
  };
  switch (type) {
    case EXPERT_CACHE_F32: of(float{}); break;
    case EXPERT_CACHE_BF16: of(Bf16{}); break;
    default: of(F16{}); break;
  }
  return (int)hipGetLastError();
}

bool moved_bad(long long T, int H, int type) {
  return type_bad(type) || H <= 0 || H > kMaxRow || T * H * size_of(type) > kMaxMoved;
}

bool rows_bad(long rows, const void* x, long stride, int H) {
  return x == nullptr || (rows > 1 && stride < H);
}

// ---- 8-bit integers -----------------------------------------------------------------------

template <class X>
int launch_quantize(const QuantizeArgs& a, hipStream_t stream) {
  // A wave a row where rows are many and short, else a workgroup: 16384 rows of 768 floats 13.0 us, by
  // workgroups 16.1; 4096 rows of 4096 bf16 16.5 and 14.0.
  const long bytes = (long)a.H * sizeof(X);
  const dim3 block(kQuantizeThreads), all(a.rows), quarter((a.rows + 3) / 4);
  if (a.rows >= 1024 && bytes <= 4096)
    hipLaunchKernelGGL((quantize_k<64, 4, X>), quarter, block, 0, stream, a);
  else if (bytes <= 4096)
    hipLaunchKernelGGL((quantize_k<256, 1, X>), all, block, 0, stream, a);
  else if (bytes <= 16384)
    hipLaunchKernelGGL((quantize_k<256, 4, X>), all, block, 0, stream, a);
  else
    hipLaunchKernelGGL((quantize_k<256, 16, X>), all, block, 0, stream, a);
  return (int)hipGetLastError();
}

template <class X>
int launch_begin(const SortArgs& s, const QuantizeArgs& q, hipStream_t stream) {
  const bool many = s.n > kSortOne;
  const int sorting = many ? (s.n - 1) / s.chunk + 1 : 1;
  const dim3 grid(sorting + (q.rows + 3) / 4);
  if (many) {
    hipLaunchKernelGGL((begin8_k<1, X, true>), grid, dim3(1024), 0, stream, s, sorting, q);
    launch_place<16, 1, true>(s, sorting, stream);
  } else if (s.n > 1024) {
    hipLaunchKernelGGL((begin8_k<4, X, false>), grid, dim3(1024), 0, stream, s, sorting, q);
  } else {
    hipLaunchKernelGGL((begin8_k<1, X, false>), grid, dim3(1024), 0, stream, s, sorting, q);
  }
  return (int)hipGetLastError();
}

template <int TM, int TN, int WM, int WN, int ST, Form FORM, class OUT>
int launch_product(Product8Args& a, long long m_tiles, int outputs, hipStream_t stream) {
  a.out_tiles = (outputs + TN - 1) / TN;
  // every die's tiles, of which the last may be cut in parts: four of less than a quarter of its units
  const long long per = (m_tiles * a.out_tiles * (FORM == Form::kPart ? a.splits : 1) + 7) / 8;
  const long long blocks = 8 * (per + 3 * kDieUnits / 4);
  hipLaunchKernelGGL((product8_k<TM, TN, WM, WN, ST, FORM, OUT>), dim3((unsigned)blocks),
                     dim3(WM * WN * kWave), 0, stream, a);
  return (int)hipGetLastError();
}

// How a dense product of 8-bit rows is cut, us in a graph on MI355X with quantize:
//   side 0   16 outputs a workgroup, the length over its waves. Few tokens and outputs: 32 tokens of
//            2048 x 2048 7.2, with tiles of 64 9.3; 48 of 4096 x 4096 14.3 and 14.4; but 16 of 4096 x
//            14336 15.9 and 15.5, and 32 of 14336 x 4096 27.8 and 21.9.
//   64       while all tiles are beside each other: 128 tokens of 4096 x 14336 (448 tiles) 19.4, with
//            tiles of 128 32.2; 512 of 4096 x 4096 (512) 21.3 and 26.8; 256 of 4096 x 14336 (896)
//            32.8 and 31.8. Long products of few tiles are cut along the length as well, at the
//            price of a launch that joins the sums: 64 tokens of 14336 x 4096 24.2, whole 36.4, 128
//            29.9 and 41.8; but 64 of 4096 x 4096 15.2 and 14.7, and 256 of 14336 x 4096 46.9 and 43.5.
//   256      where there is one for every third compute unit or more: 512 of 4096 x 14336 (112 tiles'
//            area) 44.8, with tiles of 128 45.9; 4096 of 4096 x 4096 75.5 and 100.6; 384 of 4096 x
//            14336 (84) 43 and 37
struct DensePlan {
  int side, splits;
};

DensePlan dense_plan(long T, long O, long K) {
  if (O < 8192 && (T <= 16 || (T <= 48 && K <= 4096))) return {0, 1};
  const long of_64 = ((T + 63) / 64) * ((O + 63) / 64), steps = (K + kStepBytes - 1) / kStepBytes;
  if (of_64 <= 512) {
    const long beside = 256 / of_64, long_enough = steps / 8;
    const long splits = steps < 48 ? 1 : beside < long_enough ? beside : long_enough;
    return {64, splits < 1 ? 1 : splits > 8 ? 8 : (int)splits};
  }
  return {T * O >= 96L * 65536 ? 256 : 128, 1};
}

template <int MI, class X, class OUT>
int launch_few(const Product8Args& a, const void* x, long x_stride, int H, hipStream_t stream) {
  hipLaunchKernelGGL((few8_k<MI, X, OUT>), dim3((a.N + 15) / 16),
                     dim3(kFewWaves * kWave), 0, stream, a, static_cast<const X*>(x),
                     (long long)x_stride, H);
  return (int)hipGetLastError();
}

template <class OUT>
int launch_dense(Product8Args& a, const DensePlan& plan, int* part, hipStream_t stream) {
  if (plan.side == 0) {
    if (a.rows <= 16) return launch_few<1, int8_t, OUT>(a, nullptr, 0, 0, stream);
    if (a.rows <= 32) return launch_few<2, int8_t, OUT>(a, nullptr, 0, 0, stream);
    return launch_few<4, int8_t, OUT>(a, nullptr, 0, 0, stream);
  }
  const long long m_tiles = (a.rows + plan.side - 1) / plan.side;
  if (plan.side == 256)
    return launch_product<256, 256, 2, 4, 2, Form::kDense, OUT>(a, m_tiles, a.N, stream);
  if (plan.side == 128)
    return launch_product<128, 128, 2, 2, 2, Form::kDense, OUT>(a, m_tiles, a.N, stream);
  if (plan.splits == 1)
    return launch_product<64, 64, 4, 1, 4, Form::kDense, OUT>(a, m_tiles, a.N, stream);
  JoinArgs j = {part, a.a_scale, a.w_scale, a.bias, a.out, a.out_stride,
                plan.splits, a.rows, a.N, (int)up(a.N, 4)};
  a.splits = plan.splits;
  a.N = j.stride;
  a.out = part;
  a.out_stride = j.stride;
  a.whole_stores = true;
  const int rc = launch_product<64, 64, 4, 1, 4, Form::kPart, float>(a, m_tiles, j.N, stream);
  if (rc) return rc;
  const long long blocks = ((long long)j.rows * (j.stride / 4) + kJoinThreads - 1) / kJoinThreads;
  hipLaunchKernelGGL(join8_k<OUT>, dim3((unsigned)blocks), dim3(kJoinThreads), 0, stream, j);
  return (int)hipGetLastError();
}

template <class X>
int launch_few_of(const Product8Args& a, int out_type, const void* x, long x_stride, int H,
                  hipStream_t stream) {
  if (out_type == EXPERT_CACHE_F32) return launch_few<1, X, float>(a, x, x_stride, H, stream);
  return out_type == EXPERT_CACHE_BF16 ? launch_few<1, X, Bf16>(a, x, x_stride, H, stream)
                                       : launch_few<1, X, F16>(a, x, x_stride, H, stream);
}

// The workspace of a projection: tokens in 8 bits and their scales, sums of parts of the length.
struct Linear8Layout {
  long scales, part, bytes;
};

Linear8Layout linear8_layout(const expert_cache_linear* l, int type, long T) {
  const long K = up(l->H, 16);
  Linear8Layout p = {};
  if (T == 0) return p;  // no tiles that a plan could put beside each other
  if (type != EXPERT_CACHE_INT8) {
    p.scales = up(T * K, 256);
    p.part = p.scales + up(4 * T, 256);
  }
  const DensePlan plan = dense_plan(T, l->O, K);
  p.bytes = p.part + (plan.splits > 1 ? 4L * plan.splits * T * up(l->O, 4) : 0);
  return p;
}

// Results go 16 bytes at a time by a descriptor of a tile's rows: whole cells of a row, and a range
// that 32 bits hold.
bool stores_whole(const void* out, long long stride, int width, long long rows, int size) {
  const int cell = 16 / size;
  return width % cell == 0 && aligned16(out) && (rows == 1 || stride % cell == 0) &&
         256 * stride * size < (long long)kMaxRange;
}

bool linear_bad(const expert_cache_linear* l, int type, int T) {
  if (l == nullptr || l->O <= 0 || l->H <= 0 || l->H > kMaxLength8) return true;
  if (l->w_stride % 16 || l->w_stride < l->H || l->w_stride > (1 << 22)) return true;
  if (type != EXPERT_CACHE_BF16 && type != EXPERT_CACHE_F16 && type != EXPERT_CACHE_INT8)
    return true;
  return T < 0 || T > kMaxTokens8 || l->O > (1 << 24) || (long long)T * l->O > kMaxResults8;
}

struct Moe8Plan {
  long offsets, rows, places, counts, tiles, n_tiles, q, q_scale, h, h8, h_scale, bytes;
  long max_tiles;
  int tile_rows;
};

// Rows of the experts' tiles by the pairs a slot, us a call on MI355X with 64, 128 and 256 rows: 33
// tokens, 8 of 64 slots of 2048 x 768 (4 a slot) 70, 77, 86; 128 tokens, 8 of 128 (8) 133, 134, 142;
// 1024 (64) 196, 201, 212; 2048 (128) 285, 263, 265; 1024, 2 of 8 of 4096 x 14336 (256) -, 677, 557.
int moe8_rows(long pairs, long slots) {
  return pairs >= 256 * slots ? 256 : pairs > 96 * slots ? 128 : 64;
}

Moe8Plan moe8_plan(const expert_cache_experts* e, long T, long k) {
  Moe8Plan p;
  const long n = T * k;
  p.tile_rows = moe8_rows(n, e->S);
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
  p.tiles = take(16 * p.max_tiles);
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
  if (pairs_bad(T, k) || (long long)T * e->H > (long long)kMaxRange) return true;
  const long long n = (long long)T * k;
  return n > kMaxTokens8 || n * (e->H > e->I ? e->H : e->I) > kMaxValues8;
}

template <Form FORM>
int launch_grouped(Product8Args& a, const Moe8Plan& p, hipStream_t stream) {
  if (p.tile_rows == 64)
    return launch_product<64, 128, 2, 2, 2, FORM, float>(a, p.max_tiles, a.N, stream);
  if (p.tile_rows == 128)
    return launch_product<128, 128, 2, 2, 2, FORM, float>(a, p.max_tiles, a.N, stream);
  return launch_product<256, 256, 2, 4, 2, FORM, float>(a, p.max_tiles, a.N, stream);
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
                          const int* rows, int T, int top_k, int H, void* out, long out_stride,
                          hipStream_t stream) {
  if (pairs_bad(T, top_k) || moved_bad(T, H, type)) return -1;
  if (T == 0) return 0;
  const long long n = (long long)T * top_k;
  if (rows_bad(T, x, x_stride, H) || rows_bad(n, out, out_stride, H)) return -1;
  if (places == nullptr || rows == nullptr) return -1;
  const long long out_bytes = span(n, out_stride, H, size_of(type));
  if (ranges_meet(x, span(T, x_stride, H, size_of(type)), out, out_bytes) ||
      ranges_meet(places, 4 * n, out, out_bytes) || ranges_meet(rows, 4 * n, out, out_bytes))
    return -1;
  MoveArgs a = {};
  a.x = x;
  a.x_stride = x_stride;
  a.places = places;
  a.rows = rows;
  a.out = out;
  a.out_stride = out_stride;
  a.T = T;
  a.k = top_k;
  a.H = H;
  a.n = (int)n;
  const int per = kMovePieces * 1024 / size_of(type);
  a.chunks = (H + per - 1) / per;
  const long long blocks = ((long long)T * a.chunks + kMoveWaves - 1) / kMoveWaves;
  return with_rows(type, H, out_bytes, {x, out}, {T > 1 ? x_stride : 0, n > 1 ? out_stride : 0},
                   [&](auto v, auto move) {
                     hipLaunchKernelGGL((dispatch_k<decltype(v), move.value>),
                                        dim3((unsigned)blocks), dim3(kMoveWaves * kWave), 0, stream,
                                        a);
                   });
}

int expert_cache_combine(const void* y, int type, long y_stride, const float* weights,
                         const int* places, int T, int top_k, int H, void* out, long out_stride,
                         hipStream_t stream) {
  if (pairs_bad(T, top_k) || moved_bad(T, H, type)) return -1;
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
  return with_rows(type, H, span(n, y_stride, H, size_of(type)), {y, out},
                   {n > 1 ? y_stride : 0, T > 1 ? out_stride : 0}, [&](auto v, auto move) {
                     hipLaunchKernelGGL((combine_k<decltype(v), move.value>),
                                        dim3((unsigned)blocks), dim3(kMoveWaves * kWave), 0, stream,
                                        a);
                   });
}

int expert_cache_combine_grad(const void* grad, int type, long grad_stride, const void* y,
                              long y_stride, const float* weights, const int* places,
                              const int* rows, int T, int top_k, int H, void* dy, long dy_stride,
                              float* dweights, hipStream_t stream) {
  if (pairs_bad(T, top_k) || moved_bad(T, H, type)) return -1;
  if (dy == nullptr && dweights == nullptr) return -1;
  if (T == 0) return 0;
  const long long n = (long long)T * top_k;
  if (rows_bad(T, grad, grad_stride, H) || places == nullptr || rows == nullptr) return -1;
  if (dweights && rows_bad(n, y, y_stride, H)) return -1;
  if (dy && rows_bad(n, dy, dy_stride, H)) return -1;
  const int size = size_of(type);
  const void* const in[] = {grad, dweights ? y : nullptr, weights, places, rows};
  const long long in_bytes[] = {span(T, grad_stride, H, size),
                                dweights ? span(n, y_stride, H, size) : 0,
                                weights ? 4 * n : 0, 4 * n, 4 * n};
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
  a.rows = rows;
  a.out = dy;
  a.out_stride = dy_stride;
  a.dweights = dweights;
  a.T = T;
  a.k = top_k;
  a.H = H;
  a.n = (int)n;
  const unsigned blocks = (unsigned)((n + kMoveWaves - 1) / kMoveWaves);
  return with_rows(type, H, dy_bytes, {grad, dweights ? y : nullptr, dy},
                   {T > 1 ? grad_stride : 0, dweights && n > 1 ? y_stride : 0,
                    dy && n > 1 ? dy_stride : 0},
                   [&](auto v, auto move) {
                     hipLaunchKernelGGL((combine_grad_k<decltype(v), move.value>), dim3(blocks),
                                        dim3(kMoveWaves * kWave), 0, stream, a);
                   });
}

int expert_cache_quantize(const void* x, int type, long x_stride, int T, int H, void* q,
                          long q_stride, float* scales, hipStream_t stream) {
  if (type != EXPERT_CACHE_BF16 && type != EXPERT_CACHE_F16) return -1;
  if (T < 0 || T > kMaxTokens8 || H <= 0 || H > kMaxRow) return -1;
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
  *bytes = linear8_layout(l, type, T).bytes;
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
  const Linear8Layout layout = linear8_layout(l, type, T);
  if (layout.bytes > 0 && (workspace == nullptr || !aligned16(workspace))) return -1;
  const long long x_bytes = span(T, x_stride, whole ? K : l->H, size_of(type));
  const long long out_bytes = span(T, out_stride, l->O, size_of(out_type));
  if (ranges_meet(x, x_bytes, out, out_bytes) ||
      (whole && ranges_meet(x_scales, 4LL * T, out, out_bytes)))
    return -1;
  Product8Args a = {};
  // one row may come with any stride; a tile's rows behind it have to lie behind its end
  if (T == 1) {
    x_stride = whole ? K : l->H;
    out_stride = l->O;
  }
  a.a = static_cast<const int8_t*>(x);
  a.a_stride = x_stride;
  a.a_scale = x_scales;
  a.w = static_cast<const int8_t*>(l->w);
  a.w_stride = l->w_stride;
  a.w_scale = l->scale;
  a.bias = l->bias;
  a.slab_bytes = span(l->O, l->w_stride, K, 1);
  a.rows = T;
  a.scale_rows = T;
  a.N = l->O;
  a.K = (int)K;
  a.out = out;
  a.out_stride = out_stride;
  a.whole_stores = stores_whole(out, out_stride, l->O, T, size_of(out_type));
  if (!whole && T <= 16 && T * K <= kFewValues && K <= few_longest(T)) {
    if (type == EXPERT_CACHE_BF16) return launch_few_of<Bf16>(a, out_type, x, x_stride, l->H, stream);
    return launch_few_of<F16>(a, out_type, x, x_stride, l->H, stream);
  }
  if (!whole) {
    int8_t* const q = static_cast<int8_t*>(workspace);
    float* const scales = reinterpret_cast<float*>(q + layout.scales);
    const QuantizeArgs z = {x, x_stride, T, l->H, nullptr, q, K, scales};
    const int rc = type == EXPERT_CACHE_BF16 ? launch_quantize<Bf16>(z, stream)
                                             : launch_quantize<F16>(z, stream);
    if (rc) return rc;
    a.a = q;
    a.a_stride = K;
    a.a_scale = scales;
  }
  a.a_bytes = span(T, a.a_stride, K, 1);
  const DensePlan plan = dense_plan(T, l->O, K);
  int* const part = reinterpret_cast<int*>(static_cast<char*>(workspace) + layout.part);
  if (out_type == EXPERT_CACHE_F32) return launch_dense<float>(a, plan, part, stream);
  return out_type == EXPERT_CACHE_BF16 ? launch_dense<Bf16>(a, plan, part, stream)
                                       : launch_dense<F16>(a, plan, part, stream);
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
  const long long slot = (long long)e->I * e->H;
  const Moe8Plan p = moe8_plan(e, T, top_k);
  const void* const in[] = {x, ids, topk_weights, e->w13, e->w2, e->s13, e->s2, workspace};
  const long long in_bytes[] = {span(T, x_stride, e->H, 2), n * id_bytes, 4 * n, 2 * e->S * slot,
                                e->S * slot, 8LL * e->S * e->I, 4LL * e->S * e->H, p.bytes};
  for (int i = 0; i < 8; ++i)
    if (ranges_meet(in[i], in_bytes[i], out, out_bytes)) return -1;
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
  s.tiles = reinterpret_cast<int4*>(at + p.tiles);
  s.n_tiles = ints(p.n_tiles);
  s.tile_rows = p.tile_rows;
  s.chunk = sort_chunk(s.n);
  QuantizeArgs z = {x, x_stride, T, e->H, nullptr, bytes(p.q), e->H, floats(p.q_scale)};
  int rc = e->type == EXPERT_CACHE_BF16 ? launch_begin<Bf16>(s, z, stream)
                                        : launch_begin<F16>(s, z, stream);
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
  a.tiles = s.tiles;
  a.n_tiles = s.n_tiles;
  a.pairs = s.rows;
  a.k = top_k;
  a.out = floats(p.h);
  a.out_stride = e->I;
  a.scale_rows = T;
  a.whole_stores = true;  // H and I are multiples of 16
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
  a.scale_rows = (int)n;
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
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kMoveWaves * kWave), 0, stream, m);
  };
  // The launch before has written these rows: 6000 tokens, 8 of 64 slots of 2048 x 768 (393 MB), take
  // 472 us a layer past the caches and 491 through them; 4096, 4 of 16 of 2048 x 4096 (134 MB), 592 and
  // 596.
  const bool once = 4 * n * e->H >= kOnceBytes;
  if (e->type == EXPERT_CACHE_BF16)
    once ? launch(combine_k<float, Move::kOnce, Bf16>) : launch(combine_k<float, Move::kWhole, Bf16>);
  else
    once ? launch(combine_k<float, Move::kOnce, F16>) : launch(combine_k<float, Move::kWhole, F16>);
  return (int)hipGetLastError();
}

}  // extern "C"
