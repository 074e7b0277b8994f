// libexpertcache.so: C-ABI entry points (declared in include/expert_cache.h).
//
// Argument checks run on the host before any HIP call and return -1, exactly where the
// reference's C-ABI does (kernels/expert_cache.hip:596-598, :616-618, :631-634); otherwise
// each entry point launches one kernel on the caller's stream (two: the fused one for prefill
// chunks, and the refresh above 256 experts or slots, on large grids, or where the slot ids
// overwrite the routing ids) and returns hipGetLastError().
// The library keeps no state and allocates nothing.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../include/expert_cache.h"
#include "adapters.h"
#include "align.h"
#include "experts.h"
#include "gather.h"
#include "host.h"
#include "manage.h"
#include "refresh.h"
#include "route.h"

namespace ec {
namespace {

bool manage_args_bad(int E, int S, int max_inserts, int policy) {
  if (E <= 0 || S <= 0 || S > kMaxSlots || S > kSlotMask) return true;
  if (max_inserts < 0 || max_inserts > kMaxInserts) return true;
  if (policy < 0 || policy > 1) return true;
  return false;
}

// Waves of the policy step's workgroup: one thread for every expert and every slot, and a
// quarter of one for every id (prefill chunks route far more ids than there are experts).
int waves_for(int E, int S, int ids) {
  const int n = E > S ? E : S;
  const int threads = ids / 4 > n ? ids / 4 : n;
  int w = 1;
  while (w < 16 && w * kWave < threads) w *= 2;
  return w;
}

// Calls f with the number of waves as a compile-time constant.
template <class F>
void with_waves(int w, F&& f) {
  switch (w) {
    case 1: f(std::integral_constant<int, 1>()); break;
    case 2: f(std::integral_constant<int, 2>()); break;
    case 4: f(std::integral_constant<int, 4>()); break;
    case 8: f(std::integral_constant<int, 8>()); break;
    default: f(std::integral_constant<int, 16>()); break;
  }
}

template <int IDB, bool REMAP>
int launch_manage(const ManageArgs& a, hipStream_t stream) {
  if (a.E > kLdsExperts) {
    hipLaunchKernelGGL((manage_k<16, true, IDB, REMAP>), dim3(1), dim3(16 * kWave), 0, stream,
                       EC_STEP_ARGS(a), a);
  } else {
    with_waves(waves_for(a.E, a.S, a.mk), [&](auto w) {
      hipLaunchKernelGGL((manage_k<w(), false, IDB, REMAP>), dim3(1), dim3(w() * kWave), 0,
                         stream, EC_STEP_ARGS(a), a);
    });
  }
  return (int)hipGetLastError();
}

int launch_prefetch(const ManageArgs& a, hipStream_t stream) {
  if (a.E > kLdsExperts) {
    hipLaunchKernelGGL((prefetch_k<16, true>), dim3(1), dim3(16 * kWave), 0, stream, a);
  } else {
    with_waves(waves_for(a.E, a.S, a.mk), [&](auto w) {
      hipLaunchKernelGGL((prefetch_k<w(), false>), dim3(1), dim3(w() * kWave), 0, stream, a);
    });
  }
  return (int)hipGetLastError();
}

// Both layers share E and S, so one variant serves the two workgroups.
template <int IDB>
int launch_manage_prefetch(const ManageArgs& a, const ManageArgs& p, hipStream_t stream) {
  if (a.E > kLdsExperts) {
    hipLaunchKernelGGL((manage_prefetch_k<16, true, IDB>), dim3(2), dim3(16 * kWave), 0,
                       stream, a, p);
  } else {
    with_waves(waves_for(a.E, a.S, a.mk > p.mk ? a.mk : p.mk), [&](auto w) {
      hipLaunchKernelGGL((manage_prefetch_k<w(), false, IDB>), dim3(2), dim3(w() * kWave), 0,
                         stream, a, p);
    });
  }
  return (int)hipGetLastError();
}

int launch_fused(const ManageArgs& a, const AlignArgs& g, hipStream_t stream) {
  if (a.mk <= kFusedIds) {
    with_waves(waves_for(a.E, a.S, 4 * a.mk), [&](auto w) {
      hipLaunchKernelGGL((fused_k<w()>), dim3(1), dim3(w() * kWave), 0, stream,
                         EC_STEP_ARGS(a), a, g);
    });
    return (int)hipGetLastError();
  }
  // the fills get a workgroup per 16 K outputs a side
  const int fills = g.L / 16384 < 255 ? g.L / 16384 + 1 : 256;
  with_waves(waves_for(a.E, a.S, a.mk), [&](auto w) {
    hipLaunchKernelGGL((manage_defaults_k<w()>), dim3(1 + fills), dim3(w() * kWave), 0, stream,
                       EC_STEP_ARGS(a), a, g);
  });
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  hipLaunchKernelGGL(align_k, dim3((a.mk - 1) / 1024 + 1), dim3(1024), 0, stream,
                     static_cast<const int*>(a.ids), a.mk, a.E, a.S, a.table, g);
  return (int)hipGetLastError();
}

ManageArgs make_args(const void* ids, int mk, int E, int S, int max_distinct, int max_inserts,
                     int* table, int* map_cold, int* slot_expert, long long* slot_stamp,
                     unsigned char* routed, long long* step, int* miss, int* n_miss,
                     int policy, int decay, void* out) {
  ManageArgs a;
  a.ids = ids;
  a.mk = mk;
  a.E = E;
  a.S = S;
  a.max_distinct = max_distinct;
  a.max_inserts = max_inserts;
  a.table = table;
  a.map_cold = map_cold;
  a.slot_expert = slot_expert;
  a.slot_stamp = slot_stamp;
  a.routed = routed;
  a.step = step;
  a.miss = miss;
  a.n_miss = n_miss;
  a.policy = policy;
  a.decay = decay;
  a.out = out;
  return a;
}

// ---- operators over slots -----------------------------------------------------------------

template <class X, bool BIAS>
void launch_route_of(const RouteArgs& a, hipStream_t stream) {
  const dim3 grid((a.T - 1) / kRouteWaves + 1), block(kRouteWaves * kWave);
  if (a.E <= 64)
    hipLaunchKernelGGL((route_k<X, 1, BIAS>), grid, block, 0, stream, a);
  else if (a.E <= 128)
    hipLaunchKernelGGL((route_k<X, 2, BIAS>), grid, block, 0, stream, a);
  else if (a.E <= 256)
    hipLaunchKernelGGL((route_k<X, 4, BIAS>), grid, block, 0, stream, a);
  else if (a.E <= 512)
    hipLaunchKernelGGL((route_k<X, 8, BIAS>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((route_k<X, 16, BIAS>), grid, block, 0, stream, a);
}

template <class X>
int launch_route(const RouteArgs& a, hipStream_t stream) {
  if (a.bias)
    launch_route_of<X, true>(a, stream);
  else
    launch_route_of<X, false>(a, stream);
  return (int)hipGetLastError();
}

// Longest rows of weights: the bytes of 64 of them are counted in 32 bits.
constexpr int kMaxLength = 1 << 24;
// Most tokens of a call of expert_cache_route and expert_cache_adapt, and most outputs of an
// adapter: what a grid's second dimension (65535 workgroups) holds, with room.
constexpr int kMaxTokens = 1 << 21, kMaxOutputs = 1 << 21;

bool experts_bad(const expert_cache_experts* e, int T, int top_k) {
  if (e == nullptr || e->S <= 0 || e->H <= 0 || e->I <= 0) return true;
  if (e->type != EXPERT_CACHE_BF16 && e->type != EXPERT_CACHE_F16) return true;
  const bool byte = e->weights == EXPERT_CACHE_INT8 || e->weights == EXPERT_CACHE_E4M3;
  if (!byte && e->weights != e->type) return true;
  if (e->H % (byte ? 16 : 8) || e->I % (byte ? 16 : 8)) return true;
  if (e->H > kMaxLength || e->I > kMaxLength) return true;
  if (T < 0 || top_k <= 0 || top_k > kExpertsMaxK) return true;
  return (long long)T * top_k > kExpertsMaxPairs;
}

constexpr int kUpWaves = 4, kDownWaves = 8;
constexpr int kPairTiles = 4, kPairRows = kPairTiles * kTile;

// All figures below are us a call in a graph on MI355X.

// Above 8 tokens, experts of this many weights in w2 at most take the down projection of few
// tokens. It reads an expert once for every two of its tokens (from the L2 after the first), which
// costs more than the other's third launch once the experts are large. Few / not: 16 tokens,
// top-7 of 30 slots, 480 x 80 fp8 11.8 / 14.7; 9 tokens, top-6 of 186, 448 x 1152 float16 53 / 60;
// 16 tokens, top-8 of 128, 2048 x 1408 bf16 221 / 242; 14 tokens, top-10 of 24, 6240 x 1920 int8
// 301 / 221; 16 tokens, top-2 of 8, 4096 x 7168 bf16 304 / 236.
constexpr long kFewWeights = 1 << 22;
// Up to 8 tokens few is the better one or close: 8 tokens, few / not: top-8 of 64, 2048 x 768 int8
// 46 / 51; 2048 x 1408 bf16 124 / 139; top-2 of 8, 4096 x 7168 bf16 216 / 201.
constexpr int kAlwaysFew = 8;
constexpr int kComputeUnits = 256;
// A workgroup of experts_down_k takes 16 rows, or 8 where the compute unit with the most rows then
// has fewer: a unit's workgroups run side by side, so the call lasts as long as the fullest unit.
// 8 / 16 rows, one token on 2 bf16 experts of H x 2048, us: H 2048 (8 rows a unit, or 16) 14.5 /
// 16.5; 4112 (24 or 32) to 6144 3-9 % for 8 rows (5120 27.6 / 29.3). As many either way, 16 rows
// read longer runs: 3584 (16) 21.5 / 21.2, 7168 (32) 34.6 / 34.9; with 4 tokens on 16 int8 experts
// 71.9 / 67.8 and 126.8 / 120.9. Most against the rule, of shapes up to H 16384: one token on 2
// int8 experts, 8208 x 768 21.7 / 19.4 (8 taken); 4 tokens on 16 bf16 experts, 4080 x 7168 452 /
// 476 (16 taken).
bool eight_rows(int H) {
  return (H - 1) / 8 / kComputeUnits * 8 + 8 < (H - 1) / 16 / kComputeUnits * 16 + 16;
}
// Down projection of more tokens: the waves of a workgroup share a row's length only as far as
// rows alone do not make this many workgroups. Each for itself / four together: 32 tokens, top-8
// of 64, 2048 x 512 int8 (512 workgroups) 56 / 64; 2048 x 1408 bf16 184 / 192; but 64 tokens, top-4
// of 32, 2048 x 256 bf16 (256) 36.7 / 33.6; 24 tokens, top-2 of 8, 4096 x 7168 bf16 (128) 302 /
// 249.
constexpr int kPairGroups = 512;

// How a call of expert_cache_moe is split up, and where things are in its workspace.
struct MoePlan {
  bool few;
  int groups, down_groups, splits, k_waves;
  long lo, part, meta, arrived, bytes;
};
MoePlan moe_plan(int S, int H, int I, int T, int top_k) {
  const long n = (long)T * top_k;
  MoePlan p;
  p.few = T <= kAlwaysFew || (T <= kFewTokens && (long)H * I <= kFewWeights);
  const int units = (I - 1) / kUnit + 1;
  const long all = n < S ? n : S;
  p.k_waves = 1;
  while (p.k_waves < 4 && 2 * p.k_waves <= units &&
         all * ((H - 1) / (kPairRows * (4 / p.k_waves)) + 1) < kPairGroups)
    p.k_waves *= 2;
  p.groups = p.few ? (eight_rows(H) ? 1 : 2) : 2 * kPairTiles * (4 / p.k_waves);
  p.down_groups = (H - 1) / (8 * p.groups) + 1;
  p.splits = 1;
  // Workgroups that share their rows: as fill the device, a unit a wave at least. Shared / not: 16
  // tokens, top-8 of 64, 512 x 2048 bf16 113 / 174; one token on 2 experts, 1024 x 4096 bf16 15.8 /
  // 16.4; on 8, 1024 x 512 13.0 / 12.3. Up to twice as many are worth 9 % at best (one token, 4 of
  // 1280 x 5120 bf16 39.4 / 35.9) and cost as much (int8, 2048 x 768, one token 13.9 / 15.3).
  if (p.few) {
    const int want = kComputeUnits / p.down_groups, most = (int)n * units / kDownWaves;
    p.splits = want < 2 || most < 2 ? 1 : want < most ? want : most;
  }
  p.lo = 2 * n * I;
  p.part = 4 * n * I;
  p.meta = p.part + (p.few ? 32L * p.down_groups * p.splits * p.groups * kFewTokens : 4 * n * H);
  p.arrived = p.meta + (p.few ? n * (long)sizeof(ExpertsMeta) : 0);
  p.bytes = p.arrived + (p.few ? 4L * p.down_groups : 0);
  return p;
}

template <class X, class W, bool ONCE>
int launch_moe_of(const ExpertsArgs& a, int T, int groups, hipStream_t stream) {
  const int all = a.by_slot ? a.S : a.n;
  hipLaunchKernelGGL((experts_up_k<X, W, ONCE, kUpWaves, 2>), dim3((a.I - 1) / kTile + 1, all),
                     dim3(kUpWaves * kWave), 0, stream, a);
  int rc = (int)hipGetLastError();
  if (rc) return rc;
  const dim3 down(a.down_groups, a.few ? a.splits : all);
  if (a.few) {
    if (groups == 1)
      hipLaunchKernelGGL((experts_down_k<X, W, ONCE, 1, kDownWaves, 3>), down,
                         dim3(kDownWaves * kWave), 0, stream, a);
    else
      hipLaunchKernelGGL((experts_down_k<X, W, ONCE, 2, kDownWaves, 3>), down,
                         dim3(kDownWaves * kWave), 0, stream, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((experts_pairs_k<W, ONCE, 4, kPairTiles, 1>), down, dim3(4 * kWave), 0,
                     stream, a);
  rc = (int)hipGetLastError();
  if (rc) return rc;
  hipLaunchKernelGGL((experts_sum_k<X>), dim3((a.H - 1) / 1024 + 1, T), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

// Weights whose rows are whole lines of 128 bytes are read past the caches: us past / through
// them: one token on 2 bf16 experts of 176 MB 62.8 / 67.0, on 8 fp8 experts of 44 MB 59.8 / 65.7;
// where a load's lines are shared with another one it costs: 5 tokens, H 1048, float16 23.7 / 21.1.
template <class X, class W>
int launch_moe(const ExpertsArgs& a, int T, int groups, hipStream_t stream) {
  const uintptr_t lines = reinterpret_cast<uintptr_t>(a.w13) | reinterpret_cast<uintptr_t>(a.w2) |
                          (uintptr_t)a.H * sizeof(W) | (uintptr_t)a.I * sizeof(W);
  return lines % 128 ? launch_moe_of<X, W, false>(a, T, groups, stream)
                     : launch_moe_of<X, W, true>(a, T, groups, stream);
}

bool adapters_bad(const expert_cache_adapters* l, int T) {
  if (l == nullptr || l->S <= 0 || l->O <= 0 || l->H <= 0 || l->R <= 0) return true;
  if (T < 0 || T > kMaxTokens || l->O > kMaxOutputs) return true;
  if (l->type != EXPERT_CACHE_BF16 && l->type != EXPERT_CACHE_F16) return true;
  return l->H % 8 || l->R % 8 || l->R > kAdapterMaxRank || l->H > kMaxLength;
}

constexpr int kAdapterWaves = 4;
// Up to this many tokens (few) every adapter of a tile of 16 has workgroups of its own; above
// (many) 64 tokens go through their adapters one after another. Few reads an adapter once a
// tile, many works through a tile of 64 once an adapter, and how many adapters a tile has is on
// the device only. Few / many, us in a graph, H and O 4096, one adapter and 64: 64 tokens, rank
// 16 9.4 / 15.0 and 13.2 / 142; 256 tokens, rank 16 17.2 / 15.7 and 24 / 142, rank 64 33 / 18.3
// and 76 / 191; 320 tokens, rank 16 16.8 / 16.0 and 32 / 142, rank 64 40 / 19.0 and 97 / 189;
// 1024 tokens, rank 16 32 / 18.6 and 76 / 146, rank 64 95 / 23 and 252 / 199. Steps of more than
// 256 tokens are prompts, where neighbours share an adapter.
constexpr int kAdapterFewTokens = 256;
// Up to this many tiles of 16 tokens a tile's adapters are shared out to four workgroups of
// adapters_expand_k. Four / one, us in a graph, H and O 4096: 16 tokens, rank 64, 64 adapters 14.8
// / 20.6, two 13.8 / 15.2; 33 tokens, 64 adapters 21.0 / 24.6, two 19.4 / 16.0; 64 tokens, rank 16,
// 64 adapters 13.4 / 13.5; but 128 tokens 21.9 / 18.0, 256 tokens 36 / 26.
constexpr int kAdapterPartTiles = 4;

// Workgroups that share the hidden length of a tile's product: as fill the device, a unit a wave
// at least. Half as many for many tokens: 4096 tokens, rank 64 39.3 and not 37.7 us with one
// adapter, 1024 tokens 21.1 and not 23.4, with 64 adapters 242 and not 200.
int adapter_splits(int T, int H) {
  const bool few = T <= kAdapterFewTokens;
  const int tiles = (T - 1) / (few ? kTile : kManyTokens) + 1;
  const int units = (H - 1) / kUnit + 1, waves = few ? kAdapterWaves : 2;
  const int most = (units - 1) / waves + 1, want = (few ? 512 : 256) / tiles;
  return want < 1 ? 1 : want < most ? want : most;
}

template <class X>
int launch_adapt(const AdaptersArgs& a, hipStream_t stream) {
  constexpr int W = kAdapterWaves;
  const bool few = a.T <= kAdapterFewTokens;
  const dim3 block(W * kWave);
  if (few) {
    const int tiles = (a.T - 1) / kTile + 1;
    const int parts = tiles <= kAdapterPartTiles ? 4 : 1;
    // Tiles of 16 ranks a workgroup takes at once, and workgroups that share the ranks. One / two
    // / four tiles, us in a graph, H and O 4096: 16 tokens with 64 adapters, rank 16 8.6 / - / 9.5,
    // rank 32 13.0 / 11.8 / 12.7, rank 64 13.1 / 13.2 / 15.1; one token, rank 64 9.6 / 9.6 / 11.6;
    // but 64 tokens, 64 adapters 28.6 / 27.0 / 25.5. Ranks shared / one workgroup after another:
    // one token, rank 256 24.4 / 34.8; 256 tokens, rank 256, 64 adapters 274 / 278.
    const int rows = a.R <= 16 ? 1 : a.R <= 32 || (tiles == 1 && a.R <= 64) ? 2 : 4;
    const dim3 shrink(tiles, kTile, a.splits * ((a.R - 1) / (16 * rows) + 1));
    if (rows == 1)
      hipLaunchKernelGGL((adapters_shrink_k<X, W, 1>), shrink, block, 0, stream, a);
    else if (rows == 2)
      hipLaunchKernelGGL((adapters_shrink_k<X, W, 2>), shrink, block, 0, stream, a);
    else
      hipLaunchKernelGGL((adapters_shrink_k<X, W, 4>), shrink, block, 0, stream, a);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL((adapters_expand_k<X, W, 4>), dim3(tiles, (a.O - 1) / (16 * W) + 1, parts),
                       block, 0, stream, a);
    return (int)hipGetLastError();
  }
  const int tiles = (a.T - 1) / kManyTokens + 1;
  const dim3 grid(tiles, a.splits), wide(8 * kWave);
  hipLaunchKernelGGL((adapters_shrink_many_k<X>), grid, wide, 0, stream, a);
  const int rc = (int)hipGetLastError();
  if (rc) return rc;
  hipLaunchKernelGGL((adapters_expand_many_k<X, 8>), dim3((a.O - 1) / (64 * 8) + 1, tiles), wide, 0,
                     stream, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace ec

using namespace ec;

extern "C" {

int expert_cache_manage(const int* topk_ids, int mk, int E, int S, int max_distinct,
                        int max_inserts, int* table, int* map_cold, int* slot_expert,
                        long long* slot_stamp, unsigned char* routed, long long* step,
                        int* miss, int* n_miss, int policy, int decay, hipStream_t stream) {
  if (manage_args_bad(E, S, max_inserts, policy)) return -1;
  const ManageArgs a = make_args(topk_ids, mk, E, S, max_distinct, max_inserts, table, map_cold,
                                 slot_expert, slot_stamp, routed, step, miss, n_miss, policy,
                                 decay, nullptr);
  return launch_manage<4, false>(a, stream);
}

int expert_cache_manage_remap(const void* ids, int id_bytes, int mk, int E, int S,
                              int max_distinct, int max_inserts, int* table, int* map_cold,
                              int* slot_expert, long long* slot_stamp, unsigned char* routed,
                              long long* step, int* miss, int* n_miss, int policy, int decay,
                              void* out, hipStream_t stream) {
  if (manage_args_bad(E, S, max_inserts, policy)) return -1;
  if (id_bytes != 4 && id_bytes != 8) return -1;
  if (mk > 0 && out == nullptr) return -1;
  const ManageArgs a = make_args(ids, mk, E, S, max_distinct, max_inserts, table, map_cold,
                                 slot_expert, slot_stamp, routed, step, miss, n_miss, policy,
                                 decay, out);
  return id_bytes == 8 ? launch_manage<8, true>(a, stream) : launch_manage<4, true>(a, stream);
}

int expert_cache_prefetch(const int* pred_ids, int mk, int E, int S, int max_inserts,
                          int* table, int* map_cold, int* slot_expert, long long* slot_stamp,
                          unsigned char* routed, int* miss, int* n_miss, hipStream_t stream) {
  if (manage_args_bad(E, S, max_inserts, 0) || mk < 0) return -1;
  // max_distinct = E: a prediction never reads through; no step counter is touched
  const ManageArgs a = make_args(pred_ids, mk, E, S, E, max_inserts, table, map_cold,
                                 slot_expert, slot_stamp, routed, nullptr, miss, n_miss, 0, 0,
                                 nullptr);
  return launch_prefetch(a, stream);
}

int expert_cache_manage_remap_prefetch(
    const void* ids, int id_bytes, int mk, int E, int S, int max_distinct, int max_inserts,
    int* table, int* map_cold, int* slot_expert, long long* slot_stamp, unsigned char* routed,
    long long* step, int* miss, int* n_miss, int policy, int decay, void* out,
    const int* pred_ids, int pk, int pf_max_inserts, int* pf_table, int* pf_map_cold,
    int* pf_slot_expert, long long* pf_slot_stamp, unsigned char* pf_routed, int* pf_miss,
    int* pf_n_miss, hipStream_t stream) {
  if (manage_args_bad(E, S, max_inserts, policy)) return -1;
  if (id_bytes != 4 && id_bytes != 8) return -1;
  if (mk > 0 && out == nullptr) return -1;
  if (manage_args_bad(E, S, pf_max_inserts, 0) || pk < 0) return -1;
  // the two workgroups run unordered: the layers must not share any array
  const long long e4 = 4LL * E, s4 = 4LL * S;
  if (ranges_meet(table, e4, pf_table, e4) || ranges_meet(map_cold, e4, pf_map_cold, e4) ||
      ranges_meet(slot_expert, s4, pf_slot_expert, s4) ||
      ranges_meet(slot_stamp, 2 * s4, pf_slot_stamp, 2 * s4) ||
      ranges_meet(routed, E, pf_routed, E) ||
      ranges_meet(miss, 8LL * max_inserts, pf_miss, 8LL * pf_max_inserts) ||
      ranges_meet(n_miss, 4, pf_n_miss, 4))
    return -1;
  const ManageArgs a = make_args(ids, mk, E, S, max_distinct, max_inserts, table, map_cold,
                                 slot_expert, slot_stamp, routed, step, miss, n_miss, policy,
                                 decay, out);
  const ManageArgs p = make_args(pred_ids, pk, E, S, E, pf_max_inserts, pf_table, pf_map_cold,
                                 pf_slot_expert, pf_slot_stamp, pf_routed, nullptr, pf_miss,
                                 pf_n_miss, 0, 0, nullptr);
  return id_bytes == 8 ? launch_manage_prefetch<8>(a, p, stream)
                       : launch_manage_prefetch<4>(a, p, stream);
}

int expert_cache_remap(const void* ids, int n, int id_bytes, const int* table, int E,
                       void* out, hipStream_t stream) {
  if (E <= 0 || n < 0 || (id_bytes != 4 && id_bytes != 8)) return -1;
  if (n == 0) return 0;
  const int blocks = (n + 255) / 256 < 1024 ? (n + 255) / 256 : 1024;
  if (id_bytes == 8)
    hipLaunchKernelGGL((remap_k<8>), dim3(blocks), dim3(256), 0, stream, ids, n, table, E, out);
  else
    hipLaunchKernelGGL((remap_k<4>), dim3(blocks), dim3(256), 0, stream, ids, n, table, E, out);
  return (int)hipGetLastError();
}

int expert_cache_fused(const int* topk_ids, int mk, int E, int S, int max_distinct,
                       int max_inserts, int* table, int* map_cold, int* slot_expert,
                       long long* slot_stamp, unsigned char* routed, long long* step,
                       int* miss, int* n_miss, int bs, int L, int NB, int* sorted_hot,
                       int* eids_hot, int* npad_hot, int* sorted_cold, int* eids_cold,
                       int* npad_cold, hipStream_t stream) {
  if (E <= 0 || E > kMaxAlignExperts || S <= 0 || S > kMaxSlots || S > kSlotMask) return -1;
  if (bs <= 0 || L <= 0 || NB <= 0 || mk < 0) return -1;
  if (max_inserts < 0 || max_inserts > kMaxAlignExperts) return -1;
  const ManageArgs a = make_args(topk_ids, mk, E, S, max_distinct, max_inserts, table, map_cold,
                                 slot_expert, slot_stamp, routed, step, miss, n_miss, 0, 0,
                                 nullptr);
  AlignArgs g;
  set_block_size(g, bs);
  g.L = L;
  g.NB = NB;
  g.sorted_hot = sorted_hot;
  g.eids_hot = eids_hot;
  g.npad_hot = npad_hot;
  g.sorted_cold = sorted_cold;
  g.eids_cold = eids_cold;
  g.npad_cold = npad_cold;
  return launch_fused(a, g, stream);
}

int expert_cache_refresh(const expert_cache_layer* c, const void* ids, int id_bytes, int mk,
                         void* out, hipStream_t stream) {
  if (c == nullptr || c->arrived == nullptr || mk < 0) return -1;
  if (manage_args_bad(c->E, c->S, c->S, c->policy)) return -1;
  if (id_bytes != 4 && id_bytes != 8) return -1;
  if (mk > 0 && out == nullptr) return -1;
  GatherArgs g;
  if (c->n_miss == nullptr || !gather_plan(c->dst, c->src, c->bytes, c->chunks, c->lanes, g))
    return -1;
  const ManageArgs a = make_args(ids, mk, c->E, c->S, c->E < mk ? c->E : mk, c->S, c->table,
                                 c->map_cold, c->slot_expert, c->slot_stamp, c->routed, c->step,
                                 c->miss, c->n_miss, c->policy, c->decay, out);
  const dim3 grid(c->chunks, c->lanes), block(kGatherThreads);
  // Of one launch's workgroups the first may write `out` while others still read `ids`, so
  // ids that are rewritten in place take two launches.
  const long long id_range = (long long)mk * id_bytes;
  if (c->E <= kGatherThreads && c->S <= kGatherThreads &&
      (long long)c->chunks * c->lanes <= kRefreshGroups &&
      !ranges_meet(ids, id_range, out, id_range)) {
    if (id_bytes == 8)
      hipLaunchKernelGGL((refresh_k<8>), grid, block, 0, stream, EC_STEP_ARGS(a), a, g,
                         c->arrived);
    else
      hipLaunchKernelGGL((refresh_k<4>), grid, block, 0, stream, EC_STEP_ARGS(a), a, g,
                         c->arrived);
    return (int)hipGetLastError();
  }
  const int rc = id_bytes == 8 ? launch_manage<8, true>(a, stream)
                               : launch_manage<4, true>(a, stream);
  if (rc) return rc;
  hipLaunchKernelGGL((gather_k<kGatherUnroll, true, false, false>), grid, block, 0, stream, g,
                     c->miss, c->n_miss, nullptr);
  return (int)hipGetLastError();
}

int expert_cache_gather(void* d0, const void* s0, long b0, void* d1, const void* s1, long b1,
                        void* d2, const void* s2, long b2, void* d3, const void* s3, long b3,
                        void* d4, const void* s4, long b4, void* d5, const void* s5, long b5,
                        const int* miss, const int* n_miss, int chunks, int lanes,
                        hipStream_t stream) {
  void* const dst[kGatherBufs] = {d0, d1, d2, d3, d4, d5};
  const void* const src[kGatherBufs] = {s0, s1, s2, s3, s4, s5};
  const long bytes[kGatherBufs] = {b0, b1, b2, b3, b4, b5};
  GatherArgs g;
  if (n_miss == nullptr || !gather_plan(dst, src, bytes, chunks, lanes, g)) return -1;
  hipLaunchKernelGGL((gather_k<kGatherUnroll, true, false, false>), dim3(chunks, lanes),
                     dim3(kGatherThreads), 0, stream, g, miss, n_miss, nullptr);
  return (int)hipGetLastError();
}

int expert_cache_gather_live(void* d0, const void* s0, long b0, void* d1, const void* s1,
                             long b1, void* d2, const void* s2, long b2, void* d3,
                             const void* s3, long b3, void* d4, const void* s4, long b4,
                             void* d5, const void* s5, long b5, const int* miss,
                             const int* n_miss, const int* slot_expert, int chunks, int lanes,
                             hipStream_t stream) {
  void* const dst[kGatherBufs] = {d0, d1, d2, d3, d4, d5};
  const void* const src[kGatherBufs] = {s0, s1, s2, s3, s4, s5};
  const long bytes[kGatherBufs] = {b0, b1, b2, b3, b4, b5};
  GatherArgs g;
  if (n_miss == nullptr || slot_expert == nullptr) return -1;
  if (!gather_plan(dst, src, bytes, chunks, lanes, g)) return -1;
  hipLaunchKernelGGL((gather_k<kGatherUnroll, true, false, true>), dim3(chunks, lanes),
                     dim3(kGatherThreads), 0, stream, g, miss, n_miss, slot_expert);
  return (int)hipGetLastError();
}

int expert_cache_route(const void* logits, int type, long row_stride, const float* bias, int T,
                       int E, int top_k, int scoring, int groups, int topk_groups,
                       int renormalize, float scale, float* weights, void* ids, int id_bytes,
                       hipStream_t stream) {
  if (T < 0 || T > kMaxTokens) return -1;
  if (E <= 0 || E > kRouteMaxExperts || (row_stride < E && T > 1)) return -1;
  if (scoring < 0 || scoring > 1 || (id_bytes != 4 && id_bytes != 8)) return -1;
  if (groups < 1 || groups > kRouteMaxGroups || E % groups) return -1;
  if (topk_groups < 1 || topk_groups > groups) return -1;
  if (top_k < 1 || top_k > kRouteMaxK || top_k > topk_groups * (E / groups)) return -1;
  if (type < EXPERT_CACHE_F32 || type > EXPERT_CACHE_F16) return -1;
  if (T == 0) return 0;
  if (logits == nullptr || weights == nullptr || ids == nullptr) return -1;
  const long long n = (long long)T * top_k, read = ((T - 1LL) * row_stride + E) *
                                                   (type == EXPERT_CACHE_F32 ? 4 : 2);
  if (ranges_meet(logits, read, weights, 4 * n) || ranges_meet(logits, read, ids, id_bytes * n) ||
      ranges_meet(weights, 4 * n, ids, id_bytes * n))
    return -1;
  if (bias && (ranges_meet(bias, 4LL * E, weights, 4 * n) ||
               ranges_meet(bias, 4LL * E, ids, id_bytes * n)))
    return -1;
  const RouteArgs a = {logits,       row_stride,       bias,          T,     E,       top_k, groups,
                       topk_groups,  scoring == 1,     renormalize != 0, id_bytes == 8, scale,
                       weights,      ids};
  if (type == EXPERT_CACHE_F32) return launch_route<float>(a, stream);
  return type == EXPERT_CACHE_BF16 ? launch_route<Bf16>(a, stream) : launch_route<F16>(a, stream);
}

int expert_cache_moe_workspace(const expert_cache_experts* e, int T, int top_k, long* bytes) {
  if (bytes == nullptr || experts_bad(e, T, top_k)) return -1;
  *bytes = moe_plan(e->S, e->H, e->I, T, top_k).bytes;
  return 0;
}

int expert_cache_moe(const expert_cache_experts* e, const void* x, long x_stride,
                     const float* topk_weights, const void* ids, int id_bytes, int T, int top_k,
                     void* out, long out_stride, void* workspace, hipStream_t stream) {
  if (experts_bad(e, T, top_k) || (id_bytes != 4 && id_bytes != 8)) return -1;
  if (T == 0) return 0;
  if (e->w13 == nullptr || e->w2 == nullptr || !aligned16(e->w13) || !aligned16(e->w2)) return -1;
  if (e->weights >= EXPERT_CACHE_INT8 &&
      (e->s13 == nullptr || e->s2 == nullptr || !aligned16(e->s13) || !aligned16(e->s2)))
    return -1;
  if (x == nullptr || !aligned16(x) || (T > 1 && (x_stride % 8 || x_stride < e->H))) return -1;
  if (out == nullptr || (out_stride < e->H && T > 1)) return -1;
  if (topk_weights == nullptr || ids == nullptr) return -1;
  if (workspace == nullptr || !aligned16(workspace)) return -1;
  // the last launch reads the ids and weights again while it writes the result
  const long long out_bytes = 2 * ((T - 1LL) * out_stride + e->H), n = (long long)T * top_k;
  if (ranges_meet(x, 2 * ((T - 1LL) * x_stride + e->H), out, out_bytes) ||
      ranges_meet(ids, n * id_bytes, out, out_bytes) ||
      ranges_meet(topk_weights, 4 * n, out, out_bytes))
    return -1;
  ExpertsArgs a;
  a.x = x;
  a.x_stride = x_stride;
  a.w13 = e->w13;
  a.w2 = e->w2;
  a.s13 = e->s13;
  a.s2 = e->s2;
  a.probs = topk_weights;
  a.ids = ids;
  a.n = T * top_k;
  a.k = top_k;
  a.S = e->S;
  a.H = e->H;
  a.I = e->I;
  a.wide = id_bytes == 8;
  // a workgroup for every slot where those are fewer than pairs: 32 tokens, top-8 of 128, 2048 x
  // 768 bf16 199 us, 223 with one for every pair; 64 tokens, top-4 of 32, 2048 x 256 34.4 and 45.0
  a.by_slot = a.n > a.S;
  const MoePlan plan = moe_plan(e->S, e->H, e->I, T, top_k);
  a.few = plan.few;
  a.down_groups = plan.down_groups;
  a.splits = plan.splits;
  a.k_waves = plan.k_waves;
  char* const at = static_cast<char*>(workspace);
  a.hi = reinterpret_cast<Bf16*>(at);
  a.lo = reinterpret_cast<Bf16*>(at + plan.lo);
  a.part = reinterpret_cast<float*>(at + plan.part);
  a.meta = reinterpret_cast<ExpertsMeta*>(at + plan.meta);
  a.arrived = reinterpret_cast<int*>(at + plan.arrived);
  a.out = out;
  a.out_stride = out_stride;
  if (e->type == EXPERT_CACHE_BF16) {
    if (e->weights == EXPERT_CACHE_INT8) return launch_moe<Bf16, int8_t>(a, T, plan.groups, stream);
    if (e->weights == EXPERT_CACHE_E4M3) return launch_moe<Bf16, E4m3>(a, T, plan.groups, stream);
    return launch_moe<Bf16, Bf16>(a, T, plan.groups, stream);
  }
  if (e->weights == EXPERT_CACHE_INT8) return launch_moe<F16, int8_t>(a, T, plan.groups, stream);
  if (e->weights == EXPERT_CACHE_E4M3) return launch_moe<F16, E4m3>(a, T, plan.groups, stream);
  return launch_moe<F16, F16>(a, T, plan.groups, stream);
}

int expert_cache_adapt_workspace(const expert_cache_adapters* l, int T, long* bytes) {
  if (bytes == nullptr || adapters_bad(l, T)) return -1;
  *bytes = T == 0 ? 0 : 4L * adapter_splits(T, l->H) * T * l->R;
  return 0;
}

int expert_cache_adapt(const expert_cache_adapters* l, const void* x, long x_stride,
                       const void* ids, int id_bytes, int T, const void* base,
                       long base_stride, void* out, long out_stride, void* workspace,
                       hipStream_t stream) {
  if (adapters_bad(l, T) || (id_bytes != 4 && id_bytes != 8)) return -1;
  if (T == 0) return 0;
  if (l->a == nullptr || l->b == nullptr || !aligned16(l->a) || !aligned16(l->b)) return -1;
  if (x == nullptr || !aligned16(x) || (T > 1 && (x_stride % 8 || x_stride < l->H))) return -1;
  if (base == nullptr || out == nullptr || ids == nullptr) return -1;
  if ((base_stride < l->O || out_stride < l->O) && T > 1) return -1;
  if (workspace == nullptr || !aligned16(workspace)) return -1;
  const long long out_bytes = 2 * ((T - 1LL) * out_stride + l->O);
  const bool in_place = out == base && (out_stride == base_stride || T == 1);
  if (!in_place && ranges_meet(base, 2 * ((T - 1LL) * base_stride + l->O), out, out_bytes))
    return -1;
  if (ranges_meet(x, 2 * ((T - 1LL) * x_stride + l->H), out, out_bytes) ||
      ranges_meet(ids, (long long)T * id_bytes, out, out_bytes))
    return -1;
  AdaptersArgs a;
  a.x = x;
  a.x_stride = x_stride;
  a.a = l->a;
  a.b = l->b;
  a.scales = l->scales;
  a.ids = ids;
  a.base = base;
  a.base_stride = base_stride;
  a.out = out;
  a.out_stride = out_stride;
  a.T = T;
  a.S = l->S;
  a.H = l->H;
  a.O = l->O;
  a.R = l->R;
  a.splits = adapter_splits(T, l->H);
  a.wide = id_bytes == 8;
  a.aligned = aligned16(base) && aligned16(out) &&
              (T == 1 || (base_stride % 8 == 0 && out_stride % 8 == 0));
  a.v = static_cast<float*>(workspace);
  return l->type == EXPERT_CACHE_BF16 ? launch_adapt<Bf16>(a, stream)
                                      : launch_adapt<F16>(a, stream);
}

}  // extern "C"
