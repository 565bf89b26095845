// Gated products of the chosen experts:
//   out[t] = sum_j w[t][j] down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = experts[t][j].
//
// Few pairs (token, choice; up to few_pairs): the experts' weights are read once for
// each pair by ordinary warps, two launches in all (expert_rows_gate_up, expert_rows_down).
//
// More pairs: the tensor cores, three or four launches.
//  * expert_plan sorts the pairs by expert (stable): offsets[E + 1], order[pairs].  A few
//    pairs are sorted by each block of the first product instead.
//  * expert_products<gate-up> and <down>: grouped matrix products on pairs of CTAs
//    (tcgen05, cta_group::2), persistent and warp-specialised.  The weights are the M
//    operand (128 rows a CTA) and an expert's rows the N operand (32 to 256 in steps of
//    32), so an expert with few rows costs few columns, and a batch of single tokens
//    streams each expert's weights once through tiles 32 columns wide.
//    - The rows of x are gathered by TMA (tile::gather4) through `order`: no sorted copy.
//      Four threads of four warps issue the copies, with their rows in registers.
//    - A CTA's 128 weight rows of the first product are 4 x (16 gate rows, 16 up rows),
//      one TMA box of a five-dimensional map, so that the gate and up values of a feature
//      sit in lanes l and l + 16 of one warp: one shuffle a value pair, then
//      silu(gate) * up, rounded to the operands' type for the second product.
//    - The second product's values, one pair's share of an output, stay FP32: they are terms of
//      a sum, and neighbouring features may be orders of magnitude apart.  8192 tokens x 8, hidden
//      2048: second product 268 us and combine 92 us, where 16-bit integers under one scale for 32
//      features (0.5 GB less traffic) took 258 and 66.
//  * expert_combine adds a token's shares in the order of its choices.
// Every wait is bounded (200 ms); a role that gives up records why in a device word
// (ttn_expert_mlp_fault) and the pair frees its TMEM and returns.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rows.cuh"
#include "tcgen05.cuh"

namespace ttn {
namespace {

using namespace tc;

constexpr uint32_t kAll = 0xffffffffu;
constexpr int kMaxExperts = 1024;
constexpr int kMaxChoices = 32;

struct ExpertArgs {
  const uint16_t* x;
  const int32_t* ids;
  const float* weights;
  const uint16_t *gate_up, *down;
  uint16_t* out;
  int64_t x_stride, out_stride, tokens;
  int hidden, inner, experts, top_k;
};

__device__ __forceinline__ float silu_gate(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

// ------------------------------------------------------------ few pairs
//
// A block takes 16 gated features of one pair, a warp two of them: four weight rows
// (2 gate, 2 up) against x, 16 bytes a lane and row at a time.  The activations stay
// FP32 (h: [pairs][inner]).
constexpr int kRowsThreads = 256;
constexpr int kRowsFeatures = 2;  // gated features of one warp
constexpr int kRowsBlock = kRowsThreads / 32 * kRowsFeatures;

template <typename T>
__global__ void __launch_bounds__(kRowsThreads) expert_rows_gate_up(ExpertArgs a, float* __restrict__ h, int blocks) {
  pdl_trigger();  // started after all earlier work: only expert_rows_down overlaps it
  const int64_t pair = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int f0 = (int)(blockIdx.x % blocks) * kRowsBlock + warp * kRowsFeatures;
  const int e = a.ids[pair];
  if ((unsigned)e >= (unsigned)a.experts || f0 >= a.inner) return;  // inner % 16 == 0: both features or none
  const uint16_t* x = a.x + pair / a.top_k * a.x_stride;
  const uint16_t* w = a.gate_up + ((int64_t)e * 2 * a.inner + f0) * a.hidden;
  const int64_t up = (int64_t)a.inner * a.hidden;
  float acc[2 * kRowsFeatures] = {};
#pragma unroll 2
  for (int k = lane * 8; k < a.hidden; k += 256) {
    uint4 v[2 * kRowsFeatures];
#pragma unroll
    for (int i = 0; i < kRowsFeatures; ++i) {
      v[2 * i] = __ldg(reinterpret_cast<const uint4*>(w + (int64_t)i * a.hidden + k));
      v[2 * i + 1] = __ldg(reinterpret_cast<const uint4*>(w + up + (int64_t)i * a.hidden + k));
    }
    float xs[8];
    T::unpack(__ldg(reinterpret_cast<const uint4*>(x + k)), xs);
#pragma unroll
    for (int i = 0; i < 2 * kRowsFeatures; ++i) {
      float ws[8];
      T::unpack(v[i], ws);
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i] = fmaf(ws[j], xs[j], acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2 * kRowsFeatures; ++i)
#pragma unroll
    for (int d = 16; d; d >>= 1) acc[i] += __shfl_xor_sync(kAll, acc[i], d);
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < kRowsFeatures; ++i) h[pair * a.inner + f0 + i] = silu_gate(acc[2 * i], acc[2 * i + 1]);
  }
}

// A block takes kDownRows outputs of one token, each warp the pairs warp, warp + warps, ..
// of it; the weighted sum over the pairs is taken in their order.
constexpr int kDownRows = 4;
constexpr int kDownWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kDownWarps * 32) expert_rows_down(ExpertArgs a, const float* __restrict__ h,
                                                                    int blocks) {
  __shared__ float part[kMaxChoices][kDownRows];
  const int64_t token = blockIdx.x / blocks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d0 = (int)(blockIdx.x % blocks) * kDownRows;  // hidden % 8 == 0: all rows exist
  bool waited = false;
  for (int j = warp; j < a.top_k; j += blockDim.x >> 5) {
    const int64_t pair = token * a.top_k + j;
    const int e = a.ids[pair];
    float acc[kDownRows] = {};
    const bool live = (unsigned)e < (unsigned)a.experts;
    const uint16_t* w = a.down + ((int64_t)(live ? e : 0) * a.hidden + d0) * a.inner;
    const float* hp = h + pair * a.inner;
    uint4 next[kDownRows];
    auto fetch = [&](int k) {
#pragma unroll
      for (int i = 0; i < kDownRows; ++i)
        next[i] = live && k < a.inner ? __ldg(reinterpret_cast<const uint4*>(w + (int64_t)i * a.inner + k))
                                      : make_uint4(0, 0, 0, 0);
    };
    fetch(lane * 8);
    if (!waited) {  // the weights are read while expert_rows_gate_up still runs, its h is not
      pdl_wait();
      waited = true;
    }
    if (live) {
#pragma unroll 2
      for (int k = lane * 8; k < a.inner; k += 256) {
        uint4 v[kDownRows];
#pragma unroll
        for (int i = 0; i < kDownRows; ++i) v[i] = next[i];
        fetch(k + 256);
        const float4 h0 = *reinterpret_cast<const float4*>(hp + k), h1 = *reinterpret_cast<const float4*>(hp + k + 4);
        const float hs[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
#pragma unroll
        for (int i = 0; i < kDownRows; ++i) {
          float ws[8];
          T::unpack(v[i], ws);
#pragma unroll
          for (int q = 0; q < 8; ++q) acc[i] = fmaf(ws[q], hs[q], acc[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kDownRows; ++i)
#pragma unroll
      for (int d = 16; d; d >>= 1) acc[i] += __shfl_xor_sync(kAll, acc[i], d);
    if (lane == 0) {
      const float weight = live ? a.weights[pair] : 0.0f;
#pragma unroll
      for (int i = 0; i < kDownRows; ++i) part[j][i] = live ? weight * acc[i] : 0.0f;
    }
  }
  __syncthreads();
  if (threadIdx.x < kDownRows) {
    float sum = 0.0f;
    for (int j = 0; j < a.top_k; ++j) sum += part[j][threadIdx.x];
    a.out[token * a.out_stride + d0 + threadIdx.x] = T::round(sum);
  }
}

// ------------------------------------------------------------ tensor cores

__device__ uint32_t g_expert_fault;

// Test hook (ttn_expert_mlp_test_withhold_copies): the next call's first product on the
// tensor cores issues no operand copy.
std::atomic<bool> g_withhold_next_products{false};

// offsets[e]: pairs of experts below e; order: the pairs, by expert, then by number.  One
// block an expert, each reading all ids twice (they are few and in L2), 128 a warp and load:
// no block waits for another.  The reading grows with experts x pairs: on a B200 65,536 ids of 64
// experts take 12 us and of 256 experts 19 us, 32,768 ids of 1024 experts 27 us.
constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanBatch = 4;  // loads in flight
__global__ void __launch_bounds__(kPlanThreads) expert_plan(const int32_t* __restrict__ ids, int pairs, int experts,
                                                            int vec, int32_t* __restrict__ offsets,
                                                            int32_t* __restrict__ order) {
  __shared__ int below[kPlanWarps], mine[kPlanWarps];
  pdl_trigger();
  pdl_wait();
  const int e = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int chunk = (pairs + kPlanWarps * 128 - 1) / (kPlanWarps * 128) * 128;  // ids of one warp
  const int first = warp * chunk, last = min(first + chunk, pairs);            // pairs < 2^23
  auto load = [&](int i0, int (&id)[4]) {
    const int i = i0 + lane * 4;
    if (vec && i + 4 <= last) {
      const int4 v = __ldg(reinterpret_cast<const int4*>(ids + i));
      id[0] = v.x, id[1] = v.y, id[2] = v.z, id[3] = v.w;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) id[q] = i + q < last ? ids[i + q] : -1;
    }
  };
  int less = 0, equal = 0;
  for (int i0 = first; i0 < last; i0 += 128 * kPlanBatch) {
    int id[kPlanBatch][4];
#pragma unroll
    for (int u = 0; u < kPlanBatch; ++u) load(i0 + u * 128, id[u]);
#pragma unroll
    for (int u = 0; u < kPlanBatch; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) less += (unsigned)id[u][q] < (unsigned)e, equal += id[u][q] == e;
  }
  less = __reduce_add_sync(kAll, less);
  equal = __reduce_add_sync(kAll, equal);
  if (lane == 0) below[warp] = less, mine[warp] = equal;
  __syncthreads();
  static_assert(kPlanWarps == 32, "one lane a warp");
  const int total = __reduce_add_sync(kAll, below[lane]);
  int at = total + __reduce_add_sync(kAll, lane < warp ? mine[lane] : 0);
  const int all = total + __reduce_add_sync(kAll, mine[lane]);
  if (threadIdx.x == 0) {
    offsets[e] = total;
    if (e == experts - 1) offsets[experts] = all;
  }
  if (!equal) return;
  const uint32_t before = (1u << lane) - 1;
  for (int i0 = first; i0 < last; i0 += 128 * kPlanBatch) {
    int id[kPlanBatch][4];
#pragma unroll
    for (int u = 0; u < kPlanBatch; ++u) load(i0 + u * 128, id[u]);
#pragma unroll
    for (int u = 0; u < kPlanBatch; ++u) {
      int seen = 0, ahead = 0;  // of this load: all lanes', the lower lanes'
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t vote = __ballot_sync(kAll, id[u][q] == e);
        seen += __popc(vote);
        ahead += __popc(vote & before);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (id[u][q] == e) order[at + ahead++] = i0 + u * 128 + lane * 4 + q;
      at += seen;
    }
  }
}

constexpr int kTileN = 256;      // rows of an expert in a tile, at most
constexpr int kStepK = 64;       // reduction elements of a ring stage: 128 bytes, the swizzle's width
constexpr int kMaxStages = 6;
constexpr int ring_stages(int subs) { return subs == 2 ? 4 : kMaxStages; }
constexpr uint32_t kABytes = 128 * kStepK * 2, kBBytes = kTileN / 2 * kStepK * 2;
constexpr uint32_t kRingBytes = 192 * 1024;
static_assert(kRingBytes == ring_stages(1) * (kABytes + kBBytes) && kRingBytes == ring_stages(2) * (2 * kABytes + kBBytes),
              "both rings fill the same space");
constexpr int epi_warps(bool gate_up) { return gate_up ? 12 : 8; }
constexpr int kGatherWarps = 4;  // of the first product
constexpr int kGatherRows = kTileN / 2 / kGatherWarps;
constexpr int product_threads(bool gate_up) { return 64 + 32 * epi_warps(gate_up) + (gate_up ? 32 * kGatherWarps : 0); }
// one epilogue warp of the first product: 32 rows x 16 activations
constexpr uint32_t staging_bytes(bool gate_up) { return gate_up ? 32 * 16 * 2 : 0; }

struct ProductArgs {
  int32_t *offsets, *order;
  const int32_t* ids;  // gate-up: sort these pairs here (block 0 leaves the result); null: they are sorted
  int pairs;
  uint16_t* h;      // gate-up: [pairs, sorted][inner]
  float* share;     // down: [pair][hidden]
  int experts, top_k, rows, steps, m_tiles;  // rows: weight rows of the product (inner or hidden)
  int bf16;
  int withhold;     // test hook: no operand copy, so every other role's first wait runs out
};
// Up to this many pairs every block of the first product sorts them for itself instead of a
// launch of expert_plan (3 us of the host's time a call).  With the launch / without, us: 512
// pairs of 8 experts (hidden 256, inner 128) 17.7 / 16.6, 320 of 64 (1024, 512) 55.9 / 54.1, 1024
// of 32 (1024, 512) 37.0 / 37.2, 2048 of 32 41.4 / 42.8.
constexpr int kSortHere = 1024;
struct ProductMaps {
  CUtensorMap a, b;
};
__host__ __device__ constexpr uint32_t product_smem(bool gate_up, int experts) {
  return 1024 + kRingBytes + epi_warps(gate_up) * staging_bytes(gate_up) + (gate_up ? kSortHere * 4 : 0) +
         2 * 4 * (uint32_t)(experts + 1);
}

// Tile t of the list: experts in order, of an expert its runs of rows, of a run its weight rows.
struct TileList {
  const int32_t *offsets, *tiles;  // shared memory: offsets[E + 1], runs before each expert [E + 1]
  int m_tiles, e;
  // -> expert, first weight-row tile, first sorted row, rows; t must not fall from call to call
  __device__ __forceinline__ void at(int t, int& m, int& row, int& count) {
    const int run = t / m_tiles;
    m = t - run * m_tiles;
    while (tiles[e + 1] <= run) ++e;
    const int all = offsets[e + 1] - offsets[e], runs = tiles[e + 1] - tiles[e];
    const int n = ((all + runs - 1) / runs + 31) & ~31;  // equal runs, in steps of 32 rows
    const int i = run - tiles[e];
    row = offsets[e] + i * n;
    count = min(n, all - i * n);
  }
};

// expert_plan's result for a few pairs, by all threads of a block: offsets[E + 1] and order in
// shared memory.  counts: [warps][E], room that is free for now.  Each warp counts the experts
// of its run of pairs, the runs' counts become their places, and the pairs go to them in order.
__device__ __forceinline__ void sort_pairs(const int32_t* __restrict__ ids, int pairs, int experts, int32_t* counts,
                                           int32_t* offsets, int32_t* order) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int chunk = (pairs + warps * 32 - 1) / (warps * 32) * 32;
  const int first = warp * chunk, last = min(first + chunk, pairs);
  int32_t* mine = counts + warp * experts;
  for (int e = lane; e < experts; e += 32) mine[e] = 0;
  __syncwarp();
  auto pass = [&](bool place) {
    for (int i0 = first; i0 < last; i0 += 32) {
      const int id = i0 + lane < last ? __ldg(ids + i0 + lane) : -1;
      const bool valid = (unsigned)id < (unsigned)experts;
      const uint32_t same = __match_any_sync(kAll, valid ? id : -1);
      const int before = __popc(same & ((1u << lane) - 1));
      if (place && valid) order[offsets[id] + mine[id] + before] = i0 + lane;
      __syncwarp();
      if (valid && !before) mine[id] += __popc(same);
      __syncwarp();
    }
  };
  pass(false);
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += blockDim.x) {
    int sum = 0;
    for (int w = 0; w < warps; ++w) {
      const int n = counts[w * experts + e];
      counts[w * experts + e] = sum;
      sum += n;
    }
    offsets[e] = sum;
  }
  __syncthreads();
  if (warp == 0) {
    int sum = 0;
    for (int base = 0; base < experts; base += 32) {
      const int n = base + lane < experts ? offsets[base + lane] : 0;
      int to = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(kAll, to, d);
        if (lane >= d) to += v;
      }
      if (base + lane < experts) offsets[base + lane] = sum + to - n;
      sum += __shfl_sync(kAll, to, 31);
    }
    if (lane == 0) offsets[experts] = sum;
  }
  __syncthreads();
  pass(true);
  __syncthreads();
}

// kGateUp: the first product, whose token rows are gathered from x through `order`.
// kSubs: weight-row tiles of 256 that share each stage's token rows.  1: two accumulators, so
// that a tile's epilogue overlaps the next tile's products.  2, for the first product of many
// rows an expert: a quarter fewer operand bytes a product and half the gathering (TMA takes
// about 7 cycles a gathered row, 3 a row of a tile); each sub-tile has one accumulator, and the
// next tile's products begin with sub-tile 0 alone while the epilogue still reads sub-tile 1.
// 8192 tokens x 8 of 64 experts, hidden 2048, inner 1024: 561 us with one sub-tile, 459 + 55 with
// one and a sorted copy of x, 438 with two (374 without the epilogue: at 1.6 GHz under the power
// cap the tensor cores are then the bound).
template <typename T, bool kGateUp, int kSubs>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(product_threads(kGateUp), 1)
    expert_products(ProductArgs a, const __grid_constant__ ProductMaps maps) {
  constexpr int kStages = ring_stages(kSubs), kEpiWarps = epi_warps(kGateUp), kEpiGroups = kEpiWarps / 4;
  constexpr uint32_t kStageBytes = kSubs * kABytes + kBBytes;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 4];  // full[s], empty[s], acc_full[2], acc_empty[2]
  __shared__ uint32_t tmem_slot;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const uint32_t smem0 = ((uint32_t)__cvta_generic_to_shared(smem) + 1023u) & ~1023u;
  unsigned char* generic0 = smem + (smem0 - (uint32_t)__cvta_generic_to_shared(smem));
  unsigned char* staging = generic0 + kRingBytes;
  int32_t* sorted = reinterpret_cast<int32_t*>(staging + kEpiWarps * staging_bytes(kGateUp));
  int32_t* offsets = sorted + (kGateUp ? kSortHere : 0);
  int32_t* tiles = offsets + a.experts + 1;
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(&bars[0]);
  auto full_bar = [&](int s) { return bar0 + 8 * s; };
  auto empty_bar = [&](int s) { return bar0 + 8 * (kStages + s); };
  auto acc_full = [&](int i) { return bar0 + 8 * (2 * kStages + i); };
  auto acc_empty = [&](int i) { return bar0 + 8 * (2 * kStages + 2 + i); };

  pdl_trigger();
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);   // the leader's: its producer, and both CTAs' bytes
      mbar_init(empty_bar(s), 1);  // the products' commit
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full(i), 1);
      mbar_init(acc_empty(i), 2 * kEpiWarps);  // the leader's: both CTAs' epilogue warps
    }
    mbar_init_fence();
  }
  if (warp == 1) tmem_pair_alloc((uint32_t)__cvta_generic_to_shared(&tmem_slot), 2 * kTileN);
  pdl_wait();
  const bool here = kGateUp && a.ids;
  if (here) {  // (the ring is free: no copy has been issued)
    sort_pairs(a.ids, a.pairs, a.experts, reinterpret_cast<int32_t*>(generic0), offsets, sorted);
    fence_proxy_async_smem();
    if (blockIdx.x == 0) {  // for the second product
      for (int i = tid; i <= a.experts; i += blockDim.x) a.offsets[i] = offsets[i];
      for (int i = tid; i < offsets[a.experts]; i += blockDim.x) a.order[i] = sorted[i];
    }
  }
  const int32_t* order = here ? sorted : a.order;
  if (warp == 0) {  // the list of tiles: runs of at most kTileN rows of each expert
    const int32_t* from = here ? offsets : a.offsets;
    int sum = 0;
    for (int base = 0; base < a.experts; base += 32) {
      const int e = base + lane;
      const int o = e <= a.experts ? from[e] : 0, next = e < a.experts ? from[e + 1] : o;
      int runs = (next - o + kTileN - 1) / kTileN;
      const int own = runs;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(kAll, runs, d);
        if (lane >= d) runs += v;
      }
      if (e < a.experts) tiles[e] = sum + runs - own;
      if (!here && e < a.experts) offsets[e] = o;
      sum += __shfl_sync(kAll, runs, 31);
    }
    if (lane == 0) tiles[a.experts] = sum;
    if (!here && lane == 0) offsets[a.experts] = from[a.experts];
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const int count = tiles[a.experts] * a.m_tiles;
  const int first = blockIdx.x >> 1, stride = gridDim.x >> 1;
  TileList list = {offsets, tiles, a.m_tiles, 0};
  uint32_t fault = 0;

  if (warp == 0) {  // producer, in both CTAs: this CTA's half of the operands that TMA loads
    int s = 0;
    uint32_t phase = 0;
    for (int t = first; t < count && !fault && !a.withhold; t += stride) {
      int m, row0, rows;
      list.at(t, m, row0, rows);
      const int half = ((rows + 31) & ~31) / 2;  // rows of the N operand in this CTA
      for (int step = 0; step < a.steps; ++step) {
        // a fresh barrier counts as freed; the vote keeps the lanes within one step of each other
        if (!__all_sync(kAll, mbar_wait_cluster(empty_bar(s), phase ^ 1))) {
          fault = 2;
          break;
        }
        const uint32_t sa = smem0 + s * kStageBytes, sb = sa + kSubs * kABytes;
        const uint32_t bar = cluster_addr(full_bar(s), 0);
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(full_bar(s), 2 * (kSubs * kABytes + (uint32_t)half * kStepK * 2));
#pragma unroll
          for (int u = 0; u < kSubs; ++u) {
            const int tile = m * kSubs + u;  // of 256 weight rows: 128 gated features, or 256 outputs
            if (kGateUp)
              tma_pair_load5(sa + u * kABytes, &maps.a, step * kStepK, 0, 0, tile * 8 + rank * 4, list.e, bar);
            else
              tma_pair_load3(sa + u * kABytes, &maps.a, step * kStepK, tile * 256 + rank * 128, list.e, bar);
          }
          if (!kGateUp) {
#pragma unroll
            for (int i = 0; i < kTileN / 32; ++i)
              if (i * 16 < half)
                tma_pair_load2(sb + i * 2048, &maps.b, step * kStepK, row0 + rank * half + i * 16, bar);
          }
        }
        __syncwarp();
        if (++s == kStages) s = 0, phase ^= 1;
      }
    }
    // The leader's commits arrive in this CTA too: none may be on its way when the CTA exits.
    for (int i = 0; i < kStages && !fault && !a.withhold; ++i) {
      if (!__all_sync(kAll, mbar_wait_cluster(empty_bar(s), phase ^ 1))) fault = 2;
      if (++s == kStages) s = 0, phase ^= 1;
    }
  } else if (kGateUp && warp >= 2 + kEpiWarps) {
    // Gathering warps, one thread each: every fourth copy of four rows.  A stage has 16 rows at
    // least, so each warp has a part in every stage: none falls two phases of a barrier
    // behind, where parities repeat.
    const int line = (warp - 2 - kEpiWarps) * 4;
    int s = 0;
    uint32_t phase = 0;
    for (int t = first; t < count && !fault && !a.withhold; t += stride) {
      int m, row0, rows;
      list.at(t, m, row0, rows);
      const int half = ((rows + 31) & ~31) / 2;
      int from[kGatherRows / 4][4];
#pragma unroll
      for (int i = 0; i < kGatherRows; ++i) {  // past the run's end: its last row (those columns are not stored)
        const int row = (int)rank * half + line + i / 4 * (4 * kGatherWarps) + i % 4;
        from[i / 4][i % 4] = order[row0 + min(row, rows - 1)] / a.top_k;
      }
      for (int step = 0; step < a.steps; ++step) {
        if (!__all_sync(kAll, mbar_wait_cluster(empty_bar(s), phase ^ 1))) {
          fault = 2;
          break;
        }
        const uint32_t sb = smem0 + s * kStageBytes + kSubs * kABytes + line * kStepK * 2;
        const uint32_t bar = cluster_addr(full_bar(s), 0);
        if (elect_one()) {
#pragma unroll
          for (int i = 0; i < kGatherRows / 4; ++i)
            if (line + i * 4 * kGatherWarps < half)
              tma_pair_gather4(sb + i * 512 * kGatherWarps, &maps.b, step * kStepK, from[i], bar);
        }
        __syncwarp();
        if (++s == kStages) s = 0, phase ^= 1;
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {  // one thread of the pair issues the products
      int s = 0;
      uint32_t phase = 0;
      int j = 0;
      for (int t = first; t < count && !fault; t += stride, ++j) {
        int m, row0, rows;
        list.at(t, m, row0, rows);
        // operand format: 0 = fp16, 1 = bf16, the same for both
        const uint32_t idesc = umma_idesc(256, (rows + 31) & ~31, false, false) | (a.bf16 ? 1u << 7 | 1u << 10 : 0u);
        // kSubs 1: accumulator j & 1, filled every second tile; 2: accumulator u of sub-tile u, every tile
        const int acc = kSubs == 1 ? j & 1 : 0;
        const uint32_t turn = (uint32_t)(kSubs == 1 ? j >> 1 : j) & 1;
        if (!__all_sync(kAll, mbar_wait_cluster(acc_empty(acc), turn ^ 1))) {
          fault = 4;
          break;
        }
        auto multiply = [&](int u, int stage, bool add) {  // of one stage into one accumulator
          const uint32_t base = smem0 + stage * kStageBytes;
          const uint64_t da = smem_desc(base + u * kABytes, 16, 1024, kSwizzle128B);
          const uint64_t db = smem_desc(base + kSubs * kABytes, 16, 1024, kSwizzle128B);
          const uint32_t d = tmem + (kSubs == 1 ? acc : u) * kTileN;
#pragma unroll
          for (int k = 0; k < kStepK / 16; ++k)  // 16 elements: 32 bytes along the swizzled rows
            umma_pair_ss(d, da + 2 * k, db + 2 * k, idesc, add || k > 0);
        };
        int held = 0;        // kSubs 2: stages up to this one that sub-tile 1 has not taken yet
        bool open = false;   // and whether its accumulator is free
        for (int step = 0; step < a.steps; ++step) {
          if (!__all_sync(kAll, mbar_wait_cluster(full_bar(s), phase))) {
            fault = 1;
            break;
          }
          tc_fence_after();
          const bool last = step == a.steps - 1;
          if (kSubs == 1) {
            if (elect_one()) {
              multiply(0, s, step > 0);
              umma_pair_commit(empty_bar(s));
              if (last) umma_pair_commit(acc_full(acc));
            }
          } else {
            if (elect_one()) {
              multiply(0, s, step > 0);
              if (last) umma_pair_commit(acc_full(0));
            }
            __syncwarp();
            ++held;
            if (!open) {
              const bool must = last || held == kStages;  // nothing more can be loaded before
              open = __all_sync(kAll, must ? mbar_wait_cluster(acc_empty(1), turn ^ 1)
                                           : mbar_test_cluster(acc_empty(1), turn ^ 1));
              if (must && !open) {
                fault = 4;
                break;
              }
              tc_fence_after();
            }
            if (open) {
              int stage = s - (held - 1);
              if (stage < 0) stage += kStages;
              for (; held; --held) {
                if (elect_one()) {
                  multiply(1, stage, step - (held - 1) > 0);
                  umma_pair_commit(empty_bar(stage));
                }
                __syncwarp();
                if (++stage == kStages) stage = 0;
              }
              if (last && elect_one()) umma_pair_commit(acc_full(1));
            }
          }
          __syncwarp();
          if (++s == kStages) s = 0, phase ^= 1;
        }
      }
    }
  } else if (warp < 2 + kEpiWarps) {  // epilogue: TMEM lanes 32 (warp % 4).., every kEpiGroups-th chunk of columns
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    unsigned char* own = staging + (warp - 2) * staging_bytes(kGateUp);
    int j = 0;
    for (int t = first; t < count && !fault; t += stride, ++j) {
      int m, row0, rows;
      list.at(t, m, row0, rows);
#pragma unroll 1
      for (int u = 0; u < kSubs; ++u) {
        const int acc = kSubs == 1 ? j & 1 : u, tile = m * kSubs + u;
        if (!__all_sync(kAll, mbar_wait_cluster(acc_full(acc), (uint32_t)(kSubs == 1 ? j >> 1 : j) & 1))) {
          fault = 4;
          break;
        }
        tc_fence_after();
        if (kGateUp) {
          const int f0 = tile * 128 + (int)rank * 64 + quarter * 16;
          const bool low = lane < 16;
          uint16_t* out = reinterpret_cast<uint16_t*>(own) + (low ? 0 : 16) + (lane & 15);
          for (int c = group * 32; c < rows && f0 < a.rows; c += kEpiGroups * 32) {  // a.rows is a multiple of 16
            uint32_t r[32];
            tmem_ld32(lanes + acc * kTileN + c, r);
#pragma unroll
            for (int i = 0; i < 16; ++i) {  // lanes below 16 take column 2i, the others 2i + 1
              const float even = __uint_as_float(r[2 * i]), odd = __uint_as_float(r[2 * i + 1]);
              const float other = __shfl_xor_sync(kAll, low ? odd : even, 16);
              const float g = low ? even : other, u = low ? other : odd;
              out[i * 32] = T::round(__fdividef(g, 1.0f + __expf(-g)) * u);
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // two lanes a row: whole 32-byte sectors
              const int n = i * 16 + (lane >> 1), q = lane & 1;
              if (c + n < rows)
                reinterpret_cast<uint4*>(a.h + (int64_t)(row0 + c + n) * a.rows + f0)[q] =
                    reinterpret_cast<const uint4*>(own)[n * 2 + q];
            }
            __syncwarp();
          }
        } else {
          // A lane has one feature of 32 pairs: each pair's 32 features are one 128-byte line.
          const int f = tile * 256 + (int)rank * 128 + quarter * 32 + lane;
          for (int c = group * 32; c < rows && f - lane < a.rows; c += kEpiGroups * 32) {
            const int own_pair = c + lane < rows ? order[row0 + c + lane] : 0;
            uint32_t r[32];
            tmem_ld32(lanes + acc * kTileN + c, r);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int pair = __shfl_sync(kAll, own_pair, i);
              if (c + i < rows && f < a.rows) a.share[(int64_t)pair * a.rows + f] = __uint_as_float(r[i]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(acc_empty(acc), 0));
      }
    }
  }
  if (fault) {
    atomicOr(&g_expert_fault, fault);
    // copies that are still in flight into either CTA land long before this
    const uint64_t start = global_ns();
    while (global_ns() - start < 5000000ull) __nanosleep(1000);
  }
  tc_fence_before();
  __syncthreads();
  cluster_barrier();
  tc_fence_after();
  if (warp == 1) tmem_pair_dealloc(tmem, 2 * kTileN);
}

// out[token] = sum of weight * share over the token's choices, in their order; 4 features a thread.
constexpr int kCombineThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kCombineThreads, 3) expert_combine(ExpertArgs a, const float* __restrict__ share,
                                                                  FastDiv groups) {
  pdl_trigger();
  pdl_wait();
  const uint32_t i = blockIdx.x * kCombineThreads + threadIdx.x;
  const uint32_t token = groups.div(i), f = (i - token * groups.d) * 4;
  if (token >= a.tokens) return;
  float sum[4] = {};
  constexpr int kBatch = 8;  // choices whose loads are in flight together
  for (int j0 = 0; j0 < a.top_k; j0 += kBatch) {
    const int64_t pair0 = (int64_t)token * a.top_k + j0;
    const int32_t* ids = a.ids + pair0;
    const float* weights = a.weights + pair0;
    const float* from = share + pair0 * a.hidden + f;
    float w[kBatch];
    float4 v[kBatch];
    uint32_t live = 0;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)  // shares of pairs without an expert were never written
      if (j0 + j < a.top_k && (unsigned)ids[j] < (unsigned)a.experts) live |= 1u << j;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (!(live >> j & 1u)) continue;
      v[j] = __ldcs(reinterpret_cast<const float4*>(from + (int64_t)j * a.hidden));
      w[j] = weights[j];
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (!(live >> j & 1u)) continue;
      sum[0] = fmaf(w[j], v[j].x, sum[0]);
      sum[1] = fmaf(w[j], v[j].y, sum[1]);
      sum[2] = fmaf(w[j], v[j].z, sum[2]);
      sum[3] = fmaf(w[j], v[j].w, sum[3]);
    }
  }
  *reinterpret_cast<uint2*>(a.out + token * a.out_stride + f) = make_uint2(T::round2(sum[0], sum[1]), T::round2(sum[2], sum[3]));
}

// Up to how many pairs each reads its expert's weights by itself, on ordinary warps: where all
// those readings are few bytes, or few pairs meet many experts, so that they read most of them once.
// The tensor cores' four dependent launches take 15 us and more.  Both sides measured (rows /
// tensor cores, us; bf16): hidden 256, inner 128, 8 experts: 128 pairs 8.7 / 15.1, 256 pairs 14.5 /
// 15.6, 512 pairs 26 / 17; 512, 256, 16: 128 pairs (101 MB) 16.1 / 16.8; 1024, 512, 32: 40 pairs
// (126 MB) 24 / 32, 64 pairs 32 / 33, 128 pairs 51 / 33; 2048, 1024, 8: 20 pairs (252 MB) 34 / 29;
// 2048, 1024, 64: 32 pairs (403 MB) 63 / 73, 48 pairs 87 / 80.
int64_t few_pairs(int64_t hidden, int64_t inner, int64_t experts) {
  const int64_t bytes = 6 * hidden * inner;  // of one expert's weights
  return std::max(std::min<int64_t>(256, 128 * 1000 * 1000 / bytes), std::min<int64_t>(32, experts / 2));
}

// Whether the first product takes two sub-tiles: experts with many rows, no more padding of
// the weight rows, and tiles enough for every pair of SMs.  64 experts, hidden 2048, inner 1024,
// 8 choices, both products: 1024 tokens (128 rows an expert) 198.5 us with two, 198.8 with one,
// 2048 tokens 264 / 287, 4096 tokens 437 / 487.  (The second one does not gain: its
// sub-tiles take half as many steps, and their longer epilogues then stand alone, 345 us
// against 258 at 8192 tokens x 8 of 64 experts, hidden 2048, inner 1024.)
constexpr int64_t kSubRows = 128;
bool two_subs(int64_t pairs, int64_t experts, int64_t inner) {
  const int64_t tiles = (inner + 127) / 128;
  return pairs >= kSubRows * experts && tiles % 2 == 0 && pairs / kTileN * (tiles / 2) >= 2 * (sm_count() / 2);
}

struct Sizes {
  int64_t pairs;
  bool rows;                        // the few-pairs kernels
  int64_t order, h, share, total;   // byte offsets into the workspace (offsets at 0)
};
bool sizes(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k, Sizes* s) {
  if (tokens < 0 || hidden < 1 || inner < 1 || experts < 1 || experts > kMaxExperts || top_k < 1 ||
      top_k > kMaxChoices || tokens > INT32_MAX / 256 / top_k || hidden > (1 << 20) || inner > (1 << 20))
    return false;
  auto pad = [](int64_t bytes) { return (bytes + 255) / 256 * 256; };
  s->pairs = tokens * top_k;
  const int64_t few = few_pairs(hidden, inner, experts);
  s->rows = s->pairs <= few;
  if (s->rows) {
    s->order = s->h = s->share = 0;
    s->total = pad(s->pairs * inner * 4);
  } else {
    s->order = pad((experts + 1) * 4);
    s->h = s->order + pad(s->pairs * 4);
    s->share = s->h + pad(s->pairs * inner * 2);
    // never less than a smaller batch needs, whose activations are FP32
    s->total = std::max(s->share + pad(s->pairs * hidden * 4), pad(few * inner * 4));
  }
  return true;
}

ttn_status encode_map(const char* name, CUtensorMap* map, bool bf16, int rank, const void* base, const cuuint64_t* dims,
                      const cuuint64_t* strides, const cuuint32_t* box) {
  const auto encode = tensor_map_encoder();
  if (!encode) return fail(TTN_CUDA_ERROR, "%s: cuTensorMapEncodeTiled is not available", name);
  const cuuint32_t unit[5] = {1, 1, 1, 1, 1};
  const CUresult r = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            (cuuint32_t)rank, const_cast<void*>(base), dims, strides, box, unit,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TTN_UNSUPPORTED, "%s: cuTensorMapEncodeTiled %d", name, (int)r);
  return TTN_OK;
}

template <typename T>
ttn_status launch_products(const char* name, const ExpertArgs& a, const Sizes& s, unsigned char* ws, cudaStream_t stream) {
  constexpr bool bf16 = std::is_same<T, BF16>::value;
  int32_t *offsets = (int32_t*)ws, *order = (int32_t*)(ws + s.order);
  uint16_t* h = (uint16_t*)(ws + s.h);
  float* share = (float*)(ws + s.share);
  const cuuint64_t hidden = a.hidden, inner = a.inner, experts = a.experts;
  ProductMaps gate, down;
  {  // gate-up weights: (hidden, 16 rows, gate | up, inner / 16, expert)
    const cuuint64_t dims[5] = {hidden, 16, 2, inner / 16, experts};
    const cuuint64_t str[4] = {hidden * 2, inner * hidden * 2, 16 * hidden * 2, 2 * inner * hidden * 2};
    const cuuint32_t box[5] = {kStepK, 16, 2, 4, 1};
    TTN_TRY(encode_map(name, &gate.a, bf16, 5, a.gate_up, dims, str, box));
  }
  {  // x: one row a box, four rows a gather
    const cuuint64_t dims[2] = {hidden, (cuuint64_t)a.tokens};
    const cuuint64_t str[1] = {(cuuint64_t)a.x_stride * 2};
    const cuuint32_t box[2] = {kStepK, 1};
    TTN_TRY(encode_map(name, &gate.b, bf16, 2, a.x, dims, str, box));
  }
  {
    const cuuint64_t dims[3] = {inner, hidden, experts};
    const cuuint64_t str[2] = {inner * 2, hidden * inner * 2};
    const cuuint32_t box[3] = {kStepK, 128, 1};
    TTN_TRY(encode_map(name, &down.a, bf16, 3, a.down, dims, str, box));
  }
  {
    const cuuint64_t dims[2] = {inner, (cuuint64_t)s.pairs};
    const cuuint64_t str[1] = {inner * 2};
    const cuuint32_t box[2] = {kStepK, 16};
    TTN_TRY(encode_map(name, &down.b, bf16, 2, h, dims, str, box));
  }
  const bool here = s.pairs <= kSortHere;
  if (!here)
    TTN_TRY(cuda_check(launch_pdl(expert_plan, dim3((unsigned)a.experts), dim3(kPlanThreads), 0, stream, a.ids,
                                (int)s.pairs, a.experts, (int)((uintptr_t)a.ids % 16 == 0), offsets, order),
                     name));
  const int64_t runs = s.pairs / kTileN + (s.pairs < a.experts ? s.pairs : a.experts);  // at most
  auto products = [&](auto kernel, bool gate_up, int subs, const ProductMaps& maps, int rows, int length) {
    const int tile = (gate_up ? 128 : 256) * subs;  // features of a tile
    const uint32_t smem = product_smem(gate_up, a.experts);
    ProductArgs p = {};
    p.offsets = offsets, p.order = order, p.h = h, p.share = share;
    p.ids = here && gate_up ? a.ids : nullptr, p.pairs = (int)s.pairs;
    p.experts = a.experts, p.top_k = a.top_k, p.rows = rows;
    p.steps = (length + kStepK - 1) / kStepK;
    p.m_tiles = (rows + tile - 1) / tile;
    p.bf16 = bf16;
    p.withhold = gate_up && g_withhold_next_products.exchange(false);
    TTN_TRY(ensure_dynamic_smem((const void*)kernel, (int)smem));
    const int64_t pairs_of_sms = sm_count() / 2, most = runs * p.m_tiles;
    const unsigned grid = 2 * (unsigned)(most < pairs_of_sms ? most : pairs_of_sms);
    return cuda_check(launch_pdl(kernel, dim3(grid), dim3(product_threads(gate_up)), smem, stream, p, maps), name);
  };
  if (two_subs(s.pairs, a.experts, a.inner))
    TTN_TRY(products(expert_products<T, true, 2>, true, 2, gate, a.inner, a.hidden));
  else
    TTN_TRY(products(expert_products<T, true, 1>, true, 1, gate, a.inner, a.hidden));
  TTN_TRY(products(expert_products<T, false, 1>, false, 1, down, a.hidden, a.inner));
  const int64_t items = a.tokens * (a.hidden / 4);
  return cuda_check(launch_pdl(expert_combine<T>, dim3((unsigned)((items + kCombineThreads - 1) / kCombineThreads)),
                               dim3(kCombineThreads), 0, stream, a, (const float*)share,
                               FastDiv((uint32_t)(a.hidden / 4))),
                    name);
}

template <typename T>
ttn_status launch_experts(const char* name, const ExpertArgs& a, const Sizes& s, void* workspace, cudaStream_t stream) {
  if (!s.rows) return launch_products<T>(name, a, s, (unsigned char*)workspace, stream);
  float* h = (float*)workspace;
  const int64_t pairs = s.pairs;
  const int gate_blocks = (a.inner + kRowsBlock - 1) / kRowsBlock, down_blocks = a.hidden / kDownRows;
  expert_rows_gate_up<T><<<(unsigned)(pairs * gate_blocks), kRowsThreads, 0, stream>>>(a, h, gate_blocks);
  TTN_TRY(launch_check(name));
  const int warps = a.top_k < kDownWarps ? a.top_k : kDownWarps;
  return cuda_check(launch_pdl(expert_rows_down<T>, dim3((unsigned)(a.tokens * down_blocks)), dim3(warps * 32), 0,
                               stream, a, (const float*)h, down_blocks),
                    name);
}

}  // namespace
}  // namespace ttn

using namespace ttn;

extern "C" {

size_t ttn_expert_mlp_workspace_size(int64_t tokens, int64_t hidden, int64_t inner, int64_t num_experts,
                                     int64_t top_k) {
  Sizes s;
  return sizes(tokens, hidden, inner, num_experts, top_k, &s) ? (size_t)s.total : 0;
}

ttn_status ttn_expert_mlp(int dtype, const void* x, int64_t x_row_stride, int64_t tokens, int64_t hidden,
                          const int32_t* experts, const float* weights, int64_t top_k, const void* gate_up,
                          const void* down, int64_t num_experts, int64_t inner, void* out, int64_t out_row_stride,
                          void* workspace, size_t workspace_bytes, ttn_stream stream) {
  const char* name = "ttn_expert_mlp";
  if (dtype != TTN_F16 && dtype != TTN_BF16)
    return fail(TTN_UNSUPPORTED, "%s: dtype %d is not float16/bfloat16", name, dtype);
  Sizes s;
  if (!sizes(tokens, hidden, inner, num_experts, top_k, &s))
    return fail(TTN_INVALID_ARG,
                "%s: tokens %lld, hidden %lld, inner %lld, experts %lld (1..%d) or top_k %lld (1..%d) out of range", name,
                (long long)tokens, (long long)hidden, (long long)inner, (long long)num_experts, kMaxExperts,
                (long long)top_k, kMaxChoices);
  if (hidden % 8 || inner % 16)
    return fail(TTN_UNSUPPORTED, "%s: hidden must be a multiple of 8 and inner of 16", name);
  // the combine's 32-bit index of 4 outputs; 2^23 pairs and 2^20 rows keep every other count below 2^31
  if (tokens * hidden > (1ll << 34) - 4096)
    return fail(TTN_UNSUPPORTED, "%s: tokens * hidden must be below 2^34 - 4095", name);
  if (tokens == 0) return TTN_OK;
  if (!x || !experts || !weights || !gate_up || !down || !out) return fail(TTN_INVALID_ARG, "%s: null pointer", name);
  if (((uintptr_t)x | (uintptr_t)gate_up | (uintptr_t)down | (uintptr_t)out) % 16)
    return fail(TTN_INVALID_ARG, "%s: x, gate_up, down and out must be 16-byte aligned", name);
  if (((uintptr_t)experts | (uintptr_t)weights) % 4)
    return fail(TTN_INVALID_ARG, "%s: experts and weights must be 4-byte aligned", name);
  if (tokens > 1 && (x_row_stride % 8 || out_row_stride % 8 || x_row_stride < hidden || out_row_stride < hidden))
    return fail(TTN_INVALID_ARG, "%s: row strides must be multiples of 8 and at least hidden", name);
  if (workspace_bytes < (size_t)s.total || (s.total && (!workspace || (uintptr_t)workspace % 256)))
    return fail(TTN_INVALID_ARG, "%s: workspace must be 256-byte aligned and hold %lld bytes", name,
                (long long)s.total);
  ExpertArgs a;
  a.x = (const uint16_t*)x;
  a.ids = experts;
  a.weights = weights;
  a.gate_up = (const uint16_t*)gate_up;
  a.down = (const uint16_t*)down;
  a.out = (uint16_t*)out;
  a.x_stride = tokens > 1 ? x_row_stride : hidden;
  a.out_stride = tokens > 1 ? out_row_stride : hidden;
  a.tokens = tokens;
  a.hidden = (int)hidden, a.inner = (int)inner, a.experts = (int)num_experts, a.top_k = (int)top_k;
  return dtype == TTN_F16 ? launch_experts<F16>(name, a, s, workspace, (cudaStream_t)stream)
                          : launch_experts<BF16>(name, a, s, workspace, (cudaStream_t)stream);
}

void ttn_expert_mlp_test_withhold_copies(void) { g_withhold_next_products.store(true); }

ttn_status ttn_expert_mlp_fault(uint32_t* fault) {
  const char* name = "ttn_expert_mlp_fault";
  if (!fault) return fail(TTN_INVALID_ARG, "%s: null pointer", name);
  TTN_TRY(cuda_check(cudaMemcpyFromSymbol(fault, g_expert_fault, sizeof(uint32_t)), name));
  const uint32_t zero = 0;
  return cuda_check(cudaMemcpyToSymbol(g_expert_fault, &zero, sizeof(zero)), name);
}

}  // extern "C"
