// Log probabilities of given tokens, entropy and the largest alternatives of vocabulary
// rows, in one pass over the logits.
//
// With m the running maximum, d = scale (x - m): S = sum e^d and A = sum e^d d are kept
// in FP32 and rescaled when m rises, so log p(x) = d - log S and the entropy is
// log S - A / S (both terms >= 0: no cancellation).
//
// The alternatives ride along.  A warp reads 32 16-byte vectors (a segment: 256 16-bit
// logits) at a time and needs their maximum for m anyway; it leaves that maximum in
// shared memory.  The n largest logits of a row lie in the n segments with the largest
// maxima (in the order value, then segment: an element elsewhere has n segment maxima
// ahead of it), so afterwards only those n segments are read again (they are in L2) and
// only their elements that come no later than the n-th segment maximum are compared.
//
// A row is read by a cluster of 1 to 8 CTAs, one slice each; CTA 0 joins their (m, S, A)
// and their sorted lists through distributed shared memory.
//
// Bound: the row's bytes; the arithmetic (about 6 instructions and one exp2 a logit) has
// to stay below the 11 issue slots a 16-bit logit at copy speed.
#include <cooperative_groups.h>

#include <type_traits>

#include "rows.cuh"

namespace ttn {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpUnroll = 4;  // vectors in flight a thread
constexpr int64_t kLpMaxVocabulary = 1 << 20;
constexpr uint32_t kAll = 0xffffffffu;
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;

struct LpArgs {
  const void* logits;
  int64_t row_stride;  // elements
  const int64_t* tokens;
  int64_t rows;
  int vocabulary, slice;  // slice: segments of one CTA
  int top;
  float scale;
  float *logprobs, *entropy, *top_logprobs;
  int32_t* top_tokens;
};

// Value key and place in one integer: a larger one comes first (ties: the lower place).
// 0 is no element; masked logits (key 0) are none.
__device__ __forceinline__ uint64_t entry(uint32_t key, uint32_t place) {
  return key ? (uint64_t)key << 32 | (uint32_t)~place : 0ull;
}

// Sorts one entry a lane, largest first (bitonic).
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) {
      const uint64_t o = __shfl_xor_sync(kAll, v, d);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0 || size == 32);
      v = larger ? max(v, o) : min(v, o);
    }
  return v;
}
// The 32 largest of two sorted lists, sorted: `other` reversed against `list`, then a bitonic merge.
__device__ __forceinline__ uint64_t merge32(uint64_t list, uint64_t other, int lane) {
  uint64_t v = max(list, __shfl_sync(kAll, other, 31 - lane));
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const uint64_t o = __shfl_xor_sync(kAll, v, d);
    v = (lane & d) == 0 ? max(v, o) : min(v, o);
  }
  return v;
}

struct LpPart {  // what a warp or a CTA knows of its part of the row
  float m, s, a;
  uint32_t top_key;  // key of the largest logit
};
// b joined to a: both rescaled to the larger maximum.  A part without live logits has s = 0.
__device__ __forceinline__ LpPart join(const LpPart& a, const LpPart& b, float c) {
  LpPart r;
  r.top_key = max(a.top_key, b.top_key);
  if (b.s == 0.0f || a.s == 0.0f) {
    const LpPart& o = b.s == 0.0f ? a : b;
    r.m = o.m, r.s = o.s, r.a = o.a;
    return r;
  }
  r.m = fmaxf(a.m, b.m);
  const float ta = fmaxf((a.m - r.m) * c, -256.0f), tb = fmaxf((b.m - r.m) * c, -256.0f);
  const float fa = exp2f(ta), fb = exp2f(tb);
  r.s = a.s * fa + b.s * fb;
  r.a = (a.a + a.s * ta) * fa + (b.a + b.s * tb) * fb;
  return r;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads) token_logprobs(LpArgs a) {
  extern __shared__ uint32_t seg_key[];  // [segments of the slice], only with a.top
  __shared__ uint64_t lists[kLpWarps][32];
  __shared__ uint64_t buffer[kLpWarps][64];
  __shared__ LpPart parts[kLpWarps];
  __shared__ LpPart cta_part;
  __shared__ uint64_t cta_list[32];
  constexpr int kVec = T::kVec;
  constexpr int kSeg = 32 * kVec;
  using raw = typename T::raw;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int64_t row = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const raw* base = static_cast<const raw*>(a.logits) + row * a.row_stride;
  // Vectors sit on 16-byte boundaries: place p of the row is element p + shift of vector 0 on.
  const int shift = (int)(((uintptr_t)base & 15u) / sizeof(raw));
  const int length = a.vocabulary + shift;
  const int segments = (length + kSeg - 1) / kSeg;
  const int seg0 = rank * a.slice, seg1 = min(segments, seg0 + a.slice);
  const float c = a.scale * kLog2e;

  // One vector of a lane: whole where it lies inside the row, else element by element
  // with -inf outside.
  auto load = [&](int seg) {
    const int at = seg * kSeg + lane * kVec - shift;
    uint4 v;
    if (at >= 0 && at + kVec <= a.vocabulary) {
      v = __ldg(reinterpret_cast<const uint4*>(base + at));
    } else {
      constexpr raw kNone = sizeof(raw) == 4 ? (raw)0xff800000u : std::is_same<T, F16>::value ? (raw)0xfc00u : (raw)0xff80u;
      __align__(16) raw e[kVec];
#pragma unroll
      for (int i = 0; i < kVec; ++i) e[i] = at + i >= 0 && at + i < a.vocabulary ? base[at + i] : kNone;
      v = *reinterpret_cast<uint4*>(e);
    }
    return v;
  };

  LpPart p = {0.0f, 0.0f, 0.0f, 0u};  // m: the warp's; s, a: this lane's
  bool started = false;
  for (int seg = seg0 + warp; seg < seg1; seg += kLpWarps * kLpUnroll) {
    uint4 v[kLpUnroll];
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u)
      if (seg + u * kLpWarps < seg1) v[u] = load(seg + u * kLpWarps);
#pragma unroll
    for (int u = 0; u < kLpUnroll; ++u) {
      if (seg + u * kLpWarps >= seg1) break;
      float f[kVec];
      T::unpack(v[u], f);
      uint32_t k = 0;
#pragma unroll
      for (int i = 0; i < kVec; ++i) k = max(k, order_key(f[i]));
      k = __reduce_max_sync(kAll, k);
      if (a.top && lane == 0) seg_key[seg + u * kLpWarps - seg0] = k;
      if (!k) continue;  // nothing but masked logits
      p.top_key = max(p.top_key, k);
      const float sm = key_value(k);
      if (!started || sm > p.m) {  // the same in all lanes
        if (started) {
          const float t = fmaxf((p.m - sm) * c, -256.0f), scale = exp2f(t);
          p.a = (p.a + p.s * t) * scale;
          p.s *= scale;
        }
        p.m = sm;
        started = true;
      }
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float t = fmaxf((f[i] - p.m) * c, -256.0f);  // masked logits: e = 0 and t finite
        const float e = ex2_approx(t);
        p.s += e;
        p.a = fmaf(e, t, p.a);
      }
    }
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    p.s += __shfl_xor_sync(kAll, p.s, d);
    p.a += __shfl_xor_sync(kAll, p.a, d);
  }
  if (lane == 0) parts[warp] = p;
  __syncthreads();
  if (threadIdx.x == 0) {
    LpPart all = parts[0];
    for (int i = 1; i < kLpWarps; ++i) all = join(all, parts[i], c);
    cta_part = all;
  }

  if (a.top) {
    // sorted lists of the largest entries: one a warp, joined pairwise
    auto join_lists = [&](uint64_t list) {
      lists[warp][lane] = list;
      for (int half = kLpWarps / 2; half; half >>= 1) {
        __syncthreads();
        if (warp < half) {
          list = merge32(list, lists[warp + half][lane], lane);
          lists[warp][lane] = list;
        }
      }
      __syncthreads();
      return lists[0][lane];
    };
    const int count = max(seg1 - seg0, 0);
    uint64_t list = 0;
    for (int i = warp * 32; i < count; i += kLpThreads) {
      const uint64_t mine = i + lane < count ? entry(seg_key[i + lane], i + lane) : 0ull;
      if (__any_sync(kAll, mine > __shfl_sync(kAll, list, 31))) list = merge32(list, sort32(mine, lane), lane);
    }
    const uint64_t best = join_lists(list);
    // the n-th largest segment maximum: no element behind it is among the n largest
    const uint32_t floor_key = (uint32_t)(__shfl_sync(kAll, best, a.top - 1) >> 32);
    list = 0;
    int held = 0;
    uint64_t* mine = buffer[warp];
    __syncthreads();  // lists[0] is read
    for (int j = warp; j < a.top; j += kLpWarps) {
      const uint64_t chosen = __shfl_sync(kAll, best, j);
      if (!chosen) break;
      const int seg = seg0 + (int)~(uint32_t)chosen;
      const uint4 v = load(seg);
      float f[kVec];
      T::unpack(v, f);
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const uint32_t k = order_key(f[i]);
        const bool in = k && k >= floor_key;
        const uint32_t vote = __ballot_sync(kAll, in);
        if (!vote) continue;
        if (in) mine[held + __popc(vote & ((1u << lane) - 1))] = entry(k, seg * kSeg + lane * kVec + i - shift);
        held += __popc(vote);
        __syncwarp();
        if (held >= 32) {
          list = merge32(list, sort32(mine[lane], lane), lane);
          __syncwarp();
          const uint64_t rest = mine[32 + lane];
          __syncwarp();
          mine[lane] = rest;
          held -= 32;
          __syncwarp();
        }
      }
    }
    if (held) list = merge32(list, sort32(lane < held ? mine[lane] : 0ull, lane), lane);
    list = join_lists(list);
    if (warp == 0) cta_list[lane] = list;
  }
  if (ranks > 1)
    cluster.sync();
  else
    __syncthreads();
  if (rank == 0 && warp == 0) {
    LpPart all = cta_part;
    uint64_t list = a.top ? cta_list[lane] : 0ull;
    for (int r = 1; r < ranks; ++r) {
      all = join(all, *cluster.map_shared_rank(&cta_part, r), c);
      if (a.top) list = merge32(list, cluster.map_shared_rank(cta_list, r)[lane], lane);
    }
    const float nan = __int_as_float(0x7fffffff), ninf = -__int_as_float(0x7f800000);
    const bool bad = all.top_key >= 0xff800000u;  // +inf or NaN
    const bool empty = all.top_key == 0u;
    const float log_total = logf(all.s);
    auto logp = [&](float x) { return bad ? nan : empty || x == ninf ? ninf : (x - all.m) * a.scale - log_total; };
    if (lane == 0) {
      if (a.logprobs) {
        const int64_t token = a.tokens[row];
        a.logprobs[row] = token >= 0 && token < a.vocabulary ? logp(T::get(base[token])) : 0.0f;
      }
      if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.0f : log_total - all.a / all.s * kLn2;
    }
    if (lane < a.top) {
      const uint32_t k = (uint32_t)(list >> 32);
      a.top_logprobs[row * a.top + lane] = bad ? nan : k ? logp(key_value(k)) : ninf;
      a.top_tokens[row * a.top + lane] = k ? (int32_t)~(uint32_t)list : -1;
    }
  }
  if (ranks > 1) cluster.sync();  // the other CTAs' shared memory is read above
}

template <typename T>
ttn_status launch_logprobs(const char* name, LpArgs a, cudaStream_t stream) {
  constexpr int kSeg = 32 * T::kVec;
  const int segments = (int)((a.vocabulary + T::kVec - 1 + kSeg - 1) / kSeg);  // at the largest shift
  // Few rows: split each over a cluster, as long as a CTA keeps two rounds of its warps.
  int ranks = 1;
  while (ranks < 8 && a.rows * ranks * 2 <= 2 * sm_count() && segments > ranks * kLpWarps * kLpUnroll) ranks *= 2;
  a.slice = (segments + ranks - 1) / ranks;
  const size_t smem = a.top ? (size_t)a.slice * 4 : 0;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(a.rows * ranks));
  config.blockDim = dim3(kLpThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = (unsigned)ranks;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  return cuda_check(cudaLaunchKernelEx(&config, token_logprobs<T>, a), name);
}

}  // namespace
}  // namespace ttn

using namespace ttn;

extern "C" ttn_status ttn_token_logprobs(const ttn_tensor* logits, const int64_t* tokens, float scale, int64_t top,
                                         float* logprobs, float* entropy, float* top_logprobs, int32_t* top_tokens,
                                         ttn_stream stream) {
  const char* name = "ttn_token_logprobs";
  TTN_TRY(validate_rows(logits, name));
  const int64_t rows = logits->sizes[0], v = logits->sizes[1];
  if (v < 1 || v > kLpMaxVocabulary)
    return fail(TTN_UNSUPPORTED, "%s: vocabulary %lld outside [1, 2^20]", name, (long long)v);
  if (v > 1 && logits->strides[1] != 1) return fail(TTN_UNSUPPORTED, "%s: the last stride must be 1", name);
  if (top < 0 || top > kLpMaxTop || top > v)
    return fail(TTN_UNSUPPORTED, "%s: top %lld outside [0, min(%d, vocabulary)]", name, (long long)top, kLpMaxTop);
  if (!(scale > 0.0f) || scale > 1e30f) return fail(TTN_INVALID_ARG, "%s: scale must be positive and finite", name);
  if (rows > INT32_MAX / 8) return fail(TTN_UNSUPPORTED, "%s: too many rows", name);
  if (rows == 0) return TTN_OK;
  if (top && (!top_logprobs || !top_tokens)) return fail(TTN_INVALID_ARG, "%s: null top output", name);
  if (!tokens != !logprobs) return fail(TTN_INVALID_ARG, "%s: tokens and logprobs go together", name);
  if ((uintptr_t)tokens % 8 || (uintptr_t)logprobs % 4 || (uintptr_t)entropy % 4 || (uintptr_t)top_logprobs % 4 ||
      (uintptr_t)top_tokens % 4)
    return fail(TTN_INVALID_ARG, "%s: tokens and outputs must be aligned to their elements", name);
  LpArgs a;
  a.logits = logits->data;
  a.row_stride = rows > 1 ? logits->strides[0] : 0;
  a.tokens = tokens;
  a.rows = rows;
  a.vocabulary = (int)v;
  a.slice = 0;
  a.top = (int)top;
  a.scale = scale;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_tokens = top_tokens;
  if (logits->dtype == TTN_F32) return launch_logprobs<F32>(name, a, (cudaStream_t)stream);
  if (logits->dtype == TTN_F16) return launch_logprobs<F16>(name, a, (cudaStream_t)stream);
  return launch_logprobs<BF16>(name, a, (cudaStream_t)stream);
}
