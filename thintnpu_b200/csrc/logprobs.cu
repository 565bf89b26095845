// Log probabilities of given tokens, entropy and the largest alternatives of vocabulary
// rows, in one pass over the logits.
//
// With c = scale log2 e and t = c (x - the running maximum): S = sum 2^t and A = sum 2^t t are
// kept in FP32 and rescaled when the maximum rises.  log2 p(x) = t - log2 S, and the entropy is
// log2 S - A / S in units of log 2 (both terms >= 0: no cancellation).  The difference comes
// first, so that t's error is 2^-23 |t| at most however large x is (finite masks such as -1e10,
// the lowest values); one fused multiply-add with a rounded c * maximum saves half an instruction
// a logit (4096 x 128,000 bf16: 208 us for 212) but is off by 2^-24 c |x|.
//
// The alternatives ride along.  A warp reads segments of 64 16-byte vectors (512 16-bit
// logits) and needs their maxima anyway; it leaves them in shared memory.  The n-th
// largest of 32 lanes' maxima over those is a floor: n elements are at least that large, so
// the n largest of the row lie in the segments whose maximum reaches it.  Only those (about
// 30 of 250 for n = 20) are read again (they are in L2), and their elements from the floor
// up, usually n to 2n, are put in order by counting the larger ones.
//
// A row is read by a cluster of 1 to 8 CTAs, one slice each; CTA 0 joins their (maximum, S, A)
// and their sorted lists through distributed shared memory.
//
// Without that many live segments in a slice (a 16-bit row below about 10,000 logits, or one
// split over CTAs below 128,000) there is no floor, every element qualifies and the sorted lists
// take over: with n = 20 one row of 32,000 takes 43 us, one of 128,000 9.3 us.
//
// Bound: the row's bytes; the arithmetic (about 8.5 instructions a logit with its exp2, 11.4 with
// all else a row needs) has to stay below the 11 issue slots a 16-bit logit at copy speed.
#include <cooperative_groups.h>

#include <cfloat>
#include <type_traits>

#include "rows.cuh"

namespace ttn {
namespace {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpMaxTop = 32;
constexpr int kLpGroup = 2;     // vectors of a lane in a segment
constexpr int kLpRing = 4;      // segment slots of a warp
constexpr int kLpMaxRanks = 8;  // CTAs of a row
constexpr int kLpHeld = 512;    // candidates of a CTA (>= 32 a warp)
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

// Sorts one key or entry a lane, largest first (bitonic).  Not inlined, as merge32: code that
// runs at most once a row should not be long.
template <typename K>
__device__ __noinline__ K sort32(K v, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) {
      const K o = __shfl_xor_sync(kAll, v, d);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0 || size == 32);
      v = larger ? max(v, o) : min(v, o);
    }
  return v;
}
// The 32 largest of two sorted lists, sorted: `other` reversed against `list`, then a bitonic merge.
template <typename K>
__device__ __noinline__ K merge32(K list, K other, int lane) {
  K v = max(list, __shfl_sync(kAll, other, 31 - lane));
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const K o = __shfl_xor_sync(kAll, v, d);
    v = (lane & d) == 0 ? max(v, o) : min(v, o);
  }
  return v;
}
struct LpPart {  // what a warp or a CTA knows of its part of the row
  float s, a;        // S, A
  uint32_t top_key;  // key of the largest logit
};
// What takes a t of the maximum `from` to one of the maximum `to`, no further than where 2^t is 0.
__device__ __forceinline__ float apart(float from, float to, float c) { return fmaxf((from - to) * c, -256.0f); }
// b joined to a: both rescaled to the larger maximum.  A part without live logits has s = 0.
__device__ __forceinline__ LpPart join(const LpPart& a, const LpPart& b, float c) {
  LpPart r;
  r.top_key = max(a.top_key, b.top_key);
  if (b.s == 0.0f || a.s == 0.0f) {  // one has nothing
    const LpPart& o = b.s == 0.0f ? a : b;
    r.s = o.s, r.a = o.a;
    return r;
  }
  const float most = key_value(r.top_key);
  const float ta = apart(key_value(a.top_key), most, c), tb = apart(key_value(b.top_key), most, c);
  const float fa = exp2f(ta), fb = exp2f(tb);
  r.s = a.s * fa + b.s * fb;
  r.a = (a.a + a.s * ta) * fa + (b.a + b.s * tb) * fb;
  return r;
}

// Joins the parts of the first `count` lanes (a power of two), pairwise; lane 0 has the whole.
__device__ __forceinline__ LpPart join_lanes(LpPart p, int count, float c) {
  for (int d = 1; d < count; d <<= 1) {
    const LpPart o = {__shfl_xor_sync(kAll, p.s, d), __shfl_xor_sync(kAll, p.a, d),
                      __shfl_xor_sync(kAll, p.top_key, d)};
    p = join(p, o, c);
  }
  return p;
}

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 4) token_logprobs(LpArgs a) {
  extern __shared__ float seg_top[];  // largest logit of each segment of the slice, only with a.top
  __shared__ uint4 ring[kLpWarps * kLpRing * kLpGroup * 32];
  __shared__ uint64_t buffer[kLpHeld];
  __shared__ int held;
  __shared__ LpPart parts[kLpWarps];
  __shared__ LpPart cta_part;
  __shared__ uint64_t cta_list[32];
  constexpr int kVec = T::kVec;
  constexpr int kSeg = kLpGroup * 32 * kVec;
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
  float given = 0.0f;  // thread 0 of CTA 0: the given token's logit
  bool has_given = false;
  if (threadIdx.x == 0) {
    held = 0;
    if (rank == 0 && a.logprobs) {
      const int64_t token = a.tokens[row];
      has_given = token >= 0 && token < a.vocabulary;
      if (has_given) given = T::get(base[token]);
    }
  }

  // One vector of a lane: whole where it lies inside the row, else element by element with
  // -inf outside.  `inside`: the whole segment lies inside.
  auto whole = [&](int seg) { return seg * kSeg >= shift && (seg + 1) * kSeg <= length; };
  auto load = [&](int seg, int g, bool inside) {
    const int at = seg * kSeg + (g * 32 + lane) * kVec - shift;
    if (inside || (at >= 0 && at + kVec <= a.vocabulary)) return __ldg(reinterpret_cast<const uint4*>(base + at));
    constexpr raw kNone = sizeof(raw) == 4 ? (raw)0xff800000u : std::is_same<T, F16>::value ? (raw)0xfc00u : (raw)0xff80u;
    __align__(16) raw e[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) e[i] = at + i >= 0 && at + i < a.vocabulary ? base[at + i] : kNone;
    return *reinterpret_cast<uint4*>(e);
  };

  // the maximum is the warp's, S and A this lane's, in two halves (packed arithmetic)
  const float ninf = -__int_as_float(0x7f800000);
  float most = ninf;
  bool bad = false;  // a NaN or +inf
  unsigned long long s2 = 0, a2 = 0;
  auto add = [&](int seg, const uint4 (&v)[kLpGroup]) {
    float rise = T::largest(v[0]);
#pragma unroll
    for (int g = 1; g < kLpGroup; ++g) rise = max_nan(rise, T::largest(v[g]));
    rise = warp_largest(rise);
    if (a.top && lane == 0) seg_top[seg - seg0] = rise;
    if (rise == ninf) return;  // nothing but masked logits
    if (!(rise <= most)) {  // the same in all lanes
      if (rise < __int_as_float(0x7f800000)) {
        if (most != ninf) {
          const float t = apart(most, rise, c), shrink = exp2f(t);
          a2 = f2_mul(f2_fma(s2, f2_pack(t, t), a2), f2_pack(shrink, shrink));
          s2 = f2_mul(s2, f2_pack(shrink, shrink));
        }
        most = rise;
      } else {
        bad = true;
      }
    }
#pragma unroll
    for (int g = 0; g < kLpGroup; ++g) {
      float f[kVec];
      T::unpack(v[g], f);
#pragma unroll
      for (int i = 0; i < kVec; i += 2) {
        const float2 d =
            f2_unpack(f2_mul(f2_add(f2_pack(f[i], f[i + 1]), f2_pack(-most, -most)), f2_pack(c, c)));
        const float t0 = fmaxf(d.x, -256.0f), t1 = fmaxf(d.y, -256.0f);  // masked logits: 2^t = 0 and t finite
        const unsigned long long e = f2_pack(ex2_approx(t0), ex2_approx(t1));
        s2 = f2_add(s2, e);
        a2 = f2_fma(e, f2_pack(t0, t1), a2);
      }
    }
  };
  auto fetch = [&](int seg, uint4 (&to)[kLpGroup]) {
#pragma unroll
    for (int g = 0; g < kLpGroup; ++g) to[g] = load(seg, g, false);
  };
  // This warp's segments seg, seg + kLpWarps, .. below end: those that the row does not fill (its
  // first and last at most) are loaded with guards.
  int seg = seg0 + warp, end = seg1, edge = -1;
  if (seg < end && !whole(seg)) {
    edge = seg;
    seg += kLpWarps;
  }
  const int final_seg = seg + (end - 1 - seg) / kLpWarps * kLpWarps;
  if (seg < end && !whole(final_seg)) {
    if (edge >= 0) {  // both ends
      uint4 v[kLpGroup];
      fetch(edge, v);
      add(edge, v);
    }
    edge = final_seg;
    end = final_seg;
  }
  // The others go through a ring of segment slots in shared memory: a lane copies its own
  // vectors asynchronously and reads them back itself, so nothing but its copies' completion
  // is waited for, and loads in flight cost no registers.
  uint4* slot = ring + (warp * kLpRing * kLpGroup) * 32 + lane;
  const uint4* from = reinterpret_cast<const uint4*>(base + (int64_t)seg * kSeg - shift) + lane;
  const int whole_segs = seg < end ? (end - seg + kLpWarps - 1) / kLpWarps : 0;
  auto copy = [&](int i) {
    if (i < whole_segs) {
#pragma unroll
      for (int g = 0; g < kLpGroup; ++g)
        cp_async16(slot + ((i % kLpRing) * kLpGroup + g) * 32, from + ((int64_t)i * kLpWarps * kLpGroup + g) * 32);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kLpRing - 1; ++i) copy(i);
  if (edge >= 0) {
    uint4 v[kLpGroup];
    fetch(edge, v);
    add(edge, v);
  }
  for (int i = 0; i < whole_segs; ++i) {
    copy(i + kLpRing - 1);
    cp_async_wait<kLpRing - 1>();
    uint4 v[kLpGroup];
#pragma unroll
    for (int g = 0; g < kLpGroup; ++g) v[g] = slot[((i % kLpRing) * kLpGroup + g) * 32];
    add(seg + i * kLpWarps, v);
  }
  const float2 s_halves = f2_unpack(s2), a_halves = f2_unpack(a2);
  LpPart p = {s_halves.x + s_halves.y, a_halves.x + a_halves.y, bad ? kAll : order_key(most)};
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    p.s += __shfl_xor_sync(kAll, p.s, d);
    p.a += __shfl_xor_sync(kAll, p.a, d);
  }
  if (lane == 0) parts[warp] = p;
  __syncthreads();
  if (warp == 0) {
    const LpPart all = join_lanes(parts[lane % kLpWarps], kLpWarps, c);
    if (lane == 0) cta_part = all;
  }

  if (a.top) {
    const int count = max(seg1 - seg0, 0), own = (count - warp + kLpWarps - 1) / kLpWarps;
    // floor: the n-th largest of the lanes' maxima over the segment maxima (n <= 32)
    uint32_t key = 0;
    for (int i = lane; i < count; i += 32) key = max(key, order_key(seg_top[i]));
    const uint32_t floor_key = __shfl_sync(kAll, sort32(key, lane), a.top - 1);
    const float floor_value = key_value(floor_key);  // -inf: fewer live segments than that
    // First the elements from the floor up are gathered in no particular order, and each one's
    // place is the number of larger ones.  Where they are too many for that (many equal or
    // rising logits), a second time into sorted lists, one a warp: once a list is full only what
    // beats its n-th entry gets in.
    uint64_t list = 0, last = 0;
    // Elements below the bar are passed over: masked ones, and once a list is full those equal
    // to its n-th entry too, as they come later.
    float bar = floor_value == ninf ? -FLT_MAX : floor_value;
    for (bool sorted = false;; sorted = true) {
      for (int i0 = 0; i0 < own; i0 += 32) {
        const int i = i0 + lane;
        const float t = i < own ? seg_top[i * kLpWarps + warp] : ninf;
        uint32_t open = __ballot_sync(kAll, !(t < bar));
        while (open) {  // two segments' loads in flight
          const int s0 = seg0 + (i0 + __ffs(open) - 1) * kLpWarps + warp;
          open &= open - 1;
          const int s1 = open ? seg0 + (i0 + __ffs(open) - 1) * kLpWarps + warp : s0;
          const bool two = open != 0;
          open &= open - 1;
          uint4 v[2][kLpGroup];
#pragma unroll
          for (int g = 0; g < kLpGroup; ++g) {
            v[0][g] = load(s0, g, whole(s0));
            v[1][g] = load(s1, g, whole(s1));
          }
          uint32_t reach = 0;  // bit (u * kLpGroup + g) * kVec + q
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int g = 0; g < kLpGroup; ++g) {
              float f[kVec];
              T::unpack(v[u][g], f);
#pragma unroll
              for (int q = 0; q < kVec; ++q)
                reach |= (uint32_t)(!(f[q] < bar)) << ((u * kLpGroup + g) * kVec + q);
            }
          if (!two) reach &= (1u << (kLpGroup * kVec)) - 1;
          while (__any_sync(kAll, reach)) {  // few: each element is read once more by itself
            uint64_t e = 0;
            if (reach) {
              const int bit = __ffs(reach) - 1, g = bit / kVec;
              reach &= reach - 1;
              const int place = (g < kLpGroup ? s0 : s1) * kSeg + ((g % kLpGroup) * 32 + lane) * kVec + bit % kVec - shift;
              if (place >= 0 && place < a.vocabulary) e = entry(order_key(T::get(base[place])), place);
            }
            if (!sorted) {
              const uint32_t vote = __ballot_sync(kAll, e != 0);
              int at = 0;
              if (lane == 0) at = atomicAdd(&held, __popc(vote));
              at = __shfl_sync(kAll, at, 0) + __popc(vote & ((1u << lane) - 1));
              if (e && at < kLpHeld) buffer[at] = e;
            } else if (__any_sync(kAll, e > last)) {
              list = merge32(list, sort32(e > last ? e : (uint64_t)0, lane), lane);
              last = __shfl_sync(kAll, list, a.top - 1);
              if (last) bar = key_value((uint32_t)(last >> 32) + 1);  // the next value up
            }
          }
          if (!sorted && __any_sync(kAll, *static_cast<volatile int*>(&held) > kLpHeld)) open = 0, i0 = own;  // too many
        }
      }
      __syncthreads();
      if (sorted || held <= kLpHeld) break;
    }
    if (held <= kLpHeld) {
      for (int i = threadIdx.x; i < max(held, 32); i += kLpThreads) {
        const uint64_t e = i < held ? buffer[i] : 0ull;
        int place = i < held ? 0 : i;  // places that no entry takes hold none
#pragma unroll 4
        for (int j = 0; j < held; ++j) place += i < held && buffer[j] > e;
        if (place < 32) cta_list[place] = e;
      }
    } else {
      buffer[warp * 32 + lane] = list;
      for (int half = kLpWarps / 2; half; half >>= 1) {
        __syncthreads();
        if (warp < half) {
          list = merge32(list, buffer[(warp + half) * 32 + lane], lane);
          buffer[warp * 32 + lane] = list;
        }
      }
      if (warp == 0) cta_list[lane] = list;
    }
  }
  if (ranks > 1)
    cluster.sync();
  else
    __syncthreads();
  if (rank == 0 && warp == 0) {
    uint64_t lists_of[kLpMaxRanks];
#pragma unroll
    for (int r = 0; r < kLpMaxRanks; ++r)  // all remote reads in flight together
      lists_of[r] = a.top && r < ranks ? cluster.map_shared_rank(cta_list, r)[lane] : 0ull;
    LpPart all = join_lanes(*cluster.map_shared_rank(&cta_part, lane & (ranks - 1)), ranks, c);
    all.s = __shfl_sync(kAll, all.s, 0);  // one lane's sum, so that a token has one value wherever it is listed
#pragma unroll
    for (int half = kLpMaxRanks / 2; half; half >>= 1)
      if (half < ranks) {
#pragma unroll
        for (int r = 0; r < half; ++r) lists_of[r] = merge32(lists_of[r], lists_of[r + half], lane);
      }
    const uint64_t list = lists_of[0];
    const float nan = __int_as_float(0x7fffffff);
    const bool bad = all.top_key >= 0xff800000u;  // +inf or NaN
    const bool empty = all.top_key == 0u;
    const float log_total = log2f(all.s);
    const float m = key_value(all.top_key), log_p_m = -log_total * kLn2;
    // (over halves: the difference of two finite logits stays finite)
    auto logp = [&](float x) {
      return bad ? nan : empty || x == ninf ? ninf : fmaf(0.5f * x - 0.5f * m, 2.0f * a.scale, log_p_m);
    };
    if (lane == 0) {
      if (a.logprobs) a.logprobs[row] = has_given ? logp(given) : 0.0f;
      if (a.entropy) a.entropy[row] = bad ? nan : empty ? 0.0f : (log_total - all.a / all.s) * kLn2;
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
  constexpr int kSeg = kLpGroup * 32 * T::kVec;
  const int segments = (int)((a.vocabulary + T::kVec - 1 + kSeg - 1) / kSeg);  // at the largest shift
  // Few rows: split each over a cluster, as long as a CTA keeps two rounds of its warps.
  int ranks = 1;
  while (ranks < kLpMaxRanks && a.rows * ranks * 2 <= 2 * sm_count() && segments > ranks * kLpWarps * 2) ranks *= 2;
  a.slice = (segments + ranks - 1) / ranks;
  const size_t smem = a.top ? (size_t)a.slice * 4 : 0;
  TTN_TRY(ensure_dynamic_smem((const void*)token_logprobs<T>, (int)smem));
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
  if (!(scale >= 1e-6f && scale <= 1e6f)) return fail(TTN_INVALID_ARG, "%s: scale must be in [1e-6, 1e6]", name);
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
