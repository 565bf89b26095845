// Routing to experts: for each row of logits x, scores s = softmax(x) or sigmoid(x), the
// top_k experts by s + bias (inside the best groups, where there are groups) and their
// weights, s itself, renormalised over the chosen ones if asked.
//
// One warp a row.  Lane l holds the experts l*w .. l*w + w - 1 (w = ceil(E / 32)) in
// registers as order-preserving integer keys; each choice is one warp-wide integer
// maximum and a ballot, whose lowest lane holds the lowest index among ties.
//
// The order is the mathematical one, not that of rounded scores.  softmax and sigmoid
// rise with x, so without a bias the rank is x itself.  With a bias (or a group's sum of
// two scores) ranks are fp32 sums with an error below kBand; neighbours in the chosen
// order that lie closer than that are ranked again in 64 bits -- one candidate a lane --
// and rows whose choice of groups is that close take route_exact.  On N(0, 1.5) logits
// with 256 experts about one row in two hundred has such neighbours.
//
// Bound: a row of 256 fp32 logits is 1 KB of reading (0.16 us a thousand rows at copy
// speed); the chain of top_k choices costs more than that, so the kernel is bound by
// instruction issue and latency, and rows are spread over as many warps as fit.
#include "rows.cuh"

namespace ttn {
namespace {

constexpr int kRouteThreads = 128;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxTopK = 16;  // leaves 16 lanes for candidates behind the last choice
constexpr uint32_t kAll = 0xffffffffu;
// Two fp32 ranks further apart than kBand * max(1, |rank|) are in the order of their exact
// values: expf (2 ulp), x - max, the division and the sum's own error leave s within
// 8 * 2^-24 of its value (s <= 1), the bias addition rounds by |rank| 2^-24 more, twice that
// for a difference, and a group's sum of two doubles it again: 36 * 2^-24 = 2.2e-6.
constexpr float kBand = 2.5e-6f;

struct RouteArgs {
  const void* logits;
  int64_t row_stride, col_stride;  // elements
  const float* bias;               // [E] or null
  int64_t rows;
  int experts, width;              // width = ceil(E / 32): experts of one lane
  int top_k, groups, group_size, top_groups, group_top;
  int sigmoid, renormalize;
  int by_logit;                    // the rank is the logit itself
  int vec;                         // a lane's experts can be read as 16-byte vectors
  int lanes;                       // lanes of one group when that is a power of two, else 0
  float scale;
  float* weights;
  int32_t* ids;
};

template <typename T>
__device__ __forceinline__ float logit(const RouteArgs& a, int64_t row, int e) {
  return T::get(static_cast<const typename T::raw*>(a.logits)[row * a.row_stride + e * a.col_stride]);
}
__device__ __forceinline__ float warp_max(float v) { return key_value(__reduce_max_sync(kAll, order_key(v))); }
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {  // the same order in every call
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ float sigmoid_score(float x) { return __fdividef(1.0f, 1.0f + expf(-x)); }

// Larger first, NaN before all, equal ranks in index order; -inf is never chosen.
__device__ __forceinline__ bool ahead(double a, int ia, double b, int ib) {
  const bool na = a != a, nb = b != b;
  if (na || nb) return na && (!nb || ia < ib);
  return a > b || (a == b && ia < ib);
}
__device__ __forceinline__ void best_of(double& v, int& i) {
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const double ov = __shfl_xor_sync(kAll, v, d);
    const int oi = __shfl_xor_sync(kAll, i, d);
    if (ahead(ov, oi, v, i)) v = ov, i = oi;
  }
}

// exp(x - m) summed over the row's live experts in 64 bits.
template <typename T>
__device__ double exact_total(const RouteArgs& a, int64_t row, float m, int lane) {
  double z = 0;
  for (int e = lane; e < a.experts; e += 32) z += exp((double)logit<T>(a, row, e) - (double)m);
  return warp_sum(z);
}
template <typename T>
__device__ double exact_rank(const RouteArgs& a, int64_t row, int e, float m, double total) {
  const double x = (double)logit<T>(a, row, e);
  if (x == -HUGE_VAL) return x;
  double s = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)m) / total;
  return a.bias ? s + (double)a.bias[e] : s;
}

// The choice of one row in 64 bits throughout: lane j gets the expert of choice j (or -1).
// Only for rows whose groups are too close to tell apart in fp32, so it is written for size.
template <typename T>
__device__ __noinline__ int route_exact(const RouteArgs& a, int64_t row, float m, int lane) {
  const double total = a.sigmoid ? 1.0 : exact_total<T>(a, row, m, lane);
  uint32_t kept = 1u;
  if (a.groups > 1) {
    double strength = -HUGE_VAL;  // lane g: group g
    for (int g = 0; g < a.groups; ++g) {
      double sum = -HUGE_VAL;
      int taken = -1;
      for (int n = 0; n < a.group_top && n < a.group_size; ++n) {
        double v = -HUGE_VAL;
        int at = a.experts;
        for (int e = g * a.group_size + lane; e < (g + 1) * a.group_size; e += 32) {
          const double r = exact_rank<T>(a, row, e, m, total);
          if (e != taken && ahead(r, e, v, at)) v = r, at = e;
        }
        best_of(v, at);
        if (v != -HUGE_VAL) sum = n ? sum + v : v;
        taken = at;
      }
      if (lane == g) strength = sum;
    }
    int rank = 0;
    for (int g = 0; g < a.groups; ++g)
      if (ahead(__shfl_sync(kAll, strength, g), g, strength, lane)) ++rank;
    kept = __ballot_sync(kAll, lane < a.groups && rank < a.top_groups);
  }
  int mine = -1, last_at = -1;
  double last = 0;
  for (int j = 0; j < a.top_k; ++j) {  // the best expert behind the last choice
    double v = -HUGE_VAL;
    int at = a.experts;
    for (int e = lane; e < a.experts; e += 32) {
      if (!(kept >> (e / a.group_size) & 1u)) continue;
      const double r = exact_rank<T>(a, row, e, m, total);
      if (last_at >= 0 && !ahead(last, last_at, r, e)) continue;
      if (r != -HUGE_VAL && ahead(r, e, v, at)) v = r, at = e;
    }
    best_of(v, at);
    if (at >= a.experts) break;
    last = v, last_at = at;
    if (lane == j) mine = at;
  }
  return mine;
}

// W: room for a lane's experts (>= a.width).
template <typename T, int W>
__global__ void __launch_bounds__(kRouteThreads) route_rows(RouteArgs a) {
  extern __shared__ uint32_t shared_keys[];  // [warps][E], only where groups and lanes do not line up
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kRouteWarps + warp;
  if (row >= a.rows) return;  // whole warps
  const int w = a.width, first = lane * w;

  float x[W];
#pragma unroll
  for (int i = 0; i < W; ++i) x[i] = -__int_as_float(0x7f800000);
  constexpr int kV = W < T::kVec ? W : T::kVec;
  if (a.vec) {
    const typename T::raw* p = static_cast<const typename T::raw*>(a.logits) + row * a.row_stride + first;
#pragma unroll
    for (int i = 0; i + kV <= W; i += kV) {
      if (kV < T::kVec || i >= w || first + i >= a.experts) continue;
      if (first + i + kV <= a.experts) {
        float f[T::kVec];
        T::unpack(*reinterpret_cast<const uint4*>(p + i), f);
#pragma unroll
        for (int j = 0; j < kV; ++j) x[i + j] = f[j];
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j)
          if (first + i + j < a.experts) x[i + j] = T::get(p[i + j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < w && first + i < a.experts) x[i] = logit<T>(a, row, first + i);
  }

  // The row's maximum; a NaN or +inf in a softmax row makes every score NaN.
  float m = 0.0f;
  bool poisoned = false;
  if (!a.sigmoid) {
    uint32_t k = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) k = max(k, order_key(x[i]));
    m = key_value(__reduce_max_sync(kAll, k));
    poisoned = m != m || m == __int_as_float(0x7f800000);
    if (poisoned) m = __int_as_float(0x7fffffff);
  }
  float total = 0.0f;  // sum of exp(x - m)
  if (!a.sigmoid && !(a.by_logit && a.renormalize)) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < w && x[i] != -__int_as_float(0x7f800000)) total += expf(x[i] - m);
    total = warp_sum(total);
  }

  uint32_t key[W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    key[i] = 0;
    if (i >= w || x[i] == -__int_as_float(0x7f800000)) continue;
    float r = x[i];
    if (!a.by_logit) {
      r = a.sigmoid ? sigmoid_score(x[i]) : __fdividef(expf(x[i] - m), total);
      if (a.bias) r += a.bias[first + i];
    }
    key[i] = poisoned ? kAll : order_key(r);
  }

  bool exact = false;
  if (a.groups > 1) {
    uint32_t t1 = 0, t2 = 0;  // lane g: the two best keys of group g
    if (a.lanes) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        t2 = max(t2, min(t1, key[i]));
        t1 = max(t1, key[i]);
      }
      for (int d = 1; d < a.lanes; d <<= 1) {
        const uint32_t o1 = __shfl_xor_sync(kAll, t1, d), o2 = __shfl_xor_sync(kAll, t2, d);
        t2 = max(min(t1, o1), max(t2, o2));
        t1 = max(t1, o1);
      }
      t1 = __shfl_sync(kAll, t1, lane * a.lanes);
      t2 = __shfl_sync(kAll, t2, lane * a.lanes);
    } else {
      uint32_t* k = shared_keys + warp * a.experts;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < w && first + i < a.experts) k[first + i] = key[i];
      __syncwarp();
      if (lane < a.groups)
        for (int e = lane * a.group_size; e < (lane + 1) * a.group_size; ++e) {
          t2 = max(t2, min(t1, k[e]));
          t1 = max(t1, k[e]);
        }
    }
    const float strength =
        a.group_top == 2 && t2 ? key_value(t1) + key_value(t2) : key_value(t1);
    const uint32_t gk = lane < a.groups ? (t1 ? order_key(strength) : 0u) : 0u;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const uint32_t o = __shfl_sync(kAll, gk, g);
      rank += o > gk || (o == gk && g < lane);
    }
    const uint32_t kept = __ballot_sync(kAll, lane < a.groups && rank < a.top_groups);
    if (!a.by_logit && a.top_groups < a.groups) {
      const uint32_t in = __ballot_sync(kAll, lane < a.groups && rank == a.top_groups - 1);
      const uint32_t out = __ballot_sync(kAll, lane < a.groups && rank == a.top_groups);
      const float inner = __shfl_sync(kAll, strength, __ffs(in) - 1);
      const float outer = __shfl_sync(kAll, strength, __ffs(out) - 1);
      exact = inner - outer <= kBand * fmaxf(1.0f, fabsf(inner));  // false for infinities and NaN
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (!(kept >> (min(first + i, a.experts - 1) / a.group_size) & 1u)) key[i] = 0;
  }

  int mine = -1;           // lane j: the expert of choice j
  uint32_t mine_key = 0;
  if (!exact) {
    uint32_t bk = 0;
    int bi = 0;
    auto rescan = [&]() {
      bk = 0;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (key[i] > bk) bk = key[i], bi = i;
    };
    rescan();
    auto choose = [&](int j) {  // false when nothing is left
      const uint32_t top = __reduce_max_sync(kAll, bk);
      if (!top) return false;
      const int src = __ffs(__ballot_sync(kAll, bk == top)) - 1;
      const int e = src * w + __shfl_sync(kAll, bi, src);
      if (lane == j) mine = e, mine_key = top;
      if (lane == src) {
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (i == bi) key[i] = 0;
        rescan();
      }
      return true;
    };
    int n = 0;
    while (n < a.top_k && choose(n)) ++n;
    if (!a.by_logit) {
      // Neighbours too close for fp32: lane j against lane j + 1.  Equal logits with equal
      // biases have equal ranks in any precision and stand in index order already.
      bool left = n == a.top_k;
      uint32_t close = 0;
      while (true) {
        if (left && n < 32) {
          left = choose(n);
          if (left) ++n;
        }
        const float xl = mine >= 0 ? logit<T>(a, row, mine) : 0.0f, bl = mine >= 0 && a.bias ? a.bias[mine] : 0.0f;
        const float v = key_value(mine_key), vn = __shfl_down_sync(kAll, v, 1);
        const float xn = __shfl_down_sync(kAll, xl, 1), bn = __shfl_down_sync(kAll, bl, 1);
        const bool in_band = lane + 1 < n && v - vn <= kBand * fmaxf(1.0f, fabsf(v));
        close = __ballot_sync(kAll, in_band && !(xl == xn && bl == bn));
        // the order matters down to the last choice, and behind it as far as the run of
        // neighbours within the band (equal ones too) goes
        const uint32_t run = __ballot_sync(kAll, in_band);
        if (!left || n <= a.top_k || !(run >> (n - 2) & 1u)) break;
        if (n == 32) {
          exact = true;
          break;
        }
      }
      if (close && !exact) {
        const double z = a.sigmoid ? 1.0 : exact_total<T>(a, row, m, lane);
        const double d = lane < n ? exact_rank<T>(a, row, mine, m, z) : -HUGE_VAL;
        int rank = 0;
        for (int j = 0; j < n; ++j)
          rank += ahead(__shfl_sync(kAll, d, j), __shfl_sync(kAll, mine, j), d, mine) ? 1 : 0;
        int sorted = -1;
        for (int j = 0; j < n; ++j) {
          const int r = __shfl_sync(kAll, rank, j), e = __shfl_sync(kAll, mine, j);
          if (r == lane) sorted = e;
        }
        mine = sorted;
      }
    }
  }
  if (exact) mine = route_exact<T>(a, row, m, lane);
  if (lane >= a.top_k) mine = -1;

  // Weights, one choice a lane.  Renormalised softmax needs only the chosen logits, taken
  // relative to their own maximum; so do sigmoids so small that s = e^x to fp32 (x < -20).
  const float xm = mine >= 0 ? logit<T>(a, row, mine) : -__int_as_float(0x7f800000);
  float s = 0.0f;
  const float chosen = a.renormalize ? warp_max(xm) : 0.0f;
  if (mine >= 0) {
    if (a.sigmoid)
      s = a.renormalize && chosen < -20.0f ? expf(xm - chosen) : 1.0f / (1.0f + expf(-xm));
    else
      s = poisoned ? m : a.renormalize ? expf(xm - chosen) : expf(xm - m) / total;
  }
  if (a.renormalize) {
    const float sum = warp_sum(s);
    s = sum == 0.0f ? 0.0f : s / sum;
  }
  if (lane < a.top_k) {
    a.weights[row * a.top_k + lane] = mine >= 0 ? s * a.scale : 0.0f;
    a.ids[row * a.top_k + lane] = mine;
  }
}

template <typename T>
void launch_route(const RouteArgs& a, size_t smem, cudaStream_t stream) {
  const unsigned grid = (unsigned)((a.rows + kRouteWarps - 1) / kRouteWarps);
  auto go = [&](auto kernel) { kernel<<<grid, kRouteThreads, smem, stream>>>(a); };
  if (a.width <= 2)
    go(route_rows<T, 2>);
  else if (a.width <= 4)
    go(route_rows<T, 4>);
  else if (a.width <= 8)
    go(route_rows<T, 8>);
  else if (a.width <= 16)
    go(route_rows<T, 16>);
  else
    go(route_rows<T, 32>);
}

}  // namespace
}  // namespace ttn

using namespace ttn;

extern "C" ttn_status ttn_route_experts(const ttn_tensor* logits, const float* bias, int64_t top_k, int64_t groups,
                                        int64_t top_groups, int32_t group_top, uint32_t flags, float scale,
                                        float* weights, int32_t* experts, ttn_stream stream) {
  const char* name = "ttn_route_experts";
  TTN_TRY(validate_rows(logits, name));
  if (flags & ~(TTN_ROUTE_SIGMOID | TTN_ROUTE_RENORMALIZE))
    return fail(TTN_INVALID_ARG, "%s: unknown flags 0x%x", name, flags);
  const int64_t rows = logits->sizes[0], e = logits->sizes[1];
  if (e < 1 || e > 1024) return fail(TTN_UNSUPPORTED, "%s: %lld experts outside [1, 1024]", name, (long long)e);
  if (top_k < 1 || top_k > kMaxTopK || top_k > e)
    return fail(TTN_UNSUPPORTED, "%s: top_k %lld outside [1, min(%d, experts)]", name, (long long)top_k, kMaxTopK);
  if (groups < 1 || groups > 32 || e % groups)
    return fail(TTN_INVALID_ARG, "%s: groups must divide the experts and be in [1, 32]", name);
  if (top_groups < 1 || top_groups > groups)
    return fail(TTN_INVALID_ARG, "%s: top_groups must be in [1, groups]", name);
  if (group_top != 1 && group_top != 2) return fail(TTN_INVALID_ARG, "%s: group_top must be 1 or 2", name);
  if (!(scale == scale) || scale > 3.0e38f || scale < -3.0e38f)
    return fail(TTN_INVALID_ARG, "%s: scale must be finite", name);
  if (rows > (int64_t)kRouteWarps * INT32_MAX) return fail(TTN_UNSUPPORTED, "%s: too many rows", name);
  if (rows == 0) return TTN_OK;
  if (!weights || !experts) return fail(TTN_INVALID_ARG, "%s: null output", name);
  if ((uintptr_t)weights % 4 || (uintptr_t)experts % 4 || (uintptr_t)bias % 4)
    return fail(TTN_INVALID_ARG, "%s: weights, experts and bias must be 4-byte aligned", name);

  RouteArgs a;
  a.logits = logits->data;
  a.row_stride = rows > 1 ? logits->strides[0] : 0;
  a.col_stride = e > 1 ? logits->strides[1] : 1;
  a.bias = bias;
  a.rows = rows;
  a.experts = (int)e;
  a.width = (int)((e + 31) / 32);
  a.top_k = (int)top_k;
  a.groups = top_groups == groups ? 1 : (int)groups;  // all groups kept: none matter
  a.group_size = (int)(e / a.groups);
  a.top_groups = (int)top_groups;
  a.group_top = group_top;
  a.sigmoid = flags & TTN_ROUTE_SIGMOID ? 1 : 0;
  a.renormalize = flags & TTN_ROUTE_RENORMALIZE ? 1 : 0;
  a.by_logit = !bias && (a.groups == 1 || group_top == 1 || a.group_size == 1);
  const int64_t size = row_dtype_size(logits->dtype);
  a.vec = a.col_stride == 1 && a.width * size % 16 == 0 && (uintptr_t)logits->data % 16 == 0 &&
          a.row_stride * size % 16 == 0;
  a.lanes = 0;
  if (a.groups > 1 && a.group_size % a.width == 0) {
    const int lanes = a.group_size / a.width;
    if ((lanes & (lanes - 1)) == 0) a.lanes = lanes;
  }
  a.scale = scale;
  a.weights = weights;
  a.ids = experts;
  const size_t smem = a.groups > 1 && !a.lanes ? (size_t)kRouteWarps * e * 4 : 0;
  if (logits->dtype == TTN_F32)
    launch_route<F32>(a, smem, (cudaStream_t)stream);
  else if (logits->dtype == TTN_F16)
    launch_route<F16>(a, smem, (cudaStream_t)stream);
  else
    launch_route<BF16>(a, smem, (cudaStream_t)stream);
  return launch_check(name);
}
