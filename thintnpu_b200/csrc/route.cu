// Routing to experts: for each row of logits x, scores s = softmax(x) or sigmoid(x), the
// top_k experts by s + bias (inside the best groups, where there are groups) and their
// weights, s itself, renormalised over the chosen ones if asked.
//
// One warp a row.  Lane l holds the experts l*w .. l*w + w - 1 (w = ceil(E / 32)) in
// registers.  The k-th largest of the lanes' maxima is a floor: k experts are at least that
// good, so the k best are among those that reach it -- a few more than k.  They are packed
// together, one a lane, and each one's place is the number of better ones (ties: of lower
// index).  Rows with more than 32 such experts (many ties) choose one after the other: a
// warp-wide maximum and a ballot, whose lowest lane holds the lowest index among ties.
//
// The order is the mathematical one, not that of rounded scores.  softmax and sigmoid
// rise with x, so without a bias the rank is x itself.  With a bias (or a group's sum of
// two scores) ranks are fp32 sums with an error below rank_band; neighbours in the chosen
// order that lie closer than that are ranked again in 64 bits, one candidate a lane, and so
// are the groups' best where a group kept and one left out are that close.  On
// N(0, 1.5) logits with 256 experts about one row in two hundred has such neighbours.
//
// Bound: a row of 256 fp32 logits is 1 KB of reading (0.16 us a thousand rows at copy
// speed), but about a thousand instructions with a bias and groups: the kernel is bound by
// instruction issue.  On a B200 16,384 such rows take 23.9 us (62 us when each choice was a
// warp-wide maximum and close groups took the whole row in 64 bits).
#include <cfloat>

#include "rows.cuh"

namespace ttn {
namespace {

constexpr int kRouteThreads = 128;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kMaxTopK = 16;  // leaves 16 lanes for candidates behind the last choice
constexpr uint32_t kAll = 0xffffffffu;
// Two fp32 ranks further apart than band * max(1, |rank|) are in the order of their exact
// values.  With u = 2^-24: a sigmoid score is within 8 u (exp2 and reciprocal approximations
// of 2 ulp, the argument's rounding, 1 + e); a softmax score within (W + 19) u, as its
// total of W terms a lane and five shuffles rounds W + 4 times and each term is within 6 u
// (s |x - m| <= 0.37).  The bias addition rounds by |rank| u more; a difference of two doubles
// that.  A group's strength, the sum of two ranks r and q, is within twice a score's error and
// (|r| + |q| + |r + q|) u, which large biases of opposite sign leave far above |r + q| u, and its
// sum with that bound rounds once more: 0.6 band * max(1, |r| + |q|) bounds it (with band = 36 u:
// 16 + 3 (|r| + |q|) <= 19 max(1, |r| + |q|)).
template <int W>
__device__ __forceinline__ float rank_band(bool sigmoid) {
  return (sigmoid ? 4.0f * 9.0f : 4.0f * (W + 20.0f)) * 5.9604645e-8f;
}

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
  int bias_vec;                    // so can their biases
  int lanes;                       // lanes of one group when that is a power of two, else 0
  float scale;
  float* weights;
  int32_t* ids;
};

template <typename T>
__device__ __forceinline__ float logit(const RouteArgs& a, int64_t row, int e) {
  return T::get(static_cast<const typename T::raw*>(a.logits)[row * a.row_stride + e * a.col_stride]);
}
template <typename V>
__device__ __forceinline__ V warp_sum(V v) {  // the same order in every call
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(kAll, v, d);
  return v;
}
__device__ __forceinline__ float sigmoid_score(float x) { return sigmoid_fast_f32(x); }

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
  if (a.by_logit) return m != m ? (double)m : x;  // m is NaN in a softmax row with a NaN or +inf
  double s = a.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double)m) / total;
  return a.bias ? s + (double)a.bias[e] : s;  // -inf with a bias of -inf: never chosen
}

// The choice of one row in 64 bits throughout: lane j gets the expert of choice j (or -1).
// Only for rows with NaN ranks or with more than 32 experts too close to tell apart in fp32,
// so it is written for size.  ranks: room for the row's ranks in shared memory.
template <typename T>
__device__ __noinline__ int route_exact(const RouteArgs& a, int64_t row, float m, int lane, double* ranks) {
  const double total = a.sigmoid || a.by_logit ? 1.0 : exact_total<T>(a, row, m, lane);
  for (int e = lane; e < a.experts; e += 32) ranks[e] = exact_rank<T>(a, row, e, m, total);
  __syncwarp();
  uint32_t kept = 1u;
  if (a.groups > 1) {
    double t1 = -HUGE_VAL, t2 = -HUGE_VAL;  // lane g: the two best of group g
    if (lane < a.groups)
      for (int e = lane * a.group_size; e < (lane + 1) * a.group_size; ++e) {
        const double r = ranks[e];
        if (ahead(r, 0, t1, 0)) {
          t2 = t1;
          t1 = r;
        } else if (ahead(r, 0, t2, 0)) {
          t2 = r;
        }
      }
    const double strength = a.group_top == 2 && t2 != -HUGE_VAL ? t1 + t2 : t1;
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
      const double r = ranks[e];
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
__global__ void __launch_bounds__(kRouteThreads, W <= 8 ? 12 : 4) route_rows(RouteArgs a) {
  extern __shared__ double shared_ranks[];  // [warps][E]
  __shared__ float2 packed[kRouteWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * kRouteWarps + warp;
  if (row >= a.rows) return;  // whole warps
  const int w = a.width, first = lane * w;
  const float ninf = -__int_as_float(0x7f800000), band = rank_band<W>(a.sigmoid);

  float v[W];  // logits, then ranks; -inf: none
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] = ninf;
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
        for (int j = 0; j < kV; ++j) v[i + j] = f[j];
      } else {
#pragma unroll
        for (int j = 0; j < kV; ++j)
          if (first + i + j < a.experts) v[i + j] = T::get(p[i + j]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (i < w && first + i < a.experts) v[i] = logit<T>(a, row, first + i);
  }
  auto largest = [&]() {
    float l = v[0];
#pragma unroll
    for (int i = 1; i < W; ++i) l = max_nan(l, v[i]);
    return l;
  };

  // The row's maximum; a NaN or +inf in a softmax row makes every score NaN.
  float m = 0.0f, inverse = 0.0f;  // inverse: 1 / sum of exp(x - m)
  bool poisoned = false;
  if (!a.sigmoid) {
    m = warp_largest(largest());
    poisoned = !(m < __int_as_float(0x7f800000));
    if (poisoned) m = __int_as_float(0x7fffffff);
    if (!(a.by_logit && a.renormalize)) {
      float total = 0.0f;
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (v[i] != ninf) total += exp_fast(v[i] - m);
      inverse = __frcp_rn(warp_sum(total));
    }
  }
  if (!a.by_logit) {
    float bias[W];
#pragma unroll
    for (int i = 0; i < W; ++i) bias[i] = 0.0f;
    if (a.bias && a.bias_vec) {  // w and the experts are multiples of 4
#pragma unroll
      for (int i = 0; i + 4 <= W; i += 4)
        if (i < w && first + i < a.experts) F32::unpack(*reinterpret_cast<const uint4*>(a.bias + first + i), reinterpret_cast<float(&)[4]>(bias[i]));
    } else if (a.bias) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < w && first + i < a.experts) bias[i] = a.bias[first + i];
    }
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i >= w) continue;
      float r = a.sigmoid ? sigmoid_score(v[i]) : exp_fast(v[i] - m) * inverse;
      if (a.bias) r += bias[i];
      if (v[i] != ninf) v[i] = r;
    }
  }

  const float lane_best = largest();
  bool exact = poisoned || __any_sync(kAll, lane_best != lane_best);
  if (a.groups > 1 && !exact) {
    float t1 = ninf, t2 = ninf;  // lane g: the two best ranks of group g
    if (a.lanes) {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        t2 = fmaxf(t2, fminf(t1, v[i]));
        t1 = fmaxf(t1, v[i]);
      }
      for (int d = 1; d < a.lanes; d <<= 1) {
        const float o1 = __shfl_xor_sync(kAll, t1, d), o2 = __shfl_xor_sync(kAll, t2, d);
        t2 = fmaxf(fminf(t1, o1), fmaxf(t2, o2));
        t1 = fmaxf(t1, o1);
      }
      t1 = __shfl_sync(kAll, t1, lane * a.lanes);
      t2 = __shfl_sync(kAll, t2, lane * a.lanes);
    } else {
      float* k = reinterpret_cast<float*>(shared_ranks + warp * a.experts);
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (i < w && first + i < a.experts) k[first + i] = v[i];
      __syncwarp();
      if (lane < a.groups)
        for (int e = lane * a.group_size; e < (lane + 1) * a.group_size; ++e) {
          t2 = fmaxf(t2, fminf(t1, k[e]));
          t1 = fmaxf(t1, k[e]);
        }
    }
    // two ranks are added as halves: the sum of two finite ones stays finite
    const bool two = a.group_top == 2 && t2 != ninf;
    const float half = a.group_top == 2 ? 0.5f : 1.0f;
    const float strength = lane >= a.groups ? ninf : two ? 0.5f * t1 + 0.5f * t2 : half * t1;
    int rank = 0;
    for (int g = 0; g < a.groups; ++g) {
      const float o = __shfl_sync(kAll, strength, g);
      rank += o > strength || (o == strength && g < lane);
    }
    uint32_t kept = __ballot_sync(kAll, lane < a.groups && rank < a.top_groups);
    if (!a.by_logit) {
      // how far the strength may be off; an infinite rank is the same in any precision
      const float size = two ? 0.5f * fabsf(t1) + 0.5f * fabsf(t2) : half * fabsf(t1);
      const float off = fabsf(strength) < __int_as_float(0x7f800000) ? 0.6f * band * fmaxf(half, size) : 0.0f;
      const float least_kept = -warp_largest(kept >> lane & 1u ? off - strength : ninf);
      const float most_left = warp_largest(kept >> lane & 1u ? ninf : strength + off);
      if (most_left != ninf && least_kept <= most_left) {
        // A group kept and one left out are too close for fp32: the experts that can
        // be among their group's group_top, one a lane, ranked in 64 bits.
        const float least = two ? t2 : t1;
        int n = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const float bar = __shfl_sync(kAll, least, min(first + i, a.experts - 1) / a.group_size);
          const bool can = v[i] != ninf && (v[i] >= bar || v[i] >= bar - band * fmaxf(1.0f, fabsf(bar)));  // bar: +inf too
          const uint32_t vote = __ballot_sync(kAll, can);
          const int at = n + __popc(vote & ((1u << lane) - 1));
          if (can && at < 32) packed[warp][at].y = __int_as_float(first + i);
          n += __popc(vote);
        }
        __syncwarp();
        exact = n > 32;
        if (!exact) {
          const int e = lane < n ? __float_as_int(packed[warp][lane].y) : 0;
          const double z = a.sigmoid ? 1.0 : exact_total<T>(a, row, m, lane);
          const double d = exact_rank<T>(a, row, e, m, z);
          double d1 = -HUGE_VAL, d2 = -HUGE_VAL;  // lane g: the two best of group g
          for (int j = 0; j < n; ++j) {
            const double o = __shfl_sync(kAll, d, j);
            if (__shfl_sync(kAll, e, j) / a.group_size != lane) continue;
            if (o > d1) {
              d2 = d1;
              d1 = o;
            } else if (o > d2) {
              d2 = o;
            }
          }
          const double sum = a.group_top == 2 && d2 != -HUGE_VAL ? d1 + d2 : d1;
          rank = 0;
          for (int g = 0; g < a.groups; ++g) rank += ahead(__shfl_sync(kAll, sum, g), g, sum, lane);
          kept = __ballot_sync(kAll, lane < a.groups && rank < a.top_groups);
        }
        __syncwarp();
      }
    }
    if (a.lanes) {  // a lane's experts are of one group
      if (!(kept >> (lane / a.lanes) & 1u)) {
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = ninf;
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (!(kept >> (min(first + i, a.experts - 1) / a.group_size) & 1u)) v[i] = ninf;
    }
  }

  int mine = -1;      // lane j: the expert of choice j
  float val = ninf;   // and its rank
  if (!exact) {
    // Neighbours too close for fp32: lane j against lane j + 1 of the first n.  Equal logits with
    // equal biases have equal ranks in any precision and stand in index order already.
    // close: pairs to be ranked again; run: pairs within the band, equal ones too
    auto neighbours = [&](int n, uint32_t& close, uint32_t& run) {
      const float next = __shfl_down_sync(kAll, val, 1);
      const bool in_band = lane + 1 < n && val - next <= band * fmaxf(1.0f, fabsf(val));
      run = __ballot_sync(kAll, in_band);
      close = 0;
      if (!run) return;
      const float xl = mine >= 0 ? logit<T>(a, row, mine) : 0.0f, bl = mine >= 0 && a.bias ? a.bias[mine] : 0.0f;
      const float xn = __shfl_down_sync(kAll, xl, 1), bn = __shfl_down_sync(kAll, bl, 1);
      close = __ballot_sync(kAll, in_band && !(xl == xn && bl == bn));
    };
    uint32_t close = 0, run = 0;
    int n = 0;
    bool done = false;
    {
      float best = v[0];
#pragma unroll
      for (int i = 1; i < W; ++i) best = fmaxf(best, v[i]);
      float floor_rank = ninf;
      // two more than the choices where the order behind the last one may matter
      const int want = a.by_logit ? a.top_k : a.top_k + 2;
      for (int j = 0; j < want; ++j) {  // equal maxima count once: the floor is no higher for it
        floor_rank = warp_largest(best);
        if (floor_rank == ninf) break;
        if (best == floor_rank) best = ninf;
      }
      const uint32_t before = (1u << lane) - 1;
      const float bar = fmaxf(floor_rank, -FLT_MAX);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const bool in = v[i] >= bar;
        const uint32_t vote = __ballot_sync(kAll, in);
        const int at = n + __popc(vote & before);
        if (in && at < 32) packed[warp][at] = make_float2(v[i], __int_as_float(first + i));
        n += __popc(vote);
      }
      __syncwarp();
      if (n <= 32) {
        const float2 c = lane < n ? packed[warp][lane] : make_float2(ninf, 0.0f);
        const int e = __float_as_int(c.y);
        int place = 0;
        for (int j = 0; j < n; ++j) {
          const float2 o = packed[warp][j];
          place += o.x > c.x || (o.x == c.x && __float_as_int(o.y) < e);
        }
        __syncwarp();
        if (lane < n) packed[warp][place] = c;
        __syncwarp();
        if (lane < n) {
          const float2 own = packed[warp][lane];
          val = own.x;
          mine = __float_as_int(own.y);
        }
        if (!a.by_logit) neighbours(n, close, run);
        // settled unless a run of neighbours from the last choice on reaches the last candidate
        const uint32_t behind = n > a.top_k ? run >> (a.top_k - 1) : 0u;
        done = a.by_logit || n <= a.top_k || (~behind & ((1u << (n - a.top_k)) - 1)) != 0 || floor_rank == ninf;
        if (done && n > a.top_k) close &= (1u << (a.top_k - 1 + __ffs(~behind))) - 1;
      }
    }
    if (!done) {  // one after the other, as far as the run goes
      n = 0;
      mine = -1;
      val = ninf;
      float best = ninf;
      int bi = 0;
      auto rescan = [&]() {
        best = ninf;
#pragma unroll
        for (int i = 0; i < W; ++i)
          if (v[i] > best) best = v[i], bi = i;
      };
      rescan();
      auto choose = [&](int j) {  // false when nothing is left
        const float top = warp_largest(best);
        if (top == ninf) return false;
        const int src = __ffs(__ballot_sync(kAll, best == top)) - 1;
        const int e = src * w + __shfl_sync(kAll, bi, src);
        if (lane == j) mine = e, val = top;
        if (lane == src) {
#pragma unroll
          for (int i = 0; i < W; ++i)
            if (i == bi) v[i] = ninf;
          rescan();
        }
        return true;
      };
      while (n < a.top_k && choose(n)) ++n;
      if (!a.by_logit) {
        bool left = n == a.top_k;
        while (true) {
          if (left && n < 32) {
            left = choose(n);
            if (left) ++n;
          }
          neighbours(n, close, run);
          if (!left || n <= a.top_k || !(run >> (n - 2) & 1u)) break;
          if (n == 32) {
            exact = true;
            break;
          }
        }
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
  if (exact) mine = route_exact<T>(a, row, m, lane, shared_ranks + warp * a.experts);
  if (lane >= a.top_k) mine = -1;

  // Weights, one choice a lane.  Renormalised softmax needs only the chosen logits, taken
  // relative to their own maximum; so do sigmoids so small that s = e^x to fp32 (x < -20).
  // Where all chosen scores are 0 in 64 bits (logits of the lowest value), so is their sum.
  const float xm = mine >= 0 ? logit<T>(a, row, mine) : ninf;
  float s = 0.0f;
  const float chosen = a.renormalize ? warp_largest(xm) : 0.0f;
  const bool vanished = a.renormalize && (a.sigmoid ? chosen : chosen - m) < -745.13322f;  // e^that < 2^-1074
  if (mine >= 0 && !vanished) {
    if (a.sigmoid)
      s = a.renormalize && chosen < -20.0f ? expf(xm - chosen) : __fdividef(1.0f, 1.0f + expf(-xm));
    else
      s = poisoned ? m : a.renormalize ? expf(xm - chosen) : expf(xm - m) * inverse;
  }
  if (a.renormalize) {
    const float sum = warp_sum(s);
    s = sum == 0.0f ? 0.0f : __fdividef(s, sum);
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
  a.group_top = a.group_size == 1 ? 1 : group_top;
  a.sigmoid = flags & TTN_ROUTE_SIGMOID ? 1 : 0;
  a.renormalize = flags & TTN_ROUTE_RENORMALIZE ? 1 : 0;
  a.by_logit = !bias && (a.groups == 1 || a.group_top == 1);
  const int64_t size = row_dtype_size(logits->dtype);
  a.vec = a.col_stride == 1 && a.width * size % 16 == 0 && (uintptr_t)logits->data % 16 == 0 &&
          a.row_stride * size % 16 == 0;
  a.bias_vec = bias && a.width % 4 == 0 && e % 4 == 0 && (uintptr_t)bias % 16 == 0;
  a.lanes = 0;
  if (a.groups > 1 && a.group_size % a.width == 0) {
    const int lanes = a.group_size / a.width;
    if ((lanes & (lanes - 1)) == 0) a.lanes = lanes;
  }
  a.scale = scale;
  a.weights = weights;
  a.ids = experts;
  const size_t smem = (size_t)kRouteWarps * e * sizeof(double);  // 32 KB at most
  if (logits->dtype == TTN_F32)
    launch_route<F32>(a, smem, (cudaStream_t)stream);
  else if (logits->dtype == TTN_F16)
    launch_route<F16>(a, smem, (cudaStream_t)stream);
  else
    launch_route<BF16>(a, smem, (cudaStream_t)stream);
  return launch_check(name);
}
