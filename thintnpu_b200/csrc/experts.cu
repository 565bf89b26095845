// Gated products of the chosen experts:
//   out[t] = sum_j w[t][j] down[e] (silu(gate[e] x[t]) * (up[e] x[t])),  e = experts[t][j].
//
// Few pairs (token, choice): the experts' weights are read once for each pair by
// ordinary warps, two launches in all (expert_rows_gate_up, expert_rows_down).
#include "rows.cuh"

namespace ttn {
namespace {

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
  for (int j = warp; j < a.top_k; j += blockDim.x >> 5) {
    const int64_t pair = token * a.top_k + j;
    const int e = a.ids[pair];
    float acc[kDownRows] = {};
    const bool live = (unsigned)e < (unsigned)a.experts;
    if (live) {
      const uint16_t* w = a.down + ((int64_t)e * a.hidden + d0) * a.inner;
      const float* hp = h + pair * a.inner;
#pragma unroll 2
      for (int k = lane * 8; k < a.inner; k += 256) {
        uint4 v[kDownRows];
#pragma unroll
        for (int i = 0; i < kDownRows; ++i)
          v[i] = __ldg(reinterpret_cast<const uint4*>(w + (int64_t)i * a.inner + k));
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

struct Sizes {
  int64_t h, total;
};
bool sizes(int64_t tokens, int64_t hidden, int64_t inner, int64_t experts, int64_t top_k, Sizes* s) {
  if (tokens < 0 || hidden < 1 || inner < 1 || experts < 1 || experts > kMaxExperts || top_k < 1 ||
      top_k > kMaxChoices || tokens > INT32_MAX / 256 / top_k || hidden > (1 << 20) || inner > (1 << 20))
    return false;
  const int64_t pairs = tokens * top_k;
  s->h = 0;
  s->total = (pairs * inner * 4 + 255) / 256 * 256;
  return true;
}

template <typename T>
ttn_status launch_experts(const char* name, const ExpertArgs& a, void* workspace, cudaStream_t stream) {
  float* h = (float*)workspace;
  const int64_t pairs = a.tokens * a.top_k;
  const int gate_blocks = (a.inner + kRowsBlock - 1) / kRowsBlock, down_blocks = a.hidden / kDownRows;
  if (pairs * gate_blocks > INT32_MAX || a.tokens * down_blocks > INT32_MAX)
    return fail(TTN_UNSUPPORTED, "%s: too many tokens for these sizes", name);
  expert_rows_gate_up<T><<<(unsigned)(pairs * gate_blocks), kRowsThreads, 0, stream>>>(a, h, gate_blocks);
  TTN_TRY(launch_check(name));
  const int warps = a.top_k < kDownWarps ? a.top_k : kDownWarps;
  expert_rows_down<T><<<(unsigned)(a.tokens * down_blocks), warps * 32, 0, stream>>>(a, h, down_blocks);
  return launch_check(name);
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
  return dtype == TTN_F16 ? launch_experts<F16>(name, a, workspace, (cudaStream_t)stream)
                          : launch_experts<BF16>(name, a, workspace, (cudaStream_t)stream);
}

}  // extern "C"
