// Score rows (router logits, vocabulary logits, token activations) in fp32, fp16 or
// bf16: element types, 16-byte vector loads and an order-preserving integer key.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace ttn {

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The largest value of the warp, NaN if there is one.
__device__ __forceinline__ float warp_largest(float v) {
  float r;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

struct F32 {
  using raw = uint32_t;
  // the largest of a vector's elements, NaN if one is
  static __device__ __forceinline__ float largest(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)),
                   max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr int kVec = 4;  // elements in 16 bytes
  static __device__ __forceinline__ float get(raw b) { return __uint_as_float(b); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
};
struct F16 {
  using raw = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(raw b) { return __half2float(__ushort_as_half(b)); }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const __half2* h = reinterpret_cast<const __half2*>(&v);
    const float2 f = __half22float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ float2 two(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
    __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ raw round(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = two(w[i]);
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
};
struct BF16 {
  using raw = uint16_t;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(raw b) { return __uint_as_float((uint32_t)b << 16); }
  static __device__ __forceinline__ float largest(const uint4& v) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const float2 f = __bfloat1622float2(__hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ float2 two(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t round2(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
  }
  static __device__ __forceinline__ raw round(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = two(w[i]);
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
};

// Key of a value in an order where NaN comes first, then the larger value; equal values
// (-0 and +0 among them) have equal keys.  -inf, which nothing chooses, has key 0.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 -> +0
  return b == 0xff800000u ? 0u : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
// The value of a key (NaN for the NaN key, -inf for key 0).
__device__ __forceinline__ float key_value(uint32_t k) {
  if (k == 0u) return -__int_as_float(0x7f800000);
  if (k == 0xffffffffu) return __int_as_float(0x7fffffff);
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

inline bool row_dtype(int dtype) { return dtype == TTN_F16 || dtype == TTN_F32 || dtype == TTN_BF16; }
inline int64_t row_dtype_size(int dtype) { return dtype == TTN_F32 ? 4 : 2; }

// A [rows, cols] view of scores: f16, bf16 or f32.
inline ttn_status validate_rows(const ttn_tensor* t, const char* name) {
  if (!t) return fail(TTN_INVALID_ARG, "%s: null descriptor", name);
  if (t->ndim != 2) return fail(TTN_INVALID_ARG, "%s: logits must have two dims, not %d", name, t->ndim);
  if (!row_dtype(t->dtype))
    return fail(TTN_UNSUPPORTED, "%s: dtype %d is not float16/bfloat16/float32", name, t->dtype);
  if (t->sizes[0] < 0 || t->sizes[1] < 0) return fail(TTN_INVALID_ARG, "%s: negative size", name);
  if (t->sizes[0] && t->sizes[1]) {
    if (!t->data) return fail(TTN_INVALID_ARG, "%s: null data pointer", name);
    if ((uintptr_t)t->data % row_dtype_size(t->dtype))
      return fail(TTN_INVALID_ARG, "%s: data pointer not aligned to its element size", name);
  }
  return TTN_OK;
}

}  // namespace ttn
