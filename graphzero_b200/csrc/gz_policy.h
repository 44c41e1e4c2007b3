// Rows of policy scores: what drawing actions from them (policy_sample.cu) and
// their loss (policy_loss.cu) share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "gz_internal.h"
#include "gz_sm100.h"

namespace gz {
namespace policy {

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
// 16 bytes of floats rounded to T.
template <typename T> __device__ __forceinline__ uint4 pack(const float* x);
template <> __device__ __forceinline__ uint4 pack<float>(const float* x) {
  const float4 v = make_float4(x[0], x[1], x[2], x[3]);
  return *(const uint4*)&v;
}
template <> __device__ __forceinline__ uint4 pack<__half>(const float* x) {
  uint4 v;
  for (int k = 0; k < 4; ++k) ((__half2*)&v)[k] = __floats2half2_rn(x[2 * k], x[2 * k + 1]);
  return v;
}
template <> __device__ __forceinline__ uint4 pack<__nv_bfloat16>(const float* x) {
  uint4 v;
  for (int k = 0; k < 4; ++k) ((__nv_bfloat162*)&v)[k] = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
  return v;
}
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

struct RowArgs {
  const void* logits;
  const uint8_t* mask;
  int64_t logits_stride, mask_stride;
  int actions;
};

// Order-preserving map of floats to unsigned integers (-0 below +0 is undone
// by adding 0 first).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Maximum over the warp's lanes (no lane holds a NaN).
__device__ __forceinline__ float warp_max(float x) {
  return key_value(__reduce_max_sync(~0u, order_key(x)));
}

// V scores of a vector as floats.
template <typename T> __device__ __forceinline__ void unpack(uint4 raw, float* x);
template <> __device__ __forceinline__ void unpack<float>(uint4 raw, float* x) {
  for (int k = 0; k < 4; ++k) x[k] = __uint_as_float((&raw.x)[k]);
}
template <> __device__ __forceinline__ void unpack<__half>(uint4 raw, float* x) {
  for (int k = 0; k < 4; ++k) *(float2*)(x + 2 * k) = __half22float2(((const __half2*)&raw)[k]);
}
template <> __device__ __forceinline__ void unpack<__nv_bfloat16>(uint4 raw, float* x) {
  for (int k = 0; k < 4; ++k) {  // a bf16 is the upper half of its float
    x[2 * k] = __uint_as_float((&raw.x)[k] << 16);
    x[2 * k + 1] = __uint_as_float((&raw.x)[k] & 0xffff0000u);
  }
}

// Visibility of V actions, a bit each.
template <int V> __device__ __forceinline__ uint32_t visible_bits(const uint8_t* mask, bool aligned) {
  uint32_t bits = 0;
  if (aligned) {
    uint32_t w[V / 4];
    if (V == 4) w[0] = __ldg((const uint32_t*)mask);
    else *(uint2*)w = __ldg((const uint2*)mask);
#pragma unroll
    for (int k = 0; k < V; ++k) bits |= ((w[k / 4] >> (8 * (k % 4)) & 0xff) != 0) << k;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) bits |= (__ldg(mask + k) != 0) << k;
  }
  return bits;
}

// Maximum of a vector's visible scores and m.
template <bool kMasked, typename T>
__device__ __forceinline__ float max_vector(float m, uint4 raw, uint32_t bits) {
  constexpr int V = 16 / (int)sizeof(T);
  float f[V];
  unpack<T>(raw, f);
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (!kMasked || (bits >> k & 1)) m = fmaxf(m, f[k]);
  return m;
}
template <typename T2> __device__ __forceinline__ T2 max_pairs(uint4 raw) {
  const T2* p = (const T2*)&raw;
  return __hmax2(__hmax2(p[0], p[1]), __hmax2(p[2], p[3]));
}
template <> __device__ __forceinline__ float max_vector<false, __half>(float m, uint4 raw, uint32_t) {
  const float2 f = __half22float2(max_pairs<__half2>(raw));
  return fmaxf(m, fmaxf(f.x, f.y));
}
template <> __device__ __forceinline__ float max_vector<false, __nv_bfloat16>(float m, uint4 raw, uint32_t) {
  const float2 f = __bfloat1622float2(max_pairs<__nv_bfloat162>(raw));
  return fmaxf(m, fmaxf(f.x, f.y));
}

inline gz_status bad(const char* who, const char* what) { return set_last_error(GZ_ERR_INVALID_ARG, "%s: %s", who, what); }

inline gz_status check_rows(const gz_policy_rows* r, const char* who) {
  if (!r) return bad(who, "null argument");
  if (r->rows < 0 || r->rows > INT32_MAX) return bad(who, "rows must be 0 .. 2^31 - 1");
  if (r->actions < 1 || r->actions > GZ_POLICY_MAX_ACTIONS)
    return set_last_error(GZ_ERR_INVALID_ARG, "%s: actions must be 1 .. %d", who, GZ_POLICY_MAX_ACTIONS);
  if (r->dtype < GZ_F32 || r->dtype > GZ_BF16) return bad(who, "bad dtype");
  if (r->logits_stride < 0 || r->mask_stride < 0) return bad(who, "negative stride");
  if (r->rows > 0 && !r->logits) return bad(who, "null logits");
  return GZ_OK;
}

inline RowArgs row_args(const gz_policy_rows* r) {
  return {r->logits, r->mask, r->logits_stride, r->mask_stride, r->actions};
}

inline gz_status launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GZ_OK : set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

}  // namespace policy
}  // namespace gz
