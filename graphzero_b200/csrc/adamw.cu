// AdamW over many tensors in one launch, states in 32 or 8 bits
// (gz_adamw_*).
//
// A plan cuts every tensor into chunks of whole 256-element blocks and keeps
// the tensors' table and the chunk list on the device; a step launches one
// block of threads per chunk.  The gradients' addresses change from step to
// step, so they travel as kernel arguments.  So does what depends on the step's
// number t, worked out by the host; a step that is captured to be replayed
// counts on the device instead, where a kernel of one thread works the same out
// before the others.
//
// Every operation of the update is rounded by itself (no contraction), so a
// step reproduces an elementwise evaluation of the formulas bit for bit; that
// matters for 8-bit states, where a last-bit difference before the rounding
// could come out as a whole grain.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "gz_internal.h"
#include "gz_round.h"

namespace gz {
namespace {

constexpr int kBlock = GZ_ADAMW_BLOCK;
constexpr int kThreads = 256, kStepBlocks = 3;
constexpr int kPerLane = kBlock / 32;  // elements of a block per lane
constexpr int kGradsPerLaunch = 416;   // addresses and types per launch (3.7 KB of arguments)

struct Tensor {
  float* param;
  void* copy;
  void *m, *v;
  float *m_scale, *v_scale;
  int64_t n;
  uint64_t first;  // index of its first element over all tensors, each rounded up to whole blocks
  double weight_decay, lr_scale;
  int copy_dtype;
};

struct Chunk {
  int32_t tensor;
  uint32_t block;  // first block of the chunk
};

struct Grads {
  const void* p[kGradsPerLaunch];
  uint8_t dtype[kGradsPerLaunch];
};

// What depends on the step's number t.
struct Timed {
  double lr_corrected;  // lr / (1 - beta1^t)
  float correct2;       // 1 / sqrt(1 - beta2^t)
  uint32_t key;         // of the rounding
};

// t as the device counts it, and what depends on it in a counted step.
struct Count {
  int64_t t;
  Timed timed;
};

struct StepArgs {
  const Tensor* tensors;
  const Chunk* chunks;     // of this launch
  int first_tensor;        // grads.p[0] belongs to it
  uint32_t blocks;         // blocks per chunk
  double lr;
  float beta1, one_beta1, beta2, one_beta2, eps;
  float grad_scale, max_norm;  // max_norm 0: no clipping
  int64_t t;               // of a step that is not counted on the device
  Timed timed;
  Count* count;
  double* partial;         // sums of squares, one per chunk of the plan
  unsigned* arrived;
  int chunk_base, chunk_count;  // first chunk of this launch, chunks of the plan
  float* norm;
};

// A lane's eight elements of a 256-element block: four from 4 lane on and four
// from 128 + 4 lane on, so that every access of a warp is one run of memory.
constexpr int kRun = 4;
__device__ __forceinline__ int place(int lane, int k) { return (k / kRun) * (kBlock / 2) + lane * kRun + k % kRun; }

// Vector accesses of a lane's elements i, i + 1, .. i + 3.
__device__ __forceinline__ void load4(float* x, const float* p) { *(float4*)x = __ldcs((const float4*)p); }
__device__ __forceinline__ void load4(float* x, const __half* p) {
  const uint2 raw = __ldcs((const uint2*)p);
  const float2 a = __half22float2(*(const __half2*)&raw.x), b = __half22float2(*(const __half2*)&raw.y);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
__device__ __forceinline__ void load4(float* x, const __nv_bfloat16* p) {
  const uint2 raw = __ldcs((const uint2*)p);
  x[0] = __uint_as_float(raw.x << 16), x[1] = __uint_as_float(raw.x & 0xffff0000u);
  x[2] = __uint_as_float(raw.y << 16), x[3] = __uint_as_float(raw.y & 0xffff0000u);
}

// Gradients of a lane, zeros beyond the tensor's end.  `vector`: a whole block
// whose gradients are aligned to four of them.
__device__ __forceinline__ void load_grads(float* x, const void* g, int dtype, int64_t at, int lane, int64_t n, bool vector) {
#pragma unroll
  for (int k = 0; k < kPerLane; k += kRun) {
    const int64_t i = at + place(lane, k);
    if (vector) {
      if (dtype == GZ_F32) load4(x + k, (const float*)g + i);
      else if (dtype == GZ_F16) load4(x + k, (const __half*)g + i);
      else load4(x + k, (const __nv_bfloat16*)g + i);
    } else {
#pragma unroll
      for (int q = 0; q < kRun; ++q) {
        x[k + q] = 0.f;
        if (i + q >= n) continue;
        if (dtype == GZ_F32) x[k + q] = ((const float*)g)[i + q];
        else if (dtype == GZ_F16) x[k + q] = __half2float(((const __half*)g)[i + q]);
        else x[k + q] = __bfloat162float(((const __nv_bfloat16*)g)[i + q]);
      }
    }
  }
}
__device__ __forceinline__ bool grads_aligned(const void* g, int dtype) {
  return ((uintptr_t)g & (dtype == GZ_F32 ? 15 : 7)) == 0;
}

// Sum of squares: eight products added in pairs in 32 bits, everything above
// them in 64.  Where 32 bits do not hold the products (gradients beyond 2^64
// overflow; below a sum of 2^-100 lost bits could count) those are taken in 64
// too.  One block's last arrival adds the chunks' sums, in their order.
__global__ void __launch_bounds__(kThreads) norm_kernel(StepArgs a, const __grid_constant__ Grads grads) {
  __shared__ double sums[kThreads / 32];
  __shared__ bool last;
  const Chunk c = a.chunks[blockIdx.x];
  const int64_t n = a.tensors[c.tensor].n;
  const void* g = grads.p[c.tensor - a.first_tensor];
  const int dtype = grads.dtype[c.tensor - a.first_tensor];
  const int lane = threadIdx.x % 32;
  const bool aligned = grads_aligned(g, dtype);
  double sum = 0;
  if (g)
#pragma unroll 2
    for (uint32_t b = threadIdx.x / 32; b < a.blocks; b += kThreads / 32) {
      const int64_t at = (int64_t)(c.block + b) * kBlock;
      if (at >= n) break;
      float x[kPerLane];
      load_grads(x, g, dtype, at, lane, n, aligned && at + kBlock <= n);
      float y[kPerLane];
#pragma unroll
      for (int k = 0; k < kPerLane; ++k) y[k] = x[k] * x[k];
      const float s = ((y[0] + y[1]) + (y[2] + y[3])) + ((y[4] + y[5]) + (y[6] + y[7]));
      if (s >= 0x1p-100f && s < INFINITY) {
        sum += (double)s;
      } else {
#pragma unroll
        for (int k = 0; k < kPerLane; ++k) sum += (double)x[k] * x[k];
      }
    }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) sums[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < kThreads / 32; ++w) sum += sums[w];
    a.partial[a.chunk_base + blockIdx.x] = sum;
    __threadfence();
    last = atomicAdd(a.arrived, 1u) == (unsigned)a.chunk_count - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  sum = 0;
  for (int i = threadIdx.x; i < a.chunk_count; i += kThreads) sum += __ldcg(&a.partial[i]);
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) sums[threadIdx.x / 32] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0;
    for (int w = 0; w < kThreads / 32; ++w) sum += sums[w];
    *a.norm = (float)(sqrt(sum) * fabs((double)a.grad_scale));
    *a.arrived = 0;
  }
}

// Scale of a block whose largest magnitude is `most`: the power of two that
// brings it into (224, 448].
__device__ __forceinline__ int scale_exponent(float most) {
  const uint32_t b = __float_as_uint(most);
  if (b == 0) return 0;
  return max((int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u), -126);
}
__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// x (already scaled, finite) rounded down or up by u = h 2^-16 to a value of the
// 8-bit format: a multiple of a grain of 2^(e - 3), e the exponent, at least -6.
// From 2^-6 on that is the float's upper 12 bits after adding u of a grain to
// its bits; below, the sum is taken in 32 bits.
__device__ __forceinline__ float to_8bit(float x, uint32_t h) {
  return __uint_as_float((__float_as_uint(x) + (h << 4)) & 0xfff00000u);
}
constexpr float kSmall = 0x1p-6f;
template <bool kRoot> __device__ __forceinline__ float small_to_8bit(float x, uint32_t h) {
  float q = floorf(__fadd_rn(fabsf(x) * 512.f, (float)h * 0x1p-16f));
  if (kRoot && q == 0.f && x > 0.f) q = 1.f;  // a root stays positive: m over it must not run away
  return copysignf(q * 0x1p-9f, x);
}
// Four such values' codes, and back.
__device__ __forceinline__ uint32_t codes(const float* q) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(q[0], q[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(q[2], q[3]), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
__device__ __forceinline__ void values(float* x, uint32_t c) {
#pragma unroll
  for (int k = 0; k < 4; k += 2) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> (8 * k)), __NV_E4M3);
    const float2 f = __half22float2(*(const __half2*)&h);
    x[k] = f.x;
    x[k + 1] = f.y;
  }
}

// Largest magnitude over the warp (as bits: they order like the values).
__device__ __forceinline__ float warp_most(const float* x) {
  uint32_t most = 0;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) most = max(most, __float_as_uint(x[k]) & 0x7fffffffu);
  most = __reduce_max_sync(~0u, most);
  if (most >= 0x7f800000u) {  // of the finite ones
    most = 0;
#pragma unroll
    for (int k = 0; k < kPerLane; ++k) {
      const uint32_t b = __float_as_uint(x[k]) & 0x7fffffffu;
      if (b < 0x7f800000u) most = max(most, b);
    }
    most = __reduce_max_sync(~0u, most) | 0x80000000u;  // the sign tells
  }
  return __uint_as_float(most);
}

// What a lane reads of a whole, aligned block.
template <int kBits> struct Raw {
  float4 p[2];
  uint4 g[2];  // as read: four floats, or four 16-bit numbers in x and y
  float4 m[kBits == 32 ? 2 : 1], v[kBits == 32 ? 2 : 1];
  uint32_t mc[2], vc[2];
  float ms, vs;

  __device__ __forceinline__ void load(const Tensor& t, const void* grad, int dtype, uint32_t block, int lane) {
    const int64_t at = (int64_t)block * kBlock;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int64_t i = at + place(lane, k * kRun);
      p[k] = __ldcs((const float4*)(t.param + i));
      if (dtype == GZ_F32) {
        g[k] = __ldcs((const uint4*)((const float*)grad + i));
      } else {
        const uint2 h = __ldcs((const uint2*)((const uint16_t*)grad + i));
        g[k] = make_uint4(h.x, h.y, 0, 0);
      }
      if (kBits == 32) {
        m[k] = __ldcs((const float4*)((const float*)t.m + i));
        v[k] = __ldcs((const float4*)((const float*)t.v + i));
      } else {
        mc[k] = __ldcs((const uint32_t*)((const uint8_t*)t.m + i));
        vc[k] = __ldcs((const uint32_t*)((const uint8_t*)t.v + i));
      }
    }
    if (kBits == 8) {
      ms = t.m_scale[block];
      vs = t.v_scale[block];
    }
  }
  __device__ __forceinline__ void grads(float* x, int dtype) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float* y = x + k * kRun;
      if (dtype == GZ_F32) {
        *(uint4*)y = g[k];
      } else if (dtype == GZ_F16) {
        *(float2*)y = __half22float2(*(const __half2*)&g[k].x);
        *(float2*)(y + 2) = __half22float2(*(const __half2*)&g[k].y);
      } else {
        y[0] = __uint_as_float(g[k].x << 16), y[1] = __uint_as_float(g[k].x & 0xffff0000u);
        y[2] = __uint_as_float(g[k].y << 16), y[3] = __uint_as_float(g[k].y & 0xffff0000u);
      }
    }
  }
};

__host__ __device__ inline Timed timed_at(int64_t t, double lr, double beta1, double beta2, uint32_t seed) {
  return {lr / (1.0 - pow(beta1, (double)t)), (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t))),
          mix32((uint32_t)t * 0x9E3779B9u + seed)};
}

// One thread: the step's number where the host has not given it (t = 0).
__global__ void count_kernel(Count* count, int64_t t, double lr, double beta1, double beta2, uint32_t seed) {
  if (t == 0) t = count->t + 1;
  count->t = t;
  count->timed = timed_at(t, lr, beta1, beta2, seed);
}

// The numbers of a step that a chunk's tensor goes by.
template <bool kCounted> struct Rates {
  float decay, step, scale, correct2;
  uint32_t key;
  __device__ Rates(const StepArgs& a, const Tensor& t) {
    const Timed& timed = kCounted ? a.count->timed : a.timed;
    correct2 = timed.correct2;
    key = timed.key;
    decay = (float)(1.0 - a.lr * t.lr_scale * t.weight_decay);
    step = (float)(timed.lr_corrected * t.lr_scale);
    scale = a.grad_scale;
    if (a.max_norm > 0.f) {
      const float clip = __fdiv_rn(a.max_norm, __fadd_rn(*a.norm, 1e-6f));
      scale = __fmul_rn(scale, clip > 1.f ? 1.f : clip);  // (fminf would take a NaN for 1: no clipping)
    }
  }
};

// The update of a lane's elements; v holds the root of the second moment going
// in with 8-bit states, and root the new one's.
template <int kBits, bool kCounted>
__device__ __forceinline__ void update(const StepArgs& a, const Rates<kCounted>& rate, float* x, float* p, float* m, float* v, float* root) {
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    if (kBits == 8) v[k] = __fmul_rn(v[k], v[k]);
    x[k] = __fmul_rn(x[k], rate.scale);
    m[k] = __fadd_rn(__fmul_rn(m[k], a.beta1), __fmul_rn(x[k], a.one_beta1));
    v[k] = __fadd_rn(__fmul_rn(v[k], a.beta2), __fmul_rn(__fmul_rn(x[k], x[k]), a.one_beta2));
    root[k] = __fsqrt_rn(v[k]);
    const float move = __fdiv_rn(m[k], __fadd_rn(__fmul_rn(root[k], rate.correct2), a.eps));
    p[k] = __fsub_rn(__fmul_rn(p[k], rate.decay), __fmul_rn(move, rate.step));
  }
}

// Rounds a block's new states to 8 bits and stores them.
__device__ __forceinline__ void store_8bit(uint32_t key, const Tensor& t, uint32_t block, int lane, float* m, float* root) {
  const int64_t at = (int64_t)block * kBlock;
  const float m_most = warp_most(m), v_most = warp_most(root);
  const int me = scale_exponent(fabsf(m_most)), ve = scale_exponent(fabsf(v_most));
  const float m_down = power(-me), v_down = power(-ve);
  const bool odd = signbit(m_most) || signbit(v_most);  // something is not finite
  const uint32_t first = (uint32_t)(t.first + at) + lane * kRun + key;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    const uint32_t h = mix32(first + place(0, k));
    const float x = __fmul_rn(m[k], m_down), y = __fmul_rn(root[k], v_down);
    m[k] = to_8bit(x, h & 0xffffu);
    root[k] = to_8bit(y, h >> 16);
    if (fabsf(x) < kSmall || y < kSmall) {
      if (fabsf(x) < kSmall) m[k] = small_to_8bit<false>(x, h & 0xffffu);
      if (y < kSmall) root[k] = small_to_8bit<true>(y, h >> 16);
    }
    if (odd) {
      if (!isfinite(x)) m[k] = NAN;
      if (!isfinite(y)) root[k] = NAN;
    }
  }
#pragma unroll
  for (int k = 0; k < kPerLane; k += kRun) {
    __stcs((uint32_t*)((uint8_t*)t.m + at + place(lane, k)), codes(m + k));
    __stcs((uint32_t*)((uint8_t*)t.v + at + place(lane, k)), codes(root + k));
  }
  if (lane == 0) {
    t.m_scale[block] = power(me);
    t.v_scale[block] = power(ve);
  }
}

// A block at a tensor's end, or of one that is not aligned: element by element.
template <int kBits, bool kCounted>
__device__ __noinline__ void step_ragged(const StepArgs& a, const Tensor* tensor, const void* g, int dtype, uint32_t block, int lane) {
  const Tensor t = *tensor;
  const Rates<kCounted> rate(a, t);
  const int64_t at = (int64_t)block * kBlock;
  float x[kPerLane], p[kPerLane], m[kPerLane], v[kPerLane], root[kPerLane];
  const float ms = kBits == 8 ? t.m_scale[block] : 1.f, vs = kBits == 8 ? t.v_scale[block] : 1.f;
#pragma unroll
  for (int k = 0; k < kPerLane; k += kRun) {
    if (kBits == 8) {  // states are whole blocks
      values(m + k, *(const uint32_t*)((const uint8_t*)t.m + at + place(lane, k)));
      values(v + k, *(const uint32_t*)((const uint8_t*)t.v + at + place(lane, k)));
    }
  }
  load_grads(x, g, dtype, at, lane, t.n, false);
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    const int64_t i = at + place(lane, k);
    const bool in = i < t.n;
    p[k] = in ? t.param[i] : 0.f;
    if (kBits == 32) {
      m[k] = in ? ((const float*)t.m)[i] : 0.f;
      v[k] = in ? ((const float*)t.v)[i] : 0.f;
    } else {
      m[k] = in ? __fmul_rn(m[k], ms) : 0.f;
      v[k] = in ? __fmul_rn(v[k], vs) : 0.f;
    }
  }
  update<kBits, kCounted>(a, rate, x, p, m, v, root);
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) {
    const int64_t i = at + place(lane, k);
    if (i >= t.n) continue;
    t.param[i] = p[k];
    if (kBits == 32) {
      ((float*)t.m)[i] = m[k];
      ((float*)t.v)[i] = v[k];
    }
    if (t.copy) {
      if (t.copy_dtype == GZ_F16) ((__half*)t.copy)[i] = __float2half_rn(p[k]);
      else ((__nv_bfloat16*)t.copy)[i] = __float2bfloat16_rn(p[k]);
    }
  }
  if (kBits == 8) store_8bit(rate.key, t, block, lane, m, root);
}

// A warp per 256-element block, several in turn; with 8-bit states the next
// block is read while one is worked on.  Every array is read and written once,
// past the caches (nothing is used again within the step): bound by memory.
template <int kBits, bool kCounted>
__global__ void __launch_bounds__(kThreads, kStepBlocks) step_kernel(const __grid_constant__ StepArgs a, const __grid_constant__ Grads grads) {
  const Chunk c = a.chunks[blockIdx.x];
  const Tensor t = a.tensors[c.tensor];
  const void* g = grads.p[c.tensor - a.first_tensor];
  const int dtype = grads.dtype[c.tensor - a.first_tensor];
  if (!kCounted && blockIdx.x == 0 && threadIdx.x == 0) a.count->t = a.t;  // for a counted step after this one
  if (!g) return;
  const int lane = threadIdx.x % 32;
  const Rates<kCounted> rate(a, t);
  bool aligned = grads_aligned(g, dtype) && ((uintptr_t)t.param & 15) == 0 && ((uintptr_t)t.copy & 7) == 0;
  if (kBits == 32) aligned = aligned && (((uintptr_t)t.m | (uintptr_t)t.v) & 15) == 0;
  const uint32_t end = min((uint32_t)((t.n + kBlock - 1) / kBlock), c.block + a.blocks);
  const uint32_t whole = aligned ? min((uint32_t)(t.n / kBlock), end) : 0;  // whole blocks end here
  uint32_t b = c.block + threadIdx.x / 32;
  Raw<kBits> next;
  if (b < whole) next.load(t, g, dtype, b, lane);
#pragma unroll 2
  for (; b < whole; b += kThreads / 32) {
    const Raw<kBits> now = next;
    if (kBits == 8 && b + kThreads / 32 < whole) next.load(t, g, dtype, b + kThreads / 32, lane);
    float x[kPerLane], p[kPerLane], m[kPerLane], v[kPerLane], root[kPerLane];
    now.grads(x, dtype);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      *(float4*)(p + k * kRun) = now.p[k];
      if (kBits == 32) {
        *(float4*)(m + k * kRun) = now.m[k];
        *(float4*)(v + k * kRun) = now.v[k];
      } else {
        values(m + k * kRun, now.mc[k]);
        values(v + k * kRun, now.vc[k]);
#pragma unroll
        for (int q = k * kRun; q < (k + 1) * kRun; ++q) {
          m[q] = __fmul_rn(m[q], now.ms);
          v[q] = __fmul_rn(v[q], now.vs);
        }
      }
    }
    update<kBits, kCounted>(a, rate, x, p, m, v, root);
#pragma unroll
    for (int k = 0; k < kPerLane; k += kRun) {
      const int64_t i = (int64_t)b * kBlock + place(lane, k);
      __stcs((float4*)(t.param + i), *(const float4*)(p + k));
      if (kBits == 32) {
        __stcs((float4*)((float*)t.m + i), *(const float4*)(m + k));
        __stcs((float4*)((float*)t.v + i), *(const float4*)(v + k));
      }
      if (t.copy) {
        uint2 raw;
        if (t.copy_dtype == GZ_F16) {
          ((__half2*)&raw)[0] = __floats2half2_rn(p[k], p[k + 1]);
          ((__half2*)&raw)[1] = __floats2half2_rn(p[k + 2], p[k + 3]);
        } else {
          ((__nv_bfloat162*)&raw)[0] = __floats2bfloat162_rn(p[k], p[k + 1]);
          ((__nv_bfloat162*)&raw)[1] = __floats2bfloat162_rn(p[k + 2], p[k + 3]);
        }
        __stcs((uint2*)((uint16_t*)t.copy + i), raw);
      }
    }
    if (kBits == 8) store_8bit(rate.key, t, b, lane, m, root);
    else if (b + kThreads / 32 < whole) next.load(t, g, dtype, b + kThreads / 32, lane);
  }
  for (; b < end; b += kThreads / 32) step_ragged<kBits, kCounted>(a, a.tensors + c.tensor, g, dtype, b, lane);
}

}  // namespace
}  // namespace gz

using namespace gz;

struct gz_adamw {
  int device = 0, state_bits = 32, count = 0;
  uint32_t blocks_per_chunk = 0;
  void* arena = nullptr;  // tensors | chunks | partial sums | count, norm and counter of blocks
  Tensor* d_tensors = nullptr;
  Chunk* d_chunks = nullptr;
  double* d_partial = nullptr;
  Count* d_count = nullptr;
  unsigned* d_arrived = nullptr;
  float* d_norm = nullptr;
  std::vector<int> chunk_start;  // per tensor, and the total
};

namespace {

gz_status bad(const char* who, const char* what) { return set_last_error(GZ_ERR_INVALID_ARG, "%s: %s", who, what); }

gz_status cuda_failed(const char* who, cudaError_t e) {
  return set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

struct Device {  // the plan's device for the scope
  int prev = -1;
  bool changed = false, ok = false;
  explicit Device(int d) {
    ok = cudaGetDevice(&prev) == cudaSuccess;
    if (ok && prev != d) {
      changed = ok = cudaSetDevice(d) == cudaSuccess;
    }
  }
  ~Device() {
    if (changed) cudaSetDevice(prev);
  }
};

// Whether two of the buffers that a step writes overlap: blocks of threads would
// race for them.
bool any_overlap(const std::vector<Tensor>& tensors, int state_bits) {
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  auto add = [&](const void* p, uint64_t bytes) {
    if (p && bytes) spans.push_back({(uintptr_t)p, (uintptr_t)p + bytes});
  };
  for (const Tensor& t : tensors) {
    const uint64_t n = (uint64_t)t.n, blocks = (n + kBlock - 1) / kBlock, state = state_bits == 8 ? blocks * kBlock : 4 * n;
    add(t.param, 4 * n);
    add(t.copy, 2 * n);
    add(t.m, state);
    add(t.v, state);
    if (state_bits == 8) {
      add(t.m_scale, 4 * blocks);
      add(t.v_scale, 4 * blocks);
    }
  }
  std::sort(spans.begin(), spans.end());
  for (size_t k = 1; k < spans.size(); ++k)
    if (spans[k].first < spans[k - 1].second) return true;
  return false;
}

gz_status create(const gz_adamw_tensor* tensors, int count, int state_bits, int device, gz_adamw* a) {
  const char* who = "gz_adamw_create";
  std::vector<Tensor> table((size_t)count);
  std::vector<Chunk> chunks;
  uint64_t first = 0;
  for (int k = 0; k < count; ++k) {
    const gz_adamw_tensor& t = tensors[k];
    if (t.n < 0 || t.n > (int64_t)UINT32_MAX * (kBlock / 2)) return bad(who, "bad tensor size");
    if (t.n > 0 && (!t.param || !t.m || !t.v)) return bad(who, "null tensor");
    if (t.copy && t.copy_dtype != GZ_F16 && t.copy_dtype != GZ_BF16) return bad(who, "the copy must be fp16 or bf16");
    if (!(t.weight_decay >= 0) || !isfinite(t.weight_decay) || !(t.lr_scale >= 0) || !isfinite(t.lr_scale))
      return bad(who, "weight_decay and lr_scale must be finite and at least 0");
    if (state_bits == 8 && t.n > 0) {
      if (!t.m_scale || !t.v_scale) return bad(who, "8-bit states need scales");
      if (((uintptr_t)t.m | (uintptr_t)t.v) % 16) return bad(who, "8-bit states must be 16-byte aligned");
    }
    table[k] = {t.param, t.copy, t.m, t.v, t.m_scale, t.v_scale, t.n, first, t.weight_decay, t.lr_scale,
                t.copy_dtype};
    first += (uint64_t)(t.n + kBlock - 1) / kBlock * kBlock;
  }
  if (any_overlap(table, state_bits)) return bad(who, "weights, copies or states overlap");
  a->device = device;
  a->state_bits = state_bits;
  a->count = count;
  // a block of the plan's units per warp and round; with many, more rounds
  // until there are some sixteen chunks an SM
  const uint64_t all_blocks = first / kBlock;
  a->blocks_per_chunk = 8;
  while (a->blocks_per_chunk < 64 && all_blocks / a->blocks_per_chunk > 148 * 32) a->blocks_per_chunk *= 2;
  for (int k = 0; k < count; ++k) {
    a->chunk_start.push_back((int)chunks.size());
    const uint64_t blocks = (uint64_t)(table[k].n + kBlock - 1) / kBlock;
    for (uint64_t b = 0; b < blocks; b += a->blocks_per_chunk) chunks.push_back({k, (uint32_t)b});
    if (chunks.size() > (size_t)INT32_MAX) return bad(who, "too many elements");
  }
  a->chunk_start.push_back((int)chunks.size());

  int devices = 0;
  if (cudaError_t e = cudaGetDeviceCount(&devices)) return cuda_failed(who, e);
  if (device < 0 || device >= devices) return set_last_error(GZ_ERR_INVALID_ARG, "%s: device %d of %d", who, device, devices);
  Device on(device);
  if (!on.ok) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, device);
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  const size_t tb = up(sizeof(Tensor) * table.size()), cb = up(sizeof(Chunk) * chunks.size()), pb = up(8 * chunks.size());
  if (cudaError_t e = cudaMalloc(&a->arena, tb + cb + pb + 256)) return cuda_failed(who, e);
  char* p = (char*)a->arena;
  a->d_tensors = (Tensor*)p;
  a->d_chunks = (Chunk*)(p + tb);
  a->d_partial = (double*)(p + tb + cb);
  a->d_count = (Count*)(p + tb + cb + pb);
  a->d_norm = (float*)(a->d_count + 1);
  a->d_arrived = (unsigned*)(a->d_norm + 1);
  static_assert(sizeof(Count) + 8 <= 256, "they fit the arena's end");
  cudaError_t e = cudaMemset(a->d_count, 0, 256);
  if (e == cudaSuccess && count) e = cudaMemcpy(a->d_tensors, table.data(), sizeof(Tensor) * table.size(), cudaMemcpyHostToDevice);
  if (e == cudaSuccess && !chunks.empty())
    e = cudaMemcpy(a->d_chunks, chunks.data(), sizeof(Chunk) * chunks.size(), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  return e == cudaSuccess ? GZ_OK : cuda_failed(who, e);
}

}  // namespace

extern "C" gz_status gz_adamw_create(const gz_adamw_tensor* tensors, int count, int state_bits, int device,
                                     gz_adamw** out) {
  const char* who = "gz_adamw_create";
  if (!out) return bad(who, "null argument");
  *out = nullptr;
  if (count < 0 || (count > 0 && !tensors)) return bad(who, "null argument");
  if (state_bits != 8 && state_bits != 32) return bad(who, "states have 8 or 32 bits");
  gz_adamw* a = nullptr;
  gz_status s;
  try {
    a = new gz_adamw;
    s = create(tensors, count, state_bits, device, a);
  } catch (const std::bad_alloc&) {
    s = set_last_error(GZ_ERR_CAPACITY, "%s: out of host memory", who);
  }
  if (s != GZ_OK) {
    if (a) gz_adamw_destroy(a);
    return s;
  }
  *out = a;
  return GZ_OK;
}

extern "C" gz_status gz_adamw_destroy(gz_adamw* a) {
  if (!a) return GZ_OK;
  if (a->arena) {
    Device on(a->device);
    cudaFree(a->arena);
  }
  delete a;
  return GZ_OK;
}

extern "C" gz_status gz_adamw_step(gz_adamw* a, const void* const* d_grads, const int32_t* grad_dtypes,
                                   const gz_adamw_config* cfg, float* d_norm, void* stream) {
  const char* who = "gz_adamw_step";
  if (!a || !cfg || (a->count > 0 && !d_grads)) return bad(who, "null argument");
  if (!(cfg->lr >= 0) || !isfinite(cfg->lr)) return bad(who, "lr must be finite and at least 0");
  if (!(cfg->beta1 >= 0 && cfg->beta1 < 1) || !(cfg->beta2 >= 0 && cfg->beta2 < 1)) return bad(who, "betas must be in [0, 1)");
  if (!(cfg->eps >= 0) || !isfinite(cfg->eps)) return bad(who, "eps must be finite and at least 0");
  if (!(cfg->max_norm >= 0)) return bad(who, "max_norm must be at least 0");
  if (cfg->step < 0) return bad(who, "steps count from 1 (0: counted on the device)");
  for (int k = 0; grad_dtypes && k < a->count; ++k)
    if (grad_dtypes[k] < GZ_F32 || grad_dtypes[k] > GZ_BF16) return bad(who, "bad gradient dtype");
  Device on(a->device);
  if (!on.ok) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, a->device);
  const cudaStream_t s = (cudaStream_t)stream;
  StepArgs args{};
  args.tensors = a->d_tensors;
  args.blocks = a->blocks_per_chunk;
  args.lr = cfg->lr;
  args.beta1 = (float)cfg->beta1;
  args.one_beta1 = (float)(1.0 - cfg->beta1);
  args.beta2 = (float)cfg->beta2;
  args.one_beta2 = (float)(1.0 - cfg->beta2);
  args.eps = (float)cfg->eps;
  args.grad_scale = cfg->grad_scale;
  args.max_norm = (float)cfg->max_norm;
  if (!isfinite(args.max_norm)) args.max_norm = 0.f;  // an infinite limit clips nothing
  const bool counted = cfg->step == 0;
  args.t = cfg->step;
  args.count = a->d_count;
  if (!counted) args.timed = timed_at(cfg->step, cfg->lr, cfg->beta1, cfg->beta2, (uint32_t)cfg->seed);
  args.partial = a->d_partial;
  args.arrived = a->d_arrived;
  args.chunk_count = a->chunk_start.back();
  args.norm = d_norm ? d_norm : a->d_norm;
  if (counted || args.chunk_count == 0) {
    count_kernel<<<1, 1, 0, s>>>(a->d_count, cfg->step, cfg->lr, cfg->beta1, cfg->beta2, (uint32_t)cfg->seed);
    if (cudaError_t e = cudaGetLastError()) return cuda_failed(who, e);
  }
  if (d_norm && args.chunk_count == 0)
    if (cudaError_t e = cudaMemsetAsync(d_norm, 0, sizeof(float), s)) return cuda_failed(who, e);
  Grads g;
  for (int pass = cfg->max_norm > 0 || d_norm ? 0 : 1; pass < 2; ++pass)
    for (int k = 0; k < a->count; k += kGradsPerLaunch) {
      const int end = k + kGradsPerLaunch < a->count ? k + kGradsPerLaunch : a->count;
      const int base = a->chunk_start[k], n = a->chunk_start[end] - base;
      if (!n) continue;
      for (int i = k; i < end; ++i) {
        g.p[i - k] = d_grads[i];
        g.dtype[i - k] = (uint8_t)(grad_dtypes ? grad_dtypes[i] : GZ_F32);
      }
      args.first_tensor = k;
      args.chunks = a->d_chunks + base;
      args.chunk_base = base;
      if (pass == 0) norm_kernel<<<n, kThreads, 0, s>>>(args, g);
      else if (a->state_bits == 8) (counted ? step_kernel<8, true> : step_kernel<8, false>)<<<n, kThreads, 0, s>>>(args, g);
      else (counted ? step_kernel<32, true> : step_kernel<32, false>)<<<n, kThreads, 0, s>>>(args, g);
      if (cudaError_t e = cudaGetLastError()) return cuda_failed(who, e);
    }
  return GZ_OK;
}

extern "C" gz_status gz_adamw_get_steps(gz_adamw* a, int64_t* steps) {
  const char* who = "gz_adamw_get_steps";
  if (!a || !steps) return bad(who, "null argument");
  Device on(a->device);
  if (!on.ok) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, a->device);
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(steps, &a->d_count->t, sizeof(int64_t), cudaMemcpyDeviceToHost);
  return e == cudaSuccess ? GZ_OK : cuda_failed(who, e);
}

extern "C" gz_status gz_adamw_set_steps(gz_adamw* a, int64_t steps) {
  const char* who = "gz_adamw_set_steps";
  if (!a) return bad(who, "null argument");
  if (steps < 0) return bad(who, "steps must be at least 0");
  Device on(a->device);
  if (!on.ok) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, a->device);
  cudaError_t e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&a->d_count->t, &steps, sizeof(int64_t), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  return e == cudaSuccess ? GZ_OK : cuda_failed(who, e);
}
