// Drawing actions from rows of policy scores, and the policy loss with its
// gradient (gz_policy_sample, gz_policy_loss).  One block per row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "gz_internal.h"

namespace gz {
namespace {

constexpr int kThreads = 256;

template <typename T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float x) { return __float2bfloat16_rn(x); }

struct RowArgs {
  const void* logits;
  const uint8_t* mask;
  int64_t logits_stride, mask_stride;
  int actions;
};

struct SampleArgs {
  RowArgs rows;
  gz_sample_config cfg;
  const float* noise;
  int64_t noise_stride;
  int32_t* action;
  float* logp;
};

struct LossArgs {
  RowArgs rows;
  const float* target;
  int64_t target_stride;
  const int32_t* label;
  const float* weight;
  float scale;
  float* loss;
  void* grad;
  int64_t grad_stride;
};

struct MaxOp {
  template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; }
};
struct SumOp {
  template <typename V> __device__ V operator()(V a, V b) const { return a + b; }
};

// Every thread gets the reduction of all threads' x, in a fixed order.
template <typename V, typename Op>
__device__ V block_reduce(V x, Op op, V* slots) {
  for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(~0u, x, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) slots[threadIdx.x / 32] = x;
  __syncthreads();
  x = slots[0];
  for (int w = 1; w < kThreads / 32; ++w) x = op(x, slots[w]);
  return x;
}

// Order-preserving map of floats to unsigned integers (-0 below +0 is undone
// by adding 0 first).
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// exp(d) in units of 2^-44 (d <= 0): 2^18 actions sum below 2^63.
__device__ __forceinline__ uint64_t fixed_weight(float e) { return __float2ull_rd(e * 17592186044416.f); }

// The score of action j, -inf where it takes no part.
template <typename T>
__device__ __forceinline__ float score(const T* x, const uint8_t* mask, int j) {
  if (mask && !mask[j]) return -INFINITY;
  const float v = to_f32(x[j]);
  return v > -INFINITY ? fminf(v, FLT_MAX) : -INFINITY;
}

// Rank order as one number: higher scores first, at equal scores lower indices.
__device__ __forceinline__ uint64_t rank_key(float x, int j) {
  return (uint64_t)order_key(x) << 18 | (uint64_t)(GZ_POLICY_MAX_ACTIONS - 1 - j);
}

// The threshold of top_k and of top_p is the rank key of the last action kept,
// found by bisection on the key's 50 bits: each step counts (or weighs) what
// lies at or above the middle.
template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ float sf[kThreads / 32];
  __shared__ uint64_t su[kThreads / 32];
  const int64_t row = blockIdx.x;
  const int A = a.rows.actions;
  const T* x = (const T*)a.rows.logits + row * a.rows.logits_stride;
  const uint8_t* mask = a.rows.mask ? a.rows.mask + row * a.rows.mask_stride : nullptr;
  const float temperature = fminf(a.cfg.d_temperature ? a.cfg.d_temperature[row] : a.cfg.temperature, FLT_MAX);
  const float top_p = a.cfg.d_top_p ? a.cfg.d_top_p[row] : a.cfg.top_p;
  const float min_p = fminf(a.cfg.d_min_p ? a.cfg.d_min_p[row] : a.cfg.min_p, 1.f);
  const int top_k = a.cfg.d_top_k ? a.cfg.d_top_k[row] : a.cfg.top_k;
  const bool greedy = !(temperature > 0.f);

  float top = -INFINITY;
  for (int j = threadIdx.x; j < A; j += kThreads) top = fmaxf(top, score(x, mask, j));
  top = block_reduce(top, MaxOp(), sf);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) {
      a.action[row] = -1;
      if (a.logp) a.logp[row] = 0.f;
    }
    return;
  }
  auto depth = [&](float v) { return __fdiv_rn(v - top, temperature); };
  uint64_t last = 0;  // rank key of the last action kept
  if (greedy || top_k == 1 || !(top_p > 0.f)) {
    uint64_t best = 0;
    for (int j = threadIdx.x; j < A; j += kThreads) {
      const float v = score(x, mask, j);
      if (v > -INFINITY) best = MaxOp()(best, rank_key(v, j));
    }
    last = block_reduce(best, MaxOp(), su);
  } else {
    // the largest key with at least top_k keys at or above it
    if (top_k > 0 && top_k < A) {
      for (int bit = 49; bit >= 0; --bit) {
        const uint64_t mid = last | 1ull << bit;
        uint64_t c = 0;
        for (int j = threadIdx.x; j < A; j += kThreads) {
          const float v = score(x, mask, j);
          c += v > -INFINITY && rank_key(v, j) >= mid;
        }
        if (block_reduce(c, SumOp(), su) >= (uint64_t)top_k) last = mid;
      }
    }
    if (top_p < 1.f) {
      uint64_t z = 0;
      for (int j = threadIdx.x; j < A; j += kThreads) {
        const float v = score(x, mask, j);
        if (v > -INFINITY && rank_key(v, j) >= last) z += fixed_weight(expf(depth(v)));
      }
      const double goal = (double)top_p * (double)block_reduce(z, SumOp(), su);
      // the largest key with at least the goal's weight at or above it
      uint64_t cut = 0;
      for (int bit = 49; bit >= 0; --bit) {
        const uint64_t mid = cut | 1ull << bit;
        uint64_t s = 0;
        for (int j = threadIdx.x; j < A; j += kThreads) {
          const float v = score(x, mask, j);
          if (v > -INFINITY && rank_key(v, j) >= mid) s += fixed_weight(expf(depth(v)));
        }
        if ((double)block_reduce(s, SumOp(), su) >= goal) cut = mid;
      }
      last = MaxOp()(last, cut);
    }
  }
  // the draw among the kept actions, and their weight
  const float* noise = a.noise ? a.noise + row * a.noise_stride : nullptr;
  uint64_t best = 0, z = 0;
  for (int j = threadIdx.x; j < A; j += kThreads) {
    const float v = score(x, mask, j);
    if (v == -INFINITY || rank_key(v, j) < last) continue;
    float s = 0.f;
    if (!greedy) {
      const float d = depth(v), e = expf(d);
      if (e < min_p) continue;
      z += fixed_weight(e);
      s = d + (noise ? noise[j] : 0.f);
      if (!(s >= -INFINITY)) s = -INFINITY;
    }
    best = MaxOp()(best, rank_key(s, j));
  }
  z = block_reduce(z, SumOp(), su);
  best = block_reduce(best, MaxOp(), su);
  if (threadIdx.x == 0) {
    const int j = GZ_POLICY_MAX_ACTIONS - 1 - (int)(best & (GZ_POLICY_MAX_ACTIONS - 1));
    a.action[row] = j;
    if (a.logp) a.logp[row] = greedy ? 0.f : depth(score(x, mask, j)) - logf((float)((double)z * 0x1p-44));
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) loss_kernel(LossArgs a) {
  __shared__ float sf[kThreads / 32];
  const int64_t row = blockIdx.x;
  const int A = a.rows.actions;
  const T* x = (const T*)a.rows.logits + row * a.rows.logits_stride;
  const uint8_t* mask = a.rows.mask ? a.rows.mask + row * a.rows.mask_stride : nullptr;
  const float* target = a.target ? a.target + row * a.target_stride : nullptr;
  const int label = a.target ? -1 : a.label[row];
  T* grad = a.grad ? (T*)a.grad + row * a.grad_stride : nullptr;

  float top = -INFINITY;
  bool nan = false;
  for (int j = threadIdx.x; j < A; j += kThreads) {
    if (mask && !mask[j]) continue;
    const float v = to_f32(x[j]);
    nan |= v != v;
    top = fmaxf(top, v);
  }
  top = block_reduce(nan ? INFINITY : top, MaxOp(), sf);  // +inf makes the sums below NaN
  const bool live = top != -INFINITY;
  float z = 0.f, mass = 0.f, cross = 0.f;
  if (live)
    for (int j = threadIdx.x; j < A; j += kThreads) {
      if (mask && !mask[j]) continue;
      const float d = to_f32(x[j]) - top;
      z += top < INFINITY ? expf(d) : NAN;
      const float t = target ? target[j] : (j == label ? 1.f : 0.f);
      mass += t;
      if (t != 0.f) cross += t * d;
    }
  z = block_reduce(z, SumOp(), sf);
  mass = block_reduce(mass, SumOp(), sf);
  cross = block_reduce(cross, SumOp(), sf);
  const float w = a.weight ? a.weight[row] : 1.f;
  if (threadIdx.x == 0) a.loss[row] = live ? w * (mass * logf(z) - cross) : 0.f;
  if (!grad) return;
  const float share = mass / z, scale = w * a.scale;
  for (int j = threadIdx.x; j < A; j += kThreads) {
    float g = 0.f;
    if (live && !(mask && !mask[j])) {
      const float t = target ? target[j] : (j == label ? 1.f : 0.f);
      g = scale * (expf(to_f32(x[j]) - top) * share - t);
    }
    grad[j] = from_f32<T>(g);
  }
}

gz_status bad(const char* who, const char* what) { return set_last_error(GZ_ERR_INVALID_ARG, "%s: %s", who, what); }

gz_status check_rows(const gz_policy_rows* r, const char* who) {
  if (!r) return bad(who, "null argument");
  if (r->rows < 0 || r->rows > INT32_MAX) return bad(who, "rows must be 0 .. 2^31 - 1");
  if (r->actions < 1 || r->actions > GZ_POLICY_MAX_ACTIONS)
    return set_last_error(GZ_ERR_INVALID_ARG, "%s: actions must be 1 .. %d", who, GZ_POLICY_MAX_ACTIONS);
  if (r->dtype < GZ_F32 || r->dtype > GZ_BF16) return bad(who, "bad dtype");
  if (r->logits_stride < 0 || r->mask_stride < 0) return bad(who, "negative stride");
  if (r->rows > 0 && !r->logits) return bad(who, "null logits");
  return GZ_OK;
}

RowArgs row_args(const gz_policy_rows* r) {
  return {r->logits, r->mask, r->logits_stride, r->mask_stride, r->actions};
}

gz_status launched(const char* who) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GZ_OK : set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}

}  // namespace
}  // namespace gz

using namespace gz;

extern "C" gz_status gz_policy_sample(const gz_policy_rows* rows, const gz_sample_config* cfg, const float* d_noise,
                                      int64_t noise_stride, int32_t* d_action, float* d_logp, void* stream) {
  const char* who = "gz_policy_sample";
  if (gz_status s = check_rows(rows, who)) return s;
  if (!cfg) return bad(who, "null argument");
  if (!cfg->d_temperature && !(cfg->temperature >= 0.f)) return bad(who, "temperature must be at least 0");
  if (!cfg->d_top_k && cfg->top_k < 0) return bad(who, "top_k must be at least 0");
  if (!cfg->d_top_p && !(cfg->top_p >= 0.f && cfg->top_p <= 1.f)) return bad(who, "top_p must be 0 .. 1");
  if (!cfg->d_min_p && !(cfg->min_p >= 0.f && cfg->min_p <= 1.f)) return bad(who, "min_p must be 0 .. 1");
  if (noise_stride < 0) return bad(who, "negative stride");
  if (rows->rows == 0) return GZ_OK;
  if (!d_action) return bad(who, "null actions");
  const SampleArgs a{row_args(rows), *cfg, d_noise, noise_stride, d_action, d_logp};
  const cudaStream_t s = (cudaStream_t)stream;
  const unsigned grid = (unsigned)rows->rows;
  if (rows->dtype == GZ_F32) sample_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else if (rows->dtype == GZ_F16) sample_kernel<__half><<<grid, kThreads, 0, s>>>(a);
  else sample_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  return launched(who);
}

extern "C" gz_status gz_policy_loss(const gz_policy_rows* rows, const float* d_target, int64_t target_stride,
                                    const int32_t* d_label, const float* d_weight, float grad_scale, float* d_loss,
                                    void* d_grad, int64_t grad_stride, void* stream) {
  const char* who = "gz_policy_loss";
  if (gz_status s = check_rows(rows, who)) return s;
  if (target_stride < 0 || grad_stride < 0) return bad(who, "negative stride");
  if (rows->rows == 0) return GZ_OK;
  if (!d_target == !d_label) return bad(who, "give either targets or labels");
  if (!d_loss) return bad(who, "null loss");
  if (d_grad && rows->rows > 1 && grad_stride < rows->actions) return bad(who, "gradient rows overlap");
  const LossArgs a{row_args(rows), d_target, target_stride, d_label, d_weight, grad_scale, d_loss, d_grad, grad_stride};
  const cudaStream_t s = (cudaStream_t)stream;
  const unsigned grid = (unsigned)rows->rows;
  if (rows->dtype == GZ_F32) loss_kernel<float><<<grid, kThreads, 0, s>>>(a);
  else if (rows->dtype == GZ_F16) loss_kernel<__half><<<grid, kThreads, 0, s>>>(a);
  else loss_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  return launched(who);
}
