// AdamW over many tensors in one launch, states in 32 or 8 bits
// (gz_adamw_*).
//
// A plan cuts every tensor into chunks of whole 256-element blocks and keeps
// the tensors' table and the chunk list on the device; a step launches one
// block of threads per chunk.  The gradients' addresses change from step to
// step, so they travel as kernel arguments.
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

#include <new>
#include <vector>

#include "gz_internal.h"
#include "gz_round.h"

namespace gz {
namespace {

constexpr int kBlock = GZ_ADAMW_BLOCK;
constexpr int kThreads = 256;
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

struct StepArgs {
  const Tensor* tensors;
  const Chunk* chunks;     // of this launch
  int first_tensor;        // grads.p[0] belongs to it
  uint32_t blocks;         // blocks per chunk
  double lr, lr_corrected;  // lr, lr / (1 - beta1^t)
  float beta1, one_beta1, beta2, one_beta2, eps, correct2;  // correct2 = 1 / sqrt(1 - beta2^t)
  float grad_scale, max_norm;
  uint32_t key;            // of the rounding
  double* partial;         // sums of squares, one per chunk of the plan
  unsigned* arrived;
  int chunk_base, chunk_count;  // first chunk of this launch, chunks of the plan
  float* norm;
};

__device__ __forceinline__ float load_grad(const void* g, int dtype, int64_t i) {
  if (dtype == GZ_F32) return ((const float*)g)[i];
  if (dtype == GZ_F16) return __half2float(((const __half*)g)[i]);
  return __bfloat162float(((const __nv_bfloat16*)g)[i]);
}

__global__ void __launch_bounds__(kThreads) norm_kernel(StepArgs a, const __grid_constant__ Grads grads) {
  __shared__ double sums[kThreads / 32];
  __shared__ bool last;
  const Chunk c = a.chunks[blockIdx.x];
  const Tensor& t = a.tensors[c.tensor];
  const void* g = grads.p[c.tensor - a.first_tensor];
  const int dtype = grads.dtype[c.tensor - a.first_tensor];
  const int64_t begin = (int64_t)c.block * kBlock;
  const int64_t end = min(t.n, begin + (int64_t)a.blocks * kBlock);
  double sum = 0;
  if (g)
    for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
      const float x = load_grad(g, dtype, i);
      sum += (double)x * x;
    }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = sum;
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
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = sum;
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

// x (already scaled) as an 8-bit float, rounded down or up by u in [0, 1).
__device__ __forceinline__ uint8_t to_8bit(float x, float u, bool nonzero) {
  const float y = fabsf(x);
  const int e = max((int)(__float_as_uint(y) >> 23) - 127, -6);
  float q = floorf(__fadd_rn(__fmul_rn(y, power(3 - e)), u));
  if (nonzero && q == 0.f && y > 0.f) q = 1.f;
  q = copysignf(__fmul_rn(q, power(e - 3)), x);
  return (uint8_t)__nv_cvt_float_to_fp8(q, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float from_8bit(uint8_t q) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
}

__device__ __forceinline__ float warp_max(float x) {
  for (int o = 16; o; o >>= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
  return x;
}

// A warp per 256-element block, eight neighbouring elements per lane.
template <int kBits>
__global__ void __launch_bounds__(kThreads) step_kernel(StepArgs a, const __grid_constant__ Grads grads) {
  const Chunk c = a.chunks[blockIdx.x];
  const Tensor t = a.tensors[c.tensor];
  const void* g = grads.p[c.tensor - a.first_tensor];
  const int dtype = grads.dtype[c.tensor - a.first_tensor];
  if (!g) return;
  const int lane = threadIdx.x % 32;
  const float decay = (float)(1.0 - a.lr * t.lr_scale * t.weight_decay);
  const float step = (float)(a.lr_corrected * t.lr_scale);
  float scale = a.grad_scale;
  if (a.max_norm > 0.f) scale = __fmul_rn(scale, fminf(__fdiv_rn(a.max_norm, __fadd_rn(*a.norm, 1e-6f)), 1.f));
  const uint32_t blocks = (uint32_t)((t.n + kBlock - 1) / kBlock);
  const uint32_t end = min(blocks, c.block + a.blocks);
  for (uint32_t b = c.block + threadIdx.x / 32; b < end; b += kThreads / 32) {
    const int64_t at = (int64_t)b * kBlock + lane * kPerLane;
    float m[kPerLane], v[kPerLane], root[kPerLane];
    const float ms = kBits == 8 ? t.m_scale[b] : 1.f, vs = kBits == 8 ? t.v_scale[b] : 1.f;
    float m_most = 0.f, v_most = 0.f;
    for (int k = 0; k < kPerLane; ++k) {
      const int64_t i = at + k;
      m[k] = v[k] = root[k] = 0.f;
      if (i >= t.n) continue;
      const float x = __fmul_rn(load_grad(g, dtype, i), scale);
      if (kBits == 8) {
        m[k] = __fmul_rn(from_8bit(((const uint8_t*)t.m)[i]), ms);
        const float r = __fmul_rn(from_8bit(((const uint8_t*)t.v)[i]), vs);
        v[k] = __fmul_rn(r, r);
      } else {
        m[k] = ((const float*)t.m)[i];
        v[k] = ((const float*)t.v)[i];
      }
      m[k] = __fadd_rn(__fmul_rn(m[k], a.beta1), __fmul_rn(x, a.one_beta1));
      v[k] = __fadd_rn(__fmul_rn(v[k], a.beta2), __fmul_rn(__fmul_rn(x, x), a.one_beta2));
      root[k] = __fsqrt_rn(v[k]);
      const float move = __fdiv_rn(m[k], __fadd_rn(__fmul_rn(root[k], a.correct2), a.eps));
      const float p = __fsub_rn(__fmul_rn(t.param[i], decay), __fmul_rn(move, step));
      t.param[i] = p;
      if (t.copy) {
        if (t.copy_dtype == GZ_F16) ((__half*)t.copy)[i] = __float2half_rn(p);
        else ((__nv_bfloat16*)t.copy)[i] = __float2bfloat16_rn(p);
      }
      if (kBits == 32) {
        ((float*)t.m)[i] = m[k];
        ((float*)t.v)[i] = v[k];
      }
      if (isfinite(m[k])) m_most = fmaxf(m_most, fabsf(m[k]));
      if (isfinite(root[k])) v_most = fmaxf(v_most, root[k]);
    }
    if (kBits == 8) {
      const int me = scale_exponent(warp_max(m_most)), ve = scale_exponent(warp_max(v_most));
      for (int k = 0; k < kPerLane; ++k) {
        const uint32_t h = mix32((uint32_t)(t.first + at + k) + a.key);
        ((uint8_t*)t.m)[at + k] = to_8bit(__fmul_rn(m[k], power(-me)), (float)(h & 0xffffu) * 0x1p-16f, false);
        ((uint8_t*)t.v)[at + k] = to_8bit(__fmul_rn(root[k], power(-ve)), (float)(h >> 16) * 0x1p-16f, true);
      }
      if (lane == 0) {
        t.m_scale[b] = power(me);
        t.v_scale[b] = power(ve);
      }
    }
  }
}

}  // namespace
}  // namespace gz

using namespace gz;

struct gz_adamw {
  int device = 0, state_bits = 32, count = 0;
  uint32_t blocks_per_chunk = 0;
  void* arena = nullptr;  // tensors | chunks | partial sums | counter and norm
  Tensor* d_tensors = nullptr;
  Chunk* d_chunks = nullptr;
  double* d_partial = nullptr;
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
  a->device = device;
  a->state_bits = state_bits;
  a->count = count;
  a->blocks_per_chunk = 8;
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
  a->d_arrived = (unsigned*)(p + tb + cb + pb);
  a->d_norm = (float*)(a->d_arrived + 1);
  cudaError_t e = cudaMemset(a->d_arrived, 0, 256);
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
  if (cfg->step < 1) return bad(who, "steps count from 1");
  for (int k = 0; grad_dtypes && k < a->count; ++k)
    if (grad_dtypes[k] < GZ_F32 || grad_dtypes[k] > GZ_BF16) return bad(who, "bad gradient dtype");
  Device on(a->device);
  if (!on.ok) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, a->device);
  const cudaStream_t s = (cudaStream_t)stream;
  StepArgs args{};
  args.tensors = a->d_tensors;
  args.blocks = a->blocks_per_chunk;
  args.lr = cfg->lr;
  args.lr_corrected = cfg->lr / (1.0 - pow(cfg->beta1, (double)cfg->step));
  args.beta1 = (float)cfg->beta1;
  args.one_beta1 = (float)(1.0 - cfg->beta1);
  args.beta2 = (float)cfg->beta2;
  args.one_beta2 = (float)(1.0 - cfg->beta2);
  args.eps = (float)cfg->eps;
  args.correct2 = (float)(1.0 / sqrt(1.0 - pow(cfg->beta2, (double)cfg->step)));
  args.grad_scale = cfg->grad_scale;
  args.max_norm = (float)cfg->max_norm;
  args.key = mix32((uint32_t)cfg->step * 0x9E3779B9u + (uint32_t)cfg->seed);
  args.partial = a->d_partial;
  args.arrived = a->d_arrived;
  args.chunk_count = a->chunk_start.back();
  args.norm = d_norm ? d_norm : a->d_norm;
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
      else if (a->state_bits == 8) step_kernel<8><<<n, kThreads, 0, s>>>(args, g);
      else step_kernel<32><<<n, kThreads, 0, s>>>(args, g);
      if (cudaError_t e = cudaGetLastError()) return cuda_failed(who, e);
    }
  return GZ_OK;
}
