// Drawing actions from rows of policy scores, and the policy loss with its
// gradient (gz_policy_sample, gz_policy_loss).  One block per row.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "gz_internal.h"
#include "gz_sm100.h"

namespace cg = cooperative_groups;

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
  int64_t first_row, end_row;  // of this launch
  int cluster;                 // blocks per row
};

constexpr int64_t kRowsPerLaunch = 1 << 26;  // rows x 16 blocks stay a valid grid
constexpr int kSliceVecs = 3200;             // 16-byte vectors of a block's slice of a row

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

// ---- loss -------------------------------------------------------------------

// What a part of a row contributes: m the largest visible score, z the sum of
// exp(x - m), mass and cross the sums of t and t (x - m).  With m = -inf
// (nothing above it so far) cross is relative to 0.
struct Part {
  float m, z, mass, cross;
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float exp_of(float d) { return sm100::ex2_approx(d * 1.44269504f); }

__device__ __forceinline__ Part merge(Part a, Part b) {
  const float m = fmaxf(a.m, b.m), ref = base_of(m);
  a.z *= a.m == m ? 1.f : exp_of(a.m - m);
  b.z *= b.m == m ? 1.f : exp_of(b.m - m);
  if (a.mass != 0.f) a.cross += a.mass * (base_of(a.m) - ref);
  if (b.mass != 0.f) b.cross += b.mass * (base_of(b.m) - ref);
  return {m, a.z + b.z, a.mass + b.mass, a.cross + b.cross};
}

// Maximum over the warp's lanes (no lane holds a NaN).
__device__ __forceinline__ float warp_max(float x) {
  const uint32_t k = __reduce_max_sync(~0u, order_key(x));
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Sums over the warp's lanes, of parts relative to the same m.
template <bool kDense>
__device__ __forceinline__ Part warp_sum(Part p) {
  for (int o = 16; o; o >>= 1) {
    p.z += __shfl_xor_sync(~0u, p.z, o);
    if (kDense) {
      p.mass += __shfl_xor_sync(~0u, p.mass, o);
      p.cross += __shfl_xor_sync(~0u, p.cross, o);
    }
  }
  return p;
}

__device__ __forceinline__ void copy_async(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// V scores of a vector as floats.
template <typename T> __device__ __forceinline__ void unpack(uint4 raw, float* x) {
  const T* e = (const T*)&raw;
#pragma unroll
  for (int k = 0; k < 16 / (int)sizeof(T); ++k) x[k] = to_f32(e[k]);
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

template <int V> __device__ __forceinline__ void load_floats(const float* p, bool aligned, float* x) {
#pragma unroll
  for (int k = 0; k < V; k += 4)
    if (aligned) *(float4*)(x + k) = __ldg((const float4*)(p + k));
    else
      for (int i = k; i < k + 4; ++i) x[i] = __ldg(p + i);
}

// One row's pointers and how it splits: `head` scores before its first 16-byte
// boundary, `vecs` vectors of 16 bytes, the rest after the last boundary
// (ends = head + rest, at most 14).
template <typename T> struct LossRow {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* x;
  const uint8_t* mask;
  const float* target;
  T* grad;
  int actions, head, vecs, ends, label;
  float label_x;
  bool mask_aligned, target_aligned, grad_aligned;

  __device__ LossRow(const LossArgs& a, int64_t row, bool dense) {
    actions = a.rows.actions;
    x = (const T*)a.rows.logits + row * a.rows.logits_stride;
    mask = a.rows.mask ? a.rows.mask + row * a.rows.mask_stride : nullptr;
    target = dense ? a.target + row * a.target_stride : nullptr;
    grad = a.grad ? (T*)a.grad + row * a.grad_stride : nullptr;
    head = min(actions, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    vecs = (actions - head) / V;
    ends = actions - vecs * V;
    mask_aligned = (((uintptr_t)mask + head) & (V - 1)) == 0;
    target_aligned = (((uintptr_t)target + 4 * head) & 15) == 0;
    grad_aligned = (((uintptr_t)grad + sizeof(T) * head) & 15) == 0;
    // a label's score comes straight from memory, in every thread
    label = -1;
    label_x = 0.f;
    if (!dense) {
      label = a.label[row];
      if (label < 0 || label >= actions || (mask && !mask[label])) label = -1;
      else label_x = to_f32(x[label]);
    }
  }
  __device__ int end_index(int i) const { return i < head ? i : actions - ends + i; }
  __device__ uint32_t seen(int v) const {
    return mask ? visible_bits<V>(mask + head + v * V, mask_aligned) : (1u << V) - 1;
  }
  __device__ bool seen_at(int j) const { return !mask || __ldg(mask + j); }
  __device__ void targets(int v, float* t) const { load_floats<V>(target + head + v * V, target_aligned, t); }
  // The gradient of vector v: g = exp(x - top) share - scale t where seen.
  template <bool kDense>
  __device__ void write(int v, uint4 raw, uint32_t bits, float top, float share, float scale) const {
    float g[V];
    if (bits) {
      float t[V];
      unpack<T>(raw, g);
      if (kDense) targets(v, t);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        g[k] = exp_of(g[k] - top) * share;
        if (kDense) g[k] -= scale * t[k];
        if (!(bits >> k & 1)) g[k] = 0.f;
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = 0.f;
    }
    const unsigned at = (unsigned)(label - head - v * V);
    if (!kDense && at < V) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k == (int)at) g[k] -= scale;
    }
    store(v, g);
  }
  __device__ void store(int v, const float* g) const {
    T* to = grad + head + v * V;
    if (grad_aligned) {
      uint4 out;
      T* o = (T*)&out;
#pragma unroll
      for (int k = 0; k < V; ++k) o[k] = from_f32<T>(g[k]);
      *(uint4*)to = out;
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) to[k] = from_f32<T>(g[k]);
    }
  }
};

// A row's loss and the factors of its gradient.
struct Result {
  float top, share, scale, loss;
};

template <bool kDense>
__device__ __forceinline__ Result result_of(Part p, const LossArgs& a, int64_t row, int label, float label_x) {
  const bool live = p.m != -INFINITY || p.z != p.z;
  const float top = base_of(p.m), w = a.weight ? a.weight[row] : 1.f;
  if (!kDense) {
    p.mass = label >= 0 ? 1.f : 0.f;
    p.cross = label >= 0 ? label_x - top : 0.f;
  }
  const float scale = live ? w * a.scale : 0.f;
  return {top, live ? scale * (p.mass / p.z) : 0.f, scale, live ? w * (p.mass * logf(p.z) - p.cross) : 0.f};
}

// Adds a vector's visible scores to the sums relative to p.m.
template <typename T, bool kDense>
__device__ __forceinline__ void add_vector(Part& p, uint4 raw, uint32_t bits, const LossRow<T>& r, int v) {
  constexpr int V = 16 / (int)sizeof(T);
  const float ref = base_of(p.m);
  float f[V], t[V];
  unpack<T>(raw, f);
  if (kDense) r.targets(v, t);
#pragma unroll
  for (int k = 0; k < V; ++k)
    if (bits >> k & 1) {
      const float d = f[k] - ref;
      p.z += exp_of(d);
      if (kDense) {
        p.mass += t[k];
        if (t[k] != 0.f) p.cross += t[k] * d;
      }
    }
}

// Short rows: a warp each, four a block, scores in registers.
constexpr int kWarpVecs = 4;  // 16-byte vectors a lane
template <typename T, bool kDense>
__global__ void __launch_bounds__(128) loss_warp_kernel(LossArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lane = threadIdx.x % 32;
  const int64_t row = a.first_row + (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= a.end_row) return;
  const LossRow<T> r(a, row, kDense);
  uint32_t seen[kWarpVecs];
  uint4 raw[kWarpVecs];
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i) {
    const int v = i * 32 + lane;
    seen[i] = v < r.vecs ? r.seen(v) : 0;
    if (seen[i]) raw[i] = __ldg((const uint4*)(r.x + r.head) + v);
  }
  const int ej = r.end_index(lane);
  const bool end_seen = lane < r.ends && r.seen_at(ej);
  const float ex = end_seen ? to_f32(r.x[ej]) : -INFINITY, et = kDense && end_seen ? r.target[ej] : 0.f;

  Part p{ex, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i) {
    float f[V];
    unpack<T>(raw[i], f);
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (seen[i] >> k & 1) p.m = fmaxf(p.m, f[k]);
  }
  p.m = warp_max(fmaxf(p.m, -INFINITY));
  const float top = base_of(p.m);
  if (end_seen) {
    p.z = exp_of(ex - top);
    p.mass = et;
    if (et != 0.f) p.cross = et * (ex - top);
  }
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i)
    if (seen[i]) add_vector<T, kDense>(p, raw[i], seen[i], r, i * 32 + lane);
  p = warp_sum<kDense>(p);
  const Result q = result_of<kDense>(p, a, row, r.label, r.label_x);
  if (lane == 0) a.loss[row] = q.loss;
  if (!r.grad) return;
  if (lane < r.ends)
    r.grad[ej] = from_f32<T>(end_seen ? exp_of(ex - q.top) * q.share - q.scale * (kDense ? et : ej == r.label) : 0.f);
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i)
    if (i * 32 + lane < r.vecs) r.template write<kDense>(i * 32 + lane, raw[i], seen[i], q.top, q.share, q.scale);
}

// Longer rows: a block each, or a slice of a row per block of a cluster.
//
// Bound by memory: scores, mask and targets are read once, the gradient is
// written once.  Two ways through a slice:
//  - Its scores are copied to shared memory (asynchronously, all at once, so
//    that few registers keep many bytes in flight) and passed over three times
//    there: maximum, sums, gradient.  Targets are read in the second pass and
//    again, from the caches, in the third.
//  - Under a mask that leaves at most kListed actions of the slice visible
//    (legal moves: some 30 of 4672), only these are read at all: the mask gives
//    their list in order, scores and targets are gathered, the gradient is
//    zeros plus the listed ones.  That leaves the mask's byte and the
//    gradient's bytes per action to move.
// A cluster's blocks exchange maximum and sums through distributed shared
// memory, once, each relative to its own maximum.
constexpr int kListed = 256;
constexpr int kLossThreads = 256;

template <typename T, bool kDense>
__global__ void __launch_bounds__(kLossThreads) loss_kernel(LossArgs a) {
  constexpr int V = 16 / (int)sizeof(T);
  extern __shared__ uint4 shared[];
  __shared__ Part slots[kLossThreads / 32], whole;
  __shared__ int counts[kLossThreads / 32];
  const int tid = threadIdx.x, n = blockDim.x, warps = n / 32;
  const int parts = a.cluster, rank = blockIdx.x % parts;
  const int64_t row = a.first_row + blockIdx.x / parts;
  const LossRow<T> r(a, row, kDense);
  const int per = (r.vecs + parts - 1) / parts, begin = min(r.vecs, rank * per), end = min(r.vecs, begin + per);
  const bool has_end = rank == 0 && tid < r.ends;  // the ragged scores, one a thread
  const int ej = r.end_index(tid);

  int listed = -1;  // visible actions of the slice, if they are few
  int* index = (int*)shared;
  float2* entry = (float2*)(index + kListed);  // score and target
  if (r.mask) {
    const bool end_seen = has_end && r.seen_at(ej);
    int mine = end_seen;
    for (int v = begin + tid; v < end; v += n) mine += __popc(r.seen(v));
    int before = mine;  // inclusive sum over the warp's lanes
    for (int o = 1; o < 32; o *= 2) {
      const int up = __shfl_up_sync(~0u, before, o);
      if (tid % 32 >= o) before += up;
    }
    if (tid % 32 == 31) counts[tid / 32] = before;
    __syncthreads();
    int total = 0, base = 0;
    for (int w = 0; w < warps; ++w) {
      if (w == tid / 32) base = total;
      total += counts[w];
    }
    if (total <= kListed) {
      listed = total;
      int at = base + before - mine;
      if (end_seen) index[at++] = ej;
      for (int v = begin + tid; v < end && at < base + before; v += n)
        for (uint32_t bits = r.seen(v); bits; bits &= bits - 1) index[at++] = r.head + v * V + __ffs(bits) - 1;
      if (r.grad) {
        if (has_end) r.grad[ej] = from_f32<T>(0.f);
        const float zero[V] = {};
        for (int v = begin + tid; v < end; v += n) r.store(v, zero);
      }
      __syncthreads();
      for (int i = tid; i < listed; i += n) entry[i] = {to_f32(r.x[index[i]]), kDense ? r.target[index[i]] : 0.f};
    }
  }
  Part p{-INFINITY, 0.f, 0.f, 0.f};
  float ex = -INFINITY, et = 0.f;
  bool end_seen = false;
  if (listed >= 0) {
    for (int i = tid; i < listed; i += n) p.m = fmaxf(p.m, entry[i].x);
  } else {
    for (int v = begin + tid; v < end; v += n) copy_async(&shared[v - begin], (const uint4*)(r.x + r.head) + v);
    if (has_end && r.seen_at(ej)) {
      end_seen = true;
      ex = to_f32(r.x[ej]);
      if (kDense) et = r.target[ej];
    }
    wait_copies();  // a thread reads only what it has copied itself
    p.m = fmaxf(p.m, ex);
    for (int v = begin + tid; v < end; v += n) {
      float f[V];
      unpack<T>(shared[v - begin], f);
      const uint32_t bits = r.seen(v);
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (bits >> k & 1) p.m = fmaxf(p.m, f[k]);
    }
  }
  p.m = warp_max(p.m);
  if (tid % 32 == 0) slots[tid / 32].m = p.m;
  __syncthreads();
  p.m = warp_max(tid % 32 < warps ? slots[tid % 32].m : -INFINITY);
  const float ref = base_of(p.m);
  if (listed >= 0) {
    for (int i = tid; i < listed; i += n) {
      const float2 e = entry[i];
      p.z += exp_of(e.x - ref);
      p.mass += e.y;
      if (e.y != 0.f) p.cross += e.y * (e.x - ref);
    }
  } else {
    if (end_seen) {
      p.z = exp_of(ex - ref);
      p.mass = et;
      if (et != 0.f) p.cross = et * (ex - ref);
    }
    for (int v = begin + tid; v < end; v += n)
      if (const uint32_t bits = r.seen(v)) add_vector<T, kDense>(p, shared[v - begin], bits, r, v);
  }
  p = warp_sum<kDense>(p);
  __syncthreads();  // the maxima have been read
  if (tid % 32 == 0) slots[tid / 32] = p;
  __syncthreads();
  p = slots[0];
  for (int w = 1; w < warps; ++w) {
    p.z += slots[w].z;
    p.mass += slots[w].mass;
    p.cross += slots[w].cross;
  }
  if (parts > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    if (tid == 0) whole = p;
    cluster.sync();
    p = *cluster.map_shared_rank(&whole, 0);
    for (int k = 1; k < parts; ++k) p = merge(p, *cluster.map_shared_rank(&whole, k));
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // done reading the others
  }
  const Result q = result_of<kDense>(p, a, row, r.label, r.label_x);
  if (rank == 0 && tid == 0) a.loss[row] = q.loss;
  if (r.grad) {
    if (listed >= 0) {
      for (int i = tid; i < listed; i += n) {
        const float2 e = entry[i];
        const float t = kDense ? e.y : index[i] == r.label ? 1.f : 0.f;
        r.grad[index[i]] = from_f32<T>(exp_of(e.x - q.top) * q.share - q.scale * t);
      }
    } else {
      if (has_end)
        r.grad[ej] = from_f32<T>(end_seen ? exp_of(ex - q.top) * q.share - q.scale * (kDense ? et : ej == r.label) : 0.f);
      for (int v = begin + tid; v < end; v += n)
        r.template write<kDense>(v, shared[v - begin], r.seen(v), q.top, q.share, q.scale);
    }
  }
  if (parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, bool kDense>
cudaError_t launch_loss(LossArgs a, int64_t rows, cudaStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  const int vecs = a.rows.actions / V;
  cudaError_t e = cudaSuccess;
  for (int64_t first = 0; first < rows && e == cudaSuccess; first += kRowsPerLaunch) {
    const int64_t n = rows - first < kRowsPerLaunch ? rows - first : kRowsPerLaunch;
    a.first_row = first;
    a.end_row = first + n;
    if (vecs <= 32 * kWarpVecs) {
      loss_warp_kernel<T, kDense><<<(unsigned)((n + 3) / 4), 128, 0, stream>>>(a);
      e = cudaGetLastError();
      continue;
    }
    // the slice: small enough that four blocks fit an SM's shared memory, and
    // with few rows smaller still, until the blocks fill the device
    int cluster = 1;
    while (cluster < 16 && (vecs + cluster - 1) / cluster > kSliceVecs) cluster *= 2;
    while (cluster < 16 && n * cluster < 148 && vecs / cluster >= 512) cluster *= 2;
    const int per = (vecs + cluster - 1) / cluster;
    const int threads = min(kLossThreads, max(64, (per / 8 + 31) / 32 * 32));
    const size_t smem = max((size_t)per * 16, (size_t)kListed * 12);
    a.cluster = cluster;
    auto kernel = loss_kernel<T, kDense>;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && cluster == 16)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) break;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(n * cluster));
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = cluster > 1;
    e = cudaLaunchKernelEx(&c, kernel, a);
  }
  return e;
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
  const LossArgs a{row_args(rows), d_target, target_stride, d_label, d_weight, grad_scale, d_loss, d_grad, grad_stride, 0, 0, 1};
  const cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (rows->dtype == GZ_F32) e = d_target ? launch_loss<float, true>(a, rows->rows, s) : launch_loss<float, false>(a, rows->rows, s);
  else if (rows->dtype == GZ_F16) e = d_target ? launch_loss<__half, true>(a, rows->rows, s) : launch_loss<__half, false>(a, rows->rows, s);
  else e = d_target ? launch_loss<__nv_bfloat16, true>(a, rows->rows, s) : launch_loss<__nv_bfloat16, false>(a, rows->rows, s);
  return e == cudaSuccess ? GZ_OK : set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}
