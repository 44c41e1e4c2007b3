// The policy loss and its gradient (gz_policy_loss).
#include "gz_policy.h"

namespace gz {
namespace policy {
namespace {

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
constexpr int kSharedPerSM = 227 * 1024;
constexpr int kSliceVecs = 6400;             // 16-byte vectors of a block's slice of a row: two blocks fit an SM
constexpr int kMostScores = (kSliceVecs + 8) * 16;  // bytes of a slice, its end rounded up to 16 actions

// What a part of a row contributes: m the largest visible score, z the sum of
// exp(x - m), mass and cross the sums of t and t (x - m).  With m = -inf
// (nothing above it so far) cross is relative to 0.
struct Part {
  float m, z, mass, cross;
};

__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ float exp_of(float d) { return sm100::ex2_approx(d * 1.44269504f); }

// exp(x - ref) as one multiply-add and a power of two, 2^(a x + c): c rounds
// -a ref, and the factor 2^(a ref + c) that this leaves on every term is taken
// out of the sums by `fix`.  Its exponent is up to half a unit in the last place
// of 1.44 |ref|, so below |ref| = 2^30 at most 64, and both powers stay far
// within range.  From 2^30 on the next float below ref is 64 or more away: all
// that differs from ref adds nothing to a sum that ref's 1 is in, at a = 1
// (2^-64) as at a = log2 e (e^-64), and a = 1 needs no rounding.
struct Scale {
  float a, c, fix;
  __device__ explicit Scale(float ref) {
    a = fabsf(ref) < 0x1p30f ? 1.44269504f : 1.f;
    c = -__fmul_rn(ref, a);
    fix = sm100::ex2_approx(-__fmaf_rn(ref, a, c));
  }
  __device__ float operator()(float x) const { return sm100::ex2_approx(__fmaf_rn(x, a, c)); }
  __device__ float2 operator()(float2 x) const {
    const float2 y = __ffma2_rn(x, make_float2(a, a), make_float2(c, c));
    return make_float2(sm100::ex2_approx(y.x), sm100::ex2_approx(y.y));
  }
};

__device__ __forceinline__ Part merge(Part a, Part b) {
  const float m = fmaxf(a.m, b.m), ref = base_of(m);
  a.z *= a.m == m ? 1.f : exp_of(a.m - m);
  b.z *= b.m == m ? 1.f : exp_of(b.m - m);
  if (a.mass != 0.f) a.cross += a.mass * (base_of(a.m) - ref);
  if (b.mass != 0.f) b.cross += b.mass * (base_of(b.m) - ref);
  return {m, a.z + b.z, a.mass + b.mass, a.cross + b.cross};
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
// Ends a group of copies; waits for all of this thread's groups but the last kLeft.
__device__ __forceinline__ void end_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

template <int V> __device__ __forceinline__ void load_floats(const float* p, bool aligned, float* x) {
#pragma unroll
  for (int k = 0; k < V; k += 4)
    if (aligned) *(float4*)(x + k) = __ldg((const float4*)(p + k));
    else
      for (int i = k; i < k + 4; ++i) x[i] = __ldg(p + i);
}

// A row's loss and the factors of its gradient.
struct Result {
  Scale e;
  float share, scale, loss;
};

// Actions of each of a row's slices: whole groups of 16, so that all slices
// have their row's alignment.
__host__ __device__ inline int slice_actions(int actions, int slices) {
  return slices == 1 ? actions : (actions + slices * 16 - 1) / (slices * 16) * 16;
}

// A row's slice: its pointers and how it splits into `head` scores before its
// first 16-byte boundary, `vecs` vectors of 16 bytes and the rest after the
// last boundary (ends = head + rest, at most 14).  The label counts from the
// slice's first action, and lies outside where it is another slice's.
template <typename T> struct LossRow {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* x;
  const uint8_t* mask;
  const float* target;
  T* grad;
  int actions, head, vecs, ends, label;
  float label_x, weight;
  bool labelled, mask_aligned, target_aligned, grad_aligned;

  __device__ LossRow(const LossArgs& a, int64_t row, int rank, bool dense) {
    const int size = slice_actions(a.rows.actions, a.cluster), first = rank * size;
    actions = min(size, a.rows.actions - first);
    x = (const T*)a.rows.logits + row * a.rows.logits_stride;
    mask = a.rows.mask ? a.rows.mask + row * a.rows.mask_stride : nullptr;
    // a label's score comes straight from memory, in every thread
    label = -1 - first;
    label_x = 0.f;
    if (!dense) {
      const int j = a.label[row];
      if (j >= 0 && j < a.rows.actions && !(mask && !mask[j])) {
        label = j - first;
        label_x = to_f32(x[j]);
      }
    }
    labelled = label >= -first;
    weight = a.weight ? a.weight[row] : 1.f;
    x += first;
    if (mask) mask += first;
    target = dense ? a.target + row * a.target_stride + first : nullptr;
    grad = a.grad ? (T*)a.grad + row * a.grad_stride + first : nullptr;
    head = min(actions, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    vecs = (actions - head) / V;
    ends = actions - vecs * V;
    mask_aligned = (((uintptr_t)mask + head) & (V - 1)) == 0;
    target_aligned = (((uintptr_t)target + 4 * head) & 15) == 0;
    grad_aligned = (((uintptr_t)grad + sizeof(T) * head) & 15) == 0;
  }
  __device__ int end_index(int i) const { return i < head ? i : actions - ends + i; }
  __device__ uint32_t seen(int v) const {
    return mask ? visible_bits<V>(mask + head + v * V, mask_aligned) : (1u << V) - 1;
  }
  __device__ bool seen_at(int j) const { return !mask || __ldg(mask + j); }
  __device__ void targets(int v, float* t) const { load_floats<V>(target + head + v * V, target_aligned, t); }
  // The gradient of vector v, exp(x - top) share - scale t where seen; a
  // label's -scale is not in it.
  template <bool kDense, bool kMasked>
  __device__ void write(int v, uint4 raw, uint32_t bits, const Scale& e, float share, float scale) const {
    float g[V], t[V];
    unpack<T>(raw, g);
    if (kDense) targets(v, t);
#pragma unroll
    for (int k = 0; k < V; k += 2) {
      float2 y = __fmul2_rn(e(make_float2(g[k], g[k + 1])), make_float2(share, share));
      if (kDense) y = __ffma2_rn(make_float2(-scale, -scale), make_float2(t[k], t[k + 1]), y);
      g[k] = !kMasked || (bits >> k & 1) ? y.x : 0.f;
      g[k + 1] = !kMasked || (bits >> k & 2) ? y.y : 0.f;
    }
    store(v, g);
  }
  // Stores the label's gradient over the one written with its vector, by the
  // thread that wrote that: thread tid of n has the vectors tid, tid + n, ...
  __device__ void store_label(int tid, int n, const Result& q) const {
    const int at = label - head;
    if (at >= 0 && at < vecs * V && at / V % n == tid) grad[label] = from_f32<T>(q.e(label_x) * q.share - q.scale);
  }
  __device__ void store(int v, const float* g) const {
    T* to = grad + head + v * V;
    if (grad_aligned) {
      *(uint4*)to = pack<T>(g);
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) to[k] = from_f32<T>(g[k]);
    }
  }
};

template <bool kDense>
__device__ __forceinline__ Result result_of(Part p, float grad_scale, float w, bool labelled, float label_x) {
  const bool live = p.m != -INFINITY || p.z != p.z;
  const float top = base_of(p.m);
  if (!kDense) {
    p.mass = labelled ? 1.f : 0.f;
    p.cross = labelled ? label_x - top : 0.f;
  }
  const float scale = live ? w * grad_scale : 0.f;
  const Scale e(top);
  return {e, live ? scale * (p.mass / p.z) * e.fix : 0.f, scale, live ? w * (p.mass * logf(p.z) - p.cross) : 0.f};
}

// Adds a vector's visible scores to the sums relative to ref; z in two halves.
template <bool kDense, bool kMasked, typename T>
__device__ __forceinline__ void add_vector(Part& p, float2& z, uint4 raw, uint32_t bits, const LossRow<T>& r, int v,
                                           const Scale& scale, float ref) {
  constexpr int V = 16 / (int)sizeof(T);
  float f[V], t[V];
  unpack<T>(raw, f);
  if (kDense) r.targets(v, t);
#pragma unroll
  for (int k = 0; k < V; k += 2) {
    float2 e = scale(make_float2(f[k], f[k + 1]));
    if (kMasked) {
      if (!(bits >> k & 1)) e.x = 0.f;
      if (!(bits >> k & 2)) e.y = 0.f;
    }
    z = __fadd2_rn(z, e);
  }
  if (kDense) {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if ((!kMasked || (bits >> k & 1)) && t[k] != 0.f) {
        p.mass += t[k];
        p.cross += t[k] * (f[k] - ref);
      }
  }
}

// Short rows: a warp each, four a block, scores in registers.
constexpr int kWarpVecs = 4;  // 16-byte vectors a lane
template <typename T, bool kDense>
__global__ void __launch_bounds__(128) loss_warp_kernel(LossArgs a) {
  const int lane = threadIdx.x % 32;
  const int64_t row = a.first_row + (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= a.end_row) return;
  const LossRow<T> r(a, row, 0, kDense);
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
  for (int i = 0; i < kWarpVecs; ++i)
    if (seen[i]) p.m = max_vector<true, T>(p.m, raw[i], seen[i]);
  p.m = warp_max(fmaxf(p.m, -INFINITY));
  const float top = base_of(p.m);
  const Scale e(top);
  if (end_seen) {
    p.z = e(ex);
    p.mass = et;
    if (et != 0.f) p.cross = et * (ex - top);
  }
  float2 z = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i)
    if (seen[i]) add_vector<kDense, true>(p, z, raw[i], seen[i], r, i * 32 + lane, e, top);
  p.z += z.x + z.y;
  p = warp_sum<kDense>(p);
  p.z *= e.fix;
  const Result q = result_of<kDense>(p, a.scale, r.weight, r.labelled, r.label_x);
  if (lane == 0) a.loss[row] = q.loss;
  if (!r.grad) return;
  if (lane < r.ends)
    r.grad[ej] = from_f32<T>(end_seen ? q.e(ex) * q.share - q.scale * (kDense ? et : ej == r.label) : 0.f);
#pragma unroll
  for (int i = 0; i < kWarpVecs; ++i) {
    const int v = i * 32 + lane;
    if (v >= r.vecs) continue;
    const float zero[16 / sizeof(T)] = {};
    if (seen[i]) r.template write<kDense, true>(v, raw[i], seen[i], q.e, q.share, q.scale);
    else r.store(v, zero);
  }
  if (!kDense) r.store_label(lane, 32, q);
}

// Longer rows: a block each, or a slice of a row per block of a cluster, in
// two ways.
//  - Dense: scores (from shared memory, where a copy without registers has put
//    them), mask and targets are passed over twice, for the sums and for the
//    gradient; what is not in shared memory comes from the caches the second
//    time.  Scores, mask and targets are read and the gradient is written once:
//    bound by memory, next by the two exponentials an action.
//  - Listed: under a mask that leaves at most kListed actions of the slice
//    visible (legal moves: some 30 of 4672) only these are read at all.  The
//    mask gives their list in an order fixed by position, scores and targets
//    are gathered, the gradient is zeros with the listed ones stored over
//    them: the mask's byte and the gradient's bytes are what is left to move,
//    209 MB of 497 on 8192 rows of 4672 in 46 us, 4.6 TB/s.
// A cluster's blocks exchange maximum and sums through distributed shared
// memory, once.
constexpr int kListed = 256;
constexpr int kLossThreads = 384, kListedThreads = 256;  // most threads of a block

constexpr int kMostSlices = 16;

struct LossShared {
  Part slots[kLossThreads / 32], merged[2][kLossThreads / 32];
  int counts[kListedThreads / 32];
  alignas(16) Part inbox[2][kMostSlices];  // the cluster's parts, the block's rows in turn
  uint64_t filled[2];
  int gave_up;
};

// The cluster's blocks send each other their parts: 16 bytes each into every
// inbox, whose barrier counts the bytes; nobody waits for another's copies.
__device__ __forceinline__ void open_inbox(int cluster, LossShared& sh) {
  if (cluster == 1) return;
  if (threadIdx.x == 0) {
    sh.gave_up = 0;
    sm100::mbar_init(&sh.filled[0], 1);
    sm100::mbar_init(&sh.filled[1], 1);
    sm100::fence_mbar_init();
  }
  __syncthreads();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void wait_cluster() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// All blocks' parts, joined in the blocks' order, for the block's row number
// `turn`, once all are there.  A wait that lasts longer than `limit_ns` gives
// up: its thread gets a NaN for every sum, and its block for all rows after
// this one, without sending or waiting again (the others, then short of its
// parts, give up in their turn).  So what is written is right or NaN, a program
// loses a few waits at most, and no inbox gets a part of another row's.
constexpr uint64_t kWaitLimitNs = 4000000000ull;

__device__ __forceinline__ Part no_part() { return {NAN, NAN, NAN, NAN}; }
__device__ __forceinline__ bool gave_up(const LossShared& sh) { return *(const volatile int*)&sh.gave_up; }

__device__ __forceinline__ void send_part(Part p, int cluster, int rank, unsigned turn, LossShared& sh) {
  if (threadIdx.x >= cluster) return;
  uint32_t to, bar;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(sm100::smem_u32(&sh.inbox[turn & 1][rank])), "r"(threadIdx.x));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(sm100::smem_u32(&sh.filled[turn & 1])), "r"(threadIdx.x));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
               "r"(__float_as_uint(p.m)), "r"(__float_as_uint(p.z)), "r"(__float_as_uint(p.mass)),
               "r"(__float_as_uint(p.cross)), "r"(bar)
               : "memory");
}

__device__ __forceinline__ Part receive_parts(int cluster, unsigned turn, LossShared& sh, uint64_t limit_ns) {
  const Part* inbox = sh.inbox[turn & 1];
  uint64_t* filled = &sh.filled[turn & 1];
  if (threadIdx.x == 0) sm100::mbar_arrive_expect_tx(filled, cluster * sizeof(Part));
  const uint64_t began = sm100::global_timer_ns();
  uint32_t done = 0;
  while (!done) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(sm100::smem_u32(filled)), "r"(turn >> 1 & 1)
        : "memory");
    if (!done && sm100::global_timer_ns() - began > limit_ns) {
      *(volatile int*)&sh.gave_up = 1;
      return no_part();
    }
  }
  Part p = inbox[0];
  for (int k = 1; k < cluster; ++k) p = merge(p, inbox[k]);
  return p;
}

// Both.  A block is at most one row ahead of the others (it needs their parts),
// so two inboxes in turn never mix.
__device__ __forceinline__ Part exchange(Part p, int cluster, int rank, unsigned turn, LossShared& sh) {
  if (turn == 0) wait_cluster();  // every inbox is open
  if (gave_up(sh)) return no_part();
  send_part(p, cluster, rank, turn, sh);
  return receive_parts(cluster, turn, sh, kWaitLimitNs);
}

// Maximum over the block.
__device__ __forceinline__ float block_max(float m, LossShared& sh) {
  m = warp_max(m);
  if (threadIdx.x % 32 == 0) sh.slots[threadIdx.x / 32].m = m;
  __syncthreads();
  m = warp_max(threadIdx.x % 32 < blockDim.x / 32 ? sh.slots[threadIdx.x % 32].m : -INFINITY);
  __syncthreads();
  return m;
}

// Sums over the block of parts relative to one m.
template <bool kDense>
__device__ __forceinline__ Part block_sum(Part p, LossShared& sh) {
  p = warp_sum<kDense>(p);
  if (threadIdx.x % 32 == 0) sh.slots[threadIdx.x / 32] = p;
  __syncthreads();
  p = threadIdx.x % 32 < blockDim.x / 32 ? sh.slots[threadIdx.x % 32] : Part{p.m, 0.f, 0.f, 0.f};
  return warp_sum<kDense>(p);
}

// A part relative to m, which is no less than its own reference.
template <bool kDense> __device__ __forceinline__ Part rebased(Part p, float m) {
  if (p.m != m) {
    p.z *= exp_of(p.m - m);
    if (kDense && p.mass != 0.f) p.cross += p.mass * (base_of(p.m) - base_of(m));
    p.m = m;
  }
  return p;
}

// Sums over the block of parts each relative to its own m; `slots` are not in
// use until the block has met again.
template <bool kDense>
__device__ __forceinline__ Part block_merge(Part p, Part* slots) {
  p = warp_sum<kDense>(rebased<kDense>(p, warp_max(p.m)));
  if (threadIdx.x % 32 == 0) slots[threadIdx.x / 32] = p;
  __syncthreads();
  p = threadIdx.x % 32 < blockDim.x / 32 ? slots[threadIdx.x % 32] : Part{-INFINITY, 0.f, 0.f, 0.f};
  return warp_sum<kDense>(rebased<kDense>(p, warp_max(p.m)));
}

// Joins the cluster's parts and stores the row's loss.
template <bool kDense>
__device__ __forceinline__ Result join(Part p, const LossArgs& a, int64_t row, int rank, unsigned turn, float weight,
                                       bool labelled, float label_x, LossShared& sh) {
  if (a.cluster > 1) p = exchange(p, a.cluster, rank, turn, sh);
  const Result q = result_of<kDense>(p, a.scale, weight, labelled, label_x);
  if (rank == 0 && threadIdx.x == 0) a.loss[row] = q.loss;
  return q;
}
// A block's shared memory stays until the others have sent what they send.
__device__ __forceinline__ void leave(int cluster) {
  if (cluster == 1) return;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  wait_cluster();
}

// Sums may be taken relative to any score near the row's largest: those beyond
// 2^64, 0 or NaN are taken again, relative to the maximum.
__device__ __forceinline__ bool in_range(float z) { return z > 0.f && z < 0x1p64f; }

// The dense way under a mask: scores, mask and targets are read from memory for
// the sums and again, from the caches, for the gradient.  The sums' first
// reference is the largest of a sample, each thread's first vector; where the
// sample has nothing above -inf (the row may begin with hidden actions) the
// maximum is looked for before any sum counts.  A call of its own, so that the
// listed way does not pay for its registers.
template <typename T, bool kDense>
__device__ __noinline__ void masked_dense_slice(const LossArgs& a, LossShared& sh) {
  const int tid = threadIdx.x, n = blockDim.x;
  const int rank = blockIdx.x % a.cluster;
  const int64_t row = a.first_row + blockIdx.x / a.cluster;
  const LossRow<T> r(a, row, rank, kDense);
  const uint4* from = (const uint4*)(r.x + r.head);
  const bool has_end = tid < r.ends;  // the ragged scores, one a thread
  const int ej = r.end_index(tid);
  const bool end_seen = has_end && r.seen_at(ej);
  const float ex = end_seen ? to_f32(r.x[ej]) : -INFINITY, et = kDense && end_seen ? r.target[ej] : 0.f;
  Part p{fmaxf(ex, -INFINITY), 0.f, 0.f, 0.f};
  if (tid < r.vecs) p.m = max_vector<true, T>(p.m, __ldg(from + tid), r.seen(tid));
  for (bool sample = true;; sample = false) {
    const float m = block_max(p.m, sh), ref = base_of(m);
    const Scale scale(ref);
    p = {m, 0.f, 0.f, 0.f};
    float2 z = {end_seen ? scale(ex) : 0.f, 0.f};
    if (end_seen && et != 0.f) {
      p.mass = et;
      p.cross = et * (ex - ref);
    }
#pragma unroll 2
    for (int v = tid; v < r.vecs; v += n) add_vector<kDense, true>(p, z, __ldg(from + v), r.seen(v), r, v, scale, ref);
    p.z = z.x + z.y;
    p = block_sum<kDense>(p, sh);
    p.z *= scale.fix;
    if (!sample || (m > -INFINITY && in_range(p.z))) break;
    p.m = fmaxf(ex, -INFINITY);
    for (int v = tid; v < r.vecs; v += n) p.m = max_vector<true, T>(p.m, __ldg(from + v), r.seen(v));
    __syncthreads();  // the sums have been read
  }
  const Result q = join<kDense>(p, a, row, rank, 0, r.weight, r.labelled, r.label_x, sh);
  if (!r.grad) return;
  if (has_end)
    r.grad[ej] = from_f32<T>(end_seen ? q.e(ex) * q.share - q.scale * (kDense ? et : ej == r.label) : 0.f);
#pragma unroll 2
  for (int v = tid; v < r.vecs; v += n)
    r.template write<kDense, true>(v, __ldg(from + v), r.seen(v), q.e, q.share, q.scale);
  if (!kDense) r.store_label(tid, n, q);
}

// Non-zero bytes of a word, counted.
__device__ __forceinline__ int nonzero_bytes(uint32_t w) { return __popc(__vcmpne4(w, 0) & 0x01010101u); }

// False, with nothing done, where the slice has more than kListed visible actions.
template <typename T, bool kDense>
__device__ __forceinline__ bool listed_slice(const LossArgs& a, int* index, LossShared& sh) {
  float2* entry = (float2*)(index + kListed);  // score and target
  const int tid = threadIdx.x, n = blockDim.x;
  const int rank = blockIdx.x % a.cluster;
  const int64_t row = a.first_row + blockIdx.x / a.cluster;
  const LossRow<T> r(a, row, rank, kDense);
  // groups of 16 mask bytes, and those before and after them
  const int head = min(r.actions, (int)(-(uintptr_t)r.mask & 15));
  const int groups = (r.actions - head) / 16, ends = r.actions - groups * 16;
  const int ej = tid < head ? tid : r.actions - ends + tid;
  const uint4* group = (const uint4*)(r.mask + head);
  const bool end_seen = tid < ends && r.mask[ej];
  int mine = end_seen;
#pragma unroll 2
  for (int u = tid; u < groups; u += n) {
    const uint4 w = __ldg(group + u);
    if (w.x | w.y | w.z | w.w) mine += nonzero_bytes(w.x) + nonzero_bytes(w.y) + nonzero_bytes(w.z) + nonzero_bytes(w.w);
  }
  int at = mine;  // sum over the warp's lanes up to this one
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int up = __shfl_up_sync(~0u, at, o);
    if (tid % 32 >= o) at += up;
  }
  if (tid % 32 == 31) sh.counts[tid / 32] = at;
  __syncthreads();
  int total = 0;
  at -= mine;
#pragma unroll
  for (int w = 0; w < kListedThreads / 32; ++w)
    if (w < n / 32) {
      if (w < tid / 32) at += sh.counts[w];
      total += sh.counts[w];
    }
  if (total > kListed) return false;  // the same in all threads
  if (mine) {
    if (end_seen) index[at++] = ej, --mine;
    for (int u = tid; u < groups && mine; u += n) {
      const uint4 w = __ldg(group + u);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        for (uint32_t bits = __vcmpne4(k == 0 ? w.x : k == 1 ? w.y : k == 2 ? w.z : w.w, 0) & 0x01010101u; bits;
             bits &= bits - 1, --mine)
          index[at++] = head + u * 16 + k * 4 + (__ffs(bits) - 1) / 8;
    }
  }
  if (r.grad) {
    constexpr int V = 16 / (int)sizeof(T);
    const T zero = from_f32<T>(0.f);
    const int skip = min(r.actions, (int)(-(uintptr_t)r.grad & 15) / (int)sizeof(T));
    const int vecs = (r.actions - skip) / V, rest = r.actions - vecs * V;
    if (tid < rest) r.grad[tid < skip ? tid : r.actions - rest + tid] = zero;
    uint4* vec = (uint4*)(r.grad + skip);
#pragma unroll 4
    for (int v = tid; v < vecs; v += n) vec[v] = make_uint4(0, 0, 0, 0);
  }
  __syncthreads();
  Part p{-INFINITY, 0.f, 0.f, 0.f};
  for (int i = tid; i < total; i += n) {
    const int j = index[i];
    const float2 e = {to_f32(r.x[j]), kDense ? r.target[j] : j == r.label ? 1.f : 0.f};
    entry[i] = e;
    p.m = fmaxf(p.m, e.x);
  }
  p.m = block_max(p.m, sh);
  const float ref = base_of(p.m);
  const Scale scale(ref);
  for (int i = tid; i < total; i += n) {
    const float2 e = entry[i];
    p.z += scale(e.x);
    p.mass += e.y;
    if (e.y != 0.f) p.cross += e.y * (e.x - ref);
  }
  p = block_sum<kDense>(p, sh);
  p.z *= scale.fix;
  const Result q = join<kDense>(p, a, row, rank, 0, r.weight, r.labelled, r.label_x, sh);
  if (r.grad)
    for (int i = tid; i < total; i += n) r.grad[index[i]] = from_f32<T>(q.e(entry[i].x) * q.share - q.scale * entry[i].y);
  return true;
}

// A thread's sums over its share of a slice, relative to the largest score of
// the first vector that has one above -inf (or to a given one).
template <typename T, bool kDense> struct ShareSum {
  Part p{-INFINITY, 0.f, 0.f, 0.f};
  float2 z{0.f, 0.f};
  Scale scale{0.f};

  // From relative to nothing to relative to m.
  __device__ void refer(float m) {
    p.m = m;
    scale = Scale(base_of(m));
    if (kDense && p.mass != 0.f) p.cross -= p.mass * base_of(m);
  }
  __device__ void add(const LossRow<T>& r, int v, uint4 raw) {
    if (p.m == -INFINITY) refer(max_vector<false, T>(-INFINITY, raw, 0));
    add_vector<kDense, false>(p, z, raw, 0, r, v, scale, base_of(p.m));
  }
  __device__ void add(float x, float t) {
    if (p.m == -INFINITY) refer(fmaxf(x, -INFINITY));
    z.x += scale(x);
    if (kDense && t != 0.f) {
      p.mass += t;
      p.cross += t * (x - base_of(p.m));
    }
  }
  __device__ Part sum() const { return {p.m, (z.x + z.y) * scale.fix, p.mass, p.cross}; }
};

// Without a mask the blocks stay and take rows in turn, and one loop over a
// thread's vectors does everything at once: the row's gradient from the scores
// in shared memory, the copy of the next row's scores into the place just read,
// and, kBehind vectors behind, the next row's sums.  So reading, writing and
// both exponentials share the time: 2048 rows of 100003 bf16 scores in 168 us,
// 4.9 TB/s (a copy of these bytes takes 132 us).  In three passes with four
// blocks an SM to overlap them it took 178 us, the same loop with 512 or 256
// threads a block 174 and 179 us, with four smaller slices a row 225 us.
constexpr int kBehind = 4;

template <typename T, bool kDense>
__global__ void __launch_bounds__(kLossThreads, 2) loss_kernel(const __grid_constant__ LossArgs a) {
  extern __shared__ uint4 scores[];
  __shared__ LossShared sh;
  const int tid = threadIdx.x, n = blockDim.x, rank = blockIdx.x % a.cluster;
  const int64_t step = gridDim.x / a.cluster;
  int64_t row = a.first_row + blockIdx.x / a.cluster;
  open_inbox(a.cluster, sh);
  LossRow<T> now(a, row, rank, kDense);
  now.vecs = 0;  // nothing to write yet
  Result q{Scale(0.f), 0.f, 0.f, 0.f};
  float ex = 0.f, et = 0.f;
  unsigned turn = 0;
  for (bool first = true;; first = false) {
    // the gradient of `now` (not at first), the sums of `next`
    const int64_t next_row = first ? row : row + step;
    const bool more = next_row < a.end_row;
    LossRow<T> next(a, more ? next_row : a.first_row, rank, kDense);
    if (!more) next.vecs = 0;
    const uint4* from = (const uint4*)(next.x + next.head);
    float next_ex = 0.f, next_et = 0.f;  // the thread's ragged score
    if (more && tid < next.ends) {
      const int ej = next.end_index(tid);
      next_ex = to_f32(next.x[ej]);
      next_et = kDense ? next.target[ej] : 0.f;
    }
    ShareSum<T, kDense> sum;
    const int most = max(now.vecs, next.vecs);
    int v = tid;
    for (int k = 0; v < most; v += n, ++k) {
      if (v < now.vecs && now.grad) now.template write<kDense, false>(v, scores[v], 0, q.e, q.share, q.scale);
      if (v < next.vecs) copy_async(&scores[v], from + v);
      end_copies();
      if (k >= kBehind) {
        wait_copies<kBehind>();
        if (v - kBehind * n < next.vecs) sum.add(next, v - kBehind * n, scores[v - kBehind * n]);
      }
    }
    if (!first && now.grad) {
      const int ej = now.end_index(tid);
      if (tid < now.ends) now.grad[ej] = from_f32<T>(q.e(ex) * q.share - q.scale * (kDense ? et : ej == now.label));
      if (!kDense) now.store_label(tid, n, q);
    }
    if (!more) break;
    wait_copies<0>();
    for (v = max(tid, v - kBehind * n); v < next.vecs; v += n) sum.add(next, v, scores[v]);
    if (tid < next.ends) sum.add(next_ex, next_et);
    ex = next_ex;
    et = next_et;
    Part p = sum.sum();
    // one thread out of range makes the whole NaN
    if (!(in_range(p.z) || (p.m == -INFINITY && p.z == 0.f))) p.z = NAN;
    p = block_merge<kDense>(p, sh.merged[turn & 1]);
    if (p.z != p.z) {  // relative to the slice's maximum instead
      float m = tid < next.ends ? fmaxf(ex, -INFINITY) : -INFINITY;
      for (v = tid; v < next.vecs; v += n) m = max_vector<false, T>(m, scores[v], 0);
      m = block_max(m, sh);
      sum = ShareSum<T, kDense>();
      if (m > -INFINITY) sum.refer(m);
      for (v = tid; v < next.vecs; v += n) sum.add(next, v, scores[v]);
      if (tid < next.ends) sum.add(ex, et);
      p = block_merge<kDense>(sum.sum(), sh.slots);
      __syncthreads();
    }
    q = join<kDense>(p, a, next_row, rank, turn++, next.weight, next.labelled, next.label_x, sh);
    now = next;
    row = next_row;
  }
  leave(a.cluster);
}

template <typename T, bool kDense>
__global__ void __launch_bounds__(kListedThreads, 8) loss_masked_kernel(const __grid_constant__ LossArgs a) {
  __shared__ LossShared sh;
  __shared__ __align__(8) int list[kListed * 3];
  open_inbox(a.cluster, sh);
  if (!listed_slice<T, kDense>(a, list, sh)) {
    __syncthreads();
    masked_dense_slice<T, kDense>(a, sh);
  }
  leave(a.cluster);
}

// Two blocks that wait for parts nobody sends.  *status: 1 where every thread's
// first wait gave up, the next row was given up at once, and a row's loss and
// gradient come out as NaN; else 0.
__global__ void __cluster_dims__(2, 1, 1) wait_limit_kernel(uint64_t limit_ns, int* status) {
  __shared__ LossShared sh;
  open_inbox(2, sh);
  wait_cluster();
  Part p = receive_parts(2, 0, sh, limit_ns);
  bool fine = p.z != p.z;
  __syncthreads();
  const uint64_t began = sm100::global_timer_ns();
  p = exchange({0.f, 1.f, 1.f, 0.f}, 2, blockIdx.x, 1, sh);
  fine = fine && p.z != p.z && sm100::global_timer_ns() - began < limit_ns;
  const Result dense = result_of<true>(p, 1.f, 1.f, false, 0.f), label = result_of<false>(p, 1.f, 1.f, true, 0.f);
  for (const Result& q : {dense, label}) {
    const float grad = q.e(0.f) * q.share;
    fine = fine && q.loss != q.loss && grad != grad;
  }
  if (!fine) atomicAnd(status, 0);
  leave(2);
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
    // the slice: small enough that two blocks fit an SM's shared memory, and
    // with few rows smaller still, until the blocks fill the device
    int cluster = 1;
    while (cluster < 16 && (vecs + cluster - 1) / cluster > kSliceVecs) cluster *= 2;
    while (cluster < 16 && n * cluster < 148 && vecs / cluster >= 512) cluster *= 2;
    const int per = slice_actions(a.rows.actions, cluster) / V;
    const bool masked = a.rows.mask != nullptr;
    const int threads = masked ? min(kListedThreads, max(64, (per / 12 + 31) / 32 * 32))
                               : min(kLossThreads, max(64, (per / 8 + 31) / 32 * 32));
    const size_t smem = masked ? 0 : (size_t)per * 16;
    a.cluster = cluster;
    auto kernel = masked ? loss_masked_kernel<T, kDense> : loss_kernel<T, kDense>;
    // (48 KB go without asking, the kernel's own few included; the limit is the
    // kernel's, not the call's: every call asks for the same, so that calls of
    // several threads do not take it from each other)
    if (smem > 40 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostScores);
    if (e == cudaSuccess && cluster == 16)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) break;
    cudaLaunchConfig_t c{};
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cluster;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    c.attrs = &at;
    c.numAttrs = cluster > 1;
    int64_t rows_at_once = n;
    if (!masked) {
      // what the device holds: by shared memory, and by registers and threads
      const int resident = max(1, min(min((int)(kSharedPerSM / (smem + 2048)), 1024 / threads), 16));
      int most = max(1, 148 * resident / cluster);
      // clusters of 2 always pack (an SM holds 2 blocks); others may not fill
      // every GPC, and one cluster too many would cost a whole second round
      if (cluster > 2 && n * cluster > 148) {
        c.gridDim = dim3((unsigned)(most * cluster));
        e = cudaOccupancyMaxActiveClusters(&most, kernel, &c);
        if (e != cudaSuccess) break;
        most = max(1, most);
      }
      rows_at_once = min(n, (int64_t)most);
    }
    c.gridDim = dim3((unsigned)(rows_at_once * cluster));
    e = cudaLaunchKernelEx(&c, kernel, a);
  }
  return e;
}

}  // namespace
}  // namespace policy
}  // namespace gz

using namespace gz;
using namespace gz::policy;

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

extern "C" gz_status gz_selftest_cluster_wait_timeout(int device, int limit_us) {
  const char* who = "gz_selftest_cluster_wait_timeout";
  if (limit_us <= 0 || limit_us > 10000000) return bad(who, "limit_us out of range");
  int before = 0, fine = 1;
  int* status = nullptr;
  cudaError_t e = cudaGetDevice(&before);
  if (e == cudaSuccess) e = cudaSetDevice(device);
  if (e != cudaSuccess) return set_last_error(GZ_ERR_CUDA, "%s: cannot select CUDA device %d", who, device);
  e = cudaMalloc(&status, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpy(status, &fine, sizeof(int), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) {
    wait_limit_kernel<<<2, 64>>>(limit_us * 1000ull, status);
    e = cudaGetLastError();
  }
  if (e == cudaSuccess) e = cudaMemcpy(&fine, status, sizeof(int), cudaMemcpyDeviceToHost);
  cudaFree(status);
  cudaSetDevice(before);
  if (e != cudaSuccess) return set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  if (!fine) return GZ_OK;
  return set_last_error(GZ_ERR_TIMEOUT, "%s: bounded waits gave up after %d us and left NaN (expected)", who, limit_us);
}
