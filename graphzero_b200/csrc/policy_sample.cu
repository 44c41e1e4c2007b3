// Drawing actions from rows of policy scores (gz_policy_sample).
//
// A row's order is that of its rank keys: the score's bits in an order-
// preserving form, then the index, so that no two are alike, and the kept
// actions of top_k and top_p are those from some rank key on.  Reading a row is
// bound by memory, choosing from it by the latency of its steps; so a row is
// read once, the few actions that can be kept go to a list in shared memory,
// and the rest is done there, by one warp where the list is short:
//  - Masked rows of up to 5120 actions (legal moves): a warp lists the visible
//    ones, sixteen mask bytes at a time, and reads scores and noise of these
//    alone.  4096 rows of 4672 with top_p and min_p: 13 us, 1.5 TB/s of mask.
//  - Other rows: a block reads the row once for its best score, its vectors'
//    maxima and, where top_p needs it, its sum of exponentials.  A bound below
//    which (nearly always) nothing is kept gives the list (draw_long).  256 rows
//    of 131072 bf16 scores with top_p 0.92: 33 us, of which 17 read the rows
//    (10 at the copy rate); the rest is steps of one after the other.
//  - Where the list is too long or not enough (a wide share of a flat row, a
//    large top_k), a histogram over the scores finds the bin that the last kept
//    action lies in, and only that bin is listed and sorted; if it overflows the
//    list (equal scores), the last rank key is found by bisection.
// The draw is an argmax over the kept actions; noise is read for these alone,
// or, where nearly all are kept, a vector at a time.
//
// Weights exp(d) of listed actions are summed as whole numbers of 2^-44, so
// that neither the list's order nor that of the atomics matters; sums over
// whole rows are 32-bit floats in an order given by the row's length and
// alignment.
#include "gz_policy.h"

namespace gz {
namespace policy {
namespace {

struct SampleArgs {
  RowArgs rows;
  gz_sample_config cfg;
  const float* noise;
  int64_t noise_stride;
  int32_t* action;
  float* logp;
  int64_t first_row, end_row;  // of this launch
};

constexpr int kList = 2048;          // keys a block's list holds
constexpr int kMaskedList = 1024, kMaskedThreads = 128;  // the same for blocks of four masked rows, and their threads
constexpr int kSampleThreads = 512;  // most threads of a block
constexpr int kReachBit = 16;       // lowest bit of a score that the search for a list's bound looks at
constexpr int kMaximaVecs = 24576;  // vectors of a row whose maxima are kept (96 KB; up to 22700 two blocks fit an SM)
constexpr int64_t kRowsPerLaunch = 1 << 28;

// e = exp(d), 0 .. 1, in units of 2^-44, cut off: 2^18 actions sum below 2^63.
__device__ __forceinline__ uint64_t fixed_weight(float e) {
  const uint32_t b = __float_as_uint(e);
  return (uint64_t)(b & 0x7fffffu | 0x800000u) << 21 >> min(63u, 127 - (b >> 23));  // 24 bits, shifted by the exponent
}

// Rank order as one number: higher scores first, at equal scores lower indices.
__device__ __forceinline__ uint64_t rank_key(float x, int j) {
  return (uint64_t)order_key(x) << 18 | (uint64_t)(GZ_POLICY_MAX_ACTIONS - 1 - j);
}
__device__ __forceinline__ int key_index(uint64_t k) {
  return GZ_POLICY_MAX_ACTIONS - 1 - (int)(k & (GZ_POLICY_MAX_ACTIONS - 1));
}
__device__ __forceinline__ float key_score(uint64_t k) { return key_value((uint32_t)(k >> 18)); }

// The threads that share a row: a warp, or the block.
template <bool kWarp> struct Team {
  uint64_t* slots;  // a word per warp
  int tid, n;
  __device__ void sync() const {
    if (kWarp) __syncwarp();
    else __syncthreads();
  }
  template <typename V, typename Op> __device__ V reduce(V x, Op op) const {
#pragma unroll
    for (int o = 16; o; o >>= 1) x = op(x, __shfl_xor_sync(~0u, x, o));
    if (kWarp) return x;
    V* s = (V*)slots;
    __syncthreads();
    if (tid % 32 == 0) s[tid / 32] = x;
    __syncthreads();
    x = s[0];
    for (int w = 1; w < n / 32; ++w) x = op(x, s[w]);
    return x;
  }
  template <typename V> __device__ V max(V x) const {
    return reduce(x, [](V a, V b) { return a > b ? a : b; });
  }
  template <typename V> __device__ V sum(V x) const {
    return reduce(x, [](V a, V b) { return a + b; });
  }
  // Sum of the x of the threads before this one.
  __device__ uint64_t before(uint64_t x) const {
    uint64_t up = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const uint64_t y = __shfl_up_sync(~0u, up, o);
      if (tid % 32 >= o) up += y;
    }
    uint64_t sum = up - x;
    if (kWarp) return sum;
    __syncthreads();
    if (tid % 32 == 31) slots[tid / 32] = up;
    __syncthreads();
    for (int w = 0; w < tid / 32; ++w) sum += slots[w];
    return sum;
  }
};

// kMask: vectors are read through the mask.
template <typename T, bool kMask> struct Row {
  static constexpr int V = 16 / (int)sizeof(T);
  const T* x;
  const uint8_t* mask;
  const float* noise;
  int actions, head, vecs, ends;  // scores before the first 16-byte boundary, vectors, scores beside them
  bool mask_aligned;

  __device__ Row(const SampleArgs& a, int64_t row) {
    actions = a.rows.actions;
    x = (const T*)a.rows.logits + row * a.rows.logits_stride;
    mask = a.rows.mask ? a.rows.mask + row * a.rows.mask_stride : nullptr;
    noise = a.noise ? a.noise + row * a.noise_stride : nullptr;
    head = min(actions, (int)(-(uintptr_t)x & 15) / (int)sizeof(T));
    vecs = (actions - head) / V;
    ends = actions - vecs * V;
    mask_aligned = (((uintptr_t)mask + head) & (V - 1)) == 0;
  }
  __device__ int end_index(int i) const { return i < head ? i : actions - ends + i; }
  __device__ float end_score(int i) const {
    const int j = end_index(i);
    return kMask && !mask[j] ? -INFINITY : to_f32(x[j]);
  }
  // A vector's scores, -inf where masked.
  __device__ __forceinline__ uint4 vector(int v) const {
    const uint4* p = (const uint4*)(x + head) + v;
    if (!kMask) return __ldg(p);
    const uint32_t bits = visible_bits<V>(mask + head + v * V, mask_aligned);
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (bits) raw = __ldg(p);
    T* e = (T*)&raw;
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (!(bits >> k & 1)) e[k] = from_f32<T>(-INFINITY);
    return raw;
  }
};

// f(first, bits) for this thread's share of a mask, sixteen bytes at a time and
// the bytes beside the whole sixteens one by one: bits of visible actions from
// `first` on, none of them 0.  Needs at least 30 threads.
template <int kAhead, typename T, typename F, bool kMask> __device__ __forceinline__ void each_visible(const Row<T, kMask>& r, int tid, int n, F f) {
  const int head = min(r.actions, (int)(-(uintptr_t)r.mask & 15));
  const int groups = (r.actions - head) / 16, ends = r.actions - groups * 16;
  const int ej = tid < head ? tid : r.actions - ends + tid;
  if (tid < ends && r.mask[ej]) f(ej, 1u);
  const uint4* group = (const uint4*)(r.mask + head);
  for (int u0 = tid; u0 < groups; u0 += kAhead * n) {
    uint4 w[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) w[i] = u0 + i * n < groups ? __ldg(group + u0 + i * n) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (!(w[i].x | w[i].y | w[i].z | w[i].w)) continue;
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // the bytes' flags, gathered into four bits
        const uint32_t c = __vcmpne4(k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w, 0) & 0x08040201u;
        bits |= (c * 0x01010101u >> 24) << (4 * k);
      }
      f(head + (u0 + i * n) * 16, bits);
    }
  }
}

// f(j, score) for this thread's share of the visible actions.
template <typename T, typename F, bool kMask> __device__ __forceinline__ void each(const Row<T, kMask>& r, int tid, int n, F f) {
  auto one = [&](int j, float v) {
    if (v > -INFINITY) f(j, fminf(v, FLT_MAX));  // a NaN counts as -inf
  };
  if (tid < r.ends) one(r.end_index(tid), r.end_score(tid));
  for (int v = tid; v < r.vecs; v += n) {
    constexpr int V = 16 / (int)sizeof(T);
    float x[V];
    unpack<T>(r.vector(v), x);
#pragma unroll
    for (int k = 0; k < V; ++k) one(r.head + v * V + k, x[k]);
  }
}

struct Filters {
  float temperature, top_p, min_p;
  int top_k;
  bool greedy;  // the best action alone

  __device__ Filters(const gz_sample_config& c, int64_t row) {
    // (of a NaN the end that keeps the fewest actions is taken: 0, 0 and 1)
    temperature = c.d_temperature ? c.d_temperature[row] : c.temperature;
    if (temperature > 0.f) temperature = fminf(fmaxf(temperature, 1e-30f), FLT_MAX);  // its reciprocal stays finite
    top_p = c.d_top_p ? c.d_top_p[row] : c.top_p;
    min_p = fminf(c.d_min_p ? c.d_min_p[row] : c.min_p, 1.f);
    top_k = c.d_top_k ? c.d_top_k[row] : c.top_k;
    greedy = !(temperature > 0.f) || top_k == 1 || !(top_p > 0.f);
  }
  __device__ float depth(float x, float top) const { return temperature == 1.f ? x - top : __fdiv_rn(x - top, temperature); }
};

__device__ __forceinline__ void answer(const SampleArgs& a, int64_t row, int action, float logp) {
  a.action[row] = action;
  if (a.logp) a.logp[row] = logp;
}

// The best of a row's noisy scores so far, and the kept weight.
struct Draw {
  uint64_t best = 0, weight = 0;
  __device__ void add(const Filters& f, float top, float x, int j, const float* noise) {
    const float d = f.depth(x, top), e = expf(d);
    if (e < f.min_p) return;
    weight += fixed_weight(e);
    const float s = noise ? d + noise[j] : d;
    const uint64_t key = rank_key(s >= -INFINITY ? s : -INFINITY, j);
    if (key > best) best = key;
  }
  template <typename T, bool kWarp, bool kMask>
  __device__ void finish(const SampleArgs& a, int64_t row, const Team<kWarp>& team, const Row<T, kMask>& r, const Filters& f, float top) {
    weight = team.sum(weight);
    best = team.max(best);
    if (team.tid == 0) {
      const int j = key_index(best);
      answer(a, row, j, f.depth(fminf(to_f32(r.x[j]), FLT_MAX), top) - logf((float)((double)weight * 0x1p-44)));
    }
  }
};

// Sorts keys[0 .. size) downwards; the memory behind them up to a power of two is used.
template <bool kWarp> __device__ void sort_keys(const Team<kWarp>& team, uint64_t* keys, int size) {
  int p = 2;
  while (p < size) p *= 2;
  for (int i = size + team.tid; i < p; i += team.n) keys[i] = 0;
  team.sync();
  for (int k = 2; k <= p; k *= 2)
    for (int h = k / 2; h; h /= 2) {
      for (int i = team.tid; i < p / 2; i += team.n) {
        const int lo = 2 * i - (i & (h - 1)), hi = lo + h;
        const uint64_t x = keys[lo], y = keys[hi];
        if ((x < y) == ((lo & k) == 0)) {
          keys[lo] = y;
          keys[hi] = x;
        }
      }
      team.sync();
    }
}

// How many of the sorted keys[0 .. m) have less than `goal` before them, where
// `above` lies before the first and a key counts its weight, or 1.
template <bool kWeights, bool kWarp>
__device__ int keys_before(const Team<kWarp>& team, const uint64_t* keys, int m, const Filters& f, float top, double goal,
                           uint64_t above, uint64_t* total) {
  const int per = (m + team.n - 1) / team.n, lo = min(m, team.tid * per), hi = min(m, lo + per);
  auto weight = [&](int i) { return kWeights ? fixed_weight(expf(f.depth(key_score(keys[i]), top))) : 1ull; };
  uint64_t mine = 0;
  for (int i = lo; i < hi; ++i) mine += weight(i);
  uint64_t sum = above + team.before(mine);
  if (total) {
    *total = team.max(sum + mine);
    if (goal < 0) goal = -goal * (double)*total;  // a share of the keys' own weight
  }
  int c = 0;
  for (int i = lo; i < hi && (double)sum < goal; ++i, ++c) sum += weight(i);
  return team.sum(c);
}

// Draws from a list of a row's best actions: all that can be kept.  size: keys
// in memory, of which `count` are not 0.  row_weight < 0: the list is the whole
// row or top_k's; else the row's weight, and false comes back if the list does
// not reach top_p's share of it.
template <typename T, bool kWarp, bool kMask>
__device__ bool draw_from_list(const SampleArgs& a, int64_t row, const Team<kWarp>& team, const Row<T, kMask>& r, const Filters& f,
                               uint64_t* keys, int size, int count, float top, double row_weight) {
  if ((f.top_k > 0 && f.top_k < count) || f.top_p < 1.f) {
    sort_keys(team, keys, size);
    size = f.top_k > 0 ? min(count, f.top_k) : count;
    if (f.top_p < 1.f) {
      uint64_t total;
      const double goal = row_weight < 0 ? -(double)f.top_p : f.top_p * row_weight;
      const int kept = keys_before<true>(team, keys, size, f, top, goal, 0, &total);
      if (row_weight >= 0 && (double)total < goal) return false;
      size = max(1, kept);
    }
  }
  Draw d;
  for (int i = team.tid; i < size; i += team.n)
    if (keys[i]) d.add(f, top, key_score(keys[i]), key_index(keys[i]), r.noise);
  d.finish(a, row, team, r, f, top);
  return true;
}

// Draws from at most kFew actions, in any order, with one warp: every key's rank
// and the weight before it come from comparing it with all others.  A lane
// brings kMine of them, j < 0 for none.  row_weight and the answer as in
// draw_from_list.
constexpr int kFew = 64, kMine = kFew / 32;
struct FewShared {
  uint64_t key[kFew], weight[kFew];
};
template <typename T, bool kMask>
__device__ __forceinline__ bool draw_from_few(const SampleArgs& a, int64_t row, const Row<T, kMask>& r, const Filters& f, const int* j,
                                              const float* x, double row_weight, FewShared& sh) {
  const Team<true> team{nullptr, (int)threadIdx.x % 32, 32};
  float noise[kMine], d[kMine], e[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) noise[i] = r.noise && j[i] >= 0 ? r.noise[j[i]] : 0.f;
  uint64_t key[kMine], best = 0;
  int count = 0;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const bool in = j[i] >= 0 && x[i] > -INFINITY;  // a NaN counts as -inf
    key[i] = in ? rank_key(fminf(x[i], FLT_MAX), j[i]) : 0;
    if (key[i] > best) best = key[i];
    count += __popc(__ballot_sync(~0u, in));
  }
  best = team.max(best);
  if (!best || f.greedy) {
    if (team.tid == 0) answer(a, row, best ? key_index(best) : -1, 0.f);
    return true;
  }
  const float top = key_score(best);
  uint64_t weight[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    d[i] = f.depth(key_score(key[i]), top);
    e[i] = key[i] ? expf(d[i]) : 0.f;
    weight[i] = fixed_weight(e[i]);
  }
  bool keep[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) keep[i] = key[i] != 0;
  if ((f.top_k > 0 && f.top_k < count) || f.top_p < 1.f) {
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      sh.key[team.tid + 32 * i] = key[i];
      sh.weight[team.tid + 32 * i] = weight[i];
    }
    team.sync();
    int rank[kMine] = {};
    uint64_t before[kMine] = {}, sum = 0;
    int full = 0;  // keys lie below it
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      const uint32_t some = __ballot_sync(~0u, key[i] != 0);
      if (some) full = 32 * i + 32 - __clz(some);
    }
#pragma unroll 4
    for (int q = 0; q < full; ++q) {
      const uint64_t k = sh.key[q], w = sh.weight[q];
#pragma unroll
      for (int i = 0; i < kMine; ++i)
        if (k > key[i]) {
          ++rank[i];
          before[i] += w;
        }
    }
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      if (f.top_k > 0) keep[i] = keep[i] && rank[i] < f.top_k;
      if (keep[i]) sum += weight[i];
    }
    if (f.top_p < 1.f) {
      const double total = (double)team.sum(sum), goal = f.top_p * (row_weight < 0 ? total : row_weight);
      if (total < goal) return false;
#pragma unroll
      for (int i = 0; i < kMine; ++i) keep[i] = keep[i] && ((double)before[i] < goal || rank[i] == 0);
    }
  }
  uint64_t sum = 0;
  best = 0;
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    if (keep[i] && e[i] >= f.min_p) {
      sum += weight[i];
      const float s = d[i] + noise[i];
      const uint64_t k = rank_key(s >= -INFINITY ? s : -INFINITY, key_index(key[i]));
      if (k > best) best = k;
    }
  sum = team.sum(sum);
  best = team.max(best);
  // the drawn action's lane answers
#pragma unroll
  for (int i = 0; i < kMine; ++i)
    if (key[i] && key_index(key[i]) == key_index(best)) answer(a, row, key_index(best), d[i] - logf((float)((double)sum * 0x1p-44)));
  return true;
}

// Rows of at most kFew actions: a warp each, four a block.
template <typename T> __global__ void __launch_bounds__(128) sample_warp_kernel(SampleArgs a) {
  __shared__ FewShared few[4];
  const int64_t row = a.first_row + (int64_t)blockIdx.x * 4 + threadIdx.x / 32;
  if (row >= a.end_row) return;
  const int lane = threadIdx.x % 32;
  const Row<T, false> r(a, row);
  const Filters f(a.cfg, row);
  int j[kMine];
  float x[kMine];
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int k = lane + 32 * i;
    j[i] = k < r.actions && !(r.mask && !r.mask[k]) ? k : -1;
    x[i] = k < r.actions ? to_f32(r.x[k]) : -INFINITY;
  }
  draw_from_few(a, row, r, f, j, x, -1.0, few[threadIdx.x / 32]);
}

// The rank key of the last kept action: the largest with at least `goal` (a
// count, or a weight) at or above it.
template <bool kWeights, typename T, bool kMask>
__device__ __noinline__ uint64_t last_by_bisection(const Team<false>& team, const Row<T, kMask>& r, const Filters& f, float top, double goal) {
  uint64_t last = 0;
  for (int bit = 49; bit >= 0; --bit) {
    const uint64_t mid = last | 1ull << bit;
    uint64_t s = 0;
    each(r, team.tid, team.n, [&](int j, float x) {
      if (rank_key(x, j) >= mid) s += kWeights ? fixed_weight(expf(f.depth(x, top))) : 1ull;
    });
    if ((double)team.sum(s) >= goal) last = mid;
  }
  return last;
}

// The same through a histogram, in the list's memory, over `span` below the best
// score (what lies deeper is found by bisection if need be).
// Scores below `from` are known not to be kept.
template <bool kWeights, int kSize, typename T, bool kMask>
__device__ __noinline__ uint64_t last_by_bins(const Team<false>& team, const Row<T, kMask>& r, const Filters& f, float top, double goal,
                                              float from, float span, uint64_t* memory, int* counter) {
  __shared__ uint64_t above;
  __shared__ int found;
  constexpr int kBins = kSize;
  uint32_t *low = (uint32_t*)memory, *high = low + kBins;
  const float scale = kBins / span, per_score = 1.44269504f / f.temperature;
  auto bin = [&](float x) { return min(kBins - 1, (int)((top - x) * scale)); };  // falls as x rises, weakly
  team.sync();
  for (int i = team.tid; i < kBins; i += team.n) low[i] = high[i] = 0;
  if (team.tid == 0) *counter = 0, found = kBins;
  team.sync();
  each(r, team.tid, team.n, [&](int, float x) {
    if (x < from) return;
    // (the bins' weights by the fast exponential; the boundary bin's by the list's)
    const uint64_t w = kWeights ? fixed_weight(sm100::ex2_approx((x - top) * per_score)) : 1;
    if (!w) return;
    // in two halves, for only 32-bit adds are done in shared memory at once
    const int b = bin(x);
    const uint32_t old = atomicAdd(&low[b], (uint32_t)w), up = (uint32_t)(w >> 32) + (old + (uint32_t)w < old);
    if (up) atomicAdd(&high[b], up);
  });
  team.sync();
  const int per = kBins / team.n, lo = team.tid * per;  // n divides kBins or the rest is the last thread's
  const int hi = team.tid == team.n - 1 ? kBins : lo + per;
  uint64_t mine = 0;
  auto weight = [&](int i) { return (uint64_t)high[i] << 32 | low[i]; };
  for (int i = lo; i < hi; ++i) mine += weight(i);
  uint64_t sum = team.before(mine);
  for (int i = lo; i < hi; ++i) {
    if ((double)sum < goal && (double)(sum + weight(i)) >= goal) {
      found = i;
      above = sum;
    }
    sum += weight(i);
  }
  team.sync();
  const int b = found;
  const uint64_t base = above;
  if (b == kBins) return last_by_bisection<kWeights>(team, r, f, top, goal);  // out of reach by rounding
  team.sync();  // the bins have been read
  each(r, team.tid, team.n, [&](int j, float x) {
    if (bin(x) == b) {
      const int at = atomicAdd(counter, 1);
      if (at < kSize) memory[at] = rank_key(x, j);
    }
  });
  team.sync();
  const int m = *counter;
  if (m > kSize) return last_by_bisection<kWeights>(team, r, f, top, goal);
  sort_keys(team, memory, m);
  const int kept = keys_before<kWeights>(team, memory, m, f, top, goal, base, nullptr);
  const uint64_t last = memory[max(0, kept - 1)];
  team.sync();
  return last;
}

template <int kSize> struct Shared {
  uint64_t slots[kSampleThreads / 32], list[kSize];
  alignas(8) int hit[kSize];
  int hits, counter;
  bool done;
  uint32_t bound, sums[3];
};

// Draws from a row's actions from the rank key `last` on (0: all): the scores
// from the caches once more, and the noise.  The kept weight is summed in 32
// bits (under a mask in whole numbers).  Noisy scores are compared as they are
// defined, but with a temperature the division is done only for vectors whose
// upper bound, from a product with its reciprocal, could still win.  256
// unfiltered rows of 131072 bf16 scores, draw_long's pass included: 60 us at
// temperature 1, 76 us at 0.8 (3.3 and 2.7 TB/s of scores and noise), bound by
// instructions.
template <typename T, bool kMask>
__device__ void draw_from_all(const SampleArgs& a, int64_t row, const Team<false>& team, const Row<T, kMask>& r, const Filters& f, float top,
                              uint64_t last) {
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = team.tid, n = team.n;
  const float* noise = r.noise ? r.noise + r.head : nullptr;
  const bool aligned = ((uintptr_t)noise & 15) == 0;
  const float least = last ? key_score(last) : -FLT_MAX, per = 1.f / f.temperature;
  const float above = least < FLT_MAX ? least : INFINITY;  // kept whatever its index is; +inf counts as FLT_MAX
  const int last_index = last ? key_index(last) : GZ_POLICY_MAX_ACTIONS;
  float most = -INFINITY, z = 0.f;
  uint64_t weight = 0;  // the same in whole numbers, under a mask: whatever the mask's alignment to the scores
  int where = -1;
  auto load = [&](int v, float* x, float* g) {  // scores, -inf where not kept
    unpack<T>(r.vector(v), x);
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
      if (noise) {
        const float* p = noise + v * V + k;
        q = aligned ? __ldg((const float4*)p) : make_float4(__ldg(p), __ldg(p + 1), __ldg(p + 2), __ldg(p + 3));
      }
      *(float4*)(g + k) = q;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const bool kept = x[k] > above || (x[k] >= least && r.head + v * V + k <= last_index);
      x[k] = kept ? fminf(x[k], FLT_MAX) : -INFINITY;
    }
  };
  auto noisy = [&](float x, float g) { return x > -INFINITY ? f.depth(x, top) + g : -INFINITY; };
#pragma unroll 2
  for (int v = tid; v < r.vecs; v += n) {
    float x[V], g[V], m = -INFINITY;
    load(v, x, g);
    if (f.min_p > 0.f) {
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (x[k] > -INFINITY && expf(f.depth(x[k], top)) < f.min_p) x[k] = -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = (x[k] - top) * per;
      const float e = sm100::ex2_approx(d * 1.44269504f);
      if (kMask) weight += fixed_weight(e);
      else z += e;
      // d is within 2^-22 |d| of the quotient
      m = fmaxf(m, f.temperature == 1.f ? d + g[k] : fmaf(d, -0x1p-21f, d + g[k]));
    }
    if (f.temperature != 1.f && m + fabsf(m) * 0x1p-21f >= most) {
      m = -INFINITY;
#pragma unroll
      for (int k = 0; k < V; ++k) m = fmaxf(m, noisy(x[k], g[k]));
    }
    if (m > most) {
      most = m;
      where = v;
    }
  }
  uint64_t best = 0;
  if (where >= 0) {
    float x[V], g[V];
    load(where, x, g);
#pragma unroll
    for (int k = V - 1; k >= 0; --k)
      if (noisy(x[k], g[k]) == most && !(f.min_p > 0.f && expf(f.depth(x[k], top)) < f.min_p)) best = rank_key(most, r.head + where * V + k);
  }
  if (tid < r.ends) {
    const int j = r.end_index(tid);
    const float x = fminf(r.end_score(tid), FLT_MAX);
    if (r.end_score(tid) > -INFINITY && rank_key(x, j) >= last && !(f.min_p > 0.f && expf(f.depth(x, top)) < f.min_p)) {
      const float d = f.depth(x, top), s = d + (r.noise ? r.noise[j] : 0.f);
      const float e = sm100::ex2_approx((x - top) * per * 1.44269504f);
      if (kMask) weight += fixed_weight(e);
      else z += e;
      const uint64_t key = rank_key(s >= -INFINITY ? s : -INFINITY, j);
      if (key > best) best = key;
    }
  }
  z = kMask ? (float)((double)team.sum(weight) * 0x1p-44) : team.sum(z);
  best = team.max(best);
  if (!best || key_score(best) == -INFINITY) {  // no noisy score above -inf: the first of the kept actions
    best = 0;
    each(r, tid, n, [&](int j, float x) {
      const uint64_t key = rank_key(-INFINITY, j);
      if (rank_key(x, j) >= last && expf(f.depth(x, top)) >= f.min_p && key > best) best = key;
    });
    best = team.max(best);
  }
  if (tid == 0) {
    const int j = key_index(best);
    answer(a, row, j, f.depth(fminf(to_f32(r.x[j]), FLT_MAX), top) - logf(z));
  }
}

// Draws from a list of m actions, at most kRanked, in any order, with the block:
// a key's rank and the weight before it come from comparing it with all others.
// row_weight and the answer as in draw_from_list.
constexpr int kRanked = 256;
template <typename T, int kSize, bool kMask>
__device__ bool draw_by_rank(const SampleArgs& a, int64_t row, const Team<false>& team, const Row<T, kMask>& r, const Filters& f,
                             Shared<kSize>& sh, int m, float top, double row_weight) {
  static_assert(2 * kRanked <= kSize, "keys, and the weights before them, lie in the list");
  uint64_t *key = sh.list, *before = sh.list + kRanked, *weight = (uint64_t*)sh.hit;
  const int tid = team.tid, n = team.n;
  for (int i = tid; i < m; i += n) weight[i] = fixed_weight(expf(f.depth(key_score(key[i]), top)));
  __syncthreads();
  const bool cut = f.top_k > 0 && f.top_k < m;
  uint64_t sum = 0;
  for (int i = tid; i < m; i += n) {
    const uint64_t mine = key[i];
    uint64_t w = 0;
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < m; ++j)
      if (key[j] > mine) {
        w += weight[j];
        ++rank;
      }
    const bool in = !cut || rank < f.top_k;
    if (in) sum += weight[i];
    before[i] = in ? w : ~0ull;
  }
  double goal = 0x1p64;  // of the weight before a kept action; above every sum
  if (f.top_p < 1.f) {
    const double total = (double)team.sum(sum);
    goal = f.top_p * (row_weight < 0 ? total : row_weight);
    if (total < goal) return false;
  }
  Draw d;
  for (int i = tid; i < m; i += n)
    if (before[i] != ~0ull && ((double)before[i] < goal || before[i] == 0)) d.add(f, top, key_score(key[i]), key_index(key[i]), r.noise);
  d.finish(a, row, team, r, f, top);
  return true;
}

// Draws by top_p from a list of m actions, more than kRanked, without sorting it.
// Weights in units of 2^-22, cut off, are summed above a score that a search
// over its bits raises as far as the goal is surely reached; what is left has
// few actions too many, and those go one by one, the least first, by exact
// weights.  False: not done (the list or the cut weights do not reach the goal,
// or too many actions are at the boundary).
template <typename T, int kSize, bool kWarp, bool kMask>
__device__ bool draw_by_weight(const SampleArgs& a, int64_t row, const Team<kWarp>& team, const Row<T, kMask>& r, const Filters& f,
                               Shared<kSize>& sh, int m, float from, float top, double row_weight) {
  const int tid = team.tid, n = team.n;
  const double goal = f.top_p * row_weight, cut = goal * 0x1p-22 + 1;
  if (cut >= 0x1p31) return false;
  const uint32_t goal22 = (uint32_t)cut + 1;
  uint32_t* weight = (uint32_t*)sh.hit;
  for (int i = tid; i < m; i += n) weight[i] = (uint32_t)(fixed_weight(expf(f.depth(key_score(sh.list[i]), top))) >> 22);
  if (!kWarp && tid < 3) sh.sums[tid] = 0;
  team.sync();
  int round = 0;
  auto above = [&](uint32_t score) {  // weight of the scores from this one on
    uint32_t c = 0;
    for (int i = tid; i < m; i += n)
      if ((uint32_t)(sh.list[i] >> 18) >= score) c += weight[i];
    c = __reduce_add_sync(~0u, c);
    if (kWarp) return c;
    uint32_t* sum = &sh.sums[round % 3];
    if (tid % 32 == 0 && c) atomicAdd(sum, c);
    if (tid == 0) sh.sums[(round + 1) % 3] = 0;
    ++round;
    __syncthreads();
    return *sum;
  };
  // (a sum that passes 2^32 only looks too small: the score is raised less)
  const uint32_t low = order_key(from), high = order_key(top);
  if (above(low) < goal22) return false;
  const int first = 31 - __clz(low ^ high | 1);
  uint32_t score = high & ~((2u << first) - 1);
#pragma unroll 1
  for (int bit = first; bit >= (sizeof(T) == 2 ? 13 : 6); --bit)
    if (above(score | 1u << bit) >= goal22) score |= 1u << bit;
  // the list's actions from `score` on
  uint64_t sum = 0;
  for (int i = tid; i < m; i += n)
    if ((uint32_t)(sh.list[i] >> 18) >= score) sum += fixed_weight(expf(f.depth(key_score(sh.list[i]), top)));
  sum = team.sum(sum);
  uint64_t least = 0;  // the last key that is dropped
  for (int round = 0;; ++round) {
    uint64_t key = ~0ull;
    for (int i = tid; i < m; i += n) {
      const uint64_t k = sh.list[i];
      if ((uint32_t)(k >> 18) >= score && k > least && k < key) key = k;
    }
    key = team.reduce(key, [](uint64_t x, uint64_t y) { return x < y ? x : y; });
    const uint64_t w = fixed_weight(expf(f.depth(key_score(key), top)));
    if ((double)(sum - w) < goal) break;
    if (round == 16) return false;
    sum -= w;
    least = key;
  }
  Draw d;
  for (int i = tid; i < m; i += n) {
    const uint64_t k = sh.list[i];
    if ((uint32_t)(k >> 18) >= score && k > least) d.add(f, top, key_score(k), key_index(k), r.noise);
  }
  d.finish(a, row, team, r, f, top);
  return true;
}

// A row with a block.  maxima: a float for every vector of the row, or null.
// kMask: it is read through its mask.
template <typename T, bool kMask, int kSize>
__device__ __forceinline__ void draw_long(const SampleArgs& a, int64_t row, Shared<kSize>& sh, float* maxima) {
  constexpr int V = 16 / (int)sizeof(T);
  const int tid = threadIdx.x, n = blockDim.x;
  const Team<false> team{sh.slots, tid, n};
  const Row<T, kMask> r(a, row);
  const Filters f(a.cfg, row);
  const bool by_count = f.top_k > 0 && f.top_k < r.actions, by_weight = f.top_p < 1.f;
  const bool row_weighs = by_weight && !by_count && !f.greedy;
  const float per_score = 1.44269504f / f.temperature;

  // the thread's best action and, where top_p asks for the row's weight, its
  // sum of exponentials relative to the best of its first vector
  uint64_t best = 0;
  float z = 0.f, z_base = -INFINITY;
  bool z_fine = false;
  float most = -INFINITY, base = 0.f;
  int where = -1;
  float2 sum = {0.f, 0.f};
  constexpr int kAhead = 4;
  for (int v0 = tid; v0 < r.vecs; v0 += kAhead * n) {
    uint4 raw[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (v0 + i * n < r.vecs) raw[i] = r.vector(v0 + i * n);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (v0 + i * n >= r.vecs) continue;
      const float m = fminf(max_vector<false, T>(-INFINITY, raw[i], 0), FLT_MAX);
      if (maxima) maxima[v0 + i * n] = m;
      if (m > most) {
        most = m;
        where = v0 + i * n;
      }
      if (row_weighs) {
        if (z_base == -INFINITY) {
          z_base = m;
          base = m == -INFINITY ? 0.f : m;
        }
        float x[V];
        unpack<T>(raw[i], x);
#pragma unroll
        for (int k = 0; k < V; k += 2) {
          const float2 d = __fadd2_rn(make_float2(x[k], x[k + 1]), make_float2(-base, -base));
          const float2 y = __fmul2_rn(d, make_float2(per_score, per_score));
          sum = __fadd2_rn(sum, make_float2(sm100::ex2_approx(y.x), sm100::ex2_approx(y.y)));
        }
      }
    }
  }
  if (where >= 0) {
    float x[V];
    unpack<T>(r.vector(where), x);
#pragma unroll
    for (int k = V - 1; k >= 0; --k)
      if (x[k] >= most) best = rank_key(most, r.head + where * V + k);  // (+inf counts as FLT_MAX, a NaN is none)
  }
  z = sum.x + sum.y;
  if (tid < r.ends) {
    const float x = fminf(r.end_score(tid), FLT_MAX);
    if (r.end_score(tid) > -INFINITY) {
      const uint64_t key = rank_key(x, r.end_index(tid));
      if (key > best) best = key;
      if (z_base == -INFINITY) z_base = x;
      z += sm100::ex2_approx((x - z_base) * per_score);
    }
  }
  z_fine = z_base == -INFINITY ? z == 0.f : z > 0.f && z < 0x1p64f;
  const uint64_t mine = best;
  best = team.max(best);
  if (!best || f.greedy) {
    if (tid == 0) answer(a, row, best ? key_index(best) : -1, 0.f);
    return;
  }
  const float top = key_score(best);

  uint64_t last = 0;  // rank key of the last action that top_k and top_p keep
  if (by_count || by_weight) {
    double row_weight = -1.0;
    if (row_weighs) {
      if (__syncthreads_and(z_fine)) {
        z *= z_base > -INFINITY ? sm100::ex2_approx((z_base - top) * per_score) : 0.f;
      } else {  // beyond what a sum relative to some score holds
        z = 0.f;
        each(r, tid, n, [&](int, float x) { z += expf(f.depth(x, top)); });
      }
      row_weight = (double)team.sum(z) * 0x1p44;
    }
    // Bounds for the list.  For top_k the largest number that top_k threads' best
    // scores reach; one warp searches for it, over the scores' upper 16 bits.
    // Not so where top_k is above the number of threads, nor where the leading
    // bits that those scores' keys share are all 0 (scores on both sides of 0, or
    // of -2 where none is positive): such rows have no list and take the
    // histogram (256 rows of 131072 with top_k 50: 26 us with the list, 229 us
    // with scores 4 lower that do without).
    // For top_p the scores of a weight of 1/256, then 1/2048 of what top_p leaves
    // out; no more than 256 / (1 - top_p) actions reach the first, and what lies
    // below it is often little.  Rows of up to kList actions are flatter at
    // their sizes: 1/4, then one times the share per action (4096 rows of 500
    // with top_p 0.9 take 39 us from 1/16 and 1/512 on, 24 us so).
    float bounds[2] = {-INFINITY, -INFINITY};
    if (!by_count) {
      const float out = (float)((1.0 - f.top_p) * row_weight * 0x1p-44);
      const bool flat = r.actions <= kList;
      const float first = flat ? fmaxf(r.actions / 4, 64) : 256.f, second = flat ? r.actions : 2048.f;
      bounds[0] = top + fminf(logf(out / first), 0.f) * f.temperature;
      bounds[1] = top + fminf(logf(out / second), 0.f) * f.temperature;
    } else if (f.top_k <= n) {
      uint32_t* scores = (uint32_t*)sh.list;
      scores[tid] = (uint32_t)(mine >> 18);
      __syncthreads();
      if (tid < 32) {
        uint32_t score[kSampleThreads / 32], least = ~0u, most = 0;
#pragma unroll
        for (int i = 0; i < kSampleThreads / 32; ++i) {
          score[i] = i < n / 32 ? scores[tid + 32 * i] : 0;
          if (score[i]) {
            least = min(least, score[i]);
            most = max(most, score[i]);
          }
        }
        auto above = [&](uint32_t mid) {
          int c = 0;
#pragma unroll
          for (int i = 0; i < kSampleThreads / 32; ++i) c += score[i] >= mid;
          return __reduce_add_sync(~0u, c);
        };
        least = __reduce_min_sync(~0u, least);
        most = __reduce_max_sync(~0u, most);
        // the bits that all scores share need no search
        const int first = 31 - __clz(least ^ most | 1);
        uint32_t bound = above(1) >= f.top_k ? most & ~((2u << first) - 1) : 0;
        if (bound)
#pragma unroll 1
          for (int bit = first; bit >= kReachBit; --bit)
            if (above(bound | 1u << bit) >= f.top_k) bound |= 1u << bit;
        if (tid == 0) sh.bound = bound;
      }
      __syncthreads();
      if (sh.bound) bounds[0] = key_value(sh.bound);
    }
    for (int attempt = 0; attempt < 2 && bounds[attempt] > -INFINITY; ++attempt) {
      const float from = bounds[attempt];
      if (tid == 0) sh.counter = sh.hits = 0;
      __syncthreads();
      auto take = [&](int j, float x) {
        if (x >= from) {
          const int at = atomicAdd(&sh.counter, 1);
          if (at < kSize) sh.list[at] = rank_key(x, j);
        }
      };
      if (tid < r.ends && r.end_score(tid) > -INFINITY) take(r.end_index(tid), fminf(r.end_score(tid), FLT_MAX));
      auto take_vector = [&](int v, uint4 raw) {
        float x[V];
        unpack<T>(raw, x);
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (x[k] == x[k]) take(r.head + v * V + k, fminf(x[k], FLT_MAX));
      };
      if (maxima) {  // each thread's own vectors' maxima; then their scores, all at once
#pragma unroll 8
        for (int v = tid; v < r.vecs; v += n)
          if (maxima[v] >= from) {
            const int at = atomicAdd(&sh.hits, 1);
            if (at < kSize) sh.hit[at] = v;
          }
        __syncthreads();
        const int hits = sh.hits;
        if (hits > kSize) {
          __syncthreads();  // all have seen it
          continue;
        }
        for (int h = tid; h < hits; h += n) take_vector(sh.hit[h], r.vector(sh.hit[h]));
      } else {
        constexpr int kAhead = 4;
        for (int v0 = tid; v0 < r.vecs; v0 += kAhead * n) {
          uint4 raw[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (v0 + i * n < r.vecs) raw[i] = r.vector(v0 + i * n);
#pragma unroll
          for (int i = 0; i < kAhead; ++i)
            if (v0 + i * n < r.vecs && max_vector<false, T>(-INFINITY, raw[i], 0) >= from) take_vector(v0 + i * n, raw[i]);
        }
      }
      __syncthreads();
      const int m = sh.counter;
      // Few by one warp, which has no barriers to wait for; in small blocks
      // more too; in large ones all threads compare keys (256 rows of 131072
      // with top_p 0.92: 35 us, against 43 with one warp for these; 4096 rows
      // of 500 with top_p 0.9, two warps a row: 25 us, against 67 with both).
      const bool few = m <= kFew, alone = few || (!by_count && n < 256 && m <= 2 * kRanked);
      if (alone) {
        if (tid < 32) {
          bool done;
          if (few) {
            int j[kMine];
            float x[kMine];
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
              const uint64_t key = tid + 32 * i < m ? sh.list[tid + 32 * i] : 0;
              j[i] = key ? key_index(key) : -1;
              x[i] = key_score(key);
            }
            done = draw_from_few(a, row, r, f, j, x, row_weight, *(FewShared*)(sh.list + kFew));
          } else {
            done = draw_by_weight(a, row, Team<true>{nullptr, tid, 32}, r, f, sh, m, from, top, row_weight);
          }
          if (tid == 0) sh.done = done;
        }
        __syncthreads();
        if (sh.done) return;
      }
      if (few) {
      } else if (m <= kRanked && n >= 256) {
        if (draw_by_rank(a, row, team, r, f, sh, m, top, row_weight)) return;
      } else if (m <= kSize) {
        if (!by_count && !alone && draw_by_weight(a, row, team, r, f, sh, m, from, top, row_weight)) return;
        if (draw_from_list(a, row, team, r, f, sh.list, m, m, top, row_weight)) return;
      }
      __syncthreads();  // all have read the count, and the list
    }
    if (by_count) {
      // twice the depth of the least of the threads' best scores
      const float depth = team.max(mine ? top - key_score(mine) : 0.f), span = 2.f * depth;
      last = last_by_bins<false, kSize>(team, r, f, top, (double)f.top_k, -INFINITY, span, sh.list, &sh.counter);
    }
    if (by_weight) {
      if (by_count) {
        uint64_t w = 0;
        each(r, tid, n, [&](int j, float x) {
          if (rank_key(x, j) >= last) w += fixed_weight(expf(f.depth(x, top)));
        });
        row_weight = (double)team.sum(w);
      }
      // all actions of less than (1 - top_p) / actions of the weight have less
      // than 1 - top_p of it together: the share is reached before them
      const float least = (float)((1.0 - f.top_p) * row_weight * 0x1p-44) / r.actions * 0.999f;
      const float from = least > 1e-30f ? top + (logf(fminf(least, 1.f)) - 0.001f) * f.temperature : -INFINITY;
      const uint64_t cut = last_by_bins<true, kSize>(team, r, f, top, f.top_p * row_weight, from, 31.f * f.temperature, sh.list, &sh.counter);
      if (cut > last) last = cut;
    }
  }
  draw_from_all(a, row, team, r, f, top, last);
}

// A call of its own, so that rows that fit the list do not pay for its registers.
template <typename T, int kSize> __device__ __noinline__ void draw_masked_long(const SampleArgs& a, int64_t row, Shared<kSize>& sh) {
  draw_long<T, true>(a, row, sh, nullptr);
}

// Masked rows, a warp each, four a block: the mask gives the visible actions'
// indices; of up to kFew of them scores and noise are read at once.  Rows with
// more than fit a list are taken by the whole block afterwards.
template <typename T> __global__ void __launch_bounds__(kMaskedThreads, 8) sample_masked_kernel(const __grid_constant__ SampleArgs a) {
  constexpr int kRows = kMaskedThreads / 32, kIndices = 256;
  __shared__ union {
    Shared<kMaskedList> whole;
    struct {
      int index[kIndices], count;
      union {
        FewShared few;
        uint64_t list[kIndices];
      };
    } part[kRows];
  } sh;
  const int team_id = threadIdx.x / 32, tid = threadIdx.x % 32;
  const int64_t row = a.first_row + (int64_t)blockIdx.x * kRows + team_id;
  const bool in = row < a.end_row;
  const Row<T, false> r(a, in ? row : a.first_row);
  if (tid == 0) sh.part[team_id].count = 0;
  __syncwarp();
  if (in)
    each_visible<10>(r, tid, 32, [&](int first, uint32_t bits) {
      int at = atomicAdd(&sh.part[team_id].count, __popc(bits));
      for (; bits; bits &= bits - 1, ++at)
        if (at < kIndices) sh.part[team_id].index[at] = first + __ffs(bits) - 1;
    });
  __syncwarp();
  const int count = in ? sh.part[team_id].count : 0;
  if (in && count <= kIndices) {
    const Filters f(a.cfg, row);
    const int* index = sh.part[team_id].index;
    if (count <= kFew) {
      int j[kMine];
      float x[kMine];
#pragma unroll
      for (int i = 0; i < kMine; ++i) {
        j[i] = tid + 32 * i < count ? index[tid + 32 * i] : -1;
        x[i] = j[i] >= 0 ? to_f32(r.x[j[i]]) : -INFINITY;
      }
      draw_from_few(a, row, r, f, j, x, -1.0, sh.part[team_id].few);
    } else {
      const Team<true> team{nullptr, tid, 32};
      uint64_t* keys = sh.part[team_id].list;
      uint64_t best = 0;
      int seen = 0;
      for (int i = tid; i < count; i += 32) {
        const float x = to_f32(r.x[index[i]]);
        const uint64_t key = x > -INFINITY ? rank_key(fminf(x, FLT_MAX), index[i]) : 0;
        keys[i] = key;
        seen += key != 0;
        if (key > best) best = key;
      }
      best = team.max(best);
      seen = team.sum(seen);
      team.sync();
      if (!best || f.greedy) {
        if (tid == 0) answer(a, row, best ? key_index(best) : -1, 0.f);
      } else {
        draw_from_list(a, row, team, r, f, keys, count, seen, key_score(best), -1.0);
      }
    }
  }
  const bool over = count > kIndices;
  if (!__syncthreads_or(over)) return;
  for (int t = 0; t < kRows; ++t)
    if (__syncthreads_or(over && team_id == t)) {
      draw_masked_long<T>(a, a.first_row + (int64_t)blockIdx.x * kRows + t, sh.whole);
      __syncthreads();
    }
}

template <typename T, int kSize, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_long_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ Shared<kSize> sh;
  extern __shared__ float maxima[];
  draw_long<T, false>(a, a.first_row + blockIdx.x, sh, a.rows.actions / (16 / (int)sizeof(T)) <= kMaximaVecs ? maxima : nullptr);
}

// Long masked rows, a block each: up to kRanked visible actions are listed, of
// more the row's vectors are gone through as without a mask.
template <typename T> __global__ void __launch_bounds__(kSampleThreads, 2) sample_long_masked_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ Shared<kList> sh;
  extern __shared__ float maxima[];
  const int64_t row = a.first_row + blockIdx.x;
  const int tid = threadIdx.x, n = blockDim.x;
  const Row<T, true> r(a, row);
  if (tid == 0) sh.hits = sh.counter = 0;
  __syncthreads();
  each_visible<4>(r, tid, n, [&](int first, uint32_t bits) {
    int at = atomicAdd(&sh.hits, __popc(bits));
    for (; bits; bits &= bits - 1, ++at)
      if (at < kRanked) sh.hit[at] = first + __ffs(bits) - 1;
  });
  __syncthreads();
  const int visible = sh.hits;
  if (visible > kRanked) {
    __syncthreads();
    draw_long<T, true>(a, row, sh, a.rows.actions / (16 / (int)sizeof(T)) <= kMaximaVecs ? maxima : nullptr);
    return;
  }
  const Team<false> team{sh.slots, tid, n};
  const Filters f(a.cfg, row);
  uint64_t best = 0;
  for (int i = tid; i < visible; i += n) {
    const int j = sh.hit[i];
    const float x = to_f32(r.x[j]);
    if (!(x > -INFINITY)) continue;  // a NaN counts as -inf
    const uint64_t key = rank_key(fminf(x, FLT_MAX), j);
    sh.list[atomicAdd(&sh.counter, 1)] = key;
    if (key > best) best = key;
  }
  best = team.max(best);
  if (!best || f.greedy) {
    if (tid == 0) answer(a, row, best ? key_index(best) : -1, 0.f);
    return;
  }
  draw_by_rank(a, row, team, r, f, sh, sh.counter, key_score(best), -1.0);
}

template <typename T> cudaError_t launch_sample(SampleArgs a, int64_t rows, cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  for (int64_t first = 0; first < rows && e == cudaSuccess; first += kRowsPerLaunch) {
    const int64_t n = rows - first < kRowsPerLaunch ? rows - first : kRowsPerLaunch;
    a.first_row = first;
    a.end_row = first + n;
    const int A = a.rows.actions;
    if (A <= kFew) {
      sample_warp_kernel<T><<<(unsigned)((n + 3) / 4), 128, 0, stream>>>(a);
    } else {
      // masked, a warp for up to 5120 actions (ten mask loads a lane)
      if (a.rows.mask && A <= 5120) {
        sample_masked_kernel<T><<<(unsigned)((n + 3) / 4), kMaskedThreads, 0, stream>>>(a);
      } else {
        // 32 scores a thread, so that there are many best scores to choose from
        const int threads = min(kSampleThreads, max(32, (A / 32 + 31) / 32 * 32));
        const int vecs = A / (16 / (int)sizeof(T));
        const size_t smem = vecs <= kMaximaVecs ? (size_t)vecs * 4 : 0;
        if (threads <= 64) {
          sample_long_kernel<T, 512, 64><<<(unsigned)n, threads, smem, stream>>>(a);
        } else {
          auto kernel = a.rows.mask ? sample_long_masked_kernel<T> : sample_long_kernel<T, kList, kSampleThreads>;
          // (48 KB go without asking, some 25 KB of the kernel's own included)
          if (smem > 16 * 1024)
            e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaximaVecs * 4);
          if (e != cudaSuccess) break;
          kernel<<<(unsigned)n, threads, smem, stream>>>(a);
        }
      }
    }
    e = cudaGetLastError();
  }
  return e;
}

}  // namespace
}  // namespace policy
}  // namespace gz

using namespace gz;
using namespace gz::policy;

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
  const SampleArgs a{row_args(rows), *cfg, d_noise, noise_stride, d_action, d_logp, 0, 0};
  const cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (rows->dtype == GZ_F32) e = launch_sample<float>(a, rows->rows, s);
  else if (rows->dtype == GZ_F16) e = launch_sample<__half>(a, rows->rows, s);
  else e = launch_sample<__nv_bfloat16>(a, rows->rows, s);
  return e == cudaSuccess ? GZ_OK : set_last_error(GZ_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
}
