// Log probabilities of given tokens from a row of logits x[0..V):
//   m = max x, Z = sum exp(x - m), lp(v) = x_v - m - log Z,
//   entropy = log Z - sum exp(x - m) (x - m) / Z   (a logit of -inf adds nothing),
// and the n largest lp with their ids (ties to the lowest id). All in fp32. A
// row holding NaN or +inf gives NaN log probabilities and entropy, as does one
// with nothing but -inf; a token outside [0, V) gives NaN. Among the
// alternatives NaN counts as the largest value.
//
// One pass over the logits; the bound is their bytes (at 2 bytes a logit and
// 6.5 TB/s an SM takes 11.6 logits a clock: 0.7 of its exponentials and about
// 7 of the 11 instructions a logit may cost). A row goes to one CTA or, when
// there are few rows, to a cluster of 2 to 8 whose partial results rank 0
// joins through distributed shared memory in rank order. Every warp streams a
// part of the row through a ring of its own in shared memory (bulk copies, the
// ends of a row off the 16-byte grid by plain loads), so that no warp waits for
// another; a thread takes 16 or 32 logits (64 bytes) at a time, keeps its own
// running maximum and sums, and raises the maximum at most once for them.
// Alternatives: a logit is a candidate when it reaches a bound that n logits of
// the CTA's part reach for certain: with k = ceil(n / warps), the least over the
// warps of the k-th largest of its 32 lane maxima. The bound rises as the pass
// goes on, so of V random logits only some hundreds are looked at again. It cannot
// rise while a warp has seen fewer than k logits above -inf: where a mask leaves only
// a few ids, or one range of them, every logit is looked at (32 rows of 152064 with 10
// ids or 1000 in a row allowed, 20 alternatives: 56 and 60 us, against 18).
// Candidates wait in a buffer per warp, cut back to its n largest when full; at
// the end the CTA ranks the survivors by counting.
// In a CUDA graph, 2048 rows of 152064 bf16 logits: 105 us without alternatives, 125
// with 8 (91% and 76% of the copy bandwidth; in a call, inputs alternating, 137);
// 1024 rows in fp32 with 8 111 (85%); instruction issue bounds it. 32 rows: 8 us
// without, 13 with 5, 18 with 20: a chain of latencies (the copies, two steps of 32
// logits a thread, the candidates, the joins, one meeting of the cluster).
#include <cooperative_groups.h>

#include "common.cuh"
#include "f32x2.cuh"

namespace cg = cooperative_groups;

namespace tf {
namespace {

constexpr int kTopMax = 32;
constexpr int kCap = 128;      // candidates of a warp
constexpr int kMaxCluster = 8;

// Order of the alternatives: value descending (NaN first), then id ascending,
// as one unsigned 64-bit key; every logit of a row has a key of its own, above 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  uint32_t u = __float_as_uint(v + 0.f);  // -0 orders as +0
  u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return v != v ? 0xffffffffu : u;
}
__device__ __forceinline__ float value_of(uint32_t order) {
  return __uint_as_float((order & 0x80000000u) ? order ^ 0x80000000u : ~order);
}
__device__ __forceinline__ uint64_t key_of(uint32_t order, uint32_t id) { return ((uint64_t)order << 32) | (uint32_t)~id; }

// max(a, b), NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// sum over logits of e = 2^t and of e t, t = (x - m) log2(e), for a running maximum m
struct Sums {
  float m, z, w;
};

// s's sums relative to a maximum m >= s.m (m may be -inf: nothing seen yet)
__device__ __forceinline__ Sums rebase(const Sums& s, float m) {
  if (s.m == m || s.m == -INFINITY) return {m, s.z, s.w};
  const float t = (s.m - m) * kLog2e, f = ex2(t);
  return {m, s.z * f, (s.w + s.z * fmaxf(t, -150.f)) * f};
}
// The sum over a warp's lanes, the same on all of them.
__device__ __forceinline__ Sums join_warp(Sums s) {
  float m = s.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  s = rebase(s, m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.z += __shfl_xor_sync(0xffffffffu, s.z, o);
    s.w += __shfl_xor_sync(0xffffffffu, s.w, o);
  }
  return s;
}

template <typename T>
struct Batch {
  static constexpr int kPer = 16 / (int)sizeof(T);  // logits of a 16-byte load
  static constexpr int kLoads = 4;
  static constexpr int kBatch = kLoads * kPer;      // logits of a thread at a time
  uint4 raw[kLoads];
  static __device__ __forceinline__ uint32_t lowest_word() {
    return std::is_same_v<T, float> ? 0xff800000u : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;  // -inf
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& v = raw[i / 4];
    return (i & 3) == 0 ? v.x : (i & 3) == 1 ? v.y : (i & 3) == 2 ? v.z : v.w;
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (std::is_same_v<T, float>) return __uint_as_float(word(e));
    const uint32_t w = word(e / 2);
    if constexpr (std::is_same_v<T, __nv_bfloat16>) return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return (e & 1) ? __high2float(h) : __low2float(h);
  }
  // The largest (NaN if there is one).
  __device__ __forceinline__ float largest() const {
    if constexpr (std::is_same_v<T, float>) {
      float m = get(0);
#pragma unroll
      for (int e = 1; e < kBatch; ++e) m = max_nan(m, get(e));
      return m;
    } else {
      uint32_t m = word(0);
#pragma unroll
      for (int i = 1; i < kBatch / 2; ++i) m = max_words(m, word(i));
      return of_word(m);
    }
  }
  static __device__ __forceinline__ uint32_t max_words(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (std::is_same_v<T, __half>)
      asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else
      asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float of_word(uint32_t w) {
    Batch<T> two;
    two.raw[0].x = w;
    return max_nan(two.get(0), two.get(1));
  }
  // The least, -inf included (NaN need not show).
  __device__ __forceinline__ float least() const {
    if constexpr (std::is_same_v<T, float>) {
      float m = get(0);
#pragma unroll
      for (int e = 1; e < kBatch; ++e) m = fminf(m, get(e));
      return m;
    } else {
      uint32_t m = word(0);
#pragma unroll
      for (int i = 1; i < kBatch / 2; ++i) {
        if constexpr (std::is_same_v<T, __half>)
          asm("min.f16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
        else
          asm("min.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(word(i)));
      }
      Batch<T> two;
      two.raw[0].x = m;
      return fminf(two.get(0), two.get(1));
    }
  }
};

struct LogprobArgs {
  const void* logits;
  int64_t ld;
  const int64_t* tokens;
  int V, top;
  float* logprob;
  float* entropy;
  float* top_lp;
  int64_t* top_ids;
};

template <int kWarps, int kStages, int kStageBytes>
struct Shared {
  uint8_t ring[kWarps][kStages][kStageBytes];
  uint64_t cand[kWarps][kCap];               // candidates of each warp
  uint64_t list[kWarps * kTopMax];           // the CTA's survivors
  uint64_t best[kTopMax];                    // the CTA's n largest, in order
  uint64_t peers[kMaxCluster * kTopMax];     // of each CTA of the cluster (rank 0's copy is read)
  uint64_t full[kWarps][kStages];            // stage landed
  uint32_t bound[kWarps];                    // k-th largest lane maximum of each warp, so far
  Sums sums[kWarps], cta[kMaxCluster];       // cta: of each CTA of the cluster (rank 0's copy is read)
  int count;
};
// stages of 2 KiB: two hold enough 16-bit logits to work on while the next come
template <typename T, int kThreads>
using SharedOf = Shared<kThreads / 32, std::is_same_v<T, float> ? 3 : 2, 32 * 16 * Batch<T>::kLoads>;

// The n largest of a warp's `count` candidates to its front, in order. Returns how many there are.
__device__ __noinline__ int cut_back(uint64_t* cand, int count, int n) {
  const int lane = threadIdx.x & 31;
  uint64_t mine[kCap / 32];
  int rank[kCap / 32];
#pragma unroll
  for (int i = 0; i < kCap / 32; ++i) {
    mine[i] = lane + 32 * i < count ? cand[lane + 32 * i] : 0;
    rank[i] = 0;
  }
  for (int j = 0; j < count; ++j) {
    const uint64_t k = cand[j];
#pragma unroll
    for (int i = 0; i < kCap / 32; ++i) rank[i] += k > mine[i] ? 1 : 0;
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kCap / 32; ++i)
    if (mine[i] && rank[i] < n) cand[rank[i]] = mine[i];
  __syncwarp();
  return count < n ? count : n;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) logprobs_kernel(const LogprobArgs a) {
  using B = Batch<T>;
  using Sh = SharedOf<T, kThreads>;
  constexpr int kBatch = B::kBatch, kStages = (int)(sizeof(Sh::full[0]) / sizeof(uint64_t));
  extern __shared__ __align__(128) uint8_t smem_lp[];
  Sh& sh = *reinterpret_cast<Sh*>(smem_lp);
  pdl_trigger();
  pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  auto arrived = cluster.barrier_arrive();  // every CTA of the cluster has begun (waited for below)
  const int64_t row = blockIdx.y;
  const int parts = (int)gridDim.x, part = (int)blockIdx.x;  // the cluster's CTAs share the row
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int threads = kThreads, warps = kThreads / 32;
  const T* x = (const T*)a.logits + row * a.ld;
  const int n = a.top;
  float chosen = NAN;  // the given token's logit
  if (part == 0 && tid == 0) {
    const int64_t t = a.tokens[row];
    if (t >= 0 && t < a.V) chosen = Num<T>::to_f(x[t]);
  }

  // [0, head) and [tail, V) off the 16-byte grid; vectors of 16 bytes between
  int head = (int)(((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / sizeof(T));
  head = head < a.V ? head : a.V;
  const int vectors = (a.V - head) / B::kPer, tail = head + vectors * B::kPer;
  // this warp's vectors, in steps of 32 x kLoads
  const int slot = part * warps + warp, slots = parts * warps;
  const int v_begin = (int)((int64_t)vectors * slot / slots), v_end = (int)((int64_t)vectors * (slot + 1) / slots);
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  constexpr int kSpan = 32 * B::kLoads;
  const int steps = (v_end - v_begin + kSpan - 1) / kSpan;
  uint64_t* full = sh.full[warp];
  auto fetch = [&](int step) {  // lane 0
    const int v = v_begin + step * kSpan, left = v_end - v;
    const uint32_t bytes = (uint32_t)(left < kSpan ? left : kSpan) * 16;
    mbar_arrive_expect_tx(&full[step % kStages], bytes);
    bulk_load(sh.ring[warp][step % kStages], body + v, bytes, &full[step % kStages]);
  };
  if (lane == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1);
    fence_mbarrier_init();
    for (int i = 0; i < kStages && i < steps; ++i) fetch(i);
  }
  __syncwarp();

  // Running sums of this thread. While |m| < 1024 they are relative to c, the
  // rounded m log2(e), and a logit takes one multiply-add: t = x log2(e) - c.
  // Beyond (`far`, from then on) the rounding of the product would show, and
  // t = (x - m) log2(e) with the difference taken first.
  float m_run = -INFINITY, c = 0.f, z = 0.f, w = 0.f;
  bool far = false;
  auto shift = [&](float d) {  // the reference moves down by d = old - new, in log2 units
    const float f = ex2(d);
    w = fmaf(z, fmaxf(d, -150.f), w) * f;
    z *= f;
  };
  auto raise = [&](float m) {  // to a maximum m > m_run
    const bool seen = m_run > -INFINITY;
    if (!far && !(fabsf(m) < 1024.f)) {
      if (seen) shift(fmaf(-m_run, kLog2e, c));  // from c to m_run itself
      far = true;
    }
    if (far) {
      if (seen) shift((m_run - m) * kLog2e);
    } else {
      const float c_new = m * kLog2e;
      if (seen) shift(c - c_new);
      c = c_new;
    }
    m_run = m;
  };
  auto add_careful = [&](float v) {  // any logit: -inf counts as 2^-150 (0 in fp32, and 0 x -150 too)
    const float m = fmaxf(m_run, -3.402823466e38f);
    const float t = max_nan(far ? (v - m) * kLog2e : fmaf(v, kLog2e, -c), -150.f), e = ex2(t);
    z += e;
    w = fmaf(e, t, w);
  };
  uint32_t lane_max = 0;  // order of this lane's largest logit
  uint64_t* cand = sh.cand[warp];
  int count = 0;
  uint64_t floor_key = 0;  // candidates are above it
  float least = NAN;       // a bound read earlier: bounds only rise, so it holds still (NaN: none)
  const int k = n > 0 ? (n + warps - 1) / warps : 0;

  // raise this warp's bound: the k-th largest of its lane maxima
  auto publish = [&]() {
    uint32_t v = lane_max, top = 0;
    for (int i = 0;; ++i) {
      top = __reduce_max_sync(0xffffffffu, v);
      if (i == k - 1) break;
      const unsigned who = __ballot_sync(0xffffffffu, v == top);
      if (lane == __ffs(who) - 1) v = 0;
    }
    if (lane == 0) *(volatile uint32_t*)&sh.bound[warp] = top;
  };
  auto bound = [&]() {  // the least of the warps' bounds, as a value (0, nothing seen yet: NaN)
    const uint32_t u =
        __reduce_min_sync(0xffffffffu, lane < warps ? *(volatile uint32_t*)&sh.bound[lane] : 0xffffffffu);
    return value_of(u);
  };
  auto offer = [&](float v, uint32_t id, bool valid) {
    const uint64_t key = key_of(order_of(v), id);
    const bool take = valid && !(v < least) && key > floor_key;
    const unsigned who = __ballot_sync(0xffffffffu, take);
    if (count + __popc(who) > kCap) {
      __syncwarp();
      count = cut_back(cand, count, n);
      if (count == n) floor_key = cand[n - 1];
    }
    if (take) cand[count + __popc(who & ((1u << lane) - 1))] = key;
    count += __popc(who);
    __syncwarp();
  };

  bool ok = true, synced = false;
  auto step = [&](int i, bool whole) {
    const uint4* stage = reinterpret_cast<const uint4*>(sh.ring[warp][i % kStages]) + lane;
    const int v0 = v_begin + i * kSpan + lane;
    B b;
    if (whole) {
#pragma unroll
      for (int j = 0; j < B::kLoads; ++j) b.raw[j] = stage[32 * j];
    } else {
      const uint32_t w = B::lowest_word();
#pragma unroll
      for (int j = 0; j < B::kLoads; ++j) b.raw[j] = v0 + 32 * j < v_end ? stage[32 * j] : make_uint4(w, w, w, w);
    }
    const float big = b.largest();
    if (big > m_run) raise(big);
    if (b.least() > -1e38f && !far) {  // no -inf: no product overflows
      const uint64_t scale = pair(kLog2e, kLog2e), shift2 = pair(-c, -c);
      uint64_t zz = pair(z, 0.f), ww = pair(w, 0.f);
#pragma unroll
      for (int e = 0; e < kBatch; e += 2) {
        const uint64_t t = fma2(pair(b.get(e), b.get(e + 1)), scale, shift2);
        float t0, t1;
        unpair(t, t0, t1);
        const uint64_t p = pair(ex2(t0), ex2(t1));
        zz = add2(zz, p);
        ww = fma2(p, t, ww);
      }
      float z1, w1;
      unpair(zz, z, z1);
      unpair(ww, w, w1);
      z += z1;
      w += w1;
    } else {
#pragma unroll
      for (int e = 0; e < kBatch; ++e) add_careful(b.get(e));
    }
    if (n > 0 && __any_sync(0xffffffffu, !(big < least))) {
      if (v0 < v_end && !(big < least)) {
        const uint32_t o = order_of(big);
        lane_max = o > lane_max ? o : lane_max;
      }
      publish();
      if (!synced) __syncthreads();  // every warp has a bound
      synced = true;
      least = bound();
      // lanes with logits that reach it (seldom more than one): the warp looks
      // through the lane's logits, one each
      unsigned who = __ballot_sync(0xffffffffu, !(big < least));
      while (who) {
        const int src = __ffs(who) - 1, e = lane % kBatch, v = v0 - lane + src + (e / B::kPer) * 32;
        who &= who - 1;
        const T* at = reinterpret_cast<const T*>(stage - lane + src + (e / B::kPer) * 32) + e % B::kPer;
        offer(Num<T>::to_f(*at), (uint32_t)(head + v * B::kPer + e % B::kPer), lane < kBatch && v < v_end);
      }
    }
  };
  for (int i = 0; i < steps; ++i) {
    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[i % kStages], (uint32_t)(i / kStages) & 1u, nullptr, 0));
    if (!ok) break;
    if (i < steps - 1) step(i, true);
    else step(i, false);
    __syncwarp();  // the stage is read: fill it again
    if (lane == 0 && i + kStages < steps) fetch(i + kStages);
  }
  if (!ok)  // a copy that has not come in a second (below: NaN); the others in flight land before the CTA exits
    for (int i = 0; i < kStages && i < steps; ++i) mbar_wait_bounded(&full[i], 0u, nullptr, 0);
  if (n > 0 && !synced) {  // nothing here, but the other warps wait for a bound
    if (lane == 0) sh.bound[warp] = 0;
    __syncthreads();
  }
  // the ends of the row, by the last part's first warp
  const int ends = head + (a.V - tail);
  if (part == parts - 1 && warp == 0 && ends > 0) {
    const int id = lane < head ? lane : tail + (lane - head);
    const bool valid = lane < ends;
    const float v = valid ? Num<T>::to_f(x[id]) : -INFINITY;
    if (v > m_run) raise(v);
    if (valid) add_careful(v);
    if (n > 0) {
      least = bound();
      offer(v, (uint32_t)id, valid);
    }
  }

  // join the lanes, the warps, the CTAs (in that order: a fixed one)
  if (!far && m_run > -INFINITY) shift(fmaf(-m_run, kLog2e, c));  // all relative to a maximum from here on
  Sums s = join_warp({m_run, z, w});
  if (!ok) s.z = NAN;  // a copy that never came: the row has no result
  if (lane == 0) sh.sums[warp] = s;
  if (tid == 0) sh.count = 0;
  if (tid < kTopMax) sh.best[tid] = 0;
  __syncthreads();
  if (n > 0) {
    // the candidates that reach the last bound, to one list (seldom more than it holds)
    const float last = bound();
    const uint32_t order = last != last ? 0 : order_of(last);
    for (bool again = false;; again = true) {
      for (int i = 0; i < count; i += 32) {
        const uint64_t key = i + lane < count ? cand[i + lane] : 0;
        const bool take = i + lane < count && (uint32_t)(key >> 32) >= order;
        const unsigned who = __ballot_sync(0xffffffffu, take);
        int at = 0;
        if (lane == 0 && who) at = atomicAdd(&sh.count, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (take && at < warps * kTopMax) sh.list[at] = key;
      }
      __syncthreads();
      if (again || sh.count <= warps * kTopMax) break;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      if (count > n) count = cut_back(cand, count, n);
      __syncthreads();
    }
  }
  auto rank_list = [&](const uint64_t* list, int total) {  // the n largest of `total` to best, in order
    constexpr int kSplit = 8;                              // lanes that count for one
    for (int i0 = 0; i0 < total; i0 += threads / kSplit) {
      const int i = i0 + tid / kSplit;
      const uint64_t key = i < total ? list[i] : 0;
      int rank = 0;
#pragma unroll 4
      for (int j = tid % kSplit; j < total; j += kSplit) rank += list[j] > key ? 1 : 0;
#pragma unroll
      for (int o = kSplit / 2; o > 0; o >>= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (tid % kSplit == 0 && key && rank < n) sh.best[rank] = key;
    }
  };
  if (n > 0) rank_list(sh.list, sh.count);
  Sums all = join_warp(lane < warps ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f});
  cluster.barrier_wait(std::move(arrived));
  if (parts > 1) {
    Sh* root = cluster.map_shared_rank(&sh, 0);
    __syncthreads();  // `best` is complete
    if (tid == 0) root->cta[part] = all;
    if (tid < n) root->peers[part * n + tid] = sh.best[tid];
    cluster.sync();
    if (part != 0) return;
    all = join_warp(lane < parts ? sh.cta[lane] : Sums{-INFINITY, 0.f, 0.f});
    if (n > 0) rank_list(sh.peers, parts * n);
  }
  __syncthreads();
  // a row of nothing but -inf has no distribution
  const float lz = all.m == -INFINITY ? NAN : logf(all.z);
  if (tid == 0) {
    a.logprob[row] = (chosen - all.m) - lz;
    a.entropy[row] = lz - all.w * kLn2 / all.z;
  }
  if (tid < n) {
    const uint32_t id = ~(uint32_t)sh.best[tid];
    a.top_ids[row * n + tid] = id;
    a.top_lp[row * n + tid] = (value_of((uint32_t)(sh.best[tid] >> 32)) - all.m) - lz;
  }
}

template <typename T, int kThreads>
int go_logprobs(dim3 grid, dim3 cluster, const LogprobArgs& a, cudaStream_t st) {
  constexpr auto kern = logprobs_kernel<T, kThreads>;
  constexpr size_t smem = sizeof(SharedOf<T, kThreads>);
  const int rc = allow_smem<kern>("token_logprobs", smem);
  if (rc != TF_OK) return rc;
  return launch_ex("token_logprobs", kern, grid, dim3(kThreads), smem, st, cluster, a);
}

template <typename T>
int launch_logprobs(const LogprobArgs& a, int64_t M, cudaStream_t st) {
  // Few rows (their clusters of 8 x 512 threads all resident at 1024 threads an
  // SM): the latency of a row counts, so the widest cluster. Else CTAs of 256
  // threads, in clusters as wide as lets all rows be resident at once.
  const int64_t room = (int64_t)num_sms() * 1024;
  const bool wide = M * kMaxCluster * 512 <= room;
  int parts = wide ? kMaxCluster : 1;
  while (!wide && parts < kMaxCluster && M * parts * 2 * 256 <= room) parts *= 2;
  const dim3 grid((unsigned)parts, (unsigned)M), cluster((unsigned)parts, 1, 1);
  if (wide) return go_logprobs<T, 512>(grid, cluster, a, st);
  return go_logprobs<T, 256>(grid, cluster, a, st);
}

}  // namespace
}  // namespace tf

extern "C" int tf_token_logprobs(const void* logits, int64_t ld, const int64_t* tokens, int64_t M, int64_t V,
                                 int32_t top, int dtype, float* logprob, float* entropy, float* top_logprobs,
                                 int64_t* top_ids, void* stream) {
  using namespace tf;
  if (M < 0 || V <= 0 || V > (1 << 30) || M > INT32_MAX || ld < V)
    return fail(TF_ERR_BAD_SHAPE, "token_logprobs: bad shape (M=%lld, V=%lld, ld=%lld)", (long long)M, (long long)V,
                (long long)ld);
  if (top < 0 || top > kTopMax || top > V)
    return fail(TF_ERR_BAD_ARG, "token_logprobs: top %d (0 to %d, at most V)", top, kTopMax);
  if (dtype != TF_F16 && dtype != TF_BF16 && dtype != TF_F32)
    return fail(TF_ERR_BAD_DTYPE, "token_logprobs: unsupported dtype %d", dtype);
  if (M == 0) return TF_OK;
  if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids)))
    return fail(TF_ERR_BAD_ARG, "token_logprobs: null pointer");
  const size_t item = dtype == TF_F32 ? 4 : 2;
  if (!aligned(logits, item)) return fail(TF_ERR_UNALIGNED, "token_logprobs: logits must be aligned to their type");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // rows go to the grid's y axis, at most 65535 of them
  for (int64_t r0 = 0; r0 < M; r0 += 65535) {
    const int64_t rows = M - r0 < 65535 ? M - r0 : 65535;
    const LogprobArgs a{(const char*)logits + r0 * ld * (int64_t)item, ld, tokens + r0, (int)V, top, logprob + r0,
                        entropy + r0, top ? top_logprobs + r0 * top : nullptr, top ? top_ids + r0 * top : nullptr};
    const int rc = dtype == TF_F16    ? launch_logprobs<__half>(a, rows, st)
                   : dtype == TF_BF16 ? launch_logprobs<__nv_bfloat16>(a, rows, st)
                                      : launch_logprobs<float>(a, rows, st);
    if (rc != TF_OK) return rc;
  }
  return TF_OK;
}
