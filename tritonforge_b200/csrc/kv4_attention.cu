// Single-token attention over the 4-bit KV cache (format: kv4.cuh): for each
// sequence b and query head h, over its first lens[b] positions,
//   out = sum_t p_t v_t,  p = softmax_t(scale q . k_t),
// with k_t, v_t the values the codes stand for, (code - zero) * scale:
//   q . k_t = s_t (sum_d q_d c_td - z_t sum_d q_d)   per group of channels,
//   out     = sum_t p_t s_t (c_td - z_t).
// Softmax and accumulators are in fp32, the output is rounded once; a sequence
// without positions gives zeros. The bound is the bytes of the cached rows.
//
// Products: mma.sync on the codes themselves. A 4-bit code under the mask
// 0x000f000f is a subnormal fp16 number, code 2^-24, under 0x00f000f0 16 times
// that: no conversion at all, the powers of two go into the other operand or
// into the result. The tensor cores line addends up by their exponents, a
// subnormal's being -14 whatever its leading zeros, and drop what lies 2^-24 below
// the largest: beside a code of 8 addends are kept to 2^-17 of it under the first
// mask, to 2^-21 under the second. The values' sums, from which the zero points take
// most away again, use the second for both nibbles (a shift; 32 x 4096, 64 / 8
// heads: 37.3 -> 37.9 us; code - zero as normal numbers 48). Scores keep the first
// for every other nibble: 2^-15 of the largest |q| a product, which does not show
// beside the rounded weights (the second for all of them: 39.9 us, errors against
// 64 bits equal, also with one channel of q 400 times the others).
// Per 16 positions a warp takes S^T = K Q^T (rows: positions,
// columns: up to 8 query heads of the kv head) and O^T += V^T P^T; a row of the
// cache is read as it lies, its channels in whatever order the nibbles come
// (the same for q). tcgen05 would want the codes as 16-bit operands in shared
// memory: 4 times the cache's bytes through it.
// q is scaled by a power of two per head to fp16's upper range; P s, rounded to
// fp16, is kept below 2^15 by the running maximum of the scores and a running
// power of two above the value scales (both raised only when passed by 2^3).
// The zero points multiply the rounded P s too, so each value's weight is
// rounded once.
//
// Work split: a unit is 128 positions of one row (sequence, kv head and block of
// up to 8 query heads); CTAs take equal shares of all units in order, whatever
// the lengths are, and not less than kMinUnits each while that leaves a share
// per row. A row inside one share is finished there; a row cut by shares leaves
// (m, l, O) pieces in the workspace. The last CTA to leave one of a group of
// about sqrt(pieces) joins the group, the last of the groups the row, always in
// order: results do not depend on timing. One warp streams the share through a
// ring in shared memory (bulk copies), four compute, 32 positions of a unit each.
//
// In a CUDA graph, 32 x 4096 positions: 38.1 us with 64 / 8 heads of 128, 58% of the
// copy bandwidth, 25.9 with 28 / 4, 14.0 with 14 / 2 heads of 64; rotating and
// appending the new token too (the fused form) 44.3, 29.9 and 16.8. Two or three
// warps a scheduler issue in 47% of the cycles, each waiting for its own chain of
// products, exponentials and shuffles, and about 8 us go to the start and the joins:
// that is all of it for short batches (300 positions: 5.0 us, fused 6.6; 16 sequences
// of 1125 on average, 28 / 4 heads: 14.0, fused 17.8).
#include "kv4.cuh"

namespace tf {
namespace {

constexpr int kHeads = 8;         // query heads of a row
constexpr int kUnit = 128;        // positions of a unit
constexpr int kWarps = 4;         // computing warps, 32 positions of a unit each
constexpr int kMinUnits = 4;      // of a share
constexpr int kThreads = 32 * (kWarps + 1);
// CTAs per SM. At D = 128 registers count: two at 168 (batch 32 x 4096, 72B
// shape: 37.5 us) beat three at 128 (42), six or eight warps each at 144 and 112
// (44, 43) and one (57); at D = 64 warps do: three.
template <int D>
constexpr int kCtasPerSm = D == 64 ? 3 : 2;
constexpr float kRaise = 3.f;     // log2 of how far scores may pass the running maximum
constexpr float kNorm = 2048.f;   // P s below 2^11 at the running maximum and scale

struct Kv4Args {
  const void* q;   // [B, hq, D], or the projection rows (kRope)
  int64_t q_ld;    // elements between the rows of two sequences
  const void* cos_t;
  const void* sin_t;
  Kv4Cache c;
  void* out;
  const int* lens;  // positions attended; kRope: the new token's position
  int B, hq, hkv, blocks, per_block;  // blocks of per_block query heads per kv head
  int64_t t_max;
  float scale;
  int* err;
  float* pieces;   // [2 per CTA][Piece floats]
  int* arrived;    // [2 levels][2 per CTA], zero between launches
};

template <int D>
constexpr int piece_floats() { return kHeads * D + 2 * kHeads; }  // O, m, l

template <int D, int GS>
struct Stage {
  static constexpr int G = D / GS;
  uint8_t k[kUnit][D / 2];
  uint8_t v[kUnit][D / 2];
  uint32_t kp[kUnit][G];
  uint32_t vp[kUnit][G];
};

template <int D, int GS>
struct Smem {
  static constexpr int kStages = 4;
  Stage<D, GS> ring[kStages];
  float o[kWarps][kHeads][D];
  float m[kWarps][kHeads], l[kWarps][kHeads];
  uint64_t full[kStages], freed[kStages];
  int64_t total, skipped;  // units in all, units of the sequences before `first`
  int64_t shares;          // CTAs with work
  int first;               // sequence of this CTA's first unit
  int last;                // this CTA joins the row
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Position (of 16) of row i of the S^T tile, column i of V^T: any order does;
// this one spreads both operands' shared-memory reads over the banks.
__device__ __forceinline__ int position_of(int i) {
  const int c = (i & 7) >> 1;
  return (i & 8) + ((i & 1) ? (c ^ 1) + 4 : c);
}

// One piece of a CTA's share: units [u0, u1) of `units`, all of one row.
struct Piece {
  int b, kh, hb;
  int tiles;           // units of the row
  int t0, t1;          // this CTA's
  int64_t row_u0;      // the row's first unit, of all
  int len;
};

// Walks a share [u, end) row by row. b, skipped: the sequence of unit u and the
// units before it.
struct Walk {
  int64_t u, end, skipped;
  int b;
};
template <bool kRope>
__device__ __forceinline__ int length_of(const Kv4Args& a, int b) {
  int64_t n = a.lens[b];
  if (kRope) n = n >= 0 && n < a.t_max ? n + 1 : 0;  // the new token's position must lie in the cache
  return (int)(n < 0 ? 0 : (n > a.t_max ? a.t_max : n));
}
template <bool kRope>
__device__ __forceinline__ bool next_piece(const Kv4Args& a, Walk& w, Piece& p) {
  if (w.u >= w.end) return false;
  const int rows = a.hkv * a.blocks;
  for (;;) {  // sequences without positions own no unit
    p.len = length_of<kRope>(a, w.b);
    p.tiles = (p.len + kUnit - 1) / kUnit;
    if (w.u < w.skipped + (int64_t)p.tiles * rows) break;
    w.skipped += (int64_t)p.tiles * rows;
    ++w.b;
  }
  const int64_t in = w.u - w.skipped;
  const int row = (int)(in / p.tiles);
  p.b = w.b;
  p.kh = row / a.blocks;
  p.hb = row % a.blocks;
  p.t0 = (int)(in - (int64_t)row * p.tiles);
  p.row_u0 = w.skipped + (int64_t)row * p.tiles;
  const int64_t left = w.end - w.u;
  p.t1 = left < p.tiles - p.t0 ? p.t0 + (int)left : p.tiles;
  w.u += p.t1 - p.t0;
  return true;
}

// Eight rotated channels [d, d + 8) of a head's row (transformers' roundings).
template <typename T, int D>
__device__ __forceinline__ void rotate8(const T* row, const T* cs, const T* sn, int d, float* y) {
  const int other = d < D / 2 ? d + D / 2 : d - D / 2;
  Half8<T> x, o, c, s;
  x.raw = *reinterpret_cast<const uint4*>(row + d);
  o.raw = *reinterpret_cast<const uint4*>(row + other);
  c.raw = *reinterpret_cast<const uint4*>(cs + d);
  s.raw = *reinterpret_cast<const uint4*>(sn + d);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float turned = d < D / 2 ? -o.get(e) : o.get(e);
    y[e] = round_to<T>(round_to<T>(x.get(e) * c.get(e)) + round_to<T>(turned * s.get(e)));
  }
}

// The new token's key (rotated) and value, quantised by a warp into position
// `at` of the unit in shared memory and into the cache.
template <typename T, int D, int GS>
__device__ __forceinline__ void append(const Kv4Args& a, const Piece& p, Stage<D, GS>& st, int at) {
  constexpr int G = D / GS, kLanes = D / 16;
  const int lane = threadIdx.x & 31, i = lane % kLanes;
  const bool key = lane < kLanes, mine = lane < 2 * kLanes;  // other lanes repeat the value's
  const int pos = p.len - 1;
  const T* row = reinterpret_cast<const T*>(a.q) + p.b * a.q_ld +
                 (int64_t)(a.hq + p.kh + (key ? 0 : a.hkv)) * D;
  Half8<T> x1, x2;
  if (key) {
    const T* cs = (const T*)a.cos_t + (int64_t)pos * D;
    const T* sn = (const T*)a.sin_t + (int64_t)pos * D;
    float y1[8], y2[8];
    rotate8<T, D>(row, cs, sn, 8 * i, y1);
    rotate8<T, D>(row, cs, sn, D / 2 + 8 * i, y2);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x1.set(e, y1[e]);
      x2.set(e, y2[e]);
    }
  } else {
    x1.raw = *reinterpret_cast<const uint4*>(row + 8 * i);
    x2.raw = *reinterpret_cast<const uint4*>(row + D / 2 + 8 * i);
  }
  __syncwarp();
  uint32_t w1, w2, params;
  kv4_quantize_row<T, D, GS>(x1, x2, i, w1, w2, params);
  if (mine) {
    const int64_t at_row = ((int64_t)p.b * a.hkv + p.kh) * a.t_max + pos;
    uint8_t* to[2] = {(key ? st.k : st.v)[at], (key ? a.c.k : a.c.v) + at_row * (D / 2)};
    uint32_t* par[2] = {(key ? st.kp : st.vp)[at],
                        reinterpret_cast<uint32_t*>(key ? a.c.k_params : a.c.v_params) + at_row * G};
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      *reinterpret_cast<uint32_t*>(to[y] + 4 * i) = w1;
      *reinterpret_cast<uint32_t*>(to[y] + D / 4 + 4 * i) = w2;
      if (i < G) par[y][i] = params;
    }
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the stage is filled again
  __syncwarp();
}

// Joins n pieces of a row (k0, k0 + step, ...; slot_of(k) of the workspace), in
// that order, into one piece (into the first one's place) or the row's output.
// By the kWarps computing warps; a thread takes four channels of kPer heads,
// four pieces at a time (their loads wait together).
template <typename T, int D, typename Slot>
__device__ __forceinline__ void join(float* pieces, Slot slot_of, int k0, int step, int n, int heads, float* into,
                                     T* out) {
  constexpr int kPer = (kHeads * D / 4 + 32 * kWarps - 1) / (32 * kWarps);
  const int tid = threadIdx.x;
  float4 o[kPer];
  float m[kPer], l[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    o[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[j] = -INFINITY;
    l[j] = 0.f;
  }
  for (int b = 0; b < n; b += 4) {
    float4 v[4][kPer];
    float mk[4][kPer], lk[4][kPer];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float* q = pieces + (int64_t)slot_of(k0 + (b + k < n ? b + k : n - 1) * step) * piece_floats<D>();
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int i = 4 * (tid + j * 32 * kWarps);
        if (b + k < n && i < heads * D) {
          v[k][j] = __ldcg(reinterpret_cast<const float4*>(q + i));
          mk[k][j] = __ldcg(q + kHeads * D + i / D);
          lk[k][j] = __ldcg(q + kHeads * D + kHeads + i / D);
        } else {
          v[k][j] = make_float4(0.f, 0.f, 0.f, 0.f);
          mk[k][j] = -INFINITY;
          lk[k][j] = 0.f;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const float top = fmaxf(fmaxf(fmaxf(mk[0][j], mk[1][j]), fmaxf(mk[2][j], mk[3][j])), m[j]);
      const float f = m[j] > -INFINITY ? ex2(m[j] - top) : 1.f;
      o[j] = make_float4(o[j].x * f, o[j].y * f, o[j].z * f, o[j].w * f);
      l[j] *= f;
      m[j] = top;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float g = mk[k][j] > -INFINITY ? ex2(mk[k][j] - top) : 1.f;
        o[j].x = fmaf(v[k][j].x, g, o[j].x);
        o[j].y = fmaf(v[k][j].y, g, o[j].y);
        o[j].z = fmaf(v[k][j].z, g, o[j].z);
        o[j].w = fmaf(v[k][j].w, g, o[j].w);
        l[j] = fmaf(lk[k][j], g, l[j]);
      }
    }
  }
  if (into) named_barrier(1, 32 * kWarps);  // every piece is read
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int i = 4 * (tid + j * 32 * kWarps);
    if (i >= heads * D) continue;
    if (into) {
      __stcg(reinterpret_cast<float4*>(into + i), o[j]);
      if (i % D == 0) {
        __stcg(into + kHeads * D + i / D, m[j]);
        __stcg(into + kHeads * D + kHeads + i / D, l[j]);
      }
    } else {
      const float inv = 1.f / l[j];
      const T y[4] = {Num<T>::from_f(o[j].x * inv), Num<T>::from_f(o[j].y * inv), Num<T>::from_f(o[j].z * inv),
                      Num<T>::from_f(o[j].w * inv)};
      *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(y);
    }
  }
}

template <typename T, int D, int GS, bool kRope>
__global__ void __launch_bounds__(kThreads, kCtasPerSm<D>) kv4_attn_kernel(const Kv4Args a) {
  constexpr int G = D / GS;
  constexpr int KW = GS / 32;          // words of a lane's part of a key group
  constexpr int VB = GS / 16;          // bytes of a lane's part of a value group
  constexpr int kTiles = D / 16;       // 16-channel tiles of O^T
  using Sm = Smem<D, GS>;
  constexpr int kStages = Sm::kStages;
  extern __shared__ __align__(128) uint8_t smem_kv4[];
  Sm& sm = *reinterpret_cast<Sm*>(smem_kv4);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rows = a.hkv * a.blocks;
  pdl_trigger();
  pdl_wait();

  if (warp == kWarps) {
    if (lane == 0) {
      for (int i = 0; i < kStages; ++i) {
        mbar_init(&sm.full[i], 1);
        mbar_init(&sm.freed[i], kWarps);
      }
      fence_mbarrier_init();
    }
    // units in all, then the sequence that this CTA's first unit belongs to
    auto units_of = [&](int b) { return b < a.B ? (length_of<kRope>(a, b) + kUnit - 1) / kUnit : 0; };
    int64_t total = 0, full_rows = 0;
    int t = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      t = units_of(b0 + lane);
      total += __reduce_add_sync(0xffffffffu, (unsigned)t);
      full_rows += __popc(__ballot_sync(0xffffffffu, t > 0));
    }
    total *= rows;
    full_rows *= rows;
    int64_t shares = (total + kMinUnits - 1) / kMinUnits;
    shares = shares > full_rows ? shares : full_rows;
    shares = shares < gridDim.x ? shares : gridDim.x;
    const int64_t begin = shares > 0 ? (int64_t)blockIdx.x * total / shares : 0;
    int64_t before = 0;
    int first = 0;
    for (int b0 = 0; b0 < a.B; b0 += 32) {
      if (a.B > 32) t = units_of(b0 + lane);
      int sum = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned who = __ballot_sync(0xffffffffu, (before + sum) * rows > begin);
      if (who) {
        const int src = __ffs(who) - 1;
        first = b0 + src;
        before += __shfl_sync(0xffffffffu, sum - t, src);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
      sm.total = total;
      sm.shares = shares;
      sm.first = first;
      sm.skipped = before * rows;
    }
  }
  // sequences without positions: zeros
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (length_of<kRope>(a, b) == 0)
      for (int i = tid; i < a.hq * D / 8; i += kThreads)
        reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.out) + (int64_t)b * a.hq * D)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  const int64_t total = sm.total;
  const int64_t shares = sm.shares;  // at most `total`: every share holds a unit
  if (blockIdx.x >= shares) return;
  const int64_t share0 = (int64_t)blockIdx.x * total / shares;
  Walk walk{share0, (int64_t)(blockIdx.x + 1) * total / shares, sm.skipped, sm.first};
  Piece p;

  if (warp == kWarps) {
    // ------------------------------------------------------------- copies
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      while (ok && next_piece<kRope>(a, walk, p)) {
        const int64_t row0 = ((int64_t)p.b * a.hkv + p.kh) * a.t_max;
        for (int t = p.t0; t < p.t1; ++t, ++it) {
          const int slot = it % kStages;
          if (it >= kStages && !mbar_wait_bounded(&sm.freed[slot], (uint32_t)(it / kStages - 1) & 1u, a.err, 1)) {
            ok = false;
            break;
          }
          const int64_t row = row0 + (int64_t)t * kUnit;
          // whole 16-position tiles (the cache's length is a multiple of 16)
          int n = (p.len - t * kUnit + 15) & ~15;
          n = n < kUnit ? n : kUnit;
          Stage<D, GS>& st = sm.ring[slot];
          mbar_arrive_expect_tx(&sm.full[slot], (uint32_t)(n * (D + 8 * G)));
          bulk_load(st.k, a.c.k + row * (D / 2), (uint32_t)(n * (D / 2)), &sm.full[slot]);
          bulk_load(st.kp, (const uint32_t*)a.c.k_params + row * G, (uint32_t)(n * 4 * G), &sm.full[slot]);
          bulk_load(st.v, a.c.v + row * (D / 2), (uint32_t)(n * (D / 2)), &sm.full[slot]);
          bulk_load(st.vp, (const uint32_t*)a.c.v_params + row * G, (uint32_t)(n * 4 * G), &sm.full[slot]);
        }
      }
      if (!ok)  // what is in flight lands before the CTA exits
        for (int i = (it > kStages ? it - kStages : 0); i < it; ++i)
          mbar_wait_bounded(&sm.full[i % kStages], (uint32_t)(i / kStages) & 1u, a.err, 4);
    }
    return;
  }

  // -------------------------------------------------------------- compute
  const int r = lane >> 2, c = lane & 3;
  int it = 0;
  bool alive = true;  // a wait gave up: the rest is walked through without work
  while (next_piece<kRope>(a, walk, p)) {
    const int heads = min(a.per_block, a.hq / a.hkv - p.hb * a.per_block);
    const int h0 = p.kh * (a.hq / a.hkv) + p.hb * a.per_block;
    const int pos = p.len - 1;  // kRope: the new token's
    // q of head r in the codes' channel order: pairs of nibbles (0, 4), (1, 5), (2, 6), (3, 7) of a word
    uint32_t qf[G * KW][4];
    float f_r = 0.f, qz_r[G];  // of head r: score = s (f C - z qz)
    {
      float x[G * KW][8], big = 0.f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          float* y = x[g * KW + w];
          const int d = g * GS + c * (GS / 4) + 8 * w;
          if (r < heads) {
            const T* row = reinterpret_cast<const T*>(a.q) + p.b * a.q_ld + (int64_t)(h0 + r) * D;
            if constexpr (kRope) {
              rotate8<T, D>(row, (const T*)a.cos_t + (int64_t)pos * D, (const T*)a.sin_t + (int64_t)pos * D, d, y);
            } else {
              Half8<T> v;
              v.raw = *reinterpret_cast<const uint4*>(row + d);
#pragma unroll
              for (int e = 0; e < 8; ++e) y[e] = v.get(e);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = 0.f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum += y[e];
            big = fmaxf(big, fabsf(y[e]));
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qz_r[g] = sum * a.scale * 1.4426950408889634f;
      }
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, 2));
      int up = 14 - ((int)(__float_as_uint(big) >> 23) - 127);  // big 2^up in [2^14, 2^15)
      up = big > 0.f && big < INFINITY ? max(-100, min(up, 120)) : 0;
      const float lift = __uint_as_float((uint32_t)(127 + up) << 23);
      f_r = __uint_as_float((uint32_t)(127 + 24 - up) << 23) * a.scale * 1.4426950408889634f;
#pragma unroll
      for (int i = 0; i < G * KW; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float by = (e & 1) ? lift * 0.0625f : lift;
          qf[i][e] = half2_of(x[i][e] * by, x[i][e + 4] * by);
        }
    }
    // of the heads 2c, 2c + 1 of this lane's scores
    const float f0 = __shfl_sync(0xffffffffu, f_r, 8 * c), f1 = __shfl_sync(0xffffffffu, f_r, 8 * c + 4);
    float qz0[G], qz1[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      qz0[g] = __shfl_sync(0xffffffffu, qz_r[g], 8 * c);
      qz1[g] = __shfl_sync(0xffffffffu, qz_r[g], 8 * c + 4);
    }

    float acc[kTiles][4], za[G][2];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
    for (int g = 0; g < G; ++g) za[g][0] = za[g][1] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    float top = 0.f, norm = 0.f;  // power of two above the value scales seen, 2^11 / top

    const int tok = 32 * warp + position_of(r);  // and + 8; of the second tile + 16, + 24
    const int vtok = 32 * warp + position_of(2 * c), vtok1 = 32 * warp + position_of(2 * c + 1);  // and + 8
    for (int t = p.t0; t < p.t1; ++t, ++it) {
      const int slot = it % kStages;
      alive = __all_sync(0xffffffffu, alive && mbar_wait_bounded(&sm.full[slot], (uint32_t)(it / kStages) & 1u, a.err, 2));
      const int left = p.len - t * kUnit;  // positions of the unit that count
      Stage<D, GS>& st = sm.ring[slot];
      // the row's last position is the new token: the copy in shared memory is of what was there before
      if (kRope && alive && left <= kUnit && (left - 1) / 32 == warp) append<T, D, GS>(a, p, st, left - 1);
      if (alive && 32 * warp < left) {
        // scores of positions tok + 16 u (+ 8), heads 2c, 2c + 1
        float x[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int ta = tok + 16 * u, tb = ta + 8;
          x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            uint32_t ka[KW], kb[KW];
            const uint32_t* pa = reinterpret_cast<const uint32_t*>(&st.k[ta][g * (GS / 2)]) + c * KW;
            const uint32_t* pb = reinterpret_cast<const uint32_t*>(&st.k[tb][g * (GS / 2)]) + c * KW;
            if constexpr (KW == 4) {
              *reinterpret_cast<uint4*>(ka) = *reinterpret_cast<const uint4*>(pa);
              *reinterpret_cast<uint4*>(kb) = *reinterpret_cast<const uint4*>(pb);
            } else {
              *reinterpret_cast<uint2*>(ka) = *reinterpret_cast<const uint2*>(pa);
              *reinterpret_cast<uint2*>(kb) = *reinterpret_cast<const uint2*>(pb);
            }
            const Kv4Group ga = kv4_unpack_params<T>(st.kp[ta][g]), gb = kv4_unpack_params<T>(st.kp[tb][g]);
            float s[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};  // two chains
#pragma unroll
            for (int w = 0; w < KW; ++w) {
              const uint32_t f[4] = {ka[w] & 0x000f000fu, kb[w] & 0x000f000fu, ka[w] & 0x00f000f0u,
                                     kb[w] & 0x00f000f0u};
              mma16816(s, f, qf[g * KW + w][0], qf[g * KW + w][1]);
              const uint32_t ha = ka[w] >> 8, hb = kb[w] >> 8;
              const uint32_t e[4] = {ha & 0x000f000fu, hb & 0x000f000fu, ha & 0x00f000f0u, hb & 0x00f000f0u};
              mma16816(s2, e, qf[g * KW + w][2], qf[g * KW + w][3]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[e] += s2[e];
            x[u][0] = fmaf(ga.scale, fmaf(s[0], f0, -ga.zero * qz0[g]), x[u][0]);
            x[u][1] = fmaf(ga.scale, fmaf(s[1], f1, -ga.zero * qz1[g]), x[u][1]);
            x[u][2] = fmaf(gb.scale, fmaf(s[2], f0, -gb.zero * qz0[g]), x[u][2]);
            x[u][3] = fmaf(gb.scale, fmaf(s[3], f1, -gb.zero * qz1[g]), x[u][3]);
          }
        }
        uint32_t vp[2][2][G];  // value parameters of the same positions
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int g = 0; g < G; ++g) vp[u][e][g] = st.vp[tok + 16 * u + 8 * e][g];
        if (32 * warp + 32 > left) {  // positions past the length hold anything
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (tok + 16 * u + 8 * e >= left) {
                x[u][2 * e] = x[u][2 * e + 1] = -INFINITY;
#pragma unroll
                for (int g = 0; g < G; ++g) vp[u][e][g] = 0u;
              }
        }
        float sc = 0.f;
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int u = 0; u < 2; ++u)
            sc = fmaxf(sc, fmaxf(kv4_unpack_params<T>(vp[u][0][g]).scale, kv4_unpack_params<T>(vp[u][1][g]).scale));
        float x0 = fmaxf(fmaxf(x[0][0], x[0][2]), fmaxf(x[1][0], x[1][2]));
        float x1 = fmaxf(fmaxf(x[0][1], x[0][3]), fmaxf(x[1][1], x[1][3]));
        if (__any_sync(0xffffffffu, x0 > m0 + kRaise || x1 > m1 + kRaise || sc > top)) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, o));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, o));
          }
          sc = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(sc)));  // scales are not negative
          const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
          // the power of two above sc, at least 2^-60 (stored scales are 0 or above 2^-25)
          const uint32_t e = (__float_as_uint(sc) >> 23) + 1;
          const float new_top = fmaxf(top, __uint_as_float((e < 67 ? 67u : e > 253 ? 253u : e) << 23));
          const float keep = top > 0.f ? top / new_top : 0.f;
          const float r0 = m0 > -INFINITY ? ex2(m0 - n0) : 0.f, r1 = m1 > -INFINITY ? ex2(m1 - n1) : 0.f;
          l0 *= r0;
          l1 *= r1;
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            acc[i][0] *= r0 * keep;
            acc[i][1] *= r1 * keep;
            acc[i][2] *= r0 * keep;
            acc[i][3] *= r1 * keep;
          }
#pragma unroll
          for (int g = 0; g < G; ++g) {
            za[g][0] *= r0 * keep;
            za[g][1] *= r1 * keep;
          }
          m0 = n0;
          m1 = n1;
          top = new_top;
          norm = kNorm / top;
        }
        uint32_t pb[2][G][2];  // P s, heads in rows: the B operand of O^T += V^T P^T
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float p0 = ex2(x[u][0] - m0), p1 = ex2(x[u][1] - m1), p2 = ex2(x[u][2] - m0), p3 = ex2(x[u][3] - m1);
          l0 += p0 + p2;
          l1 += p1 + p3;
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const Kv4Group va = kv4_unpack_params<T>(vp[u][0][g]), vb = kv4_unpack_params<T>(vp[u][1][g]);
            const float sa = va.scale * norm, sb = vb.scale * norm;
            const uint32_t ha = half2_of(p0 * sa, p1 * sa), hb = half2_of(p2 * sb, p3 * sb);
            const float2 ra = __half22float2(*reinterpret_cast<const __half2*>(&ha));
            const float2 rb = __half22float2(*reinterpret_cast<const __half2*>(&hb));
            za[g][0] = fmaf(ra.x, va.zero, fmaf(rb.x, vb.zero, za[g][0]));
            za[g][1] = fmaf(ra.y, va.zero, fmaf(rb.y, vb.zero, za[g][1]));
            pb[u][g][0] = transpose8x8(ha);
            pb[u][g][1] = transpose8x8(hb);
          }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int g = 0; g < G; ++g) {
            uint32_t vw[4][VB / 4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int at = ((k & 1) ? vtok1 : vtok) + 16 * u + 8 * (k >> 1);
              const uint32_t* pv = reinterpret_cast<const uint32_t*>(&st.v[at][g * (GS / 2)]) + r * (VB / 4);
              if constexpr (VB == 8)
                *reinterpret_cast<uint2*>(vw[k]) = *reinterpret_cast<const uint2*>(pv);
              else
                vw[k][0] = *pv;
            }
#pragma unroll
            for (int j = 0; j < VB; ++j) {
              const uint32_t sel = 0x4400u + 0x1111u * (j & 3);  // byte j of both, in bits 0-7 and 16-23
              const uint32_t lo = __byte_perm(vw[0][j / 4], vw[1][j / 4], sel);
              const uint32_t hi = __byte_perm(vw[2][j / 4], vw[3][j / 4], sel);
              const uint32_t f[4] = {(lo << 4) & 0x00f000f0u, lo & 0x00f000f0u, (hi << 4) & 0x00f000f0u, hi & 0x00f000f0u};
              mma16816(acc[g * VB + j], f, pb[u][g][0], pb[u][g][1]);
            }
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.freed[slot]);
    }

    // ------------------------------------------- join the warps of the CTA
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        za[g][0] += __shfl_xor_sync(0xffffffffu, za[g][0], o);
        za[g][1] += __shfl_xor_sync(0xffffffffu, za[g][1], o);
      }
    }
    const float back = top * (1.f / kNorm);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int j = 0; j < VB; ++j) {
        const float* v = acc[g * VB + j];
        const int d = g * GS + r * (GS / 8) + 2 * j;
        const float two20 = 1048576.f;
        *reinterpret_cast<float2*>(&sm.o[warp][2 * c][d]) =
            make_float2((v[0] * two20 - za[g][0]) * back, (v[2] * two20 - za[g][0]) * back);
        *reinterpret_cast<float2*>(&sm.o[warp][2 * c + 1][d]) =
            make_float2((v[1] * two20 - za[g][1]) * back, (v[3] * two20 - za[g][1]) * back);
      }
    if (r == 0) {
      sm.m[warp][2 * c] = m0;
      sm.m[warp][2 * c + 1] = m1;
      sm.l[warp][2 * c] = l0;
      sm.l[warp][2 * c + 1] = l1;
    }
    named_barrier(1, 32 * kWarps);
    const bool whole = p.t0 == 0 && p.t1 == p.tiles;
    // pieces: slot 2 CTA for a row begun in an earlier share, 2 CTA + 1 for one that begins here
    float* piece = a.pieces + (int64_t)(2 * blockIdx.x + (p.row_u0 < share0 ? 0 : 1)) * piece_floats<D>();
    T* out = reinterpret_cast<T*>(a.out) + ((int64_t)p.b * a.hq + h0) * D;
    for (int i = 4 * tid; i < heads * D; i += 4 * 32 * kWarps) {
      const int h = i / D, d = i % D;
      float m = sm.m[0][h], l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) m = fmaxf(m, sm.m[w][h]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp without positions has m = -inf, l = 0 and o = 0; NaN in l or o stays
        const float f = sm.m[w][h] > -INFINITY ? ex2(sm.m[w][h] - m) : 1.f;
        const float4 v = *reinterpret_cast<const float4*>(&sm.o[w][h][d]);
        o.x = fmaf(v.x, f, o.x);
        o.y = fmaf(v.y, f, o.y);
        o.z = fmaf(v.z, f, o.z);
        o.w = fmaf(v.w, f, o.w);
        l = fmaf(sm.l[w][h], f, l);
      }
      if (whole) {
        const float inv = 1.f / l;
        const T y[4] = {Num<T>::from_f(o.x * inv), Num<T>::from_f(o.y * inv), Num<T>::from_f(o.z * inv),
                        Num<T>::from_f(o.w * inv)};
        *reinterpret_cast<uint2*>(out + i) = *reinterpret_cast<const uint2*>(y);
      } else {
        __stcg(reinterpret_cast<float4*>(piece + i), o);
        if (d == 0) {
          __stcg(piece + kHeads * D + h, m);
          __stcg(piece + kHeads * D + kHeads + h, l);
        }
      }
    }
    if (!whole) {
      auto cta_of = [&](int64_t u) { return (int)(((u + 1) * shares - 1) / total); };
      const int first = cta_of(p.row_u0), n = cta_of(p.row_u0 + p.tiles - 1) - first + 1;
      int group = n;  // pieces of a group: up to 16 at once
      if (n > 16)
        for (group = 5; group * group < n;) ++group;
      const int mine = (int)blockIdx.x - first, g = mine / group, groups = (n + group - 1) / group;
      // slot of piece k of the row: begun here (k = 0), or in an earlier share
      auto slot_of = [&](int k) { return 2 * (first + k) + (k == 0 ? 1 : 0); };
      auto arrive_last = [&](int level, int k, int of) {  // the last of `of` CTAs to leave its piece?
        named_barrier(1, 32 * kWarps);
        if (tid == 0) {
          // releases what the CTA's threads wrote before the barrier, acquires what others released
          int* count = a.arrived + level * 2 * gridDim.x + slot_of(k);
          int old;
          asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(count) : "memory");
          sm.last = old == of - 1;
          if (sm.last) *count = 0;
        }
        named_barrier(1, 32 * kWarps);
        return sm.last != 0;
      };
      const int in_group = min(group, n - g * group);
      if (arrive_last(0, g * group, in_group)) {
        if (groups == 1) {
          join<T, D>(a.pieces, slot_of, 0, 1, n, heads, nullptr, out);
        } else {
          join<T, D>(a.pieces, slot_of, g * group, 1, in_group, heads,
                     a.pieces + (int64_t)slot_of(g * group) * piece_floats<D>(), out);
          if (arrive_last(1, 0, groups))
            join<T, D>(a.pieces, slot_of, 0, group, groups, heads, nullptr, out);
        }
      }
    }
    named_barrier(1, 32 * kWarps);  // the joined values are read before the next row's overwrite them
  }
}

// Bytes of the pieces of either head size's grid.
template <int D>
int64_t pieces_of() { return (int64_t)2 * num_sms() * kCtasPerSm<D> * piece_floats<D>() * (int64_t)sizeof(float); }
int64_t pieces_bytes() { return pieces_of<64>() > pieces_of<128>() ? pieces_of<64>() : pieces_of<128>(); }

template <typename T, int D, int GS, bool kRope>
int go_kv4(const Kv4Args& a, cudaStream_t st) {
  constexpr auto kern = kv4_attn_kernel<T, D, GS, kRope>;
  const int rc = allow_smem<kern>("kv4_decode_attention", sizeof(Smem<D, GS>));
  if (rc != TF_OK) return rc;
  return launch_ex("kv4_decode_attention", kern, dim3((unsigned)(num_sms() * kCtasPerSm<D>)), dim3(kThreads), sizeof(Smem<D, GS>), st,
                   dim3(1, 1, 1), a);
}

template <typename T, bool kRope>
int launch_kv4_attention(const Kv4Args& a, int head_dim, int group, cudaStream_t st) {
  if (head_dim == 64) return go_kv4<T, 64, 64, kRope>(a, st);
  if (group == 64) return go_kv4<T, 128, 64, kRope>(a, st);
  return go_kv4<T, 128, 128, kRope>(a, st);
}

// The two entry points' common checks and launch; cos_t: the fused one.
int kv4_attention(const char* what, const void* q, int64_t q_ld, const void* cos_t, const void* sin_t, const Kv4Cache& c,
                  void* out, const int* lens, int64_t B, int hq, int hkv, int head_dim, int group, int64_t t_max,
                  float scale, int dtype, void* workspace, size_t workspace_bytes, cudaStream_t st) {
  const int rc = kv4_check(what, c, B, hkv, head_dim, group, t_max, dtype);
  if (rc != TF_OK) return rc;
  if (hq <= 0 || hq % hkv || B > 65535)
    return fail(TF_ERR_BAD_SHAPE, "%s: bad shape (B=%lld, hq=%d, hkv=%d)", what, (long long)B, hq, hkv);
  if (B == 0) return TF_OK;
  if (!q || !out || !lens) return fail(TF_ERR_BAD_ARG, "%s: null pointer", what);
  if (q_ld % 8 || !aligned(q, 16) || !aligned(out, 16) || !aligned(cos_t, 16) || !aligned(sin_t, 16))
    return fail(TF_ERR_UNALIGNED, "%s: q rows, rotary tables and out must be 16-byte aligned", what);
  if (!(scale > 0.f) || !(scale < INFINITY)) return fail(TF_ERR_BAD_ARG, "%s: scale %g must be positive", what, (double)scale);
  const size_t need = tf_kv4_attention_workspace_bytes();
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(TF_ERR_WORKSPACE, "%s: 16-byte aligned workspace of %zu bytes required", what, need);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int ratio = hq / hkv, blocks = (int)cdiv(ratio, kHeads);
  const Kv4Args a{q, q_ld, cos_t, sin_t, c, out, lens, (int)B, hq, hkv, blocks, (int)cdiv(ratio, blocks), t_max, scale,
                  reinterpret_cast<int*>(ws), reinterpret_cast<float*>(ws + 256),
                  reinterpret_cast<int*>(ws + 256 + pieces_bytes())};
  if (cos_t)
    return dtype == TF_F16 ? launch_kv4_attention<__half, true>(a, head_dim, group, st)
                           : launch_kv4_attention<__nv_bfloat16, true>(a, head_dim, group, st);
  return dtype == TF_F16 ? launch_kv4_attention<__half, false>(a, head_dim, group, st)
                         : launch_kv4_attention<__nv_bfloat16, false>(a, head_dim, group, st);
}

}  // namespace
}  // namespace tf

// Pieces and arrival counters of a fixed number of CTAs: one size for every shape.
extern "C" size_t tf_kv4_attention_workspace_bytes(void) {
  using namespace tf;
  return (size_t)(256 + pieces_bytes() + 4 * (int64_t)num_sms() * kCtasPerSm<64> * sizeof(int));
}

extern "C" int tf_kv4_decode_attention(const void* q, const uint8_t* k_codes, const void* k_params,
                                       const uint8_t* v_codes, const void* v_params, void* out, const int* lens,
                                       int64_t B, int32_t hq, int32_t hkv, int32_t head_dim, int32_t group,
                                       int64_t t_max, float scale, int dtype, void* workspace, size_t workspace_bytes,
                                       void* stream) {
  using namespace tf;
  const Kv4Cache c{(uint8_t*)k_codes, (void*)k_params, (uint8_t*)v_codes, (void*)v_params};
  return kv4_attention("kv4_decode_attention", q, (int64_t)hq * head_dim, nullptr, nullptr, c, out, lens, B, hq, hkv,
                       head_dim, group, t_max, scale, dtype, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream));
}

extern "C" int tf_kv4_decode_attention_rope(const void* qkv, int64_t ld_qkv, const void* cos_table,
                                            const void* sin_table, uint8_t* k_codes, void* k_params, uint8_t* v_codes,
                                            void* v_params, const int* pos, void* out, int64_t B, int32_t hq,
                                            int32_t hkv, int32_t head_dim, int32_t group, int64_t t_max, float scale,
                                            int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tf;
  const Kv4Cache c{k_codes, k_params, v_codes, v_params};
  if (B > 0 && (!cos_table || !sin_table)) return fail(TF_ERR_BAD_ARG, "kv4_decode_attention_rope: null pointer");
  if (ld_qkv < (int64_t)(hq + 2 * (int64_t)hkv) * head_dim)
    return fail(TF_ERR_BAD_SHAPE, "kv4_decode_attention_rope: ld_qkv %lld for %d + 2 x %d heads", (long long)ld_qkv, hq,
                hkv);
  return kv4_attention("kv4_decode_attention_rope", qkv, ld_qkv, cos_table, sin_table, c, out, pos, B, hq, hkv,
                       head_dim, group, t_max, scale, dtype, workspace, workspace_bytes,
                       static_cast<cudaStream_t>(stream));
}
