// Attention over packed prompts: for query i of a sequence with Lq queries and
// Lk keys (its queries are the last Lq of its Lk positions),
//   out[i, h] = sum_j p_ij v_j,  p = softmax_j(scale q_i . k_j),
// over the keys j of the same sequence, with causal masking j <= i + Lk - Lq.
// Query head h reads key head h / (hq / hkv). Scores, softmax and sums are in
// fp32 and the output is rounded once; a query that sees no key gives zeros.
//
// One pass over the keys with a running maximum m and sum l per query (4 D
// flops per query head and visible key: the tensor cores bound it, and the
// exponentials, one per pair at 16 per clock and SM, weigh as much as the two
// products at D = 128 and twice that at D = 64).
//
// Tile: 128 rows = the G = hq / hkv query heads of a kv head x 128 / G tokens,
// so that a tile's rows share keys whatever G is and the causal diagonal wastes
// half a block of 128 keys for 128 / G tokens instead of for 128. A CTA runs
// two tiles (consecutive tokens) over the same key blocks: while the softmax of
// one runs on the CUDA cores, the products of the other run on the tensor
// cores. TMA brings Q once and K, V blocks through a ring; S = Q K^T goes to
// TMEM, four warps per tile (one row per thread) turn it into P in place (16
// bits, over half of the S columns, the product with V starting when three quarters
// are there), and O += P V takes P from TMEM.
// CTAs stay (one per SM) and take pairs of tiles from a counter, those with the
// most keys first; the next pair's Q and keys come while the last one ends. With
// few pairs and long keys some or all pairs are cut into `splits` ranges of key
// blocks that leave (m, l, O) in the workspace; a second kernel joins them in
// order, all SMs at once (joined by the last CTA to arrive they cost 15 us at the
// end).
// m is raised only when a block's maximum passes it by 2^8: until then p is
// relative to an older maximum, which costs no precision in fp32 sums and 16-bit
// floating-point P, and O in TMEM needs no rescaling. The S product of block
// j + 1 follows the P V product of block j in one thread's order, so its
// completion tells that O is at rest.
// P is rounded to the 16-bit type (products of 16-bit operands); l sums the
// unrounded values.
// Masked values are multiplied by p = 0, so one that is not finite turns rows
// that do not see it into NaN. A CTA that meets a non-finite output runs the
// pair (or the range of its keys) once more when its slot is free again, with such
// values replaced by zero in shared memory and the first key of each channel's noted:
// rows that do not see them come out as if they were not there, and in the others
// the channel becomes what the sum is, an infinity or NaN.
//
// In a CUDA graph, 8192 tokens of 64 / 8 heads of 128: 850 us, 79% of the measured
// tensor rate (980 in a run of seconds, under the power cap); 701 queries over 9702
// keys 93 us; 4099 tokens in 11 prompts of 28 / 4 heads 37; 6000 tokens of 14 / 2
// heads of 64 114; 37 tokens of them 8. A pair of tiles takes 3300 to 3500 cycles a
// block for 2048 of products: a tile's own chain (scores to registers and maximum
// 720, powers and P 1500, the last quarter's product and the next S 1000) is what
// is left, TMEM being full; a pair costs 2000 to 4000 cycles more for its first
// block and its output.
#include "f32x2.cuh"
#include "packed.cuh"
#include "tcgen05.cuh"

namespace tf {
namespace {

using namespace tc;

struct PromptArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h, o_t, o_h;  // element strides of tokens and heads
  const int* cu_q;
  const int* cu_k;
  int64_t tq, tk;
  int S, hq, hkv, causal;
  float scale;
  int splits;         // ranges of key blocks that a pair is cut into, if it is
  int max_cut;        // pairs x kv heads that may be cut
  int whole;          // nonzero: as many pairs as make whole rounds of all CTAs are not cut
  int max_pairs;      // pairs per kv head at most
  int* err;
  int* next;          // pairs taken beyond the first of each CTA, and CTAs that are done: zero between launches
  int* cut;           // [0] pairs x kv heads that were cut, [1] those before them; then (sequence, pair) of each
  float* pieces;      // [pairs][splits][2][Piece]
  uint32_t idesc_s, idesc_s_half, idesc_o;  // tcgen05 instruction descriptors of S = Q K^T (128, 64 keys) and of P V
};

// Where one sequence lies: queries [q0, q0 + lq), keys [k0, k0 + lk).
struct Span {
  int q0, lq, k0, lk;
};
__device__ __forceinline__ Span span_of(const PromptArgs& a, int s) {
  const int q0 = (int)packed_offset(a.cu_q, s, a.tq), q1 = (int)packed_offset(a.cu_q, s + 1, a.tq);
  const int k0 = (int)packed_offset(a.cu_k, s, a.tk), k1 = (int)packed_offset(a.cu_k, s + 1, a.tk);
  return {q0, q1 > q0 ? q1 - q0 : 0, k0, k1 > k0 ? k1 - k0 : 0};
}
// Keys that query i of the sequence sees.
__device__ __forceinline__ int keys_seen(const PromptArgs& a, const Span& sp, int i) {
  if (!a.causal) return sp.lk;
  const int n = i + 1 + sp.lk - sp.lq;
  return n < 0 ? 0 : (n > sp.lk ? sp.lk : n);
}

constexpr int kRows = 128;                 // rows of a tile, keys of a block
constexpr int kSoftmaxWarps = 8;           // four per tile
constexpr int kThreads = 32 * (kSoftmaxWarps + 4);  // and a warpgroup of TMA, MMA and two idle warps
// Registers: 384 threads at 168 = 64512 = 256 x 208 + 128 x 88. With 168 for all
// the softmax reads half of its scores twice (8192 tokens: 890 us instead of
// 856), or spills (1100).
constexpr int kRegsSoftmax = 208, kRegsControl = 88;
constexpr float kRaise = 8.f;              // log2 of how far a score may pass the running maximum

// What the CTA works on next: two tiles of `nt` tokens of one sequence and kv
// head, over a range of key blocks.
struct Item {
  Span sp;
  int kh, i0;         // kv head, first query of tile 0 (relative to the sequence)
  int b0, nb[2];      // first key block, blocks of each tile from there
  int split;          // range of `splits`, or -1: all of it
  int index;          // of the pair and kv head, for `pieces`
  int pair;
  int valid, clean;   // clean: non-finite values are replaced by zero
  int dirty;          // met a non-finite output: to be cleaned
};

template <int D>
struct Layout {
  static constexpr int kTile = kRows * D * 2;            // bytes of a Q tile, K block or V block
  static constexpr int kSlots = D == 128 ? 4 : 8;        // K and V blocks in flight
  static constexpr int kRing = 2 * kTile;                // after the two Q tiles
  static constexpr int kOut = kRing + kSlots * kTile;    // a 32 x 64 piece of the output per softmax warp
  static constexpr int kBars = kOut + 8 * 4096;          // barriers, items
  static constexpr int kControl = 1536;
  static constexpr int kBytes = kBars + kControl + 1024;  // + alignment of the base to 1024
  // At D = 64 the lower half of S is made as soon as P's first part is written,
  // for the maximum to start on (6000 tokens, 14 / 2 heads: 130 -> 118 us). At
  // D = 128 S of 64 keys takes as long as of 96 (Q's rows come from shared memory
  // at its full bandwidth either way): 8192 tokens 865 -> 930 us.
  static constexpr bool kLowFirst = D == 64;
  static constexpr int kFirst = 3;  // quarters of P whose product starts first (8192 tokens: 861 us with 2, 853 with 3)
  static constexpr int kPiece = kRows * (D + 2);         // floats of a piece: O [D / 4][128][4], m, l
};

template <int D>
struct Control {
  uint64_t full[Layout<D>::kSlots];   // block landed
  uint64_t freed[Layout<D>::kSlots];  // products done with it
  uint64_t q_full, q_free;            // both Q tiles landed; their products done
  uint64_t s_low[2], s_full[2];       // [tile] S of the next block complete: keys 0-63 (kLowFirst), all
  uint64_t p_full[2][2];              // [tile][half] P written (keys 0-63, 64-127)
  uint64_t o_full[2];                 // [tile] O complete
  uint64_t item_full[2], item_free[2];
  uint64_t idle;                      // every product complete
  uint64_t bad_full;                  // `bad` is of the whole item
  // of the item that is being cleaned: first key of each channel whose value is +inf or NaN, -inf or NaN
  int bad[2][D];
  Item item[2];
  int abort;
  uint32_t tmem;
};

// Second pass: a warp replaces the values of a V block in shared memory that
// are not finite by zero, before the tensor cores read it, and notes the first
// key of the sequence (key0: the block's first) of each channel's. (Not inlined:
// without its code the loop of products is 0.7% faster.)
template <typename T, int D>
__device__ __noinline__ void clean_block(uint8_t* block, int key0, int lk, int (*bad)[D]) {
  constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u;
  uint4* v = reinterpret_cast<uint4*>(block);
#pragma unroll 1
  for (int i = threadIdx.x & 31; i < kRows * D / 8; i += 32) {
    const uint4 x = v[i];
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
    bool any = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) any |= ((w[e / 2] >> (16 * (e & 1))) & kExp) == kExp;
    if (!any) continue;
    // 64 channels (128 bytes, their 16-byte units swizzled) per key and half
    const int in = (i / 8) % kRows, key = key0 + in, d0 = i / (8 * kRows) * 64 + ((i ^ in) & 7) * 8;
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = (w[0] >> (16 * (e & 1))) & 0xffffu;
      if ((h & kExp) == kExp) {
        w[0] &= (e & 1) ? 0x0000ffffu : 0xffff0000u;
        const bool nan = (h & 0x7fffu) != kExp;
        if (key < lk && (nan || h == kExp)) atomicMin(&bad[0][d0 + e], key);
        if (key < lk && (nan || h != kExp)) atomicMin(&bad[1][d0 + e], key);
      }
      if (e & 1) {  // the next word to the front
        const uint32_t done = w[0];
        w[0] = w[1];
        w[1] = w[2];
        w[2] = w[3];
        w[3] = done;
      }
    }
    v[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
}

// 32 columns of this warp's 32 lanes (one lane per thread): the load, and the
// wait after which the registers may be used.
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      :
      "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld32(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               :
      "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
        "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
        "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
        "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]),
        "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The MMA warp issues in step, one lane by predicate: without a branch around
// them the operands stay in uniform registers, and a 128 x 128 x 16 product
// leaves only 64 cycles to issue the next.
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r;
}
// Descriptors: the upper words are one constant (128-byte swizzle, atoms of 8
// rows 1 KiB apart), the lower ones address and leading offset.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) { return (saddr >> 4) | ((lbo >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " mov.b64 da, {%1, %6};\n mov.b64 db, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n"
      " mov.b64 db, {%2, %6};\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint32_t leader, uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.b32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(smem_u32(bar)),
      "r"(leader)
      : "memory");
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Names the pairs of all sequences by one index, longest first (a pair's level:
// the number of its last keys in steps of a pair's queries); a warp's work, each
// lane a sequence. With more than 32 sequences: the pairs in order, the last one
// first.
struct Pairs {
  int total, level, before;  // pairs; present level, pairs above it
  int n, low, width;         // of this lane's sequence: pairs, level of the first; queries of a pair
  Span mine;                 // this lane's sequence
  __device__ __forceinline__ int of(const PromptArgs& a, int s) const {
    return s < a.S ? (span_of(a, s).lq + width - 1) / width : 0;
  }
  __device__ __forceinline__ void init(const PromptArgs& a, int queries) {
    const int lane = threadIdx.x & 31;
    width = queries;
    mine = lane < a.S ? span_of(a, lane) : Span{0, 0, 0, 0};
    n = (mine.lq + width - 1) / width;
    low = mine.lk > mine.lq ? (mine.lk - mine.lq) / width : 0;
    level = INT32_MAX;
    before = 0;
    total = 0;
    for (int s0 = 0; s0 < a.S; s0 += 32)
      total += (int)__reduce_add_sync(0xffffffffu, (unsigned)(s0 ? of(a, s0 + lane) : n));
    total = total < a.max_pairs ? total : a.max_pairs;
  }
  // index < total, not below an earlier one
  __device__ __forceinline__ void find(const PromptArgs& a, int index, int& seq, int& pair) {
    const int lane = threadIdx.x & 31;
    if (a.S <= 32) {
      for (;; --level) {  // (down to the next level that has a pair: there is one, index < total)
        level = __reduce_max_sync(0xffffffffu, n > 0 && low <= level ? min(level, low + n - 1) : 0);
        const unsigned here = __ballot_sync(0xffffffffu, low <= level && level < low + n);
        if (index < before + __popc(here)) {
          const bool it = (here >> lane & 1u) && __popc(here & ((1u << lane) - 1)) == index - before;
          seq = __ffs(__ballot_sync(0xffffffffu, it)) - 1;
          pair = level - __shfl_sync(0xffffffffu, low, seq);
          return;
        }
        before += __popc(here);
      }
    }
    // (more than a warp of sequences)
    const int want = total - 1 - index;
    int sum0 = 0;
    for (int s0 = 0;; s0 += 32) {
      const int m = of(a, s0 + lane);
      int sum = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const unsigned who = __ballot_sync(0xffffffffu, sum0 + sum > want);
      if (who) {
        const int src = __ffs(who) - 1;
        seq = s0 + src;
        pair = want - sum0 - __shfl_sync(0xffffffffu, sum - m, src);
        return;
      }
      sum0 += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    prompt_attn_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                       const __grid_constant__ CUtensorMap vmap, const PromptArgs a) {
  using L = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  Control<D>& ct = *reinterpret_cast<Control<D>*>(smem + L::kBars);
  static_assert(sizeof(Control<D>) <= L::kControl, "control block");
  volatile int* abort_flag = &ct.abort;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.hkv, nt = kRows / G;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kSlots; ++i) {
      mbar_init(&ct.full[i], 1);
      mbar_init(&ct.freed[i], 1);
    }
    mbar_init(&ct.q_full, 1);
    mbar_init(&ct.q_free, 1);
    for (int w = 0; w < 2; ++w) {
      mbar_init(&ct.s_low[w], 1);
      mbar_init(&ct.s_full[w], 1);
      mbar_init(&ct.p_full[w][0], 4);
      mbar_init(&ct.p_full[w][1], 4);
      mbar_init(&ct.o_full[w], 1);
      mbar_init(&ct.item_full[w], 1);
      mbar_init(&ct.item_free[w], kSoftmaxWarps + 1);
    }
    mbar_init(&ct.idle, 1);
    mbar_init(&ct.bad_full, 1);
    ct.abort = 0;
    fence_mbarrier_init();
  }
  // Q rows past G x nt, which no copy writes: zeros, whose scores never raise a maximum
  for (int e = threadIdx.x; e < 2 * (D / 64) * (kRows - G * nt) * 8; e += kThreads) {
    const int r = G * nt + (e / 8) % (kRows - G * nt), part = e / 8 / (kRows - G * nt);
    *reinterpret_cast<uint4*>(smem + part * (kRows * 128) + r * 128 + (e % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  pdl_wait();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&ct.tmem))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem = ct.tmem;
  // a wait that every lane of the warp makes; false (and the CTA ends) when it gives up
  auto wait = [&](uint64_t* bar, uint32_t parity, int bit) {
    const bool ok = __all_sync(0xffffffffu, !*abort_flag && mbar_wait_bounded(bar, parity & 1u, a.err, bit));
    if (!ok) *abort_flag = 1;
    return ok;
  };

  // the same where the phase is mostly complete already
  auto ready = [&](uint64_t* bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity & 1u))) return true;
    return wait(bar, parity, 2);
  };

  // (a warpgroup's warps execute the same setmaxnreg)
  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (warp == kSoftmaxWarps) {
      // ------------------------------------------------- pairs and their loads
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
      }
      Pairs pairs;
      pairs.init(a, 2 * nt);
      const int heads = pairs.total * a.hkv;  // pairs x kv heads, the first `uncut` of them not cut
      const int rounds = a.whole ? heads / (int)gridDim.x * (int)gridDim.x : 0;
      const int uncut = a.splits == 1 ? heads : max(rounds, heads - a.max_cut);
      const int items = uncut + (heads - uncut) * a.splits;
      int n_items = 0, n_q = 0, it = 0;
      bool ok = true;
      // into the next slot, which is free
      auto put = [&](const Span& sp, int pair, int kh, int split, int index, int clean) {
        const int slot = n_items & 1;
        Item t;
        t.sp = sp;
        t.kh = kh;
        t.i0 = pair * 2 * nt;
        int nb = 0;
        for (int w = 0; w < 2; ++w) {  // key blocks that the tile's last query needs
          const int i = t.i0 + w * nt, last = i + nt - 1 < t.sp.lq ? i + nt - 1 : t.sp.lq - 1;
          t.nb[w] = i < t.sp.lq ? (keys_seen(a, t.sp, last) + kRows - 1) / kRows : 0;
          nb = t.nb[w] > nb ? t.nb[w] : nb;
        }
        t.b0 = 0;
        if (split >= 0) {
          t.b0 = (int)((int64_t)nb * split / a.splits);
          const int end = (int)((int64_t)nb * (split + 1) / a.splits);
          nb = end - t.b0;
          for (int w = 0; w < 2; ++w) {
            const int e = t.nb[w] < end ? t.nb[w] : end;
            t.nb[w] = e > t.b0 ? e - t.b0 : 0;
          }
          nb = t.nb[1] > t.nb[0] ? t.nb[1] : t.nb[0];
        }
        t.split = split;
        t.index = index;
        t.pair = pair;
        t.valid = 1;
        t.clean = clean;
        t.dirty = 0;
        if (lane == 0) {
          ct.item[slot] = t;
          mbar_arrive(&ct.item_full[slot]);
        }
        ++n_items;
        if (nb == 0) return;
        if (n_q > 0) ok = wait(&ct.q_free, (uint32_t)(n_q - 1), 1);
        if (!ok) return;
        ++n_q;
        if (lane == 0) {
          mbar_arrive_expect_tx(&ct.q_full, (uint32_t)(2 * G * nt * D * 2));
          for (int w = 0; w < 2; ++w)
            for (int half = 0; half < D / 64; ++half)
              tma_load_3d(smem + w * L::kTile + half * (kRows * 128), &qmap, &ct.q_full, 64 * half, kh * G,
                          t.sp.q0 + t.i0 + w * nt);
          for (int j = 0; j < 2 * nb; ++j, ++it) {  // K0, V0, K1, V1, ...
            const int s = it % L::kSlots;
            if (*abort_flag || (it >= L::kSlots &&
                                !mbar_wait_bounded(&ct.freed[s], (uint32_t)(it / L::kSlots - 1) & 1u, a.err, 1))) {
              *abort_flag = 1;
              break;
            }
            mbar_arrive_expect_tx(&ct.full[s], (uint32_t)L::kTile);
            for (int half = 0; half < D / 64; ++half)
              tma_load_3d(smem + L::kRing + s * L::kTile + half * (kRows * 128), (j & 1) ? &vmap : &kmap, &ct.full[s],
                          64 * half, kh, t.sp.k0 + (t.b0 + (j >> 1)) * kRows);
          }
        }
        __syncwarp();
        ok = !*abort_flag;
      };
      // waits for item i: true if it met a non-finite output and is to be run again
      auto dirty = [&](int i) {
        ok = ok && wait(&ct.item_free[i & 1], (uint32_t)(i / 2), 1);
        return ok && __shfl_sync(0xffffffffu, *(volatile int*)&ct.item[i & 1].dirty, 0) != 0;
      };
      Span sp;  // of pair `id`, looked up while the items before it are at work
      int seq = -1, pair = 0;
      for (int id = blockIdx.x, next = 0;;) {
        const bool more = id < items;
        const int range = id < uncut ? -1 : (id - uncut) % a.splits;
        const int g = id < uncut ? id : uncut + (id - uncut) / a.splits;
        if (more && seq < 0) {
          if (lane == 0) next = atomicAdd(a.next, 1);
          pairs.find(a, g / a.hkv, seq, pair);
          if (a.S <= 32) {
            sp = {__shfl_sync(0xffffffffu, pairs.mine.q0, seq), __shfl_sync(0xffffffffu, pairs.mine.lq, seq),
                  __shfl_sync(0xffffffffu, pairs.mine.k0, seq), __shfl_sync(0xffffffffu, pairs.mine.lk, seq)};
          } else {
            sp = span_of(a, seq);
          }
        }
        // the item that held the next slot; at the end the one in the other slot too
        int old = n_items - 2;
        bool again = old >= 0 && dirty(old);
        if (!more && !again && n_items > 0) again = dirty(old = n_items - 1);
        if (!ok || !(more || again)) break;
        if (again) {
          Item& was = ct.item[old & 1];
          const Span was_sp = was.sp;
          const int was_pair = was.pair, was_kh = was.kh, was_split = was.split, was_index = was.index;
          __syncwarp();
          if (lane == 0) was.dirty = 0;
          put(was_sp, was_pair, was_kh, was_split, was_index, 1);
        } else {
          if (range == 0 && lane == 0) {  // for the kernel that joins the ranges
            a.cut[2 + 2 * (g - uncut)] = seq;
            a.cut[3 + 2 * (g - uncut)] = pair;
          }
          put(sp, pair, g % a.hkv, range, g - uncut, 0);
          id = (int)gridDim.x + __shfl_sync(0xffffffffu, next, 0);
          seq = -1;
        }
      }
      if (lane == 0) {
        if (ok) {  // no more
          ct.item[n_items & 1].valid = 0;
          mbar_arrive(&ct.item_full[n_items & 1]);
        }
        if (blockIdx.x == 0) {
          a.cut[0] = heads - uncut;
          a.cut[1] = uncut;
        }
        if (atomicAdd(a.next + 1, 1) == (int)gridDim.x - 1) {  // the last CTA to take a pair: nobody counts any more
          a.next[0] = 0;
          a.next[1] = 0;
        }
      }
      if (lane == 0) {
        if (*abort_flag) {  // the copies in flight land before the CTA exits
          if (n_q > 0) mbar_wait_bounded(&ct.q_full, (uint32_t)(n_q - 1) & 1u, a.err, 4);
          for (int i = (it > L::kSlots ? it - L::kSlots : 0); i < it; ++i)
            mbar_wait_bounded(&ct.full[i % L::kSlots], (uint32_t)(i / L::kSlots) & 1u, a.err, 4);
        }
      }
    } else if (warp == kSoftmaxWarps + 1) {
      // ---------------------------------------------------------------- MMA
      const uint32_t leader = elect_one();
      const uint32_t base = __shfl_sync(0xffffffffu, smem_u32(smem), 0), tm = __shfl_sync(0xffffffffu, tmem, 0);
      int n_items = 0, n_q = 0, slot = 0;  // slot: of the ring, the next block's
      uint32_t slot_phase = 0;             // its parity
      uint32_t done[2] = {0, 0};           // blocks of each tile so far
      for (bool ok = true; ok; ++n_items) {
        ok = ready(&ct.item_full[n_items & 1], (uint32_t)(n_items / 2));
        if (!ok) break;
        Item& item = ct.item[n_items & 1];
        if (!__shfl_sync(0xffffffffu, item.valid, 0)) break;
        const int n0 = __shfl_sync(0xffffffffu, item.nb[0], 0), n1 = __shfl_sync(0xffffffffu, item.nb[1], 0);
        const int nb = n1 > n0 ? n1 : n0;
        const int clean = __shfl_sync(0xffffffffu, item.clean, 0);
        if (nb > 0) {
          auto next_slot = [&]() {
            if (++slot == L::kSlots) {
              slot = 0;
              slot_phase ^= 1u;
            }
          };
          auto ring = [&](int i) { return base + L::kRing + (uint32_t)i * L::kTile; };
          // S = Q K_j^T over n keys from `key` on (rows of 128 B)
          auto s_product = [&](int tile, int key, int n, int k_slot, uint64_t* bar) {
            const uint32_t qa = desc_low(base + tile * L::kTile, 16), ka = desc_low(ring(k_slot) + key * 128, 16);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t off = ((uint32_t)(ks / 4) * (kRows * 128) + (uint32_t)(ks % 4) * 32) >> 4;
              mma_ss(leader, tm + tile * 128 + key, qa + off, ka + off, n == kRows ? a.idesc_s : a.idesc_s_half,
                     ks > 0 ? 1u : 0u);
            }
            commit_if(leader, bar);
          };
          // O (+)= P V_j over the keys [16 k0, 16 k1) of the block; V: 64 channels x 8
          // keys atoms, 1 KiB per 8 keys
          auto o_product = [&](int tile, bool first, int k0, int k1, int v_slot) {
            const uint32_t va = desc_low(ring(v_slot), kRows * 128), pa = tm + tile * 128 + 64;
#pragma unroll
            for (int k = k0; k < k1; ++k)
              mma_ts(leader, tm + 256 + tile * D, pa + k * 8, va + k * (2048 >> 4), a.idesc_o, (k > k0 || !first) ? 1u : 0u);
          };
          if (clean) {  // what `bad` holds is read until the item before is done
            ok = wait(&ct.item_free[(n_items - 1) & 1], (uint32_t)((n_items - 1) / 2), 2);
            for (int e = lane; e < 2 * D; e += 32) (&ct.bad[0][0])[e] = INT32_MAX;
            __syncwarp();
          }
          ok = ok && ready(&ct.q_full, (uint32_t)n_q) && ready(&ct.full[slot], slot_phase);
          ++n_q;
          if (ok) {
            tc_fence_after();
            if constexpr (L::kLowFirst) {
              if (n0 > 0) s_product(0, 0, 64, slot, &ct.s_low[0]);
              if (n1 > 0) s_product(1, 0, 64, slot, &ct.s_low[1]);
              if (n0 > 0) s_product(0, 64, 64, slot, &ct.s_full[0]);
              if (n1 > 0) s_product(1, 64, 64, slot, &ct.s_full[1]);
            } else {
              if (n0 > 0) s_product(0, 0, kRows, slot, &ct.s_full[0]);
              if (n1 > 0) s_product(1, 0, kRows, slot, &ct.s_full[1]);
            }
            commit_if(leader, &ct.freed[slot]);
            if (nb == 1) commit_if(leader, &ct.q_free);
            next_slot();
          }
          for (int j = 0; ok && j < nb; ++j) {
            const int v_slot = slot;
            ok = ready(&ct.full[slot], slot_phase);
            next_slot();
            const int k_slot = slot;
            if (ok && j + 1 < nb) {
              ok = ready(&ct.full[slot], slot_phase);
              next_slot();
            }
            if (ok && clean) {
              clean_block<T, D>(smem + L::kRing + v_slot * L::kTile, (item.b0 + j) * kRows, item.sp.lk, ct.bad);
              if (j + 1 == nb && lane == 0) mbar_arrive(&ct.bad_full);
            }
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
              const int n = tile ? n1 : n0;
              if (!ok || j >= n) continue;
              const uint32_t phase = done[tile] + j;
              ok = ready(&ct.p_full[tile][1], phase);
              if (!ok) continue;
              tc_fence_after();
              o_product(tile, j == 0, 8 - 2 * L::kFirst, 8, v_slot);
              // every score of block j is in registers by now
              if (L::kLowFirst && j + 1 < n) s_product(tile, 0, 64, k_slot, &ct.s_low[tile]);
              ok = ready(&ct.p_full[tile][0], phase);
              if (!ok) continue;
              tc_fence_after();
              o_product(tile, false, 0, 8 - 2 * L::kFirst, v_slot);
              if (j + 1 < n) s_product(tile, L::kLowFirst ? 64 : 0, L::kLowFirst ? 64 : kRows, k_slot, &ct.s_full[tile]);
              else commit_if(leader, &ct.o_full[tile]);
            }
            if (!ok) break;
            commit_if(leader, &ct.freed[v_slot]);
            if (j + 1 < nb) commit_if(leader, &ct.freed[k_slot]);
            if (j + 2 == nb) commit_if(leader, &ct.q_free);
          }
          done[0] += n0;
          done[1] += n1;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ct.item_free[n_items & 1]);
      }
      commit_if(leader, &ct.idle);  // this warp goes on only after its last product
      mbar_wait_bounded(&ct.idle, 0u, a.err, 8);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    // ------------------------------------------------------------ softmax
    const int tile = warp >> 2, row = (warp & 3) * 32 + lane;
    const int row_i = row / G, row_h = row % G;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + tile * 128, o_addr = tmem + lanes + 256 + tile * D;
    const float c = a.scale * 1.4426950408889634f;
    uint32_t done = 0, n_o = 0, n_clean = 0;  // blocks, O products and cleaned items so far
    bool ok = true;
    for (int n_items = 0; ok; ++n_items) {
      ok = wait(&ct.item_full[n_items & 1], (uint32_t)(n_items / 2), 2);
      if (!ok) break;
      Item& item = ct.item[n_items & 1];
      if (!item.valid) break;
      const Span sp = item.sp;
      const int i = item.i0 + tile * nt + row_i, h = item.kh * G + row_h;
      const bool real = row < G * nt && i < sp.lq;
      const int key0 = item.b0 * kRows;
      const int n = real ? keys_seen(a, sp, i) : 0;           // keys this row sees, in all
      const int n_first = item.i0 + tile * nt < sp.lq ? keys_seen(a, sp, item.i0 + tile * nt) : 0;
      const int n_blocks = item.nb[tile];
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_blocks; ++j) {
        ok = ready(L::kLowFirst ? &ct.s_low[tile] : &ct.s_full[tile], done + j);
        if (!ok) break;
        tc_fence_after();
        const bool edge = key0 + (j + 1) * kRows > n_first;  // some row does not see all of the block
        const int lim = n - key0 - j * kRows;
        // The row's 128 scores stay in registers from the maximum to P.
        uint32_t x[4][32];
        float mx0 = -INFINITY, mx1 = -INFINITY;
        auto take_max = [&](int q) {
          if (edge) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (32 * q + e >= lim) x[q][e] = 0xff800000u;  // -inf
          }
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            mx0 = fmaxf(mx0, __uint_as_float(x[q][e]));
            mx1 = fmaxf(mx1, __uint_as_float(x[q][e + 1]));
          }
        };
        tmem_ld32_issue(s_addr, x[0]);
        tmem_ld32_issue(s_addr + 32, x[1]);
        tmem_wait_ld32(x[0]);
        tmem_wait_ld32(x[1]);
        if constexpr (L::kLowFirst) {
          take_max(0);
          take_max(1);
          ok = ready(&ct.s_full[tile], done + j);
          if (!ok) break;
          tc_fence_after();
        }
        tmem_ld32_issue(s_addr + 64, x[2]);
        tmem_ld32_issue(s_addr + 96, x[3]);
        if constexpr (!L::kLowFirst) {
          take_max(0);
          take_max(1);
        }
        tmem_wait_ld32(x[2]);
        tmem_wait_ld32(x[3]);
        take_max(2);
        take_max(3);
        const float mx = fmaxf(mx0, mx1);
        // raise the running maximum (and rescale O) only when this block passes it by far
        const bool raise = mx > m && (mx - m) * c > kRaise;
        if (__any_sync(0xffffffffu, raise)) {
          const float f = raise && m > -INFINITY ? ex2((m - mx) * c) : (raise ? 0.f : 1.f);
          if (raise) m = mx;
          l *= f;
          if (j > 0) {
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += 16) {
              uint32_t o[16];
              tmem_ld16(o_addr + d0, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(o_addr + d0, o);
            }
          }
        }
        const float mc = m > -INFINITY ? m * c : 0.f;
        const uint64_t c2 = pair(c, c), mc2 = pair(-mc, -mc);
        uint64_t l2a = 0, l2b = 0;  // (0, 0)
        auto powers = [&](int q) {  // 32 scores -> 16 words of P, over the upper columns of S
          uint32_t p[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float t0, t1;
            unpair(fma2(pair(__uint_as_float(x[q][e]), __uint_as_float(x[q][e + 1])), c2, mc2), t0, t1);
            const float p0 = ex2(t0), p1 = ex2(t1);
            if (e & 2) l2a = add2(l2a, pair(p0, p1));
            else l2b = add2(l2b, pair(p0, p1));
            p[e / 2] = pack2<T>(p0, p1);
          }
          tmem_st16(s_addr + 64 + 16 * q, p);
        };
        auto half_done = [&](int half) {
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ct.p_full[tile][half]);
        };
#pragma unroll
        for (int q = 4 - L::kFirst; q < 4; ++q) powers(q);
        half_done(1);
#pragma unroll
        for (int q = 0; q < 4 - L::kFirst; ++q) powers(q);
        half_done(0);
        {
          float a0, a1, b0, b1;
          unpair(l2a, a0, a1);
          unpair(l2b, b0, b1);
          l += (a0 + a1) + (b0 + b1);
        }
      }
      if (!ok) break;
      done += n_blocks;
      if (n_blocks > 0) {
        ok = wait(&ct.o_full[tile], n_o, 2);
        if (!ok) break;
        ++n_o;
      }
      if (item.clean) {
        ok = wait(&ct.bad_full, n_clean, 2);
        if (!ok) break;
        ++n_clean;
      }
      tc_fence_after();
      // of a cleaned item: what channel d of this row's sum is, where the row sees a value that is not finite
      auto patch = [&](auto&& store) {
        for (int d = 0; d < D; ++d) {
          const bool up = n > ct.bad[0][d], down = n > ct.bad[1][d];
          if (up || down) store(d, up && down ? NAN : up ? INFINITY : -INFINITY);
        }
      };
      bool finite = true;
      if (item.split < 0) {
        // Through shared memory, 64 channels at a time: a warp's stores then cover
        // four rows' 128 bytes each, where 16 bytes of 32 rows take eight times
        // the cycles (3600 a tile).
        uint8_t* stage = smem + L::kOut + warp * 4096;  // [32 rows][8 units of 16 bytes, unit ^ row % 8]
        const float inv = n > 0 ? 1.f / l : 0.f;        // (a row that sees no key has zeros in O)
        const uint64_t inv2 = pair(inv, inv);
        const int64_t mine = real ? (int64_t)(sp.q0 + i) * a.o_t + (int64_t)h * a.o_h : -1;
        int64_t at[8];  // where the rows that this lane stores a unit of go
#pragma unroll
        for (int r = 0; r < 8; ++r) at[r] = __shfl_sync(0xffffffffu, mine, 4 * r + lane / 8);
        uint64_t check2[2] = {0, 0};  // NaN when an output is not finite
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 64) {
          uint32_t o[2][32];
          if (n_blocks > 0) {
            tmem_ld32_issue(o_addr + d0, o[0]);
            tmem_ld32_issue(o_addr + d0 + 32, o[1]);
            tmem_wait_ld32(o[0]);
            tmem_wait_ld32(o[1]);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[0][e] = o[1][e] = 0u;
          }
#pragma unroll
          for (int u = 0; u < 8; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t* y = &o[u / 4][8 * (u & 3) + 2 * e];
              const uint64_t x = mul2(pair(__uint_as_float(y[0]), __uint_as_float(y[1])), inv2);
              check2[e & 1] = fma2(x, 0ull, check2[e & 1]);
              float x0, x1;
              unpair(x, x0, x1);
              w[e] = pack2<T>(x0, x1);
            }
            *reinterpret_cast<uint4*>(stage + lane * 128 + (u ^ (lane & 7)) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int rr = 4 * r + lane / 8, unit = lane & 7;
            const uint4 x = *reinterpret_cast<const uint4*>(stage + rr * 128 + (unit ^ (rr & 7)) * 16);
            if (at[r] >= 0) *reinterpret_cast<uint4*>((T*)a.out + at[r] + d0 + 8 * unit) = x;
          }
          __syncwarp();
        }
        float c0, c1, c2, c3;
        unpair(check2[0], c0, c1);
        unpair(check2[1], c2, c3);
        const float check = (c0 + c1) + (c2 + c3);
        finite = check == check;
        if (item.clean && real)
          patch([&](int d, float x) { ((T*)a.out)[mine + d] = Num<T>::from_f(l > 0.f ? x : NAN); });
      } else {
        float* piece = a.pieces + (((int64_t)item.index * a.splits + item.split) * 2 + tile) * L::kPiece;
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 16) {
          uint32_t o[16];
          if (n_blocks > 0) {
            tmem_ld16(o_addr + d0, o);
          } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = 0u;
          }
          float check = 0.f;  // NaN when a sum is not finite
#pragma unroll
          for (int e = 0; e < 16; ++e) check = fmaf(__uint_as_float(o[e]), 0.f, check);
          finite = finite && check == check;
          if (real)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              __stcg(reinterpret_cast<uint4*>(piece) + (d0 + e) / 4 * kRows + row,
                     make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]));
          __syncwarp();
        }
        if (real) {
          __stcg(piece + D * kRows + row, m);
          __stcg(piece + (D + 1) * kRows + row, l);
          if (item.clean) patch([&](int d, float x) { __stcg(piece + (d / 4 * kRows + row) * 4 + d % 4, x); });
        }
      }
      if (!item.clean && __any_sync(0xffffffffu, real && !finite) && lane == 0) *(volatile int*)&item.dirty = 1;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ct.item_free[n_items & 1]);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Joins the pieces of one tile's ranges, in order: a CTA per (pair, kv head,
// tile), 16 channels of a row per thread and step.
constexpr int kJoinThreads = 256, kMaxSplits = 32;
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) prompt_join_kernel(const PromptArgs a) {
  constexpr int64_t kStep = 2 * Layout<D>::kPiece;
  __shared__ float weight[kMaxSplits][kRows];
  pdl_trigger();
  pdl_wait();
  const int index = (int)(blockIdx.x >> 1), tile = (int)(blockIdx.x & 1);
  if (index >= a.cut[0]) return;
  const int G = a.hq / a.hkv, nt = kRows / G, kh = (a.cut[1] + index) % a.hkv;
  const Span sp = span_of(a, a.cut[2 + 2 * index]);
  const int i0 = (2 * a.cut[3 + 2 * index] + tile) * nt, rows = min(G * nt, (sp.lq - i0) * G);
  if (rows <= 0) return;
  const float* first = a.pieces + ((int64_t)index * a.splits * 2 + tile) * Layout<D>::kPiece;
  const float c = a.scale * 1.4426950408889634f;
  if ((int)threadIdx.x < rows) {
    const int r = threadIdx.x;
    const float* ms = first + D * kRows + r;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      weight[k][r] = ms[k * kStep];
      top = fmaxf(top, weight[k][r]);
    }
#pragma unroll 4
    for (int k = 0; k < a.splits; ++k) {
      const float mk = weight[k][r], f = mk > -INFINITY ? ex2((mk - top) * c) : 1.f;
      sum += ms[k * kStep + kRows] * f;
      weight[k][r] = f;
    }
    const float inv = keys_seen(a, sp, i0 + r / G) > 0 ? 1.f / sum : 0.f;
    for (int k = 0; k < a.splits; ++k) weight[k][r] *= inv;
  }
  __syncthreads();
  for (int u = threadIdx.x; u < rows * (D / 16); u += kJoinThreads) {
    const int r = u % rows, col = u / rows;
    float4 x[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) x[y] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 3
    for (int k = 0; k < a.splits; ++k) {
      const float f = weight[k][r];
      const float4* q = reinterpret_cast<const float4*>(first + k * kStep) + r;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const float4 v = q[(4 * col + y) * kRows];
        x[y].x = fmaf(v.x, f, x[y].x);
        x[y].y = fmaf(v.y, f, x[y].y);
        x[y].z = fmaf(v.z, f, x[y].z);
        x[y].w = fmaf(v.w, f, x[y].w);
      }
    }
    uint32_t w[8];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      w[2 * y] = pack2<T>(x[y].x, x[y].y);
      w[2 * y + 1] = pack2<T>(x[y].z, x[y].w);
    }
    uint4* o = reinterpret_cast<uint4*>((T*)a.out + (int64_t)(sp.q0 + i0 + r / G) * a.o_t + (int64_t)(kh * G + r % G) * a.o_h +
                                        16 * col);
    o[0] = make_uint4(w[0], w[1], w[2], w[3]);
    o[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

constexpr size_t kFixedBytes = 8192;  // error word, counters, the table of pairs that were cut
constexpr int64_t kCutWords = (int64_t)(kFixedBytes - 256) / 4;

// How a problem is cut: pairs of tiles per kv head (at most) and ranges of key
// blocks per pair. A pair's CTA holds an SM, so with few pairs per SM the time
// is that of the SM that takes one more than the others, or of the longest pair.
// Of these cuts the one is taken for which a count in units of a block's time is
// least: no pair; every pair; where the pairs are about as long as each other,
// those beyond whole rounds of all SMs. Ranges are of equal length, four blocks
// or more; one costs about 2 blocks on top of its own and the join 3, and more
// with more ranges. 701 queries over 9702 keys, 192 pairs: 106 us with every pair
// in two, 124 in three, 96 with the last 44 in three (600
// over 20600, 152 pairs: 408 us in two, 359 with the last four in 25).
struct Plan {
  int64_t pairs, cut;  // per kv head; pairs x kv heads that may be cut
  int splits, whole;
  size_t bytes;
};
Plan plan_of(int64_t tq, int64_t tk, int S, int hq, int hkv, int head_dim) {
  constexpr float kRange = 2.f;
  const int nt = kRows / (hq / hkv);
  // sum of ceil(lq / (2 nt)) at most
  Plan p{S == 1 ? cdiv(tq, 2 * nt) : tq / (2 * nt) + (S < tq ? S : tq), 0, 1, 0, kFixedBytes};
  const int64_t base = p.pairs * hkv, sms = num_sms(), rest = base % sms;
  if (base <= 0 || S <= 0) return p;
  const bool alike = tk >= 2 * tq;  // or from nothing to all keys, the longest first
  const float longest = (float)tk / (float)S / kRows;
  const float mean = tk > tq ? longest - (float)tq / (float)(2 * S * (int64_t)kRows) : longest / 2.f;
  auto uneven = [&](int s) {  // every pair in s ranges, the longest first
    const float all = (float)base * (mean + kRange * (float)s) / (float)sms, one = longest / (float)s + kRange;
    return all > one ? all : one;
  };
  float best = alike ? (float)cdiv(base, sms) * (mean + kRange) : uneven(1);
  for (int s = 2; s <= kMaxSplits && (float)(4 * s) <= longest; ++s) {
    const float join = 3.f + 0.25f * (float)s;
    auto take = [&](float time, int64_t cut, int whole) {
      if (time >= best || 2 + 2 * cut > kCutWords) return;
      best = time;
      p.splits = s;
      p.cut = cut;
      p.whole = whole;
    };
    const float range = mean / (float)s + kRange;
    if (alike) {
      take(join + (float)cdiv(base * s, sms) * range, base, 0);
      if (rest < base)
        take(join + (float)(base / sms) * (mean + kRange) + (float)cdiv(rest * s, sms) * range,
             2 * rest < sms ? 2 * rest : sms, 1);  // (the pairs may be fewer than counted here)
    } else {
      take(join + uneven(s), base, 0);
    }
  }
  if (p.splits > 1) p.bytes += (size_t)(p.cut * p.splits * 2 * kRows * (head_dim + 2)) * sizeof(float);
  return p;
}

template <typename T, int D>
int launch_prompt(const PromptArgs& args, size_t workspace_bytes, cudaStream_t st) {
  using L = Layout<D>;
  PromptArgs a = args;
  const int G = a.hq / a.hkv, nt = kRows / G;
  const CUtensorMapDataType ty =
      std::is_same_v<T, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const uint32_t ab = std::is_same_v<T, __half> ? 0u : 1u;
  // fp32 accumulators, both operands 16-bit, N >> 3 and M >> 4; B of the second product is N-major
  a.idesc_s_half = (1u << 4) | (ab << 7) | (ab << 10) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  a.idesc_s = (1u << 4) | (ab << 7) | (ab << 10) | ((uint32_t)(kRows >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);
  a.idesc_o = (1u << 4) | (ab << 7) | (ab << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
              ((uint32_t)(kRows >> 4) << 24);
  CUtensorMap qm, km, vm;
  // (channel, head, token); an axis of one element may have any stride: give it the row's
  auto map = [&](CUtensorMap* m, const void* p, int64_t heads, int64_t tokens, int64_t sh, int64_t st_, uint32_t bh,
                 uint32_t bt) {
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)heads, (uint64_t)tokens};
    const uint64_t strides[2] = {(uint64_t)(heads > 1 ? sh : D) * 2, (uint64_t)(tokens > 1 ? st_ : D) * 2};
    const uint32_t box[3] = {64, bh, bt};
    return encode_tensor_map_3d(m, ty, p, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  int rc = map(&qm, a.q, a.hq, a.tq, a.q_h, a.q_t, (uint32_t)G, (uint32_t)nt);
  if (rc == TF_OK) {
    // no keys at all: the maps are never used, but must name something
    const bool none = a.tk == 0;
    rc = map(&km, none ? a.q : a.k, none ? a.hq : a.hkv, none ? a.tq : a.tk, none ? a.q_h : a.k_h,
             none ? a.q_t : a.k_t, 1, kRows);
    if (rc == TF_OK)
      rc = map(&vm, none ? a.q : a.v, none ? a.hq : a.hkv, none ? a.tq : a.tk, none ? a.q_h : a.v_h,
               none ? a.q_t : a.v_t, 1, kRows);
  }
  if (rc != TF_OK) return rc;
  const Plan plan = plan_of(a.tq, a.tk, a.S, a.hq, a.hkv, D);
  if (plan.pairs * a.hkv > INT32_MAX / 64) return fail(TF_ERR_BAD_SHAPE, "prompt_attention: too many tiles");
  a.max_pairs = (int)plan.pairs;
  a.splits = workspace_bytes >= plan.bytes ? plan.splits : 1;
  a.max_cut = (int)plan.cut;
  a.whole = plan.whole;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.err);
  a.next = reinterpret_cast<int*>(ws + 128);
  a.cut = reinterpret_cast<int*>(ws + 256);
  a.pieces = reinterpret_cast<float*>(ws + kFixedBytes);
  constexpr auto kern = prompt_attn_kernel<T, D>;
  rc = allow_smem<kern>("prompt_attention", L::kBytes);
  if (rc != TF_OK) return rc;
  const int64_t items = plan.pairs * a.hkv * (int64_t)a.splits;
  rc = launch_ex("prompt_attention", kern, dim3((unsigned)(items < num_sms() ? items : num_sms())), dim3(kThreads),
                 L::kBytes, st, dim3(1, 1, 1), qm, km, vm, a);
  if (rc != TF_OK || a.splits == 1) return rc;
  return launch_ex("prompt_attention join", prompt_join_kernel<T, D>, dim3((unsigned)(2 * plan.cut)),
                   dim3(kJoinThreads), 0, st, dim3(1, 1, 1), a);
}

}  // namespace
}  // namespace tf

extern "C" size_t tf_prompt_attention_workspace_bytes(int64_t Tq, int64_t Tk, int32_t S, int32_t hq, int32_t hkv,
                                                      int32_t head_dim) {
  using namespace tf;
  if (Tq <= 0 || Tk < 0 || S <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || hq / hkv > kRows) return kFixedBytes;
  return plan_of(Tq, Tk, S, hq, hkv, head_dim).bytes;
}

extern "C" int tf_prompt_attention(const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k,
                                   int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_h, void* out, int64_t o_stride_t, int64_t o_stride_h,
                                   const int* cu_q, const int* cu_k, int32_t S, int64_t Tq, int64_t Tk, int32_t hq,
                                   int32_t hkv, int32_t head_dim, int32_t causal, float scale, int dtype,
                                   void* workspace, size_t workspace_bytes, void* stream) {
  using namespace tf;
  if (S < 0 || Tq < 0 || Tk < 0 || hq <= 0 || hkv <= 0 || hq % hkv || Tq > INT32_MAX || Tk > INT32_MAX)
    return fail(TF_ERR_BAD_SHAPE, "prompt_attention: bad shape (S=%d, Tq=%lld, Tk=%lld, hq=%d, hkv=%d)", S,
                (long long)Tq, (long long)Tk, hq, hkv);
  if (dtype != TF_F16 && dtype != TF_BF16)
    return fail(TF_ERR_BAD_DTYPE, "prompt_attention: unsupported dtype %d", dtype);
  if (head_dim != 64 && head_dim != 128)
    return fail(TF_ERR_UNSUPPORTED, "prompt_attention: head_dim %d (64 or 128)", head_dim);
  if (hq / hkv > 128) return fail(TF_ERR_UNSUPPORTED, "prompt_attention: %d q heads per kv head (max 128)", hq / hkv);
  if (Tq == 0) return TF_OK;
  if (S == 0) return fail(TF_ERR_BAD_SHAPE, "prompt_attention: %lld queries in no sequence", (long long)Tq);
  if (!q || !out || !cu_q || !cu_k || (Tk > 0 && (!k || !v)))
    return fail(TF_ERR_BAD_ARG, "prompt_attention: null pointer");
  if (!(scale > 0.f) || !(scale < INFINITY))
    return fail(TF_ERR_BAD_ARG, "prompt_attention: scale %g must be positive", (double)scale);
  if (!workspace || workspace_bytes < kFixedBytes || !aligned(workspace, 16))
    return fail(TF_ERR_WORKSPACE, "prompt_attention: 16-byte aligned workspace of at least %zu bytes required", kFixedBytes);
  const int64_t strides[] = {q_stride_t, q_stride_h, k_stride_t, k_stride_h, v_stride_t, v_stride_h, o_stride_t,
                             o_stride_h};
  const int64_t sizes[] = {Tq, hq, Tk, hkv, Tk, hkv, Tq, hq};
  for (int i = 0; i < 8; ++i)
    if (sizes[i] > 1 && (strides[i] < head_dim || strides[i] % 8))
      return fail(TF_ERR_UNALIGNED, "prompt_attention: strides must be multiples of 8 elements, at least head_dim");
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16))
    return fail(TF_ERR_UNALIGNED, "prompt_attention: q, k, v and out must be 16-byte aligned");
  PromptArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.q_t = q_stride_t;
  a.q_h = q_stride_h;
  a.k_t = k_stride_t;
  a.k_h = k_stride_h;
  a.v_t = v_stride_t;
  a.v_h = v_stride_h;
  a.o_t = o_stride_t;
  a.o_h = o_stride_h;
  a.cu_q = cu_q;
  a.cu_k = cu_k;
  a.tq = Tq;
  a.tk = Tk;
  a.S = S;
  a.hq = hq;
  a.hkv = hkv;
  a.causal = causal;
  a.scale = scale;
  a.err = static_cast<int*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TF_F16) return head_dim == 64 ? launch_prompt<__half, 64>(a, workspace_bytes, st)
                                              : launch_prompt<__half, 128>(a, workspace_bytes, st);
  return head_dim == 64 ? launch_prompt<__nv_bfloat16, 64>(a, workspace_bytes, st)
                        : launch_prompt<__nv_bfloat16, 128>(a, workspace_bytes, st);
}
