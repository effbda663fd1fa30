// Writing and reading the 4-bit KV cache (format: kv4.cuh), one pass over the
// rows. A row (one token's key or value of one kv head) is taken by D / 16
// lanes, each holding channels [8i, 8i + 8) and [D/2 + 8i, D/2 + 8i + 8): two
// 16-byte loads, the group minima and maxima by shuffles, and the two channels
// of a rotary pair always in one lane.
// 20011 tokens of 8 heads of 128, bf16, groups of 128: written in 27.4 us, read in
// 22.7, 58% and 70% of the copy bandwidth (104 MB each; with 14 / 2 heads of 64 or
// few tokens it is the launch); 64 query and 8 key heads rotated and keys and values
// written in 196 us, 62% (801 MB). Instruction issue bounds both: about 15
// instructions a channel and lane to write, and loads of 4 bytes a lane to read.
#include "kv4.cuh"
#include "packed.cuh"

namespace tf {
namespace {

struct Kv4Rows {
  Kv4Cache c;
  const int* cu;     // [S + 1] packed offsets
  const int* start;  // [S] first cache position of each sequence, or null (0)
  const int* slots;  // [S] cache row of each sequence, or null (its index)
  int64_t T, B, t_max;
  int S, hkv;
};

// Cache row (in rows of D channels) of packed token t's kv head 0, or -1 outside
// the cache or in no sequence (before cu[0], from cu[S] on); the other heads'
// follow t_max rows apart. `pos` is its position.
__device__ __forceinline__ int64_t cache_row(const Kv4Rows& a, int64_t t, int64_t& pos) {
  const int s = packed_sequence(a.cu, a.S, t);
  const int64_t in = t - a.cu[s];
  pos = in + (a.start ? a.start[s] : 0);
  const int64_t b = a.slots ? a.slots[s] : s;
  if (in < 0 || t >= a.cu[s + 1] || pos < 0 || pos >= a.t_max || b < 0 || b >= a.B) return -1;
  return b * a.hkv * a.t_max + pos;
}

// A warp takes a token's head rows, 32 / (D / 16) at a time; the grid's y axis
// splits them where there are few tokens. Head rows are [q heads (kRope)] | k
// heads | v heads. kRope: q and k are views of the projection rows, rotated in
// place with transformers' roundings: round(round(x cos) + round(rotate_half(x) sin)).
template <typename T, int D, int G, bool kRope>
__global__ void __launch_bounds__(256) kv4_write_kernel(const Kv4Rows a, T* q, const T* k, const T* v, int64_t q_t,
                                                        int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h, int hq,
                                                        const T* __restrict__ cos_t, const T* __restrict__ sin_t) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, li = lane % kLanes;
  const int rows = (kRope ? hq : 0) + 2 * a.hkv;
  const int groups = (rows + kRows - 1) / kRows;
  const int g0 = groups * (int)blockIdx.y / (int)gridDim.y, g1 = groups * (int)(blockIdx.y + 1) / (int)gridDim.y;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32);
  int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5), next_pos = 0;
  int64_t next_row = t < a.T ? cache_row(a, t, next_pos) : -1;
  for (; t < a.T; t += step) {
    const int64_t pos = next_pos, row0 = next_row;
    if (t + step < a.T) next_row = cache_row(a, t + step, next_pos);  // beside this token's loads
#pragma unroll 1  // (registers: five blocks per SM; unrolled twice 30.7 us)
    for (int g = g0; g < g1; ++g) {
      int r = g * kRows + lane / kLanes;
      const bool active = r < rows;
      if (!active) r = rows - 1;
      const int kind = kRope ? (r < hq ? 0 : r < hq + a.hkv ? 1 : 2) : (r < a.hkv ? 1 : 2);
      const int h = kind == 0 ? r : r - (kRope ? hq : 0) - (kind == 2 ? a.hkv : 0);
      const T* src = kind == 0 ? q + t * q_t + h * D : kind == 1 ? k + t * k_t + h * k_h : v + t * v_t + h * v_h;
      Half8<T> x1, x2;
      x1.raw = *reinterpret_cast<const uint4*>(src + 8 * li);
      x2.raw = *reinterpret_cast<const uint4*>(src + D / 2 + 8 * li);
      if constexpr (kRope) {
        if (kind != 2 && row0 >= 0) {
          Half8<T> c1, c2, s1, s2;
          c1.raw = *reinterpret_cast<const uint4*>(cos_t + pos * D + 8 * li);
          c2.raw = *reinterpret_cast<const uint4*>(cos_t + pos * D + D / 2 + 8 * li);
          s1.raw = *reinterpret_cast<const uint4*>(sin_t + pos * D + 8 * li);
          s2.raw = *reinterpret_cast<const uint4*>(sin_t + pos * D + D / 2 + 8 * li);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float u = x1.get(e), w = x2.get(e);
            x1.set(e, round_to<T>(u * c1.get(e)) + round_to<T>(-w * s1.get(e)));
            x2.set(e, round_to<T>(w * c2.get(e)) + round_to<T>(u * s2.get(e)));
          }
          if (active) {
            T* dst = const_cast<T*>(src);
            *reinterpret_cast<uint4*>(dst + 8 * li) = x1.raw;
            *reinterpret_cast<uint4*>(dst + D / 2 + 8 * li) = x2.raw;
          }
        }
      }
      uint32_t w1, w2, params;
      kv4_quantize_row<T, D, G>(x1, x2, li, w1, w2, params);
      if (active && kind != 0 && row0 >= 0) {
        const int64_t row = row0 + (int64_t)h * a.t_max;
        uint8_t* codes = (kind == 1 ? a.c.k : a.c.v) + row * (D / 2);
        *reinterpret_cast<uint32_t*>(codes + 4 * li) = w1;
        *reinterpret_cast<uint32_t*>(codes + D / 4 + 4 * li) = w2;
        if (li < D / G) reinterpret_cast<uint32_t*>(kind == 1 ? a.c.k_params : a.c.v_params)[row * (D / G) + li] = params;
      }
    }
  }
}

template <typename T, int D, int G>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Rows a, T* k, T* v, int64_t k_t, int64_t k_h,
                                                       int64_t v_t, int64_t v_h) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = D / 16, kRows = 32 / kLanes;
  const int lane = threadIdx.x & 31, li = lane % kLanes;
  const int rows = 2 * a.hkv;
  const int groups = (rows + kRows - 1) / kRows;
  const int g0 = groups * (int)blockIdx.y / (int)gridDim.y, g1 = groups * (int)(blockIdx.y + 1) / (int)gridDim.y;
  const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32);
  int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5), next_pos = 0;
  int64_t next_row = t < a.T ? cache_row(a, t, next_pos) : -1;
  for (; t < a.T; t += step) {
    const int64_t row0 = next_row;
    if (t + step < a.T) next_row = cache_row(a, t + step, next_pos);  // beside this token's loads
#pragma unroll 4
    for (int g = g0; g < g1; ++g) {
      const int r = g * kRows + lane / kLanes;
      if (r >= rows) continue;
      const bool key = r < a.hkv;
      const int h = key ? r : r - a.hkv;
      uint4 o1 = make_uint4(0u, 0u, 0u, 0u), o2 = o1;
      if (row0 >= 0) {
        const int64_t row = row0 + (int64_t)h * a.t_max;
        const uint8_t* c = (key ? a.c.k : a.c.v) + row * (D / 2);
        const uint32_t* pr = reinterpret_cast<const uint32_t*>(key ? a.c.k_params : a.c.v_params) + row * (D / G);
        o1 = kv4_values<T>(*reinterpret_cast<const uint32_t*>(c + 4 * li), pr[0]);
        o2 = kv4_values<T>(*reinterpret_cast<const uint32_t*>(c + D / 4 + 4 * li), pr[G == D ? 0 : 1]);
      }
      T* dst = key ? k + t * k_t + h * k_h : v + t * v_t + h * v_h;
      *reinterpret_cast<uint4*>(dst + 8 * li) = o1;
      *reinterpret_cast<uint4*>(dst + D / 2 + 8 * li) = o2;
    }
  }
}

// Blocks of eight warps, a token per warp, `per_sm` per SM at most (writing 10,
// two rounds of those that fit: 27.0 us against 29.2 with one and 28.0 with a
// token each; reading 16: 22.9, with 10 24.5); with few tokens a token's head
// rows are spread over the y axis.
dim3 row_grid(int64_t T, int rows, int head_dim, int per_sm) {
  const int groups = (int)cdiv(rows, 32 / (head_dim / 16));
  const int64_t cap = (int64_t)num_sms() * per_sm, blocks = cdiv(T, 8);
  int64_t y = cdiv((int64_t)num_sms() * 4, blocks);
  y = y < groups ? y : groups;
  return dim3((unsigned)(blocks < cap ? blocks : cap), (unsigned)y);
}

int check_packed(const char* what, int64_t T, int S, const int* cu) {
  if (T < 0 || S < 0 || T > INT32_MAX) return fail(TF_ERR_BAD_SHAPE, "%s: bad packed shape", what);
  if (T > 0 && S == 0) return fail(TF_ERR_BAD_SHAPE, "%s: %lld tokens in no sequence", what, (long long)T);
  if (T > 0 && !cu) return fail(TF_ERR_BAD_ARG, "%s: null cu_seqlens", what);
  return TF_OK;
}

// (the stride of an axis of one element counts for nothing)
int check_rows(const char* what, const void* k, const void* v, int64_t k_t, int64_t k_h, int64_t v_t, int64_t v_h,
               int64_t T, int hkv) {
  if (!k || !v) return fail(TF_ERR_BAD_ARG, "%s: null pointer", what);
  const bool tokens = T > 1 && (k_t < 0 || v_t < 0 || k_t % 8 || v_t % 8);
  const bool heads = hkv > 1 && (k_h < 0 || v_h < 0 || k_h % 8 || v_h % 8);
  if (tokens || heads || !aligned(k, 16) || !aligned(v, 16))
    return fail(TF_ERR_UNALIGNED, "%s: rows must be 16-byte aligned", what);
  return TF_OK;
}

// f(T, D, G) over the supported (type, head size, group) combinations
template <typename F>
int kv4_dispatch(int dtype, int head_dim, int group, F&& f) {
  auto by_type = [&](auto zero) {
    if (head_dim == 64) return f(zero, std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
    if (group == 64) return f(zero, std::integral_constant<int, 128>{}, std::integral_constant<int, 64>{});
    return f(zero, std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{});
  };
  return dtype == TF_F16 ? by_type((__half*)nullptr) : by_type((__nv_bfloat16*)nullptr);
}

}  // namespace
}  // namespace tf

extern "C" int tf_kv4_write(const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                            int64_t v_stride_h, uint8_t* k_codes, void* k_params, uint8_t* v_codes, void* v_params,
                            const int* cu, const int* start, const int* slots, int32_t S, int64_t T, int64_t B,
                            int32_t hkv, int32_t head_dim, int32_t group, int64_t t_max, int dtype, void* stream) {
  using namespace tf;
  const Kv4Cache c{k_codes, k_params, v_codes, v_params};
  int rc = kv4_check("kv4_write", c, B, hkv, head_dim, group, t_max, dtype);
  if (rc == TF_OK) rc = check_packed("kv4_write", T, S, cu);
  if (rc != TF_OK || T == 0) return rc;
  rc = check_rows("kv4_write", k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, T, hkv);
  if (rc != TF_OK) return rc;
  const Kv4Rows a{c, cu, start, slots, T, B, t_max, S, hkv};
  return kv4_dispatch(dtype, head_dim, group, [&](auto type, auto d, auto g) {
    using E = std::remove_pointer_t<decltype(type)>;
    return launch_ex("kv4_write", kv4_write_kernel<E, d.value, g.value, false>,
                     row_grid(T, 2 * hkv, head_dim, 10), dim3(256), 0, static_cast<cudaStream_t>(stream),
                     dim3(1, 1, 1), a, (E*)nullptr, (const E*)k, (const E*)v, (int64_t)0, k_stride_t, k_stride_h,
                     v_stride_t, v_stride_h, 0, (const E*)nullptr, (const E*)nullptr);
  });
}

extern "C" int tf_rope_kv4_write(void* qkv, int64_t ld_qkv, const void* cos_table, const void* sin_table,
                                 uint8_t* k_codes, void* k_params, uint8_t* v_codes, void* v_params, const int* cu,
                                 const int* start, const int* slots, int32_t S, int64_t T, int64_t B, int32_t hq,
                                 int32_t hkv, int32_t head_dim, int32_t group, int64_t t_max, int dtype, void* stream) {
  using namespace tf;
  const Kv4Cache c{k_codes, k_params, v_codes, v_params};
  int rc = kv4_check("rope_kv4_write", c, B, hkv, head_dim, group, t_max, dtype);
  if (rc == TF_OK) rc = check_packed("rope_kv4_write", T, S, cu);
  if (rc != TF_OK) return rc;
  if (hq < 0 || ld_qkv < (int64_t)(hq + 2 * hkv) * head_dim)
    return fail(TF_ERR_BAD_SHAPE, "rope_kv4_write: ld_qkv %lld for %d + 2 x %d heads", (long long)ld_qkv, hq, hkv);
  if (T == 0) return TF_OK;
  if (!qkv || !cos_table || !sin_table) return fail(TF_ERR_BAD_ARG, "rope_kv4_write: null pointer");
  if (ld_qkv % 8 || !aligned(qkv, 16) || !aligned(cos_table, 16) || !aligned(sin_table, 16))
    return fail(TF_ERR_UNALIGNED, "rope_kv4_write: qkv rows and rotary tables must be 16-byte aligned");
  const Kv4Rows a{c, cu, start, slots, T, B, t_max, S, hkv};
  return kv4_dispatch(dtype, head_dim, group, [&](auto type, auto d, auto g) {
    using E = std::remove_pointer_t<decltype(type)>;
    E* q = (E*)qkv;
    const int64_t dd = head_dim;
    return launch_ex("rope_kv4_write", kv4_write_kernel<E, d.value, g.value, true>,
                     row_grid(T, hq + 2 * hkv, head_dim, 10), dim3(256), 0, static_cast<cudaStream_t>(stream),
                     dim3(1, 1, 1), a, q, (const E*)(q + hq * dd), (const E*)(q + (hq + hkv) * dd), ld_qkv, ld_qkv, dd,
                     ld_qkv, dd, hq, (const E*)cos_table, (const E*)sin_table);
  });
}

extern "C" int tf_kv4_read(const uint8_t* k_codes, const void* k_params, const uint8_t* v_codes, const void* v_params,
                           void* k, int64_t k_stride_t, int64_t k_stride_h, void* v, int64_t v_stride_t,
                           int64_t v_stride_h, const int* cu, const int* start, const int* slots, int32_t S, int64_t T,
                           int64_t B, int32_t hkv, int32_t head_dim, int32_t group, int64_t t_max, int dtype,
                           void* stream) {
  using namespace tf;
  const Kv4Cache c{(uint8_t*)k_codes, (void*)k_params, (uint8_t*)v_codes, (void*)v_params};
  int rc = kv4_check("kv4_read", c, B, hkv, head_dim, group, t_max, dtype);
  if (rc == TF_OK) rc = check_packed("kv4_read", T, S, cu);
  if (rc != TF_OK || T == 0) return rc;
  rc = check_rows("kv4_read", k, v, k_stride_t, k_stride_h, v_stride_t, v_stride_h, T, hkv);
  if (rc != TF_OK) return rc;
  if ((T > 1 && (k_stride_t < head_dim || v_stride_t < head_dim)) ||
      (hkv > 1 && (k_stride_h < head_dim || v_stride_h < head_dim)))
    return fail(TF_ERR_BAD_SHAPE, "kv4_read: output rows overlap");
  const Kv4Rows a{c, cu, start, slots, T, B, t_max, S, hkv};
  return kv4_dispatch(dtype, head_dim, group, [&](auto type, auto d, auto g) {
    using E = std::remove_pointer_t<decltype(type)>;
    return launch_ex("kv4_read", kv4_read_kernel<E, d.value, g.value>, row_grid(T, 2 * hkv, head_dim, 16),
                     dim3(256), 0, static_cast<cudaStream_t>(stream), dim3(1, 1, 1), a, (E*)k, (E*)v, k_stride_t,
                     k_stride_h, v_stride_t, v_stride_h);
  });
}
