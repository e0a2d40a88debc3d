// The paged cache in 4 bits on gfx950: appending keys and values to it, and reading
// them back.
//
// A head's row of D elements is held in blocks of 32: 32 codes E2M1 (a sign and one of
// 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte with the even element in the low bits, and
// one byte E8M0, 127 + e, for the block's scale 2^e -- the element and block formats of
// the OCP Microscaling specification (MXFP4), which gfx950 converts in hardware.  The
// scale is the smallest power of two (from 2^-126) that keeps the block's largest
// magnitude within 6, where the specification's own choice would let magnitudes past 6
// saturate; a code is the value over the scale, rounded to nearest, ties to the even
// code.  A scale of a power of two makes every step but that rounding exact, so the
// codes do not depend on the order or the width of the arithmetic.  Byte 255 marks a
// block that holds an infinity or a NaN, all of which then reads as NaN.
//
// Codes: [pages, 2, heads, slots, D / 2], scales: [pages, 2, heads, slots, D / 32] bytes
// (any strides but the last).  4 lanes take a block, 8 elements each.  Bound by the
// bytes: 16-bit k and v in, 4.25 bits an element out.
#include <type_traits>

#include "bfa_append.h"
#include "bfa_device.h"
#include "bfa_host.h"
#include "bfa_internal.h"

namespace bfa {

// AppendArgs addresses the codes (strides in bytes); the scales' strides beside it.
struct Fp4Args {
  AppendArgs a;
  uint8_t* scales;
  int64_t s_sp, s_skv, s_sh, s_ss;
  void* k_out;  // gather: [tokens, heads, D]
  void* v_out;
  int64_t tokens;
  FastDiv per_token;  // 2 * heads * D / 8
};

// A workgroup takes 256 N chunks of 8 elements, N to a lane, in order of token, K or V,
// head, element.  Its first lanes find where its tokens go (three dependent reads a
// token, while the elements' loads are in flight) and leave that in the LDS: with each
// lane finding its own token's place, one chunk a lane, 6000 tokens of 8 x 128 took
// 14.8 us to append, the loads' latency and that one's after another.
constexpr int FP4_TOKENS = 256 * 4 / 8 + 2;  // of a workgroup at most: 8 chunks a token at least
struct Fp4Place {
  int64_t codes, scales;  // byte offsets of the token's slot, -1: it has none
};
__device__ __forceinline__ void fp4_places(const Fp4Args& f, int64_t t0, int64_t t1, Fp4Place* places) {
  const AppendArgs& a = f.a;
  const int64_t t = t0 + threadIdx.x;
  if (t <= t1) {
    Fp4Place p{-1, -1};
    const AppendKey key = append_key(a, t);
    if (!(a.indptr && key.seq == -1)) {  // (request -1 is padding, which is no error)
      int64_t page = 0, slot = 0;
      const int bad = append_resolve(a, key, page, slot);
      if (bad) flag_status(a.status, bad);
      else p = Fp4Place{page * a.c_sp + slot * a.c_ss, page * f.s_sp + slot * f.s_ss};
    }
    places[threadIdx.x] = p;
  }
  __syncthreads();
}

// chunk i: its token, K or V, head and first element
struct Fp4Item {
  int64_t t;
  uint32_t kv, h, e;
};
__device__ __forceinline__ Fp4Item fp4_item(const Fp4Args& f, uint32_t i) {
  Fp4Item it;
  it.t = f.per_token.div(i);
  const uint32_t r = i - static_cast<uint32_t>(it.t) * f.per_token.d;
  it.kv = f.a.chunks_per_kv.div(r);
  const uint32_t q = r - it.kv * f.a.chunks_per_kv.d;
  it.h = f.a.chunks_per_head.div(q);
  it.e = (q - it.h * f.a.chunks_per_head.d) * 8;
  return it;
}

// 8 elements as codes, with the scale byte of their block, which 4 lanes share
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], uint32_t& byte) {
  // largest magnitude of the block, as bits (a NaN's are above an infinity's)
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(x[i]) & 0x7fffffffu);
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(most), 0xB1, 0xF, 0xF, false)));
  most = max(most, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(most), 0x4E, 0xF, 0xF, false)));
  // 1.m x 2^E stays within 6 x 2^e = 1.5 x 2^(e + 2) with e = E - 2, or E - 1 where 1.m > 1.5
  const int e = max(static_cast<int>(most >> 23) - 129 + ((most & 0x7fffffu) > 0x400000u ? 1 : 0), -126);
  const bool finite = most < 0x7f800000u;
  byte = finite ? static_cast<uint32_t>(e + 127) : 255u;
  const float scale = __uint_as_float(byte << 23);
  uint32_t w = 0;
  if (finite) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  }
  return w;
}

template <int DT, bool VEC, int N>
__global__ __launch_bounds__(256) void kv_fp4_append_kernel(Fp4Args f) {
  using T = typename Elem<DT>::T;
  const AppendArgs& a = f.a;
  __shared__ Fp4Place places[FP4_TOKENS];
  const uint32_t total = static_cast<uint32_t>(f.tokens) * f.per_token.d, i0 = blockIdx.x * 256u * N;
  const uint32_t last = min(i0 + 256u * N, total) - 1;
  Fp4Item it[N];
  float x[N][8];
#pragma unroll
  for (int n = 0; n < N; ++n) {  // (a lane past the end takes the last chunk, and stores nothing)
    it[n] = fp4_item(f, min(i0 + 256u * n + threadIdx.x, last));
    const T* src = it[n].kv == 0 ? static_cast<const T*>(a.k) + it[n].t * a.k_st + it[n].h * a.k_sh
                                 : static_cast<const T*>(a.v) + it[n].t * a.v_st + it[n].h * a.v_sh;
    if constexpr (VEC) {
      load8_nt<DT>(src + it[n].e, x[n]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[n][i] = Elem<DT>::to_f32(src[it[n].e + i]);
    }
  }
  const int64_t t0 = f.per_token.div(i0);
  fp4_places(f, t0, f.per_token.div(last), places);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    uint32_t byte;
    const uint32_t w = fp4_codes(x[n], byte);
    const Fp4Place p = places[it[n].t - t0];
    if (i0 + 256u * n + threadIdx.x > last || p.codes < 0) continue;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.cache) + p.codes + it[n].kv * a.c_skv + it[n].h * a.c_sh + it[n].e / 2) = w;
    if ((threadIdx.x & 3) == 0)
      f.scales[p.scales + it[n].kv * f.s_skv + it[n].h * f.s_sh + it[n].e / 32] = static_cast<uint8_t>(byte);
  }
}

// 8 codes and their scale as fp32, exactly
__device__ __forceinline__ void fp4_values(uint32_t w, uint32_t byte, float (&x)[8]) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float scale = __uint_as_float(byte << 23);
  const f32x2 v0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 0), v1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 1);
  const f32x2 v2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 2), v3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, 3);
  x[0] = v0.x; x[1] = v0.y; x[2] = v1.x; x[3] = v1.y;
  x[4] = v2.x; x[5] = v2.y; x[6] = v3.x; x[7] = v3.y;
}

template <int DT, int N>
__global__ __launch_bounds__(256) void kv_fp4_gather_kernel(Fp4Args f) {
  using T = typename Elem<DT>::T;
  const AppendArgs& a = f.a;
  __shared__ Fp4Place places[FP4_TOKENS];
  const uint32_t total = static_cast<uint32_t>(f.tokens) * f.per_token.d, i0 = blockIdx.x * 256u * N;
  const uint32_t last = min(i0 + 256u * N, total) - 1;
  const int64_t t0 = f.per_token.div(i0);
  fp4_places(f, t0, f.per_token.div(last), places);
  Fp4Item it[N];
  uint32_t w[N], byte[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    it[n] = fp4_item(f, min(i0 + 256u * n + threadIdx.x, last));
    const Fp4Place p = places[it[n].t - t0];
    w[n] = byte[n] = 0;  // (no place: zeros)
    if (p.codes >= 0) {
      w[n] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.cache) + p.codes + it[n].kv * a.c_skv +
                                                it[n].h * a.c_sh + it[n].e / 2);
      byte[n] = f.scales[p.scales + it[n].kv * f.s_skv + it[n].h * f.s_sh + it[n].e / 32];
    }
  }
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (i0 + 256u * n + threadIdx.x > last) continue;
    float x[8];
    fp4_values(w[n], byte[n], x);
    T* dst = static_cast<T*>(it[n].kv == 0 ? f.k_out : f.v_out) + (it[n].t * a.heads + it[n].h) * a.head_dim + it[n].e;
    store8<DT>(dst, x);
  }
}

// Checks and fills what the append and the gather share.
static int fp4_args(const char* what, const void* codes, const void* scales, int64_t num_pages, int64_t slots,
                    int64_t num_kv_heads, int64_t head_dim, const int64_t (&cs)[4], const int64_t (&ss)[4],
                    const void* kv_indices, int kv_indices_dtype, int64_t num_indices, const int32_t* kv_indptr,
                    const void* batch_indices, int batch_indices_dtype, int64_t num_seqs, const void* positions,
                    int positions_dtype, int64_t num_tokens, int32_t* status, Fp4Args* out) {
  BFA_REQUIRE(num_tokens >= 0 && num_kv_heads >= 0 && head_dim >= 0, "%s: bad geometry", what);
  BFA_REQUIRE(head_dim % 32 == 0, "%s: head_dim %lld (a multiple of 32)", what, static_cast<long long>(head_dim));
  const int64_t lim = int64_t{1} << 31;
  BFA_REQUIRE(num_tokens < lim && num_kv_heads < lim && head_dim < lim / 8 && num_kv_heads * (head_dim / 4) < lim &&
                  num_tokens * (num_kv_heads * (head_dim / 4)) < lim,
              "%s: too many elements in one call", what);
  for (int i = 0; i < 4; ++i)
    BFA_REQUIRE(cs[i] % 4 == 0, "%s: the codes' strides must be multiples of 4 bytes", what);
  BFA_REQUIRE((reinterpret_cast<uintptr_t>(codes) & 3) == 0, "%s: the codes must be 4-byte aligned", what);
  Fp4Args f{};
  const int rc = fill_append_args(what, const_cast<void*>(codes), BFA_DTYPE_F32, num_pages, slots, cs[0], cs[1], cs[2], cs[3],
                                  kv_indices, kv_indices_dtype, num_indices, kv_indptr, batch_indices, batch_indices_dtype,
                                  num_seqs, positions, positions_dtype, slots, status, &f.a);
  if (rc != BFA_OK) return rc;
  f.a.heads = static_cast<uint32_t>(num_kv_heads);
  f.a.head_dim = static_cast<uint32_t>(head_dim);
  f.scales = static_cast<uint8_t*>(const_cast<void*>(scales));
  f.s_sp = ss[0]; f.s_skv = ss[1]; f.s_sh = ss[2]; f.s_ss = ss[3];
  f.tokens = num_tokens;
  if (num_tokens > 0 && num_kv_heads > 0 && head_dim > 0) {
    BFA_REQUIRE(codes && scales && positions, "%s: null pointer", what);
    BFA_REQUIRE(num_indices == 0 || kv_indices, "%s: null kv_indices", what);
    f.a.chunks_per_head = FastDiv(static_cast<uint32_t>(head_dim / 8));
    f.a.chunks_per_kv = FastDiv(static_cast<uint32_t>(num_kv_heads * (head_dim / 8)));
    f.per_token = FastDiv(static_cast<uint32_t>(num_kv_heads * (head_dim / 4)));
  }
  *out = f;
  return BFA_OK;
}

// 4 chunks a lane where that leaves at least two workgroups a CU: 64 tokens of 8 x 128,
// 64 workgroups of one chunk a lane, are latency, 3.7 us; 6000 tokens take 10.1 us to
// append (31 MB, 3.1 TB/s) and 8.9 to gather with four chunks, 14.8 and 13.0 with one.
static bool fp4_many(const Fp4Args& f) { return f.tokens * f.per_token.d >= int64_t{512} * 1024; }
static dim3 fp4_grid(const Fp4Args& f, int n) {
  return dim3(static_cast<unsigned>(cdiv(f.tokens * f.per_token.d, 256 * n)));
}

}  // namespace bfa

using namespace bfa;

extern "C" int bfa_append_paged_kv_fp4(const void* k, const void* v, int kv_dtype, int64_t num_tokens,
                                       int64_t num_kv_heads, int64_t head_dim, int64_t k_stride_token,
                                       int64_t k_stride_head, int64_t v_stride_token, int64_t v_stride_head,
                                       void* codes, void* scales, int64_t num_pages, int64_t page_size,
                                       int64_t stride_page, int64_t stride_kv, int64_t stride_head,
                                       int64_t stride_slot, int64_t scale_stride_page, int64_t scale_stride_kv,
                                       int64_t scale_stride_head, int64_t scale_stride_slot, const void* kv_indices,
                                       int kv_indices_dtype, int64_t num_indices, const int32_t* kv_indptr,
                                       const void* batch_indices, int batch_indices_dtype, int64_t num_seqs,
                                       const void* positions, int positions_dtype, int32_t* status, void* stream) {
  const char* what = "bfa_append_paged_kv_fp4";
  BFA_REQUIRE(is_float_dtype(kv_dtype), "%s: bad dtype", what);
  Fp4Args f{};
  const int rc = fp4_args(what, codes, scales, num_pages, page_size, num_kv_heads, head_dim,
                          {stride_page, stride_kv, stride_head, stride_slot},
                          {scale_stride_page, scale_stride_kv, scale_stride_head, scale_stride_slot}, kv_indices,
                          kv_indices_dtype, num_indices, kv_indptr, batch_indices, batch_indices_dtype, num_seqs, positions,
                          positions_dtype, num_tokens, status, &f);
  if (rc != BFA_OK) return rc;
  if (num_tokens == 0 || num_kv_heads == 0 || head_dim == 0) return BFA_OK;
  BFA_REQUIRE(k && v, "%s: null pointer", what);
  f.a.k = k; f.a.v = v;
  f.a.k_st = k_stride_token; f.a.k_sh = k_stride_head;
  f.a.v_st = v_stride_token; f.a.v_sh = v_stride_head;
  const auto m8 = [](int64_t x) { return x % 8 == 0; };
  const bool vec = m8(k_stride_token) && m8(k_stride_head) && m8(v_stride_token) && m8(v_stride_head) && aligned16(k) && aligned16(v);
  const hipStream_t s = as_stream(stream);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (!vec) hipLaunchKernelGGL((kv_fp4_append_kernel<DT, false, 1>), fp4_grid(f, 1), dim3(256), 0, s, f);
    else if (fp4_many(f)) hipLaunchKernelGGL((kv_fp4_append_kernel<DT, true, 4>), fp4_grid(f, 4), dim3(256), 0, s, f);
    else hipLaunchKernelGGL((kv_fp4_append_kernel<DT, true, 1>), fp4_grid(f, 1), dim3(256), 0, s, f);
  };
  switch (kv_dtype) {
    case BFA_DTYPE_BF16: launch(std::integral_constant<int, BFA_DTYPE_BF16>{}); break;
    case BFA_DTYPE_F16: launch(std::integral_constant<int, BFA_DTYPE_F16>{}); break;
    default: launch(std::integral_constant<int, BFA_DTYPE_F32>{}); break;
  }
  return check_launch(what);
}

extern "C" int bfa_gather_paged_kv_fp4(const void* codes, const void* scales, int64_t num_pages, int64_t page_size,
                                       int64_t num_kv_heads, int64_t head_dim, int64_t stride_page, int64_t stride_kv,
                                       int64_t stride_head, int64_t stride_slot, int64_t scale_stride_page,
                                       int64_t scale_stride_kv, int64_t scale_stride_head, int64_t scale_stride_slot,
                                       const void* kv_indices, int kv_indices_dtype, int64_t num_indices,
                                       const int32_t* kv_indptr, const void* batch_indices, int batch_indices_dtype,
                                       int64_t num_seqs, const void* positions, int positions_dtype,
                                       int64_t num_tokens, void* k_out, void* v_out, int out_dtype, int32_t* status,
                                       void* stream) {
  const char* what = "bfa_gather_paged_kv_fp4";
  BFA_REQUIRE(is_float_dtype(out_dtype), "%s: bad dtype", what);
  Fp4Args f{};
  const int rc = fp4_args(what, codes, scales, num_pages, page_size, num_kv_heads, head_dim,
                          {stride_page, stride_kv, stride_head, stride_slot},
                          {scale_stride_page, scale_stride_kv, scale_stride_head, scale_stride_slot}, kv_indices,
                          kv_indices_dtype, num_indices, kv_indptr, batch_indices, batch_indices_dtype, num_seqs, positions,
                          positions_dtype, num_tokens, status, &f);
  if (rc != BFA_OK) return rc;
  if (num_tokens == 0 || num_kv_heads == 0 || head_dim == 0) return BFA_OK;
  BFA_REQUIRE(k_out && v_out && aligned16(k_out) && aligned16(v_out), "%s: outputs must be 16-byte aligned", what);
  f.k_out = k_out; f.v_out = v_out;
  const hipStream_t s = as_stream(stream);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (fp4_many(f)) hipLaunchKernelGGL((kv_fp4_gather_kernel<DT, 4>), fp4_grid(f, 4), dim3(256), 0, s, f);
    else hipLaunchKernelGGL((kv_fp4_gather_kernel<DT, 1>), fp4_grid(f, 1), dim3(256), 0, s, f);
  };
  switch (out_dtype) {
    case BFA_DTYPE_BF16: launch(std::integral_constant<int, BFA_DTYPE_BF16>{}); break;
    case BFA_DTYPE_F16: launch(std::integral_constant<int, BFA_DTYPE_F16>{}); break;
    default: launch(std::integral_constant<int, BFA_DTYPE_F32>{}); break;
  }
  return check_launch(what);
}
