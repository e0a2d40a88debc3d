// RMSNorm of every query and key head and their rotation by position, in one pass,
// on gfx950 (Qwen3: models/qwen3.py:257-309 applies q_norm, k_norm and rotary_emb to
// the projection's output one after the other):
//
//   x' = x / sqrt(mean(x^2) + eps) * w,   y1 = x1' cos - x2' sin,  y2 = x2' cos + x1' sin
//
// with the halves x1', x2' of a head's row and the position's row of the fp32
// cos | sin table.  All of it in fp32, rounded once, to the type of x.
//
// A row (one head of one token) is taken by L = D / 16 lanes (the next power of two),
// each with 8 elements of either half: the pairs of the rotation are in one lane, the
// sum of squares takes log2 L lane exchanges, and a row's loads and stores are 16
// bytes a lane.  Bound by the bytes of q and k, in and out.
#include "bfa_device.h"
#include "bfa_host.h"

namespace bfa {

struct QkArgs {
  const void* x[2];  // q, k
  void* y[2];
  const void* w[2];
  int64_t st[2], sh[2];  // token, head strides; the outputs are contiguous [tokens, heads, D]
  uint32_t heads[2];
  uint32_t rows_per_token;
  FastDiv per_token;
  int64_t tokens;
  int32_t dim;
  int w_dt;
  float eps;
  const void* positions;
  int pos_i64;
  const float* table;
  int64_t max_pos;
  int* status;
};

__device__ __forceinline__ int64_t qk_position(const QkArgs& a, int64_t t, bool& ok) {
  int64_t p = a.pos_i64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
  if (p < 0) p += a.max_pos;  // as a torch index
  ok = p >= 0 && p < a.max_pos;
  return ok ? p : 0;
}

__device__ __forceinline__ void load8_any(const void* p, int dt, int64_t i, float (&v)[8]) {
  if (dt == BFA_DTYPE_F32) load8<BFA_DTYPE_F32>(static_cast<const float*>(p) + i, v);
  else if (dt == BFA_DTYPE_BF16) load8<BFA_DTYPE_BF16>(static_cast<const uint16_t*>(p) + i, v);
  else load8<BFA_DTYPE_F16>(static_cast<const uint16_t*>(p) + i, v);
}

// 16-byte rows: L lanes a row, 256 / L rows a workgroup.
template <int DT, int L>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(QkArgs a) {
  using T = typename Elem<DT>::T;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
  if (row >= a.tokens * a.rows_per_token) return;  // whole groups of L lanes
  const int j = threadIdx.x % L, half = a.dim / 2;
  const bool act = 8 * j < half;
  const int64_t t = a.per_token.div(static_cast<uint32_t>(row));
  uint32_t h = static_cast<uint32_t>(row) - static_cast<uint32_t>(t) * a.rows_per_token;
  const int s = h >= a.heads[0];
  if (s) h -= a.heads[0];
  const int e = act ? 8 * j : 0;
  const T* x = static_cast<const T*>(a.x[s]) + t * a.st[s] + h * a.sh[s] + e;
  float x1[8], x2[8], c[8], n[8];
  load8<DT>(x, x1);
  load8<DT>(x + half, x2);
  bool ok;
  const int64_t p = qk_position(a, t, ok);
  if (!ok && j == 0) flag_status(a.status, BFA_STATUS_INDEX_OOB);
  const float* cs = a.table + p * a.dim + e;
  load8<BFA_DTYPE_F32>(cs, c);
  load8<BFA_DTYPE_F32>(cs + half, n);
  if (a.w[s]) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += x1[i] * x1[i] + x2[i] * x2[i];
    sum = group_sum<L>(act ? sum : 0.f);
    const float r = 1.0f / sqrtf(sum / static_cast<float>(a.dim) + a.eps);
    float w1[8], w2[8];
    load8_any(a.w[s], a.w_dt, e, w1);
    load8_any(a.w[s], a.w_dt, half + e, w2);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x1[i] = x1[i] * r * w1[i];
      x2[i] = x2[i] * r * w2[i];
    }
  }
  if (!act) return;
  float y1[8], y2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    y1[i] = ok ? x1[i] * c[i] - x2[i] * n[i] : 0.f;
    y2[i] = ok ? x2[i] * c[i] + x1[i] * n[i] : 0.f;
  }
  T* y = static_cast<T*>(a.y[s]) + (t * a.heads[s] + h) * a.dim + e;
  store8<DT>(y, y1);
  store8<DT>(y + half, y2);
}

// Any even head_dim and any alignment: a wave a row, a pair of the rotation a lane.
template <int DT>
__global__ __launch_bounds__(256) void qk_norm_rope_scalar_kernel(QkArgs a) {
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= a.tokens * a.rows_per_token) return;
  const int lane = threadIdx.x & 63, half = a.dim / 2;
  const int64_t t = a.per_token.div(static_cast<uint32_t>(row));
  uint32_t h = static_cast<uint32_t>(row) - static_cast<uint32_t>(t) * a.rows_per_token;
  const int s = h >= a.heads[0];
  if (s) h -= a.heads[0];
  const int64_t x0 = t * a.st[s] + h * a.sh[s], y0 = (t * a.heads[s] + h) * a.dim;
  bool ok;
  const int64_t p = qk_position(a, t, ok);
  if (!ok && lane == 0) flag_status(a.status, BFA_STATUS_INDEX_OOB);
  float r = 1.f;
  if (a.w[s]) {
    float sum = 0.f;
    for (int i = lane; i < a.dim; i += 64) {
      const float v = load1<DT>(a.x[s], x0 + i);
      sum += v * v;
    }
    r = 1.0f / sqrtf(group_sum<64>(sum) / static_cast<float>(a.dim) + a.eps);
  }
  for (int i = lane; i < half; i += 64) {
    float u = load1<DT>(a.x[s], x0 + i), v = load1<DT>(a.x[s], x0 + half + i);
    if (a.w[s]) {
      u = u * r * load_any(a.w[s], a.w_dt, i);
      v = v * r * load_any(a.w[s], a.w_dt, half + i);
    }
    const float c = a.table[p * a.dim + i], n = a.table[p * a.dim + half + i];
    store1<DT>(a.y[s], y0 + i, ok ? u * c - v * n : 0.f);
    store1<DT>(a.y[s], y0 + half + i, ok ? v * c + u * n : 0.f);
  }
}

template <int DT>
static void launch_qk(const QkArgs& a, bool vec, hipStream_t s) {
  const int64_t rows = a.tokens * a.rows_per_token;
  auto grid = [&](int64_t per) { return dim3(static_cast<unsigned>(cdiv(rows, per))); };
  if (!vec) {
    hipLaunchKernelGGL((qk_norm_rope_scalar_kernel<DT>), grid(4), dim3(256), 0, s, a);
  } else if (a.dim <= 32) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 2>), grid(128), dim3(256), 0, s, a);
  } else if (a.dim <= 64) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 4>), grid(64), dim3(256), 0, s, a);
  } else if (a.dim <= 128) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 8>), grid(32), dim3(256), 0, s, a);
  } else if (a.dim <= 256) {
    hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 16>), grid(16), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((qk_norm_rope_kernel<DT, 64>), grid(4), dim3(256), 0, s, a);
  }
}

}  // namespace bfa

using namespace bfa;

extern "C" int bfa_qk_norm_rope(const void* query, int64_t q_heads, int64_t q_stride_token, int64_t q_stride_head,
                                void* query_out, const void* key, int64_t k_heads, int64_t k_stride_token,
                                int64_t k_stride_head, void* key_out, int dtype, int64_t num_tokens,
                                int64_t head_dim, const void* q_norm_weight, const void* k_norm_weight,
                                int weight_dtype, float eps, const void* positions, int positions_dtype,
                                const float* cos_sin_cache, int64_t max_position, int32_t* status, void* stream) {
  const char* what = "bfa_qk_norm_rope";
  BFA_REQUIRE(is_float_dtype(dtype), "%s: bad dtype", what);
  BFA_REQUIRE((!q_norm_weight && !k_norm_weight) || is_float_dtype(weight_dtype), "%s: bad weight dtype", what);
  BFA_REQUIRE(positions_dtype == BFA_DTYPE_I32 || positions_dtype == BFA_DTYPE_I64, "%s: positions must be int32/int64", what);
  BFA_REQUIRE(num_tokens >= 0 && q_heads >= 0 && k_heads >= 0 && head_dim > 0 && head_dim % 2 == 0 && head_dim < 65536,
              "%s: bad geometry (head_dim must be even)", what);
  const int64_t lim = int64_t{1} << 31;
  BFA_REQUIRE(q_heads < lim && k_heads < lim && num_tokens < lim && (q_heads + k_heads) * std::max<int64_t>(num_tokens, 1) < lim,
              "%s: 2^31 rows or more", what);
  if (num_tokens == 0 || q_heads + k_heads == 0) return BFA_OK;
  BFA_REQUIRE((q_heads == 0 || (query && query_out)) && (k_heads == 0 || (key && key_out)) && positions && cos_sin_cache,
              "%s: null pointer", what);
  BFA_REQUIRE(max_position > 0, "%s: empty rotary table", what);
  QkArgs a{};
  a.x[0] = query; a.x[1] = key;
  a.y[0] = query_out; a.y[1] = key_out;
  a.w[0] = q_norm_weight; a.w[1] = k_norm_weight;
  a.st[0] = q_stride_token; a.st[1] = k_stride_token;
  a.sh[0] = q_stride_head; a.sh[1] = k_stride_head;
  a.heads[0] = static_cast<uint32_t>(q_heads); a.heads[1] = static_cast<uint32_t>(k_heads);
  a.rows_per_token = a.heads[0] + a.heads[1];
  a.per_token = FastDiv(a.rows_per_token);
  a.tokens = num_tokens; a.dim = static_cast<int32_t>(head_dim);
  a.w_dt = weight_dtype; a.eps = eps;
  a.positions = positions; a.pos_i64 = positions_dtype == BFA_DTYPE_I64;
  a.table = cos_sin_cache; a.max_pos = max_position;
  a.status = status;
  const auto m8 = [](int64_t v) { return v % 8 == 0; };
  const bool vec = head_dim % 16 == 0 && head_dim <= 1024 && m8(q_stride_token) && m8(q_stride_head) && m8(k_stride_token) &&
                   m8(k_stride_head) && aligned16(query) && aligned16(key) && aligned16(query_out) && aligned16(key_out) &&
                   aligned16(q_norm_weight) && aligned16(k_norm_weight) && aligned16(cos_sin_cache);
  int64_t lanes = 64;  // of a row
  if (vec && head_dim <= 256)
    for (lanes = 2; lanes * 16 < head_dim;) lanes *= 2;
  BFA_REQUIRE(cdiv(num_tokens * (q_heads + k_heads), 256 / lanes) < (int64_t{1} << 24),  // (a launch has 2^32 threads)
              "%s: too many rows in one call", what);
  const hipStream_t s = as_stream(stream);
  switch (dtype) {
    case BFA_DTYPE_BF16: launch_qk<BFA_DTYPE_BF16>(a, vec, s); break;
    case BFA_DTYPE_F16: launch_qk<BFA_DTYPE_F16>(a, vec, s); break;
    default: launch_qk<BFA_DTYPE_F32>(a, vec, s); break;
  }
  return check_launch(what);
}
