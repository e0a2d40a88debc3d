// Attention of a ragged batch over one paged cache on gfx950, with a sliding
// window and a few first tokens that stay visible, the cache in 16 bits or in 4.
//
//   o_r = sum_j p_rj v_j / sum_j p_rj,   p_rj = exp(scale q_r . k_j - max_j)
//
// over the keys j that row r sees (bfa_paged.h); a row that sees none is 0.  A row
// is a query token and one of the Hq / Hkv query heads of a kv head, so a key that
// is read serves all of them.  Scores, maxima, sums and accumulators are fp32; the
// weights p are rounded to the queries' 16-bit type for the matrix product (by at most
// half a step, 2^-8 of p in bf16 and 2^-11 in fp16), since the matrix cores take V in
// that type, and the sum below adds them before that; the output is rounded once.
//
// The 4-bit cache holds E2M1 codes, two to a byte, and a power-of-two scale (E8M0)
// for each 32 elements of a row.  v_cvt_scalef32_pk_bf16_fp4 gives two elements'
// bf16 values, scale included, exactly; in fp16 the scale is taken 2^-4 times (a
// value of 4 x 2^14, which an fp16 key of 57344 and more has, is past fp16) and
// scores and output 2^4 times.
//
// The matrix work is done transposed, S^T = K Q^T and O^T = V^T P^T, with
// v_mfma_f32_16x16x32: a lane owns one row (lane % 16), its maximum and its sum,
// and P^T is the second product's B operand in the registers that hold it.  V^T
// comes from the row-major V tile in the LDS by the transposing reads
// (ds_read_b64_tr_b16: of 16 lanes, lane s passes the address of row s / 4,
// elements 4 (s % 4) .. +3, and gets element s of each of the four rows).
//
// Work is cut by the device itself (locate below), from the lengths that only it
// needs to know: an item is a block of rows and a range of its key tiles, so that
// one long request among short ones, or a few rows over a long cache, still fill
// the chip, and a captured graph follows the lengths of each replay.
#include <limits.h>

#include <cmath>

#include <type_traits>

#include "bfa_device.h"
#include "bfa_host.h"
#include "bfa_paged.h"
#include "bfa_paged_scan.h"

namespace bfa {

typedef __attribute__((ext_vector_type(8))) __bf16 pa_bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 pa_f16x8_t;
typedef __attribute__((ext_vector_type(4))) float pa_f32x4_t;
typedef __attribute__((ext_vector_type(4))) short pa_s16x4_t;
typedef __attribute__((address_space(3))) pa_s16x4_t pa_lds_s16x4_t;

struct PagedArgs {
  const uint16_t* q;  // [tokens, Hq, D], token / head strides
  int64_t q_st, q_sh;
  const uint8_t* cache;           // 16-bit elements, or codes
  uint32_t c_sp, c_ss;            // page, slot strides in 16-byte units
  int64_t c_skv, c_sh;            // K|V, head strides in bytes
  const uint8_t* scales;          // of the 4-bit cache
  uint32_t s_sp, s_ss;            // its strides in bytes
  int64_t s_skv, s_sh;
  int64_t num_pages;
  const int32_t* indices;
  int64_t num_indices;
  const int32_t* kv_indptr;
  const int32_t* last;
  const int32_t* qo_indptr;
  int32_t num_seqs;
  int64_t tokens;
  uint32_t hq, hkv;
  FastDiv group, ps, heads;       // Hq / Hkv, page size, Hkv
  float sl2, oscale;              // |scale| x log2(e) (1 for a scale of 0), factor of the output
  uint32_t qand, qxor;            // on pairs of query values: zero them, turn their signs
  PagedShape shape;
  int32_t sinks;
  uint16_t* out;                  // [tokens, Hq * D], row stride out_st
  int64_t out_st;
  int32_t split, target, least;   // split 0: an item is a block
  int32_t shift;                  // of the sum of the work
  int32_t nblocks, items;         // bounds of the blocks and the items
  int4* plan;                     // [items, 2] the items, where a launch of its own finds them
  float* acc;                     // [items, Hkv, BM, D] partial sums
  float* ml;                      // [items, Hkv, BM, 2] their maxima and sums
  int4* table;                    // [nblocks] (first item, items, first query row, rows) of a block
  int* status;
};

template <bool BF16>
__device__ __forceinline__ pa_f32x4_t pa_mfma(const uint4& a, const uint4& b, pa_f32x4_t c) {
  if constexpr (BF16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pa_bf16x8_t, a),
                                                   __builtin_bit_cast(pa_bf16x8_t, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(pa_f16x8_t, a),
                                                  __builtin_bit_cast(pa_f16x8_t, b), c, 0, 0, 0);
  }
}

template <bool BF16>
__device__ __forceinline__ uint32_t pa_pack(float lo, float hi) {
  if constexpr (BF16) {
    return pack_bf16x2(lo, hi);
  } else {
    return static_cast<uint32_t>(f32_to_f16_bits(lo)) | (static_cast<uint32_t>(f32_to_f16_bits(hi)) << 16);
  }
}

// 8 codes (a dword, the first element in the low 4 bits) as 16-bit values times the
// power of two in `scale`'s exponent
template <bool BF16>
__device__ __forceinline__ uint4 pa_from4(uint32_t w, float scale) {
  if constexpr (BF16) {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3)));
  } else {
    return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 0)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 1)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 2)),
                      __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, 3)));
  }
}
// a scale byte as the float whose exponent the conversion takes; 255 stands for NaN
template <bool BF16>
__device__ __forceinline__ float pa_scale(uint32_t byte) {
  if constexpr (!BF16) byte = byte == 255u ? 255u : byte < 4u ? 0u : byte - 4u;
  return __uint_as_float(byte << 23);
}

// whether a word holds a 16-bit infinity or NaN
template <bool BF16>
__device__ __forceinline__ bool pa_nonfinite(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}
// zeros in place of infinities and NaN; whether there were any
template <bool BF16>
__device__ __forceinline__ bool pa_make_finite(uint4& v) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  if (!(pa_nonfinite<BF16>(v.x) || pa_nonfinite<BF16>(v.y) || pa_nonfinite<BF16>(v.z) || pa_nonfinite<BF16>(v.w))) return false;
  auto fix = [](uint32_t w) { return ((w & e) == e ? 0u : w & 0xffffu) | ((w & (e << 16)) == (e << 16) ? 0u : w & 0xffff0000u); };
  v = make_uint4(fix(v.x), fix(v.y), fix(v.z), fix(v.w));
  return true;
}

// word j of a quarter row of codes (8 or 16 bytes)
__device__ __forceinline__ uint32_t pa_word(const uint4& c, int j) { return j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w; }
__device__ __forceinline__ uint32_t pa_word(const uint2& c, int j) { return j == 0 ? c.x : c.y; }

// ------------------------------------------------------------------- tiles
// A K or V tile in the LDS: rows of GK = D / 8 granules of 16 bytes.  Granule G of
// row r is at slot G ^ f(r).  K: the 16 rows of a fragment read then meet in no bank
// (as 256-byte rows, 64 banks: all of G; as 128-byte rows, two to the 256 bytes,
// r / 2).  V: of a transposing read's four rows, two granules each, no pair meets,
// and neither do the four rows of a write of the 4-bit form, a quarter row a lane.
template <int D>
__device__ __forceinline__ int k_slot(int r, int G) {
  if constexpr (D == 128) return G ^ (r & 15);
  else return G ^ ((r >> 1) & 7);
}
template <int D>
__device__ __forceinline__ int v_slot(int r, int G) {
  if constexpr (D == 128) return G ^ (((r >> 1) & 1) * 5 | (r & 1) << 1 | ((r >> 2) & 1) << 3);
  else return G ^ (((r >> 1) & 3) << 1);
}

// The V^T operand of 32 keys and 16 head-dim columns (block jd), key position 4 b + i
// of lane group g holding key 16 b + 4 g + i, which is where S^T left its score.
template <int D>
__device__ __forceinline__ uint4 v_fragment(const uint4* tile, int key0, int jd, int lane) {
  constexpr int GK = D / 8;
  const int s = lane & 15, r = key0 + 4 * (lane >> 4) + (s >> 2);
  const int G = 2 * jd + ((s & 3) >> 1);
  uint2 w[2];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint2* p = reinterpret_cast<const uint2*>(tile + (r + 16 * b) * GK + v_slot<D>(r + 16 * b, G)) + (s & 1);
    w[b] = __builtin_bit_cast(
        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds_s16x4_t*)(const_cast<uint2*>(p))));
  }
  return make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
}

// Softmax and O^T += V^T P^T of one tile of 16 KC keys for RB blocks of 16 rows;
// sc: the masked scores of keys 16 c + 4 (lane / 16) + i, not yet times `sl2` (scale x
// log2 e, not negative).  With the row's reference m, the largest score times sl2,
// rounded, a weight is 2^(s sl2 - m): one multiply-add and one v_exp.  m's rounding error
// is the same in every weight and in the sum and goes out with the division; from 2^16
// on, where it could carry a weight past the type, the product is rounded first, as m's
// was.  m follows a larger score only when that is more than LAG above it: weights then
// reach 2^LAG, which fp32 sums and 16-bit weights do not mind, and most tiles after a
// row's first few leave the accumulators alone.  (Measured, 8192 tokens of 32 heads of
// 128 over a window of 4096, and 64 requests of up to 8000 tokens in 4 bits: 483 and
// 78.7 us with LAG 0, 474 and 79.4 with 2, 463 and 76.3 with 6.  A row's largest weight
// is 1 with LAG 0, which 16 bits hold exactly; with 6 it is rounded as the others are,
// and the largest error of an output is 1.1 to 1.15 times that of LAG 0.)
template <bool BF16, int D, int KC, int RB>
__device__ __forceinline__ void attend(pa_f32x4_t (&sc)[RB][KC], float sl2, float (&m)[RB], float (&l)[RB],
                                       pa_f32x4_t (&o)[RB][D / 16], const uint4* vt, int lane) {
  constexpr int OJ = D / 16;
  constexpr float LAG = 6.f;
  float mul[RB], ref[RB], sum[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) mx = fmaxf(mx, sc[rb][c][i]);
    mx = lanes4_max(mx) * sl2;
    if (__any(mx - m[rb] > LAG)) {
      const float top = fmaxf(m[rb], mx);
      const float alpha = __builtin_amdgcn_exp2f(m[rb] - (top == -INFINITY ? 0.f : top));
      m[rb] = top;
      l[rb] *= alpha;
#pragma unroll
      for (int j = 0; j < OJ; ++j) o[rb][j] *= alpha;
    }
    ref[rb] = m[rb] == -INFINITY ? 0.f : m[rb];
    mul[rb] = sl2;
    sum[rb] = 0.f;
    if (__any(fabsf(ref[rb]) >= 65536.f)) {
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[rb][c][i] = sc[rb][c][i] * sl2 - ref[rb];
      mul[rb] = 1.f, ref[rb] = 0.f;
    }
  }
  // The weights of the first 32 keys, then their products with V between the weights of
  // the next 32: the matrix core works while the wave computes exponentials.
  auto weight = [&](int rb, int c, int i) {
    sc[rb][c][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[rb][c][i], mul[rb], -ref[rb]));
    sum[rb] += sc[rb][c][i];
  };
  uint4 pf[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) weight(rb, c, i);
#pragma unroll
  for (int h = 0; h < KC / 2; ++h) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      pf[rb] = make_uint4(pa_pack<BF16>(sc[rb][2 * h][0], sc[rb][2 * h][1]),
                          pa_pack<BF16>(sc[rb][2 * h][2], sc[rb][2 * h][3]),
                          pa_pack<BF16>(sc[rb][2 * h + 1][0], sc[rb][2 * h + 1][1]),
                          pa_pack<BF16>(sc[rb][2 * h + 1][2], sc[rb][2 * h + 1][3]));
#pragma unroll
    for (int j = 0; j < OJ; ++j) {
      const uint4 vf = v_fragment<D>(vt, 32 * h, j, lane);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) o[rb][j] = pa_mfma<BF16>(vf, pf[rb], o[rb][j]);
      if (h + 1 < KC / 2) {  // 8 weights of each row block over the OJ steps
#pragma unroll
        for (int w = 8 / OJ * j; w < 8 / OJ * (j + 1); ++w)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) weight(rb, 2 * h + 2 + w / 4, w % 4);
      }
    }
  }
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) l[rb] += sum[rb];
}

// Scores of keys that a row does not see, or that do not exist, to -inf whatever they
// were.  hi: the row's position, lo: the first key of its window.
template <int KC, int RB>
__device__ __forceinline__ void hide(pa_f32x4_t (&sc)[RB][KC], uint64_t exists, int key0, const int32_t (&hi)[RB],
                                     const int32_t (&lo)[RB], int32_t sinks, int lane) {
#pragma unroll
  for (int c = 0; c < KC; ++c) {
    const uint32_t there = static_cast<uint32_t>(exists >> (16 * c)) >> (4 * (lane >> 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int32_t key = key0 + 16 * c + 4 * (lane >> 4) + i;
      const int32_t gone = ((there >> i) & 1) - 1, in = (key - sinks) >> 31;  // all ones: no such key; a sink
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const int32_t hidden = gone | ((hi[rb] - key) >> 31) | (((key - lo[rb]) >> 31) & ~in);
        sc[rb][c][i] = hidden < 0 ? -INFINITY : sc[rb][c][i];
      }
    }
  }
}

// first key of the window of a row at position p
__device__ __forceinline__ int32_t window_from(int32_t p, int32_t window) {
  return window > 0 && p >= window ? p - window + 1 : 0;
}

// Whether rows at positions first .. last see the keys key0 .. key0 + n - 1
// differently: not all of them see all.
__device__ __forceinline__ bool tile_edge(int32_t key0, int n, int32_t first, int32_t last, int32_t window,
                                          int32_t sinks) {
  if (key0 + n - 1 > first) return true;
  return key0 < window_from(last, window) && key0 + n > sinks;
}

// ------------------------------------------------------------------- items
struct Item {
  PagedSeq s;
  int32_t block, chunk, chunks;  // chunks 0: no item
};

__device__ __forceinline__ PagedSeq request(const PagedArgs& a, int32_t b, bool& bad) {
  bad = false;
  if (b >= a.num_seqs) return PagedSeq{0, 0, 0, 0, 0};
  return paged_seq(a.qo_indptr[b], a.qo_indptr[b + 1], a.kv_indptr[b], a.kv_indptr[b + 1], a.last[b], a.tokens,
                   a.num_indices, static_cast<int32_t>(a.ps.d), bad);
}

// the line of the table that the merge reads for a block
__device__ __forceinline__ int4 table_line(const PagedArgs& a, const PagedSeq& s, int32_t block, int32_t chunks, int32_t item) {
  const int32_t group = static_cast<int32_t>(a.group.d), row0 = block * a.shape.bm;
  return make_int4(item, chunks, s.q0 * group + row0, min(a.shape.bm, s.qlen * group - row0));
}

// Item x of the grid, for up to 64 requests: every wave finds it by itself, a request a
// lane.  The sum of the work (the key tiles of all blocks) gives the tiles to an item,
// the running sum of the items the request that owns item x.  An item's first workgroup
// fills its block's line of the table that the merge reads, and workgroups past the last
// item the lines past the last block.
constexpr int32_t PA_INLINE_SEQS = 64;
__device__ __forceinline__ Item locate(const PagedArgs& a, int32_t x, bool writes_table) {
  bool bad;
  const PagedSeq s = request(a, threadIdx.x & 63, bad);
  const PagedSplit sp = paged_split(s, a.shape);
  if (bad && x == 0 && writes_table) flag_status(a.status, BFA_STATUS_INDEX_OOB);
  int32_t per = INT_MAX;
  if (a.split)
    per = paged_per_item(__builtin_amdgcn_readlane(scan_lanes(paged_work(sp, a.shift)), 63), a.shift, a.target, a.least);
  const int32_t chunks = sp.chunks(per), end = scan_lanes(paged_items(sp, per)), start = lane_before(end);
  const uint64_t owner = __ballot(x >= start && x < end);
  const int src = owner ? __builtin_ctzll(owner) : 63;
  auto rd = [&](int32_t v) { return __builtin_amdgcn_readlane(v, src); };
  Item it{};
  if (owner) {
    it.s = PagedSeq{rd(s.q0), rd(s.qlen), rd(s.page0), rd(s.npages), rd(s.kvlen)};
    it.chunks = rd(chunks);
    const int32_t in = x - rd(start);
    it.block = it.chunks > 1 ? in / it.chunks : in;
    it.chunk = in - it.block * it.chunks;
  }
  if (a.split && writes_table) {
    // (read out here, where every lane is active: the compiler may compute what a lane
    // read gives away under the branch that uses it)
    const int32_t bend = scan_lanes(sp.blocks);
    const int32_t at = owner ? rd(lane_before(bend)) + it.block : rd(bend) + (x - rd(end));
    if (threadIdx.x == 0 && it.chunk == 0 && at < a.nblocks)
      a.table[at] = owner ? table_line(a, it.s, it.block, it.chunks, x) : make_int4(0, 0, 0, 0);
  }
  return it;
}

// The same for more requests, by one workgroup ahead of the others: all items, and the
// table, 1024 requests at a time.  (512 requests of one key each: 99 us with the items
// found by every workgroup for itself, a pass of 64 requests after another, 41 so.  One
// pass is cheaper than the launch: 64 requests of one key 8.8 us found inline and 13.4
// planned, one of 4000 keys 12.1 and 16.6, 64 of up to 4000 in a window 181 and 186.)
__global__ __launch_bounds__(1024) void paged_plan_kernel(PagedArgs a) {
  __shared__ int32_t item_end[1024], block_end[1024], wave_sum[2][16];
  const int tid = threadIdx.x, wid = tid >> 6;
  // sum of v over the workgroup up to and with this thread, and over all of it
  auto scan = [&](int32_t v, int k, int32_t& all) {
    int32_t end = scan_lanes(v);
    if ((tid & 63) == 63) wave_sum[k][wid] = end;
    __syncthreads();
    int32_t before = 0;
    all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wid) before = paged_add(before, wave_sum[k][w]);
      all = paged_add(all, wave_sum[k][w]);
    }
    __syncthreads();
    return paged_add(end, before);
  };
  int32_t per = INT_MAX;
  if (a.split) {
    int32_t work = 0, all;
    for (int32_t b = tid; b < a.num_seqs; b += 1024) {
      bool bad;
      work = paged_add(work, paged_work(paged_split(request(a, b, bad), a.shape), a.shift));
    }
    scan(work, 0, all);
    per = paged_per_item(all, a.shift, a.target, a.least);
  }
  int32_t items = 0, blocks = 0;  // of the requests before
  for (int32_t b0 = 0; b0 < a.num_seqs; b0 += 1024) {
    bool bad;
    const PagedSplit sp = paged_split(request(a, b0 + tid, bad), a.shape);
    if (bad) flag_status(a.status, BFA_STATUS_INDEX_OOB);
    int32_t all_items, all_blocks;
    item_end[tid] = scan(paged_items(sp, per), 0, all_items);
    block_end[tid] = scan(sp.blocks, 1, all_blocks);
    __syncthreads();
    for (int32_t x = tid; x < all_items && items + x < a.items; x += 1024) {
      int lo = 0, hi = 1023;  // the first request that ends past x
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (item_end[mid] > x) hi = mid;
        else lo = mid + 1;
      }
      bool ignored;
      const PagedSeq s = request(a, b0 + lo, ignored);
      const int32_t chunks = paged_split(s, a.shape).chunks(per), in = x - (lo ? item_end[lo - 1] : 0);
      const int32_t block = in / chunks, chunk = in - block * chunks;
      a.plan[2 * (items + x)] = make_int4(s.q0, s.qlen, s.page0, s.npages);
      a.plan[2 * (items + x) + 1] = make_int4(s.kvlen, block, chunk, chunks);
      const int32_t at = paged_add(blocks, paged_add(lo ? block_end[lo - 1] : 0, block));
      if (a.split && chunk == 0 && at < a.nblocks) a.table[at] = table_line(a, s, block, chunks, items + x);
    }
    items = paged_add(items, all_items);
    blocks = paged_add(blocks, all_blocks);
    __syncthreads();
  }
  for (int32_t x = items + tid; x < a.items; x += 1024) a.plan[2 * x + 1] = make_int4(0, 0, 0, 0);
  if (a.split)
    for (int32_t at = blocks + tid; at < a.nblocks; at += 1024) a.table[at] = make_int4(0, 0, 0, 0);
}

// (in scalar registers: the compiler does not see by itself that a wave's lanes agree,
// and kept the key loops' counters and branches in vector ones)
__device__ __forceinline__ Item find_item(const PagedArgs& a, int32_t x, bool writes_table) {
  Item it;
  if (!a.plan) {
    it = locate(a, x, writes_table);
  } else {
    const int4 p = a.plan[2 * x], q = a.plan[2 * x + 1];
    it = Item{PagedSeq{p.x, p.y, p.z, p.w, q.x}, q.y, q.z, q.w};
  }
  auto rd = [](int32_t v) { return __builtin_amdgcn_readfirstlane(v); };
  return Item{PagedSeq{rd(it.s.q0), rd(it.s.qlen), rd(it.s.page0), rd(it.s.npages), rd(it.s.kvlen)}, rd(it.block), rd(it.chunk),
              rd(it.chunks)};
}

// The rows of a block: positions and query addresses.
struct Rows {
  int32_t row0, n;            // rows of the request, of the block
  int32_t first, last;        // positions of its first and last row
};
template <int BM>
__device__ __forceinline__ Rows block_rows(const PagedArgs& a, const Item& it) {
  Rows r;
  r.row0 = it.block * BM;
  r.n = min(BM, it.s.qlen * static_cast<int32_t>(a.group.d) - r.row0);
  const int32_t base = it.s.kvlen - it.s.qlen;
  r.first = base + static_cast<int32_t>(a.group.div(r.row0));
  r.last = base + static_cast<int32_t>(a.group.div(r.row0 + r.n - 1));
  return r;
}

// 8 query values, with the scale's sign
__device__ __forceinline__ uint4 query_words(const PagedArgs& a, const uint16_t* p) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  return make_uint4((v.x & a.qand) ^ a.qxor, (v.y & a.qand) ^ a.qxor, (v.z & a.qand) ^ a.qxor, (v.w & a.qand) ^ a.qxor);
}

// Address of a key: offsets of its row in the cache (16-byte units) and, in the
// 4-bit cache, of its scales; ok: the key exists.
struct KeyRow {
  uint32_t off, soff;
  bool ok;
};
__device__ __forceinline__ int32_t key_entry(const PagedArgs& a, const PagedSeq& s, int32_t key) {
  key = max(min(key, s.kvlen - 1), 0);  // (the caller has keys: kvlen > 0)
  return a.indices[s.page0 + static_cast<int32_t>(a.ps.div(key))];
}
template <bool FP4>
__device__ __forceinline__ KeyRow key_row(const PagedArgs& a, const PagedSeq& s, int32_t key, int32_t id) {
  KeyRow r{0, 0, key < s.kvlen};
  const int64_t page = paged_page(id, a.num_pages);
  if (r.ok && page < 0) {
    flag_status(a.status, BFA_STATUS_INDEX_OOB);
    r.ok = false;
  }
  if (r.ok) {
    const uint32_t slot = static_cast<uint32_t>(key) - a.ps.div(key) * a.ps.d;
    r.off = static_cast<uint32_t>(page) * a.c_sp + slot * a.c_ss;
    if constexpr (FP4) r.soff = static_cast<uint32_t>(page) * a.s_sp + slot * a.s_ss;
  }
  return r;
}
// The rows of a key tile.  P16 (the page size is a multiple of 16): 16 keys from a
// multiple of 16 lie on one page, so a lane resolves such a group (lane c group c), and
// a load's address is the group's, in scalar registers, and an offset that the lane
// keeps; otherwise a lane resolves a key, and loads take their rows' offsets from it.
// (It is fewer instructions, 300 in place of 393 on the vector unit per 32 keys of the
// 4-bit decode form, and lets the prefill form stage by DMA: 8192 tokens of 32 heads of
// 128 over a window of 4096 567 -> 464 us, 64 requests of up to 4000 keys 182 -> 175,
// 30 requests of up to 8000 in 4 bits 17.3 -> 15.7.)
template <bool FP4, bool P16, int KT>
struct KeyTile {
  KeyRow kr;
  uint64_t exists;  // of the tile's keys

  static constexpr uint64_t all() { return KT == 64 ? ~uint64_t{0} : (uint64_t{1} << (KT & 63)) - 1; }
  // the page list's entry that this lane resolves; asked for a tile ahead of its use
  static __device__ __forceinline__ int32_t entry(const PagedArgs& a, const PagedSeq& s, int32_t key0, int lane) {
    return key_entry(a, s, key0 + (P16 ? 16 * (lane & (KT / 16 - 1)) : lane & (KT - 1)));
  }
  __device__ __forceinline__ KeyTile(const PagedArgs& a, const PagedSeq& s, int32_t key0, int32_t id, int lane) {
    if constexpr (P16) {
      const int32_t key = key0 + 16 * (lane & (KT / 16 - 1));
      kr = key_row<FP4>(a, s, key, id);
      const uint64_t groups = __ballot(kr.ok || key >= s.kvlen);
      exists = all();
      if ((groups & ((1u << (KT / 16)) - 1)) != (1u << (KT / 16)) - 1) {
#pragma unroll
        for (int c = 0; c < KT / 16; ++c)
          if (!((groups >> c) & 1)) exists &= ~(uint64_t{0xffff} << (16 * c));
      }
      const int32_t left = s.kvlen - key0;
      if (left < KT) exists &= (uint64_t{1} << left) - 1;
    } else {
      kr = key_row<FP4>(a, s, key0 + (lane & (KT - 1)), id);
      exists = __ballot(kr.ok) & all();
    }
  }
  // offset (16-byte units) of row 16 c + base + sub, `sub` the lane's: of the group and
  // the row's own in bytes, or of the row
  __device__ __forceinline__ const uint8_t* row(const uint8_t* p, uint32_t stride, int c, int base, int sub, uint32_t part) const {
    if constexpr (P16) {
      const uint64_t g = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(kr.off), c))) * 16;
      return p + g + static_cast<uint32_t>(base) * stride + (static_cast<uint32_t>(sub) * stride + part);
    } else {
      return p + static_cast<uint64_t>(__shfl(kr.off, 16 * c + base + sub)) * 16 + part;
    }
  }
  __device__ __forceinline__ const uint8_t* scale(const uint8_t* p, uint32_t stride, int c, int sub, uint32_t part) const {
    if constexpr (P16) {
      return p + static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(kr.soff), c)) + (static_cast<uint32_t>(sub) * stride + part);
    } else {
      return p + __shfl(kr.soff, 16 * c + sub) + part;
    }
  }
};
__device__ __forceinline__ uint4 zero_unless(bool ok, const uint4& v) {
  return make_uint4(ok ? v.x : 0u, ok ? v.y : 0u, ok ? v.z : 0u, ok ? v.w : 0u);
}
__device__ __forceinline__ uint2 zero_unless(bool ok, const uint2& v) { return make_uint2(ok ? v.x : 0u, ok ? v.y : 0u); }

// What the tiles i0, i0 + step, .. of a block left out: infinities and NaN of V in tiles
// that some row does not see all of, for the rows that see their key.  Runs only
// where there are any, after the last tile.
template <bool BF16, int D, bool FP4, int KT, int RB>
__device__ __forceinline__ void poison(const PagedArgs& a, const PagedSeq& s, int32_t first, int32_t last, const KeyTiles& kt,
                                       int32_t i0, int32_t i1, int32_t step, uint32_t h, const int32_t (&hi)[RB],
                                       const int32_t (&lo)[RB], pa_f32x4_t (&o)[RB][D / 16], int lane) {
  using E = Elem<BF16 ? BFA_DTYPE_BF16 : BFA_DTYPE_F16>;
  const uint8_t* vbase = a.cache + h * a.c_sh + a.c_skv;
  for (int32_t i = i0; i < i1; i += step) {
    const int32_t key0 = kt.at(i) * KT;
    if (!tile_edge(key0, KT, first, last, a.shape.window, a.sinks)) continue;
    for (int32_t key = key0; key < min(key0 + KT, s.kvlen); ++key) {
      const KeyRow kr = key_row<FP4>(a, s, key, key_entry(a, s, key));
      if (!kr.ok) continue;
      const uint8_t* row = vbase + static_cast<uint64_t>(kr.off) * 16;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        const int d = 16 * j + 4 * (lane >> 4);
        uint2 w;
        if constexpr (FP4) {
          const float f = pa_scale<BF16>(a.scales[h * a.s_sh + a.s_skv + kr.soff + d / 32]);
          const uint4 v = pa_from4<BF16>(*reinterpret_cast<const uint16_t*>(row + d / 2), f);
          w = make_uint2(v.x, v.y);
        } else {
          w = *reinterpret_cast<const uint2*>(row + 2 * d);
        }
        if (!(pa_nonfinite<BF16>(w.x) || pa_nonfinite<BF16>(w.y))) continue;
        const float v[4] = {E::to_f32(static_cast<uint16_t>(w.x & 0xffffu)), E::to_f32(static_cast<uint16_t>(w.x >> 16)),
                            E::to_f32(static_cast<uint16_t>(w.y & 0xffffu)), E::to_f32(static_cast<uint16_t>(w.y >> 16))};
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(fabsf(v[e]) < INFINITY) && key <= hi[rb] && (key >= lo[rb] || key < a.sinks)) o[rb][j][e] += v[e];
      }
    }
  }
}

// ------------------------------------------------------------------ decode
// Blocks of 16 rows, one kv head, 4 waves: wave w takes key tiles w, w + 4, ... of
// the item by itself, with its own running state, and the four meet in the LDS at
// the end.  K fragments go from the cache straight to the registers that the
// product reads; V goes through the wave's own LDS tile, for the transposing reads.
// The page ids of the next tile are asked for during a tile's work; its rows are not
// (a second tile's registers cost more than they hid: the CU's other waves fill the
// wait).  Bound by the cache's bytes: 64 requests of 32 heads of 128 on 8,
// window 4000, 931 MB, in 176 us are 5.3 TB/s, above a large copy's 4.9.  In 4 bits the
// conversions weigh as much: 64 requests of up to 8000 keys, 281 MB, in 72 us, 3.9 TB/s.
template <bool BF16, int D, bool FP4, bool P16>
__global__ __launch_bounds__(256, 3) void paged_decode_kernel(PagedArgs a) {
  constexpr int KT = 32, KC = KT / 16;
  constexpr int GK = D / 8, QJ = D / 32, OJ = D / 16;
  constexpr int VN = FP4 ? KT / 16 : KT * GK / 64;  // V loads of a lane: a quarter row of codes, or a granule
  using Code = std::conditional_t<FP4 && D == 64, uint2, uint4>;  // a quarter row of codes, or a granule
  __shared__ uint4 vbuf[4][KT * GK];
  __shared__ float2 state[4][16];

  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t x = a.heads.div(blockIdx.x), h = blockIdx.x - x * a.hkv;
  const int32_t index = static_cast<int32_t>(x);
  const Item it = find_item(a, index, h == 0);
  if (it.chunks == 0) return;
  const Rows rows = block_rows<16>(a, it);
  const KeyTiles kt = paged_key_tiles(rows.first, rows.last, it.s.kvlen, a.shape);
  const int32_t per = paged_even(kt.count, it.chunks);
  const int32_t i0 = min(it.chunk * per, kt.count), i1 = min(i0 + per, kt.count);

  // this lane's row: its query, as the B operand of S^T, and its position
  uint4 qf[QJ];
  int32_t hi[1], lo[1];
  {
    const uint32_t r = rows.row0 + min(lane & 15, rows.n - 1), t = a.group.div(r);
    const uint16_t* qrow =
        a.q + (it.s.q0 + static_cast<int64_t>(t)) * a.q_st + (h * a.group.d + (r - t * a.group.d)) * a.q_sh;
    // (the 4-bit form's lane holds columns D / 4 (lane / 16) .. of a key, which then
    // are its columns of the query)
#pragma unroll
    for (int j = 0; j < QJ; ++j)
      qf[j] = query_words(a, qrow + (FP4 ? D / 4 * g4 + 8 * j : 32 * j + 8 * g4));
    hi[0] = it.s.kvlen - it.s.qlen + static_cast<int32_t>(t);
    lo[0] = window_from(hi[0], a.shape.window);
  }

  float m[1] = {-INFINITY}, l[1] = {0.f};
  pa_f32x4_t o[1][OJ];
#pragma unroll
  for (int j = 0; j < OJ; ++j) o[0][j] = pa_f32x4_t{};

  const uint8_t* kbase = a.cache + h * a.c_sh;
  const uint8_t* ksc = FP4 ? a.scales + h * a.s_sh : nullptr;
  const uint32_t cstride = a.c_ss * 16;  // of the slots, in bytes
  struct Tile {
    uint4 k[FP4 ? 1 : KC][FP4 ? 1 : QJ];
    Code kc[FP4 ? KC : 1], v[VN];
    uint32_t ks[FP4 ? KC : 1], vs[FP4 ? VN : 1];
  };
  using Keys = KeyTile<FP4, P16, KT>;
  auto entry = [&](int32_t i) { return Keys::entry(a, it.s, kt.at(min(i, kt.count - 1)) * KT, lane); };
  auto issue = [&](const Keys& keys) {
    Tile t;
    if constexpr (FP4) {
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        t.kc[c] = *reinterpret_cast<const Code*>(keys.row(kbase, cstride, c, 0, lane & 15, D / 8 * g4));
        t.ks[c] = *keys.scale(ksc, a.s_ss, c, lane & 15, D / 4 * g4 / 32);
      }
#pragma unroll
      for (int i = 0; i < VN; ++i) {
        t.v[i] = *reinterpret_cast<const Code*>(keys.row(kbase + a.c_skv, cstride, i, 0, lane >> 2, D / 8 * (lane & 3)));
        t.vs[i] = *keys.scale(ksc + a.s_skv, a.s_ss, i, lane >> 2, D / 4 * (lane & 3) / 32);
      }
    } else {
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        const uint8_t* row = keys.row(kbase, cstride, c, 0, lane & 15, 16 * g4);
#pragma unroll
        for (int j = 0; j < QJ; ++j) t.k[c][j] = *reinterpret_cast<const uint4*>(row + 64 * j);
      }
#pragma unroll
      for (int i = 0; i < VN; ++i)
        t.v[i] = *reinterpret_cast<const uint4*>(
            keys.row(kbase + a.c_skv, cstride, 64 / GK * i / 16, 64 / GK * i % 16, lane / GK, 16 * (lane % GK)));
    }
    return t;
  };

  uint4* vt = vbuf[wid];
  bool odd = false;
  int32_t i = i0 + wid;
  if (i < i1) {
    int32_t id = entry(i);
    for (; i < i1; i += 4) {
      const int32_t key0 = kt.at(i) * KT;
      const bool edge = tile_edge(key0, KT, rows.first, rows.last, a.shape.window, a.sinks);
      const int32_t id2 = entry(i + 4);
      const Keys keys(a, it.s, key0, id, lane);
      const Tile cur = issue(keys);
      id = id2;
      // S^T = K Q^T
      pa_f32x4_t sc[1][KC];
#pragma unroll
      for (int c = 0; c < KC; ++c) sc[0][c] = pa_f32x4_t{};
#pragma unroll
      for (int j = 0; j < QJ; ++j)
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if constexpr (FP4) {
            sc[0][c] = pa_mfma<BF16>(pa_from4<BF16>(pa_word(cur.kc[c], j), pa_scale<BF16>(cur.ks[c])), qf[j], sc[0][c]);
          } else {
            sc[0][c] = pa_mfma<BF16>(cur.k[c][j], qf[j], sc[0][c]);
          }
        }
      const bool whole = keys.exists == Keys::all();
      if (edge || !whole) hide<KC, 1>(sc, keys.exists, key0, hi, lo, a.sinks, lane);
      // V -> LDS; rows that do not exist as zeros, since 0 x a NaN would poison the sum,
      // and likewise what is not finite in a tile that some row does not see all of
      __builtin_amdgcn_wave_barrier();
      if constexpr (FP4) {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int r = 16 * i + (lane >> 2);
          Code c = cur.v[i];
          float s = pa_scale<BF16>(cur.vs[i]);
          if (!whole) {
            const bool ok = (keys.exists >> r) & 1;
            c = zero_unless(ok, c);
            s = ok ? s : 1.f;
          }
#pragma unroll
          for (int k = 0; k < QJ; ++k) {
            uint4 x = pa_from4<BF16>(pa_word(c, k), s);
            if (edge) odd |= pa_make_finite<BF16>(x);
            vt[r * GK + v_slot<D>(r, QJ * (lane & 3) + k)] = x;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < VN; ++i) {
          const int r = 64 / GK * i + lane / GK;
          uint4 x = cur.v[i];
          if (!whole) x = zero_unless((keys.exists >> r) & 1, x);
          if (edge) odd |= pa_make_finite<BF16>(x);
          vt[r * GK + v_slot<D>(r, lane % GK)] = x;
        }
      }
      asm volatile("" ::: "memory");  // (one wave's LDS accesses happen in order)
      __builtin_amdgcn_wave_barrier();
      attend<BF16, D, KC, 1>(sc, a.sl2, m, l, o, vt, lane);
      asm volatile("" ::: "memory");
    }
  }

  if (__any(odd)) poison<BF16, D, FP4, KT, 1>(a, it.s, rows.first, rows.last, kt, i0 + wid, i1, 4, h, hi, lo, o, lane);

  // the four waves' states meet: granule G (4 columns) of row r at slot G ^ r
  l[0] = lanes4_sum(l[0]);
  float4* ob = reinterpret_cast<float4*>(vt);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < OJ; ++j)
    ob[(lane & 15) * (D / 4) + ((4 * j + g4) ^ (lane & 15))] = make_float4(o[0][j][0], o[0][j][1], o[0][j][2], o[0][j][3]);
  if (lane < 16) state[wid][lane] = make_float2(m[0], l[0]);
  __syncthreads();
  const int r = tid >> 4;  // 16 lanes a row, D / 16 columns each
  if (r >= rows.n) return;
  float mx = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, state[w][r].x);
  const float ref = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  float4 acc[D / 64] = {};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float2 st = state[w][r];
    const float f = __builtin_amdgcn_exp2f(st.x - ref);
    sum += f * st.y;
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
      const float4 v = reinterpret_cast<const float4*>(vbuf[w])[r * (D / 4) + ((D / 64 * (tid & 15) + c) ^ r)];
      acc[c].x += f * v.x; acc[c].y += f * v.y; acc[c].z += f * v.z; acc[c].w += f * v.w;
    }
  }
  if (it.chunks == 1) {
    const uint32_t rr = rows.row0 + r, t = a.group.div(rr);
    uint16_t* orow = a.out + (it.s.q0 + static_cast<int64_t>(t)) * a.out_st +
                     (h * a.group.d + (rr - t * a.group.d)) * static_cast<int64_t>(D) + D / 16 * (tid & 15);
    const float inv = sum == 0.f ? 0.f : a.oscale / sum;
    if constexpr (D == 128) {
      *reinterpret_cast<uint4*>(orow) =
          make_uint4(pa_pack<BF16>(acc[0].x * inv, acc[0].y * inv), pa_pack<BF16>(acc[0].z * inv, acc[0].w * inv),
                     pa_pack<BF16>(acc[1].x * inv, acc[1].y * inv), pa_pack<BF16>(acc[1].z * inv, acc[1].w * inv));
    } else {
      *reinterpret_cast<uint2*>(orow) =
          make_uint2(pa_pack<BF16>(acc[0].x * inv, acc[0].y * inv), pa_pack<BF16>(acc[0].z * inv, acc[0].w * inv));
    }
  } else {
    const int64_t slot = (static_cast<int64_t>(index) * a.hkv + h) * 16 + r;
    float4* dst = reinterpret_cast<float4*>(a.acc + slot * D) + D / 64 * (tid & 15);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) dst[c] = acc[c];
    if ((tid & 15) == 0) reinterpret_cast<float2*>(a.ml)[slot] = make_float2(mx, sum);
  }
}

// ----------------------------------------------------------------- prefill
// Blocks of 64 RB rows, one kv head, 4 waves of 16 RB rows each over the same key
// tiles of 64, which all of them load into the LDS, two tiles deep: the next one's rows
// are on their way during a tile's matrix work, by DMA where a tile's keys lie on whole
// 16-key pages of 16-bit elements, in registers otherwise.  RB is 2 where there are rows
// for it, since a K or V fragment read from the LDS then feeds two products.  Bound by
// what the waves issue between the products, the softmax above all (85 % of the cycles
// issue, 37 % of them to the matrix cores, no bank conflicts): 8192 tokens of 32 heads of
// 128 on 8, window 4096, 413 GFLOP, in 460 us are 897 TFLOP/s; a large bf16 product has
// 1365.  In 4 bits a tile is converted once a workgroup, on its way to the LDS: 1000
// tokens of 16 heads on 8 over 9000, 70 GFLOP, in 105 us with the join.
template <bool BF16, int D, bool FP4, bool P16, int RB>
__global__ __launch_bounds__(256, 2) void paged_prefill_kernel(PagedArgs a) {
  constexpr int KT = 64, KC = 4, BM = 64 * RB;
  constexpr int GK = D / 8, QJ = D / 32, OJ = D / 16;
  constexpr int NL = FP4 ? 1 : GK / 4;  // rows of a tile that a thread loads (a granule, or a quarter row of codes)
  using Code = std::conditional_t<FP4 && D == 64, uint2, uint4>;
  __shared__ uint4 kbuf[2][KT * GK];
  __shared__ uint4 vbuf[2][KT * GK];

  const int tid = threadIdx.x, lane = tid & 63, g4 = lane >> 4;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t x = a.heads.div(blockIdx.x), h = blockIdx.x - x * a.hkv;
  // the last blocks of a request see the most keys: they go first
  const int32_t grid_items = static_cast<int32_t>(a.heads.div(gridDim.x));
  const int32_t index = grid_items - 1 - static_cast<int32_t>(x);
  const Item it = find_item(a, index, h == 0);
  if (it.chunks == 0) return;
  const Rows rows = block_rows<BM>(a, it);
  const KeyTiles kt = paged_key_tiles(rows.first, rows.last, it.s.kvlen, a.shape);
  const int32_t per = paged_even(kt.count, it.chunks);
  const int32_t i0 = min(it.chunk * per, kt.count), i1 = min(i0 + per, kt.count);

  uint4 qf[RB][QJ];
  int32_t hi[RB], lo[RB];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const uint32_t r = rows.row0 + min(16 * (RB * wid + rb) + (lane & 15), rows.n - 1), t = a.group.div(r);
    const uint16_t* qrow =
        a.q + (it.s.q0 + static_cast<int64_t>(t)) * a.q_st + (h * a.group.d + (r - t * a.group.d)) * a.q_sh;
#pragma unroll
    for (int j = 0; j < QJ; ++j) qf[rb][j] = query_words(a, qrow + 32 * j + 8 * g4);
    hi[rb] = it.s.kvlen - it.s.qlen + static_cast<int32_t>(t);
    lo[rb] = window_from(hi[rb], a.shape.window);
  }
  // positions of this wave's first and last row (a wave without rows repeats the last)
  const int32_t base = it.s.kvlen - it.s.qlen;
  const int32_t wfirst = base + static_cast<int32_t>(a.group.div(rows.row0 + min(16 * RB * wid, rows.n - 1)));
  const int32_t wlast = base + static_cast<int32_t>(a.group.div(rows.row0 + min(16 * RB * wid + 16 * RB - 1, rows.n - 1)));
  const bool idle = 16 * RB * wid >= rows.n;

  float m[RB], l[RB];
  pa_f32x4_t o[RB][OJ];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    m[rb] = -INFINITY;
    l[rb] = 0.f;
#pragma unroll
    for (int j = 0; j < OJ; ++j) o[rb][j] = pa_f32x4_t{};
  }

  // staging: load n takes row 16 c + base + sub of the tile, a wave the rows of one group
  constexpr int WR = FP4 ? 16 : 64 / GK;  // rows of a wave in one load
  const int sub = FP4 ? lane >> 2 : lane / GK, part = FP4 ? lane & 3 : lane % GK;
  auto row0_of = [&](int n) { return WR * wid + 4 * WR * n; };
  const uint8_t* kbase = a.cache + h * a.c_sh;
  const uint8_t* ksc = FP4 ? a.scales + h * a.s_sh : nullptr;
  const uint32_t cstride = a.c_ss * 16;
  using Keys = KeyTile<FP4, P16, KT>;
  // 16-bit rows of P16 pages go to the LDS by DMA, 64 granules in the order of their
  // slots an instruction (a lane fetches the granule that belongs in its slot: f(r) of
  // its row is the same in every load); the others through registers.
  constexpr bool DMA = !FP4 && P16;
  const uint32_t kl = lds_addr(kbuf), vl = lds_addr(vbuf);
  const uint32_t koff = DMA ? sub * cstride + 16 * k_slot<D>(row0_of(0) + sub, part) : 0;
  const uint32_t voff = DMA ? sub * cstride + 16 * v_slot<D>(row0_of(0) + sub, part) : 0;
  struct Tile {
    Code k[NL], v[NL];
    uint32_t ks, vs;
  };
  auto entry = [&](int32_t i) { return Keys::entry(a, it.s, kt.at(min(i, kt.count - 1)) * KT, lane); };
  auto copy = [&](const Keys& keys, int b) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r0 = row0_of(n);
      const uint8_t* p = kbase + static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(keys.kr.off), r0 / 16))) * 16 +
                         static_cast<uint32_t>(r0 % 16) * cstride;
      const uint32_t at = (b * KT + r0) * GK * 16;
      dma16(p, koff, kl + at);
      dma16(p + a.c_skv, voff, vl + at);
    }
  };
  auto issue = [&](const Keys& keys) {
    Tile t;
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r0 = row0_of(n);
      const uint8_t* p = keys.row(kbase, cstride, r0 / 16, r0 % 16, sub, (FP4 ? D / 8 : 16) * part);
      t.k[n] = *reinterpret_cast<const Code*>(p);
      t.v[n] = *reinterpret_cast<const Code*>(p + a.c_skv);
      if constexpr (FP4) {
        const uint8_t* f = keys.scale(ksc, a.s_ss, r0 / 16, sub, D / 4 * part / 32);
        t.ks = *f;
        t.vs = f[a.s_skv];
      }
    }
    return t;
  };
  // a tile into the LDS, rows that do not exist as zeros, and so what is not finite in
  // a V tile that some row does not see all of
  bool odd = false;
  auto store = [&](const Tile& t, int b, uint64_t exists, bool edge) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r = row0_of(n) + sub;
      Code kc = t.k[n], vc = t.v[n];
      float fk = 1.f, fv = 1.f;
      if constexpr (FP4) fk = pa_scale<BF16>(t.ks), fv = pa_scale<BF16>(t.vs);
      if (exists != Keys::all()) {
        const bool ok = (exists >> r) & 1;
        kc = zero_unless(ok, kc), vc = zero_unless(ok, vc);
        fk = ok ? fk : 1.f, fv = ok ? fv : 1.f;
      }
      if constexpr (FP4) {
#pragma unroll
        for (int k = 0; k < QJ; ++k) {
          uint4 xv = pa_from4<BF16>(pa_word(vc, k), fv);
          if (edge) odd |= pa_make_finite<BF16>(xv);
          kbuf[b][r * GK + k_slot<D>(r, QJ * part + k)] = pa_from4<BF16>(pa_word(kc, k), fk);
          vbuf[b][r * GK + v_slot<D>(r, QJ * part + k)] = xv;
        }
      } else {
        if (edge) odd |= pa_make_finite<BF16>(vc);
        kbuf[b][r * GK + k_slot<D>(r, part)] = kc;
        vbuf[b][r * GK + v_slot<D>(r, part)] = vc;
      }
    }
  };
  // the same for a tile that is in the LDS already
  auto mend = [&](int b, uint64_t exists, bool edge) {
#pragma unroll
    for (int n = 0; n < NL; ++n) {
      const int r = row0_of(n) + sub, at = r * GK + part;
      const bool ok = (exists >> r) & 1;
      uint4 v = vbuf[b][at];
      if (!ok) kbuf[b][at] = vbuf[b][at] = make_uint4(0, 0, 0, 0);
      else if (edge && pa_make_finite<BF16>(v)) odd = true, vbuf[b][at] = v;
    }
    __syncthreads();
  };
  // a tile has arrived in buffer b, and every wave is done with the other
  auto arrive = [&](int b, uint64_t exists, bool edge) {
    if constexpr (DMA) {
      wait_vmem();
      __syncthreads();
      if (edge || exists != Keys::all()) mend(b, exists, edge);
    } else {
      __syncthreads();
    }
  };
  auto wg_edge = [&](int32_t i) {
    return tile_edge(kt.at(i) * KT, KT, rows.first, rows.last, a.shape.window, a.sinks);
  };
  if (i0 < i1) {
    uint64_t exists, ahead;
    Tile cur;
    {
      const Keys keys(a, it.s, kt.at(i0) * KT, entry(i0), lane);
      exists = ahead = keys.exists;
      if constexpr (DMA) copy(keys, 0);
      else cur = issue(keys);
    }
    int32_t id = entry(i0 + 1);
    if constexpr (!DMA) store(cur, 0, exists, wg_edge(i0));
    arrive(0, exists, wg_edge(i0));
    for (int32_t i = i0; i < i1; ++i) {
      const int b = (i - i0) & 1;
      const bool more = i + 1 < i1;
      const int32_t id2 = entry(i + 2);
      if (more) {
        const Keys keys(a, it.s, kt.at(i + 1) * KT, id, lane);
        ahead = keys.exists;
        if constexpr (DMA) copy(keys, b ^ 1);
        else cur = issue(keys);
      }
      id = id2;
      const int32_t key0 = kt.at(i) * KT;
      // (a wave skips a tile that none of its rows sees)
      if (!idle && key0 <= wlast && (key0 + KT > window_from(wfirst, a.shape.window) || key0 < a.sinks)) {
        pa_f32x4_t sc[RB][KC];
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int rb = 0; rb < RB; ++rb) sc[rb][c] = pa_f32x4_t{};
#pragma unroll
        for (int j = 0; j < QJ; ++j)
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const int r = 16 * c + (lane & 15);
            const uint4 kf = kbuf[b][r * GK + k_slot<D>(r, 4 * j + g4)];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) sc[rb][c] = pa_mfma<BF16>(kf, qf[rb][j], sc[rb][c]);
          }
        if (tile_edge(key0, KT, wfirst, wlast, a.shape.window, a.sinks) || exists != Keys::all())
          hide<KC, RB>(sc, exists, key0, hi, lo, a.sinks, lane);
        attend<BF16, D, KC, RB>(sc, a.sl2, m, l, o, vbuf[b], lane);
      }
      if (more) {
        if constexpr (!DMA) store(cur, b ^ 1, ahead, wg_edge(i + 1));
        exists = ahead;
        arrive(b ^ 1, exists, wg_edge(i + 1));
      }
    }
    if (__syncthreads_or(odd)) poison<BF16, D, FP4, KT, RB>(a, it.s, rows.first, rows.last, kt, i0, i1, 1, h, hi, lo, o, lane);
  }

#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    l[rb] = lanes4_sum(l[rb]);
    const int r = 16 * (RB * wid + rb) + (lane & 15);
    if (r >= rows.n) continue;
    if (it.chunks == 1) {
      const uint32_t rr = rows.row0 + r, t = a.group.div(rr);
      uint16_t* orow = a.out + (it.s.q0 + static_cast<int64_t>(t)) * a.out_st +
                       (h * a.group.d + (rr - t * a.group.d)) * static_cast<int64_t>(D) + 4 * g4;
      const float inv = l[rb] == 0.f ? 0.f : a.oscale / l[rb];
#pragma unroll
      for (int j = 0; j < OJ; ++j)
        *reinterpret_cast<uint2*>(orow + 16 * j) = make_uint2(pa_pack<BF16>(o[rb][j][0] * inv, o[rb][j][1] * inv),
                                                              pa_pack<BF16>(o[rb][j][2] * inv, o[rb][j][3] * inv));
    } else {
      const int64_t slot = (static_cast<int64_t>(index) * a.hkv + h) * BM + r;
      float4* dst = reinterpret_cast<float4*>(a.acc + slot * D) + g4;
#pragma unroll
      for (int j = 0; j < OJ; ++j) dst[4 * j] = make_float4(o[rb][j][0], o[rb][j][1], o[rb][j][2], o[rb][j][3]);
      if (lane < 16) reinterpret_cast<float2*>(a.ml)[slot] = make_float2(m[rb], l[rb]);
    }
  }
}

// ------------------------------------------------------------------- merge
// Joins the items of each block that has several: a wave takes a row, or up to 16
// items of it at a time where there are more and the workgroup's four waves share the
// row (30000 keys of one request, 128 items: attention and join 42.3 us with a wave a
// row, 35.0 so; 256 items 49 and 38.5); D / 4 lanes have 4 columns each, the 64 /
// (D / 4) groups of lanes every such item, and meet by lane exchanges, the waves in the
// LDS, in one order whatever runs first.
template <bool BF16, int D, int BM>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a) {
  constexpr int L = D / 4, NG = 64 / L;
  __shared__ float4 wacc[4][L];
  __shared__ float wsum[4];
  const uint32_t block = a.heads.div(blockIdx.x), h = blockIdx.x - block * a.hkv;
  const int4 line = a.table[block];
  const int32_t items = line.y, n = line.w;
  if (items <= 1 || !paged_line_inside(line.x, items, line.z, n, a.items, a.tokens * a.group.d, BM)) return;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, sub = lane / L, col = lane % L;
  const bool wide = items > 16;
  const int step_r = (wide ? 1 : 4) * gridDim.y;
  for (int r = wide ? blockIdx.y : blockIdx.y * 4 + wid; r < n; r += step_r) {
    const int64_t slot0 = (static_cast<int64_t>(line.x) * a.hkv + h) * BM + r, step = static_cast<int64_t>(a.hkv) * BM;
    const float2* ml = reinterpret_cast<const float2*>(a.ml) + slot0;
    float mx = -INFINITY;
    for (int z = lane; z < items; z += 64) mx = fmaxf(mx, ml[z * step].x);
    mx = lanes4_max(group16_max_dpp(mx));
    const float ref = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    float4 acc = {};
    auto add = [&](int z0, auto n) {  // the items from z0, n at most
      constexpr int U = decltype(n)::value / NG;
      float2 st[U];
      float4 v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int z = min(z0 + NG * u + sub, items - 1);
        st[u] = ml[z * step];
        v[u] = reinterpret_cast<const float4*>(a.acc + (slot0 + z * step) * D)[col];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (z0 + NG * u + sub >= items) continue;
        const float f = __builtin_amdgcn_exp2f(st[u].x - ref);
        sum += f * st[u].y;
        acc.x += f * v[u].x; acc.y += f * v[u].y; acc.z += f * v[u].z; acc.w += f * v[u].w;
      }
    };
    // (1000 tokens over 9000 in 4 bits, four items a block: 116.7 us with loads for 16, most
    // of them again for the last item, and 110.4 so)
    if (items <= 4) add(0, std::integral_constant<int, 4>{});
    else for (int z0 = wide ? 16 * wid : 0; z0 < items; z0 += wide ? 64 : 16) add(z0, std::integral_constant<int, 16>{});
#pragma unroll
    for (int d = L; d < 64; d *= 2) {
      sum += __shfl_xor(sum, d);
      acc.x += __shfl_xor(acc.x, d); acc.y += __shfl_xor(acc.y, d);
      acc.z += __shfl_xor(acc.z, d); acc.w += __shfl_xor(acc.w, d);
    }
    if (wide) {  // (the same for the whole workgroup)
      if (sub == 0) wacc[wid][col] = acc;
      if (lane == 0) wsum[wid] = sum;
      __syncthreads();
      sum = wsum[0] + wsum[1] + wsum[2] + wsum[3];
      const float4 p = wacc[0][col], q = wacc[1][col], s = wacc[2][col], t = wacc[3][col];
      acc = make_float4(p.x + q.x + s.x + t.x, p.y + q.y + s.y + t.y, p.z + q.z + s.z + t.z, p.w + q.w + s.w + t.w);
      __syncthreads();
    }
    if (sub || (wide && wid)) continue;
    const float inv = sum == 0.f ? 0.f : a.oscale / sum;
    const uint32_t rr = static_cast<uint32_t>(line.z) + r, t = a.group.div(rr);
    uint16_t* orow = a.out + static_cast<int64_t>(t) * a.out_st + (h * a.group.d + (rr - t * a.group.d)) * static_cast<int64_t>(D);
    reinterpret_cast<uint2*>(orow)[col] =
        make_uint2(pa_pack<BF16>(acc.x * inv, acc.y * inv), pa_pack<BF16>(acc.z * inv, acc.w * inv));
  }
}

// -------------------------------------------------------------------- plan
struct PagedPlan {
  int bm, rb;                     // rows of a block; rb 0: the decode form
  PagedShape shape;
  int32_t split, target, least, shift, nblocks, items;
  int64_t acc_bytes, ml_bytes, table_bytes, plan_bytes;
  int64_t total() const { return acc_bytes + ml_bytes + table_bytes + plan_bytes; }
};

// The form follows the rows of an average request and the whole call's work, and the
// items the workgroups that fill the chip; the lengths themselves stay on the device.
static PagedPlan paged_plan(int64_t tokens, int64_t num_seqs, int64_t group, int64_t hkv, int64_t d,
                            int64_t num_indices, int64_t page_size, int64_t window, int64_t sinks) {
  PagedPlan p{};
  const int64_t rows = tokens * group;
  // tiles of 128 rows by 64 keys, over all kv heads, if every request had the average
  const int64_t keys = cdiv(num_indices * page_size, num_seqs), seen = window > 0 ? std::min(keys, window + sinks + 64) : keys;
  const int64_t big = (rows / 128 + num_seqs) * hkv * cdiv(seen, 64);
  // Blocks of 16 rows for requests of as few, and where 128-row blocks would be so few
  // tiles that the chip is not full; of 128 where the work is ample and rows fill them.
  // us with blocks of 16 / 64 / 128 (`big`): a prompt of 100, 16 heads on 8 (32)
  // 9.3 / 9.3 / 11.0; three of 300, window 130 (about 300) 12.8 / 17.9 / 21.8; one of 500, 32 on
  // 8 (1024) 23.7 / 20.9 / 24.8; four of up to 1000, 16 on 8 (about 2000) 34.4 / 32.8 /
  // 39.7; one of 2000, 32 on 8 (16128) 165 / 73.4 / 75.8; 500 tokens over 3000, 32 on 4 of
  // 64 (6016) 59.5 / 46.5 / 43.8; 200 over 6000, 32 on 8 (5264) 111 / 80 / 48.4; 1000 over
  // 9000 in 4 bits, 16 on 8 (18048) 189 / 152 / 112; 8192 tokens 1763 / 702 / 476.
  p.rb = rows <= 16 * num_seqs || big < 600 ? 0 : rows <= 64 * num_seqs || big < 3000 ? 1 : 2;
  const int forced = tuning(BFA_TUNE_PAGED_ROWS);  // planner override
  if (forced == 16 || forced == 64 || forced == 128) p.rb = forced / 64;
  p.bm = p.rb == 0 ? 16 : 64 * p.rb;
  const int64_t kt = p.rb == 0 ? 32 : 64;
  p.shape = paged_shape(p.bm, static_cast<int32_t>(group), static_cast<int32_t>(kt), static_cast<int32_t>(window),
                        static_cast<int32_t>(sinks));
  p.nblocks = static_cast<int32_t>(std::min(rows, rows / p.bm + num_seqs));
  // Key tiles of an item at least: one for each wave of the decode form; 8 of the prefill
  // form, whose split pays for partial sums of 64 rows and more (the prompt of 500 above
  // in blocks of 64: 20.7 us whole, 28.6 split).
  p.least = p.rb == 0 ? 4 : 8;
  const int64_t all = cdiv(num_indices * page_size, kt) + num_seqs;  // key tiles of all requests
  const int64_t most = std::min<int64_t>(all, p.shape.most);        // of a block
  const int64_t work = p.rb == 0 ? std::min(all, p.nblocks * most) : p.nblocks * std::min(most, cdiv(all, num_seqs));
  // Workgroups to aim for.  Decode: about 24 tiles (of one kv head) each, from 640, below
  // which the chip is not full, to 2048, past which partial sums cost more than evenness
  // gains.  us at 512 / 768 / 1024 / 2048 (work x kv heads): one request of 30000 keys
  // (7500) 31 / - / 34.6 / 37.8; 8 of up to 4000 in 4 bits 16.0 / 14.9 / 19.4 / -; 64 of up to
  // 8000 in 4 bits 79.9 / 83.7 / - / 75.8, and 84 at 4096; 64 of up to 16000, window 4000,
  // - / 187 / - / 177.  Prefill: two a CU, which is what its LDS holds; at 256 / 512 / 768 /
  // 1024: 1000 tokens over 9000 in 4 bits 170 / 113 / 135 / 121, 200 over 6000 60.6 / 48.7 /
  // 58.9 / 57.5.
  int64_t wgs = p.rb == 0 ? std::min<int64_t>(std::max<int64_t>(work * hkv / 24, 640), 2048) : 512;
  const int wanted = tuning(BFA_TUNE_PAGED_WG);  // planner override
  if (wanted > 0) wgs = wanted;
  p.target = static_cast<int32_t>(std::max<int64_t>(1, std::min(cdiv(wgs, hkv), work / p.least)));
  // (blocks that are many times the workgroups the chip holds are even as they are)
  p.split = most > p.least && (p.rb == 0 ? p.nblocks * hkv < 8192 : p.nblocks * hkv < 1024);
  if (wanted >= 0) p.split = wanted > 0 && most > p.least;
  p.items = p.nblocks + (p.split ? p.target : 0);
  while (p.nblocks * ((most >> p.shift) + 1) > PAGED_MOST) ++p.shift;
  if (num_seqs > PA_INLINE_SEQS) p.plan_bytes = static_cast<int64_t>(p.items) * 32;
  if (p.split) {
    const int64_t slots = static_cast<int64_t>(p.items) * hkv * p.bm;
    p.acc_bytes = slots * d * 4;
    p.ml_bytes = cdiv(slots * 8, 16) * 16;
    p.table_bytes = static_cast<int64_t>(p.nblocks) * 16;
  }
  return p;
}

static bool paged_head_dim(int64_t d) { return d == 64 || d == 128; }

// what the 32-bit arithmetic of the kernels holds
static int paged_limits(const char* what, int64_t tokens, int64_t num_seqs, int64_t hq, int64_t hkv, int64_t d,
                        int64_t num_indices, int64_t page_size) {
  BFA_REQUIRE(tokens >= 0 && num_seqs >= 0 && hq > 0 && hkv > 0 && num_indices >= 0 && page_size > 0, "%s: bad geometry", what);
  BFA_REQUIRE(hq % hkv == 0, "%s: %lld query heads do not share %lld kv heads evenly", what,
              static_cast<long long>(hq), static_cast<long long>(hkv));
  if (!paged_head_dim(d))
    return set_error(BFA_ERR_UNSUPPORTED, "%s: head_dim %lld (64 or 128)", what, static_cast<long long>(d));
  const int64_t lim = int64_t{1} << 31;
  BFA_REQUIRE(num_seqs < lim / 2 && num_indices < lim && page_size < lim && num_indices * page_size < lim,
              "%s: 2^31 cached tokens or more", what);
  BFA_REQUIRE(tokens < lim && hq < lim && tokens * (hq / hkv) < lim / 2 &&
                  (tokens * (hq / hkv) / 16 + num_seqs + 1024) * hkv < lim / 2,
              "%s: too many query rows", what);
  return BFA_OK;
}

}  // namespace bfa

using namespace bfa;

extern "C" int64_t bfa_paged_attention_workspace_size(int64_t tokens, int64_t num_seqs, int64_t num_q_heads,
                                                      int64_t num_kv_heads, int64_t head_dim, int64_t num_indices,
                                                      int64_t page_size, int64_t window, int64_t sinks, int cache_dtype) {
  if (tokens <= 0 || num_seqs <= 0 ||
      paged_limits("bfa_paged_attention_workspace_size", tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, num_indices,
                   page_size) != BFA_OK)
    return 0;
  return paged_plan(tokens, num_seqs, num_q_heads / num_kv_heads, num_kv_heads, head_dim, num_indices, page_size, window,
                    sinks).total();
}

extern "C" int bfa_paged_attention(
    const void* query, int dtype, int64_t num_tokens, int64_t num_q_heads, int64_t q_stride_token,
    int64_t q_stride_head, const void* cache, int cache_dtype, int64_t num_pages, int64_t num_kv_heads,
    int64_t page_size, int64_t head_dim, int64_t stride_page, int64_t stride_kv, int64_t stride_head,
    int64_t stride_slot, const void* scales, int64_t scale_stride_page, int64_t scale_stride_kv,
    int64_t scale_stride_head, int64_t scale_stride_slot, const int32_t* kv_indices, int64_t num_indices,
    const int32_t* kv_indptr, const int32_t* kv_last_page_len, const int32_t* qo_indptr, int64_t num_seqs,
    float scale, int64_t window, int64_t sinks, void* out, int64_t out_stride_token, void* workspace,
    int64_t workspace_bytes, int32_t* status, void* stream) {
  const char* what = "bfa_paged_attention";
  BFA_REQUIRE(dtype == BFA_DTYPE_BF16 || dtype == BFA_DTYPE_F16, "%s: queries must be bf16 or fp16", what);
  const bool fp4 = cache_dtype == BFA_DTYPE_FP4;
  BFA_REQUIRE(fp4 || cache_dtype == dtype, "%s: the cache must have the queries' dtype, or 4 bits", what);
  const int rc = paged_limits(what, num_tokens, num_seqs, num_q_heads, num_kv_heads, head_dim, num_indices, page_size);
  if (rc != BFA_OK) return rc;
  BFA_REQUIRE(num_pages >= 0 && window >= 0 && sinks >= 0, "%s: negative pages, window or sinks", what);
  const auto pos = [](int64_t a, int64_t b, int64_t c, int64_t d) { return a >= 0 && b >= 0 && c >= 0 && d >= 0; };
  BFA_REQUIRE(pos(stride_page, stride_kv, stride_head, stride_slot) &&
                  (!fp4 || pos(scale_stride_page, scale_stride_kv, scale_stride_head, scale_stride_slot)),
              "%s: negative cache strides", what);
  const int64_t unit = fp4 ? 16 : 8;  // elements (bytes of codes) in 16 bytes
  BFA_REQUIRE(q_stride_token % 8 == 0 && q_stride_head % 8 == 0 && out_stride_token % 8 == 0 &&
                  stride_page % unit == 0 && stride_kv % unit == 0 && stride_head % unit == 0 && stride_slot % unit == 0 &&
                  aligned16(query) && aligned16(cache) && aligned16(out) && aligned16(workspace),
              "%s: tensors must be 16-byte aligned with strides in multiples of 16 bytes", what);
  if (num_tokens == 0 || num_seqs == 0) return BFA_OK;
  BFA_REQUIRE(query && out && qo_indptr && kv_indptr && kv_last_page_len, "%s: null pointer", what);
  BFA_REQUIRE(num_indices == 0 || (kv_indices && cache && (!fp4 || scales) && num_pages > 0), "%s: null cache or page list", what);
  const int64_t span = num_pages > 0 ? (num_pages - 1) * (stride_page / unit) + (page_size - 1) * (stride_slot / unit) : 0;
  const int64_t sspan = fp4 && num_pages > 0 ? (num_pages - 1) * scale_stride_page + (page_size - 1) * scale_stride_slot : 0;
  const int64_t lim32 = int64_t{1} << 32;
  BFA_REQUIRE(num_pages < (int64_t{1} << 31) && stride_page / unit < lim32 && stride_slot / unit < lim32 && span < lim32 &&
                  scale_stride_page < lim32 && scale_stride_slot < lim32 && sspan < lim32,
              "%s: a cache beyond 64 GiB", what);
  const int64_t win = window >= (int64_t{1} << 31) ? 0 : window;  // (wider than any cache: no window)
  const int64_t snk = std::min<int64_t>(sinks, (int64_t{1} << 31) - 1);
  const int64_t group = num_q_heads / num_kv_heads;
  const PagedPlan p = paged_plan(num_tokens, num_seqs, group, num_kv_heads, head_dim, num_indices, page_size, win, snk);
  BFA_REQUIRE(p.items * num_kv_heads < (int64_t{1} << 24), "%s: too many query rows", what);  // (a launch has 2^32 threads)
  BFA_REQUIRE(p.total() == 0 || (workspace && workspace_bytes >= p.total()), "%s: workspace too small", what);

  PagedArgs a{};
  a.q = static_cast<const uint16_t*>(query);
  a.q_st = q_stride_token; a.q_sh = q_stride_head;
  a.cache = static_cast<const uint8_t*>(cache);
  const int64_t bytes = fp4 ? 1 : 2;
  a.c_sp = static_cast<uint32_t>(stride_page / unit); a.c_ss = static_cast<uint32_t>(stride_slot / unit);
  a.c_skv = stride_kv * bytes; a.c_sh = stride_head * bytes;
  a.scales = static_cast<const uint8_t*>(scales);
  a.s_sp = static_cast<uint32_t>(scale_stride_page); a.s_ss = static_cast<uint32_t>(scale_stride_slot);
  a.s_skv = scale_stride_kv; a.s_sh = scale_stride_head;
  a.num_pages = num_pages;
  a.indices = kv_indices; a.num_indices = num_indices;
  a.kv_indptr = kv_indptr; a.last = kv_last_page_len; a.qo_indptr = qo_indptr;
  a.num_seqs = static_cast<int32_t>(num_seqs);
  a.tokens = num_tokens;
  a.hq = static_cast<uint32_t>(num_q_heads); a.hkv = static_cast<uint32_t>(num_kv_heads);
  a.group = FastDiv(static_cast<uint32_t>(group));
  a.ps = FastDiv(static_cast<uint32_t>(page_size));
  a.heads = FastDiv(a.hkv);
  const float back = fp4 && dtype == BFA_DTYPE_F16 ? 16.f : 1.f;
  a.sl2 = scale == 0.f ? 1.f : fabsf(scale * 1.4426950408889634f) * back;
  a.qand = scale == 0.f ? 0u : 0xffffffffu;
  a.qxor = scale < 0.f ? 0x80008000u : 0u;
  a.oscale = back;
  a.shape = p.shape; a.sinks = static_cast<int32_t>(snk);
  a.out = static_cast<uint16_t*>(out); a.out_st = out_stride_token;
  a.split = p.split; a.target = p.target; a.least = p.least; a.shift = p.shift;
  a.nblocks = p.nblocks; a.items = p.items;
  char* ws = static_cast<char*>(workspace);
  a.acc = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(ws + p.acc_bytes);
  a.table = reinterpret_cast<int4*>(ws + p.acc_bytes + p.ml_bytes);
  a.plan = p.plan_bytes ? reinterpret_cast<int4*>(ws + p.acc_bytes + p.ml_bytes + p.table_bytes) : nullptr;
  a.status = status;
  const hipStream_t s = as_stream(stream);
  const dim3 grid(static_cast<unsigned>(p.items * num_kv_heads));
  if (a.plan) hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(1024), 0, s, a);
  const bool p16 = page_size % 16 == 0 && stride_slot / unit < (int64_t{1} << 23) && scale_stride_slot < (int64_t{1} << 27);
  auto launch = [&](auto bf, auto dd, auto four, auto by16) {
    constexpr bool B = decltype(bf)::value, F = decltype(four)::value, P = decltype(by16)::value;
    constexpr int DD = decltype(dd)::value;
    const unsigned blocks = static_cast<unsigned>(p.nblocks * num_kv_heads);
    // Workgroups of the merge over a block's rows, up to one for the four of a pass.  us of
    // attention and join with 8 / 32: 200 tokens over 6000, 56 blocks of 128 rows, 48.7 /
    // 46.1; 1000 over 9000 in 4 bits, 128 blocks, 110.4 / 112.3.
    const unsigned over = std::min(std::max(2048 / blocks, 8u), static_cast<unsigned>(p.bm / 4));
    if (p.rb == 0) {
      hipLaunchKernelGGL((paged_decode_kernel<B, DD, F, P>), grid, dim3(256), 0, s, a);
      if (p.split) hipLaunchKernelGGL((paged_merge_kernel<B, DD, 16>), dim3(blocks, blocks < 512 ? 4 : 1), dim3(256), 0, s, a);
    } else if (p.rb == 1) {
      hipLaunchKernelGGL((paged_prefill_kernel<B, DD, F, P, 1>), grid, dim3(256), 0, s, a);
      if (p.split) hipLaunchKernelGGL((paged_merge_kernel<B, DD, 64>), dim3(blocks, over), dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((paged_prefill_kernel<B, DD, F, P, 2>), grid, dim3(256), 0, s, a);
      if (p.split) hipLaunchKernelGGL((paged_merge_kernel<B, DD, 128>), dim3(blocks, over), dim3(256), 0, s, a);
    }
  };
  auto with_d = [&](auto bf, auto four) {
    auto with_p = [&](auto dd) {
      if (p16) launch(bf, dd, four, std::true_type{}); else launch(bf, dd, four, std::false_type{});
    };
    if (head_dim == 64) with_p(std::integral_constant<int, 64>{}); else with_p(std::integral_constant<int, 128>{});
  };
  if (dtype == BFA_DTYPE_BF16) {
    if (fp4) with_d(std::true_type{}, std::true_type{}); else with_d(std::true_type{}, std::false_type{});
  } else {
    if (fp4) with_d(std::false_type{}, std::true_type{}); else with_d(std::false_type{}, std::false_type{});
  }
  return check_launch(what);
}
