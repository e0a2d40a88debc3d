// A step's batch from its requests' lengths, on gfx950: the page lists in CSR form,
// the offsets of the new tokens, and each token's request, position and cache slot
// (what build_paged_kv_indices, kernels/kv_cache_utils.py:81-118, and the page
// manager's loops around it, engine/page_manager.py:159-218, build on the host).
//
//   kv_indptr[b + 1] = sum over c <= b of ceil(seq_c / page_size), qo_indptr of query_c
//   kv_indices[kv_indptr[b] + j] = page_tables[b, j]
//   token qo_indptr[b] + i: request b, position p = seq_b - query_b + i,
//   slot page_tables[b, p / page_size] * page_size + p % page_size
//
// A workgroup owns a request (or, over grid.y, a part of a long one).  It sums the
// lengths of the requests before it and of all by itself, which takes one pass over
// B lengths from the L2, and so the whole batch is one launch and no workgroup waits
// for another.  Bound by that latency: two dependent reads and the writes.
#include "bfa_device.h"
#include "bfa_host.h"
#include "bfa_paged_scan.h"

namespace bfa {

struct BatchArgs {
  const void* tables;  // [num_seqs, max_pages], row stride
  int64_t table_stride;
  int64_t max_pages;
  const void* seq;
  const void* query;
  int tables_i64, seq_i64, query_i64;
  int64_t num_seqs, page_size, num_tokens, num_indices;
  int32_t* qo_indptr;
  int32_t* kv_indptr;
  int32_t* kv_indices;
  int32_t* last;
  int32_t* batch;
  int64_t* positions;
  int64_t* slots;
  int* status;
};

__device__ __forceinline__ int64_t load_int(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// A request's lengths, cut to what its page table holds; `bad` where that cut them
// or a token has no place.
struct Lengths {
  int64_t seq, query, held, pages;  // as given (not negative); tokens that have a page, pages
};
__device__ __forceinline__ Lengths request_lengths(const BatchArgs& a, int64_t b, bool& bad) {
  Lengths l;
  l.seq = load_int(a.seq, a.seq_i64, b);
  l.query = load_int(a.query, a.query_i64, b);
  const int64_t room = a.max_pages * a.page_size;
  bad = l.seq < 0 || l.query < 0 || l.seq > room || l.query > l.seq;
  l.seq = max(l.seq, static_cast<int64_t>(0));
  l.query = max(l.query, static_cast<int64_t>(0));
  l.held = min(l.seq, room);
  l.pages = (l.held + a.page_size - 1) / a.page_size;
  return l;
}

__global__ __launch_bounds__(256) void paged_batch_kernel(BatchArgs a) {
  __shared__ int32_t part[4][4];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  // pages and queries before b, and of all, held at 2^30 - 1 (there is room for fewer)
  int32_t sum[4] = {0, 0, 0, 0};
  for (int64_t c = tid; c < a.num_seqs; c += 256) {
    bool bad;
    const Lengths l = request_lengths(a, c, bad);
    const int32_t pages = static_cast<int32_t>(min<int64_t>(l.pages, PAGED_MOST));
    const int32_t query = static_cast<int32_t>(min<int64_t>(l.query, PAGED_MOST));
    sum[2] = paged_add(sum[2], pages);
    sum[3] = paged_add(sum[3], query);
    if (c < b) {
      sum[0] = paged_add(sum[0], pages);
      sum[1] = paged_add(sum[1], query);
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    sum[k] = sum_lanes(sum[k]);
    if ((tid & 63) == 0) part[tid >> 6][k] = sum[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) sum[k] = paged_add(paged_add(part[0][k], part[1][k]), paged_add(part[2][k], part[3][k]));
  const int64_t page0 = sum[0], token0 = sum[1], all_pages = sum[2], all_tokens = sum[3];
  const int64_t nt = static_cast<int64_t>(gridDim.y) * 256, first = static_cast<int64_t>(blockIdx.y) * 256 + tid;
  if (b < a.num_seqs) {
    bool bad;
    const Lengths l = request_lengths(a, b, bad);
    if (first == 0) {
      if (b == 0) a.qo_indptr[0] = a.kv_indptr[0] = 0;
      a.kv_indptr[b + 1] = static_cast<int32_t>(min(page0 + l.pages, a.num_indices));
      a.qo_indptr[b + 1] = static_cast<int32_t>(min(token0 + l.query, a.num_tokens));
      a.last[b] = l.pages > 0 ? static_cast<int32_t>(l.held - (l.pages - 1) * a.page_size) : 0;
      if (bad || page0 + l.pages > a.num_indices || token0 + l.query > a.num_tokens)
        flag_status(a.status, BFA_STATUS_INDEX_OOB);
    }
    const int64_t row = b * a.table_stride;
    for (int64_t j = first; j < min(l.pages, a.num_indices - page0); j += nt)
      a.kv_indices[page0 + j] = static_cast<int32_t>(load_int(a.tables, a.tables_i64, row + j));
    const bool narrow = static_cast<uint64_t>(l.seq | a.page_size) >> 32 == 0;
    for (int64_t i = first; i < min(l.query, a.num_tokens - token0); i += nt) {
      const int64_t p = l.seq - l.query + i;
      int64_t slot = -1;
      if (p >= 0 && p < l.held) {
        // (a 32-bit division where the operands allow it)
        const int64_t page = narrow ? static_cast<int64_t>(static_cast<uint32_t>(p) / static_cast<uint32_t>(a.page_size))
                                    : p / a.page_size;
        slot = load_int(a.tables, a.tables_i64, row + page) * a.page_size + (p - page * a.page_size);
      }
      a.batch[token0 + i] = static_cast<int32_t>(b);
      a.positions[token0 + i] = p;
      a.slots[token0 + i] = slot;
    }
  } else if (first == 0 && b == 0) {  // no requests
    a.qo_indptr[0] = a.kv_indptr[0] = 0;
  }
  // what is behind the last request
  const int64_t wg = static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x, all = nt * gridDim.x;
  for (int64_t j = all_pages + wg * 256 + tid; j < a.num_indices; j += all) a.kv_indices[j] = -1;
  for (int64_t i = all_tokens + wg * 256 + tid; i < a.num_tokens; i += all) {
    a.batch[i] = -1;
    a.positions[i] = -1;
    a.slots[i] = -1;
  }
}

}  // namespace bfa

using namespace bfa;

extern "C" int bfa_build_paged_kv_batch(const void* page_tables, int page_tables_dtype, int64_t num_seqs,
                                        int64_t max_pages, int64_t page_table_stride, const void* seq_lens,
                                        int seq_lens_dtype, const void* query_lens, int query_lens_dtype,
                                        int64_t page_size, int64_t num_tokens, int64_t num_indices,
                                        int32_t* qo_indptr, int32_t* kv_indptr, int32_t* kv_indices,
                                        int32_t* kv_last_page_len, int32_t* batch_indices, int64_t* positions,
                                        int64_t* slot_mapping, int32_t* status, void* stream) {
  const char* what = "bfa_build_paged_kv_batch";
  const auto is_int = [](int dt) { return dt == BFA_DTYPE_I32 || dt == BFA_DTYPE_I64; };
  BFA_REQUIRE(is_int(page_tables_dtype) && is_int(seq_lens_dtype) && is_int(query_lens_dtype),
              "%s: page tables and lengths must be int32/int64", what);
  const int64_t lim = int64_t{1} << 31;
  BFA_REQUIRE(num_seqs >= 0 && max_pages >= 0 && num_tokens >= 0 && num_indices >= 0 && page_table_stride >= 0, "%s: bad geometry", what);
  BFA_REQUIRE(page_size > 0, "%s: page_size must be positive", what);
  BFA_REQUIRE(num_seqs < lim / 2 && num_tokens < lim / 2 && num_indices < lim / 2 && max_pages < lim && page_size < lim,
              "%s: 2^30 requests, pages or tokens or more", what);
  BFA_REQUIRE(num_seqs < (int64_t{1} << 24), "%s: 2^24 requests or more", what);  // (a launch has 2^32 threads)
  BFA_REQUIRE(qo_indptr && kv_indptr, "%s: null pointer", what);
  BFA_REQUIRE(num_seqs == 0 || (seq_lens && query_lens && kv_last_page_len && (max_pages == 0 || page_tables)), "%s: null pointer", what);
  BFA_REQUIRE((num_indices == 0 || kv_indices) && (num_tokens == 0 || (batch_indices && positions && slot_mapping)),
              "%s: null output", what);
  BatchArgs a{};
  a.tables = page_tables; a.table_stride = page_table_stride; a.max_pages = max_pages;
  a.seq = seq_lens; a.query = query_lens;
  a.tables_i64 = page_tables_dtype == BFA_DTYPE_I64;
  a.seq_i64 = seq_lens_dtype == BFA_DTYPE_I64;
  a.query_i64 = query_lens_dtype == BFA_DTYPE_I64;
  a.num_seqs = num_seqs; a.page_size = page_size; a.num_tokens = num_tokens; a.num_indices = num_indices;
  a.qo_indptr = qo_indptr; a.kv_indptr = kv_indptr; a.kv_indices = kv_indices; a.last = kv_last_page_len;
  a.batch = batch_indices; a.positions = positions; a.slots = slot_mapping;
  a.status = status;
  // 4 entries of a page table and 2 tokens a thread at most, at 64 parts of a request at most
  const int64_t seqs = std::max<int64_t>(num_seqs, 1);
  const int64_t parts = std::max(cdiv(max_pages, 1024), cdiv(num_tokens, seqs * 512));
  const dim3 grid(static_cast<unsigned>(seqs), static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(parts, 1), 64)));
  hipLaunchKernelGGL(paged_batch_kernel, grid, dim3(256), 0, as_stream(stream), a);
  return check_launch(what);
}
