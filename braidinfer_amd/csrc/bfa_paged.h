// How a ragged batch over one paged cache is cut into work: the arithmetic that
// the paged attention kernels (paged_attn.hip) and the batch builder
// (paged_batch.hip) share with the host planner.  No loads and no GPU types here,
// so that it also compiles for the host, where every path is tested.
//
// A request s owns query rows [qo_indptr[s], qo_indptr[s+1]) and the page list
// kv_indices[kv_indptr[s] .. kv_indptr[s+1]), whose last page holds
// kv_last_page_len[s] tokens.  Its queries are its last tokens: row i of it stands
// at position kv_len - q_len + i and sees key j if j <= position and, with a
// window of W tokens and S sinks, position - j < W or j < S.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define BFA_HD __host__ __device__ __forceinline__
#else
#define BFA_HD inline
#endif

namespace bfa {

struct PagedSeq {
  int32_t q0, qlen;       // first query row, rows
  int32_t page0, npages;  // first entry of the page list, entries
  int32_t kvlen;          // tokens in the cache, the queries' own among them
};

// Request from its offsets; `bad` is set, and the request emptied or cut to what
// is there, where they do not lie inside the arrays.  tokens, num_indices: rows of
// the query tensor and entries of kv_indices (num_indices * page_size < 2^31).
BFA_HD PagedSeq paged_seq(int32_t qo0, int32_t qo1, int32_t kv0, int32_t kv1, int32_t last, int64_t tokens,
                          int64_t num_indices, int32_t page_size, bool& bad) {
  PagedSeq s{0, 0, 0, 0, 0};
  bad = false;
  if (qo0 < 0 || qo1 < qo0 || qo1 > tokens) bad = true;
  else { s.q0 = qo0; s.qlen = qo1 - qo0; }
  if (kv0 < 0 || kv1 < kv0 || kv1 > num_indices) bad = true;
  else { s.page0 = kv0; s.npages = kv1 - kv0; }
  if (s.npages > 0) {
    if (last < 0 || last > page_size) bad = true;
    last = last < 0 ? 0 : last > page_size ? page_size : last;
    s.kvlen = (s.npages - 1) * page_size + last;
  }
  return s;
}

// Page id of the cache from an entry of the page list: negative ids count from the
// end, as a torch index does; -1 if there is no such page.
BFA_HD int64_t paged_page(int64_t id, int64_t num_pages) {
  if (id < 0) id += num_pages;
  return id >= 0 && id < num_pages ? id : -1;
}

// The key tiles (of `tile` keys) that any row at positions first .. last sees, in
// order: `sinks` tiles from the front, then those from tile `from` on; count in all.
struct KeyTiles {
  int32_t sinks, from, count;
  BFA_HD int32_t at(int32_t i) const { return i < sinks ? i : from + (i - sinks); }
};

// window: 0 for none.  first and last may be negative (rows before the cache's
// first token, which see nothing).
BFA_HD KeyTiles paged_key_tiles(int32_t first, int32_t last, int32_t kvlen, int32_t window, int32_t sinks,
                                int32_t tile) {
  KeyTiles k{0, 0, 0};
  if (last >= kvlen) last = kvlen - 1;
  if (last < 0) return k;
  const int32_t all = last / tile + 1;
  if (window > 0 && first >= window) {
    k.from = (first - window + 1) / tile;
    const int32_t s = sinks / tile + (sinks % tile != 0);
    k.sinks = s < k.from ? s : k.from;
  }
  k.count = k.sinks + all - k.from;
  return k;
}

// Work items.  Request s has `blocks` blocks of `bm` rows (a row is a query token
// and one of the `group` heads of a kv head), each over at most `tiles` key tiles;
// with `per` key tiles to an item a block takes ceil(tiles / per) items.
struct PagedSplit {
  int32_t blocks, tiles;
  BFA_HD int32_t chunks(int32_t per) const { return tiles > 0 ? (tiles - 1) / per + 1 : 1; }
};

BFA_HD PagedSplit paged_split(const PagedSeq& s, int32_t group, int32_t bm, int32_t window, int32_t sinks,
                              int32_t tile) {
  PagedSplit p{0, 0};
  const int64_t rows = static_cast<int64_t>(s.qlen) * group;
  p.blocks = static_cast<int32_t>((rows + bm - 1) / bm);
  const int32_t first = s.kvlen - s.qlen;
  p.tiles = paged_key_tiles(first, s.kvlen - 1, s.kvlen, window, sinks, tile).count;
  if (window > 0) {
    // one block's rows lie within ceil(bm / group) + 1 tokens: its window's keys
    // within that many more, on one more tile than they fill, and the sinks' tiles
    const int64_t keys = static_cast<int64_t>(window) + bm / group + 2;
    const int64_t most = keys / tile + 2 + sinks / tile + 1;
    if (most < p.tiles) p.tiles = static_cast<int32_t>(most);
  }
  return p;
}

// Key tiles to an item, so that `total` tiles (the sum of blocks * tiles) make at
// most `target` items beside one for each block; at least `least`.
BFA_HD int32_t paged_per_item(int64_t total, int32_t target, int32_t least) {
  const int64_t per = (total + target - 1) / target;
  return per < least ? least : static_cast<int32_t>(per > 0x3fffffff ? 0x3fffffff : per);
}

// Key tiles of each of a block's `chunks` items, so that they are alike: with `per`
// tiles to the first and what is left to the last, the last would often be short.
BFA_HD int32_t paged_even(int32_t tiles, int32_t chunks) {
  return chunks > 1 ? tiles / chunks + (tiles % chunks != 0) : tiles;
}

}  // namespace bfa
