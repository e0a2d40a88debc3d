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

// What the cut depends on beside the lengths: `bm` rows to a block (a row is a query
// token and one of the `group` heads of a kv head), `tile` keys to a tile (a power of
// two), the window (0 for none) and the sinks, in whole tiles.
struct PagedShape {
  int32_t bm, group, tile;
  int32_t window, sink_tiles;
  int32_t most;  // bound of a block's key tiles from its window
};

BFA_HD PagedShape paged_shape(int32_t bm, int32_t group, int32_t tile, int32_t window, int32_t sinks) {
  PagedShape p{bm, group, tile, window, 0, 0x7fffffff};
  p.sink_tiles = sinks / tile + (sinks % tile != 0);
  if (window > 0) {
    // one block's rows lie within (bm - 1) / group + 2 tokens: its window's keys within
    // that many more, on two tiles more than they fill, and the sinks' tiles
    const int64_t keys = static_cast<int64_t>(window) + bm / group + 2;
    const int64_t most = keys / tile + 2 + p.sink_tiles;
    if (most < p.most) p.most = static_cast<int32_t>(most);
  }
  return p;
}

// The key tiles that any row at positions first .. last sees, in order: `sinks` tiles
// from the front, then those from tile `from` on; count in all.
struct KeyTiles {
  int32_t sinks, from, count;
  BFA_HD int32_t at(int32_t i) const { return i < sinks ? i : from + (i - sinks); }
};

// first and last may be negative (rows before the cache's first token, which see
// nothing).
BFA_HD KeyTiles paged_key_tiles(int32_t first, int32_t last, int32_t kvlen, const PagedShape& p) {
  KeyTiles k{0, 0, 0};
  if (last >= kvlen) last = kvlen - 1;
  if (last < 0) return k;
  const uint32_t tile = static_cast<uint32_t>(p.tile);
  const int32_t all = static_cast<int32_t>(static_cast<uint32_t>(last) / tile) + 1;
  if (p.window > 0 && first >= p.window) {
    k.from = static_cast<int32_t>(static_cast<uint32_t>(first - p.window + 1) / tile);
    k.sinks = p.sink_tiles < k.from ? p.sink_tiles : k.from;
  }
  k.count = k.sinks + all - k.from;
  return k;
}

// Work items.  Request s has `blocks` blocks of rows, each over at most `tiles` key
// tiles; with `per` key tiles to an item a block takes ceil(tiles / per) items.
struct PagedSplit {
  int32_t blocks, tiles;
  BFA_HD int32_t chunks(int32_t per) const {
    return tiles > per ? static_cast<int32_t>((static_cast<uint32_t>(tiles) - 1) / static_cast<uint32_t>(per)) + 1 : 1;
  }
};

BFA_HD PagedSplit paged_split(const PagedSeq& s, const PagedShape& p) {
  PagedSplit sp{0, 0};
  const uint32_t rows = static_cast<uint32_t>(s.qlen) * static_cast<uint32_t>(p.group);  // < 2^30 (checked by the caller)
  sp.blocks = static_cast<int32_t>((rows + p.bm - 1) / static_cast<uint32_t>(p.bm));
  sp.tiles = paged_key_tiles(s.kvlen - s.qlen, s.kvlen - 1, s.kvlen, p).count;
  if (sp.tiles > p.most) sp.tiles = p.most;
  return sp;
}

// Work is summed in units of 2^shift key tiles, rounded up, so that the sum of all
// requests stays below 2^30; sums are held there, which only broken offsets (whose
// requests overlap) can reach.
constexpr int32_t PAGED_MOST = 0x3fffffff;
BFA_HD int32_t paged_work(const PagedSplit& s, int32_t shift) {
  const int64_t w = static_cast<int64_t>(s.blocks) * (s.tiles > 0 ? ((s.tiles - 1) >> shift) + 1 : 0);
  return w > PAGED_MOST ? PAGED_MOST : static_cast<int32_t>(w);
}

// Key tiles to an item, so that `work` units make at most `target` items beside one for
// each block; at least `least`.
BFA_HD int32_t paged_per_item(int32_t work, int32_t shift, int32_t target, int32_t least) {
  const uint32_t units = (static_cast<uint32_t>(work) + target - 1) / static_cast<uint32_t>(target);
  const int64_t per = static_cast<int64_t>(units) << shift;
  return per < least ? least : static_cast<int32_t>(per > PAGED_MOST ? PAGED_MOST : per);
}

// Items of a request, held likewise.
BFA_HD int32_t paged_items(const PagedSplit& s, int32_t per) {
  const int64_t n = static_cast<int64_t>(s.blocks) * s.chunks(per);
  return n > PAGED_MOST ? PAGED_MOST : static_cast<int32_t>(n);
}
BFA_HD int32_t paged_add(int32_t a, int32_t b) {  // of values up to PAGED_MOST
  return a + b > PAGED_MOST ? PAGED_MOST : a + b;
}

// Whether a block's line of the merge's table, its first item, items, first query row
// and rows, lies inside what there is.  Every block's does, unless broken offsets, whose
// requests overlap, make more items than the grid has: then no item may have filled it.
BFA_HD bool paged_line_inside(int32_t item, int32_t items, int32_t row0, int32_t n, int32_t all_items, int64_t rows,
                              int32_t bm) {
  return item >= 0 && items >= 0 && n >= 0 && row0 >= 0 && items <= all_items - item && n <= bm &&
         static_cast<int64_t>(row0) + n <= rows;
}

// Key tiles of each of a block's `chunks` items, so that they are alike: with `per`
// tiles to the first and what is left to the last, the last would often be short.
BFA_HD int32_t paged_even(int32_t tiles, int32_t chunks) {
  return chunks > 1 ? tiles / chunks + (tiles % chunks != 0) : tiles;
}

}  // namespace bfa
