// Attention over a key/value cache kept in pages (flash_paged.hip) and eviction from such a cache
// (flash_evict.hip): parameter blocks and the index arithmetic both share.
#pragma once
#include "flash_common.h"

namespace fa {

// Row `key` of sequence `bi` of a cache: row key % page of page table[bi][key / page].  A cache
// without a table (max_pages == 0) is dense: sequence bi is page bi.
struct Pages {
  const int *table;      // [b, max_pages]; null: dense
  int num_pages, page, max_pages;
  uint32_t mul;          // key / page = (key * mul) >> shift for every key < 2^31
  int shift;
  int64_t k_ps, k_rs, k_hs, v_ps, v_rs, v_hs;  // page, row and head strides (elements)
  FA_HD int capacity() const { return max_pages ? max_pages * page : page; }
  // the place of a key in the sequence's row of the table, and the key's row on that page
  __device__ __forceinline__ int index(int key, int &row) const {
    const int at = (int)(((uint64_t)(uint32_t)key * mul) >> shift);
    row = key - at * page;
    return at;
  }
  // a number names a page when it lies inside the pool
  __device__ __forceinline__ bool present(int pg) const { return (unsigned)pg < (unsigned)num_pages; }
  // page of a key and its row there; -1: the page is absent
  __device__ __forceinline__ int locate(int bi, int key, int &row) const {
    if (!max_pages) { row = key; return bi; }
    const int pg = table[(int64_t)bi * max_pages + index(key, row)];
    return present(pg) ? pg : -1;
  }
};
// mul, shift of a page size: mul = ceil(2^shift / page) < 2^32 with shift = 31 + ceil(log2 page),
// so key * mul / 2^shift exceeds key / page by less than key / 2^31 / page < 1 / page
inline void set_page(Pages &p, int page) {
  int log = 0;
  while ((int64_t(1) << log) < page) ++log;
  p.page = page;
  p.shift = 31 + log;
  p.mul = (uint32_t)(((uint64_t(1) << p.shift) + page - 1) / page);
}

struct PagedParams {
  const void *q, *k, *v, *k_new, *v_new;  // the caches are written when k_new is given
  void *o;
  float *lse;                // [b, h, sq]
  const int *seqlens;        // [b] keys in the cache before the call; < 0: the sequence is idle; null: the capacity
  const float *w_in;         // [b, h_k, capacity]; null: from zero
  float *w_out;              // null: no weights
  Pages pages;
  int64_t q_bs, q_rs, q_hs, o_bs, o_rs, o_hs, kn_bs, kn_rs, kn_hs, vn_bs, vn_rs, vn_hs;
  int b, h, h_k, d, sq, n_new;
  float scale, scale_log2;
  int wl, wr, n_sink;
  int fuse_append;           // 1: the attention kernel writes the new rows itself
  int n_ct;                  // tiles of 32 columns (query head of the group x query row)
  int max_units;             // most 32-key units a column tile can visit
  int n_splits, min_units;   // workgroups that share a tile's units, fewest units of one
  // What one launch computes: column tiles [tile0, tile0 + n_tiles), numbered through (sequence, key/value head,
  // tile), whose rows ((sequence * h + head) * sq + query row) are [row0, row0 + n_rows).  All of them, unless
  // the scores of all would take more than kScoreBytes.
  int tile0, n_tiles;
  int64_t row0, n_rows;
  float *o_part, *ml_part;   // [n_splits][n_rows][tile width], [n_splits][n_rows][2]; null: n_splits == 1
  float *s_part;             // [n_rows][max_units * 32] scores, for the weights
  void *ws;
  size_t ws_bytes;
  size_t *ws_query;

  // keys of sequence bi after the call
  __device__ __forceinline__ int keys_of(int bi) const {
    if (!seqlens) return pages.capacity();
    const int n = seqlens[bi];
    return n < 0 ? 0 : (int)min((int64_t)n + n_new, (int64_t)pages.capacity());
  }
  // the units that column tile ct of a sequence with sk keys visits
  FA_HD idx::SinkTiles units(int sk, int ct) const {
    const int c0 = ct * 32, c1 = c0 + 31 < h / h_k * sq ? c0 + 31 : h / h_k * sq - 1;
    const bool one = c0 / sq == c1 / sq;  // the tile lies within one head
    const int r0 = one ? c0 % sq : 0, r1 = one ? c1 % sq : sq - 1;
    return idx::sink_tile_range(sq, sk, wl, wr, n_sink, r0, r1 - r0 + 1, 32);
  }
  // units of one split, and how many splits have any (split 0 always writes its partials)
  FA_HD int per_split(int n_units) const {
    const int even = (n_units + n_splits - 1) / n_splits;
    return ((even > min_units ? even : min_units) + 3) & ~3;
  }
};
hipError_t launch_paged(PagedParams &p, int dtype, hipStream_t stream);

struct EvictParams {
  const void *k, *v;
  void *k_out, *v_out;
  const float *w;            // [b, h_k, capacity of `from`]
  float *w_out;              // [b, h_k, capacity of `to`]
  const int *seqlens;        // [b]
  int *seqlens_out, *kept;   // [b], [b, h_k, budget]
  Pages from, to;
  int b, h_k, d, budget, n_sink, n_recent;
  int in_place;              // the caches are the same memory
};
// in place: workgroups (of 1024 threads) of one (sequence, head): slices of kEvictCols 16-byte columns of K and of
// V, and the weights
constexpr int kEvictCols = 4;
inline int evict_groups(int d) { return 2 * ((d / 8 + kEvictCols - 1) / kEvictCols) + 1; }
hipError_t launch_evict(const EvictParams &p, hipStream_t stream);

}  // namespace fa
