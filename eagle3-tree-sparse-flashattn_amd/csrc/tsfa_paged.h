// Sequences of different lengths over a paged K/V pool: what the append and
// the varlen attention share, and the attention's cut of its work.  Lengths
// live on the device (no host reads them), so every value is brought into
// range here before it addresses anything.  Plain C++: the cut is tested on
// the host as well.
#pragma once

#include <stdint.h>

#include "tsfa_plan.h"

namespace tsfa {
namespace paged {

constexpr int kMaxKeys = 1 << 30;  // keys of one sequence (kv_lens beyond are cut)

// The lengths and page lists of a call.  Sequence b owns query rows
// [q_indptr[b], q_indptr[b + 1]) and keys 0 .. kv_lens[b] - 1, key j at row
// j % page_size of the page list[j / page_size]; its list is
// kv_indices[kv_indptr[b] .. kv_indptr[b + 1]) or, without kv_indptr, the
// pt_width entries at kv_indices[b * pt_stride].
struct Seqs {
  const int32_t* q_indptr;
  const int32_t* kv_lens;
  const int32_t* kv_indptr;
  const int32_t* kv_indices;
  int64_t n_indices, pt_stride;
  int pt_width, page_shift, n_pages, batch, total_q;
};

struct Seq {
  int q0, q_len;   // query rows
  int kv_len;      // keys, at most what the list's pages hold
  int prefix;      // keys before the query tokens' own
  int64_t list;    // first entry of the page list in kv_indices
  int pages;       // entries of the list
};

TSFA_HD inline int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

TSFA_HD inline Seq seq_of(const Seqs& s, int b) {
  Seq r;
  r.q0 = (int)clamp64(s.q_indptr[b], 0, s.total_q);
  r.q_len = (int)clamp64(s.q_indptr[b + 1], r.q0, s.total_q) - r.q0;
  if (s.kv_indptr != nullptr) {
    r.list = clamp64(s.kv_indptr[b], 0, s.n_indices);
    r.pages = (int)(clamp64(s.kv_indptr[b + 1], r.list, s.n_indices) - r.list);
  } else {
    r.list = (int64_t)b * s.pt_stride;
    r.pages = s.pt_width;
  }
  const int64_t held = (int64_t)r.pages << s.page_shift;
  r.kv_len = (int)clamp64(s.kv_lens[b], 0, held < kMaxKeys ? held : kMaxKeys);
  r.prefix = r.kv_len > r.q_len ? r.kv_len - r.q_len : 0;
  return r;
}

// ---------------------------------------------------- the attention's work
// The query rows of one (sequence, kv head) are packed token-major, r = t *
// group + g, and cut into tiles of `rows`; a tile walks its keys in steps of
// `keys`.  All steps of a call, in the order (sequence, kv head, tile, step),
// form one line that is cut into equal runs, one to a workgroup: every
// workgroup gets the same number of steps whatever the lengths are, and at
// most the first and the last tile of a run are shared with its neighbours.
struct Cut {
  int rows, keys;           // tile height, keys of a step
  int group, num_kv_heads;  // query heads per kv head; kv heads
  int causal;               // no mask: a tile stops at its last token's own key
};

TSFA_HD inline int cut_tiles(const Cut& c, const Seq& s) {
  return (int)(((int64_t)s.q_len * c.group + c.rows - 1) / c.rows);
}

// Steps of tile r (at least one: a tile without keys still writes its rows).
TSFA_HD inline int tile_steps(const Cut& c, const Seq& s, int r) {
  int end = s.kv_len;
  if (c.causal) {
    const int64_t t = (((int64_t)r + 1) * c.rows - 1) / c.group;  // the tile's last token
    const int64_t lim = (int64_t)s.prefix + (t < s.q_len ? t + 1 : s.q_len);
    if (lim < end) end = (int)lim;
  }
  const int n = (int)(((int64_t)end + c.keys - 1) / c.keys);
  return n > 0 ? n : 1;
}

// Steps of one kv head of a sequence.
TSFA_HD inline int64_t head_steps(const Cut& c, const Seq& s) {
  const int n = cut_tiles(c, s);
  if (n == 0) return 0;
  if (!c.causal) return (int64_t)n * tile_steps(c, s, 0);
  int64_t sum = 0;
  for (int r = 0; r < n; ++r) sum += tile_steps(c, s, r);
  return sum;
}

// A place on the line: the next step of `tile` of kv head `kvh` of sequence b.
struct Place {
  int b, kvh, tile, step;
  Seq seq;
};

// The place `at` steps into sequence b (at < head_steps * num_kv_heads).
TSFA_HD inline Place place_in_seq(const Cut& c, const Seq& s, int b, int64_t at) {
  Place p;
  p.b = b;
  p.seq = s;
  const int64_t per = head_steps(c, s);
  p.kvh = (int)(at / per);
  int64_t left = at - p.kvh * per;
  if (!c.causal) {
    const int n = tile_steps(c, s, 0);
    p.tile = (int)(left / n);
    p.step = (int)(left - (int64_t)p.tile * n);
    return p;
  }
  p.tile = 0;
  for (int n = tile_steps(c, s, 0); left >= n; n = tile_steps(c, s, ++p.tile)) left -= n;
  p.step = (int)left;
  return p;
}

// The part [from, end) of a tile's steps that runs in one go: its page ids
// (list entries first_page .. first_page + ids - 1) and, with a mask, the
// visibility words of its units from tree_unit on (units of 32 keys, the
// first that needs them) fit the workgroup's LDS tables.
constexpr int kTableIds = 1024;
constexpr int kTreeUnits = 16;
struct Chunk {
  int end, first_page, ids, tree_unit;
};
TSFA_HD inline Chunk chunk_of(const Seq& s, int page_shift, int streams, int from, int last, bool mask) {
  Chunk c;
  c.first_page = (int)(((int64_t)from * (32 * streams)) >> page_shift);
  const int64_t lim = ((int64_t)(c.first_page + kTableIds) << page_shift) / (32 * streams);
  c.end = (int)(lim < last ? lim : last);
  const int u = from * streams;
  c.tree_unit = s.prefix / 32 > u ? s.prefix / 32 : u;
  if (mask && (int64_t)c.end * streams > c.tree_unit + kTreeUnits) c.end = (c.tree_unit + kTreeUnits) / streams;
  const int held = ((s.kv_len - 1) >> page_shift) - c.first_page + 1;
  c.ids = held < kTableIds ? held : kTableIds;
  return c;
}
// First key of the rpl rows that a load takes for keys k0 .. k0 + rpl - 1
// (rpl divides the page size): those, or the ones that hold the last key.
TSFA_HD inline int load_block(int k0, int rpl, int kv_len) {
  const int last = (kv_len - 1) & ~(rpl - 1);
  return k0 < last ? k0 : last;
}

}  // namespace paged

// ------------------------------------------------------- host-side helpers
// Checks of a page pool's description (the pages' size as the paged forward
// takes it; a dense table must hold pt_width entries for every sequence).
inline int paged_check(const int32_t* kv_indptr, int64_t n_indices, int64_t pt_stride, int pt_width, int n_pages,
                       int page_size, int batch) {
  if (n_pages <= 0 || n_indices < 0 || n_indices > INT32_MAX || page_size <= 0) return TSFA_ERR_INVALID_ARGUMENT;
  if (page_size < 16 || (page_size & (page_size - 1)) != 0) return TSFA_ERR_UNSUPPORTED;
  if (kv_indptr == nullptr && batch > 0) {
    if (pt_stride < 0 || pt_width < 0) return TSFA_ERR_INVALID_ARGUMENT;
    if (pt_stride > INT32_MAX || (batch - 1) * pt_stride + pt_width > n_indices) return TSFA_ERR_INVALID_ARGUMENT;
  }
  return TSFA_OK;
}

inline paged::Seqs make_seqs(const int32_t* q_indptr, const int32_t* kv_lens, const int32_t* kv_indptr,
                             const int32_t* kv_indices, int64_t n_indices, int64_t pt_stride, int pt_width,
                             int n_pages, int page_size, int batch, int total_q) {
  paged::Seqs s;
  s.q_indptr = q_indptr;
  s.kv_lens = kv_lens;
  s.kv_indptr = kv_indptr;
  s.kv_indices = kv_indices;
  s.n_indices = n_indices;
  s.pt_stride = pt_stride;
  s.pt_width = pt_width;
  s.page_shift = 0;
  while ((1 << s.page_shift) < page_size) ++s.page_shift;
  s.n_pages = n_pages;
  s.batch = batch;
  s.total_q = total_q;
  return s;
}

}  // namespace tsfa
