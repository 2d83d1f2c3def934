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
  int list;        // first entry of the page list in kv_indices (of 2^31 - 1 at most)
  int pages;       // entries of the list
};

TSFA_HD inline int64_t clamp64(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

TSFA_HD inline Seq seq_of(const Seqs& s, int b) {
  Seq r;
  r.q0 = (int)clamp64(s.q_indptr[b], 0, s.total_q);
  r.q_len = (int)clamp64(s.q_indptr[b + 1], r.q0, s.total_q) - r.q0;
  if (s.kv_indptr != nullptr) {
    r.list = (int)clamp64(s.kv_indptr[b], 0, s.n_indices);
    r.pages = (int)(clamp64(s.kv_indptr[b + 1], r.list, s.n_indices) - r.list);
  } else {
    r.list = (int)(b * s.pt_stride);
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
// `keys`.  All tiles of a call lie on one line in the order (sequence, kv
// head, tile), each as long as its keys, and the line is cut into equal runs,
// one to a workgroup: the run of a step is the one its start lies in, so every
// workgroup gets about the same work whatever the lengths are and at most the
// first and the last tile of a run are shared with its neighbours.
//
// The line counts 1 / group keys, step s of a tile starting s * unit past the
// tile.  With a mask every tile of a sequence sees its kv_len keys and is a
// whole number of steps long.  Without, tile r ends at its last token's own
// key, prefix + ((r + 1) rows - 1) / group, linear in r on this scale, so the
// place of a tile is a closed form both ways and no workgroup walks the tiles
// before its own (a loop over them took tens of microseconds for prompts of
// 1000 tokens).  Either way steps start a step's length apart at least, and
// `extra` steps of nothing at a tile's end stand for what starting and ending
// a tile costs, so that a run of many short tiles has fewer steps.
struct Cut {
  int rows, keys;           // tile height, keys of a step (powers of two)
  int group, num_kv_heads;  // query heads per kv head; kv heads
  int causal;               // no mask: a tile stops at its last token's own key
  int keys_shift, rows_shift;
  FastDiv by_group;
  int64_t unit;             // line length of a step: keys * group
  double inv_unit;
  int extra;                // steps that a tile's start and end cost
};

// 1 / d to 2^-48: on the device the hardware's estimate and one Newton step (a
// full division is three times the instructions, on every call's first path).
TSFA_HD inline double inverse(int64_t d) {
#ifdef __HIP_DEVICE_COMPILE__
  const double x = (double)d, r = __builtin_amdgcn_rcp(x);
  return __builtin_fma(r, __builtin_fma(-x, r, 1.0), r);
#else
  return 1.0 / (double)d;
#endif
}

inline Cut make_cut(int rows, int keys, int group, int num_kv_heads, int causal, int extra) {
  Cut c;
  c.rows = rows;
  c.keys = keys;
  c.group = group;
  c.num_kv_heads = num_kv_heads;
  c.causal = causal;
  for (c.keys_shift = 0; (1 << c.keys_shift) < keys;) ++c.keys_shift;
  for (c.rows_shift = 0; (1 << c.rows_shift) < rows;) ++c.rows_shift;
  c.by_group = make_fastdiv((uint32_t)group);
  c.unit = (int64_t)keys * group;
  c.inv_unit = inverse(c.unit);
  c.extra = extra;
  return c;
}

// x / d for 0 <= x < 2^52, inv = inverse(d).  Below 2^30 the half keeps (x +
// 1/2) / d at least 1/2 / d from a whole number, more than the 2^-18 that the
// product is off; above, the quotient is off by one at most before the
// remainder is looked at (2^52 2^-48 / d: by 16 / d).
TSFA_HD inline int64_t udiv(int64_t x, int64_t d, double inv) {
  if (x < (1 << 30)) return (int)(((double)(int)x + 0.5) * inv);
  int64_t q = (int64_t)((double)x * inv);
  int64_t r = x - q * d;
  for (; r < 0; r += d) --q;
  for (; r >= d; r -= d) ++q;
  return q;
}

TSFA_HD inline int cut_tiles(const Cut& c, const Seq& s) {
  return (int)(((int64_t)s.q_len * c.group + c.rows - 1) >> c.rows_shift);
}

// Steps of tile r (at least one: a tile without keys still writes its rows).
TSFA_HD inline int tile_steps(const Cut& c, const Seq& s, int r) {
  int end = s.kv_len;
  if (c.causal) {
    const int t = (int)fdiv(((uint32_t)r + 1) * (uint32_t)c.rows - 1, c.by_group);  // the tile's last token
    const int lim = s.prefix + (t < s.q_len ? t + 1 : s.q_len);
    if (lim < end) end = lim;
  }
  const int n = (int)(((int64_t)end + c.keys - 1) >> c.keys_shift);
  return n > 0 ? n : 1;
}

// Line lengths: tile 0 of a sequence and what each further tile adds to it,
// the first r tiles, and one kv head.
TSFA_HD inline int64_t tile_first(const Cut& c, const Seq& s) {
  if (c.causal) return ((int64_t)s.prefix + 1) * c.group + c.rows - 1 + c.unit - 1 + c.extra * c.unit;
  return (tile_steps(c, s, 0) + c.extra) * c.unit;
}
TSFA_HD inline int64_t tile_more(const Cut& c) { return c.causal ? c.rows : 0; }
TSFA_HD inline int64_t tiles_length(const Cut& c, const Seq& s, int64_t r) {
  return r * tile_first(c, s) + tile_more(c) * (r * (r - 1) / 2);
}
TSFA_HD inline int64_t head_length(const Cut& c, const Seq& s) { return tiles_length(c, s, cut_tiles(c, s)); }

// A place on the line: a step of `tile` of kv head `kvh`; from: the line from
// the tile's start to the given point.
struct Place {
  int kvh, tile, step;
  int64_t from;
};

// The first step at or behind the point x of a sequence's line (x < its
// length); tile or kvh may come out one past the sequence's last.
TSFA_HD inline Place place_in_seq(const Cut& c, const Seq& s, int64_t x) {
  Place p;
  const int n = cut_tiles(c, s);
  const int64_t head = head_length(c, s);
  p.kvh = (int)udiv(x, head, inverse(head));
  x -= p.kvh * head;
  const int64_t a = tile_first(c, s);
  if (!c.causal) {
    p.tile = (int)udiv(x, a, inverse(a));
  } else {
    // the last r with r a + rows r (r - 1) / 2 <= x: the root of the quadratic
    // with equality, taken in 32 bits and then looked at
    const float h = (float)a - 0.5f * c.rows, y = 2.0f * (float)x;
    int64_t r = (int64_t)(y / (h + __builtin_sqrtf(h * h + c.rows * y)));
    r = clamp64(r, 0, n - 1);
    while (r > 0 && tiles_length(c, s, r) > x) --r;
    while (r + 1 < n && tiles_length(c, s, r + 1) <= x) ++r;
    p.tile = (int)r;
  }
  p.from = x - tiles_length(c, s, p.tile);
  p.step = (int)udiv(p.from + c.unit - 1, c.unit, c.inv_unit);
  if (p.step >= tile_steps(c, s, p.tile)) {  // between the tile's last step and its end
    p.from -= a + tile_more(c) * p.tile;
    p.step = 0;
    if (++p.tile == n) {
      p.tile = 0;
      ++p.kvh;
    }
  }
  return p;
}

// Length of a run, at least half a step's: with fewer steps than workgroups a
// run holds one step or none.
TSFA_HD inline int64_t run_length(const Cut& c, int64_t total, int groups) {
  const int64_t per = udiv(total + groups - 1, groups, inverse(groups));
  return per > (c.unit + 1) / 2 ? per : (c.unit + 1) / 2;
}
// Steps of a tile that start before the line's point `ahead` past its start.
TSFA_HD inline int steps_before(const Cut& c, int64_t ahead, int steps) {
  if (ahead <= 0) return 0;
  const int64_t n = udiv(ahead + c.unit - 1, c.unit, c.inv_unit);
  return n < steps ? (int)n : steps;
}
// Whether the run at `at` holds steps of the tile at `tile` (each a point of
// the line; the tile's steps come from udiv, exact below 2^52).
TSFA_HD inline bool run_has_step(const Cut& c, int64_t at, int64_t per, int64_t tile) {
  return per >= c.unit || steps_before(c, at + per - tile, INT32_MAX) > steps_before(c, at - tile, INT32_MAX);
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
