// The varlen attention's cut of its work (csrc/tsfa_paged.h), over random
// sequences with lengths and lists in and out of range: every step of every
// tile belongs to exactly one run, shared tiles name the runs that hold their
// parts, every page-table and list index is in range.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <tuple>
#include <vector>

#include "tsfa_paged.h"

using namespace tsfa;
using namespace tsfa::paged;

#define CHECK(x)                                                              \
  do {                                                                        \
    if (!(x)) {                                                               \
      std::printf("case %d: %s (line %d)\n", g_case, #x, __LINE__);           \
      std::exit(1);                                                           \
    }                                                                         \
  } while (0)
static int g_case = 0;

static void check_udiv(std::mt19937_64& rng) {
  for (int i = 0; i < 2000000; ++i) {
    const int64_t d = 1 + (int64_t)(rng() >> (24 + rng() % 40));
    int64_t x = (int64_t)(rng() >> (12 + rng() % 52));
    if (i % 3 == 0) x = x / d * d;          // at a multiple, and just below one
    if (i % 3 == 1) x = x / d * d + d - 1;
    if (x < 0 || x >= ((int64_t)1 << 52)) continue;
    // the device's inverse is up to 2^-48 off either way
    for (double e : {0.0, 3.5e-15, -3.5e-15}) CHECK(udiv(x, d, inverse(d) * (1 + e)) == x / d);
  }
}

int main() {
  std::mt19937_64 rng64(3);
  check_udiv(rng64);
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (uint32_t)(hi - lo + 1)); };
  for (g_case = 0; g_case < 3000; ++g_case) {
    const bool wild = g_case % 5 == 0, dense = g_case % 3 == 0;
    const int batch = pick(1, g_case % 50 == 0 ? 150 : 9), page_shift = pick(4, 8);
    std::vector<int32_t> qi{0}, kl, pi{0};
    for (int b = 0; b < batch; ++b) {
      const int q = pick(0, 3) == 0 ? 0 : pick(0, 9) == 0 ? pick(1, 700) : pick(1, 70);
      const int p = pick(0, 4) == 0 ? 0 : pick(0, 20) == 0 ? pick(1, 60000) : pick(1, 900);
      qi.push_back(qi.back() + q);
      kl.push_back(q + p);
      pi.push_back(pi.back() + (q + p + (1 << page_shift) - 1) / (1 << page_shift));
    }
    const int total_q = qi.back();
    int width = 0;
    for (int b = 0; b < batch; ++b) width = std::max(width, pi[b + 1] - pi[b]);
    std::vector<int32_t> indices(dense ? (size_t)batch * width : (size_t)pi.back(), 0);
    if (wild) {
      for (int i = 0; i < 3; ++i) {
        kl[pick(0, batch - 1)] = (int32_t)rng();
        qi[pick(0, batch)] = pick(0, 1) ? (int32_t)rng() : pick(-5, total_q + 5);
        pi[pick(0, batch)] = (int32_t)rng();
      }
    }
    Seqs s = make_seqs(qi.data(), kl.data(), dense ? nullptr : pi.data(), indices.data(), (int64_t)indices.size(),
                       width, width, 4, 1 << page_shift, batch, total_q);
    const int rg = 1 << pick(0, 3), streams = 1 << pick(0, 2);
    const Cut c = make_cut(32 * rg, 32 * streams, pick(1, 9), pick(1, 4), pick(0, 1), pick(0, 9));
    const int groups = pick(0, 1) ? 256 : pick(1, 40);

    int64_t total = 0;
    for (int b = 0; b < batch; ++b) {
      const Seq q = seq_of(s, b);
      CHECK(q.q0 >= 0 && q.q_len >= 0 && q.q0 + q.q_len <= total_q && q.kv_len >= 0 && q.prefix >= 0);
      CHECK(q.list >= 0 && q.pages >= 0 && q.list + q.pages <= (int64_t)indices.size());
      CHECK(((int64_t)q.pages << page_shift) >= q.kv_len && q.prefix <= q.kv_len);
      total += head_length(c, q) * c.num_kv_heads;
      int64_t sum = 0;
      for (int r = 0; r < cut_tiles(c, q); ++r) {
        CHECK(tiles_length(c, q, r) == sum);
        const int64_t len = tile_first(c, q) + tile_more(c) * r;
        CHECK(len >= tile_steps(c, q, r) * c.unit);  // steps start a step's length apart
        sum += len;
      }
      CHECK(head_length(c, q) == sum);
    }
    if (total == 0 || total / c.unit > 400000) continue;
    const int64_t per = run_length(c, total, groups);
    std::map<std::tuple<int, int, int>, std::vector<std::tuple<int, int, int>>> parts;  // tile -> (run, s0, s1)
    CHECK(per * groups >= total);
    for (int run = 0; run < groups; ++run) {
      const int64_t at = run * per;
      if (at >= total) break;
      const int64_t end = std::min(at + per, total);
      int b = 0;
      int64_t before = 0;
      for (;; ++b) {
        CHECK(b < batch);
        const int64_t n = head_length(c, seq_of(s, b)) * c.num_kv_heads;
        if (before + n > at) break;
        before += n;
      }
      Seq q = seq_of(s, b);
      Place p = place_in_seq(c, q, at - before);
      int64_t left = end - (at - p.from);
      bool more = true;
      auto next = [&]() {
        do {
          if (++b >= batch) return false;
          q = seq_of(s, b);
        } while (q.q_len == 0);
        return true;
      };
      if (p.kvh == c.num_kv_heads) {
        p.kvh = 0;
        more = next();
      }
      while (more) {
        const int n = tile_steps(c, q, p.tile), s0 = p.step;
        CHECK(p.tile < cut_tiles(c, q) && p.kvh < c.num_kv_heads && s0 < n);
        const int s1 = steps_before(c, left, n);
        if (s0 >= s1) break;
        parts[{b, p.kvh, p.tile}].push_back({run, s0, s1});
        for (int c0 = s0; c0 < s1 && q.kv_len > 0;) {
          const Chunk k = chunk_of(q, page_shift, streams, c0, s1, !c.causal);
          CHECK(k.end > c0 && k.end <= s1 && k.first_page >= 0 && k.ids >= 1 && k.ids <= kTableIds);
          CHECK(k.first_page + k.ids <= q.pages);
          if (!c.causal) CHECK(k.end * streams - k.tree_unit <= kTreeUnits);
          for (int u = c0 * streams; u < k.end * streams; ++u) {
            if ((u + 1) * 32 > q.prefix) CHECK(u >= k.tree_unit);
            for (int rpl : {4, 8})
              for (int kb = 0; kb < 32; kb += rpl) {
                const int blk = load_block(u * 32 + kb, rpl, q.kv_len);
                CHECK(blk >= 0 && blk < q.kv_len);
                const int id = (blk >> page_shift) - k.first_page;
                CHECK(id >= 0 && id < k.ids);
              }
          }
          c0 = k.end;
        }
        if (s1 < n) break;
        left -= tile_first(c, q) + tile_more(c) * p.tile;
        if (left <= 0) break;
        p.step = 0;
        if (++p.tile == cut_tiles(c, q)) {
          p.tile = 0;
          if (++p.kvh == c.num_kv_heads) {
            p.kvh = 0;
            more = next();
          }
        }
      }
    }
    int64_t line = 0;
    for (int b = 0; b < batch; ++b) {
      const Seq q = seq_of(s, b);
      for (int h = 0; h < c.num_kv_heads; ++h)
        for (int t = 0; t < cut_tiles(c, q); ++t) {
          const int n = tile_steps(c, q, t);
          auto& v = parts[{b, h, t}];
          CHECK(!v.empty());
          int upto = 0;
          for (size_t i = 0; i < v.size(); ++i) {
            auto [run, s0, s1] = v[i];
            CHECK(s0 == upto && s1 > s0 && run >= std::get<0>(v[0]) + (int)i);
            upto = s1;
          }
          CHECK(upto == n);
          // the runs between the first and the last part's that hold a part are those run_has_step names
          size_t held = 0;
          for (int run = std::get<0>(v.front()); run <= std::get<0>(v.back()); ++run)
            if (run_has_step(c, run * per, per, line)) {
              CHECK(held < v.size() && std::get<0>(v[held]) == run);
              ++held;
            }
          CHECK(held == v.size());
          // the number of parts as the first run writes it for the join
          if (v.size() > 1)
            CHECK((int)udiv(line + (n - 1) * c.unit, per, inverse(per)) == std::get<0>(v.back()));
          line += tile_first(c, q) + tile_more(c) * t;
        }
    }
    CHECK(line == total);
  }
  std::printf("all invariants hold\n");
  return 0;
}
