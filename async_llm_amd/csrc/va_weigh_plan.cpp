// Host side of attention weights: the sub-request tables of a step, turned round (va_weigh.h).
#include <algorithm>
#include <climits>
#include <cstring>
#include <numeric>
#include <stdexcept>
#include <unordered_map>
#include <utility>
#include <vector>

#include "../../include/viewattn.h"
#include "va_internal.h"
#include "va_weigh.h"

namespace {

struct Visitor {
  int32_t list;  // one of `lists`
  int32_t entry;  // of its list
  int32_t place;  // -1: the whole page; a token of it, for lists of slots
  bool operator==(const Visitor& o) const { return list == o.list && entry == o.entry && place == o.place; }
};

struct Planner {
  const VaSubRequests& in;
  const VaShape& shape;
  bool rows32;  // 32-bit keys
  int num_pages, window;
  Planner(const VaSubRequests& s, const VaShape& sh, bool wide, int pages_, int w) : in(s), shape(sh), rows32(wide), num_pages(pages_), window(w) {}
  // Lists of entries that differ: readers of a shared block bring the same one, which is then looked through once.
  struct List {
    const int32_t* at;
    int32_t entries;
    bool by_slot;
    int32_t first_reader, last_reader;  // sub-requests, linked by next_reader
    bool alone;                         // none of its pages is another entry's too
  };
  std::vector<List> lists;
  std::vector<int32_t> next_reader;  // by sub-request; -1 behind the last
  std::vector<int32_t> first_visitor;  // by page, [num_pages + 1]
  std::vector<Visitor> visitors;
  std::vector<int32_t> pages, items, joins, sub_row, lo, hi;
  int64_t n_partials = 0;

  int rows_of(int s) const { return in.qo_indptr[s + 1] - in.qo_indptr[s]; }
  int skipped(int s) const { return window > 0 ? std::max(0, rows_of(s) - window) : 0; }
  // tokens of its list that row i of sub-request s sees
  int64_t seen(int s, int i) const {
    const int64_t len = in.seq_lens[s];
    return in.flags[s] & VA_SUB_CAUSAL ? std::max<int64_t>(0, len - rows_of(s) + i + 1) : len;
  }
  bool slots(int s) const { return in.flags[s] & VA_SUB_SLOTS; }
  int64_t entries(int s) const { return slots(s) ? in.seq_lens[s] : ((int64_t)in.seq_lens[s] + shape.page_size - 1) / shape.page_size; }

  int find_lists() {
    if (in.n_sub < 0 || in.n_subrows < 0) return va_fail(VA_ERR_ARG, "negative count");
    if (in.n_sub == 0) return VA_OK;
    if (!in.qo_indptr || !in.kv_indptr || !in.seq_lens || !in.flags) return va_fail(VA_ERR_ARG, "null table");
    if (in.qo_indptr[0] != 0 || in.qo_indptr[in.n_sub] != in.n_subrows || in.kv_indptr[0] != 0)
      return va_fail(VA_ERR_ARG, "tables do not start at 0 or end at n_subrows");
    const int64_t pool = (int64_t)num_pages * shape.page_size;
    next_reader.assign((size_t)in.n_sub, -1);
    std::unordered_multimap<int32_t, int32_t> by_first;  // first entry -> list
    for (int s = 0; s < in.n_sub; ++s) {
      if (in.qo_indptr[s + 1] < in.qo_indptr[s] || in.kv_indptr[s + 1] < in.kv_indptr[s] || in.seq_lens[s] < 0)
        return va_fail(VA_ERR_ARG, "sub-request %d: tables must not fall", s);
      const int64_t n = entries(s);
      if (n > in.kv_indptr[s + 1] - in.kv_indptr[s]) return va_fail(VA_ERR_ARG, "sub-request %d: %d tokens in %d entries", s, in.seq_lens[s], in.kv_indptr[s + 1] - in.kv_indptr[s]);
      if (n == 0) continue;
      if (!in.kv_indices) return va_fail(VA_ERR_ARG, "null table");
      const List list{in.kv_indices + in.kv_indptr[s], (int32_t)n, slots(s), s, s, false};
      int32_t known = -1;
      for (auto [i, end] = by_first.equal_range(list.at[0]); i != end && known < 0; ++i) {
        const List& o = lists[(size_t)i->second];
        if (o.entries == list.entries && o.by_slot == list.by_slot && !std::memcmp(o.at, list.at, (size_t)n * 4)) known = i->second;
      }
      const int32_t limit = list.by_slot ? (int32_t)pool : num_pages;
      if (const int32_t* bad = known < 0 ? outside(list, limit) : nullptr)
        return va_fail(VA_ERR_ARG, "%s %d lies outside the pool of %d pages of %d tokens", list.by_slot ? "slot" : "page", *bad, num_pages, shape.page_size);
      if (rows_of(s) == 0) continue;
      if (known < 0) {
        by_first.emplace(list.at[0], (int32_t)lists.size());
        lists.push_back(list);
      } else {
        List& o = lists[(size_t)known];
        o.last_reader = next_reader[(size_t)o.last_reader] = s;
      }
    }
    return VA_OK;
  }

  static const int32_t* outside(const List& list, int32_t limit) {
    int32_t any = 0;
    for (int32_t e = 0; e < list.entries; ++e) any |= (list.at[e] < 0) | (list.at[e] >= limit);
    return any ? std::find_if(list.at, list.at + list.entries, [&](int32_t x) { return x < 0 || x >= limit; }) : nullptr;
  }

  // Who visits the pages of the lists that are not alone.
  void find_visitors() {
    const int P = shape.page_size;
    first_visitor.assign((size_t)num_pages + 1, 0);
    auto count = [&](const List& list) {
      for (int32_t e = 0; e < list.entries; ++e) ++first_visitor[(size_t)(list.by_slot ? list.at[e] / P : list.at[e])];
    };
    for (const List& list : lists) count(list);
    bool others = false;
    for (List& list : lists) {
      int32_t more = 0;
      for (int32_t e = 0; e < list.entries && !list.by_slot; ++e) more |= first_visitor[(size_t)list.at[e]] - 1;
      list.alone = !list.by_slot && more == 0;
      others = others || !list.alone;
    }
    if (!others) return;
    first_visitor.assign((size_t)num_pages + 1, 0);
    for (const List& list : lists)
      if (!list.alone) count(list);
    int32_t sum = 0;  // (of entries, which 32 bits count)
    for (int32_t& n : first_visitor) sum += n, n = sum;
    visitors.resize((size_t)sum);
    // (from the last to the first: what was a page's end becomes its beginning)
    for (size_t l = lists.size(); l-- > 0;) {
      const List& list = lists[l];
      if (list.alone) continue;
      for (int32_t e = list.entries; e-- > 0;) {
        const int32_t x = list.at[e];
        const Visitor v = list.by_slot ? Visitor{(int32_t)l, e, x % P} : Visitor{(int32_t)l, e, -1};
        visitors[(size_t)--first_visitor[(size_t)(list.by_slot ? x / P : x)]] = v;
      }
    }
  }

  // Whether the sub-requests that read page a read page b as their next one, and nobody else does.
  bool follows(int32_t a, int32_t b) const {
    const int32_t n = first_visitor[a + 1] - first_visitor[a];
    if (n != first_visitor[b + 1] - first_visitor[b]) return false;
    const Visitor *x = &visitors[(size_t)first_visitor[a]], *y = &visitors[(size_t)first_visitor[b]];
    for (int32_t i = 0; i < n; ++i)
      if (x[i].place >= 0 || !(Visitor{x[i].list, x[i].entry + 1, -1} == y[i])) return false;
    return true;
  }

  // Tokens of a run that somebody sees, without a gap.
  struct Span {
    int64_t page_begin;
    int32_t first, end;
    int64_t row_begin, row_end;  // packed
    int pairs;  // of a tile
  };
  std::vector<Span> spans;
  // Pages that follow one another for all who read them: a list that is alone, or some of run_pages.
  struct Run {
    int32_t list;  // -1: run_pages
    int64_t begin, end;
  };
  std::vector<int32_t> run_pages;
  std::vector<Run> runs;

  void find_runs() {
    std::vector<char> done;
    for (size_t l = 0; l < lists.size(); ++l) {
      const List& list = lists[l];
      if (list.alone) {
        runs.push_back(Run{(int32_t)l, 0, list.entries});
        continue;
      }
      if (done.empty()) done.assign((size_t)num_pages, 0);
      int32_t before = -1;
      for (int32_t e = 0; e < list.entries; ++e) {
        const int32_t page = list.by_slot ? list.at[e] / shape.page_size : list.at[e];
        if (done[page]) continue;
        done[page] = 1;
        if (before < 0 || !follows(before, page)) runs.push_back(Run{-1, (int64_t)run_pages.size(), 0});
        run_pages.push_back(before = page);
        runs.back().end = (int64_t)run_pages.size();
      }
    }
  }

  // Rows of a run's visitors that see any of it: `each(sub-row, first token, end)`.
  template <typename F>
  void rows_of_run(const Run& run, F&& each) const {
    const int P = shape.page_size;
    const int64_t room = (run.end - run.begin) * P;  // (within the pool, whose slots 32 bits count)
    const Visitor itself{run.list, 0, -1};
    const Visitor *v = &itself, *last = v + 1;
    if (run.list < 0) {
      const int32_t page = run_pages[(size_t)run.begin];
      v = visitors.data() + first_visitor[page], last = visitors.data() + first_visitor[page + 1];
    }
    for (; v < last; ++v)
      for (int32_t s = lists[(size_t)v->list].first_reader; s >= 0; s = next_reader[(size_t)s])
        for (int i = skipped(s); i < rows_of(s); ++i) {
          int64_t from = 0, to = std::min(room, seen(s, i) - (int64_t)v->entry * P);
          if (v->place >= 0) from = v->place, to = seen(s, i) > v->entry ? v->place + 1 : 0;
          if (to > from) each(in.qo_indptr[s] + i, (int32_t)from, (int32_t)to);
        }
  }

  size_t n_tile_spans = 0;
  int64_t n_tile_rows = 0;

  int find_spans() {
    find_runs();
    const int G = shape.num_q_heads / shape.num_kv_heads;
    const bool halves = !rows32 && (shape.head_dim == 64 || shape.head_dim == 128 || shape.head_dim == 256);
    const size_t n = runs.size();
    std::vector<char> many(n, 0);
    std::vector<std::pair<int32_t, int32_t>> seen_parts;
    for (size_t i = 0; i < n && halves; ++i) {
      int64_t rows = 0;
      rows_of_run(runs[i], [&](int32_t, int32_t, int32_t) { ++rows; });
      many[i] = rows * G > 16;
    }
    for (int which = 1; which >= 0; --which) {  // those of tile items first
      const int pairs = which ? VA_WEIGH_TILE_ROWS : 16, unit = pairs / std::gcd(pairs, G);
      for (size_t i = 0; i < n; ++i) {
        if (many[i] != which) continue;
        const int64_t row_begin = (int64_t)sub_row.size();
        int32_t first = INT32_MAX, end = 0;
        bool places = false;  // single tokens of a page: there may be some between them that nobody sees
        rows_of_run(runs[i], [&](int32_t row, int32_t from, int32_t to) {
          sub_row.push_back(row), lo.push_back(from), hi.push_back(to);
          places = places || from > 0;
          first = std::min(first, from), end = std::max(end, to);
        });
        if ((int64_t)sub_row.size() == row_begin) continue;
        while (sub_row.size() % unit) sub_row.push_back(-1), lo.push_back(0), hi.push_back(0);
        if ((int64_t)sub_row.size() * G > INT32_MAX / 32)  // (a thread for each 16 elements of a row)
          return va_fail(VA_ERR_ARG, "too many query rows for one plan");
        Span span{(int64_t)pages.size(), first, end, row_begin, (int64_t)sub_row.size(), pairs};
        if (places) {  // a span for each part
          seen_parts.clear();
          for (size_t r = (size_t)row_begin; r < sub_row.size(); ++r)
            if (sub_row[r] >= 0) seen_parts.emplace_back(lo[r], hi[r]);
          std::sort(seen_parts.begin(), seen_parts.end());
          span.end = first;
          for (const auto& [from, to] : seen_parts) {
            if (from > span.end) spans.push_back(span), span.first = from;
            span.end = std::max(span.end, to);
          }
        }
        spans.push_back(span);
        const int32_t* from = runs[i].list < 0 ? run_pages.data() : lists[(size_t)runs[i].list].at;
        pages.insert(pages.end(), from + runs[i].begin, from + runs[i].end);
      }
      if (which) n_tile_spans = spans.size(), n_tile_rows = (int64_t)sub_row.size();
    }
    return VA_OK;
  }

  static constexpr int64_t kWorkgroups = 512;  // that run at a time
  std::vector<int32_t> strips;
  int64_t n_tile_items = 0;

  int make_items() {
    if (const int rc = make_tiles()) return rc;
    if (const int rc = make_strips()) return rc;
    if ((items.size() / VA_WEIGH_ITEM_WORDS + strips.size()) * (size_t)shape.num_kv_heads > INT32_MAX)
      return va_fail(VA_ERR_ARG, "too many work items for one launch");
    return VA_OK;
  }

  // The tiles of a span's rows that see any of its tokens [begin, end): they lie between these (a request's rows see ever more).
  void tiles_of(const Span& s, int64_t begin, int64_t end, int64_t& tile_a, int64_t& tile_b) const {
    const int G = shape.num_q_heads / shape.num_kv_heads;
    int64_t a = s.row_begin, b = s.row_end;
    while (a < b && (hi[(size_t)a] <= begin || lo[(size_t)a] >= end)) ++a;
    while (b > a && (hi[(size_t)b - 1] <= begin || lo[(size_t)b - 1] >= end)) --b;
    tile_a = a * G / s.pairs, tile_b = a == b ? tile_a : (b * G + s.pairs - 1) / s.pairs;
  }
  // Tokens [begin, begin + n_tok) under tiles [tile_a, tile_b), in `parts` items: `each(part, item words)`.
  template <typename F>
  int put_items(const Span& s, int64_t begin, int n_tok, int64_t tile_a, int64_t tile_b, int64_t parts, F&& each) {
    if (parts > 1) {
      if (n_partials + parts * n_tok > INT32_MAX) return va_fail(VA_ERR_ARG, "too many partial sums for one plan");
      const int32_t join[VA_WEIGH_JOIN_WORDS] = {(int32_t)s.page_begin, (int32_t)begin, n_tok, (int32_t)n_partials, (int32_t)parts, 0, 0, 0};
      joins.insert(joins.end(), join, join + VA_WEIGH_JOIN_WORDS);
    }
    for (int64_t p = 0; p < parts; ++p) {
      each(p);
      const int32_t item[VA_WEIGH_ITEM_WORDS] = {(int32_t)s.page_begin, (int32_t)begin, n_tok, (int32_t)(tile_a + (tile_b - tile_a) * p / parts),
                                                 (int32_t)(tile_a + (tile_b - tile_a) * (p + 1) / parts),
                                                 parts > 1 ? (int32_t)(n_partials + p * n_tok) : -1, 0, 0};
      items.insert(items.end(), item, item + VA_WEIGH_ITEM_WORDS);
    }
    if (parts > 1) n_partials += parts * n_tok;
    return VA_OK;
  }

  // Tile items of 256 tokens, with as many rows as make about 2048 workgroups of equal products, but not fewer than four tiles, nor
  // less than takes as long as a strip beside them (whose token takes about eight times as long as a token's one tile of rows).
  int make_tiles() {
    int64_t products = 0, walked = 0, tile_a, tile_b;  // (token, tile of rows); tokens of strips
    for (size_t i = 0; i < spans.size(); ++i) {
      const int64_t n = spans[i].end - spans[i].first;
      if (i >= n_tile_spans) {
        walked += n;
      } else {
        tiles_of(spans[i], spans[i].first, spans[i].end, tile_a, tile_b);
        products += n * (tile_b - tile_a);
      }
    }
    const int64_t T = VA_WEIGH_TILE_TOKENS, hkv = shape.num_kv_heads;
    const int64_t most = std::max({4 * T, products * hkv / 2048, 8 * walked * hkv / kWorkgroups});
    for (size_t i = 0; i < n_tile_spans; ++i) {
      const Span& s = spans[i];
      for (int64_t t = s.first; t < s.end; t += T) {
        const int n_tok = (int)std::min<int64_t>(T, s.end - t);
        tiles_of(s, t, t + n_tok, tile_a, tile_b);
        if (tile_a == tile_b) continue;
        if (const int rc = put_items(s, t, n_tok, tile_a, tile_b, std::min((n_tok * (tile_b - tile_a) + most - 1) / most, tile_b - tile_a), [](int64_t) {})) return rc;
      }
    }
    while (items.size() % (8 * VA_WEIGH_ITEM_WORDS)) items.push_back(0);
    n_tile_items = (int64_t)items.size() / VA_WEIGH_ITEM_WORDS;
    return VA_OK;
  }

  // Strips of equal cost, two workgroups a CU where there is that much: a token costs its key, and a quarter of that more for every
  // further tile of rows (of 32-bit rows, which have no tile items).  Tokens are cut at multiples of what the waves of a workgroup take at a time.
  int make_strips() {
    constexpr int64_t kKey = 4;
    const int row = shape.head_dim * (rows32 ? 4 : 2);
    const int hkv = shape.num_kv_heads, heads = hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;  // of a workgroup, whose four waves share them
    const int64_t least = 4 / heads * 16 * (row > 256 ? 1 : row > 128 ? 2 : 4);
    auto cost_of = [&](int64_t tiles) { return kKey + tiles - 1; };
    int64_t total = 0, pieces = 0;
    if (n_tile_spans == spans.size()) return VA_OK;
    for (size_t i = n_tile_spans; i < spans.size(); ++i) {
      const Span& s = spans[i];
      int64_t tile_a, tile_b;
      tiles_of(s, s.first, s.end, tile_a, tile_b);
      total += (s.end - s.first) * cost_of(tile_b - tile_a);
      pieces += ((int64_t)s.end - s.first + least - 1) / least * (tile_b - tile_a);
    }
    const int64_t n = std::max<int64_t>(1, std::min(pieces, std::max<int64_t>(1, kWorkgroups * heads / hkv)));
    // Strip k ends where the cost so far is nearest to (k + 1) / n of all: never more than n of them, which run at a time.
    int64_t used = 0, k = 0, target = total / n;
    strips.push_back((int32_t)n_tile_items);
    auto close_at = [&](int64_t margin) {  // begins another strip where this one is within `margin` of its end
      if (k + 1 >= n || used + margin < target || (size_t)strips.back() * VA_WEIGH_ITEM_WORDS == items.size()) return;
      strips.push_back((int32_t)(items.size() / VA_WEIGH_ITEM_WORDS));
      while (k + 1 < n && used + margin >= target) target = total * (++k + 1) / n;
    };
    for (size_t i = n_tile_spans; i < spans.size(); ++i) {
      const Span& s = spans[i];
      int64_t t = s.first;
      while (t < s.end) {
        int64_t tile_a, tile_b;
        tiles_of(s, t, s.end, tile_a, tile_b);
        if (tile_a == tile_b) break;
        const int64_t cost = cost_of(tile_b - tile_a);
        // as many tokens as the strip has room for, to the nearest cut; rows are split where the least number costs more than a strip
        const int64_t parts = std::min(tile_b - tile_a, std::max<int64_t>(1, std::min<int64_t>(least, s.end - t) * cost * n / std::max<int64_t>(1, total)));
        int64_t n_tok = least;
        close_at(parts == 1 ? least * cost / 2 : 0);
        if (parts == 1) n_tok = k + 1 < n ? std::max<int64_t>(1, ((target - used) / cost + least / 2) / least) * least : s.end - t + least;
        // (chunks start on multiples of 16 tokens of the span: pages of as many are read in runs)
        const int64_t end = std::min<int64_t>(s.end, (t + n_tok) / 16 * 16), each = (end - t) * cost / parts;
        const int rc = put_items(s, t, (int)(end - t), tile_a, tile_b, parts, [&](int64_t p) {
          if (p > 0) close_at(each / 2);
          used += each;
        });
        if (rc) return rc;
        t = end;
      }
    }
    strips.push_back((int32_t)(items.size() / VA_WEIGH_ITEM_WORDS));
    while ((strips.size() - 1) % 8) strips.push_back(strips.back());
    return VA_OK;
  }
};

int build(const VaSubRequests* subs, const VaShape* shape, int32_t over_codes, int32_t num_pages, int32_t window, int32_t* plan, int64_t capacity, VaWeighCounts* counts) {
  if (!subs || !shape || !counts) return va_fail(VA_ERR_ARG, "null pointer");
  if (shape->num_kv_heads <= 0 || shape->num_q_heads <= 0 || shape->num_q_heads % shape->num_kv_heads || shape->head_dim <= 0 || shape->page_size <= 0)
    return va_fail(VA_ERR_ARG, "bad shape");
  if (num_pages < 0 || (int64_t)num_pages * shape->page_size > INT32_MAX || window < 0)
    return va_fail(VA_ERR_ARG, "%d pages of %d tokens, window %d", (int)num_pages, (int)shape->page_size, (int)window);
  Planner p{*subs, *shape, shape->dtype == VA_F32 && !over_codes, num_pages, window};
  int rc = p.find_lists();
  if (rc) return rc;
  p.find_visitors();
  if ((rc = p.find_spans()) || (rc = p.make_items())) return rc;
  const int64_t n_rows = (int64_t)p.sub_row.size();
  const int64_t words = VA_WEIGH_HEADER_WORDS + (int64_t)p.items.size() + (int64_t)p.joins.size() + (int64_t)p.strips.size() + (int64_t)p.pages.size() + 3 * n_rows;
  if (words > INT32_MAX) return va_fail(VA_ERR_ARG, "too large a plan");
  const int64_t pairs = n_rows * (shape->num_q_heads / shape->num_kv_heads);
  counts->n_items = (int32_t)(p.items.size() / VA_WEIGH_ITEM_WORDS);
  counts->n_rows = (int32_t)n_rows;
  counts->n_joins = (int32_t)(p.joins.size() / VA_WEIGH_JOIN_WORDS);
  counts->n_spans = (int32_t)p.spans.size();
  counts->plan_words = (int32_t)words;
  // queries as up to three 16-bit numbers an element (one 32-bit one on the vector ALU), 16 bytes a row beside them, partial sums
  counts->workspace_bytes = shape->num_kv_heads * (pairs * (6 * (int64_t)shape->head_dim + 16) + 4 * p.n_partials);
  if (!plan || capacity < words) return va_fail(VA_ERR_CAPACITY, "plan needs %lld words, %lld given", (long long)words, (long long)capacity);
  int32_t* h = plan;
  std::fill(h, h + VA_WEIGH_HEADER_WORDS, 0);
  int64_t at = VA_WEIGH_HEADER_WORDS;
  auto put = [&](const std::vector<int32_t>& x) {
    std::copy(x.begin(), x.end(), plan + at);
    const int32_t begin = (int32_t)at;
    at += (int64_t)x.size();
    return begin;
  };
  h[VA_WH_MAGIC] = VA_WEIGH_MAGIC;
  h[VA_WH_N_ITEMS] = counts->n_items;
  h[VA_WH_N_ROWS] = counts->n_rows;
  h[VA_WH_N_JOINS] = counts->n_joins;
  h[VA_WH_N_PARTIALS] = (int32_t)p.n_partials;
  h[VA_WH_N_PAGES] = (int32_t)p.pages.size();
  h[VA_WH_OFF_ITEMS] = put(p.items);
  h[VA_WH_OFF_JOINS] = put(p.joins);
  h[VA_WH_N_STRIPS] = std::max((int32_t)p.strips.size() - 1, 0);
  h[VA_WH_OFF_STRIPS] = put(p.strips);
  h[VA_WH_OFF_PAGES] = put(p.pages);
  h[VA_WH_OFF_ROWS] = put(p.sub_row);
  put(p.lo);
  put(p.hi);
  h[VA_WH_HQ] = shape->num_q_heads, h[VA_WH_HKV] = shape->num_kv_heads, h[VA_WH_D] = shape->head_dim;
  h[VA_WH_CODES] = over_codes != 0;
  h[VA_WH_PAGE] = shape->page_size, h[VA_WH_DTYPE] = shape->dtype, h[VA_WH_POOL_PAGES] = num_pages, h[VA_WH_N_SUBROWS] = subs->n_subrows;
  h[VA_WH_N_TILE_ITEMS] = (int32_t)p.n_tile_items, h[VA_WH_N_TILE_ROWS] = (int32_t)p.n_tile_rows;
  return VA_OK;
}

}  // namespace

extern "C" int va_weigh_plan(const VaSubRequests* subs, const VaShape* shape, int32_t over_codes, int32_t num_pages, int32_t window, int32_t* plan_host,
                             int64_t plan_capacity_words, VaWeighCounts* counts) {
  try {
    return build(subs, shape, over_codes, num_pages, window, plan_host, plan_capacity_words, counts);
  } catch (const std::exception& e) {  // (no memory: nothing may leave a C entry)
    return va_fail(VA_ERR_CAPACITY, "planning weights: %s", e.what());
  }
}
