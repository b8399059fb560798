// Windows on the host: the page lists and tile walks that the kernels and planners
// share (window_pages, window_tiles in plan.h) against an enumeration of what is
// seen, and the windowed planners with randomized and malformed metadata, built with
// the address and undefined-behaviour sanitizers (Makefile next to this file).
// The work-list upload is a copy into host memory (hipMemcpyAsync below).
//
//   window_fuzz <iterations> <seed>
#include <algorithm>
#include <cinttypes>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <random>
#include <vector>

#include "pagedattn.h"
#include "plan_internal.h"

namespace {
char* g_ws = nullptr;
size_t g_ws_bytes = 0;
bool g_upload_inside = true;
}  // namespace

extern "C" hipError_t hipMemcpyAsync(void* dst, const void* src, size_t bytes, hipMemcpyKind,
                                     hipStream_t) {
  char* d = static_cast<char*>(dst);
  if (!g_ws || d < g_ws || bytes > g_ws_bytes || d + bytes > g_ws + g_ws_bytes) {
    g_upload_inside = false;
    return hipErrorInvalidValue;
  }
  std::memcpy(dst, src, bytes);
  return hipSuccess;
}

namespace {

std::mt19937_64 rng;

int64_t uni(int64_t lo, int64_t hi) {  // inclusive
  return std::uniform_int_distribution<int64_t>(lo, hi)(rng);
}
bool coin(double p) { return std::uniform_real_distribution<double>(0, 1)(rng) < p; }

struct Window {
  int left, sinks;
  bool sees(int64_t p, int64_t j) const { return j <= p && (j >= p - left || j < sinks); }
};

Window make_window() {
  return Window{(int)(coin(0.1) ? INT_MAX - uni(0, 3) : coin(0.2) ? 0 : uni(0, 200)),
                (int)(coin(0.1) ? INT_MAX - uni(0, 3) : coin(0.4) ? 0 : uni(0, 70))};
}

// A decode step's listed pages hold every token its newest token sees, once, and no
// others outside the hole.
const char* lists_of(const Window& w) {
  const int npages = (int)uni(0, 30), last = (int)uni(1, 16);
  const pa::WindowPages x = pa::window_pages(npages, last, w.left, w.sinks);
  const int len = npages ? (npages - 1) * 16 + last : 0;
  if (x.npages < 0 || x.npages > npages || x.shift < 0 || x.npages + x.shift != npages)
    return "listed pages";
  std::vector<int> listed(std::max(len, 1), 0);
  for (int i = 0; i < x.npages; ++i) {
    const int page = i < x.sink_pages ? i : i + x.shift;
    for (int s = 0; s < 16; ++s) {
      const int token = page * 16 + s;
      const bool hole = i * 16 + s >= x.hole_lo && i * 16 + s < x.hole_hi;
      if (token >= len) continue;
      if (!hole && !w.sees(len - 1, token)) return "an unseen token outside the hole";
      listed[token] += !hole;
    }
  }
  for (int t = 0; t < len; ++t)
    if (listed[t] != (w.sees(len - 1, t) ? 1 : 0)) return "a seen token not listed once";
  if (x.hole_hi > x.hole_lo && (x.hole_hi - 1) / 16 - x.hole_lo / 16 > 1)
    return "a hole of more than two pages";
  return nullptr;
}

// A tile's walk holds every page that one of its rows sees, once and in order, and
// no page that none sees but those its last KV tile ends with.
const char* walk_of(const Window& w) {
  const int kv_len = (int)uni(0, 900);
  const int rows = (int)uni(1, 40);
  const int p_lo = (int)uni(-20, std::max(kv_len - 1, 0));
  const int p_hi = p_lo + rows - 1;  // the last row's position
  const int kv_end = std::min(kv_len, std::max(0, p_hi + 1));
  const pa::WindowTiles x = pa::window_tiles(kv_end, p_lo, w.left, w.sinks);
  if (x.total < 0 || x.total > (kv_end + 63) / 64) return "tiles";
  int before = -1;
  std::vector<bool> walked((size_t)kv_len / 16 + 2, false);
  for (int i = 0; i < 4 * x.total; ++i) {
    const int page = pa::window_page(x, i);
    if (page <= before) return "pages out of order";
    before = page;
    if (page < (int)walked.size()) walked[page] = true;
  }
  for (int p = p_lo; p <= p_hi; ++p)
    for (int j = 0; j < kv_end; ++j)
      if (w.sees(p, j) && !walked[j / 16]) return "a seen page not walked";
  for (int page = 0; page * 16 < kv_end; ++page) {
    bool seen = page * 16 < w.sinks;
    for (int j = page * 16; j < std::min(kv_end, page * 16 + 16); ++j)
      seen = seen || j >= (int64_t)std::max(p_lo, 0) - w.left;
    if (walked[page] && !seen) return "an unseen page walked";
  }
  return nullptr;
}

// The list places of a plan's tiles are a permutation.
const char* places_of() {
  const int n = (int)uni(0, 300), slots = (int)uni(1, 120);
  std::vector<bool> taken(n, false);
  for (int i = 0; i < n; ++i) {
    const int at = pa::prefill_place(i, n, slots);
    if (at < 0 || at >= n || taken[at]) return "list places";
    taken[at] = true;
  }
  return nullptr;
}

// Extreme sizes: nothing overflows, and the walk stays inside the sequence.
const char* extremes_of(const Window& w) {
  const int64_t kv_end = INT_MAX - uni(0, 100);
  const int64_t p_lo = kv_end - uni(1, 200);
  const pa::WindowTiles x = pa::window_tiles(kv_end, p_lo, w.left, w.sinks);
  const int64_t n = (kv_end + 15) / 16;
  if (x.total < 0 || 4 * (int64_t)x.total - 4 + x.shift >= n) return "tiles of a long walk";
  const pa::WindowPages l = pa::window_pages((int)n, (int)(kv_end - 16 * (n - 1)), w.left, w.sinks);
  if (l.npages < 1 || (int64_t)l.npages + l.shift != n || l.hole_hi < l.hole_lo)
    return "lists of a long sequence";
  return nullptr;
}

struct Meta {
  std::vector<int32_t> indptr, last, qo;
  int32_t batch = 0;
  bool valid = true;
};

Meta make_meta() {
  Meta m;
  m.batch = (int32_t)uni(0, 40);
  m.indptr.assign(m.batch + 1, coin(0.3) ? (int32_t)uni(0, 5000) : 0);
  m.qo.assign(m.batch + 1, 0);
  m.last.resize(m.batch);
  for (int b = 0; b < m.batch; ++b) {
    const int np = coin(0.1) ? 0 : (int)uni(1, coin(0.2) ? 2000 : 60);
    m.indptr[b + 1] = m.indptr[b] + np;
    m.last[b] = (int32_t)uni(1, 16);
    m.qo[b + 1] = m.qo[b] + (int32_t)uni(0, np ? std::min(np * 16, 700) : 3);
  }
  if (m.batch > 0 && coin(0.3)) {
    m.valid = false;
    const int b = (int)uni(0, m.batch - 1);
    switch (uni(0, 4)) {
      case 0: m.indptr[0] = -(int32_t)uni(1, INT_MAX); break;
      case 1: m.indptr[b + 1] = m.indptr[b] - (int32_t)uni(1, 100); break;
      case 2:
        m.last[b] = (int32_t)(coin(0.5) ? uni(17, INT_MAX) : -uni(0, INT_MAX));
        m.indptr[b + 1] = m.indptr[b] + 1;
        for (int c = b + 1; c < m.batch; ++c) m.indptr[c + 1] = m.indptr[b + 1];
        break;
      case 3:
        m.indptr[b + 1] = m.indptr[b] + (int32_t)uni(134217728, INT_MAX / 2);
        for (int c = b + 1; c < m.batch; ++c) m.indptr[c + 1] = m.indptr[b + 1];
        break;
      default: m.indptr[m.batch] = INT_MAX; break;
    }
  }
  return m;
}

// n entries of T at p, inside the workspace.
template <typename T>
bool inside(const void* p, int64_t n, std::vector<T>* out) {
  const char* c = static_cast<const char*>(p);
  if (n < 0 || c < g_ws + 256 || c + n * (int64_t)sizeof(T) > g_ws + g_ws_bytes) return false;
  out->resize(n);
  if (n) std::memcpy(out->data(), c, n * sizeof(T));
  return true;
}

// The windowed decode plan deals the pages of the lists, each once.
const char* dealt(const pagedattn_plan* p, const Meta& m, const Window& w) {
  std::vector<int32_t> listed(m.batch), first(m.batch + 1, 0);
  for (int b = 0; b < m.batch; ++b) {
    listed[b] = pa::window_pages(m.indptr[b + 1] - m.indptr[b], m.last[b], w.left, w.sinks).npages;
    first[b + 1] = first[b] + listed[b];
  }
  if (p->shared || p->scratch_bytes) {
    std::vector<pa::SharedItem> whole;
    if (!inside(p->shared ? p->items_dev : p->whole_dev,
                (int64_t)(p->shared ? p->n_items : p->n_whole) * pa::kSharedMaxItems, &whole))
      return "shared items outside the workspace";
    int64_t n = 0;
    for (auto& s : whole) {
      if (s.b < 0) continue;
      if (s.b >= m.batch || s.npages != listed[s.b] || s.ind_lo != first[s.b] ||
          (s.npages > 0 && s.last != m.last[s.b]))
        return "shared item";
      ++n;
    }
    if (n != (int64_t)m.batch * p->hkv) return "shared items missing";
    if (p->shared) return nullptr;
  }
  const int hg = 1 << p->hg_shift;
  std::vector<int32_t> wave_ptr;
  std::vector<pa::DecodeItem> items;
  if (!inside(p->wave_ptr_dev, (int64_t)p->n_items + 1, &wave_ptr) ||
      !inside(p->items_dev, wave_ptr.back(), &items))
    return "items outside the workspace";
  std::sort(items.begin(), items.end(),
            [](auto& x, auto& y) { return x.page_lo < y.page_lo; });
  std::map<std::pair<int, int>, int> pages;
  for (auto& i : items) {
    if (i.b < 0 || i.b >= m.batch) return "item";
    int& at = pages[{i.b, i.h}];
    if (i.page_lo != at || i.page_hi < i.page_lo || i.page_hi > listed[i.b])
      return "pages not dealt once";
    at = i.page_hi;
  }
  for (int b = 0; b < m.batch; ++b)
    for (int h = 0; h < p->hkv; h += hg)
      if (pages[{b, h}] != listed[b]) return "listed pages not dealt";
  return nullptr;
}

// A windowed prefill plan's list holds every query token once.
const char* tiled(const pagedattn_plan* p, const Meta& m) {
  std::vector<pa::PrefillItem> items;
  if (!inside(p->items_dev, p->n_items, &items)) return "tiles outside the workspace";
  std::sort(items.begin(), items.end(), [](auto& x, auto& y) { return x.q_lo < y.q_lo; });
  std::vector<int> at(m.batch, 0);
  for (auto& i : items) {
    if (i.b < 0 || i.b >= m.batch || i.q_lo != at[i.b] || i.q_hi <= i.q_lo ||
        i.q_hi - i.q_lo > p->q_tile)
      return "query tokens not covered once";
    at[i.b] = i.q_hi;
  }
  for (int b = 0; b < m.batch; ++b)
    if (at[b] != m.qo[b + 1] - m.qo[b]) return "query tokens not covered";
  return nullptr;
}

}  // namespace

int main(int argc, char** argv) {
  const int64_t iters = argc > 1 ? std::atoll(argv[1]) : 2000;
  rng.seed(argc > 2 ? std::strtoull(argv[2], nullptr, 10) : 1);
  g_ws_bytes = (size_t)64 << 20;
  g_ws = static_cast<char*>(std::aligned_alloc(256, g_ws_bytes));
  if (!g_ws) return 2;
  int failures = 0, plans = 0;
  for (int64_t it = 0; it < iters && !failures; ++it) {
    const Window w = make_window();
    const char* wrong = lists_of(w);
    if (!wrong) wrong = walk_of(w);
    if (!wrong) wrong = places_of();
    if (!wrong) wrong = extremes_of(w);
    const Meta m = make_meta();
    const bool bad_window = coin(0.1);
    const Window given = bad_window ? Window{(int)uni(-5, -1), (int)uni(1, 9)} : w;
    pagedattn_plan* plan = pagedattn_plan_create();
    int rc;
    const bool decode = coin(0.5);
    if (decode)
      rc = pagedattn_decode_plan_window(plan, m.indptr.data(), m.last.data(), m.batch, 32, 8, 128,
                                        16, coin(0.5) ? 0 : (int)uni(-1, 40), given.left,
                                        given.sinks, g_ws, g_ws_bytes, nullptr);
    else
      rc = pagedattn_prefill_plan_window(plan, m.qo.data(), m.indptr.data(), m.last.data(), m.batch,
                                         32, 8, 128, 16, given.left, given.sinks, g_ws,
                                         g_ws_bytes, nullptr);
    const char* msg = pagedattn_last_error();
    if (rc < PAGEDATTN_OK || rc > PAGEDATTN_ERR_PLAN || !g_upload_inside ||
        (rc != PAGEDATTN_OK && !(msg && msg[0])) ||
        (rc == PAGEDATTN_OK) != (m.valid && !bad_window && g_upload_inside))
      wrong = decode ? "decode plan's status" : "prefill plan's status";
    if (!wrong && rc == PAGEDATTN_OK) {
      ++plans;
      wrong = decode ? dealt(plan, m, w) : tiled(plan, m);
    }
    pagedattn_plan_destroy(plan);
    if (wrong) {
      ++failures;
      std::fprintf(stderr, "iteration %" PRId64 ": %s (window_left %d, sinks %d, status %d: %s)\n",
                   it, wrong, given.left, given.sinks, rc, msg ? msg : "");
    }
  }
  std::free(g_ws);
  std::printf("window_fuzz: %" PRId64 " iterations, %d plans, %d failures\n", iters, plans,
              failures);
  return failures ? 1 : 0;
}
