// Runs the walk of csrc/paged_walk.cuh on the host, every piece of the line,
// and checks what it hands out against the units counted one by one.  Built
// and called by tests/test_paged_line_cpu.py.
#include <cstdio>

#include "paged_walk.cuh"

using namespace xb::paged;

namespace {

struct Unit {  // of the plain enumeration: sequences, KV heads, query tiles
  int b, kvh, token, rows, first_pos, keys;
};

struct Units {
  const Line& a;
  int b = -1, kvh = 0, n = 0, s0 = 0, base = 0;
  int64_t j = 0;
  bool next(Unit& u) {
    if (b >= 0 && (j + 1) * a.tpt < n) {
      ++j;
    } else if (b >= 0 && kvh + 1 < a.KVH && n > 0) {
      ++kvh;
      j = 0;
    } else {
      kvh = 0;
      j = 0;
      do {
        if (++b >= a.B) return false;
        s0 = std::min(std::max(a.q_start[b], 0), a.T);
        n = std::min(std::max(a.q_start[b + 1], s0), a.T) - s0;
        const int64_t held = std::min<int64_t>(std::max(a.kv_len[b], 0), (int64_t)a.max_pages * a.page_size);
        base = (int)(held - n);
      } while (n == 0);
    }
    const int done = (int)(j * a.tpt), tokens = std::min(a.tpt, n - done);
    u = Unit{b, kvh, s0 + done, tokens * a.n_rep, base + done, std::max(base + done + tokens, 0)};
    return true;
  }
};

template <int TK, typename I>
int check(const Line& a, int pieces, char* msg, size_t len, int64_t* units, double* weight) {
  // every sequence's place on the line, as the kernels' scan over the sequences gives it
  I total = 0;
  for (int b = 0; b < a.B; ++b) total += load_seq<I>(a, b).perh * a.KVH;
  *weight = (double)total;
  const I share = share_of(a, total, pieces);
  Units truth{a};
  Unit u;
  *units = 0;
  bool open = false;  // unit u goes on behind the piece before
  int last = -1, t = 0, sb = 0;
  I start = 0;
  for (int p = 0; p < pieces; ++p) {
    const I lo = p * share;
    if (lo >= total) break;
    Found<I> f;
    f.b = -1;
    for (; sb < a.B; ++sb) {  // the sequence that holds the piece's start
      const Seq<I> q = load_seq<I>(a, sb);
      const I c = q.perh * a.KVH;
      if (c > 0 && start <= lo && lo - start < c) {
        f = Found<I>{start, sb, q.s0, q.n, q.len};
        break;
      }
      start += c;
    }
    if (f.b < 0) return snprintf(msg, len, "piece %d of %d starts in no sequence", p, pieces), 1;
    Walk<I> w;
    Segment g;
    place(a, w, p, share, total, f);
    for (bool more = segment<TK>(a, w, g); more; more = next_unit(a, w) && segment<TK>(a, w, g)) {
      if (g.starts == (int)open) return snprintf(msg, len, "piece %d: starts = %d, but a unit is open: %d", p, g.starts, open), 2;
      if (g.starts) {
        if (!truth.next(u)) return snprintf(msg, len, "piece %d: more units than there are", p), 3;
        ++*units;
        t = 0;
      }
      if (g.b != u.b || g.kvh != u.kvh || g.token != u.token || g.rows != u.rows || g.first_pos != u.first_pos ||
          g.keys != u.keys)
        return snprintf(msg, len, "piece %d: unit of sequence %d, head %d, token %d with %d keys where %d, %d, %d with %d is due",
                        p, g.b, g.kvh, g.token, g.keys, u.b, u.kvh, u.token, u.keys), 4;
      const int tiles = (int)(((int64_t)g.keys + TK - 1) / TK);
      if (g.t0 != t || g.t1 < g.t0 || g.t1 > tiles || (g.ends && g.t1 != tiles))
        return snprintf(msg, len, "piece %d: tiles %d to %d of %d, from %d on are due", p, g.t0, g.t1, tiles, t), 5;
      t = g.t1;
      if (g.starts && !g.ends) {
        last = g.last;
        if (last <= p || last >= pieces) return snprintf(msg, len, "piece %d: a unit is said to end in piece %d of %d", p, last, pieces), 6;
      }
      if (!g.starts && g.ends != (p == last)) return snprintf(msg, len, "a unit said to end in piece %d: ends = %d in %d", last, g.ends, p), 7;
      open = !g.ends;
    }
  }
  if (open) return snprintf(msg, len, "the last unit does not end"), 8;
  if (truth.next(u)) return snprintf(msg, len, "%lld units were handed out, the next of sequence %d is left", (long long)*units, u.b), 9;
  return 0;
}

}  // namespace

// rows: 8, 16 (a piece per warp) or 128 (a piece per CTA); bits: 0 as the host chooses, 32 or 64
extern "C" int paged_line(int rows, int T, int B, int KVH, int n_rep, int page_size, int max_pages, int ctas, int bits,
                          const int32_t* q_start, const int32_t* kv_len, char* msg, size_t len, int64_t* units,
                          double* weight, double* bound, int* wide) {
  Line a;
  a.q_start = q_start;
  a.kv_len = kv_len;
  a.T = T;
  a.B = B;
  a.KVH = KVH;
  a.n_rep = n_rep;
  a.page_size = page_size;
  a.max_pages = max_pages;
  line_kernel(a, rows);
  *bound = line_bound(a);
  *wide = bits == 0 ? line_is_wide(a, ctas) : bits == 64;
  if (rows <= kFewRows)
    return *wide ? check<kFewTK, int64_t>(a, ctas * kFewWarps, msg, len, units, weight)
                 : check<kFewTK, int>(a, ctas * kFewWarps, msg, len, units, weight);
  return *wide ? check<kTcTK, int64_t>(a, ctas, msg, len, units, weight)
               : check<kTcTK, int>(a, ctas, msg, len, units, weight);
}
