// The work of a paged attention call as one line, and the walk over a piece of
// it (csrc/paged.cu says what a unit, its weight and a cut are).  Integer
// arithmetic only, the same on the host, so that it can be run without a GPU.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define XB_LINE_FN __device__ __forceinline__
#else
#include <algorithm>
#define XB_LINE_FN inline
#endif

namespace xb {
namespace paged {

#ifdef __CUDACC__
__device__ __forceinline__ int32_t line_read(const int32_t* p) { return __ldg(p); }
__device__ __forceinline__ float line_rcp(float x) { return __frcp_rn(x); }
#else
using std::max;
using std::min;
inline int32_t line_read(const int32_t* p) { return *p; }
inline float line_rcp(float x) { return 1.0f / x; }
#endif

struct Line {
  const int32_t *q_start, *kv_len;
  int T, B, KVH, n_rep, tpt, page_size, max_pages;
  int min_share, over, snap;
};

constexpr int kFewTK = 32, kTcTK = 64;  // keys of a tile of the two kernels
constexpr int kFewRows = 16;            // rows of a tile of the few-row kernel (at most)
constexpr int kFewWarps = 8;            // its warps in a CTA, each with a piece of the line

// What belongs to the kernel with tiles of `rows` rows (8 or kFewRows: few
// rows; 128: tcgen05).  A unit's fixed cost and the smallest cut and piece were
// found by measurement, in keys.
inline void line_kernel(Line& a, int rows) {
  const bool few = rows <= kFewRows;
  a.tpt = rows / a.n_rep;
  a.over = few ? 16 : 192;
  a.snap = few ? 32 : 128;
  a.min_share = few ? 32 : 288;
}

// The line's weight is at most this whatever the device arrays hold: every
// sequence at most all tokens' query tiles per KV head, each of at most the
// table's positions (starts that ascend give far less).
inline double line_bound(const Line& a) {
  return (double)a.B * a.KVH * ((double)a.T / a.tpt + 1) * ((double)a.max_pages * a.page_size + a.over + a.tpt);
}

// Below 2^30 an int holds it, the pieces' rounding included.
inline bool line_is_wide(const Line& a, int ctas) {
  return line_bound(a) + (double)a.min_share * ctas * 2 * kFewWarps >= (double)(1 << 30);
}

// I: int where the host has seen that the line's weight stays below 2^30
// whatever the device arrays hold, else int64_t (the walks are a good part of a short
// call's instructions).
template <typename I>
struct Seq {
  int s0, n;      // first packed token, number of new tokens
  int len, base;  // keys held, keys before the new tokens (negative: the first tokens see none)
  int nt;         // query tiles
  I perh;         // weight of one KV head
};

// Weight of tiles 0 .. j - 1: each the fixed cost and the keys its last token
// sees, base + tpt (i + 1) for tile i, up to n for the last.  Where the sequence
// holds fewer keys than it brings tokens (base < 0) the first tiles see none;
// tokens without a key weigh nothing, however many they are.
template <typename I>
XB_LINE_FN I cum_keys(const Line& a, const Seq<I>& q, int j) {
  const int z = q.base < 0 ? (int)((unsigned)-q.base / (unsigned)a.tpt) : 0;  // tiles without a key
  if (j <= z) return (I)j * a.over;
  const int m = j - z;  // the product of two tile numbers may pass 2^31 before it is halved
  const I keys = (I)((int64_t)m * q.base + (int64_t)a.tpt * ((int64_t)m * (z + 1 + j) / 2));
  return (I)j * a.over + keys - (j < q.nt ? 0 : a.tpt * q.nt - q.n);
}

template <typename I>
XB_LINE_FN Seq<I> make_seq(const Line& a, int s0, int n, int len) {
  Seq<I> q;
  q.s0 = s0;
  q.n = n;
  q.len = len;
  q.base = len - n;
  q.nt = n <= a.tpt ? (n > 0) : (n + a.tpt - 1) / a.tpt;
  q.perh = q.nt == 0 ? (I)0 : q.nt == 1 ? (I)a.over + len : cum_keys(a, q, q.nt);
  return q;
}

template <typename I>
XB_LINE_FN Seq<I> load_seq(const Line& a, int b) {
  const int s0 = min(max(line_read(a.q_start + b), 0), a.T);
  const int s1 = min(max(line_read(a.q_start + b + 1), s0), a.T);
  return make_seq<I>(a, s0, s1 - s0, min(max(line_read(a.kv_len + b), 0), a.max_pages * a.page_size));
}

// Where a piece starts: a sequence, its first point on the line and its numbers.
template <typename I>
struct Found {
  I start;
  int b, s0, n, len;  // b < 0: the piece is empty
};

// A walk over one piece [lo, hi) of the line.
template <typename I>
struct Walk {
  I lo, hi, share;
  int snap;  // cuts this close to a unit's end or first key move there
  I u0;    // where the current unit starts
  I ulen;  // its weight
  int b, kvh, j;
  Seq<I> q;
};

// The part of one unit that belongs to a piece.
struct Segment {
  int b, kvh;
  int token, rows;   // first packed token and rows of the query tile
  int first_pos;     // position of the tile's first token (may be negative)
  int keys;          // keys the unit's last token sees; 0 when none of its tokens sees any
  int t0, t1;        // key tiles of this part
  int starts, ends;  // the unit starts / ends in this piece
  int last;          // where it starts and goes on: the piece in which it ends
};

// Share of `pieces` equal pieces of the line: at least total / pieces (the
// product is rounded up by more than the float error; every thread of the grid
// computes the same value).
template <typename I>
XB_LINE_FN I share_of(const Line& a, I total, int pieces) {
  const I share = (I)((float)total * line_rcp((float)pieces) * 1.000001f) + 1;
  return share < a.min_share ? a.min_share : share;
}

// How far a cut moves to a unit's boundary: a part of one costs a warp or CTA
// as much as `snap` keys (starting the second unit, merging the parts), but no
// piece may grow by more than two thirds, nor lie between two moved cuts.
template <typename I>
XB_LINE_FN int cut_snap(const Line& a, I share) {
  return (int)min((I)a.snap, (share - a.over) / 3);
}

template <typename I>
XB_LINE_FN I unit_weight(const Line& a, const Walk<I>& w) {
  return (I)a.over + max(w.q.base + min(a.tpt * (w.j + 1), w.q.n), 0);
}

// Places a walk at piece `piece`'s start.
template <typename I>
XB_LINE_FN void place(const Line& a, Walk<I>& w, int piece, I share, I total, const Found<I>& f) {
  w.share = share;
  w.snap = cut_snap(a, share);
  w.lo = piece * share;
  w.hi = total - w.lo < share ? total : w.lo + share;
  w.b = f.b;
  w.q = make_seq<I>(a, f.s0, f.n, f.len);
  I in = w.lo - f.start;
  w.kvh = 0;
  if (in >= w.q.perh) {
    w.kvh = (int)(in / w.q.perh);
    in -= w.kvh * w.q.perh;
  }
  w.j = 0;
  w.u0 = f.start + w.kvh * w.q.perh;
  if (w.q.nt > 1) {
    int lo = 0, hi = w.q.nt - 1;  // the last tile j with cum(j) <= in
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (cum_keys(a, w.q, mid) <= in) lo = mid;
      else hi = mid - 1;
    }
    w.j = lo;
    w.u0 += cum_keys(a, w.q, lo);
  }
  w.ulen = unit_weight(a, w);
}

// Steps to the next unit; false behind the piece's last one.
template <typename I>
XB_LINE_FN bool next_unit(const Line& a, Walk<I>& w) {
  w.u0 += w.ulen;
  if (w.u0 >= w.hi) return false;
  if (++w.j >= w.q.nt) {
    w.j = 0;
    if (++w.kvh >= a.KVH) {
      w.kvh = 0;
      do {
        if (++w.b >= a.B) return false;
        w.q = load_seq<I>(a, w.b);
      } while (w.q.n == 0);
    }
  }
  w.ulen = unit_weight(a, w);
  return true;
}

// The part of the current unit that belongs to this piece, stepping over a
// unit whose cut was moved away; false when nothing is left.
template <int TK, typename I>
XB_LINE_FN bool segment(const Line& a, Walk<I>& w, Segment& g) {
  for (;;) {
    const I cut0 = w.lo - w.u0, cut1 = w.hi - w.u0;  // the piece's ends inside the unit
    g.starts = cut0 < a.over + w.snap;
    if (!g.starts && w.ulen - cut0 < w.snap) {  // only at the piece's start: the unit ended in the piece before
      if (!next_unit(a, w)) return false;
      continue;
    }
    if (cut1 < a.over + w.snap && cut1 < w.ulen) return false;  // the unit starts in the next piece
    g.ends = w.ulen - cut1 < w.snap;
    const int done = w.j * a.tpt;
    const int tokens = min(a.tpt, w.q.n - done);
    g.b = w.b;
    g.kvh = w.kvh;
    g.token = w.q.s0 + done;
    g.rows = tokens * a.n_rep;
    g.first_pos = w.q.base + done;
    g.keys = max(g.first_pos + tokens, 0);
    const int nk = (int)(((unsigned)g.keys + TK - 1) / TK);
    g.t0 = g.starts ? 0 : min((int)((unsigned)(cut0 - a.over) / TK), nk);  // cuts fall on tile boundaries
    g.t1 = g.ends ? nk : min((int)((unsigned)(cut1 - a.over) / TK), nk);
    if (g.starts && !g.ends) {
      // the piece that holds the unit's last key, or the one before it if that cut was moved to the unit's end
      const I end = w.u0 + w.ulen;
      I last = (end - 1) / w.share;
      if (last * w.share > w.u0 && end - last * w.share < w.snap) --last;
      g.last = (int)last;
    }
    return true;
  }
}

}  // namespace paged
}  // namespace xb
