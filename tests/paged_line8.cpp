// The walk of csrc/paged_walk.cuh as the few-row kernel over 8-bit pages takes it
// where there are many keys: tiles of 64 keys, 12 pieces a CTA of 8-row tiles.
// Built and called by tests/test_paged8_line_cpu.py.
#include "paged_line.cpp"

extern "C" int paged_line8(int rows, int T, int B, int KVH, int n_rep, int page_size, int max_pages, int ctas, int bits,
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
  line_kernel(a, rows, kFewTK8);
  *bound = line_bound(a);
  *wide = bits == 0 ? line_is_wide(a, ctas) : bits == 64;
  const int pieces = ctas * (rows == 8 ? 12 : kFewWarps);
  return *wide ? check<kFewTK8, int64_t>(a, pieces, msg, len, units, weight)
               : check<kFewTK8, int>(a, pieces, msg, len, units, weight);
}
