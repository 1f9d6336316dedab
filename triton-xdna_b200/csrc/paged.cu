// Operators of a paged KV cache: RoPE of packed new tokens with the write of
// their keys and values into pages, causal grouped-query attention of those
// tokens over the pages, and page copies inside the pool.
//
// The contiguous counterparts are xb_rope_kv_bf16 and xb_attention_bf16
// (csrc/llm.cu; examples/qwen2_5/model.py:851-889 and kernels/attention.py:
// 27-122).  There every sequence of a batch has the same length; here a step
// packs the new tokens of many sequences without padding:
//
//   q_start [B + 1]  tokens q_start[b] .. q_start[b + 1] - 1 belong to sequence b
//   kv_len  [B]      positions sequence b holds, its new tokens included
//   table   [B, max_pages]  the pages of each sequence, in order
//   pages   [n_pages, KVH, page, D] bf16, any strides with unit last one
//
// All three live on the device and are read by the kernels, so a captured
// graph serves every step of the same batch size.  Token i (0-based) of the
// n_b = q_start[b + 1] - q_start[b] new ones sits at position
// kv_len[b] - n_b + i and sees the keys 0 .. that position.
//
// Nothing the device holds can make a kernel leave its buffers: token ranges
// are clamped to the rows given, lengths to what the table can hold, and a
// page id outside the pool reads as zeros (attention) or is skipped (writes)
// and sets the flag that xb_page_status reports.
#include "common.cuh"
#include "paged_walk.cuh"
#include "tc.cuh"

namespace xb {
namespace paged {

using namespace tc;
typedef __nv_bfloat16 bf16;

__device__ int g_bad_page = 0;      // a page id outside the pool, or a position without a page
__device__ int g_taken = 0;         // a flag on its way to the host (take_flag)
__device__ int g_paged_status = 0;  // XB_ERR_TIMEOUT once a bounded wait ran out (xb_device_status)
constexpr uint64_t kWaitLimit = 2000000000ull;  // 2 s per wait: far above any legitimate wait

// ----------------------------------------------------------------------------- page copies

// pages[o, dst[i]] = pages[o, src[i]] for every outer index o (layer, K or V):
// a plain copy, 2 bytes moved per byte of page, HBM-bound.  The host has
// checked that no destination is a source or named twice, so the pairs may
// run in any order.  The pairs travel as kernel parameters: no upload, no
// device buffer whose lifetime a captured graph would have to share.  A thread
// moves four 16-byte vectors 256 apart (four loads in flight), a CTA 16 KB of
// the outer slab's n * vpp vectors.  2500 pages of 4 KB in 48 slabs take 164 us,
// 0.91 of the measured copy rate; 4 pages 2.2 us, the launch.
constexpr int kCopyPairs = 500;  // 4000 bytes of parameters; larger lists, and very large pages, take several launches
template <int N>
struct CopyPairs {
  int32_t src[N], dst[N];
};

template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyPairs<N> pairs, uint8_t* base,
                                                         int64_t outer_stride, int64_t page_stride, uint32_t vpp,
                                                         uint32_t total) {
  pdl_wait();
  pdl_trigger();
  uint8_t* slab = base + (int64_t)blockIdx.y * outer_stride;
  const uint32_t first = blockIdx.x * 1024u + threadIdx.x;
  int4 v[4];
  int64_t to[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t i = first + u * 256u;
    to[u] = -1;
    if (i < total) {
      const uint32_t p = i / vpp, at = i - p * vpp;
      to[u] = (int64_t)pairs.dst[p] * page_stride + (int64_t)at * 16;
      v[u] = __ldcs(reinterpret_cast<const int4*>(slab + (int64_t)pairs.src[p] * page_stride + (int64_t)at * 16));
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (to[u] >= 0) *reinterpret_cast<int4*>(slab + to[u]) = v[u];
}

// ----------------------------------------------------------------------------- RoPE + page write

struct Pages {  // K or V pages: element strides of page, head and row; rows of D contiguous elements
  bf16* p;
  int64_t page, head, row;
};

struct RopeArgs {
  const bf16* qkv;
  const float *cos_t, *sin_t;
  bf16* q;
  Pages k, v;
  const int32_t *table, *q_start, *kv_len;
  int64_t ld_qkv, ld_q, ld_table, rope_rows;
  int T, B, H, KVH, D, page_size, max_pages, n_pages;
};

// One warp per packed token.  A lane keeps one group of 8 dims (and the 8 of
// the other half they rotate with) and walks the head slots, so it reads its
// 32 table values once; 16-byte loads and stores.  HBM-bound: every element is
// read and written once.  The row does not depend on where the token belongs,
// so up to three of a lane's slots are requested before the search for the
// token's sequence, which all lanes do together (32 starts a step).  Products
// and sums are rounded separately in fp32, as examples/qwen2_5/kernels/rope.py:
// 63-66 and the contiguous kernel do: the same bits.  36500 tokens of 14 + 2 x 2
// heads take 33.8 us, 5.5 TB/s (0.85 of the measured copy).  Measured: four
// slots ahead in 94 registers 48.2 us, two in 64 41.0, loads after the search
// 47.1, three in 80 39.6; stores marked as streaming 35.8; then CTAs of two
// warps instead of eight 33.8 (four 34.2, 24 46.0): a CTA's place is taken again
// as soon as its own few tokens are done.
__global__ void __launch_bounds__(64, 12) paged_rope_kv_kernel(const RopeArgs a, int* __restrict__ bad) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x * 2 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= a.T) return;
  const int half = a.D / 2, groups = half / 8;  // groups of 8 dims of a half; divides 32
  const int c = (lane % groups) * 8, slot0 = lane / groups, step = 32 / groups;
  const int slots = a.H + 2 * a.KVH;
  const bf16* x = a.qkv + (int64_t)t * a.ld_qkv + c;
  constexpr int kAhead = 3;
  Vec16<bf16> u[kAhead], w[kAhead];
  auto load = [&](int first) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int slot = first + i * step;
      if (slot < slots) {
        u[i] = ld16_stream(x + slot * a.D);
        w[i] = ld16_stream(x + slot * a.D + half);
      }
    }
  };
  load(slot0);
  // the last b with q_start[b] <= t; empty sequences share their start with the next one
  int b = 0;
  for (int len = a.B + 1;;) {
    const int stride = (len + 31) / 32;
    const bool le = lane * stride < len && __ldg(a.q_start + b + lane * stride) <= t;
    const int n = __popc(__ballot_sync(0xffffffffu, le));
    if (n == 0) return;  // a row before the first sequence
    b += (n - 1) * stride;
    if (stride == 1) break;
    len = min(stride, len - (n - 1) * stride);
  }
  if (b >= a.B) return;  // behind the last sequence
  const int end = __ldg(a.q_start + b + 1);
  if (end <= t) return;  // (starts that do not ascend)
  const int64_t pos = (int64_t)__ldg(a.kv_len + b) - ((int64_t)end - t);
  const int64_t slot_page = pos >= 0 ? (int64_t)((uint32_t)pos / (uint32_t)a.page_size) : -1;  // pos < 2^31
  int id = -1;
  if (pos >= 0 && slot_page < a.max_pages) id = __ldg(a.table + (int64_t)b * a.ld_table + slot_page);
  const bool page_ok = id >= 0 && id < a.n_pages;
  if (!page_ok && lane == 0) atomicExch(bad, 1);
  if (pos < 0) return;
  const bool rotate = a.cos_t != nullptr;
  if (rotate && pos >= a.rope_rows) {
    if (lane == 0) atomicExch(bad, 1);
    return;
  }
  const int row = (int)(pos - slot_page * a.page_size);
  float cl[8], ch[8], sl[8], sh[8];
  if (rotate) {
    const float* cr = a.cos_t + pos * a.D;
    const float* sr = a.sin_t + pos * a.D;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      *reinterpret_cast<float4*>(&cl[e]) = __ldg(reinterpret_cast<const float4*>(cr + c + e));
      *reinterpret_cast<float4*>(&ch[e]) = __ldg(reinterpret_cast<const float4*>(cr + c + half + e));
      *reinterpret_cast<float4*>(&sl[e]) = __ldg(reinterpret_cast<const float4*>(sr + c + e));
      *reinterpret_cast<float4*>(&sh[e]) = __ldg(reinterpret_cast<const float4*>(sr + c + half + e));
    }
  }
  for (int first = slot0;;) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int slot = first + i * step;
      if (slot >= slots) break;
      if (rotate && slot < a.H + a.KVH) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x0 = __bfloat162float(u[i].v[e]), x1 = __bfloat162float(w[i].v[e]);
          u[i].v[e] = __float2bfloat16_rn(__fadd_rn(__fmul_rn(x0, cl[e]), __fmul_rn(-x1, sl[e])));
          w[i].v[e] = __float2bfloat16_rn(__fadd_rn(__fmul_rn(x1, ch[e]), __fmul_rn(x0, sh[e])));
        }
      }
      bf16* dst;
      if (slot < a.H) {
        dst = a.q + (int64_t)t * a.ld_q + slot * a.D;
      } else {
        if (!page_ok) continue;
        const bool is_k = slot < a.H + a.KVH;
        const Pages& pg = is_k ? a.k : a.v;
        dst = pg.p + id * pg.page + (slot - a.H - (is_k ? 0 : a.KVH)) * pg.head + row * pg.row;
      }
      st16_stream(dst + c, u[i]);
      st16_stream(dst + half + c, w[i]);
    }
    first += kAhead * step;
    if (first >= slots) break;
    load(first);
  }
}

// ----------------------------------------------------------------------------- attention: the work and its split
//
// A unit of work is one (sequence, KV head, query tile): `tpt` consecutive
// new tokens of a sequence times the n_rep query heads that share the KV head,
// which are the rows of one matrix tile, so every key and value is read once
// for all of them.  Query tile j of a sequence with `base` earlier positions
// sees base + min(tpt (j + 1), n) keys (none where that is negative); its weight
// is those keys plus `over`, what starting and finishing a unit costs in keys
// (csrc/paged_walk.cuh has the arithmetic).  All units laid end to end
// are one line of weight `total`; CTA c takes the piece [c share, (c + 1) share)
// of it, whatever unit boundaries lie inside, so the CTAs finish together
// however uneven the batch is (in the few-row kernel every warp has a piece).
// A cut close to a unit's first or last key moves to the unit's boundary (both
// neighbours move it the same way).  A unit that one CTA covers alone is
// written at once; one that spans several leaves a partial (O, max, sum) per
// CTA in the workspace, and a second small kernel joins them in CTA order
// (fixed order: repeatable bits).  Joining inside the first kernel, by the CTA
// in which a unit ends after waiting for the others' flags, saved the host a
// launch but no time on the GPU (64 sequences 11.0 -> 11.8 us).  The weights
// are a closed form, so a CTA finds its piece with one scan over the sequences
// and a binary search inside one, from lengths that only the device knows.

struct AttnArgs : Line {
  const bf16* q;
  bf16* out;
  const int32_t* table;
  float* ws;  // [2 G] partials, then G Meta
  int64_t ld_q, ld_out, ld_table;
  int n_pages, box_rows;
  uint32_t rep_magic;  // ceil(2^16 / n_rep)
  float scale_log2;
  int *bad, *status;
};

// What the joining kernel needs of CTA c: the unit that starts in c and goes on, and the CTA it ends in.
struct Meta {
  int last, token, rows, kvh;  // last < 0: no such unit
};

// r / n_rep for a row r < 128: the product is above the quotient by less than r / 2^16 < 1 / n_rep.
__device__ __forceinline__ int row_token(const AttnArgs& a, int r) { return (int)(((uint32_t)r * a.rep_magic) >> 16); }

// Weight of the whole line and, for the piece that starts at `first` + i times
// the share (i < N), the sequence that holds its start.  Every thread of the
// block calls this; sums and found[N] are shared.  One scan over the sequences
// when the block has a thread for each, two otherwise.  Returns the share.
template <int THREADS, int N, typename I>
__device__ __forceinline__ I find_pieces(const AttnArgs& a, int pieces, int first, I (*sums)[THREADS / 32],
                                         Found<I>* found, I* total_out) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x < N) found[threadIdx.x].b = -1;
  I total = 0, share = 0, start = 0, c = 0;
  Seq<I> q;
  for (int pass = 0; pass < 2; ++pass) {
    I run = 0;
    for (int b0 = 0; b0 < a.B; b0 += THREADS) {
      const int b = b0 + threadIdx.x;
      if (pass == 0 || a.B > THREADS) {
        c = 0;
        if (b < a.B) {
          q = load_seq<I>(a, b);
          c = q.perh * a.KVH;
        }
        I s = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const I v = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += v;
        }
        const int buf = (b0 / THREADS) & 1;
        if (lane == 31) sums[buf][warp] = s;
        __syncthreads();
        start = run + s - c;  // this sequence's first point
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) {
          const I v = sums[buf][i];
          if (i < warp) start += v;
          run += v;
        }
      }
      if (pass == 1 && c > 0) {
        I lo = first * share;
#pragma unroll
        for (int i = 0; i < N; ++i, lo += share)
          if (start <= lo && lo - start < c) found[i] = Found<I>{start, b, q.s0, q.n, q.len};
      }
    }
    if (pass == 0) {
      if (a.B > THREADS) __syncthreads();
      total = run;
      share = share_of(a, total, pieces);
    }
  }
  __syncthreads();
  *total_out = total;
  return share;
}

// ----------------------------------------------------------------------------- attention: few rows (mma.sync)
//
// For batches whose sequences bring few tokens each (decoding, verification of
// drafted tokens): at most 8 or 16 rows per unit, so the kernel is bound by
// reading K and V.  Every warp of the grid has a piece of the line of its own
// and runs through it alone: its lanes issue the TMA loads of a 32-key tile's
// page rows (128-byte swizzle) into one of the warp's two buffers, the next
// unit's tiles while the present one is computed, and the warp keeps an online
// softmax (running max and sum in fp32, P rounded to bf16 for P V as in the
// contiguous kernels).  8 warps x 2 buffers x 8 KB keep up to 128 KB per SM in
// flight.  The products run transposed on mma.sync m16n8k16, S^T = K Q^T and
// O^T = V^T P^T: keys and dims fill the 16 rows and the query rows the 8
// columns, so 8 rows take 16 MMAs a tile; with the query rows in the 16-row
// place they took 32, and those were the longest part of a short call (0.7 of
// the 1.4 us of two tiles).  A unit inside one warp's piece goes straight to
// the output; parts of one that spans warps of the CTA meet in shared memory
// after the last barrier, and what spans CTAs goes on to the joining
// kernel.  Calls of few keys are bound by latency and by fetching instructions
// (each line is cold in a new launch): every long piece of code is there once.
constexpr int kHD = 64;
constexpr int kTK = kFewTK;
constexpr int kTileBytes = kTK * kHD * 2;  // one K or V tile
constexpr int kQueue = 4;                  // segments a warp's requests may be ahead of its computation
constexpr int kPartLd = kHD + 4;           // row pitch of a partial in shared memory: conflict-free stores
// Warps x buffers of the 8-row kernel, 64 sequences of 576 keys / 160 long ones:
// 8 x 2 11.0 / 86.1 us, 8 x 3 11.0 / 90.2, 12 x 2 12.1 / 87.4, 16 x 1 13.1 / 86.5,
// 12 x 1 12.3 / 85.8, 8 x 1 11.1 / 93.8, 6 x 3 11.3 / 91.7, 4 x 4 12.6 / 116.
template <int ROWS>
struct FewCfg {
  static constexpr int kWarps = kFewWarps, kBufs = 2;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRing = kBufs * 2 * kTileBytes;  // of one warp
  static constexpr int kHead = ROWS * kPartLd * 4;      // a warp's kind 0 partial; kind 1 goes into its own ring
  static constexpr int kSmem = kWarps * (kRing + kHead) + 1024;
  static_assert(kHead <= kRing && kSmem <= 224 * 1024, "shared memory");
};

struct alignas(64) KvMaps {
  CUtensorMap k, v;  // [n_pages][KVH][page][64], box {64, box_rows, 1, 1}
};

__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t c0,
                                            int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::
          "r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

// True in one lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}

// transposes an 8 x 8 matrix of 16-bit elements held one row per four lanes
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// floats of one partial: O [rows][64], then max [rows], then sum [rows]
__host__ __device__ constexpr int64_t part_floats(int rows) { return (int64_t)rows * (kHD + 2); }

__device__ __forceinline__ void store_out4(const AttnArgs& a, int token, int kvh, int r, int d, float4 v) {
  const int tok = row_token(a, r);
  bf16* op = a.out + (int64_t)(token + tok) * a.ld_out + (kvh * a.n_rep + r - tok * a.n_rep) * kHD + d;
  uint2 pk;
  pk.x = pack2(v.x, v.y);
  pk.y = pack2(v.z, v.w);
  *reinterpret_cast<uint2*>(op) = pk;
}

template <int ROWS, typename I>
__global__ void __launch_bounds__(FewCfg<ROWS>::kThreads, 1) paged_attn_few_kernel(const __grid_constant__ KvMaps maps,
                                                                        const AttnArgs a) {
  using C = FewCfg<ROWS>;
  constexpr int kWarps = C::kWarps, kBufs = C::kBufs;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[kWarps][kBufs];
  __shared__ I sums[2][kWarps];
  __shared__ Found<I> found[kWarps];
  // A warp's parts of units that it does not cover alone: kind 0 of one that
  // started before its piece, kind 1 of one that goes on behind it.
  __shared__ Segment part[2][kWarps];
  __shared__ float part_m[2][kWarps][ROWS], part_l[2][kWarps][ROWS];
  __shared__ uint32_t comes, ends0, opens;  // one bit per warp: has a kind 0, its unit ends there, has a kind 1
  __shared__ Segment queue[kWarps][kQueue];
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  constexpr int NT = ROWS / 8;  // 8-row column tiles
  const uint32_t base_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base_u32 - smem_u32(smem_raw));
  const uint32_t ring = base_u32 + warp * C::kRing;
  // O of the two kinds of parts: the first beside the ring, the second, the
  // last thing a warp does, in its ring
  auto part_o = [&](int kind, int w_) -> float* {
    return reinterpret_cast<float*>(kind == 0 ? smem + kWarps * C::kRing + w_ * C::kHead : smem + w_ * C::kRing);
  };
  if (lane == 0) {
    for (int i = 0; i < kBufs; ++i) mbar_init(&full[warp][i], 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) {
    abort_flag = 0;
    comes = ends0 = opens = 0;
    prefetch_tmap(&maps.k);
    prefetch_tmap(&maps.v);
  }
  pdl_wait();
  pdl_trigger();
  I total;
  const I share =
      find_pieces<C::kThreads, kWarps, I>(a, gridDim.x * kWarps, blockIdx.x * kWarps, sums, found, &total);
  Meta* meta = reinterpret_cast<Meta*>(a.ws + 2 * (int64_t)gridDim.x * part_floats(kFewRows));
  if (found[0].b < 0) {  // no warp of this CTA has work
    if (threadIdx.x == 0) meta[blockIdx.x].last = -1;
    return;
  }
  if (found[warp].b >= 0) {
    const bool leader = elect_one();
    // This thread's rows: 8 n + 2 t and the next one, and the tokens they belong to
    int tok[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) tok[n][e] = row_token(a, 8 * n + 2 * t + e);
    // The walk runs with the requests; the computation follows through a small
    // queue of segments.
    Walk<I> wi;
    Segment si, sc;
    place(a, wi, (int)blockIdx.x * kWarps + warp, share, total, found[warp]);
    bool fresh = true, more_i = true;
    si.t1 = 0;
    sc.t1 = 0;
    int ni = 0;  // next tile to request
    uint32_t pushed = 0, popped = 0;
    uint32_t use = 0, issued = 0;  // tiles read / requested: buffer n % kBufs, parity (n / kBufs) & 1
    bool dead = false;  // a wait ran out: no more loads, the output is not valid
    // 32 entries of the page table row from page `win` on, one per lane: one
    // latency for many tiles
    uint32_t win = 0;
    int win_id = 0;
    uint32_t pi = 0;  // page index and row where the next tile starts
    int row = 0;
    auto window = [&](uint32_t first) {
      win = first;
      const uint32_t p = first + lane;
      win_id = p * (uint64_t)a.page_size < (uint32_t)si.keys ? __ldg(a.table + si.b * a.ld_table + p) : -1;
    };
    auto enter = [&]() {  // the first tile of a segment
      pi = (uint32_t)(ni * kTK) / (uint32_t)a.page_size;
      row = ni * kTK - (int)pi * a.page_size;
      window(pi);
    };
    // page piece by page piece (a piece never crosses a page), in uniform registers
    auto request = [&]() {
      const uint32_t buf = issued % kBufs;
      const int have = min(kTK, si.keys - ni * kTK);
      const int nb = (have + a.box_rows - 1) / a.box_rows;
      if (leader) mbar_arrive_expect_tx(&full[warp][buf], (uint32_t)(nb * a.box_rows * kHD * 2 * 2));
      uint32_t dst = ring + buf * 2 * kTileBytes;
      for (int i = 0; i < nb; ++i) {
        if (pi - win >= 32u) window(pi);
        int id = __shfl_sync(0xffffffffu, win_id, (int)(pi - win));
        if (id < 0 || id >= a.n_pages) {  // reads as zeros: a coordinate past the pool
          if (leader) atomicExch(a.bad, 1);
          id = a.n_pages;
        }
        if (leader) {
          tma_load_4d(dst, &maps.k, &full[warp][buf], 0, row, si.kvh, id);
          tma_load_4d(dst + kTileBytes, &maps.v, &full[warp][buf], 0, row, si.kvh, id);
        }
        dst += a.box_rows * kHD * 2;
        row += a.box_rows;
        if (row == a.page_size) {
          row = 0;
          ++pi;
        }
      }
      __syncwarp();
      ++issued;
      ++ni;
    };
    uint32_t qb[NT][4][2];
    auto load_q = [&]() {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = 8 * n + g, tk = row_token(a, r);
        const bf16* p = a.q + (int64_t)(sc.token + tk) * a.ld_q + (sc.kvh * a.n_rep + r - tk * a.n_rep) * kHD + 2 * t;
        const bool in = r < sc.rows;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          qb[n][kk][0] = in ? *reinterpret_cast<const uint32_t*>(p + kk * 16) : 0u;
          qb[n][kk][1] = in ? *reinterpret_cast<const uint32_t*>(p + kk * 16 + 8) : 0u;
        }
      }
    };
    int pos[NT][2], first_pos = 0;  // the last keys that this thread's rows see, and that every row sees
    int tile = 0;
    float o[NT][4][4], m[NT][2], l[NT][2];
    for (;;) {
      while (more_i) {
        if (ni < si.t1) {
          if (issued - use == kBufs) break;
          request();
        } else {
          if (pushed - popped == kQueue) break;
          more_i = (fresh || next_unit(a, wi)) && segment<kTK>(a, wi, si);
          fresh = false;
          if (!more_i) break;
          if (lane == 0) queue[warp][pushed % kQueue] = si;
          __syncwarp();
          ++pushed;
          ni = si.t0;
          if (ni < si.t1) enter();
          if (tile < sc.t1) break;  // compute meanwhile
        }
      }
      if (tile < sc.t1) {
        const uint32_t buf = use % kBufs;
        const bool landed = mbar_wait(&full[warp][buf], (use / kBufs) & 1, kWaitLimit, &abort_flag);
        if (__any_sync(0xffffffffu, !landed)) {
          atomicExch(a.status, XB_ERR_TIMEOUT);
          abort_flag = 1;
          dead = true;
          break;
        }
        const int k0 = tile * kTK;
        const uint32_t sk = ring + buf * 2 * kTileBytes, sv = sk + kTileBytes;
        const int have = min(kTK, sc.keys - k0);
        if (have < kTK) {
          // values behind the last key hold whatever the page or buffer held: a
          // NaN there would survive its zero weight
          for (int i = have * 8 + lane; i < kTK * 8; i += 32)
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + i * 16), "r"(0) : "memory");
          fence_proxy_async_smem();  // before a later TMA write to the buffer
          __syncwarp();
        }
        // S^T = K Q^T: keys are the MMA's 16 rows, query rows its 8 columns
        float s[NT][2][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int n = 0; n < NT; ++n) s[n][mt][0] = s[n][mt][1] = s[n][mt][2] = s[n][mt][3] = 0.0f;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const int mi = lane >> 3, r = mt * 16 + (mi & 1) * 8 + (lane & 7), c = 2 * kk + (mi >> 1);
            uint32_t ka[4];
            ldsm4(ka, sk + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816(s[n][mt], ka, qb[n][kk][0], qb[n][kk][1]);
          }
        }
        if (k0 + kTK - 1 > first_pos) {  // some row does not see the whole tile
#pragma unroll
          for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = k0 + mt * 16 + g + (e >> 1) * 8;
#pragma unroll
              for (int n = 0; n < NT; ++n)
                if (key > pos[n][e & 1]) s[n][mt][e] = -INFINITY;
            }
        }
        uint32_t pb[NT][4];  // P as the B operand of O^T = V^T P^T, 8 keys each
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float base[2], al[2];
          bool moved = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            // raw scores: the scale is positive, so their maximum scales to the scaled ones'
            float mx = fmaxf(fmaxf(s[n][0][e], s[n][0][e + 2]), fmaxf(s[n][1][e], s[n][1][e + 2]));
#pragma unroll
            for (int o_ = 4; o_ <= 16; o_ <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o_));
            const float mn = fmaxf(m[n][e], mx * a.scale_log2);
            base[e] = mn == -INFINITY ? 0.0f : mn;
            al[e] = ex2_approx(m[n][e] - base[e]);
            moved |= mn > m[n][e];
            m[n][e] = mn;
          }
          if (__any_sync(0xffffffffu, moved)) {
            l[n][0] *= al[0];
            l[n][1] *= al[1];
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              o[n][mt][0] *= al[0];
              o[n][mt][1] *= al[1];
              o[n][mt][2] *= al[0];
              o[n][mt][3] *= al[1];
            }
          }
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[n][mt][e] = ex2_approx(fmaf(s[n][mt][e], a.scale_log2, -base[e & 1]));
              l[n][e & 1] += s[n][mt][e];
            }
            pb[n][2 * mt] = transpose8(pack2(s[n][mt][0], s[n][mt][1]));
            pb[n][2 * mt + 1] = transpose8(pack2(s[n][mt][2], s[n][mt][3]));
          }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {  // dims 16 mt .. 16 mt + 15
            const int mi = lane >> 3, r = ks * 16 + (mi >> 1) * 8 + (lane & 7), c = 2 * mt + (mi & 1);
            uint32_t va[4];
            ldsm4_t(va, sv + r * 128 + ((c ^ (r & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma_16816(o[n][mt], va, pb[n][2 * ks], pb[n][2 * ks + 1]);
          }
        ++use;
        ++tile;
        __syncwarp();  // the buffer is read: it takes a tile further on
        if (tile < sc.t1) continue;
      } else {
        // the next segment
        if (popped == pushed) break;
        sc = queue[warp][popped % kQueue];
        ++popped;
        __syncwarp();
        load_q();
        tile = sc.t0;
        first_pos = min(sc.first_pos, sc.keys - 1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            pos[n][e] = min(sc.first_pos + tok[n][e], sc.keys - 1);
            m[n][e] = -INFINITY;
            l[n][e] = 0.0f;
          }
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) o[n][mt][0] = o[n][mt][1] = o[n][mt][2] = o[n][mt][3] = 0.0f;
        }
        if (tile < sc.t1) continue;
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int o_ = 4; o_ <= 16; o_ <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o_);
      if (sc.starts && sc.ends) {
        // neighbours in g swap a row each, so that a thread stores two dims of one row
        const int odd = g & 1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float i0 = l[n][0] == 0.0f ? 0.0f : 1.0f / l[n][0];  // no key: zeros
          const float i1 = l[n][1] == 0.0f ? 0.0f : 1.0f / l[n][1];
          const int r = 8 * n + 2 * t + odd, tk = odd ? tok[n][1] : tok[n][0];
          bf16* p = a.out + (int64_t)(sc.token + tk) * a.ld_out + (sc.kvh * a.n_rep + r - tk * a.n_rep) * kHD + (g & 6);
#pragma unroll
          for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float x0 = o[n][mt][2 * h] * i0, x1 = o[n][mt][2 * h + 1] * i1;
              const float got = __shfl_xor_sync(0xffffffffu, odd ? x0 : x1, 4);
              const uint32_t pk = odd ? pack2(got, x1) : pack2(x0, got);
              if (r < sc.rows) *reinterpret_cast<uint32_t*>(p + mt * 16 + h * 8) = pk;
            }
        }
      } else {
        const int kind = sc.starts ? 1 : 0;
        float* po = part_o(kind, warp);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * n + 2 * t + e;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
              po[r * kPartLd + mt * 16 + g] = o[n][mt][e];
              po[r * kPartLd + mt * 16 + g + 8] = o[n][mt][e + 2];
            }
            if (g == 0) {
              part_m[kind][warp][r] = m[n][e];
              part_l[kind][warp][r] = l[n][e];
            }
          }
        if (lane == 0) {
          part[kind][warp] = sc;
          atomicOr(kind ? &opens : &comes, 1u << warp);
          if (!kind && sc.ends) atomicOr(&ends0, 1u << warp);
        }
      }
    }
    if (dead) {  // loads still in flight land before the CTA's shared memory is given up
      uint64_t deadline = 0;
      for (; use < issued; ++use)
        mbar_wait_deadline(&full[warp][use % kBufs], (use / kBufs) & 1, &deadline, kWaitLimit);
    }
  }
  __syncthreads();
  // Chains of parts: one that came in from the CTA before (its parts start with
  // warp 0's kind 0), and one from every warp with a kind 1.  A chain goes on
  // through the kind 0 of the next warps until one ends the unit, or leaves
  // the CTA.  The CTA's threads form a team per chain (2, 4 or 8 of them when
  // there are several); a thread has one row's 16-byte column at a time.
  uint32_t chains = (opens << 1) | (comes & 1u);
  const int count = __popc(chains), teams = count <= 1 ? 1 : count == 2 ? 2 : count <= 4 ? 4 : 8;
  const int size = C::kThreads / teams, team = threadIdx.x / size;
  bool open_unit = false;
  for (int n = 0; chains; chains &= chains - 1, ++n) {
    const int c = __ffs((int)chains) - 2;  // the warp of the kind 1, or -1
    const uint32_t ahead = ends0 & (0xffffffffu << (c + 1));
    const int first = max(c, 0), end = ahead ? __ffs((int)ahead) - 1 : kWarps - 1;
    const Segment& p = part[c >= 0][first];
    const bool whole = c >= 0 && ahead;
    open_unit |= c >= 0 && !ahead;
    if ((n & (teams - 1)) != team) continue;
    for (int i = threadIdx.x % size; i < p.rows * 16; i += size) {
      const int r = i / 16, d = (i % 16) * 4;
      float M = -INFINITY, l = 0.0f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = first; k <= end; ++k) {
        const float m = part_m[k == c][k][r], mn = fmaxf(M, m), base = mn == -INFINITY ? 0.0f : mn;
        const float f0 = ex2_approx(M - base), f = ex2_approx(m - base);
        const float4 v = *reinterpret_cast<const float4*>(part_o(k == c, k) + r * kPartLd + d);
        acc.x = acc.x * f0 + v.x * f;
        acc.y = acc.y * f0 + v.y * f;
        acc.z = acc.z * f0 + v.z * f;
        acc.w = acc.w * f0 + v.w * f;
        l = l * f0 + part_l[k == c][k][r] * f;
        M = mn;
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        store_out4(a, p.token, p.kvh, r, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
      } else {
        float* out_part = a.ws + (2 * (int64_t)blockIdx.x + (c >= 0)) * part_floats(kFewRows);
        *reinterpret_cast<float4*>(out_part + r * kHD + d) = acc;
        if (d == 0) {
          out_part[kFewRows * kHD + r] = M;
          out_part[kFewRows * kHD + kFewRows + r] = l;
          if (r == 0 && c >= 0) meta[blockIdx.x] = Meta{p.last / kWarps, p.token, p.rows, p.kvh};
        }
      }
    }
  }
  if (!open_unit && threadIdx.x == 0) meta[blockIdx.x].last = -1;
}

// ----------------------------------------------------------------------------- attention: many rows (tcgen05)
//
// For batches whose sequences bring many tokens (prompts, chunks, mixed
// steps): units of up to 128 rows (tpt = 128 / n_rep tokens), key tiles of 64.
// Two persistent CTAs per SM, each walking its piece of the line:
//   warp 0     walks the piece, tells the others its segments through a small
//              ring, loads each unit's Q (two buffers) and streams K / V page
//              rows into a ring of four tiles (one lane per page piece, TMA,
//              128-byte swizzle);
//   warp 1     issues S_g = Q K_g^T into one of three 64-column TMEM buffers;
//   warp 2     issues O += P_g V_g; P_g is the MMA's A operand straight from
//              TMEM.  Values behind the last key are zeroed first;
//   warps 4-7  softmax, one query row per thread: scores from TMEM, bf16(P)
//              back into the first half of the same TMEM buffer (warp 3 only
//              makes the warpgroups whole, which trade registers).
// Keeping P in TMEM takes its write and its 16 KB operand read per tile off
// shared memory, whose 128 bytes a clock would otherwise be the first limit
// (Q, K, V and P reads, P writes and the TMA's writes: 640 of them a tile,
// against 512 clocks of exponentials).  S runs up to two tiles ahead, so the
// softmax never waits for scores.  One warp issuing both products held it up:
// each of a tile's eight dependent N = 64 MMAs takes some 66 clocks to issue and
// each commit some 80 (4096 tokens at position 28672: 730 us, two warps 713).
// O accumulates in TMEM relative to a per-row base that moves only when a
// tile's maximum exceeds it by more than 2^8 (bf16 keeps its 8 bits at any
// scale), and only then is O rescaled.  Warps whose 32 rows are all past the
// unit's (a single token of a decoding sequence in a mixed batch) only pass the
// tiles on.  Every wait is bounded; a timeout sets the status word, drains what
// is in flight and ends.
//
// What bounds it: the same 4096 tokens (14 heads on 2) take 666 us, 677
// TFLOP/s, at 1.75 to 1.8 of 1.965 GHz (power).  Of the 1433 clocks a tile takes
// the CTA that came first to its SM (the second: 1644) some 800 are the 64
// exponentials of each row, which at 16 a clock and SM would be 512 alone;
// waiting (110, the barrier's own latency: the scores are always there),
// TMEM load (65), maximum (230) and store (45) come in between, and
// the two CTAs fill each other's gaps only in part.  Measured no faster: maxima
// only where a row's sum of P grows past 2^16 (677 us, prompts 59.8 against
// 59.7), the next tile's scores loaded during the exponentials (713), key tiles
// of 128 with one score buffer (760 where 64 took 730), four CTAs per SM with
// one score buffer (757), three (862), longer pieces for an SM's first CTA
// (prompts 56.2 against 58.4, but the chunk 676), one in eight exponentials as a
// polynomial on the FMA pipe (652, but prompts 57.4 against 56.3).
constexpr int kTcRows = 128;
constexpr int kTcStages = 4;
constexpr int kTcSegs = 4;  // segments published ahead
constexpr int kTcQBytes = kTcRows * kHD * 2;
constexpr int kTcTileBytes = kTcTK * kHD * 2;  // one K or V tile
constexpr int kTcSmem = 2 * kTcQBytes + kTcStages * 2 * kTcTileBytes + 1024;
constexpr int kTcThreads = 256;
constexpr int kTcFewRegs = 64, kTcSoftmaxRegs = 192;  // a thread, of the two warpgroups; 128 each at launch

struct alignas(64) TcMaps {
  CUtensorMap q;  // [T][n_head][64], box {64, n_rep, tpt}
  CUtensorMap k, v;
};

// D[tmem] (+)= A[tmem] x B[smem desc], kind::f16; A: lane = row, 32-bit column = two consecutive K elements
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(
          d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 columns of the warp's TMEM lanes
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Two fp32 at a time: one instruction for a pair, each rounded as on its own.
__device__ __forceinline__ float2 fma2(float2 x, float2 y, float2 z) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n"
      " fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 x, float2 y) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return d;
}

__device__ __forceinline__ float2 mul2(float2 x, float2 y) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
  return d;
}

template <typename I>
__global__ void __launch_bounds__(kTcThreads, 2) paged_attn_tc_kernel(const __grid_constant__ TcMaps maps,
                                                                      const AttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], drain_bar[2], o_empty;
  __shared__ __align__(8) uint64_t s_full[3], p_full[3];
  __shared__ __align__(8) uint64_t kv_full[kTcStages], pv_done[kTcStages];
  __shared__ __align__(8) uint64_t seg_full[kTcSegs], seg_empty[kTcSegs];
  __shared__ Segment segs[kTcSegs];  // rows == 0: the end
  __shared__ I sums[2][kTcThreads / 32];
  __shared__ Found<I> found[1];
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t sQ = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sKV = sQ + 2 * kTcQBytes;

  if (threadIdx.x == 0) {
    mbar_init(&o_empty, 128);  // a unit's O read by the softmax warps
    for (int i = 0; i < kTcSegs; ++i) {
      mbar_init(&seg_full[i], 1);
      mbar_init(&seg_empty[i], 6);  // the MMA warps and the four softmax warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&drain_bar[i], 1);
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 128);  // Q's buffer, which the output passes through, free
    }
    for (int i = 0; i < 3; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
    }
    for (int i = 0; i < kTcStages; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&pv_done[i], 1);  // P V accumulated into O: K, V and the tile's S buffer are free
    }
    abort_flag = 0;
    mbar_fence_init();
    prefetch_tmap(&maps.q);
    prefetch_tmap(&maps.k);
    prefetch_tmap(&maps.v);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_sh;  // S / P buffers at columns 0, 64 and 128, O at 192
  pdl_wait();
  pdl_trigger();

  auto fail = [&]() {
    atomicExch(a.status, XB_ERR_TIMEOUT);
    abort_flag = 1;
  };
  Meta* meta = reinterpret_cast<Meta*>(a.ws + 2 * (int64_t)gridDim.x * part_floats(kTcRows));
  I total;
  const I share = find_pieces<kTcThreads, 1, I>(a, gridDim.x, blockIdx.x, sums, found, &total);
  // A wait of a whole warp: the same answer in every lane (false: it ran out)
  auto wait_all = [&](uint64_t* bar, int phase) -> bool {
    if (__all_sync(0xffffffffu, mbar_wait(bar, phase & 1, kWaitLimit, &abort_flag))) return true;
    fail();
    return false;
  };
  // Segment number n for a consumer warp (all its lanes); false at the end or after a timeout
  auto take = [&](int n, Segment& s) -> bool {
    if (!wait_all(&seg_full[n % kTcSegs], n / kTcSegs)) return false;
    s = segs[n % kTcSegs];
    __syncwarp();
    if (lane == 0) mbar_arrive(&seg_empty[n % kTcSegs]);
    return s.rows > 0;
  };

  // Every MMA issued completes before TMEM is released (also after an abort)
  auto drain = [&](int which, bool any) {
    if (any && elect_one()) {
      tc_commit(&drain_bar[which]);
      uint64_t deadline = 0;
      if (!mbar_wait_deadline(&drain_bar[which], 0, &deadline, kWaitLimit)) fail();
    }
    __syncwarp();
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kTcFewRegs));
    if (warp == 0) {
      // ------------------------------------------------------------ walk and TMA producer
      uint32_t issued[kTcStages];
#pragma unroll
      for (int i = 0; i < kTcStages; ++i) issued[i] = 0;
      const int boxes = kTcTK / a.box_rows;  // 1 .. 8 page pieces per tile; lane < boxes: K, the next ones: V
      const bool is_v = lane >= boxes;
      const int box = is_v ? lane - boxes : lane;
      const CUtensorMap* map = is_v ? &maps.v : &maps.k;
      const uint32_t q_bytes = (uint32_t)(a.tpt * a.n_rep * kHD * 2);
      int g = 0, lu = 0, n = 0;  // tiles, units (with tiles) and segments so far
      bool ok = true, open_unit = false;
      Walk<I> w;
      Segment s;
      bool more = found[0].b >= 0;
      if (more) {
        place(a, w, (int)blockIdx.x, share, total, found[0]);
        more = segment<kTcTK>(a, w, s);
      }
      auto publish = [&](int rows) -> bool {
        if (!wait_all(&seg_empty[n % kTcSegs], n / kTcSegs + 1)) return false;
        if (lane == 0) {
          segs[n % kTcSegs] = s;
          segs[n % kTcSegs].rows = rows;
          mbar_arrive(&seg_full[n % kTcSegs]);
        }
        __syncwarp();
        ++n;
        return true;
      };
      for (; more && ok; more = next_unit(a, w) && segment<kTcTK>(a, w, s)) {
        if (s.starts && !s.ends) {
          open_unit = true;
          if (lane == 0) meta[blockIdx.x] = Meta{s.last, s.token, s.rows, s.kvh};
        }
        ok = publish(s.rows);
        if (!ok) break;
        if (s.t0 >= s.t1) continue;
        // this lane's page of the first tile, fetched while Q's buffer may still be in use
        auto page_of = [&](int tile) -> int {
          const int key = tile * kTcTK + box * a.box_rows;
          if (lane >= 2 * boxes || key >= s.keys) return 0;
          return __ldg(a.table + s.b * a.ld_table + (uint32_t)key / (uint32_t)a.page_size);
        };
        int id = page_of(s.t0);
        ok = wait_all(&q_empty[lu & 1], (lu >> 1) + 1);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[lu & 1], q_bytes);
          asm volatile(
              "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
              "[%2];" ::"r"(sQ + (lu & 1) * kTcQBytes),
              "l"(reinterpret_cast<uint64_t>(&maps.q)), "r"(smem_u32(&q_full[lu & 1])), "r"(0), "r"(s.kvh * a.n_rep),
              "r"(s.token)
              : "memory");
        }
        ++lu;
        for (int j = s.t0; j < s.t1; ++j, ++g) {
          const int st = g % kTcStages;
          const int here = id;
          if (j + 1 < s.t1) id = page_of(j + 1);
          ok = wait_all(&pv_done[st], g / kTcStages + 1);
          if (!ok) break;
          const int have = min(kTcTK, s.keys - j * kTcTK);
          const int nb = (have + a.box_rows - 1) / a.box_rows;
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], (uint32_t)(nb * a.box_rows * kHD * 2 * 2));
          __syncwarp();
          if (lane < 2 * boxes && box < nb) {
            int page = here;
            if (page < 0 || page >= a.n_pages) {  // reads as zeros: a coordinate past the pool
              atomicExch(a.bad, 1);
              page = a.n_pages;
            }
            const uint32_t row = (uint32_t)(j * kTcTK + box * a.box_rows) % (uint32_t)a.page_size;
            tma_load_4d(sKV + st * 2 * kTcTileBytes + (is_v ? kTcTileBytes : 0) + box * a.box_rows * kHD * 2, map,
                        &kv_full[st], 0, (int)row, s.kvh, page);
          }
          issued[st] = g / kTcStages + 1;
        }
      }
      if (ok) publish(0);
      if (!open_unit && lane == 0) meta[blockIdx.x].last = -1;
      // every load issued must have landed before the CTA exits (also after an abort)
      if (lane == 0) {
        uint64_t deadline = 0;
        for (int i = lu > 2 ? lu - 2 : 0; i < lu; ++i)
          if (!mbar_wait_deadline(&q_full[i & 1], (i >> 1) & 1, &deadline, kWaitLimit)) fail();
#pragma unroll
        for (int st = 0; st < kTcStages; ++st)
          if (issued[st] && !mbar_wait_deadline(&kv_full[st], (issued[st] - 1) & 1, &deadline, kWaitLimit)) fail();
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------ S = Q K^T
      // The whole warp runs the loop and one elected lane issues: descriptors
      // differ by additions, ring positions by increments, all in uniform registers.
      constexpr uint32_t kIdS = umma_idesc(1, 1, 1, 0, 0, kTcRows, kTcTK);  // Q (K-major) x K tile (K-major)
      const bool leader = elect_one();
      const uint64_t dq = umma_desc_sw128(sQ, 16, 1024), dk = umma_desc_sw128(sKV, 16, 1024);
      bool ok = true;
      int g = 0, lu = 0;
      Segment s;
      for (int n = 0; ok && take(n, s); ++n) {
        const int tiles = __shfl_sync(0xffffffffu, s.t1 - s.t0, 0);
        if (tiles <= 0) continue;
        ok = wait_all(&q_full[lu & 1], lu >> 1);
        const uint64_t q = dq + (uint64_t)((lu & 1) * (kTcQBytes >> 4));  // descriptors count 16 bytes
        for (int j = 0; j < tiles && ok; ++j, ++g) {
          const int st = g % kTcStages, sb = g % 3;
          // S over the P of three tiles before, whose P V has completed
          ok = wait_all(&kv_full[st], g / kTcStages);
          if (ok && g >= 3) ok = wait_all(&pv_done[(g - 3) % kTcStages], (g - 3) / kTcStages);
          if (!ok) break;
          tc_fence_after();
          const uint64_t k = dk + (uint64_t)(st * (2 * kTcTileBytes >> 4));
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)  // head dim in steps of 16
              mma_f16(tmem + sb * 64, q + ks * 2, k + ks * 2, kIdS, ks > 0 ? 1u : 0u);
            tc_commit(&s_full[sb]);
          }
          __syncwarp();
        }
        ++lu;
      }
      drain(0, g > 0);
    } else if (warp == 2) {
      // ------------------------------------------------------------ O += P V
      constexpr uint32_t kIdO = umma_idesc(1, 1, 1, 0, 1, kTcRows, kHD);  // P (TMEM) x V tile (MN-major)
      const bool leader = elect_one();
      const uint64_t dv = umma_desc_sw128(sKV + kTcTileBytes, kTcTileBytes, 1024);
      bool ok = true;
      int g = 0, lu = 0;
      Segment s;
      for (int n = 0; ok && take(n, s); ++n) {
        const int tiles = __shfl_sync(0xffffffffu, s.t1 - s.t0, 0);
        if (tiles <= 0) continue;
        const int last_keys = __shfl_sync(0xffffffffu, s.keys - (s.t1 - 1) * kTcTK, 0);  // may be more than a tile
        for (int j = 0; j < tiles; ++j, ++g) {
          const int st = g % kTcStages, sb = g % 3;
          ok = wait_all(&kv_full[st], g / kTcStages);
          if (ok && j + 1 == tiles && last_keys < kTcTK) {
            // values behind the last key hold whatever the page or ring held: a
            // NaN there would survive its zero weight
            const uint32_t sv = sKV + st * 2 * kTcTileBytes + kTcTileBytes;
            for (int i = last_keys * 8 + lane; i < kTcTK * 8; i += 32)
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(sv + i * 16), "r"(0) : "memory");
            fence_proxy_async_smem();
            __syncwarp();
          }
          // P is written (and O rescaled where its base moved); a unit's first tile
          // starts O afresh, after the softmax has read the previous unit's
          ok = ok && wait_all(&p_full[sb], g / 3) && (j > 0 || lu == 0 || wait_all(&o_empty, lu - 1));
          if (!ok) break;
          tc_fence_after();
          const uint64_t d = dv + (uint64_t)(st * (2 * kTcTileBytes >> 4));
          if (leader) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)  // keys in steps of 16: 8 columns of P
              mma_f16_ts(tmem + 192, tmem + sb * 64 + ks * 8, d + ks * 128, kIdO, (ks > 0 || j > 0) ? 1u : 0u);
            tc_commit(&pv_done[st]);
          }
          __syncwarp();
        }
        ++lu;
      }
      drain(1, g > 0);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kTcSoftmaxRegs));
    // ------------------------------------------------------------ softmax: one query row per thread
    const int q4 = warp & 3;  // TMEM lane quarter
    const int r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    constexpr float kRebase = 8.0f;  // log2 of the largest P kept without rescaling
    const float2 scale2 = make_float2(a.scale_log2, a.scale_log2);
    bool ok = true;
    int g = 0, lu = 0;         // tiles, units with tiles
    uint32_t sb = 0, sph = 0;  // S buffer of tile g and its phase
    Segment s;
    for (int n = 0; ok && take(n, s); ++n) {
      const bool valid = r < s.rows;
      const bool warp_valid = q4 * 32 < s.rows;  // uniform: some row of this warp is the unit's
      const int seen = min(s.first_pos + row_token(a, r), s.keys - 1);  // the last key this row sees
      // key tiles that start up to here are seen whole by every row of the warp
      const int clear = __reduce_min_sync(0xffffffffu, valid ? seen : 0x7fffffff) - (kTcTK - 1);
      // m: the base of P (log2 units); rows past the unit's hold leftovers and have no say in moving bases
      float m = valid ? -INFINITY : INFINITY, l = 0.0f;
      const int g_end = g + max(s.t1 - s.t0, 0);
      if (!warp_valid)
        for (; ok && g < g_end; ++g) {
          ok = wait_all(&s_full[sb], sph);
          if (lane == 0) mbar_arrive(&p_full[sb]);
          if (++sb == 3) sb = 0, sph ^= 1;
        }
      for (int k0 = s.t0 * kTcTK; ok && g < g_end; k0 += kTcTK, ++g) {
        ok = wait_all(&s_full[sb], sph);
        if (!ok) break;
        tc_fence_after();
        float2 p[32];  // raw scores (the scale is positive: their maximum scales to the scaled ones')
        tmem_ld_32x32b_x32(tmem + sb * 64 + lane_off, *reinterpret_cast<uint32_t(*)[32]>(&p[0]));
        tmem_ld_32x32b_x32(tmem + sb * 64 + 32 + lane_off, *reinterpret_cast<uint32_t(*)[32]>(&p[16]));
        tmem_ld_wait();
        if (k0 > clear) {  // some row does not see the whole tile
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            if (k0 + 2 * c > seen) p[c].x = -INFINITY;
            if (k0 + 2 * c + 1 > seen) p[c].y = -INFINITY;
          }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = fmaxf(p[i].x, p[i].y);
#pragma unroll
        for (int c = 4; c < 32; ++c) mx[c & 3] = fmaxf(fmaxf(mx[c & 3], p[c].x), p[c].y);
        const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2;
        // a unit's first finite maximum moves the base from -inf
        if (__any_sync(0xffffffffu, mn > m + kRebase)) {
          const float to = fmaxf(m, mn), alpha = m == -INFINITY ? 0.0f : ex2_approx(m - to);
          l *= alpha;
          m = to;
          if (k0 > s.t0 * kTcTK) {  // O, with P_{g-1} V in it, to the new bases before P_g V adds to it
            ok = wait_all(&pv_done[(g - 1) % kTcStages], (g - 1) / kTcStages);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              uint32_t ov[16];
              tmem_ld_x16(tmem + 192 + h * 16 + lane_off, ov);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) ov[c] = __float_as_uint(__uint_as_float(ov[c]) * alpha);
              tmem_st_x16(tmem + 192 + h * 16 + lane_off, ov);
            }
          }
        }
        const float base = m == -INFINITY ? 0.0f : m;
        const float2 base2 = make_float2(-base, -base);
        float2 sum[2] = {make_float2(l, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 16; ++c) {  // P = exp2(S * scale - base)
            float2 e = fma2(p[16 * h + c], scale2, base2);
            e.x = ex2_approx(e.x);
            e.y = ex2_approx(e.y);
            sum[c & 1] = add2(sum[c & 1], e);
            pk[c] = pack2(e.x, e.y);
          }
          tmem_st_x16(tmem + sb * 64 + h * 16 + lane_off, pk);
        }
        l = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[sb]);
        if (++sb == 3) sb = 0, sph ^= 1;
      }
      if (!ok) break;
      const bool whole = s.starts && s.ends;
      float* part = a.ws + (2 * (int64_t)blockIdx.x + (s.starts ? 1 : 0)) * part_floats(kTcRows);
      if (valid && !whole) {
        part[kTcRows * kHD + r] = m;
        part[kTcRows * kHD + kTcRows + r] = l;
      }
      if (s.t0 >= s.t1) {  // no key in this part: zeros
        if (valid)
          for (int c = 0; c < 16; ++c) {
            const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
            if (!whole) *reinterpret_cast<float4*>(part + r * kHD + c * 4) = zero;
            else store_out4(a, s.token, s.kvh, r, c * 4, zero);
          }
        continue;
      }
      // Rows pass through the unit's own Q buffer (its scores are done), so
      // that a store instruction writes whole 128-byte rows: a row per thread
      // took 1.6 us a unit.  16-byte chunk c of row i at c ^ (i & 7).  What does
      // not need O comes before the wait for it.
      const uint32_t rows_base = sQ + (lu & 1) * kTcQBytes + q4 * 32 * 128;
      const uint32_t put_at = rows_base + lane * 128 + ((lane & 7) << 4);
      auto put = [&](int c, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(put_at ^ (c << 4)), "r"(x), "r"(y), "r"(z), "r"(w)
                     : "memory");
      };
      // this lane stores chunk col of rows row0 + 4 k
      const int col = lane & 7, row0 = q4 * 32 + (lane >> 3);
      const uint32_t get_at = rows_base + (lane >> 3) * 128 + ((col ^ (lane >> 3)) << 4);
      auto get = [&](int k) -> uint4 {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"((get_at ^ ((k & 1) << 6)) + k * 512)
                     : "memory");
        return v;
      };
      bf16* to[8];
      if (whole) {
        bf16* first = a.out + (int64_t)s.token * a.ld_out + (s.kvh * a.n_rep + row0) * kHD + col * 8;
        const int64_t skip = a.ld_out - a.n_rep * kHD;
#pragma unroll
        for (int k = 0; k < 8; ++k) to[k] = first + 4 * k * kHD + row_token(a, row0 + 4 * k) * skip;
      }
      const float inv = l == 0.0f ? 0.0f : __frcp_rn(l);  // no key: zeros
      // the unit's last P V, then O: read and released for the next unit
      ok = wait_all(&pv_done[(g - 1) % kTcStages], (g - 1) / kTcStages);
      if (!ok) break;
      tc_fence_after();
      float2 ov[32];
      if (warp_valid) {
        tmem_ld_32x32b_x32(tmem + 192 + lane_off, *reinterpret_cast<uint32_t(*)[32]>(&ov[0]));
        tmem_ld_32x32b_x32(tmem + 192 + 32 + lane_off, *reinterpret_cast<uint32_t(*)[32]>(&ov[16]));
        tmem_ld_wait();
      }
      tc_fence_before();
      mbar_arrive(&o_empty);
      if (warp_valid) {
        if (whole) {
          const float2 inv2 = make_float2(inv, inv);
#pragma unroll
          for (int c = 0; c < 32; ++c) ov[c] = mul2(ov[c], inv2);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            put(c, pack2(ov[4 * c].x, ov[4 * c].y), pack2(ov[4 * c + 1].x, ov[4 * c + 1].y),
                pack2(ov[4 * c + 2].x, ov[4 * c + 2].y), pack2(ov[4 * c + 3].x, ov[4 * c + 3].y));
          __syncwarp();
          uint4 v[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] = get(k);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (row0 + 4 * k < s.rows) *reinterpret_cast<uint4*>(to[k]) = v[k];
        } else {
          float* first = part + row0 * kHD + col * 4;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float2 x = ov[16 * h + 2 * c], y = ov[16 * h + 2 * c + 1];
              put(c, __float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
            }
            __syncwarp();
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = get(k);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (row0 + 4 * k < s.rows) *reinterpret_cast<uint4*>(first + 4 * k * kHD + h * 32) = v[k];
            __syncwarp();
          }
        }
        fence_proxy_async_smem();  // before the next Q's TMA write to the buffer
      }
      mbar_arrive(&q_empty[lu & 1]);
      ++lu;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// Joins the partials of the unit that starts in CTA blockIdx.x and goes on in
// the next ones: o = sum_c o_c 2^(m_c - M), l likewise.  A CTA takes 256 / (16
// LANES) rows; LANES threads share a row's 16-byte column, each with every
// LANES-th partial, and meet by shuffles in a fixed order.
template <int ROWS, int LANES>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const AttnArgs a, int ctas) {
  pdl_wait();
  pdl_trigger();
  const Meta m = reinterpret_cast<const Meta*>(a.ws + 2 * (int64_t)ctas * part_floats(ROWS))[blockIdx.x];
  constexpr int kRows = 256 / (16 * LANES);
  const int ln = threadIdx.x % LANES, col = (threadIdx.x / LANES) % 16;
  const int r = blockIdx.y * kRows + threadIdx.x / (16 * LANES), d = col * 4;
  if (m.last < 0 || (int)blockIdx.y * kRows >= m.rows) return;
  const int c0 = blockIdx.x, n = min(m.last, ctas - 1) - c0 + 1;
  float M = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = ln; i0 < n; i0 += 4 * LANES) {  // four partials in flight
    float pm[4], pl[4];
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int i = i0 + u * LANES;
      const float* p = a.ws + (2 * (int64_t)(c0 + i) + (i == 0)) * part_floats(ROWS);
      const bool in = i < n;
      pm[u] = in ? p[ROWS * kHD + r] : -INFINITY;
      pl[u] = in ? p[ROWS * kHD + ROWS + r] : 0.0f;
      v[u] = in ? *reinterpret_cast<const float4*>(p + r * kHD + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const float mn = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), M);
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float f0 = ex2_approx(M - base);
    acc = make_float4(acc.x * f0, acc.y * f0, acc.z * f0, acc.w * f0);
    l *= f0;
    M = mn;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = ex2_approx(pm[u] - base);
      acc.x += v[u].x * f;
      acc.y += v[u].y * f;
      acc.z += v[u].z * f;
      acc.w += v[u].w * f;
      l += pl[u] * f;
    }
  }
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, M, o);
    const float mn = fmaxf(M, om), base = mn == -INFINITY ? 0.0f : mn;
    const float f = ex2_approx(M - base), fo = ex2_approx(om - base);
    acc.x = acc.x * f + __shfl_xor_sync(0xffffffffu, acc.x, o) * fo;
    acc.y = acc.y * f + __shfl_xor_sync(0xffffffffu, acc.y, o) * fo;
    acc.z = acc.z * f + __shfl_xor_sync(0xffffffffu, acc.z, o) * fo;
    acc.w = acc.w * f + __shfl_xor_sync(0xffffffffu, acc.w, o) * fo;
    l = l * f + __shfl_xor_sync(0xffffffffu, l, o) * fo;
    M = mn;
  }
  if (ln == 0 && r < m.rows) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store_out4(a, m.token, m.kvh, r, d, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
  }
}

// ----------------------------------------------------------------------------- host side

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encoder() {
  static std::atomic<EncodeTiledFn> fn{nullptr};
  EncodeTiledFn f = fn.load(std::memory_order_acquire);
  if (f) return f;
  void* p = nullptr;
  cudaDriverEntryPointQueryResult q;
  cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
  if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p) return nullptr;
  f = reinterpret_cast<EncodeTiledFn>(p);
  fn.store(f, std::memory_order_release);
  return f;
}

int page_map(CUtensorMap* map, const void* p, int64_t n_pages, int64_t heads, int64_t page_size, int64_t page_ld,
             int64_t head_ld, int64_t row_ld, int box_rows, const char* what, char* err, size_t errlen) {
  EncodeTiledFn enc = encoder();
  if (!enc) {
    set_err(err, errlen, "%s: cuTensorMapEncodeTiled unavailable", what);
    return XB_ERR_CUDA;
  }
  cuuint64_t dims[4] = {(cuuint64_t)kHD, (cuuint64_t)page_size, (cuuint64_t)heads, (cuuint64_t)n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)row_ld * 2, (cuuint64_t)head_ld * 2, (cuuint64_t)page_ld * 2};
  cuuint32_t box[4] = {(cuuint32_t)kHD, (cuuint32_t)box_rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(p), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_err(err, errlen, "%s: cuTensorMapEncodeTiled failed (%d) for pages [%lld][%lld][%lld][64]", what, (int)r,
            (long long)n_pages, (long long)heads, (long long)page_size);
    return XB_ERR_CUDA;
  }
  return XB_OK;
}

// Q as [tokens][n_head][64]; a box is the rows of one unit: n_rep heads of tpt tokens.
int query_map(CUtensorMap* map, const void* q, int64_t tokens, int64_t heads, int64_t ld, int n_rep, int tpt,
              const char* what, char* err, size_t errlen) {
  EncodeTiledFn enc = encoder();
  if (!enc) {
    set_err(err, errlen, "%s: cuTensorMapEncodeTiled unavailable", what);
    return XB_ERR_CUDA;
  }
  cuuint64_t dims[3] = {(cuuint64_t)kHD, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)kHD * 2, (cuuint64_t)ld * 2};
  cuuint32_t box[3] = {(cuuint32_t)kHD, (cuuint32_t)n_rep, (cuuint32_t)tpt};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_err(err, errlen, "%s: cuTensorMapEncodeTiled failed (%d) for q [%lld][%lld][64]", what, (int)r,
            (long long)tokens, (long long)heads);
    return XB_ERR_CUDA;
  }
  return XB_OK;
}

// Addresses of the two status words on the current device, looked up once per device.
int status_words(int** bad, int** status, const char* what, char* err, size_t errlen) {
  static std::atomic<int*> words[kMaxDevices][2];  // zero-initialised (static storage)
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= kMaxDevices)) e = cudaErrorInvalidDevice;
  if (e == cudaSuccess) {
    *bad = words[dev][0].load(std::memory_order_acquire);
    *status = words[dev][1].load(std::memory_order_acquire);
    if (*bad && *status) return XB_OK;
    e = cudaGetSymbolAddress((void**)bad, g_bad_page);
    if (e == cudaSuccess) e = cudaGetSymbolAddress((void**)status, g_paged_status);
    if (e == cudaSuccess) {
      words[dev][0].store(*bad, std::memory_order_release);
      words[dev][1].store(*status, std::memory_order_release);
      return XB_OK;
    }
  }
  set_err(err, errlen, "%s: status words unavailable: %s", what, cudaGetErrorString(e));
  cudaGetLastError();
  return XB_ERR_CUDA;
}

// A flag's value, the flag cleared in the same step: a kernel on another stream
// that sets it between a copy and a clearing would not be heard.
__global__ void take_flag_kernel(int* flag) {
  pdl_wait();
  pdl_trigger();
  g_taken = atomicExch(flag, 0);
}

cudaError_t take_flag(int* flag, int* value, cudaStream_t s) {
  static std::mutex mu;  // g_taken is one word a device
  std::lock_guard<std::mutex> lock(mu);
  cudaError_t e = launch_k<false>(take_flag_kernel, 1, 1, 0, s, flag);
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(value, g_taken, sizeof(int), 0, cudaMemcpyDeviceToHost, s);
  return e == cudaSuccess ? cudaStreamSynchronize(s) : e;
}

// What a paged batch has to satisfy, device contents aside.
int check_pages(const xb_paged_kv* kv, const char* what, char* err, size_t errlen) {
  if (!kv) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  if (kv->n_pages <= 0 || kv->page_size <= 0 || kv->n_kv_head <= 0 || kv->head_dim <= 0 || kv->batch < 0 ||
      kv->max_pages <= 0 || kv->ld_table < kv->max_pages) {
    set_err(err, errlen, "%s: bad shape", what);
    return XB_ERR_INVALID;
  }
  if (kv->page_size % 8) {
    set_err(err, errlen, "%s: page_size %lld is not a multiple of 8", what, (long long)kv->page_size);
    return XB_ERR_UNSUPPORTED;
  }
  const int64_t lds[6] = {kv->k_page, kv->k_head, kv->k_row, kv->v_page, kv->v_head, kv->v_row};
  for (int64_t ld : lds)
    if (ld <= 0 || ld % 8 || ld >= (1LL << 38)) {
      set_err(err, errlen, "%s: page strides must be positive multiples of 8 elements", what);
      return XB_ERR_UNSUPPORTED;
    }
  if (kv->n_pages > 0x7ffffffeLL || kv->max_pages > 0x7fffffffLL || kv->page_size > 0x7fffffffLL ||
      kv->max_pages * kv->page_size > 0x7fffffffLL || kv->n_kv_head > 65535) {
    set_err(err, errlen, "%s: more than 2^31 - 1 pages or positions", what);
    return XB_ERR_UNSUPPORTED;
  }
  // every CTA scans the sequences, and its other warps wait (at most kWaitLimit) while it passes empty ones
  if (kv->batch > (1LL << 20)) {
    set_err(err, errlen, "%s: more than 2^20 sequences", what);
    return XB_ERR_UNSUPPORTED;
  }
  return XB_OK;
}

// Once there is work: the pointers.
int check_page_pointers(const xb_paged_kv* kv, const char* what, char* err, size_t errlen) {
  if (!kv->k_pages || !kv->v_pages || !kv->page_table || !kv->q_start || !kv->kv_len) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  if (!aligned16(kv->k_pages) || !aligned16(kv->v_pages)) {
    set_err(err, errlen, "%s: rows must be whole 16-byte vectors", what);
    return XB_ERR_UNSUPPORTED;
  }
  return XB_OK;
}

// Which attention kernel: the mma.sync one while the batch's rows per (sequence,
// KV head) fill at most one of its 16-row tiles on average; the host knows
// this much without the lengths.  Few-row / tcgen05 kernel, us in a graph, 14
// heads on 2, rows a sequence: 33 sequences of 300-4000 keys 7 13.8 / 19.1, 14
// 16.4 / 19.8, 21 23.4 / 19.7, 35 25.4 / 18.7; 160 of 500-1500 14 23.4 / 28.9, 21
// 36.5 / 30.4, 56 56.8 / 31.1.  12 heads of their own, 160 sequences: 16 89.3 /
// 110.4, 24 160.6 / 109.8.  It is an average: where one sequence brings most of
// the tokens, its 16-row units read its keys once each.  With 12 / 12 heads, 49
// single tokens and a chunk of 512 (11.2 rows on average) take 31.3 / 33.1, 99
// and 1024 with 25 / 25 113.9 / 110.5, but 199 and 3000 (16.0) 205 / 126.
bool few_rows(int64_t tokens, int64_t batch, int64_t n_rep) {
  return n_rep <= kFewRows && tokens * n_rep <= kFewRows * batch;
}

// Launch of an attention kernel, its shared-memory limit raised once per device.
template <typename M>
cudaError_t launch_main(void (*kernel)(M, AttnArgs), int ctas, int threads, int smem, cudaStream_t s, const M& maps,
                        const AttnArgs& a) {
  cudaError_t e = once_per_device(reinterpret_cast<const void*>(kernel), kOnceSmem, [&](int*) {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  return e != cudaSuccess ? e : launch_k(kernel, (unsigned)ctas, threads, smem, s, maps, a);
}

template <int ROWS, typename I>
cudaError_t launch_few(int ctas, cudaStream_t s, const KvMaps& maps, const AttnArgs& a) {
  using C = FewCfg<ROWS>;
  return launch_main(paged_attn_few_kernel<ROWS, I>, ctas, C::kThreads, C::kSmem, s, maps, a);
}

template <int N>
cudaError_t launch_copy(const int32_t* src, const int32_t* dst, int n, uint8_t* base, int64_t outer,
                        int64_t outer_stride, int64_t page_stride, uint32_t vpp, cudaStream_t s) {
  CopyPairs<N> pairs;
  memset(&pairs, 0, sizeof(pairs));
  memcpy(pairs.src, src, n * sizeof(int32_t));
  memcpy(pairs.dst, dst, n * sizeof(int32_t));
  const uint32_t total = (uint32_t)n * vpp;
  return launch_k<false>(copy_pages_kernel<N>, dim3((total + 1023u) / 1024u, (unsigned)outer), 256, 0, s, pairs, base,
                         outer_stride, page_stride, vpp, total);
}

}  // namespace paged

// The timeout flag of this file's kernels, read and cleared by xb_device_status.
cudaError_t paged_status_take(int* status, cudaStream_t s) {
  int *bad = nullptr, *flag = nullptr;
  if (paged::status_words(&bad, &flag, "", nullptr, 0)) return cudaErrorUnknown;
  return paged::take_flag(flag, status, s);
}

}  // namespace xb

using namespace xb::paged;
using xb::aligned16;
using xb::check_launch;
using xb::launch_k;
using xb::set_err;

extern "C" int xb_copy_pages(void* pages, int64_t outer, int64_t outer_bytes, int64_t n_pages, int64_t page_bytes,
                             const int32_t* src, const int32_t* dst, int64_t n, void* stream, char* err,
                             size_t errlen) {
  const char* what = "xb_copy_pages";
  if (outer < 0 || n_pages < 0 || page_bytes < 0 || n < 0) {
    set_err(err, errlen, "%s: negative size", what);
    return XB_ERR_INVALID;
  }
  if (n == 0) return XB_OK;
  if (!src || !dst) {
    set_err(err, errlen, "%s: null page list", what);
    return XB_ERR_INVALID;
  }
  if (n > n_pages || n_pages > 0x7fffffffLL) {
    set_err(err, errlen, "%s: %lld copies in a pool of %lld pages", what, (long long)n, (long long)n_pages);
    return XB_ERR_INVALID;
  }
  // one bit per page: destinations are distinct and none is a source
  uint64_t* seen = static_cast<uint64_t*>(calloc((size_t)(n_pages + 63) / 64, 8));
  if (!seen) {
    set_err(err, errlen, "%s: out of host memory", what);
    return XB_ERR_INVALID;
  }
  const char* wrong = nullptr;
  int64_t at = 0;
  for (int64_t i = 0; i < n && !wrong; ++i) {
    if (src[i] < 0 || src[i] >= n_pages) wrong = "source outside the pool", at = src[i];
    else if (dst[i] < 0 || dst[i] >= n_pages) wrong = "destination outside the pool", at = dst[i];
    else if (seen[dst[i] >> 6] >> (dst[i] & 63) & 1) wrong = "destination given twice", at = dst[i];
    else seen[dst[i] >> 6] |= 1ull << (dst[i] & 63);
  }
  for (int64_t i = 0; i < n && !wrong; ++i)
    if (seen[src[i] >> 6] >> (src[i] & 63) & 1) wrong = "page is both a source and a destination", at = src[i];
  free(seen);
  if (wrong) {
    set_err(err, errlen, "%s: %s (page %lld)", what, wrong, (long long)at);
    return XB_ERR_INVALID;
  }
  if (outer == 0 || page_bytes == 0) return XB_OK;
  if (!pages) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  if (page_bytes % 16 || outer_bytes % 16 || !aligned16(pages) || (outer > 1 && outer_bytes < n_pages * page_bytes)) {
    set_err(err, errlen, "%s: pages must be whole 16-byte vectors in slabs that do not overlap", what);
    return XB_ERR_UNSUPPORTED;
  }
  const int64_t vectors = 0xffff0000LL;  // of a launch, counted in 32 bits
  if (outer > 65535 || page_bytes / 16 > vectors) {
    set_err(err, errlen, "%s: %lld slabs of %lld-byte pages not supported", what, (long long)outer,
            (long long)page_bytes);
    return XB_ERR_UNSUPPORTED;
  }
  const uint32_t vpp = (uint32_t)(page_bytes / 16);
  const int64_t most = vectors / vpp < kCopyPairs ? vectors / vpp : kCopyPairs;
  uint8_t* base = static_cast<uint8_t*>(pages);
  for (int64_t i = 0; i < n; i += most) {
    const int c = (int)(n - i < most ? n - i : most);
    cudaError_t e = c <= 28 ? launch_copy<28>(src + i, dst + i, c, base, outer, outer_bytes, page_bytes, vpp,
                                              (cudaStream_t)stream)
                            : launch_copy<kCopyPairs>(src + i, dst + i, c, base, outer, outer_bytes, page_bytes, vpp,
                                                      (cudaStream_t)stream);
    if (e != cudaSuccess) {
      set_err(err, errlen, "%s: %s", what, cudaGetErrorString(e));
      return XB_ERR_CUDA;
    }
  }
  return check_launch(what, err, errlen);
}

extern "C" int xb_paged_rope_kv_bf16(const void* qkv, const float* cos_t, const float* sin_t, void* q_out,
                                     const xb_paged_kv* kv, int64_t tokens, int64_t n_head, int64_t rope_rows,
                                     int64_t ld_qkv, int64_t ld_q, void* stream, char* err, size_t errlen) {
  const char* what = "xb_paged_rope_kv_bf16";
  int rc = check_pages(kv, what, err, errlen);
  if (rc) return rc;
  if (tokens < 0 || n_head <= 0 || n_head > 65535) {
    set_err(err, errlen, "%s: bad shape", what);
    return XB_ERR_INVALID;
  }
  const int64_t D = kv->head_dim;
  if (D % 16 || D > 512 || 32 % (D / 16)) {
    set_err(err, errlen, "%s: head_dim %lld not supported (16, 32, 64, 128, 256, 512)", what, (long long)D);
    return XB_ERR_UNSUPPORTED;
  }
  if (tokens == 0 || kv->batch == 0) return XB_OK;
  rc = check_page_pointers(kv, what, err, errlen);
  if (rc) return rc;
  if (!qkv || !q_out || (!cos_t) != (!sin_t)) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  if (ld_qkv < (n_head + 2 * kv->n_kv_head) * D || ld_q < n_head * D) {
    set_err(err, errlen, "%s: row pitch shorter than the row", what);
    return XB_ERR_INVALID;
  }
  if (!aligned16(qkv) || !aligned16(q_out) || ld_qkv % 8 || ld_q % 8 ||
      (cos_t && (!aligned16(cos_t) || !aligned16(sin_t)))) {
    set_err(err, errlen, "%s: rows must be whole 16-byte vectors", what);
    return XB_ERR_UNSUPPORTED;
  }
  if (tokens > 0x7ffffff0LL) {
    set_err(err, errlen, "%s: too many tokens", what);
    return XB_ERR_UNSUPPORTED;
  }
  RopeArgs a;
  a.qkv = static_cast<const bf16*>(qkv);
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.q = static_cast<bf16*>(q_out);
  a.k = Pages{static_cast<bf16*>(kv->k_pages), kv->k_page, kv->k_head, kv->k_row};
  a.v = Pages{static_cast<bf16*>(kv->v_pages), kv->v_page, kv->v_head, kv->v_row};
  a.table = kv->page_table;
  a.q_start = kv->q_start;
  a.kv_len = kv->kv_len;
  a.ld_qkv = ld_qkv;
  a.ld_q = ld_q;
  a.ld_table = kv->ld_table;
  a.rope_rows = rope_rows;
  a.T = (int)tokens;
  a.B = (int)kv->batch;
  a.H = (int)n_head;
  a.KVH = (int)kv->n_kv_head;
  a.D = (int)D;
  a.page_size = (int)kv->page_size;
  a.max_pages = (int)kv->max_pages;
  a.n_pages = (int)kv->n_pages;
  int *bad = nullptr, *status = nullptr;
  rc = status_words(&bad, &status, what, err, errlen);
  if (rc) return rc;
  launch_k<false>(paged_rope_kv_kernel, (unsigned)((tokens + 1) / 2), 64, 0, (cudaStream_t)stream, a, bad);
  return check_launch(what, err, errlen);
}

extern "C" int xb_paged_attention_workspace_size(int64_t tokens, int64_t batch, int64_t n_head, int64_t n_kv_head,
                                                 size_t* bytes, char* err, size_t errlen) {
  const char* what = "xb_paged_attention_workspace_size";
  if (!bytes || tokens < 0 || batch < 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head) {
    set_err(err, errlen, "%s: bad arguments", what);
    return XB_ERR_INVALID;
  }
  int sms = 148;
  xb::sm_count(&sms);
  const bool few = few_rows(tokens, batch, n_head / n_kv_head);
  *bytes = (size_t)(few ? sms : 2 * sms) * (2 * part_floats(few ? kFewRows : kTcRows) * sizeof(float) + sizeof(Meta));
  return XB_OK;
}

extern "C" int xb_paged_attention_bf16(const void* q, void* out, const xb_paged_kv* kv, int64_t tokens,
                                       int64_t n_head, int64_t ld_q, int64_t ld_out, float scale, void* workspace,
                                       size_t workspace_bytes, void* stream, char* err, size_t errlen) {
  const char* what = "xb_paged_attention_bf16";
  int rc = check_pages(kv, what, err, errlen);
  if (rc) return rc;
  const int64_t n_kv_head = kv->n_kv_head, batch = kv->batch, n_pages = kv->n_pages, page_size = kv->page_size;
  if (tokens < 0 || n_head <= 0 || n_head % n_kv_head || n_head > 65535) {
    set_err(err, errlen, "%s: bad shape", what);
    return XB_ERR_INVALID;
  }
  if (kv->head_dim != kHD) {
    set_err(err, errlen, "%s: head_dim %lld not supported (64)", what, (long long)kv->head_dim);
    return XB_ERR_UNSUPPORTED;
  }
  if (n_head / n_kv_head > kTcRows) {
    set_err(err, errlen, "%s: %lld query heads per KV head not supported (1..128)", what,
            (long long)(n_head / n_kv_head));
    return XB_ERR_UNSUPPORTED;
  }
  const int n_rep = (int)(n_head / n_kv_head);
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(scale_log2 > 0.0f && scale_log2 < INFINITY)) {
    set_err(err, errlen, "%s: the scale must be positive and, times log2(e), finite", what);
    return XB_ERR_INVALID;
  }
  if (tokens == 0 || batch == 0) return XB_OK;
  rc = check_page_pointers(kv, what, err, errlen);
  if (rc) return rc;
  if (!q || !out) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  if (ld_q < n_head * kHD || ld_out < n_head * kHD) {
    set_err(err, errlen, "%s: row pitch shorter than the row", what);
    return XB_ERR_INVALID;
  }
  if (!aligned16(q) || !aligned16(out) || ld_q % 8 || ld_out % 8) {
    set_err(err, errlen, "%s: rows must be whole 16-byte vectors", what);
    return XB_ERR_UNSUPPORTED;
  }
  if (tokens > 0x7fffffffLL || ld_q >= (1LL << 38) || ld_out >= (1LL << 38)) {
    set_err(err, errlen, "%s: too many tokens, or too long a row pitch", what);
    return XB_ERR_UNSUPPORTED;
  }
  size_t need = 0;
  rc = xb_paged_attention_workspace_size(tokens, batch, n_head, n_kv_head, &need, err, errlen);
  if (rc) return rc;
  if (!workspace || workspace_bytes < need || !aligned16(workspace)) {
    set_err(err, errlen, "%s: needs a 16-byte aligned workspace of %zu bytes (%zu given)", what, need,
            workspace_bytes);
    return XB_ERR_INVALID;
  }
  AttnArgs a;
  a.q = static_cast<const bf16*>(q);
  a.out = static_cast<bf16*>(out);
  a.table = kv->page_table;
  a.q_start = kv->q_start;
  a.kv_len = kv->kv_len;
  a.ws = static_cast<float*>(workspace);
  a.ld_q = ld_q;
  a.ld_out = ld_out;
  a.ld_table = kv->ld_table;
  a.T = (int)tokens;
  a.B = (int)batch;
  a.KVH = (int)n_kv_head;
  a.n_rep = n_rep;
  a.page_size = (int)page_size;
  a.max_pages = (int)kv->max_pages;
  a.n_pages = (int)n_pages;
  a.scale_log2 = scale_log2;
  rc = status_words(&a.bad, &a.status, what, err, errlen);
  if (rc) return rc;
  const bool few = few_rows(tokens, batch, n_rep);
  const bool eight = few && n_rep <= 8 && tokens * n_rep <= 8 * batch;  // the same rule for half a tile
  const int tile = few ? kTK : kTcTK;
  line_kernel(a, few ? (eight ? 8 : kFewRows) : kTcRows);
  a.rep_magic = (65536u + (uint32_t)n_rep - 1u) / (uint32_t)n_rep;
  int box = 8;  // rows of one load: the largest power of two that divides a page, at most a tile
  while (box < tile && page_size % (2 * box) == 0) box *= 2;
  a.box_rows = box;
  TcMaps maps;
  memset(&maps, 0, sizeof(maps));
  rc = page_map(&maps.k, kv->k_pages, n_pages, n_kv_head, page_size, kv->k_page, kv->k_head, kv->k_row, box, what, err,
                errlen);
  if (!rc)
    rc = page_map(&maps.v, kv->v_pages, n_pages, n_kv_head, page_size, kv->v_page, kv->v_head, kv->v_row, box, what,
                  err, errlen);
  if (!rc && !few) rc = query_map(&maps.q, q, tokens, n_head, ld_q, n_rep, a.tpt, what, err, errlen);
  if (rc) return rc;
  int sms = 148;
  xb::sm_count(&sms);
  const int ctas = few ? sms : 2 * sms;
  if (line_bound(a) >= 4e18) {
    set_err(err, errlen, "%s: %lld tokens of %lld sequences over %lld pages each are too many", what,
            (long long)tokens, (long long)batch, (long long)kv->max_pages);
    return XB_ERR_UNSUPPORTED;
  }
  const bool wide = line_is_wide(a, ctas);
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e;
  if (few) {
    KvMaps pages;
    pages.k = maps.k;
    pages.v = maps.v;
    e = eight ? (wide ? launch_few<8, int64_t>(ctas, s, pages, a)
                      : launch_few<8, int>(ctas, s, pages, a))
              : (wide ? launch_few<16, int64_t>(ctas, s, pages, a)
                      : launch_few<16, int>(ctas, s, pages, a));
    if (e == cudaSuccess)
      e = launch_k(paged_attn_join_kernel<kFewRows, 4>, dim3((unsigned)ctas, kFewRows / 4), 256, 0, s, a, ctas);
  } else {
    e = wide ? launch_main(paged_attn_tc_kernel<int64_t>, ctas, kTcThreads, kTcSmem, s, maps, a)
             : launch_main(paged_attn_tc_kernel<int>, ctas, kTcThreads, kTcSmem, s, maps, a);
    if (e == cudaSuccess)
      e = launch_k(paged_attn_join_kernel<kTcRows, 1>, dim3((unsigned)ctas, kTcRows / 16), 256, 0, s, a, ctas);
  }
  if (e != cudaSuccess) {
    set_err(err, errlen, "%s: %s", what, cudaGetErrorString(e));
    return XB_ERR_CUDA;
  }
  return check_launch(what, err, errlen);
}

extern "C" int xb_page_status(void* stream, int* status, char* err, size_t errlen) {
  if (!status) {
    set_err(err, errlen, "xb_page_status: null output");
    return XB_ERR_INVALID;
  }
  int *bad = nullptr, *timeout = nullptr;
  int rc = status_words(&bad, &timeout, "xb_page_status", err, errlen);
  if (rc) return rc;
  cudaError_t e = take_flag(bad, status, (cudaStream_t)stream);
  if (e != cudaSuccess) {
    set_err(err, errlen, "xb_page_status: %s", cudaGetErrorString(e));
    return XB_ERR_CUDA;
  }
  return XB_OK;
}
