// The selection of a beam search step: of each group's beams and the whole
// vocabulary the `count` continuations with the largest sums
//
//   total[k, v] = score[k] + x[k, v] - log sum_u exp(x[k, u]),
//
// largest first, equal sums by the lowest (beam, token).  It stands beside the
// greedy choice (xb_argmax_f32, csrc/llm.cu; examples/qwen2_5/model.py:1134-1179
// and examples/gpt2/model.py:1144-1206 take the argmax of the last position's logits).
//
// A row's order of tokens is that of its logits, so the first kernel reads each
// logit once, keeps the running maximum and sum of the log-sum and the `count`
// best (logit, token) of a part of a row; the second adds the scores (in 64 bits:
// sums of two beams may lie closer than 32 tell apart) and picks among the parts'
// lists.
#include "common.cuh"

namespace xb {
namespace beam {

constexpr int kThreads = 256;
constexpr int kMaxCount = 64, kMaxBeams = 64, kMaxParts = 64;
constexpr int kBuffer = 1024;  // candidates of a part held at a time

// Orders floats as unsigned numbers (NaN aside).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
// One number that orders (logit, token): the larger logit, then the lower
// token.  -0 counts as 0.  0 is no candidate.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t token) {
  return (uint64_t)ordered(x + 0.0f) << 32 | (0xffffffffu - token);
}

__device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
  x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
}
__device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// Tokens W v .. W v + W - 1 of a row, W = 16 bytes of them; behind the row's end
// -inf.  Which thread adds up which tokens in which order thus does not depend on
// the row's address: rows that are alike have the same sum, to the bit.  A row
// that does not start on a 16-byte boundary: the 16 bytes out of the two aligned
// vectors that hold them (the second is the neighbour's first, in the L1); at its ends, where those reach
// out of the row, element by element.
template <bool ALIGNED, typename T, int W>
__device__ __forceinline__ void load_tokens(const T* row, int64_t vocab, int64_t v, float (&x)[W]) {
  const T* p = row + v * W;
  if ((ALIGNED || (v > 0 && (v + 2) * W <= vocab)) && (v + 1) * W <= vocab) {
    if constexpr (ALIGNED) {
      unpack(__ldcs(reinterpret_cast<const uint4*>(p)), x);
    } else {
      const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 15u;  // the same all along a row
      const uint4* q = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) - off);
      const uint4 lo = __ldg(q), hi = __ldg(q + (off != 0));
      uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      if (off & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
      }
      if (off & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
      }
      if (off & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 16);
      }
      unpack(make_uint4(w[0], w[1], w[2], w[3]), x);
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) x[j] = v * W + j < vocab ? Cvt<T>::to_f(p[j]) : -INFINITY;
  }
}

struct Stats {  // of a part: its maximum (-inf: none), the sum of exp(x - maximum)
  float top, sum;
};

// Keeps the `count` best of the n <= kBuffer candidates in `buf`, best first, and
// returns how many that are.  All threads; keys differ from each other, so a
// key's place is the number of larger ones.
__device__ __forceinline__ int keep_best(uint64_t* buf, uint64_t* sorted, int n, int count) {
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t mine = buf[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += buf[j] > mine;
    if (place < count) sorted[place] = mine;
  }
  __syncthreads();
  const int kept = min(n, count);
  for (int i = threadIdx.x; i < kept; i += kThreads) buf[i] = sorted[i];
  __syncthreads();
  return kept;
}

// One part of a row: `vps` vectors of 16 bytes.
template <bool ALIGNED, typename T>
__global__ void __launch_bounds__(kThreads) beam_scan_kernel(const T* __restrict__ logits, int64_t ld, int64_t vocab,
                                                             int count, int parts, int64_t vps,
                                                             uint64_t* __restrict__ lists, Stats* __restrict__ stats) {
  constexpr int W = 16 / sizeof(T), NV = 32 / W;  // 32 logits a thread at a time
  __shared__ uint64_t buf[kBuffer], sorted[kMaxCount];
  __shared__ float warp_low[kThreads / 32], warp_top[kThreads / 32], warp_sum[kThreads / 32];
  __shared__ int held;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x / (uint32_t)parts;
  const int part = blockIdx.x - (int)row * parts;
  if (threadIdx.x == 0) held = 0;
  pdl_wait();
  pdl_trigger();
  const T* x = logits + row * ld;
  const int64_t v0 = part * vps, v1 = min((vocab + W - 1) / W, v0 + vps);

  float top = -INFINITY, sum = 0.0f;
  uint64_t bar = 0;  // candidates lie above it
  float low = -3.402823466e38f;  // and so their logits at or above this
  __syncthreads();
  for (int64_t v = v0;; v += kThreads * NV) {
    const bool first = v == v0;
    float e[NV][W];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int64_t at = v + i * kThreads + threadIdx.x;
      if (at < v1) load_tokens<ALIGNED>(x, vocab, at, e[i]);
      else
#pragma unroll
        for (int j = 0; j < W; ++j) e[i][j] = -INFINITY;
    }
    // running maximum and sum
    float m = -INFINITY;  // never NaN: fmaxf passes over NaN, which the sum keeps
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) m = fmaxf(m, e[i][j]);
    const float to = fmaxf(top, m), base = to == -INFINITY ? 0.0f : to;
    constexpr float kLog2e = 1.4426950408889634f;
    float s[2] = {sum * ex2_approx((top - base) * kLog2e), 0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) s[j & 1] += ex2_approx((e[i][j] - base) * kLog2e);
    sum = s[0] + s[1];
    top = to;
    if (first) {
      // a bound below the count best: in every warp at least count / 8 threads have a maximum at or above the least of
      // the warps' own bounds
      float mine = m, bound = -3.402823466e38f;
      for (int need = (count + kThreads / 32 - 1) / (kThreads / 32); need > 0;) {
        bound = unordered(__reduce_max_sync(0xffffffffu, ordered(mine)));
        if (bound == -INFINITY) break;
        need -= __popc(__ballot_sync(0xffffffffu, mine == bound));
        if (mine == bound) mine = -INFINITY;
      }
      if (lane == 0) warp_low[warp] = bound;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kThreads / 32; ++i) bound = fminf(bound, warp_low[i]);
      low = fmaxf(low, bound);
      bar = (uint64_t)ordered(low + 0.0f) << 32;
    }
    // candidates into the buffer; where it is full its best stay, and the bar rises
    uint32_t want = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < W; ++j) want |= e[i][j] >= low ? 1u << (i * W + j) : 0u;
    int n;
    for (;;) {
      if (want) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < W; ++j)
            if (want >> (i * W + j) & 1) {
              const uint64_t key =
                  key_of(e[i][j], (uint32_t)((v + i * kThreads + threadIdx.x) * W + j));
              if (key > bar) {
                const int at = atomicAdd(&held, 1);
                if (at >= kBuffer) continue;  // stays wanted
                buf[at] = key;
              }
              want &= ~(1u << (i * W + j));
            }
      }
      __syncthreads();
      n = held;
      __syncthreads();
      if (n <= kBuffer && n < 3 * count + 64 && !first) break;
      const bool over = n > kBuffer;
      n = keep_best(buf, sorted, min(n, kBuffer), count);
      if (n == count) {
        bar = buf[count - 1];
        low = unordered((uint32_t)(bar >> 32));
      }
      if (threadIdx.x == 0) held = n;
      __syncthreads();
      if (!over) break;
    }
    if (v + kThreads * NV >= v1) break;
  }
  const int n = keep_best(buf, sorted, held, count);
  uint64_t* list = lists + (int64_t)blockIdx.x * count;
  for (int i = threadIdx.x; i < count; i += kThreads) list[i] = i < n ? buf[i] : 0;
  // the part's maximum and sum
  float m = top;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) warp_top[warp] = m;
  __syncthreads();
  m = warp_top[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) m = fmaxf(m, warp_top[i]);
  float s = sum * ex2_approx((top - (m == -INFINITY ? 0.0f : m)) * 1.4426950408889634f);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) warp_sum[warp] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kThreads / 32; ++i) s += warp_sum[i];
    stats[blockIdx.x] = Stats{m, s};
  }
}

struct Candidate {
  double total;
  uint64_t place;  // beam << 32 | token
};
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return a.total > b.total || (a.total == b.total && a.place < b.place);
}

// One group: its beams' lists joined.  At most count lists have a first entry among
// the count best first entries, and only they can hold one of the count best
// candidates; of those, entries below the count-th first entry fall away.
__global__ void __launch_bounds__(kThreads) beam_pick_kernel(const float* __restrict__ scores, int64_t ld_scores,
                                                             const uint64_t* __restrict__ lists,
                                                             const Stats* __restrict__ stats, int beams, int parts,
                                                             int count, float* __restrict__ values,
                                                             int64_t* __restrict__ parents,
                                                             int64_t* __restrict__ tokens) {
  extern __shared__ Candidate found[];  // [beams * parts] first entries, then [count * count]
  __shared__ double shift[kMaxBeams];   // score - log sum; NaN: the beam is out
  __shared__ Candidate least;
  __shared__ int n;
  pdl_wait();
  pdl_trigger();
  const int64_t g = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_lists = beams * parts;
  lists += g * total_lists * count;
  stats += g * total_lists;
  Candidate* firsts = found;
  Candidate* all = found + total_lists;
  for (int k = warp; k < beams; k += kThreads / 32) {
    float top = -INFINITY;
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, stats[k * parts + i].top);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    double sum = 0.0;
    for (int i = lane; i < parts; i += 32) {
      const Stats s = stats[k * parts + i];
      if (s.top != -INFINITY || s.sum != 0.0f) sum += (double)s.sum * exp((double)s.top - (double)top);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      const double score = scores[g * ld_scores + k], lse = (double)top + log(sum);
      shift[k] = isfinite(score) && isfinite(lse) ? score - lse : __longlong_as_double(0x7ff8000000000000ll);
    }
  }
  if (threadIdx.x == 0) {
    n = 0;
    least = Candidate{-INFINITY, ~0ull};
  }
  __syncthreads();
  // candidate i of list l; total -inf: none
  auto entry = [&](int l, int i) -> Candidate {
    const uint64_t key = lists[(int64_t)l * count + i];
    const int k = l / parts;
    const double t = shift[k] + (double)unordered((uint32_t)(key >> 32));
    Candidate c;
    c.total = key != 0 && isfinite(t) ? t : -INFINITY;
    c.place = (uint64_t)k << 32 | (0xffffffffu - (uint32_t)key);
    return c;
  };
  for (int l = threadIdx.x; l < total_lists; l += kThreads) firsts[l] = entry(l, 0);
  __syncthreads();
  for (int l = threadIdx.x; l < total_lists; l += kThreads) {
    const Candidate mine = firsts[l];
    int place = 0;
    for (int j = 0; j < total_lists; ++j) place += before(firsts[j], mine);
    if (place == count - 1 && mine.total != -INFINITY) least = mine;  // places of candidates differ
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total_lists * count; i += kThreads) {
    const int l = i / count;
    if (firsts[l].total == -INFINITY || before(least, firsts[l])) continue;
    const Candidate c = entry(l, i - l * count);
    if (c.total != -INFINITY && !before(least, c)) all[atomicAdd(&n, 1)] = c;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const Candidate mine = all[i];
    int place = 0;
    for (int j = 0; j < n; ++j) place += before(all[j], mine);
    if (place < count) {
      values[g * count + place] = (float)mine.total;
      parents[g * count + place] = (int64_t)(mine.place >> 32);
      tokens[g * count + place] = (int64_t)(mine.place & 0xffffffffu);
    }
  }
  for (int i = n + threadIdx.x; i < count; i += kThreads) {  // fewer candidates than asked for
    values[g * count + i] = -INFINITY;
    parents[g * count + i] = tokens[g * count + i] = -1;
  }
}

// Parts of a row: enough CTAs to fill the GPU a few times over, each with at least
// 2048 logits.
int parts_of(int64_t rows, int64_t vocab) {
  int sms = 148;
  sm_count(&sms);
  int64_t parts = (4 * sms + rows - 1) / rows;
  if (parts > vocab / 2048) parts = vocab / 2048;
  return (int)(parts < 1 ? 1 : parts > kMaxParts ? kMaxParts : parts);
}

// all first entries, and count entries of each of the count best lists
size_t pick_smem(int64_t beams, int parts, int64_t count) {
  return (size_t)(beams * parts + count * count) * sizeof(Candidate);
}

int check_sizes(int64_t groups, int64_t beams, int64_t vocab, int64_t count, const char* what, char* err,
                size_t errlen) {
  if (groups < 0 || beams <= 0 || vocab <= 0 || count <= 0) {
    set_err(err, errlen, "%s: bad shape", what);
    return XB_ERR_INVALID;
  }
  if (beams > kMaxBeams || count > kMaxCount || groups > (1 << 20) || vocab > 0x7fffffffLL) {
    set_err(err, errlen, "%s: at most %d beams, %d continuations, 2^20 groups and 2^31 - 1 tokens", what, kMaxBeams,
            kMaxCount);
    return XB_ERR_UNSUPPORTED;
  }
  return XB_OK;
}

}  // namespace beam
}  // namespace xb

using namespace xb::beam;
using xb::check_launch;
using xb::launch_k;
using xb::set_err;

extern "C" int xb_beam_select_workspace_size(int64_t groups, int64_t beams, int64_t vocab, int64_t count,
                                             size_t* bytes, char* err, size_t errlen) {
  const char* what = "xb_beam_select_workspace_size";
  int rc = check_sizes(groups, beams, vocab, count, what, err, errlen);
  if (rc) return rc;
  if (!bytes) {
    set_err(err, errlen, "%s: null output", what);
    return XB_ERR_INVALID;
  }
  const int64_t lists = groups * beams * (groups ? parts_of(groups * beams, vocab) : 0);
  *bytes = (size_t)(lists * (count * 8 + (int64_t)sizeof(Stats)));
  return XB_OK;
}

extern "C" int xb_beam_select(const void* logits, const float* scores, int64_t groups, int64_t beams, int64_t vocab,
                              int64_t ld, int64_t ld_scores, int64_t count, int dtype, float* values, int64_t* parents,
                              int64_t* tokens, void* workspace, size_t workspace_bytes, void* stream, char* err,
                              size_t errlen) {
  const char* what = "xb_beam_select";
  int rc = check_sizes(groups, beams, vocab, count, what, err, errlen);
  if (rc) return rc;
  if (dtype != XB_DT_BF16 && dtype != XB_DT_F32) {
    set_err(err, errlen, "%s: unsupported dtype code %d (want bf16=%d or f32=%d)", what, dtype, XB_DT_BF16, XB_DT_F32);
    return XB_ERR_UNSUPPORTED;
  }
  if (groups == 0) return XB_OK;
  if (!logits || !scores || !values || !parents || !tokens) {
    set_err(err, errlen, "%s: null pointer", what);
    return XB_ERR_INVALID;
  }
  const int64_t rows = groups * beams;
  if ((rows > 1 && ld < vocab) || (groups > 1 && ld_scores < beams)) {
    set_err(err, errlen, "%s: row pitch shorter than the row", what);
    return XB_ERR_INVALID;
  }
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == XB_DT_F32 ? 4 : 2)) {
    set_err(err, errlen, "%s: logits must be aligned to their type", what);
    return XB_ERR_UNSUPPORTED;
  }
  size_t need = 0;
  rc = xb_beam_select_workspace_size(groups, beams, vocab, count, &need, err, errlen);
  if (rc) return rc;
  if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)) {
    set_err(err, errlen, "%s: needs a 16-byte aligned workspace of %zu bytes (%zu given)", what, need,
            workspace_bytes);
    return XB_ERR_INVALID;
  }
  const int parts = parts_of(rows, vocab);
  uint64_t* lists = static_cast<uint64_t*>(workspace);
  Stats* stats = reinterpret_cast<Stats*>(lists + rows * parts * count);
  cudaStream_t s = (cudaStream_t)stream;
  const unsigned ctas = (unsigned)(rows * parts);
  const int64_t W = dtype == XB_DT_F32 ? 4 : 8, vps = ((vocab + W - 1) / W + parts - 1) / parts;
  const bool aligned = xb::aligned16(logits) && (rows == 1 || ld % W == 0);
  auto scan = [&](auto kernel, auto* x) {
    return launch_k(kernel, ctas, kThreads, 0, s, x, ld, vocab, (int)count, parts, vps, lists, stats);
  };
  cudaError_t e;
  if (dtype == XB_DT_F32) {
    const float* x = static_cast<const float*>(logits);
    e = aligned ? scan(beam_scan_kernel<true, float>, x) : scan(beam_scan_kernel<false, float>, x);
  } else {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(logits);
    e = aligned ? scan(beam_scan_kernel<true, __nv_bfloat16>, x) : scan(beam_scan_kernel<false, __nv_bfloat16>, x);
  }
  const size_t smem = pick_smem(beams, parts, count);
  if (e == cudaSuccess)
    e = xb::once_per_device(reinterpret_cast<const void*>(beam_pick_kernel), xb::kOnceSmem, [&](int*) {
      return cudaFuncSetAttribute(beam_pick_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  (int)pick_smem(kMaxBeams, kMaxParts, kMaxCount));
    });
  if (e == cudaSuccess)
    e = launch_k(beam_pick_kernel, (unsigned)groups, kThreads, smem, s, scores, ld_scores, lists, stats, (int)beams,
                 parts, (int)count, values, parents, tokens);
  if (e != cudaSuccess) {
    set_err(err, errlen, "%s: %s", what, cudaGetErrorString(e));
    return XB_ERR_CUDA;
  }
  return check_launch(what, err, errlen);
}
