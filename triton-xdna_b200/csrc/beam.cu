// The selection of a beam search step: of each group's beams and the whole
// vocabulary the `count` continuations with the largest sums
//
//   total[k, v] = score[k] + x[k, v] - log sum_u exp(x[k, u]),
//
// largest first, equal sums by the lowest beam, then the larger logit, then the
// lowest token.  It stands beside the
// greedy choice (xb_argmax_f32, csrc/llm.cu; examples/qwen2_5/model.py:1134-1179
// and examples/gpt2/model.py:1144-1206 take the argmax of the last position's logits).
//
// A row's order of tokens is that of its logits, so the first kernel reads each
// logit once, keeps the running maximum and sum of the log-sum and the `count`
// best (logit, token) of a part of a row; the second adds the scores (in 64 bits:
// two sums of a beam may lie closer than 32 tell apart) and picks among the parts'
// lists.
// What the log-sum itself is off by decides between beams whose sums lie closer
// than that: exponentials to 2^-22, added in fp32, measured at most 2^-21.7 for 64
// rows each of 1000 to 151936 logits of spread 1 to 8 (the bound is 2^-17).
#include "common.cuh"

namespace xb {
namespace beam {

constexpr int kScan = 256, kPick = 256;  // threads of the two kernels
constexpr int kResident = 4;             // CTAs of the first an SM
constexpr int kMaxCount = 64, kMaxBeams = 64;
constexpr int kLane = 16, kGroup = 32 * kLane;  // tokens that a lane and its warp take at a time
constexpr int kBlocks = 8;      // runs of groups of which a lane keeps the maximum
constexpr int kHeld = 128;      // candidates of a warp held at a time
constexpr int kPicked = 1024;   // candidates of a group's choice held at a time
constexpr float kLowest = -3.402823466e38f;
constexpr float kLog2e = 1.4426950408889634f;
// exp2(x kLog2e) = exp(x (1 + kLog2eOff)): what rounding log2(e) to fp32 does
constexpr double kLog2eOff = (double)kLog2e * 0.69314718055994530942 - 1.0;

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

// Of some tokens: their maximum (-inf: none) and sum 2^shift, the sum of exp2(x
// kLog2e).  The shift is a whole number, so sums of different shifts are brought to
// one without rounding, and x kLog2e - shift is one fused multiply-add, rounded in
// the size of its result.  Where the maximum is 2^22 or more in size (a row of
// masks of the lowest value) the shift is kFar and the sum that of exp(x - maximum).
constexpr int kFar = 0x40000000;
struct Stats {
  float top, sum;
  int shift, unused;
};
__device__ __forceinline__ int shift_of(float top) {
  return fabsf(top) < 4194304.0f ? (int)rintf(top * kLog2e) : kFar;
}
// 2^n, n <= 0
__device__ __forceinline__ float power(int n) { return n < -126 ? 0.0f : __int_as_float((n + 127) << 23); }
// The same sum with a larger maximum
__device__ __forceinline__ void raise(Stats& s, float top) {
  const int to = shift_of(top);
  if (s.shift != kFar && to != kFar) {
    s.sum *= power(min(s.shift - to, 0));  // a sum of nothing may have had any shift
  } else if (s.top != -INFINITY) {
    if (s.shift != kFar) s.sum *= ex2_approx(fmaf(-s.top, kLog2e, (float)s.shift));
    s.sum *= ex2_approx((s.top - top) * kLog2e);
    if (to != kFar) s.sum *= ex2_approx(fmaf(top, kLog2e, -(float)to));
  }
  s.top = top;
  s.shift = to;
}

// A number that at least `count` of the block's threads' `mine` reach, close to the
// largest such one (-inf where none is known): the count-th of the 2 count / warps largest
// of each warp.  `few` is shared and this call's own.  Every thread calls this.
constexpr int kFew = 2 * kMaxCount;
template <int THREADS>
__device__ __forceinline__ float reached_by(float mine, int count, float* few) {
  constexpr int kWarps = THREADS / 32;
  const int part = (2 * count + kWarps - 1) / kWarps, lane = threadIdx.x & 31;
  float* to = few + (threadIdx.x >> 5) * part;
  for (int n = 0; n < part;) {
    const float best = unordered(__reduce_max_sync(0xffffffffu, ordered(mine)));
    const bool at = mine == best;
    const uint32_t who = __ballot_sync(0xffffffffu, at);
    if (at) {
      mine = -INFINITY;
      const int i = n + __popc(who & ((1u << lane) - 1u));
      if (i < part) to[i] = best;
    }
    n += __popc(who);  // every lane, once all are -inf
  }
  __syncthreads();
  // the least of those that fewer than count are above
  const int all = part * kWarps;
  if (threadIdx.x < 32) {
    float bound = INFINITY;
    for (int i = lane; i < all; i += 32) {
      const float mine_ = few[i];
      int above = 0;
#pragma unroll 8
      for (int j = 0; j < all; ++j) above += few[j] > mine_;
      if (above < count) bound = fminf(bound, mine_);
    }
    bound = unordered(__reduce_min_sync(0xffffffffu, ordered(bound)));
    if (lane == 0) few[kFew] = bound;
  }
  __syncthreads();
  return few[kFew];
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

template <typename T>
struct Ring {  // a warp's groups of tokens on their way from memory
  static constexpr int kBytes = kGroup * (int)sizeof(T);
  static constexpr int kStages = 8 / (int)sizeof(T);
  static constexpr int kStage = kBytes + 16;  // a row may start anywhere in a vector
  static constexpr int kSmem = kScan / 32 * kStages * kStage;
};

// One part of a row: groups of tokens, by turns to the CTA's warps, which run
// on their own, each with a ring of asynchronous 16-byte copies (cp.async, 4 KB a
// warp in flight).  Which lane adds up which tokens in which order does not
// depend on the row's address, so rows that are alike have the same sum, to the
// bit.
//
// While the tokens stream by, a lane keeps its running maximum and sum and the
// maximum of each of 8 runs of its tokens, nothing else.  Then a bound that at
// least `count` lanes' maxima reach is one that the `count` best tokens reach, and
// only the few runs whose maximum reaches it are looked through again, in the ring
// or in the L2: some 20 of 2048 for count = 16.  Keeping the candidates during the
// stream took 44 instructions a token, mostly to find that there is none (94 us where
// this takes 43).
//
// What bounds it: 256 rows of 151936 fp32 logits, 156 MB, take 41.4 us with the choice,
// 3.8 TB/s.  The stream alone takes some 32: 14 instructions a token over all, memory
// at 4.9 TB/s, and 512 CTAs for 592 places (busy 75 % of the time); behind it comes
// what no CTA has other work for, the look through the runs and the lists (5), and the
// choice (4).  240 rows of 50257 in bf16 take 16.5 us, 4 of 151936 8.5: start, one group a
// warp, the bound, the lists and the second launch.  Measured (us of these three):
// CTAs of 128 threads 48.9 / 19.0 / 11.8 where 256 took 44.8 / 19.5 / 9.5; rows divided
// for 4, 6, 7, 8, 12 CTAs an SM 43.7 / 46.6 / 42.1 / 42.2 / 45.1 and 19.1 / 20.4 / 19.2 /
// 19.4 / 23.4, but for 100 rows of 50257 4 13.5 and 7 16.7; 16 runs a lane, with maxima
// of 16 bits, 42.8 / 19.8 / 10.1 where 8 take 43.9 / 19.6 / 9.9.
template <typename T>
__global__ void __launch_bounds__(kScan, kResident)
    beam_scan_kernel(const T* __restrict__ logits, int64_t ld, int64_t vocab, int count, int parts,
                     uint64_t* __restrict__ lists, Stats* __restrict__ stats) {
  using R = Ring<T>;
  constexpr int kWarps = kScan / 32;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t cand[kWarps][kHeld];
  __shared__ float run_top[kBlocks][kScan];
  __shared__ uint16_t runs[kBlocks * kScan];
  __shared__ float few[kFew + 1], warp_top[kWarps], warp_sum[kWarps];
  __shared__ int listed, total;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = blockIdx.x / (uint32_t)parts;
  const int part = blockIdx.x - (int)row * parts;
  if (threadIdx.x == 0) listed = total = 0;
  pdl_wait();
  pdl_trigger();
  const T* x = logits + row * ld;
  const int off = (int)(reinterpret_cast<uintptr_t>(x) & 15);
  const uint8_t* from = reinterpret_cast<const uint8_t*>(x) - off;
  const int64_t end = off + vocab * (int64_t)sizeof(T);
  const int64_t groups = (vocab + kGroup - 1) / kGroup;
  const int64_t p0 = part * groups / parts, g1 = (part + 1) * groups / parts, g0 = p0 + warp;
  const int n = g0 < g1 ? (int)((g1 - g0 + kWarps - 1) / kWarps) : 0;
  const int run = (int)((g1 - p0 + kWarps * kBlocks - 1) / (kWarps * kBlocks));  // groups of a run
  uint8_t* mine = ring + warp * R::kStages * R::kStage;
  const uint32_t mine_u32 = (uint32_t)__cvta_generic_to_shared(mine);

  auto fill = [&](int it) {
    if (it < n) {
      const int64_t at = (g0 + (int64_t)it * kWarps) * R::kBytes;
      const uint32_t to = mine_u32 + it % R::kStages * R::kStage + lane * 16;
      const uint8_t* src = from + at + lane * 16;
      if (at >= off && at + R::kStage <= end) {
#pragma unroll
        for (int k = 0; k < R::kBytes / 512; ++k) copy16_async(to + k * 512, src + k * 512);
        if (lane == 0 && off != 0) copy16_async(to + R::kBytes, src + R::kBytes);
      } else {
        for (int k = lane * 16; k < R::kStage; k += 512, src += 512) {
          const int64_t pos = at + k;
          if (pos >= off && pos + 16 <= end) {
            copy16_async(mine_u32 + it % R::kStages * R::kStage + k, src);
          } else {  // vectors that reach out of the row: what of them lies in it
            for (int e = 0; e < 16; e += (int)sizeof(T))
              if (pos + e >= off && pos + e < end)
                *reinterpret_cast<T*>(mine + it % R::kStages * R::kStage + k + e) =
                    *reinterpret_cast<const T*>(src + e);
          }
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < R::kStages; ++i) fill(i);

  Stats sums = {-INFINITY, 0.0f, 0, 0};
  float here = -INFINITY;  // maximum of the present run
  int left = run, block = 0;
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) run_top[i][threadIdx.x] = -INFINITY;
  for (int it = 0; it < n; ++it) {
    float v[kLane];
    asm volatile("cp.async.wait_group %0;" ::"n"(R::kStages - 1) : "memory");
    __syncwarp();
    const uint8_t* p = mine + it % R::kStages * R::kStage + off + lane * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < kLane; ++i) v[i] = Cvt<T>::to_f(*reinterpret_cast<const T*>(p + i * 32 * (int)sizeof(T)));
    const int64_t behind = vocab - (g0 + (int64_t)it * kWarps) * kGroup - lane;  // tokens from this lane's first on
    if (behind <= kGroup - 32) {
#pragma unroll
      for (int i = 0; i < kLane; ++i)
        if (i * 32 >= behind) v[i] = -INFINITY;
    }
    __syncwarp();
    if (it + R::kStages < n) fill(it + R::kStages);  // the last groups stay in the ring
    else asm volatile("cp.async.commit_group;" ::: "memory");
    float m = -INFINITY;  // never NaN: fmaxf passes over NaN, which the sum keeps
#pragma unroll
    for (int i = 0; i < kLane; ++i) m = fmaxf(m, v[i]);
    here = fmaxf(here, m);
    if (m > sums.top) raise(sums, m);
    float s[2] = {sums.sum, 0.0f};
    if (sums.shift != kFar) {
      const float base = -(float)sums.shift;
#pragma unroll
      for (int i = 0; i < kLane; ++i) s[i & 1] += ex2_approx(fmaf(v[i], kLog2e, base));
    } else {
#pragma unroll
      for (int i = 0; i < kLane; ++i) s[i & 1] += ex2_approx((v[i] - sums.top) * kLog2e);
    }
    sums.sum = s[0] + s[1];
    if (--left == 0 || it + 1 == n) {
      run_top[block++][threadIdx.x] = here;
      here = -INFINITY;
      left = run;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  uint64_t* own = cand[warp];
  int held = 0;
  uint64_t bar = 0;
  // the best `count` of this warp's candidates, best first; later ones have to lie above the last
  auto keep_best = [&]() {
    __syncwarp();
    uint64_t e[kHeld / 32];
    int place[kHeld / 32];
#pragma unroll
    for (int i = 0; i < kHeld / 32; ++i) {
      e[i] = i * 32 + lane < held ? own[i * 32 + lane] : 0;
      place[i] = 0;
    }
    for (int j = 0; j < held; ++j) {
      const uint64_t other = own[j];
#pragma unroll
      for (int i = 0; i < kHeld / 32; ++i) place[i] += other > e[i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kHeld / 32; ++i)
      if (e[i] != 0 && place[i] < count) own[place[i]] = e[i];
    __syncwarp();
    if (held >= count) {
      bar = own[count - 1];
      held = count;
    }
  };
  const float low = fmaxf(kLowest, reached_by<kScan>(sums.top, count, few));  // -inf is no candidate
  // the runs to look through
  if (sums.top >= low)
    for (int b = 0; b < block; ++b)
      if (run_top[b][threadIdx.x] >= low) runs[atomicAdd(&listed, 1)] = (uint16_t)(b * kScan + threadIdx.x);
  __syncthreads();
  // a half-warp takes a run, a lane a token of each of its groups
  const int half = warp * 2 + (lane >> 4), inside = (lane & 15) * 32;
  for (int q0 = 0; q0 < listed; q0 += 2 * kWarps) {
    const int q = q0 + half, r = q < listed ? runs[q] : 0;
    const int w = (r % kScan) >> 5, within = (r & 31) + inside, it0 = r / kScan * run;
    const int64_t gw = p0 + w;
    const int nw = gw < g1 ? (int)((g1 - gw + kWarps - 1) / kWarps) : 0;  // that warp's groups
    const uint8_t* slots = ring + w * R::kStages * R::kStage + off + within * (int)sizeof(T);
    for (int u0 = 0; u0 < run; u0 += 4) {  // four loads in flight
      float v[4];
      uint32_t token[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int it = it0 + u0 + u;
        const int64_t t = (gw + (int64_t)it * kWarps) * kGroup + within;
        v[u] = -INFINITY;
        token[u] = (uint32_t)t;
        if (q < listed && u0 + u < run && it < nw && t < vocab)
          v[u] = Cvt<T>::to_f(it + R::kStages >= nw
                                  ? *reinterpret_cast<const T*>(slots + it % R::kStages * R::kStage)
                                  : x[t]);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        uint32_t who = __ballot_sync(0xffffffffu, v[u] >= low);
        if (!who) continue;
        const uint64_t key = key_of(v[u], token[u]);
        if (held > kHeld - 32) keep_best();
        who = __ballot_sync(0xffffffffu, v[u] >= low && key > bar);
        if (who >> lane & 1) own[held + __popc(who & ((1u << lane) - 1u))] = key;
        held += __popc(who);
      }
    }
  }
  __syncthreads();  // the ring is read
  uint64_t* all = reinterpret_cast<uint64_t*>(ring);  // [kWarps * kHeld] at most
  for (int i = lane; i < held; i += 32) all[atomicAdd(&total, 1)] = own[i];
  // the part's maximum and sum
  float m = sums.top;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) warp_top[warp] = m;
  __syncthreads();
  m = warp_top[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) m = fmaxf(m, warp_top[i]);
  if (m > sums.top) raise(sums, m);
  float s = sums.sum;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) warp_sum[warp] = s;
  // a key's place is the number of larger ones
  uint64_t* list = lists + (int64_t)blockIdx.x * count;
  const int found = total;
  for (int i = threadIdx.x; i < found; i += kScan) {
    const uint64_t key = all[i];
    int place = 0;
    for (int j = 0; j < found; ++j) place += all[j] > key;
    if (place < count) list[place] = key;
  }
  for (int i = found + threadIdx.x; i < count; i += kScan) list[i] = 0;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < kWarps; ++i) s += warp_sum[i];
    stats[blockIdx.x] = Stats{m, s, sums.shift, 0};
  }
}

struct Candidate {
  double total;
  uint64_t key;
  int beam;
};
// Sums that 64 bits do not tell apart go by the beam, those of one beam by their
// logits, as the lists do.  Without branches: bf16 logits are equal often (48 x 5 beams
// 18.6 us with them, 17.5 without).
__device__ __forceinline__ bool before(const Candidate& a, const Candidate& b) {
  return (a.total > b.total) |
         ((a.total == b.total) & ((a.beam < b.beam) | ((a.beam == b.beam) & (a.key > b.key))));
}

// 2^n, n <= 0, in 64 bits
__device__ __forceinline__ double power64(int n) { return n < -1022 ? 0.0 : __hiloint2double((n + 1023) << 20, 0); }

// log sum of a row one of whose parts is relative to its maximum: all of them, relative
// to the row's (rare, and kept out of the way of what is fetched every time).
__device__ __noinline__ double far_log_sum(const Stats* stats, int parts, float top) {
  double sum = 0.0;
  for (int i = threadIdx.x & 31; i < parts; i += 32) {
    const Stats s = stats[i];
    if (s.top != -INFINITY || s.sum != 0.0f)
      sum += (double)s.sum * (s.shift == kFar ? exp((double)s.top - (double)top)
                                              : exp2(s.shift - (double)top * (double)kLog2e));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return (double)top + log(sum);
}

// One group: its beams' lists joined.  At least `count` entries reach a bound; what
// lies below it (compared in fp32, which no rounding turns round) falls away.
// Should more be left than fit, as where very many sums are equal, the choice
// goes step by step, the best of all entries behind the last choice each time.
// Latency bounds it, most of all that of fetching instructions, which are cold in
// every launch (3.4 of the 12 clocks between a warp's instructions): sums are formed
// once, and what is rare stays out of line, which took 1 us off every call (1 x 4 beams
// 9.8 -> 8.8).  Of what it adds to a call (4 us) loads and log-sums take 1.3, the bound
// 0.6.
__global__ void __launch_bounds__(kPick) beam_pick_kernel(const float* __restrict__ scores, int64_t ld_scores,
                                                          const uint64_t* __restrict__ lists,
                                                          const Stats* __restrict__ stats, int beams, int parts,
                                                          uint64_t beam_magic, int count, float* __restrict__ values,
                                                          int64_t* __restrict__ parents,
                                                          int64_t* __restrict__ tokens) {
  __shared__ Candidate found[kPicked];
  __shared__ double shifts[kMaxBeams];  // score - log sum; NaN: the beam is out
  __shared__ float few[kFew + 1];
  __shared__ int n;
  pdl_wait();
  pdl_trigger();
  const int64_t g = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int total_lists = beams * parts;
  lists += g * total_lists * count;
  stats += g * total_lists;
  // every entry of every list, a thread has every 256th: the first ones ahead of what they wait for.  Where threads have
  // one or none, every warp gets its part of them, which brings the bound close (48 x 5 beams 17.5 -> 16.5 us; of many
  // entries it would scatter the loads: 1 x 4 8.5 -> 9.9).
  const int entries = total_lists * count;
  constexpr int kAhead = 8;
  const int own = entries <= kPick ? lane * (kPick / 32) + warp : (int)threadIdx.x;
  uint64_t ahead[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int f = j * kPick + own;
    ahead[j] = f < entries ? lists[f] : 0;
  }
  if (threadIdx.x == 0) n = 0;
  for (int k = warp; k < beams; k += kPick / 32) {
    const float score = scores[g * ld_scores + k];
    float top = -INFINITY;
    int shift = -kFar;
    double sum = 0.0;
    bool far = false;
    for (int i0 = 0; i0 < parts; i0 += 32) {
      const Stats s = i0 + lane < parts ? stats[k * parts + i0 + lane] : Stats{-INFINITY, 0.0f, 0, 0};
      const bool any = s.top != -INFINITY || s.sum != 0.0f, near = any && s.shift != kFar;
      top = fmaxf(top, s.top);
      far |= any && !near;
      const int to = max(shift, __reduce_max_sync(0xffffffffu, near ? s.shift : -kFar));
      sum = sum * power64(shift - to) + (near ? (double)s.sum * power64(s.shift - to) : 0.0);
      shift = to;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    // sum 2^shift = sum exp(x (1 + off)), which exp(top off) times the sum of exp(x) is but for off (x - top).  The
    // logarithm of the sum's mantissa in 32 bits (off by 2^-24 as the sum is), the rest of it in 64.
    const int hi = __double2hiint(sum);
    const float mantissa = (float)__hiloint2double((hi & 0xfffff) | 0x3ff00000, __double2loint(sum));
    double lse = (double)logf(mantissa) + 0.69314718055994530942 * ((hi >> 20) - 1023 + shift) - kLog2eOff * top;
    bool out = !(sum > 0.0);  // NaN too
    if (__any_sync(0xffffffffu, far)) {
      lse = far_log_sum(stats + k * parts, parts, top);
      out = !isfinite(lse);
    }
    if (lane == 0) shifts[k] = isfinite(score) && !out ? score - lse : __longlong_as_double(0x7ff8000000000000ll);
  }
  __syncthreads();
  // entry f of the lists; total -inf: none
  auto candidate = [&](int f, uint64_t key) -> Candidate {
    Candidate c;
    c.beam = (int)((uint64_t)f * beam_magic >> 32);  // f / (parts * count)
    const double t = shifts[c.beam] + (double)unordered((uint32_t)(key >> 32));
    c.total = key != 0 && t == t ? t : -INFINITY;
    c.key = key;
    return c;
  };
  double sums[kAhead];
  float best = -INFINITY;
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    if (j * kPick >= entries) break;
    sums[j] = candidate(min(j * kPick + own, entries - 1), ahead[j]).total;
    best = fmaxf(best, (float)sums[j]);
  }
#pragma unroll 1
  for (int f = kAhead * kPick + threadIdx.x; f < entries; f += kPick)
    best = fmaxf(best, (float)candidate(f, lists[f]).total);
  const float bound = reached_by<kPick>(best, count, few);
  auto take = [&](double sum, int f, uint64_t key) {
    if (sum == -INFINITY || (float)sum < bound) return;
    const int at = atomicAdd(&n, 1);
    if (at < kPicked) found[at] = candidate(f, key);
  };
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    if (j * kPick >= entries) break;
    take(sums[j], j * kPick + own, ahead[j]);
  }
#pragma unroll 1
  for (int f = kAhead * kPick + threadIdx.x; f < entries; f += kPick) {
    const uint64_t key = lists[f];
    take(candidate(f, key).total, f, key);
  }
  __syncthreads();
  float* value = values + g * count;
  int64_t *parent = parents + g * count, *token = tokens + g * count;
  auto put = [&](int at, const Candidate& c) {
    value[at] = (float)c.total;
    parent[at] = c.beam;
    token[at] = (int64_t)(0xffffffffu - (uint32_t)c.key);
  };
  const int left = n;
  if (left <= kPicked) {
    for (int i0 = 0; i0 < left; i0 += kPick / 4) {  // four lanes count those before a candidate
      const int i = i0 + threadIdx.x / 4;
      const Candidate mine = found[min(i, left - 1)];
      int place = 0;
#pragma unroll 4
      for (int j = threadIdx.x & 3; j < left; j += 4) place += before(found[j], mine);
      place += __shfl_xor_sync(0xffffffffu, place, 1);
      place += __shfl_xor_sync(0xffffffffu, place, 2);
      if (i < left && place < count && (threadIdx.x & 3) == 0) put(place, mine);
    }
    for (int i = left + threadIdx.x; i < count; i += kPick) {  // fewer candidates than asked for
      value[i] = -INFINITY;
      parent[i] = token[i] = -1;
    }
    return;
  }
  Candidate last{INFINITY, 0, 0};  // the candidate before
  for (int at = 0; at < count; ++at) {
    Candidate mine{-INFINITY, 0, kMaxBeams};
#pragma unroll 1
    for (int f = threadIdx.x; f < entries; f += kPick) {
      const Candidate c = candidate(f, lists[f]);
      if ((at == 0 || before(last, c)) && before(c, mine)) mine = c;
    }
    __syncthreads();
    found[threadIdx.x] = mine;
    __syncthreads();
    for (int o = kPick / 2; o > 0; o >>= 1) {
      if (threadIdx.x < o && before(found[threadIdx.x + o], found[threadIdx.x]))
        found[threadIdx.x] = found[threadIdx.x + o];
      __syncthreads();
    }
    last = found[0];
    if (threadIdx.x == 0) put(at, last);
  }
}

// Parts of a row, the same for all rows, so that rows that are alike have the same
// sum to the bit.
int parts_of(int64_t rows, int64_t vocab) {
  int sms = 148;
  sm_count(&sms);
  const int64_t groups = (vocab + kGroup - 1) / kGroup;
  int64_t n = kResident * sms / rows;
  if (n > groups / (kScan / 32)) n = groups / (kScan / 32);  // a warp has a group at least
  return (int)(n < 1 ? 1 : n);
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
  const int64_t lists = groups ? groups * beams * parts_of(groups * beams, vocab) : 0;
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
  auto scan = [&](auto kernel, auto* x, int smem) {
    cudaError_t e = xb::once_per_device(reinterpret_cast<const void*>(kernel), xb::kOnceSmem, [&](int*) {
      return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    });
    return e != cudaSuccess ? e : launch_k(kernel, (unsigned)(rows * parts), kScan, smem, s, x, ld, vocab,
                                           (int)count, parts, lists, stats);
  };
  cudaError_t e = dtype == XB_DT_F32
                      ? scan(beam_scan_kernel<float>, static_cast<const float*>(logits), Ring<float>::kSmem)
                      : scan(beam_scan_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(logits),
                             Ring<__nv_bfloat16>::kSmem);
  if (e == cudaSuccess)
    e = launch_k(beam_pick_kernel, (unsigned)groups, kPick, 0, s, scores, ld_scores, lists, stats, (int)beams, parts,
                 ((1ull << 32) + parts * count - 1) / (parts * count), (int)count, values, parents, tokens);
  if (e != cudaSuccess) {
    set_err(err, errlen, "%s: %s", what, cudaGetErrorString(e));
    return XB_ERR_CUDA;
  }
  return check_launch(what, err, errlen);
}
