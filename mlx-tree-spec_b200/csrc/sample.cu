// Sampling one token per row of logits with temperature, top-k, top-p and
// min-p from given random numbers.
//
// Order the tokens by (logit descending, index ascending) and give token i the
// weight w_i = 2^-t_i, t = (max - x) * log2(e) / temperature. Every filter keeps a
// prefix of that order: top-k the first k, top-p the shortest prefix whose mass
// reaches p times the mass of those k, min-p the tokens of weight >= min_p. The
// sample is the first token whose cumulative mass exceeds u times the mass kept
// by all of them. So a row is never sorted: each step asks where the running
// count or mass along the order crosses a bound.
//
// A cluster of CTAs holds a row's logits in shared memory (one read of HBM).
// Small top-k (k <= 64): each warp sorts its lanes' maxima; a bound that k lanes
//   of a CTA reach leaves some tens of tokens per CTA, which CTA 0 gathers, cuts to
//   about k and puts in order. One cluster barrier in all.
// Otherwise:
//   1. The maximum, exchanged through distributed shared memory.
//   2. A histogram over t in steps of 1/32, so fine that a bin holds few tokens:
//      of counts with top-k, else of masses. The CTAs add theirs into CTA 0's.
//   3. CTA 0 finds the bins in which the bounds fall; the tokens of those bins
//      (all bins up to the last one wanted, or the sample's own bin alone) are
//      gathered in its shared memory, and a bound is resolved among the tokens of
//      its bin: histograms over t, then over (logit, index), narrow them down to
//      a hundred or so, which are put in order.
// Where the kept tokens are too many to list, the bounds are resolved one after
// the other, each with a list of its own bin, or, for a bin of thousands of
// nearly equal logits, by a radix descent over their bits.
//
// Masses. Inside a bin (t within 1/64 of bin / 32) a token's weight is m * 2^-22 *
// 2^(-bin / 32) with m an integer of 23 bits, from a float32 series of the reduced t.
// Sums over a bin's tokens are sums of integers, so they do not depend on the order of
// the atomics and results repeat bit for bit. m goes into two 32-bit shared-memory
// atomics of 12 and 11 bits (2^20 tokens do not overflow them), which is why it has no
// more bits; a 64-bit one would be a compare-and-swap loop.
//   Half a unit of m is 2^-23 of the weight, equal logits having the same rounding: a
// border between two tokens' shares is off by 2^-24 at most (half of the weights high,
// half low), by far less where many different logits come before it. The difference to the
// largest logit is a float32: exact for 16-bit logits but for those of very different
// exponents, else a rounding of 2^-24 d / temperature of the weight.
//   The running mass at a token is a whole number of 2^-43 too: the sum over the
// bins before its own, and its bin's tokens up to it, whose sum of m is rounded to
// such units once (`reach`). Whoever asks gets the same number, it never falls along
// the order, and a bin without tokens adds nothing; so a bound that is itself a
// running mass (what a filter keeps, at u = 1) is met at the token that it came from.
//
// Measured, in calls one after the other (and as a replayed graph), inputs in turn: one row
// of 131072 bf16 logits with top-k 50 and top-p 0.95 11.5 us (8.9); 128 such rows with
// settings of their own 55.6 us (54.9; the bytes alone: 5.2 us); 48 rows of 100003 float32
// with temperature alone 37.3 us (36.7; 3.0). One input that stays in L2: 49 and 34 us. A row's steps take 15-60 thousand cycles
// (load 3, maximum 3, histogram 8, plan 5, gather 6, each bound 6), mostly waits for shared
// memory and for the other CTAs, and 55 rows are at work at once.
//
// A call of few rows is bound by the latency of these steps one after the other, not
// by their work: tokens wanted are found as bit masks over 32 logits at a time, and a
// short list is ordered by counting, for each of its tokens, those before it.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace tsb {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kStep = 32;              // bins per octave of the weight
constexpr int kBins = 43 * kStep;      // a token of no bin has a mass of zero
constexpr int kBinsPerThread = (kBins + kThreads - 1) / kThreads;
constexpr int kList = 2048;            // tokens CTA 0 can hold
constexpr int kPart = kList / kMaxCluster;  // of them from each CTA, with small top-k: one per thread
constexpr int kDirectK = 64;           // top-k up to here is looked for among the lanes' maxima
constexpr int kSub = kThreads;         // bins of a narrowing histogram, one per thread
constexpr int kFewest = 128;           // tokens put in order by counting, two threads each
constexpr int kUnitM = 1 << 22;        // m of a token in the middle of its bin
constexpr int kMaxVocab = 1 << 20;
constexpr int kCtasPerSm = 3;              // by their registers
constexpr size_t kSmemPerSm = 228 * 1024;
constexpr int kMaxStage = 160 * 1024;  // bytes of logits a CTA holds in shared memory
constexpr size_t kSliceBytes = 48 * 1024;  // of logits in a CTA, while there are CTAs to split them over
constexpr int kSliceMin = 4096;            // logits of a slice that is not split further
constexpr double kMinTemperature = 8.673617379884035e-19;  // 2^-60
constexpr double kMaxTemperature = 1.2676506002282294e30;  // 2^100

struct SampleArgs {
  const void *logits;
  const float *u;
  const float *temperature, *top_p, *min_p;  // per row, or NULL and the scalar below
  const int32_t *top_k;
  double temperature_s, top_p_s, min_p_s;
  int top_k_s;
  int vocab, slice, staged;
  long long row_stride;
  int32_t *token;
  float *logprob;
};

TSB_HD float to_float(float x) { return x; }
TSB_HD float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
TSB_HD float to_float(__half x) { return __half2float(x); }

// Largest of 16 bytes of logits; NaN is skipped.
TSB_HD float max_of(const uint4 &v, float) {
  return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
TSB_HD float max_of(const uint4 &v, __nv_bfloat16) {
  const __nv_bfloat162 a = __hmax2(__hmax2(u32_as_bf2(v.x), u32_as_bf2(v.y)), __hmax2(u32_as_bf2(v.z), u32_as_bf2(v.w)));
  return fmaxf(__low2float(a), __high2float(a));
}
TSB_HD float max_of(const uint4 &v, __half) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
  const __half2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(__low2float(a), __high2float(a));
}

// A token as a number that orders like the sampling does: order-preserving bits
// of its logit (-0 as +0), then its index, lower first.
TSB_HD u64 make_token(float x, int index) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (u64)((b & 0x80000000u) ? ~b : (b | 0x80000000u)) << 32 | (uint32_t)~index;
}
TSB_HD float key_logit(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }
TSB_HD float token_logit(u64 token) { return key_logit((uint32_t)(token >> 32)); }
TSB_HD int token_index(u64 token) { return (int)~(uint32_t)token; }

struct RowScale {
  float top;           // the largest logit
  float scale, low;    // kStep * log2(e) / temperature, and what the float leaves of it
};

// Bin of a logit, never decreasing as the logit falls: round(kStep * t). At or past
// kBins for a token without mass, -inf and NaN among them (the float's bits are
// compared as a number).
TSB_HD uint32_t logit_bin(float x, const RowScale &r) {
  return __float_as_uint(fmaf(r.top - x, r.scale, 8388608.f)) - 0x4B000000u;
}
// m of a token of bin < kBins: 2^22 * 2^(-g / 32), g = kStep * t - bin in [-1/2, 1/2]
// up to the roundings of t, from the series of e^z at |z| <= 0.011 (the next term is
// below 2^-30). The last addition leaves the rounded integer in the mantissa.
TSB_HD uint32_t logit_m(float x, uint32_t bin, const RowScale &r) {
  const float d = r.top - x;
  const float b = __uint_as_float(0x4B000000u | bin) - 8388608.f;
  const float z = fmaf(d, r.low, fmaf(d, r.scale, -b)) * (-0.693147180559945f / kStep);
  const float p = fmaf(fmaf(fmaf(z, 1.f / 6.f, 0.5f), z, 1.f), z * (float)kUnitM, 8388608.f + (float)kUnitM);
  return __float_as_uint(p) & 0x7FFFFFu;
}
// Powers 2^(-i / 32).
__constant__ double kOctave[kStep] = {
    1.0, 0.97857206208770013, 0.9576032806985737, 0.93708381705514999, 0.91700404320467123, 0.89735453750155359,
    0.8781260801866497, 0.85930964906123897, 0.8408964152537145, 0.82287773907698243, 0.80524516597462714,
    0.78799042255394325, 0.77110541270397037, 0.75458221379671136, 0.73841307296974967, 0.72259040348852331,
    0.70710678118654752, 0.69195494098191597, 0.67712777346844632, 0.66261832157987064, 0.64841977732550475,
    0.63452547859586661, 0.62092890603674202, 0.60762367999023449, 0.59460355750136054, 0.58186242938878875,
    0.5693943173783458, 0.55719337129794622, 0.54525386633262887, 0.53357020033841180, 0.52213689121370688,
    0.51094857432705836};
// A mass is a whole number of 2^-43, the first token's 2^43; those of 2^20 tokens add
// up to 2^63 and a little.
constexpr u64 kOne = 1ull << 43;
constexpr double kPerUnit = 1.1368683772161603e-13;  // 2^-43
// What one unit of m is in a bin: of the first token's weight, and in units of a mass.
// `octave` is a copy of kOctave in shared memory: lanes ask for different ones.
TSB_HD double bin_unit(uint32_t bin, const double *octave) {
  return octave[bin % kStep] * __hiloint2double((int)(1023u - 22u - bin / kStep) << 20, 0);
}
TSB_HD double bin_scale(uint32_t bin, const double *octave) {
  return octave[bin % kStep] * __hiloint2double((int)(1023u + 43u - 22u - bin / kStep) << 20, 0);
}
// The running mass (or, with a scale of 1, count) at a token: `before` its bin, and m of
// its bin's tokens up to it.
TSB_HD u64 reach(u64 before, u64 m, double scale) {
  return before + (scale == 1.0 ? m : __double2ull_rn((double)m * scale));
}
TSB_HD double logit_mass(float x, const RowScale &r, const double *octave) {
  const uint32_t bin = logit_bin(x, r);
  return bin < (uint32_t)kBins ? (double)logit_m(x, bin, r) * bin_unit(bin, octave) : 0.0;
}

// With small top-k, weights are rounded to whole numbers of 2^-40 and added up: at most
// 64 tokens count, so what that changes of their sum is below 2^-35.
constexpr double kListUnit = 1099511627776.0;
TSB_HD u64 list_units(double mass) { return (u64)__double2ll_rn(mass * kListUnit); }

// How the tokens that a bound falls among are resolved.
enum Mode { kFew, kSlow, kOneBin, kRadix, kNoMass };

struct Shared {
  union {
    struct {
      unsigned int h0[kBins], h1[kBins];  // histogram: counts, or the low 12 and the high bits of m
    };
    u64 sums[kBins];                      // CTA 0: running counts or masses up to and including a bin
  };
  u64 list[kList];                        // tokens found; in CTA 0 its own from the front, the others' from the back
  ulonglong2 few[kFewest];                // tokens and their units of count or mass
  u64 order[kFewest], up_to[kFewest];     // in order, and the running units
  unsigned int sub0[kSub], sub1[kSub];
  double octave[kStep];
  float peer_top[kMaxCluster];
  float peer_cut[kMaxCluster];            // CTA 0
  unsigned int floor0[3], floor1[3];      // min-p's part of three bins: the low 12 and the high bits of m
  u64 peer_floor[kMaxCluster][3];         // CTA 0
  unsigned int peer_ties[kMaxCluster];
  u64 red[kWarps], red2[kWarps];
  u64 scan[kWarps];
  u64 found_mass, found_token, temp, last;
  int found;
  unsigned int mine, others, base, few_n, first;
  // written by CTA 0 into every CTA
  int overflow, mode, lo, hi;
  uint32_t prefix;
  int pick_rank, pick_tie;
};
constexpr size_t kSharedBytes = (sizeof(Shared) + 15) & ~size_t(15);
static_assert(kSharedBytes + kMaxStage <= 227 * 1024, "shared memory");
static_assert(kSub == 256, "a digit of the radix descent");
static_assert(kPart <= kThreads, "a thread moves one token of each part");

// Calls g(vector index) for the whole 16-byte vectors of elements [off, off + n) of
// data, which is a 16-byte boundary, and e(element index) for those at the ends. A
// thread gets the same ones every time.
template <typename T, int UNROLL, typename G, typename E>
TSB_HD void for_vectors(int off, int n, G g, E e) {
  constexpr int VEC = 16 / sizeof(T);
  const int v0 = (off + VEC - 1) / VEC, v1 = max((off + n) / VEC, v0);
#pragma unroll UNROLL
  for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads) g(v);
  const int head = min(v0 * VEC, off + n), rest = max(v1 * VEC, head);
  const int i = off + (int)threadIdx.x, j = rest + (int)threadIdx.x - 32;
  if (i < head) e(i);
  if (j >= rest && j < off + n) e(j);
}
// Calls f(element index, logit) for this CTA's logits.
template <typename T, typename F>
TSB_HD void for_logits(const T *data, int off, int n, F f) {
  constexpr int VEC = 16 / sizeof(T);
  for_vectors<T, 1>(
      off, n,
      [&](int v) {
        const uint4 w = *reinterpret_cast<const uint4 *>(data + v * VEC);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(v * VEC + j, to_float(e[j]));
      },
      [&](int i) { f(i, to_float(data[i])); });
}
// Calls f(element index, logit) for this CTA's logits that satisfy test.
template <typename T, typename P, typename F>
TSB_HD void for_hits(const T *data, int off, int n, P test, F f) {
  constexpr int VEC = 16 / sizeof(T), GROUP = 32 / VEC;
  const int v0 = (off + VEC - 1) / VEC, v1 = max((off + n) / VEC, v0);
#pragma unroll 1
  for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads * GROUP) {
    uint32_t mask = 0;
#pragma unroll
    for (int g = 0; g < GROUP; ++g) {
      if (v + g * kThreads < v1) {
        const uint4 w = *reinterpret_cast<const uint4 *>(data + (v + g * kThreads) * VEC);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) mask |= test(to_float(e[j])) ? 1u << (g * VEC + j) : 0u;
      }
    }
    for (; mask; mask &= mask - 1) {
      const int b = __ffs(mask) - 1;
      const int i = (v + (b / VEC) * kThreads) * VEC + b % VEC;
      f(i, to_float(data[i]));
    }
  }
  for_vectors<T, 1>(
      off, n, [](int) {}, [&](int i) {
        const float x = to_float(data[i]);
        if (test(x)) f(i, x);
      });
}

// Sums and inclusive scans over the block.
TSB_HD u64 block_sum(u64 v, Shared &s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.scan[threadIdx.x / 32] = v;
  __syncthreads();
  u64 all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) all += s.scan[w];
  return all;
}
TSB_HD u64 block_scan(u64 v, Shared &s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  __syncthreads();
  if (lane == 31) s.scan[warp] = v;
  __syncthreads();
  u64 before = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) before += w < warp ? s.scan[w] : 0ull;
  return before + v;
}

// Appends a token to this CTA's part of the list.
TSB_HD void append(Shared &s, u64 token) {
  const unsigned int at = atomicAdd(&s.mine, 1u);
  if (at < (unsigned int)kList) s.list[at] = token;
}
// Hands the list of every other CTA to CTA 0.
__device__ __noinline__ void send_list(Shared &s, Shared *head, bool is_head) {
  __syncthreads();
  if (is_head) return;
  const int n = min((int)s.mine, kList);
  if (threadIdx.x == 0) s.base = atomicAdd(&head->others, s.mine);  // all of them: CTA 0 sees a list too long
  __syncthreads();
  for (int e = threadIdx.x; e < n; e += kThreads) {
    const unsigned int at = s.base + e;
    if (at < (unsigned int)kList) head->list[kList - 1 - at] = s.list[e];
  }
}
TSB_HD u64 listed(const Shared &s, int e) { return s.list[e < (int)s.mine ? e : kList - 1 - (e - (int)s.mine)]; }

// CTA 0: puts few[0, n) in order: order[i] the i-th token, up_to[i] the units of it
// and those before it. Two threads per token count the tokens before it.
__device__ __noinline__ void put_in_order(Shared &s, int n) {
  const int i = threadIdx.x / 2, half = threadIdx.x % 2;
  const u64 me = i < n ? s.few[i].x : 0;
  int rank = 0;
  u64 units = 0;
#pragma unroll 4
  for (int j = half; j < n; j += 2) {
    const ulonglong2 o = s.few[j];
    rank += o.x > me;
    units += o.x >= me ? o.y : 0ull;
  }
  rank += __shfl_xor_sync(0xffffffffu, rank, 1);
  units += __shfl_xor_sync(0xffffffffu, units, 1);
  if (half == 0 && i < n) {
    s.order[rank] = me;
    s.up_to[rank] = units;
  }
  __syncthreads();
}
// The place in that order of the token with which the running count or mass reaches
// bound: the last one that starts below it. `m`: the units before the first of them.
TSB_HD int cross(Shared &s, int n, u64 before, u64 m, double scale, u64 bound) {
  if (threadIdx.x == 0) s.found = 0;
  __syncthreads();
  const int i = threadIdx.x;
  if (i > 0 && i < n && s.up_to[i] > s.up_to[i - 1] && reach(before, m + s.up_to[i - 1], scale) < bound) atomicMax(&s.found, i);
  __syncthreads();
  return s.found;
}

// CTA 0: the first of the n listed tokens of `bin` (of any bin for bin < 0, counts
// only) at or above floor_token, along the order, with which the running count or
// mass (`before` the bin) reaches bound; into s.found_token and s.found_mass (what has
// been reached with it).
__device__ __noinline__ void narrow(Shared &s, int n, int bin, u64 floor_token, bool by_count, u64 bound, u64 before,
                                    const RowScale &r) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const double scale = by_count ? 1.0 : bin_scale((uint32_t)bin, s.octave);
  u64 base = 0;  // units of the bin's tokens that have been passed
  u64 lo = floor_token, hi = ~0ull;
  bool by_t = bin >= 0;  // first by t inside the bin, which is known; then by the tokens' own range
  // a token's sub-bin by t: the fraction that logit_bin rounds away, of 256 parts
  const float first = (float)bin - 0.5f;
  auto sub_of = [&](float x) { return (int)fminf(fmaxf((fmaf(r.top - x, r.scale, -first)) * (float)kSub, 0.f), (float)(kSub - 1)); };
  int by_t_sub = -1;  // the sub-bin by t that is left
  auto in = [&](u64 t) {
    return t >= lo && t <= hi && (bin < 0 || (logit_bin(token_logit(t), r) == (uint32_t)bin &&
                                              (by_t_sub < 0 || sub_of(token_logit(t)) == by_t_sub)));
  };
  u64 least = 0, most = 0;
  bool few = n <= kFewest;
  while (!few) {
    s.sub0[tid] = 0;
    s.sub1[tid] = 0;
    if (tid == 0) s.found = 0;
    int shift = 0;
    if (!by_t) {
      least = ~0ull;
      most = 0;
      for (int e = tid; e < n; e += kThreads) {
        const u64 t = listed(s, e);
        if (in(t)) {
          least = min(least, t);
          most = max(most, t);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      if (lane == 0) { s.red[warp] = least; s.red2[warp] = most; }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        least = min(least, s.red[w]);
        most = max(most, s.red2[w]);
      }
      shift = max(0, 64 - __clzll((long long)(most - least)) - 8);
    } else {
      __syncthreads();
    }
    for (int e = tid; e < n; e += kThreads) {
      const u64 t = listed(s, e);
      if (!in(t)) continue;
      const int sub = by_t ? sub_of(token_logit(t)) : (int)((most - t) >> shift);
      const uint32_t m = by_count ? 1u : logit_m(token_logit(t), (uint32_t)bin, r);
      atomicAdd(&s.sub0[sub], m & 4095u);
      if (!by_count) atomicAdd(&s.sub1[sub], m >> 12);
    }
    __syncthreads();
    const u64 own = (u64)s.sub0[tid] + ((u64)s.sub1[tid] << 12);
    const u64 up = base + block_scan(own, s);
    // the last sub-bin that starts below the bound holds it
    if (own && reach(before, up - own, scale) < bound) atomicMax(&s.found, tid);
    __syncthreads();
    if (tid == s.found) {
      s.last = up - own;
      s.temp = by_count ? own : own / (kUnitM - (kUnitM >> 6)) + 1;  // no more tokens than this: m > 2^22 * 63 / 64
    }
    __syncthreads();
    base = s.last;
    few = s.temp <= (u64)kFewest || (!by_t && shift == 0);
    if (by_t) {
      by_t_sub = s.found;
      by_t = false;
    } else {
      const u64 width = (1ull << shift) - 1, down = (u64)s.found << shift;
      hi = most > down ? most - down : 0ull;
      lo = max(lo, hi > width ? hi - width : 0ull);
    }
    __syncthreads();
  }
  if (tid == 0) s.few_n = 0;
  __syncthreads();
  for (int e = tid; e < n; e += kThreads) {
    const u64 t = listed(s, e);
    if (in(t)) {
      const u64 m = by_count ? 1 : logit_m(token_logit(t), (uint32_t)bin, r);
      s.few[atomicAdd(&s.few_n, 1u)] = make_ulonglong2(t, m);
    }
  }
  __syncthreads();
  const int have = (int)s.few_n;
  put_in_order(s, have);
  const int at = cross(s, have, before, base, scale, bound);
  if (tid == 0) {
    s.found_token = have ? s.order[at] : 0;
    s.found_mass = reach(before, have ? base + s.up_to[at] : base, scale);
  }
  __syncthreads();
}

// CTA 0: running sums of the histogram; returns the whole.
__device__ __noinline__ u64 run_sums(Shared &s, bool masses) {
  u64 v[kBinsPerThread], run = 0;
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    const int bin = threadIdx.x * kBinsPerThread + i;
    v[i] = bin >= kBins ? 0ull : masses ? reach(0, (u64)s.h0[bin] + ((u64)s.h1[bin] << 12), bin_scale(bin, s.octave)) : (u64)s.h0[bin];
    run += v[i];
  }
  u64 up = block_scan(run, s) - run;
#pragma unroll
  for (int i = 0; i < kBinsPerThread; ++i) {
    const int bin = threadIdx.x * kBinsPerThread + i;
    up += v[i];
    if (bin < kBins) s.sums[bin] = up;
  }
  __syncthreads();
  return s.sums[kBins - 1];
}
TSB_HD u64 before_bin(const Shared &s, int bin) { return bin > 0 ? s.sums[bin - 1] : 0ull; }
// CTA 0: the bin in which the running sum reaches bound (the last that adds to it, if none does).
__device__ __noinline__ int find_bin(Shared &s, u64 bound) {
  if (threadIdx.x == 0) s.found = 0;
  __syncthreads();
  bound = min(bound, s.sums[kBins - 1]);
#pragma unroll
  for (int bin = threadIdx.x; bin < kBins; bin += kThreads) {
    const u64 here = s.sums[bin], before = before_bin(s, bin);
    if (here >= bound && before < bound) atomicMax(&s.found, bin);
  }
  __syncthreads();
  const int bin = s.found;
  __syncthreads();
  return bin;
}

// u's bound on the running mass, which the sample's cumulative mass exceeds: the
// next whole number above u * total. Past the last token it is the total.
TSB_HD u64 sample_bound(float u, u64 total) {
  const double want = u > 0.f ? (double)u * (double)total : 0.0;
  return want < (double)total ? min(__double2ull_rd(want) + 1, total) : total;
}
// top-p's bound on it, which the mass of the kept tokens reaches: at least one, which
// keeps the first token.
TSB_HD u64 top_p_bound(double p, u64 total) {
  return min(max(__double2ull_ru(fmax(p, 0.0) * (double)total), 1ull), total);
}
// Of tokens of m each in one bin, behind `base` units of it: how many reach bound, one of `most` at least.
TSB_HD u64 ties_for(u64 before, u64 base, uint32_t m, u64 most, double scale, u64 bound) {
  const double missing = bound > reach(before, base, scale) ? (double)(bound - reach(before, base, scale)) : 0.0;
  u64 j = min(max(__double2ull_ru(missing / ((double)m * scale)), 1ull), most);
  while (j > 1 && reach(before, base + (j - 1) * m, scale) >= bound) --j;  // the rounding of a unit: a step or two
  while (j < most && reach(before, base + j * m, scale) < bound) ++j;
  return j;
}
// No more tokens than this make up `mass` in a bin: m > 0.989 * 2^22, and the mass was
// rounded by half a unit, half of the smallest weight.
TSB_HD uint32_t most_tokens(u64 mass, int bin) {
  return (uint32_t)((float)mass * (float)kPerUnit * exp2f((float)bin * (1.f / kStep)) * 1.03f) + 1;
}

TSB_HD void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
TSB_HD void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
TSB_HD void cluster_barrier() {
  cluster_arrive();
  cluster_wait();
}

template <typename T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if (tid == 0) { s.mine = 0; s.others = 0; s.first = 0xffffffffu; s.overflow = 0; }
  if (tid < 3) s.floor0[tid] = s.floor1[tid] = 0;
  for (int i = tid; i < kBins; i += kThreads) s.sums[i] = 0;  // h0 and h1
  if (tid < kStep) s.octave[tid] = kOctave[tid];
  cluster_arrive();  // waited for before the first access to another CTA's shared memory
  griddep_wait();    // programmatic dependent: the logits are the previous kernel's
  griddep_launch_dependents();

  // ---- this CTA's logits, tokens [lo, lo + n): elements [off, off + n) of data
  const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
  const int lo = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - lo);
  const T *data = x + lo;
  const int off = (int)((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
  data -= off;
  const int index0 = lo - off;  // token of element 0
  constexpr int VEC = 16 / sizeof(T);
  const float u = a.u[row];
  const float temperature_row = a.temperature ? a.temperature[row] : 0.f;
  const float p_row = a.top_p ? a.top_p[row] : 0.f, floor_row = a.min_p ? a.min_p[row] : 0.f;
  const int k = a.top_k ? a.top_k[row] : a.top_k_s;
  float top = -INFINITY;  // this thread's largest logit
  {
    T *stage = reinterpret_cast<T *>(smem + kSharedBytes);
    for_vectors<T, 4>(
        off, n,
        [&](int v) {
          const uint4 w = ldg_nc_v4(data + v * VEC);
          if (a.staged) *reinterpret_cast<uint4 *>(stage + v * VEC) = w;
          top = fmaxf(top, max_of(w, T()));
        },
        [&](int i) {
          const T w = data[i];
          if (a.staged) stage[i] = w;
          top = fmaxf(top, to_float(w));
        });
    if (a.staged) data = stage;  // a thread reads back what it wrote itself
  }
  double temperature = a.temperature ? (double)temperature_row : a.temperature_s;
  const double p = a.top_p ? (double)p_row : a.top_p_s;
  const double floor_w = a.min_p ? (double)floor_row : a.min_p_s;
  const bool greedy = !(temperature > 0.0), use_p = p < 1.0, use_floor = floor_w > 0.0;
  bool use_k = k > 0 && k < a.vocab;
  temperature = fmin(fmax(temperature, kMinTemperature), kMaxTemperature);
  RowScale r;
  double per_t;  // 1 / temperature
  {
    const float guess = 1.f / (float)temperature;  // one Newton step leaves an error below 2^-44
    per_t = fma((double)guess, fma(-temperature, (double)guess, 1.0), (double)guess);
    const double scale = per_t * (1.4426950408889634 * kStep);
    r.scale = (float)scale;
    r.low = (float)(scale - (double)r.scale);
  }
  Shared *const head = cluster.map_shared_rank(&s, 0);
  auto emit = [&](float v, int token, double kept) {
    if (token >= 0) a.token[row] = token;
    if (a.logprob) {
      const double d = v == top ? 0.0 : ((double)v - (double)top) * per_t;
      const float f = (float)kept;  // log(kept) = log(f) + (kept - f) / f
      a.logprob[row] = (float)(d - ((double)logf(f) + (double)((float)(kept - (double)f) / f)));
    }
  };
  auto nothing = [&]() {
    a.token[row] = -1;
    if (a.logprob) a.logprob[row] = -INFINITY;
  };

  // ---- small top-k: the tokens that some k lanes' maxima reach
  if (!greedy && use_k && k <= kDirectK) {
    int before = 0;  // lanes of the warp with a larger maximum
#pragma unroll
    for (int o = 1; o < 32; ++o) {
      const int from = (lane + o) % 32;
      const float other = __shfl_sync(0xffffffffu, top, from);
      before += other > top || (other == top && from < lane);
    }
    if (before == (k - 1) / kWarps) s.red[warp] = __float_as_uint(top);  // ceil(k / warps) lanes of each warp reach it
    if (before == 0) s.red2[warp] = __float_as_uint(top);
    __syncthreads();
    float cut = INFINITY, most = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      cut = fminf(cut, __uint_as_float((uint32_t)s.red[w]));
      most = fmaxf(most, __uint_as_float((uint32_t)s.red2[w]));
    }
    cluster_wait();
    // each CTA has a part of CTA 0's list
    for_hits<T>(
        data, off, n, [&](float e) { return e >= cut && e > -INFINITY; },
        [&](int i, float e) {
          const unsigned int at = atomicAdd(&s.mine, 1u);
          if (at < (unsigned int)kPart) head->list[rank * kPart + at] = make_token(e, index0 + i);
        });
    __syncthreads();
    if (tid == 0) {
      head->peer_top[rank] = most;
      head->peer_cut[rank] = cut;
      head->peer_ties[rank] = s.mine;
    }
    // too many (equal logits, or hardly any live ones): all CTAs take the general way
    if (s.mine > (unsigned int)kPart && tid < ctas) cluster.map_shared_rank(&s, tid)->overflow = 1;
    cluster_barrier();
    if (!s.overflow) {
      if (rank != 0) return;
      // bring the parts together
      u64 mine[kMaxCluster];
      int at[kMaxCluster], m = 0;
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q) {
        const int part = q < ctas ? (int)s.peer_ties[q] : 0;
        at[q] = tid < part ? m + tid : -1;
        mine[q] = tid < part ? s.list[q * kPart + tid] : 0ull;
        m += part;
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < kMaxCluster; ++q)
        if (at[q] >= 0) s.list[at[q]] = mine[q];
      if (tid == 0) s.mine = (unsigned int)m;
      // a histogram of the logits between the lowest cut and the top leaves about k tokens
      for (int q = 0; q < ctas; ++q) {
        top = fmaxf(q ? top : -INFINITY, s.peer_top[q]);
        cut = fminf(cut, s.peer_cut[q]);
      }
      r.top = top;
      const float per_sub = (float)kSub / (top - cut);
      auto sub_of = [&](u64 t) { return (int)fminf((top - token_logit(t)) * per_sub, (float)(kSub - 1)); };  // NaN: the last
      s.sub0[tid] = 0;
      if (tid == 0) { s.found = 0; s.few_n = 0; }
      __syncthreads();
      for (int e = tid; e < m; e += kThreads) atomicAdd(&s.sub0[sub_of(listed(s, e))], 1u);
      __syncthreads();
      const u64 own = s.sub0[tid], up = block_scan(own, s);
      if (own && up - own < (u64)k) atomicMax(&s.found, tid);
      __syncthreads();
      int last = s.found;
      if (tid == last) s.temp = up;
      __syncthreads();
      u64 floor_token = 0;
      if (s.temp > (u64)kFewest) {  // many in one part of the histogram: find the k-th itself
        narrow(s, m, -1, 0, true, (u64)k, 0, r);
        floor_token = s.found_token;
        last = kSub;
        if (tid == 0) s.few_n = 0;
        __syncthreads();
      }
      for (int e = tid; e < m; e += kThreads) {
        const u64 t = listed(s, e);
        if (t < floor_token || sub_of(t) > last) continue;
        const float v = token_logit(t);
        const u64 w = v == top ? list_units(1.0) : top == INFINITY ? 0 : list_units(logit_mass(v, r, s.octave));
        s.few[atomicAdd(&s.few_n, 1u)] = make_ulonglong2(t, w);
      }
      __syncthreads();
      const int all = (int)s.few_n;
      put_in_order(s, all);
      const int have = min(all, k);
      if (have == 0) {
        if (tid == 0) nothing();
      } else {
        u64 kept = s.up_to[have - 1];
        if (use_p) kept = s.up_to[cross(s, have, 0, 0, 1.0, top_p_bound(p, kept))];
        if (use_floor) {  // of those in order the ones up to the last of weight >= min_p, at least the first
          __syncthreads();
          if (tid == 0) s.found = 0;
          __syncthreads();
          if (tid < have && (double)(s.up_to[tid] - (tid ? s.up_to[tid - 1] : 0ull)) >= floor_w * kListUnit) atomicMax(&s.found, tid);
          __syncthreads();
          kept = min(kept, s.up_to[s.found]);
        }
        __syncthreads();
        const int at = cross(s, have, 0, 0, 1.0, sample_bound(u, kept));
        if (tid == 0) emit(token_logit(s.order[at]), token_index(s.order[at]), (double)kept / kListUnit);
      }
      return;
    }
    cluster_barrier();  // `overflow` has been read: the CTAs go on together
    if (tid == 0) s.mine = 0;
  } else {
    cluster_wait();
  }

  // ---- 1. the largest logit
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  __syncthreads();
  if (lane == 0) s.red[warp] = __float_as_uint(top);
  __syncthreads();
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, __uint_as_float((uint32_t)s.red[w]));
  if (tid < ctas) cluster.map_shared_rank(&s, tid)->peer_top[rank] = top;
  cluster_barrier();
#pragma unroll 1
  for (int c = 0; c < ctas; ++c) top = fmaxf(top, s.peer_top[c]);

  if (top == -INFINITY) {  // every logit is -inf or NaN: there is no token to choose
    if (rank == 0 && tid == 0) nothing();
    return;
  }
  if (greedy) {
    unsigned int first = 0xffffffffu;
    for_hits<T>(
        data, off, n, [&](float v) { return v == top; },
        [&](int i, float) { first = min(first, (unsigned int)(index0 + i)); });
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first != 0xffffffffu) atomicMin(&head->first, first);
    cluster_barrier();
    if (rank == 0 && tid == 0) {
      a.token[row] = (int)s.first;
      if (a.logprob) a.logprob[row] = 0.f;
    }
    return;
  }
  r.top = top;
  const bool counted = use_k;

  auto tell = [&](int mode, int b0, int b1) {  // CTA 0 to all
    if (tid < ctas) {
      Shared *peer = cluster.map_shared_rank(&s, tid);
      peer->mode = mode;
      peer->lo = b0;
      peer->hi = b1;
    }
  };
  // All CTAs: token number `tie` (CTA 0 knows it) of those with this logit, in index order.
  auto pick = [&](float v, u64 kept, auto tie_of) {
    unsigned int ties = 0;
    for_logits<T>(data, off, n, [&](int, float e) { ties += e == v; });
    ties = (unsigned int)block_sum(ties, s);
    if (tid == 0) head->peer_ties[rank] = ties;
    cluster_barrier();
    if (rank == 0 && tid == 0) {
      unsigned int all = 0;
      for (int q = 0; q < ctas; ++q) all += s.peer_ties[q];
      unsigned int tie = min((unsigned int)tie_of(all, kept), all - 1);
      int q = 0;
      while (q < ctas - 1 && tie >= s.peer_ties[q]) tie -= s.peer_ties[q++];
      for (int c = 0; c < ctas; ++c) {
        Shared *peer = cluster.map_shared_rank(&s, c);
        peer->pick_rank = q;
        peer->pick_tie = (int)tie;
      }
      emit(v, -1, (double)kept * kPerUnit);
    }
    cluster_barrier();
    if (rank != s.pick_rank) return;
    unsigned int seen = 0;  // ties before this block of tokens
    for (int at = 0; at < n; at += kThreads) {
      const bool hit = at + tid < n && to_float(data[off + at + tid]) == v;
      const unsigned int up = (unsigned int)block_scan(hit ? 1ull : 0ull, s);
      if (hit && seen + up - 1 == (unsigned int)s.pick_tie) a.token[row] = lo + at + tid;
      for (int q = 0; q < kWarps; ++q) seen += (unsigned int)s.scan[q];
      if (seen > (unsigned int)s.pick_tie) return;
    }
  };

  if (top == INFINITY) {  // the +inf logits share all the weight equally
    pick(top, 0, [&](unsigned int all, u64 &kept) {
      u64 n = use_k ? min((u64)all, (u64)k) : (u64)all;
      if (use_p) n = top_p_bound(p, n);
      if (use_floor && floor_w > 1.0) n = 1;
      kept = n * kOne;
      return sample_bound(u, n) - 1;
    });
    return;
  }

  // ---- 2. the histogram, added up in CTA 0
  auto push = [&](bool both) {
    __syncthreads();
    if (rank != 0) {
#pragma unroll 1
      for (int i = tid; i < kBins; i += kThreads) {
        if (s.h0[i]) atomicAdd(&head->h0[i], s.h0[i]);
        if (both && s.h1[i]) atomicAdd(&head->h1[i], s.h1[i]);
      }
    }
  };
  auto count_tokens = [&]() {
    for_logits<T>(data, off, n, [&](int, float v) {
      const uint32_t bin = logit_bin(v, r);
      if (bin < (uint32_t)kBins) atomicAdd(&s.h0[bin], 1u);
    });
    push(false);
  };
  auto add_masses = [&]() {
    for_logits<T>(data, off, n, [&](int, float v) {
      const uint32_t bin = logit_bin(v, r);
      if (bin < (uint32_t)kBins) {
        const uint32_t m = logit_m(v, bin, r);
        atomicAdd(&s.h0[bin], m & 4095u);
        atomicAdd(&s.h1[bin], m >> 12);
      }
    });
    push(true);
  };
  // The mass of the weights that min-p keeps, a prefix of the bins and part of one, which
  // is one of three: t of min_p, in steps of 1 / kStep, is known to a small part of a step,
  // and a bin's tokens are within half of one. What of their m stays, of the tokens that
  // for_each gives, is added up once a row, into floor0 and floor1.
  int floor_bin = 0;  // the first of the three
  if (use_floor) {
    const float t = -log2f((float)floor_w) * (float)kStep;
    floor_bin = (int)fminf(fmaxf(rintf(t), 0.f), (float)(kBins + 1)) - 1;
  }
  auto floor_units = [&](auto for_each) {
    uint32_t m0[3] = {0, 0, 0}, m1[3] = {0, 0, 0};
    for_each([&](float v) {
      const uint32_t bin = logit_bin(v, r), at = bin - (uint32_t)floor_bin;
      if (at >= 3u || bin >= (uint32_t)kBins) return;
      const uint32_t m = logit_m(v, bin, r);
      if ((double)m * bin_unit(bin, s.octave) < floor_w) return;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        m0[i] += at == (uint32_t)i ? m & 4095u : 0u;
        m1[i] += at == (uint32_t)i ? m >> 12 : 0u;
      }
    });
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      if (!__any_sync(0xffffffffu, m1[i] != 0)) continue;  // m has 22 bits and more
      const uint32_t low = __reduce_add_sync(0xffffffffu, m0[i]), high = __reduce_add_sync(0xffffffffu, m1[i]);
      if (lane == 0) {
        atomicAdd(&s.floor0[i], low);
        atomicAdd(&s.floor1[i], high);
      }
    }
    __syncthreads();
  };
  auto floor_of = [&](int i) { return (u64)s.floor0[i] + ((u64)s.floor1[i] << 12); };
  auto floor_mass = [&](auto units) {  // CTA 0: with the running masses
    u64 mass = before_bin(s, floor_bin);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const u64 m = units(i);
      if (m) mass = reach(before_bin(s, floor_bin + i), m, bin_scale(floor_bin + i, s.octave));
    }
    return max(mass, kOne);  // always the first
  };
  auto add_floor = [&]() {
    floor_units([&](auto take) {
      for_hits<T>(
          data, off, n, [&](float v) { return logit_bin(v, r) - (uint32_t)floor_bin < 3u; }, [&](int, float v) { take(v); });
    });
    if (tid < 3) head->peer_floor[rank][tid] = floor_of(tid);
  };
  auto floor_sum = [&]() {
    return floor_mass([&](int i) {
      u64 m = 0;
      for (int q = 0; q < ctas; ++q) m += s.peer_floor[q][i];
      return m;
    });
  };
  auto gather = [&](int b0, int b1) {  // all CTAs, into CTA 0's list
    for_hits<T>(
        data, off, n, [&](float v) { return logit_bin(v, r) - (uint32_t)b0 <= (uint32_t)(b1 - b0); },
        [&](int i, float v) { append(s, make_token(v, index0 + i)); });
    send_list(s, head, rank == 0);
  };

  if (use_k) {
    count_tokens();
  } else {
    add_masses();
    if (use_floor && !use_p) add_floor();
  }
  cluster_barrier();

  // ---- 3. what to gather: CTA 0 decides
  u64 total = 0, above_floor = 0;
  int k_bin = 0;
  u64 k_before = 0, k_in = 0;  // tokens before and in top-k's bin
  if (rank == 0) {
    total = run_sums(s, !use_k);
    if (use_k) {
      use_k = (u64)k < total;  // else every token with a mass is among the first k
      k_bin = use_k ? find_bin(s, (u64)k) : kBins - 1;
      k_before = before_bin(s, k_bin);
      k_in = s.sums[k_bin] - k_before;
      tell(k_before + k_in <= (u64)kList ? kFew : kSlow, 0, k_bin);
    } else {
      int b0 = 0, b1;
      if (use_p) {
        b1 = find_bin(s, top_p_bound(p, total));
      } else {
        if (use_floor) above_floor = floor_sum();
        b0 = b1 = find_bin(s, sample_bound(u, use_floor ? min(total, above_floor) : total));
      }
      uint32_t tokens = 0;  // a bound on the tokens of the bins
      for (int bin = b0 + tid; bin <= b1; bin += kThreads) {
        const u64 mass = s.sums[bin] - before_bin(s, bin);
        if (mass) tokens += most_tokens(mass, bin);
      }
      tell(block_sum(tokens, s) <= (u64)kList ? kFew : kSlow, b0, b1);
    }
  }
  cluster_barrier();
  if (s.mode == kFew) {
    gather(s.lo, s.hi);
    cluster_barrier();
    if (rank != 0) return;
    const int m = min((int)(s.mine + s.others), kList);
    u64 floor_token = 0;
    u64 kept = total;
    if (counted) {
      // the list holds the first k, or every token with a mass: their masses by bin
      if (use_k) {
        narrow(s, m, k_bin, 0, true, (u64)k, k_before, r);
        floor_token = s.found_token;
      }
      for (int i = tid; i < kBins; i += kThreads) s.sums[i] = 0;
      __syncthreads();
      for (int e = tid; e < m; e += kThreads) {
        const u64 t = listed(s, e);
        if (t < floor_token) continue;
        const uint32_t bin = logit_bin(token_logit(t), r), w = logit_m(token_logit(t), bin, r);
        atomicAdd(&s.h0[bin], w & 4095u);
        atomicAdd(&s.h1[bin], w >> 12);
      }
      __syncthreads();
      kept = run_sums(s, true);
    }
    if (use_p) {
      const u64 bound = top_p_bound(p, kept);
      const int bin = find_bin(s, bound);
      narrow(s, m, bin, floor_token, false, bound, before_bin(s, bin), r);
      kept = s.found_mass;
    }
    if (use_floor) {
      if (counted || use_p) {  // min-p keeps a prefix of the order: what of it is in the list decides
        floor_units([&](auto take) {
#pragma unroll 1
          for (int e = tid; e < m; e += kThreads) {
            const u64 t = listed(s, e);
            if (t >= floor_token) take(token_logit(t));
          }
        });
        above_floor = floor_mass(floor_of);
      }
      kept = min(kept, above_floor);
    }
    const u64 bound = sample_bound(u, kept);
    const int bin = find_bin(s, bound);
    narrow(s, m, bin, floor_token, false, bound, before_bin(s, bin), r);
    if (tid == 0) emit(token_logit(s.found_token), token_index(s.found_token), (double)kept * kPerUnit);
    return;
  }

  // ---- many candidates: one bound after the other, each resolved inside its bin
  if (counted) {  // the masses are still to be added up
    for (int i = tid; i < kBins; i += kThreads) s.sums[i] = 0;
    cluster_barrier();
    add_masses();
  }
  if (use_floor && (counted || use_p)) add_floor();
  cluster_barrier();
  if (rank == 0) {
    if (counted) total = run_sums(s, true);
    if (use_floor) above_floor = floor_sum();
  }
  u64 kept = total;  // CTA 0
  for (int stage = 0; stage < 3; ++stage) {  // top-k, top-p, u
    if (stage == 0 ? !counted : stage == 1 && !use_p) continue;
    u64 bound = 0, mass_before = 0, count_before = 0;
    if (rank == 0) {
      if (stage == 2 && use_floor) kept = min(kept, above_floor);
      int bin;
      if (stage == 0) {
        bound = (u64)k;
        bin = k_bin;
        count_before = k_before;
      } else {
        bound = stage == 1 ? top_p_bound(p, kept) : sample_bound(u, kept);
        bin = find_bin(s, bound);
      }
      mass_before = before_bin(s, bin);
      const u64 tokens = stage == 0 ? k_in : most_tokens(s.sums[bin] - mass_before, bin);
      // nothing to resolve where every token with a mass is kept
      const int mode = stage == 0 && !use_k ? kNoMass : tokens <= (u64)kList ? kOneBin : kRadix;
      if (tid == 0) s.others = 0;
      tell(mode, bin, bin);
    }
    if (tid == 0) s.mine = 0;
    cluster_barrier();
    const int mode = s.mode, bin = s.lo;
    const double scale = bin_scale((uint32_t)bin, s.octave);
    if (mode == kNoMass) {
      cluster_barrier();  // the plan has been read: CTA 0 may write the next one
      continue;
    }
    if (mode == kOneBin) {
      gather(bin, bin);
      cluster_barrier();
      if (rank != 0) continue;
      const int m = min((int)(s.mine + s.others), kList);
      narrow(s, m, bin, 0, stage == 0, bound, stage == 0 ? count_before : mass_before, r);
      const u64 token = s.found_token;
      if (stage == 2) {
        if (tid == 0) emit(token_logit(token), token_index(token), (double)kept * kPerUnit);
      } else if (stage == 1) {
        kept = s.found_mass;
      } else {  // the mass of the first k
        u64 units = 0;
        for (int e = tid; e < m; e += kThreads) {
          const u64 t = listed(s, e);
          if (t >= token) units += logit_m(token_logit(t), (uint32_t)bin, r);
        }
        kept = reach(mass_before, block_sum(units, s), scale);
      }
      __syncthreads();
      continue;
    }
    // radix descent over the keys of the bin, eight bits at a time: counts in the
    // narrowing histogram's first half, m in two words of the list
    unsigned int *const low = reinterpret_cast<unsigned int *>(s.list), *const high = low + kSub;
    uint32_t prefix = 0;
    u64 base_m = 0, base_c = 0, ties = 0;  // CTA 0: of the bin's tokens before the prefix's, and (at the end) how many have it
    for (int shift = 24; shift >= 0; shift -= 8) {
      s.sub0[tid] = 0;
      low[tid] = 0;
      high[tid] = 0;
      __syncthreads();
      for_logits<T>(data, off, n, [&](int, float v) {
        if (logit_bin(v, r) != (uint32_t)bin) return;
        const uint32_t key = (uint32_t)(make_token(v, 0) >> 32);
        if (shift < 24 && (key >> (shift + 8)) != prefix) return;
        const uint32_t digit = (key >> shift) & 255u, m = logit_m(v, (uint32_t)bin, r);
        atomicAdd(&s.sub0[digit], 1u);
        atomicAdd(&low[digit], m & 4095u);
        atomicAdd(&high[digit], m >> 12);
      });
      cluster_barrier();
      if (rank == 0) {
        u64 m = 0, c = 0;
        const int digit = 255 - tid;  // descending
        for (int q = 0; q < ctas; ++q) {
          const Shared *peer = cluster.map_shared_rank(&s, q);
          const unsigned int *words = reinterpret_cast<const unsigned int *>(peer->list);
          c += peer->sub0[digit];
          m += (u64)words[digit] + ((u64)words[kSub + digit] << 12);
        }
        if (tid == 0) s.found = 0;
        const u64 from_m = base_m + block_scan(m, s) - m, from_c = base_c + block_scan(c, s) - c;
        const u64 start = stage == 0 ? count_before + from_c : reach(mass_before, from_m, scale);
        // the last digit with a token that starts below the bound holds it
        if (c && start < bound) atomicMax(&s.found, tid);
        __syncthreads();
        if (tid == s.found) { s.found_mass = from_m; s.temp = from_c; s.last = c; }
        __syncthreads();
        base_m = s.found_mass;
        base_c = s.temp;
        ties = s.last;
        if (tid < ctas) cluster.map_shared_rank(&s, tid)->prefix = prefix << 8 | (uint32_t)(255 - s.found);
      }
      cluster_barrier();
      prefix = s.prefix;
    }
    // every token left has the same logit: some of them come before the one wanted
    const float v = key_logit(prefix);
    u64 wanted = 0;
    if (rank == 0) {
      const uint32_t m = logit_m(v, (uint32_t)bin, r);
      wanted = stage == 0 ? min(bound - count_before - base_c, ties) : ties_for(mass_before, base_m, m, ties, scale, bound);
      if (stage < 2) kept = reach(mass_before, base_m + wanted * m, scale);
    }
    if (stage < 2) continue;
    pick(v, kept, [&](unsigned int, u64) { return wanted - 1; });
    return;
  }
}

// CTAs per row: a slice that stays in shared memory beside a second CTA, and
// more of them while there are fewer CTAs than SMs and a slice is long enough to
// be worth a barrier.
template <typename T>
int launch_sample(SampleArgs a, int rows, cudaStream_t st) {
  int ctas = 1;
  while (ctas < kMaxCluster && ((size_t)a.vocab * sizeof(T) / ctas > kSliceBytes ||
                                ((long long)rows * ctas * 2 <= sm_count() && a.vocab / ctas >= 2 * kSliceMin)))
    ctas *= 2;
  a.slice = ((a.vocab + ctas - 1) / ctas + 7) & ~7;
  const size_t stage = ((size_t)a.slice + 16 / sizeof(T)) * sizeof(T);
  // The logits stay in shared memory while two CTAs fit an SM that way, and where a CTA has
  // the SM to itself for two rounds of rows; else the later passes read them from L2, with
  // three CTAs an SM. Inputs that come from DRAM, vocabularies of 32003 to 600011: two to an SM,
  // staged is up to 25% faster at 1 to 256 rows (48 x 100003 float32: flat 36.7 us against 38.6,
  // mixed settings 34.1 / 40.1; 128 x 151936 bf16 73 / 87 and 61 / 75). One to an SM: 16 x 262144
  // float32 91 / 134 and 38 / 62, 36 rows 146 / 148 and 60 / 72, 48 rows 184 / 151 and 78 / 78,
  // 90 rows 287 / 233 and 122 / 101. (An input that is sampled again while it is in L2 hides the
  // later passes: 48 x 100003 float32, replayed, 28.7 us unstaged.)
  const size_t per_sm = kSmemPerSm / (kSharedBytes + stage + 1024);
  a.staged = stage <= kMaxStage && (per_sm >= 2 || (long long)rows * ctas <= 2LL * sm_count());
  const size_t smem = kSharedBytes + (a.staged ? stage : 0);
  static std::atomic<unsigned long long> ready{0};  // devices on which the attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TSB_ECUDA;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)(kSharedBytes + kMaxStage)) != cudaSuccess)
      return TSB_ECUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, (const SampleArgs)a) == cudaSuccess ? TSB_OK : TSB_ECUDA;
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_sample(const void *logits, int logits_dtype, int rows, int vocab, long long row_stride,
                          const float *u, const float *temperature, double temperature_all, const int32_t *top_k,
                          int top_k_all, const float *top_p, double top_p_all, const float *min_p, double min_p_all,
                          int32_t *token, float *logprob, tsb_stream_t stream) {
  if (!logits || !u || !token) return TSB_EINVAL;
  if (rows <= 0 || vocab <= 0 || (rows > 1 && row_stride < vocab)) return TSB_EINVAL;
  if (vocab > kMaxVocab || rows > 0x7fffffff / kMaxCluster) return TSB_EUNSUPPORTED;
  SampleArgs a = {};
  a.logits = logits;
  a.u = u;
  a.temperature = temperature;
  a.top_p = top_p;
  a.min_p = min_p;
  a.top_k = top_k;
  a.temperature_s = temperature_all;
  a.top_p_s = top_p_all;
  a.min_p_s = min_p_all;
  a.top_k_s = top_k_all;
  a.vocab = vocab;
  a.row_stride = row_stride;
  a.token = token;
  a.logprob = logprob;
  cudaStream_t st = (cudaStream_t)stream;
  switch (logits_dtype) {
    case TSB_MASK_BF16: return aligned(logits, 2) ? launch_sample<__nv_bfloat16>(a, rows, st) : TSB_EINVAL;
    case TSB_MASK_F16: return aligned(logits, 2) ? launch_sample<__half>(a, rows, st) : TSB_EINVAL;
    case TSB_MASK_F32: return aligned(logits, 4) ? launch_sample<float>(a, rows, st) : TSB_EINVAL;
    default: return TSB_EUNSUPPORTED;
  }
}
