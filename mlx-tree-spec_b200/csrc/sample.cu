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
//   the first k and walks with one warp. One cluster barrier in all.
// Otherwise:
//   1. The maximum, exchanged through distributed shared memory.
//   2. A histogram over t in steps of 1/32, so fine that a bin holds few tokens:
//      of counts with top-k, else of masses. The CTAs add theirs into CTA 0's.
//   3. CTA 0 finds the bins in which the bounds fall; the tokens of those bins
//      (all bins up to the last one wanted, or the sample's own bin alone) are
//      gathered in its shared memory, and a bound is resolved among the tokens of
//      its bin: histograms over their (logit, index) narrow them down to 32 or
//      fewer, which one warp sorts and walks.
// Where the kept tokens are too many to list, the bounds are resolved one after
// the other, each with a list of its own bin, or, for a bin of thousands of
// nearly equal logits, by a radix descent over their bits.
//
// Masses are integers, units of 2^-42 of the largest weight: sums do not depend
// on the order of the additions, results repeat bit for bit, and a row's mass
// stays below 2^62. A token's mass is m * 2^(19 - t's octave), m of 24 bits from a
// float32 power series of the exactly reduced t; the roundings of m are independent
// from token to token and do not add up. A bin lies in one octave, so its sum of
// m needs two 32-bit shared-memory atomics per token (12 bits each, 2^20 tokens
// do not overflow them); a 64-bit one would be a compare-and-swap loop.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

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
constexpr int kDirectK = 64;           // top-k up to here is looked for among the lanes' maxima
constexpr int kSub = kThreads;         // bins of a narrowing histogram, one per thread
constexpr u64 kOne = 1ull << 42;       // the mass of the largest weight
constexpr int kTopM = 1 << 23;         // its m
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxStage = 160 * 1024;  // bytes of logits a CTA holds in shared memory
constexpr size_t kSliceBytes = 48 * 1024;  // of logits in a CTA, while there are CTAs to split them over
constexpr int kSliceMin = 4096;            // logits of a slice that is not split further
constexpr double kMinTemperature = 8.673617379884035e-19;  // 2^-60

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

// Largest of 16 bytes of logits and m; NaN is skipped.
TSB_HD float max_of(const uint4 &v, float m, float) {
  return fmaxf(fmaxf(m, fmaxf(__uint_as_float(v.x), __uint_as_float(v.y))),
               fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
}
TSB_HD float max_of(const uint4 &v, float m, __nv_bfloat16) {
  const __nv_bfloat162 a = __hmax2(__hmax2(u32_as_bf2(v.x), u32_as_bf2(v.y)), __hmax2(u32_as_bf2(v.z), u32_as_bf2(v.w)));
  return fmaxf(m, fmaxf(__low2float(a), __high2float(a)));
}
TSB_HD float max_of(const uint4 &v, float m, __half) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
  const __half2 a = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  return fmaxf(m, fmaxf(__low2float(a), __high2float(a)));
}

// Order-preserving bits: a larger logit has a larger key, -0 that of +0.
TSB_HD uint32_t logit_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
TSB_HD float key_logit(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

// A row whose largest logit is finite.
struct RowScale {
  float top;        // the largest logit
  float bin_scale;  // kStep * c
  float c, c_low;   // log2(e) / temperature
};

// Bin of a logit, never decreasing as the logit falls: round(kStep * t). At or past
// kBins for a token without mass, -inf and NaN among them (the float's bits are
// compared as a number).
TSB_HD uint32_t logit_bin(float x, const RowScale &r) {
  return __float_as_uint(fmaf(r.top - x, r.bin_scale, 8388608.f)) - 0x4B000000u;
}

// m of a token of bin < kBins: its weight as m * 2^-(23 + bin / kStep), except that
// beyond the 19th octave, where units of 2^-42 are coarser, m is already in them.
// t is d * c with the product's and c's own rounding errors put back; 2^-t from
// the power series of e^z, |z| <= 0.36 (the next term is below 2^-26).
TSB_HD uint32_t logit_m(float x, uint32_t bin, const RowScale &r) {
  const float d = r.top - x;
  const uint32_t n = bin / kStep;
  const float t = d * r.c;
  const float t_low = fmaf(d, r.c_low, fmaf(d, r.c, -t));
  const float f = (t - (__uint_as_float(0x4B000000u | n) - 8388608.f)) + t_low;
  const float z = (0.5f - f) * 0.693147180559945f;
  float p = 1.f / 5040.f;
  p = fmaf(p, z, 1.f / 720.f);
  p = fmaf(p, z, 1.f / 120.f);
  p = fmaf(p, z, 1.f / 24.f);
  p = fmaf(p, z, 1.f / 6.f);
  p = fmaf(p, z, 0.5f);
  p = fmaf(p, z, 1.f);
  p = fmaf(p, z, 1.f);
  uint32_t m = (uint32_t)__float2int_rn(p * (0.70710678118654752f * 8388608.f));
  if (t == 0.f) m = kTopM;
  if (n > 19) m = (m + (1u << (n - 20))) >> (n - 19);
  return m;
}
// Units of 2^-42 in a sum of the m of one bin.
TSB_HD u64 bin_units(u64 m, uint32_t bin) {
  const uint32_t n = bin / kStep;
  return n < 19 ? m << (19 - n) : m;
}
TSB_HD u64 logit_mass(float x, const RowScale &r) {
  const uint32_t bin = logit_bin(x, r);
  return bin < (uint32_t)kBins ? bin_units(logit_m(x, bin, r), bin) : 0;
}
// No more tokens than this can make up `mass` units in a bin (a token's t is
// within the bin's rounding, with room to spare); past the point where a unit is
// coarse there is no useful bound.
TSB_HD u64 most_tokens(u64 mass, int bin) {
  const float least = exp2f(42.f - ((float)bin + 0.75f) / (float)kStep);
  return least >= 256.f ? mass / (u64)(least - 2.f) : ~0ull;
}

// How the tokens that a bound falls among are resolved.
enum Mode { kFew, kSlow, kOneBin, kRadix, kNoMass };

struct Shared {
  union {
    struct {
      unsigned int h0[kBins], h1[kBins];  // histogram: counts, or the low and high 12 bits of m
    };
    u64 sums[kBins];                      // CTA 0: running counts or masses up to and including a bin
  };
  u64 list[kList];                        // CTA 0: gathered tokens, key << 32 | ~index
  u64 few[kDirectK];
  unsigned int sub0[kSub], sub1[kSub];
  float peer_top[kMaxCluster];
  u64 peer_floor[kMaxCluster];            // CTA 0
  unsigned int peer_ties[kMaxCluster];
  u64 red[kWarps], red2[kWarps];
  u64 scan[kWarps];
  u64 found_mass, found_token;
  int found;
  unsigned int list_n, few_n, first;
  // written by CTA 0 into every CTA
  int mode, lo, hi;
  uint32_t prefix;
  int pick_rank, pick_tie;
};
constexpr size_t kSharedBytes = (sizeof(Shared) + 15) & ~size_t(15);
static_assert(kSharedBytes + kMaxStage <= 227 * 1024, "shared memory");
static_assert(sizeof(u64) * 256 + 256 * 4 <= sizeof(u64) * kList, "the radix histogram lies in the list");

// Calls g(vector index, its 16 bytes) for the whole vectors of elements [off, off
// + n) of data, a 16-byte boundary, and e(element index) for those at the ends. A
// thread gets the same ones every time.
template <typename T, typename G, typename E>
TSB_HD void for_vectors(const T *data, int off, int n, G g, E e) {
  constexpr int VEC = 16 / sizeof(T);
  const int v0 = (off + VEC - 1) / VEC, v1 = max((off + n) / VEC, v0);
#pragma unroll 4
  for (int v = v0 + (int)threadIdx.x; v < v1; v += kThreads) g(v);
  const int head = min(v0 * VEC, off + n) - off, rest = off + n - max(v1 * VEC, off + head);
  if ((int)threadIdx.x < head) e(off + (int)threadIdx.x);
  if ((int)threadIdx.x >= 32 && (int)threadIdx.x - 32 < rest) e(max(v1 * VEC, off + head) + (int)threadIdx.x - 32);
}
// Calls f(token index, logit) for this CTA's logits, the first of which is token lo.
template <typename T, typename F>
TSB_HD void for_logits(const T *data, int off, int lo, int n, F f) {
  constexpr int VEC = 16 / sizeof(T);
  for_vectors<T>(
      data, off, n,
      [&](int v) {
        const uint4 w = *reinterpret_cast<const uint4 *>(data + v * VEC);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(lo + v * VEC + j - off, to_float(e[j]));
      },
      [&](int i) { f(lo + i - off, to_float(data[i])); });
}

TSB_HD u64 block_sum(u64 v, Shared &s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = v;
  __syncthreads();
  u64 all = 0;
  for (int w = 0; w < kWarps; ++w) all += s.red[w];
  return all;
}

// Inclusive scan of a value per thread over the block.
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
  for (int w = 0; w < warp; ++w) before += s.scan[w];
  return before + v;
}

TSB_HD float token_logit(u64 token) { return key_logit((uint32_t)(token >> 32)); }
TSB_HD int token_index(u64 token) { return (int)~(uint32_t)token; }

// Descending bitonic sort of N = 32 or 64 values over a warp, element lane + 32 h in v[h].
template <int N>
TSB_HD void warp_sort(u64 (&v)[N / 32], int lane) {
#pragma unroll
  for (int k = 2; k <= N; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      if (j == 32) {
        const u64 a = v[0], b = v[N / 32 - 1];
        v[0] = max(a, b);
        v[N / 32 - 1] = min(a, b);
      } else {
#pragma unroll
        for (int h = 0; h < N / 32; ++h) {
          const u64 other = __shfl_xor_sync(0xffffffffu, v[h], j);
          const bool down = ((lane + 32 * h) & k) == 0, low = (lane & j) == 0;
          v[h] = down == low ? max(v[h], other) : min(v[h], other);
        }
      }
    }
  }
}
TSB_HD u64 warp_scan(u64 v, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
TSB_HD u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// CTA 0: the first token, along the order, at which `before` plus the running
// count or mass of the listed tokens of `bin` (all of the list for bin < 0, counts
// only) that are at or above `floor_token` reaches bound; into s.found_token and
// s.found_mass (the count or mass through it).
TSB_HD void narrow(Shared &s, int n, int bin, u64 floor_token, bool by_count, u64 bound, u64 before, const RowScale &r) {
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  u64 lo = floor_token, hi = ~0ull;
  auto each = [&](auto f) {
    for (int e = tid; e < n; e += kThreads) {
      const u64 t = s.list[e];
      if (t >= lo && t <= hi && (bin < 0 || logit_bin(token_logit(t), r) == (uint32_t)bin)) f(t);
    }
  };
  for (;;) {
    u64 least = ~0ull, most = 0;
    unsigned int count = 0;
    each([&](u64 t) {
      least = min(least, t);
      most = max(most, t);
      ++count;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      least = min(least, __shfl_xor_sync(0xffffffffu, least, o));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      count += __shfl_xor_sync(0xffffffffu, count, o);
    }
    __syncthreads();
    if (lane == 0) { s.red[warp] = least; s.red2[warp] = most; s.scan[warp] = count; }
    s.sub0[tid] = 0;
    s.sub1[tid] = 0;
    if (tid == 0) { s.found = 0; s.found_mass = before; s.few_n = 0; }
    __syncthreads();
    count = 0;
    for (int w = 0; w < kWarps; ++w) {
      least = min(least, s.red[w]);
      most = max(most, s.red2[w]);
      count += (unsigned int)s.scan[w];
    }
    if (count <= 32) break;
    const int shift = max(0, 64 - __clzll((long long)(most - least)) - 8);
    each([&](u64 t) {
      const unsigned int sub = (unsigned int)((most - t) >> shift);
      if (by_count) {
        atomicAdd(&s.sub0[sub], 1u);
      } else {
        const uint32_t m = logit_m(token_logit(t), (uint32_t)bin, r);
        atomicAdd(&s.sub0[sub], m & 4095u);
        atomicAdd(&s.sub1[sub], m >> 12);
      }
    });
    __syncthreads();
    const u64 own = by_count ? s.sub0[tid] : bin_units((u64)s.sub0[tid] + ((u64)s.sub1[tid] << 12), (uint32_t)bin);
    const u64 here = before + block_scan(own, s);
    if (here >= bound && here - own < bound) {
      s.found = tid;
      s.found_mass = here - own;
    }
    __syncthreads();
    before = s.found_mass;
    hi = most - ((u64)s.found << shift);
    const u64 width = (1ull << shift) - 1;
    lo = max(lo, hi > width ? hi - width : 0ull);
  }
  each([&](u64 t) { s.few[atomicAdd(&s.few_n, 1u)] = t; });
  __syncthreads();
  if (warp == 0) {
    u64 v[1] = {lane < (int)s.few_n ? s.few[lane] : 0ull};
    warp_sort<32>(v, lane);
    const u64 own = v[0] == 0 ? 0 : by_count ? 1 : logit_mass(token_logit(v[0]), r);
    const u64 here = before + warp_scan(own, lane);
    const unsigned int at = __ballot_sync(0xffffffffu, here >= bound && own);
    const int first = at ? __ffs(at) - 1 : 0;
    if (lane == first) {
      s.found_token = v[0];
      s.found_mass = here;
    }
  }
  __syncthreads();
}

// u's bound on the running mass: the first token whose cumulative mass exceeds u * total.
TSB_HD u64 sample_bound(float u, u64 total) {
  const double want = u > 0.f ? (double)u * (double)total : 0.0;
  return want >= (double)total ? total : min((u64)want + 1, total);
}
TSB_HD u64 top_p_bound(double p, u64 total) {
  const u64 b = p > 0.0 ? (u64)ceil(p * (double)total) : 1ull;
  return min(max(b, 1ull), total);
}

TSB_HD void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
TSB_HD void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T>
__global__ void __launch_bounds__(kThreads, 3) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int i = tid; i < kBins; i += kThreads) { s.h0[i] = 0; s.h1[i] = 0; }
  if (tid == 0) { s.list_n = 0; s.first = 0xffffffffu; }
  cluster_arrive();  // waited for before the first access to another CTA's shared memory
  griddep_wait();  // programmatic dependent: the logits are the previous kernel's
  griddep_launch_dependents();

  // ---- this CTA's logits [lo, lo + n), staged or read where they are
  const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
  const int lo = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - lo);
  const T *data = x + lo;
  const int off = (int)((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
  data -= off;
  const float u = a.u[row];
  double temperature = a.temperature ? a.temperature[row] : a.temperature_s;
  const double p = a.top_p ? a.top_p[row] : a.top_p_s;
  const double floor_w = a.min_p ? a.min_p[row] : a.min_p_s;
  int k = a.top_k ? a.top_k[row] : a.top_k_s;
  const bool greedy = !(temperature > 0.0);
  temperature = fmax(temperature, kMinTemperature);

  float top = -INFINITY;  // this thread's largest logit
  {
    constexpr int VEC = 16 / sizeof(T);
    T *stage = reinterpret_cast<T *>(smem + kSharedBytes);
    for_vectors<T>(
        data, off, n,
        [&](int v) {
          const uint4 w = ldg_nc_v4(data + v * VEC);
          if (a.staged) *reinterpret_cast<uint4 *>(stage + v * VEC) = w;
          top = max_of(w, top, T());
        },
        [&](int i) {
          const T w = data[i];
          if (a.staged) stage[i] = w;
          top = fmaxf(top, to_float(w));
        });
    if (a.staged) data = stage;  // a thread reads back what it wrote itself
  }
  Shared *const head = cluster.map_shared_rank(&s, 0);
  auto emit = [&](float v, int token, u64 kept) {
    if (token >= 0) a.token[row] = token;
    if (a.logprob) {
      const double d = v == top ? 0.0 : ((double)v - (double)top) / temperature;
      a.logprob[row] = (float)(d - log((double)kept / (double)kOne));
    }
  };
  const bool use_p = p < 1.0, use_floor = floor_w > 0.0;
  const u64 floor_mass = use_floor ? (u64)fmin(ceil(floor_w * (double)kOne), 2.0 * (double)kOne) : 0;
  const double c64 = 1.4426950408889634 / temperature;
  RowScale r;
  r.c = (float)c64;
  r.c_low = (float)(c64 - (double)r.c);
  r.bin_scale = (float)(c64 * kStep);

  // ---- small top-k: tokens that some k lanes' maxima reach
  if (!greedy && k > 0 && k <= kDirectK && k < a.vocab) {
    float v = top;  // the warp's lanes in descending order
#pragma unroll
    for (int g = 2; g <= 32; g <<= 1) {
#pragma unroll
      for (int j = g >> 1; j > 0; j >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, v, j);
        v = ((lane & g) == 0) == ((lane & j) == 0) ? fmaxf(v, other) : fminf(v, other);
      }
    }
    if (lane == (k - 1) / kWarps) s.red[warp] = __float_as_uint(v);  // ceil(k / warps) lanes of each warp reach it
    __syncthreads();
    float cut = __uint_as_float((uint32_t)s.red[0]);
    for (int w = 1; w < kWarps; ++w) cut = fminf(cut, __uint_as_float((uint32_t)s.red[w]));
    cluster_wait();
    for_logits<T>(data, off, lo, n, [&](int i, float e) {
      if (e >= cut && e > -INFINITY) {
        const unsigned int at = atomicAdd(&head->list_n, 1u);
        if (at < (unsigned int)kList) head->list[at] = (u64)logit_key(e) << 32 | (uint32_t)~i;
      }
    });
    cluster.sync();
    const int m = (int)head->list_n;
    cluster_arrive();  // CTA 0 stays until every CTA has read it
    if (m <= kList) {
      if (rank != 0) {
        cluster_wait();
        return;
      }
      u64 floor_token = 0;
      if (m > kDirectK) {
        narrow(s, m, -1, 0, true, (u64)k, 0, r);
        floor_token = s.found_token;
      }
      if (tid == 0) s.few_n = 0;
      __syncthreads();
      for (int e = tid; e < m; e += kThreads) {
        const u64 t = s.list[e];
        if (t >= floor_token) s.few[atomicAdd(&s.few_n, 1u)] = t;
      }
      __syncthreads();
      if (warp == 0) {
        const int have = (int)s.few_n;
        u64 t[2], own[2], up[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) t[h] = lane + 32 * h < have ? s.few[lane + 32 * h] : 0ull;
        warp_sort<kDirectK>(t, lane);
        const int kept_n = min(have, k);
        top = token_logit(__shfl_sync(0xffffffffu, t[0], 0));
        r.top = top;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e = token_logit(t[h]);
          own[h] = lane + 32 * h >= kept_n ? 0 : e == top ? kOne : top == INFINITY ? 0 : logit_mass(e, r);
        }
        up[0] = warp_scan(own[0], lane);
        const u64 first_half = __shfl_sync(0xffffffffu, up[0], 31);
        up[1] = first_half + warp_scan(own[1], lane);
        u64 kept = __shfl_sync(0xffffffffu, up[1], 31);
        // the place of the first token whose running mass reaches a bound
        auto cross = [&](u64 bound) -> int {
          const unsigned int a0 = __ballot_sync(0xffffffffu, up[0] >= bound && own[0]);
          const unsigned int a1 = __ballot_sync(0xffffffffu, up[1] >= bound && own[1]);
          return a0 ? __ffs(a0) - 1 : a1 ? __ffs(a1) + 31 : 0;
        };
        auto at = [&](const u64 (&w)[2], int i) -> u64 {
          const u64 w0 = __shfl_sync(0xffffffffu, w[0], i & 31), w1 = __shfl_sync(0xffffffffu, w[1], i & 31);
          return i < 32 ? w0 : w1;
        };
        if (kept == 0) {
          if (lane == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
          }
        } else {
          if (use_p) kept = min(kept, at(up, cross(top_p_bound(p, kept))));
          if (use_floor) {
            const u64 above = warp_sum((own[0] >= floor_mass ? own[0] : 0) + (own[1] >= floor_mass ? own[1] : 0));
            kept = min(kept, max(above, kOne));
          }
          const u64 token = at(t, cross(sample_bound(u, kept)));
          if (lane == 0) emit(token_logit(token), token_index(token), kept);
        }
      }
      cluster_wait();
      return;
    }
    cluster_wait();  // too many (equal logits, or hardly any live ones): the general way
    if (tid == 0) s.list_n = 0;
  } else {
    cluster_wait();
  }

  // ---- 1. the largest logit
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.red[warp] = __float_as_uint(top);
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, __uint_as_float((uint32_t)s.red[w]));
  if (tid < ctas) cluster.map_shared_rank(&s, tid)->peer_top[rank] = top;
  cluster.sync();
  for (int c = 0; c < ctas; ++c) top = fmaxf(top, s.peer_top[c]);

  if (top == -INFINITY) {  // every logit is -inf or NaN: there is no token to choose
    if (rank == 0 && tid == 0) {
      a.token[row] = -1;
      if (a.logprob) a.logprob[row] = -INFINITY;
    }
    return;
  }
  if (greedy) {
    unsigned int first = 0xffffffffu;
    for_logits<T>(data, off, lo, n, [&](int i, float v) { if (v == top) first = min(first, (unsigned int)i); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    if (lane == 0 && first != 0xffffffffu) atomicMin(&head->first, first);
    cluster.sync();
    if (rank == 0 && tid == 0) {
      a.token[row] = (int)s.first;
      if (a.logprob) a.logprob[row] = 0.f;
    }
    return;
  }

  r.top = top;
  bool use_k = k > 0 && k < a.vocab;
  const bool counted = use_k;

  auto tell = [&](int mode, int b0, int b1) {  // CTA 0 to all
    if (tid < ctas) {
      Shared *peer = cluster.map_shared_rank(&s, tid);
      peer->mode = mode;
      peer->lo = b0;
      peer->hi = b1;
    }
  };
  // All CTAs: the token number `tie` (CTA 0 knows it) of those with this logit, in index order.
  auto pick = [&](float v, u64 kept, auto tie_of) {
    unsigned int ties = 0;
    for_logits<T>(data, off, lo, n, [&](int, float e) { ties += e == v; });
    ties = (unsigned int)block_sum(ties, s);
    if (tid == 0) head->peer_ties[rank] = ties;
    cluster.sync();
    if (rank == 0 && tid == 0) {
      unsigned int all = 0;
      for (int q = 0; q < ctas; ++q) all += s.peer_ties[q];
      u64 tie = tie_of(all, kept);
      int q = 0;
      while (q < ctas - 1 && tie >= s.peer_ties[q]) tie -= s.peer_ties[q++];
      for (int c = 0; c < ctas; ++c) {
        Shared *peer = cluster.map_shared_rank(&s, c);
        peer->pick_rank = q;
        peer->pick_tie = (int)tie;
      }
      emit(v, -1, kept);
    }
    cluster.sync();
    if (rank != s.pick_rank) return;
    unsigned int seen = 0;  // ties before this block of tokens
    for (int at = 0; at < n; at += kThreads) {
      const bool hit = at + tid < n && to_float(data[off + at + tid]) == v;
      const unsigned int up = (unsigned int)block_scan(hit, s);
      if (hit && seen + up - 1 == (unsigned int)s.pick_tie) a.token[row] = lo + at + tid;
      for (int q = 0; q < kWarps; ++q) seen += (unsigned int)s.scan[q];
      if (seen > (unsigned int)s.pick_tie) return;
    }
  };

  if (top == INFINITY) {  // the +inf logits share all the weight equally
    pick(top, 0, [&](unsigned int all, u64 &kept) {
      kept = (u64)(use_k ? min(all, (unsigned int)k) : all) * kOne;
      if (use_p) kept = (top_p_bound(p, kept) + kOne - 1) / kOne * kOne;
      if (use_floor && floor_mass > kOne) kept = kOne;
      return (sample_bound(u, kept) + kOne - 1) / kOne - 1;
    });
    return;
  }

  // ---- 2. the histogram, added up in CTA 0
  auto push = [&](bool both) {
    __syncthreads();
    if (rank != 0) {
      for (int i = tid; i < kBins; i += kThreads) {
        if (s.h0[i]) atomicAdd(&head->h0[i], s.h0[i]);
        if (both && s.h1[i]) atomicAdd(&head->h1[i], s.h1[i]);
      }
    }
  };
  auto count_tokens = [&]() {
    for_logits<T>(data, off, lo, n, [&](int, float v) {
      const uint32_t bin = logit_bin(v, r);
      if (bin < (uint32_t)kBins) atomicAdd(&s.h0[bin], 1u);
    });
    push(false);
  };
  auto add_masses = [&]() {
    u64 above = 0;  // what min-p keeps
    for_logits<T>(data, off, lo, n, [&](int, float v) {
      const uint32_t bin = logit_bin(v, r);
      if (bin < (uint32_t)kBins) {
        const uint32_t m = logit_m(v, bin, r);
        atomicAdd(&s.h0[bin], m & 4095u);
        atomicAdd(&s.h1[bin], m >> 12);
        if (use_floor) {
          const u64 units = bin_units(m, bin);
          if (units >= floor_mass) above += units;
        }
      }
    });
    if (use_floor) {
      above = block_sum(above, s);
      if (tid == 0) head->peer_floor[rank] = above;
    }
    push(true);
  };
  // CTA 0: running sums of the histogram; returns the whole
  auto run_sums = [&](bool masses) -> u64 {
    u64 v[kBinsPerThread], run = 0;
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      const int bin = tid * kBinsPerThread + i;
      v[i] = bin >= kBins ? 0 : masses ? bin_units((u64)s.h0[bin] + ((u64)s.h1[bin] << 12), bin) : s.h0[bin];
      run += v[i];
    }
    u64 up = block_scan(run, s) - run;
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      const int bin = tid * kBinsPerThread + i;
      up += v[i];
      if (bin < kBins) s.sums[bin] = up;
    }
    __syncthreads();
    return s.sums[kBins - 1];
  };
  // CTA 0: the bin in which the running sum reaches bound
  auto find_bin = [&](u64 bound) -> int {
    if (tid == 0) s.found = kBins - 1;
    __syncthreads();
    for (int bin = tid; bin < kBins; bin += kThreads)
      if (s.sums[bin] >= bound && (bin == 0 || s.sums[bin - 1] < bound)) s.found = bin;
    __syncthreads();
    const int bin = s.found;
    __syncthreads();
    return bin;
  };
  auto before_bin = [&](int bin) -> u64 { return bin ? s.sums[bin - 1] : 0; };
  auto gather = [&](int b0, int b1) {  // all CTAs, into CTA 0's list
    for_logits<T>(data, off, lo, n, [&](int i, float v) {
      const uint32_t bin = logit_bin(v, r);
      if (bin >= (uint32_t)b0 && bin <= (uint32_t)b1) {
        const unsigned int at = atomicAdd(&head->list_n, 1u);
        if (at < (unsigned int)kList) head->list[at] = (u64)logit_key(v) << 32 | (uint32_t)~i;
      }
    });
  };

  if (use_k) count_tokens(); else add_masses();
  cluster.sync();

  // ---- 3. what to gather: CTA 0 decides
  u64 total = 0, above_floor = 0;
  int k_bin = 0;
  u64 k_before = 0, k_in = 0;                // tokens before and in top-k's bin
  if (rank == 0) {
    total = run_sums(!use_k);
    if (use_k) {
      use_k = (u64)k < total;  // else every token with a mass is among the first k
      k_bin = use_k ? find_bin((u64)k) : kBins - 1;
      k_before = before_bin(k_bin);
      k_in = s.sums[k_bin] - k_before;
      tell(k_before + k_in <= kList ? kFew : kSlow, 0, k_bin);
    } else {
      if (use_floor)
        for (int q = 0; q < ctas; ++q) above_floor += s.peer_floor[q];
      int b0 = 0, b1;
      if (use_p) {
        b1 = find_bin(top_p_bound(p, total));
      } else {
        b0 = b1 = find_bin(sample_bound(u, use_floor ? min(total, max(above_floor, kOne)) : total));
        
      }
      u64 tokens = 0;  // a bound on the tokens of the bins
      for (int bin = b0 + tid; bin <= b1; bin += kThreads) {
        const u64 mass = s.sums[bin] - before_bin(bin);
        if (mass) tokens += min(most_tokens(mass, bin), (u64)kMaxVocab);
      }
      tokens = block_sum(tokens, s);
      tell(tokens <= kList ? kFew : kSlow, b0, b1);
    }
  }
  cluster.sync();
  if (s.mode == kFew) {
    gather(s.lo, s.hi);
    cluster.sync();
    if (rank != 0) return;
    const int m = min((int)s.list_n, kList);
    u64 floor_token = 0, kept = total;
    if (counted) {
      // the list holds the first k, or every token with a mass: their masses by bin
      if (use_k) {
        narrow(s, m, k_bin, 0, true, (u64)k, k_before, r);
        floor_token = s.found_token;
      }
      for (int i = tid; i < kBins; i += kThreads) { s.h0[i] = 0; s.h1[i] = 0; }
      __syncthreads();
      for (int e = tid; e < m; e += kThreads) {
        if (s.list[e] < floor_token) continue;
        const float v = token_logit(s.list[e]);
        const uint32_t bin = logit_bin(v, r), w = logit_m(v, bin, r);
        atomicAdd(&s.h0[bin], w & 4095u);
        atomicAdd(&s.h1[bin], w >> 12);
      }
      __syncthreads();
      kept = run_sums(true);
    }
    if (use_p) {
      const u64 bound = top_p_bound(p, kept);
      const int bin = find_bin(bound);
      narrow(s, m, bin, floor_token, false, bound, before_bin(bin), r);
      kept = min(kept, s.found_mass);
    }
    if (use_floor) {
      if (counted || use_p) {  // min-p keeps a prefix of the order: what of it is in the list decides
        u64 above = 0;
        for (int e = tid; e < m; e += kThreads) {
          const u64 w = s.list[e] >= floor_token ? logit_mass(token_logit(s.list[e]), r) : 0;
          above += w >= floor_mass ? w : 0;
        }
        above_floor = block_sum(above, s);
      }
      kept = min(kept, max(above_floor, kOne));
    }
    const u64 bound = sample_bound(u, kept);
    const int bin = find_bin(bound);
    narrow(s, m, bin, floor_token, false, bound, before_bin(bin), r);
    if (tid == 0) emit(token_logit(s.found_token), token_index(s.found_token), kept);
    return;
  }

  // ---- many candidates: one bound after the other, each resolved inside its bin
  if (counted) {  // the masses are still to be added up
    for (int i = tid; i < kBins; i += kThreads) { s.h0[i] = 0; s.h1[i] = 0; }
    cluster.sync();
    add_masses();
    cluster.sync();
    if (rank == 0) {
      total = run_sums(true);
      if (use_floor)
        for (int q = 0; q < ctas; ++q) above_floor += s.peer_floor[q];
    }
  }
  u64 kept = total;  // CTA 0
  for (int stage = 0; stage < 3; ++stage) {  // top-k, top-p, u
    if (stage == 0 ? !counted : stage == 1 && !use_p) continue;
    u64 bound = 0, mass_before = 0, count_before = 0;
    if (rank == 0) {
      if (stage == 2 && use_floor) kept = min(kept, max(above_floor, kOne));
      int bin;
      if (stage == 0) {
        bound = (u64)k;
        bin = k_bin;
        count_before = k_before;
      } else {
        bound = stage == 1 ? top_p_bound(p, kept) : sample_bound(u, kept);
        bin = find_bin(bound);
      }
      mass_before = before_bin(bin);
      const u64 mass = s.sums[bin] - mass_before;
      int mode = (stage == 0 ? k_in : most_tokens(mass, bin)) <= kList ? kOneBin : kRadix;
      if (stage == 0 && !use_k) mode = kNoMass;  // every token with a mass is kept
      if (tid == 0) s.list_n = 0;
      tell(mode, bin, bin);
    }
    cluster.sync();
    const int mode = s.mode, bin = s.lo;
    if (mode == kNoMass) {
      cluster.sync();  // the plan has been read: CTA 0 may write the next one
      continue;
    }
    if (mode == kOneBin) {
      gather(bin, bin);
      cluster.sync();
      if (rank != 0) continue;
      narrow(s, min((int)s.list_n, kList), bin, 0, stage == 0, bound, stage == 0 ? count_before : mass_before, r);
      const u64 token = s.found_token;
      if (stage == 2) {
        if (tid == 0) emit(token_logit(token), token_index(token), kept);
      } else if (stage == 1) {
        kept = min(kept, s.found_mass);
      } else {  // the mass of the first k
        u64 mass = 0;
        for (int e = tid; e < min((int)s.list_n, kList); e += kThreads)
          if (s.list[e] >= token) mass += logit_mass(token_logit(s.list[e]), r);
        kept = mass_before + block_sum(mass, s);
      }
      __syncthreads();
      continue;
    }
    // radix descent over the keys of the bin, eight bits at a time; its histogram
    // of masses and counts takes the place of the list
    u64 *const rmass = s.list;
    unsigned int *const rcount = reinterpret_cast<unsigned int *>(s.list + 256);
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) { rmass[i] = 0; rcount[i] = 0; }
      __syncthreads();
      for_logits<T>(data, off, lo, n, [&](int, float v) {
        if (logit_bin(v, r) != (uint32_t)bin) return;
        const uint32_t key = logit_key(v);
        if (shift < 24 && (key >> (shift + 8)) != prefix) return;
        atomicAdd(&rcount[(key >> shift) & 255u], 1u);
        atomicAdd(&rmass[(key >> shift) & 255u], logit_mass(v, r));
      });
      cluster.sync();
      if (rank == 0) {
        u64 m = 0, c = 0;
        const int digit = 255 - tid;  // descending
        if (tid < 256) {
          for (int q = 0; q < ctas; ++q) {
            const Shared *peer = cluster.map_shared_rank(&s, q);
            m += peer->list[digit];
            c += reinterpret_cast<const unsigned int *>(peer->list + 256)[digit];
          }
        }
        if (tid == 0) s.found = 0;
        const u64 up_m = mass_before + block_scan(m, s);
        const u64 up_c = count_before + block_scan(c, s);
        const u64 here = stage == 0 ? up_c : up_m, own = stage == 0 ? c : m;
        if (tid < 256 && here >= bound && here - own < bound) {
          s.found = tid;
          s.found_mass = up_m - m;
          s.red[0] = up_c - c;
        }
        __syncthreads();
        mass_before = s.found_mass;
        count_before = s.red[0];
        if (tid < ctas) cluster.map_shared_rank(&s, tid)->prefix = prefix << 8 | (uint32_t)(255 - s.found);
      }
      cluster.sync();
      prefix = s.prefix;
    }
    // every token left has the same logit: some of them come before the one wanted
    const float v = key_logit(prefix);
    const u64 w = logit_mass(v, r);
    const u64 tie = stage == 0 ? bound - count_before - 1 : (bound - mass_before + w - 1) / max(w, 1ull) - 1;
    if (stage < 2) {
      kept = min(kept, mass_before + (tie + 1) * w);
      continue;
    }
    pick(v, kept, [&](unsigned int, u64) { return tie; });
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
  a.staged = stage <= kMaxStage;
  const size_t smem = kSharedBytes + (a.staged ? stage : 0);
  if (cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)(kSharedBytes + kMaxStage)) != cudaSuccess)
    return TSB_ECUDA;
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
