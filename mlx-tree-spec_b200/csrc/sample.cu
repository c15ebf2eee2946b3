// Sampling one token per row of logits with temperature, top-k, top-p and
// min-p from given random numbers.
//
// Order the tokens by (logit descending, index ascending) and give token i the
// weight w_i = exp((x_i - max) / temperature). Every filter keeps a prefix of
// that order: top-k the first k, top-p the shortest prefix whose mass reaches
// p times the mass of those k, min-p the tokens of weight >= min_p. The sample
// is the first token whose cumulative mass exceeds u times the mass S kept by
// all of them. So a row is never sorted: each step asks where the running count
// or mass along the order crosses a bound.
//
// A cluster of CTAs holds a row's logits in shared memory (one read of HBM).
//   1. The maximum, exchanged through distributed shared memory.
//   2. A histogram over t = (max - x) * log2(e) / temperature in steps of 1/32,
//      fine enough that a bin holds few tokens: counts alone where top-k needs no
//      more, else counts and masses.
//   3. CTA 0 adds the histograms up, finds the bins in which the bounds fall,
//      and the tokens of those bins (or of all bins up to the last one wanted,
//      when they are few) are gathered in its shared memory, sorted and walked.
// A bin with more tokens than the list holds (thousands of logits equal or
// nearly so) is resolved by a radix descent over the logits' bits instead.
//
// Masses are integers, units of 2^-42 of the largest weight: sums do not depend
// on the order of the additions, results repeat bit for bit, and a row's mass
// stays below 2^62. A weight is a float32 exponential of a 64-bit argument: its
// roundings are independent from token to token and do not add up.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace tsb {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kStep = 32;                // bins per halving of the weight
constexpr int kBins = 1408;              // 44 halvings; the last bin takes the rest, which have no mass
constexpr int kBinsPerThread = (kBins + kThreads - 1) / kThreads;
constexpr int kList = 2048;              // tokens CTA 0 can sort
constexpr int kCountOnlyK = 1024;        // top-k up to here needs no masses in the histogram
constexpr u64 kOne = 1ull << 42;         // the mass of the largest weight
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxStage = 160 * 1024;    // bytes of logits a CTA holds in shared memory

constexpr size_t kSliceBytes = 48 * 1024;  // of logits in a CTA, while there are CTAs to split them over
constexpr int kSliceMin = 4096;          // logits of a slice that is not split further

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

// Order-preserving bits: a larger logit has a larger key. -0 counts as +0; NaN
// is below everything.
TSB_HD uint32_t logit_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
TSB_HD float key_logit(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

struct RowScale {
  float top;        // the largest logit
  float bin_scale;  // kStep * log2(e) / temperature
  double c;         // log2(e) / temperature
};

// Bin of a live logit: never decreases as the logit falls.
TSB_HD int logit_bin(float x, const RowScale &r) {
  if (x == r.top) return 0;  // +inf - +inf among them
  return (int)fminf((r.top - x) * r.bin_scale, (float)(kBins - 1));
}

// Mass of a live logit: 2^42 * 2^-t, t = n + 1/2 - g, 2^g by its power series in
// g ln 2 (|g ln 2| <= 0.35: the eighth term is below 2^-27).
TSB_HD u64 logit_mass(float x, const RowScale &r) {
  if (x == r.top) return kOne;
  const double t = ((double)r.top - (double)x) * r.c;
  if (!(t < 43.0)) return 0;  // no mass (and NaN: a finite logit below +inf at an infinite temperature)
  const int n = (int)t;
  const float z = (0.5f - (float)(t - (double)n)) * 0.693147180559945f;
  float p = 1.f / 5040.f;
  p = fmaf(p, z, 1.f / 720.f);
  p = fmaf(p, z, 1.f / 120.f);
  p = fmaf(p, z, 1.f / 24.f);
  p = fmaf(p, z, 1.f / 6.f);
  p = fmaf(p, z, 0.5f);
  p = fmaf(p, z, 1.f);
  p = fmaf(p, z, 1.f);
  p *= 0.70710678118654752f;
  return __float2ull_rn(p * __uint_as_float((uint32_t)(127 + 42 - n) << 23));
}

// How the tokens that a bound falls among are resolved.
enum Mode { kFew, kSlow, kOneBin, kRadix, kNoMass };

struct Shared {
  u64 mass[kBins];        // this CTA's histogram
  u64 sum_mass[kBins];    // CTA 0: running masses of the row up to and including a bin
  u64 list[kList];        // CTA 0: gathered tokens, key << 32 | ~index
  unsigned int count[kBins];
  unsigned int sum_count[kBins];
  u64 peer_best[kMaxCluster];
  u64 peer_floor[kMaxCluster];          // CTA 0
  unsigned int peer_live[kMaxCluster];
  unsigned int peer_ties[kMaxCluster];  // CTA 0
  u64 red[kWarps];
  u64 scan_mass[kWarps];
  unsigned int scan_count[kWarps];
  u64 found_mass;
  int found;
  unsigned int list_n;
  // written by CTA 0 into every CTA
  int mode, lo, hi;
  uint32_t prefix;
  int pick_rank, pick_tie;
};

constexpr size_t kSharedBytes = (sizeof(Shared) + 15) & ~size_t(15);
static_assert(kSharedBytes + kMaxStage <= 227 * 1024, "shared memory");

// Calls f(token index, logit) for this CTA's live logits: elements [off, off + n)
// of data, a 16-byte boundary; the first is token lo.
template <typename T, typename F>
TSB_HD void for_logits(const T *data, int off, int lo, int n, F f) {
  constexpr int VEC = 16 / sizeof(T);
  for (int c = threadIdx.x * VEC; c < off + n; c += kThreads * VEC) {
    if (c >= off && c + VEC <= off + n) {
      const uint4 v = *reinterpret_cast<const uint4 *>(data + c);
      const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float x = to_float(e[j]);
        if (x > -INFINITY) f(lo + c + j - off, x);  // false for NaN too
      }
    } else {  // a vector that sticks out of the slice
      for (int i = max(c, off); i < min(c + VEC, off + n); ++i) {
        const float x = to_float(data[i]);
        if (x > -INFINITY) f(lo + i - off, x);
      }
    }
  }
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

// Inclusive scans of a value per thread over the block.
TSB_HD void block_scan(u64 &m, unsigned int &c, Shared &s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 um = __shfl_up_sync(0xffffffffu, m, o);
    const unsigned int uc = __shfl_up_sync(0xffffffffu, c, o);
    if (lane >= o) { m += um; c += uc; }
  }
  __syncthreads();
  if (lane == 31) { s.scan_mass[warp] = m; s.scan_count[warp] = c; }
  __syncthreads();
  u64 bm = 0;
  unsigned int bc = 0;
  for (int w = 0; w < warp; ++w) { bm += s.scan_mass[w]; bc += s.scan_count[w]; }
  m += bm;
  c += bc;
}

// Descending sort of list[0, n), n <= kList (padded with zeros to a power of two).
TSB_HD void sort_list(Shared &s, int n) {
  int size = 2;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) s.list[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int p = threadIdx.x; p < size / 2; p += kThreads) {
        const int i = 2 * p - (p & (j - 1)), l = i + j;
        const u64 a = s.list[i], b = s.list[l];
        if ((a < b) == ((i & k) == 0)) { s.list[i] = b; s.list[l] = a; }
      }
      __syncthreads();
    }
  }
}

// Running masses of the sorted list, into sum_mass-like storage of its own.
constexpr int kListPerThread = kList / kThreads;
struct ListMasses {
  u64 up_to[kListPerThread];  // inclusive running mass of list element thread * kListPerThread + i
  u64 own[kListPerThread];
};
TSB_HD void list_masses(Shared &s, int n, const RowScale &r, ListMasses &m) {
  u64 run = 0;
#pragma unroll
  for (int i = 0; i < kListPerThread; ++i) {
    const int e = threadIdx.x * kListPerThread + i;
    m.own[i] = e < n ? logit_mass(key_logit((uint32_t)(s.list[e] >> 32)), r) : 0;
    run += m.own[i];
    m.up_to[i] = run;
  }
  u64 all = run;
  unsigned int unused = 0;
  block_scan(all, unused, s);
#pragma unroll
  for (int i = 0; i < kListPerThread; ++i) m.up_to[i] += all - run;
}

// The first list element at which base + running mass reaches bound, into
// s.found / s.found_mass (mass through it); found = -1 if none does.
TSB_HD void list_cross(Shared &s, int n, u64 base, u64 bound, const ListMasses &m) {
  if (threadIdx.x == 0) s.found = -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kListPerThread; ++i) {
    const int e = threadIdx.x * kListPerThread + i;
    if (e < n && m.own[i] && base + m.up_to[i] >= bound && base + m.up_to[i] - m.own[i] < bound) {
      s.found = e;
      s.found_mass = base + m.up_to[i];
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

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared &s = *reinterpret_cast<Shared *>(smem);
  const cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int row = (int)blockIdx.x / ctas;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int i = tid; i < kBins; i += kThreads) { s.count[i] = 0; s.mass[i] = 0; }
  if (tid == 0) s.list_n = 0;
  griddep_wait();  // programmatic dependent: the logits are the previous kernel's
  griddep_launch_dependents();

  // ---- this CTA's logits [lo, lo + n), staged or read where they are
  const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
  const int lo = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - lo);
  const T *data = x + lo;
  const int off = (int)((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
  data -= off;
  const float u = a.u[row];
  const double temperature = a.temperature ? a.temperature[row] : a.temperature_s;
  const double p = a.top_p ? a.top_p[row] : a.top_p_s;
  const double floor_w = a.min_p ? a.min_p[row] : a.min_p_s;
  const int k = a.top_k ? a.top_k[row] : a.top_k_s;
  const bool greedy = !(temperature > 0.0);

  // ---- 1. the largest logit (lowest index first) and the number of live ones
  u64 best = 0;
  unsigned int live = 0;
  if (a.staged) {
    constexpr int VEC = 16 / sizeof(T);
    T *stage = reinterpret_cast<T *>(smem + kSharedBytes);
    for (int c = tid * VEC; c < off + n; c += kThreads * VEC) {
      if (c >= off && c + VEC <= off + n) {
        *reinterpret_cast<uint4 *>(stage + c) = ldg_nc_v4(data + c);
      } else {
        for (int i = max(c, off); i < min(c + VEC, off + n); ++i) stage[i] = data[i];
      }
    }
    data = stage;  // every thread reads back only what it wrote itself
  }
  for_logits<T>(data, off, lo, n, [&](int i, float v) {
    best = max(best, (u64)logit_key(v) << 32 | (uint32_t)~i);
    ++live;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    live += __shfl_xor_sync(0xffffffffu, live, o);
  }
  if (lane == 0) { s.scan_mass[warp] = best; s.scan_count[warp] = live; }
  __syncthreads();
  best = s.scan_mass[0];
  live = s.scan_count[0];
  for (int w = 1; w < kWarps; ++w) { best = max(best, s.scan_mass[w]); live += s.scan_count[w]; }
  if (tid < ctas) {
    Shared *peer = cluster.map_shared_rank(&s, tid);
    peer->peer_best[rank] = best;
    peer->peer_live[rank] = live;
  }
  cluster.sync();
  best = 0;
  live = 0;
  for (int c = 0; c < ctas; ++c) { best = max(best, s.peer_best[c]); live += s.peer_live[c]; }
  if (live == 0 || greedy) {  // nothing to choose, or no choice to make
    if (rank == 0 && tid == 0) {
      a.token[row] = live ? (int)~(uint32_t)best : -1;
      if (a.logprob) a.logprob[row] = live ? 0.f : -INFINITY;
    }
    return;
  }
  RowScale r;
  r.top = key_logit((uint32_t)(best >> 32));
  r.c = 1.4426950408889634 / temperature;
  r.bin_scale = (float)(r.c * kStep);
  const bool use_k = k > 0 && (unsigned int)k < live, use_p = p < 1.0, use_floor = floor_w > 0.0;
  const u64 floor_mass = use_floor ? (u64)fmin(ceil(floor_w * (double)kOne), 2.0 * (double)kOne) : 0;

  // ---- 2. the histogram, and the mass of the weights that min-p keeps
  Shared *const head = cluster.map_shared_rank(&s, 0);
  auto histogram = [&](bool with_mass) {
    u64 above = 0;
    for_logits<T>(data, off, lo, n, [&](int, float v) {
      const int bin = logit_bin(v, r);
      if (with_mass) {
        const u64 m = logit_mass(v, r);
        if (m) atomicAdd(&s.mass[bin], m);
        if (m >= floor_mass) above += m;
      }
      atomicAdd(&s.count[bin], 1u);
    });
    above = block_sum(above, s);
    if (tid == 0) head->peer_floor[rank] = above;
  };
  // CTA 0: adds the cluster's histograms up into running sums
  u64 total = 0, above_floor = 0;
  auto add_up = [&](bool with_mass) {
    u64 m[kBinsPerThread];
    unsigned int c[kBinsPerThread];
    u64 run_m = 0;
    unsigned int run_c = 0;
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      const int bin = tid * kBinsPerThread + i;
      m[i] = 0;
      c[i] = 0;
      if (bin < kBins) {
        for (int q = 0; q < ctas; ++q) {
          const Shared *peer = cluster.map_shared_rank(&s, q);
          c[i] += peer->count[bin];
          if (with_mass) m[i] += peer->mass[bin];
        }
      }
      run_m += m[i];
      run_c += c[i];
    }
    u64 up_m = run_m;
    unsigned int up_c = run_c;
    block_scan(up_m, up_c, s);
    up_m -= run_m;
    up_c -= run_c;
#pragma unroll
    for (int i = 0; i < kBinsPerThread; ++i) {
      const int bin = tid * kBinsPerThread + i;
      up_m += m[i];
      up_c += c[i];
      if (bin < kBins) { s.sum_mass[bin] = up_m; s.sum_count[bin] = up_c; }
    }
    __syncthreads();
    total = s.sum_mass[kBins - 1];
    above_floor = 0;
    for (int q = 0; q < ctas; ++q) above_floor += s.peer_floor[q];
  };
  // CTA 0: the bin in which the running count or mass reaches bound (the last one if none does)
  auto find_bin = [&](bool by_count, u64 bound) -> int {
    if (tid == 0) s.found = kBins - 1;
    __syncthreads();
    for (int bin = tid; bin < kBins; bin += kThreads) {
      const u64 here = by_count ? s.sum_count[bin] : s.sum_mass[bin];
      const u64 before = bin == 0 ? 0 : by_count ? s.sum_count[bin - 1] : s.sum_mass[bin - 1];
      if (here >= bound && before < bound) s.found = bin;
    }
    __syncthreads();
    const int bin = s.found;
    __syncthreads();
    return bin;
  };
  auto tell = [&](int mode, int b0, int b1) {  // CTA 0 to all
    if (tid < ctas) {
      Shared *peer = cluster.map_shared_rank(&s, tid);
      peer->mode = mode;
      peer->lo = b0;
      peer->hi = b1;
    }
  };
  auto gather = [&](int b0, int b1) {  // all CTAs, into CTA 0's list
    for_logits<T>(data, off, lo, n, [&](int i, float v) {
      const int bin = logit_bin(v, r);
      if (bin >= b0 && bin <= b1) head->list[atomicAdd(&head->list_n, 1u)] = (u64)logit_key(v) << 32 | (uint32_t)~i;
    });
  };
  auto emit = [&](uint32_t key, int token, u64 kept) {
    if (token >= 0) a.token[row] = token;
    if (a.logprob) {
      const float v = key_logit(key);
      const double d = v == r.top ? 0.0 : ((double)v - (double)r.top) / temperature;
      a.logprob[row] = (float)(d - log((double)kept / (double)kOne));
    }
  };

  const bool with_mass = !(use_k && k <= kCountOnlyK);
  histogram(with_mass);
  cluster.sync();
  u64 base = 0;  // CTA 0: mass before the gathered bins
  if (rank == 0) {
    add_up(with_mass);
    int b0 = 0, b1;
    if (use_k) {
      b1 = find_bin(true, (u64)k);
    } else if (use_p) {
      b1 = find_bin(false, top_p_bound(p, total));
    } else {
      const u64 kept = use_floor ? min(total, max(above_floor, kOne)) : total;
      b0 = b1 = find_bin(false, sample_bound(u, kept));
      base = b0 ? s.sum_mass[b0 - 1] : 0;
    }
    const unsigned int in = s.sum_count[b1] - (b0 ? s.sum_count[b0 - 1] : 0);
    tell(in <= kList ? kFew : kSlow, b0, b1);
  }
  cluster.sync();
  if (s.mode == kFew) {
    gather(s.lo, s.hi);
    cluster.sync();
    if (rank != 0) return;
    const int m = (int)s.list_n;
    sort_list(s, m);
    ListMasses lm;
    list_masses(s, m, r, lm);
    u64 kept = total;
    if (use_k) {  // mass of the first k: the bins gathered hold them
      if (tid == (k - 1) / kListPerThread) s.found_mass = lm.up_to[(k - 1) % kListPerThread];
      __syncthreads();
      kept = s.found_mass;
      __syncthreads();
    }
    if (use_p) {
      list_cross(s, m, 0, top_p_bound(p, kept), lm);
      kept = min(kept, s.found_mass);
      __syncthreads();
    }
    if (use_floor) {
      u64 above = 0;
      if (use_k || use_p) {  // min-p's tokens are a prefix of the order: those of them in the list decide
#pragma unroll
        for (int i = 0; i < kListPerThread; ++i) above += lm.own[i] >= floor_mass ? lm.own[i] : 0;
        above = block_sum(above, s);
      } else {
        above = above_floor;
      }
      kept = min(kept, max(above, kOne));
    }
    list_cross(s, m, base, sample_bound(u, kept), lm);
    if (tid == 0) {
      const u64 e = s.list[max(s.found, 0)];
      emit((uint32_t)(e >> 32), (int)~(uint32_t)e, kept);
    }
    return;
  }

  // ---- many candidates: one bound after the other, each resolved inside its bin
  if (!with_mass) {
    for (int i = tid; i < kBins; i += kThreads) s.count[i] = 0;
    __syncthreads();
    histogram(true);
    cluster.sync();
    if (rank == 0) add_up(true);
  }
  u64 kept = total;  // CTA 0
  for (int stage = 0; stage < 3; ++stage) {
    if (stage == 0 ? !use_k : stage == 1 && !use_p) continue;
    u64 bound = 0, mass_before = 0, count_before = 0;
    if (rank == 0) {
      if (stage == 2 && use_floor) kept = min(kept, max(above_floor, kOne));
      bound = stage == 0 ? (u64)k : stage == 1 ? top_p_bound(p, kept) : sample_bound(u, kept);
      const int bin = find_bin(stage == 0, bound);
      mass_before = bin ? s.sum_mass[bin - 1] : 0;
      count_before = bin ? s.sum_count[bin - 1] : 0;
      const bool none = s.sum_mass[bin] == mass_before;  // the k-th token has no mass: nor has any after it
      if (tid == 0) s.list_n = 0;
      tell(none ? kNoMass : s.sum_count[bin] - count_before <= kList ? kOneBin : kRadix, bin, bin);
      if (none) kept = mass_before;
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
      const int m = (int)s.list_n;
      sort_list(s, m);
      ListMasses lm;
      list_masses(s, m, r, lm);
      if (stage == 0) {
        const int e = (int)(bound - count_before) - 1;
        if (tid == e / kListPerThread) s.found_mass = mass_before + lm.up_to[e % kListPerThread];
        __syncthreads();
      } else {
        list_cross(s, m, mass_before, bound, lm);
      }
      if (stage == 2) {
        if (tid == 0) {
          const u64 e = s.list[max(s.found, 0)];
          emit((uint32_t)(e >> 32), (int)~(uint32_t)e, kept);
        }
      } else {
        kept = min(kept, s.found_mass);
      }
      __syncthreads();
      continue;
    }
    // radix descent over the keys of the bin, eight bits at a time
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += kThreads) { s.count[i] = 0; s.mass[i] = 0; }
      __syncthreads();
      for_logits<T>(data, off, lo, n, [&](int, float v) {
        const uint32_t key = logit_key(v);
        if (logit_bin(v, r) != bin || (shift < 24 && (key >> (shift + 8)) != prefix)) return;
        atomicAdd(&s.count[(key >> shift) & 255u], 1u);
        atomicAdd(&s.mass[(key >> shift) & 255u], logit_mass(v, r));
      });
      cluster.sync();
      if (rank == 0) {
        u64 m = 0;
        unsigned int c = 0;
        const int digit = 255 - tid;  // descending
        if (tid < 256) {
          for (int q = 0; q < ctas; ++q) {
            const Shared *peer = cluster.map_shared_rank(&s, q);
            m += peer->mass[digit];
            c += peer->count[digit];
          }
        }
        u64 up_m = m;
        unsigned int up_c = c;
        if (tid == 0) s.found = -1;
        block_scan(up_m, up_c, s);
        const u64 here = stage == 0 ? count_before + up_c : mass_before + up_m;
        const u64 before = stage == 0 ? here - c : here - m;
        if (tid < 256 && here >= bound && before < bound) s.found = tid;
        __syncthreads();
        if (tid == s.found) {
          s.red[0] = mass_before + up_m - m;
          s.red[1] = count_before + up_c - c;
        }
        __syncthreads();
        mass_before = s.red[0];
        count_before = s.red[1];
        if (tid < ctas) cluster.map_shared_rank(&s, tid)->prefix = prefix << 8 | (uint32_t)(255 - s.found);
      }
      cluster.sync();
      prefix = s.prefix;
    }
    // every token left has the same key: `tie` of them come before the one wanted
    const u64 w = logit_mass(key_logit(prefix), r);
    u64 tie = 0;
    if (rank == 0) {
      tie = stage == 0 ? bound - count_before - 1 : (bound - mass_before + w - 1) / w - 1;
      if (stage < 2) kept = min(kept, mass_before + (tie + 1) * w);
    }
    if (stage < 2) continue;
    unsigned int ties = 0;
    for_logits<T>(data, off, lo, n, [&](int, float v) { ties += logit_key(v) == prefix; });
    ties = (unsigned int)block_sum(ties, s);
    if (tid == 0) head->peer_ties[rank] = ties;
    cluster.sync();
    if (rank == 0) {
      if (tid == 0) {
        int q = 0;
        while (q < ctas - 1 && tie >= s.peer_ties[q]) tie -= s.peer_ties[q++];
        for (int c = 0; c < ctas; ++c) {
          Shared *peer = cluster.map_shared_rank(&s, c);
          peer->pick_rank = q;
          peer->pick_tie = (int)tie;
        }
        emit(prefix, -1, kept);
      }
    }
    cluster.sync();
    if (rank != s.pick_rank) return;
    // the tie in index order: this CTA's tokens, a block of them at a time
    unsigned int seen = 0;
    for (int at = 0; at < n; at += kThreads) {
      const bool hit = at + tid < n && logit_key(to_float(data[off + at + tid])) == prefix;
      u64 unused = 0;
      unsigned int up = hit;
      block_scan(unused, up, s);
      if (hit && seen + up - 1 == (unsigned int)s.pick_tie) a.token[row] = lo + at + tid;
      __syncthreads();
      for (int q = 0; q < kWarps; ++q) seen += s.scan_count[q];
      if (seen > (unsigned int)s.pick_tie) return;
    }
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
