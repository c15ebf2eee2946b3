// Sampling one token per row of logits with temperature, top-k, top-p and
// min-p from given random numbers.
//
// Order the tokens by (logit descending, index ascending) and give token i the
// weight w_i = exp((x_i - max) / temperature). Every filter keeps a prefix of
// that order: top-k the first k, top-p the shortest prefix whose mass reaches
// p times the mass of those k, min-p the tokens of weight >= min_p. The sample
// is the first token whose cumulative mass exceeds u times the mass S kept by
// all of them. So nothing has to be sorted: each step is one question, "where
// does the running count or mass along the order cross a bound", answered by a
// radix descent over the logits' bits with histograms of counts and masses.
//
// Masses are integers (units of 2^-42 of the largest weight), so sums do not
// depend on the order of the additions and results repeat bit for bit; a
// row's mass stays below 2^62. Weights are rounded to that unit once.
#include <cuda_fp16.h>
#include "sm100.cuh"

namespace tsb {
namespace {

constexpr int kThreads = 1024;
constexpr int kBins = 256;
constexpr double kUnit = 4398046511104.0;  // 2^42: the mass of the largest weight
constexpr int kMaxVocab = 1 << 20;

struct SampleArgs {
  const void *logits;
  const float *u;
  const float *temperature, *top_p, *min_p;  // per row, or NULL and the scalar below
  const int32_t *top_k;
  float temperature_s, top_p_s, min_p_s;
  int top_k_s;
  int rows, vocab;
  long long row_stride;
  int32_t *token;
  float *logprob;
};

TSB_HD float load_logit(const float *p, int i) { return p[i]; }
TSB_HD float load_logit(const __nv_bfloat16 *p, int i) { return __bfloat162float(p[i]); }
TSB_HD float load_logit(const __half *p, int i) { return __half2float(p[i]); }

// Order-preserving bits: a larger logit has a larger key. -0 counts as +0;
// NaN is below everything. Keys up to kKeyMasked (-inf) are never chosen.
constexpr uint32_t kKeyMasked = 0x007FFFFFu;
TSB_HD uint32_t logit_key(float x) {
  if (x != x) return 0u;
  const uint32_t b = __float_as_uint(x + 0.f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
TSB_HD float key_logit(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k); }

struct RowState {
  uint32_t kmax;
  double inv_t;  // 1 / temperature
};

// Weight of a logit in units of 2^-42; the largest logit's is exactly one.
TSB_HD double weight(uint32_t key, const RowState &r) {
  if (key <= kKeyMasked) return 0.0;
  if (key == r.kmax) return 1.0;
  const double w = exp(((double)key_logit(key) - (double)key_logit(r.kmax)) * r.inv_t);
  return w >= 0.0 ? w : 0.0;  // a finite logit below +inf at an infinite temperature: no weight
}
TSB_HD unsigned long long mass_units(double w) { return (unsigned long long)__double2ll_rn(w * kUnit); }

struct Shared {
  unsigned long long mass[kBins];
  unsigned int count[kBins];
  unsigned long long red[32];
  unsigned long long out[3];
  unsigned int pick;
};

TSB_HD unsigned long long block_sum(unsigned long long v, Shared &s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = v;
  __syncthreads();
  v = s.red[threadIdx.x % 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct Cross {
  uint32_t key;                // the crossing token's logit
  int tie;                     // its place among the tokens of that key, from 0
  unsigned long long mass;     // mass up to and including it
};

// The first token of the order at which the running count (by_count) or mass
// reaches `bound` (at least 1, at most the row's total).
template <typename T>
__device__ Cross cross(const T *x, int vocab, const RowState &r, bool by_count, unsigned long long bound, Shared &s) {
  uint32_t prefix = 0;
  unsigned long long mass_above = 0, count_above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) { s.mass[i] = 0; s.count[i] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const uint32_t key = logit_key(load_logit(x, i));
      if (key <= kKeyMasked || (shift < 24 && (key >> (shift + 8)) != prefix)) continue;
      const uint32_t bin = (key >> shift) & (kBins - 1);
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], mass_units(weight(key, r)));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long m = mass_above, c = count_above;
      int bin = kBins - 1;
      for (; bin > 0; --bin) {
        if ((by_count ? c + s.count[bin] : m + s.mass[bin]) >= bound) break;
        m += s.mass[bin];
        c += s.count[bin];
      }
      s.out[0] = m;
      s.out[1] = c;
      s.pick = bin;
    }
    __syncthreads();
    mass_above = s.out[0];
    count_above = s.out[1];
    prefix = shift == 24 ? s.pick : (prefix << 8 | s.pick);
    __syncthreads();
  }
  // every token left has the same key, and so the same weight
  const unsigned long long w = mass_units(weight(prefix, r));
  const unsigned long long tie = by_count ? bound - count_above - 1 : (w ? (bound - mass_above + w - 1) / w - 1 : 0);
  return Cross{prefix, (int)tie, mass_above + (tie + 1) * w};
}

// Index of token number `tie` (from 0, in index order) among those of `key`.
template <typename T>
__device__ int tie_index(const T *x, int vocab, uint32_t key, int tie, Shared &s) {
  int seen = 0;
  for (int base = 0; base < vocab; base += kThreads) {
    const int i = base + threadIdx.x;
    const bool hit = i < vocab && logit_key(load_logit(x, i)) == key;
    const unsigned ballot = __ballot_sync(0xffffffffu, hit);
    __syncthreads();
    if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = __popc(ballot);
    if (threadIdx.x == 0) s.pick = 0xffffffffu;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < (int)threadIdx.x / 32) before += (int)s.red[w];
      all += (int)s.red[w];
    }
    if (hit && seen + before + __popc(ballot & ((1u << (threadIdx.x % 32)) - 1u)) == tie) s.pick = i;
    __syncthreads();
    if (s.pick != 0xffffffffu) return (int)s.pick;
    seen += all;
  }
  return -1;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
  __shared__ Shared s;
  griddep_wait();  // programmatic dependent: the logits are the previous kernel's
  griddep_launch_dependents();
  const int row = blockIdx.x;
  const T *x = static_cast<const T *>(a.logits) + (size_t)row * a.row_stride;
  const float temperature = a.temperature ? a.temperature[row] : a.temperature_s;
  const float p = a.top_p ? a.top_p[row] : a.top_p_s;
  const float floor_w = a.min_p ? a.min_p[row] : a.min_p_s;
  int k = a.top_k ? a.top_k[row] : a.top_k_s;
  if (k <= 0 || k > a.vocab) k = a.vocab;
  const bool greedy = !(temperature > 0.f);
  if (greedy) k = 1;

  unsigned long long best = 0, live = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const uint32_t key = logit_key(load_logit(x, i));
    best = max(best, (unsigned long long)key);
    live += key > kKeyMasked;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (threadIdx.x % 32 == 0) s.red[threadIdx.x / 32] = best;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) best = max(best, s.red[w]);
  live = block_sum(live, s);
  if (live == 0) {  // every logit is -inf or NaN: there is no token to choose
    if (threadIdx.x == 0) {
      a.token[row] = -1;
      if (a.logprob) a.logprob[row] = -INFINITY;
    }
    return;
  }
  RowState r;
  r.kmax = (uint32_t)best;
  r.inv_t = greedy ? 1.0 : 1.0 / (double)temperature;

  unsigned long long total = 0, above_floor = 0;
  for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
    const double w = weight(logit_key(load_logit(x, i)), r);
    total += mass_units(w);
    if (w >= (double)floor_w) above_floor += mass_units(w);
  }
  total = block_sum(total, s);
  above_floor = block_sum(above_floor, s);
  if ((unsigned long long)k < live) total = cross(x, a.vocab, r, true, (unsigned long long)k, s).mass;
  if (p < 1.f) {
    unsigned long long bound = p > 0.f ? (unsigned long long)ceil((double)p * (double)total) : 1ull;
    bound = min(max(bound, 1ull), total);
    total = min(total, cross(x, a.vocab, r, false, bound, s).mass);
  }
  if (floor_w > 0.f) total = min(total, max(above_floor, (unsigned long long)kUnit));

  const float u = a.u[row];
  const double want = u > 0.f ? (double)u * (double)total : 0.0;
  const unsigned long long bound = want >= (double)total ? total : min((unsigned long long)want + 1, total);
  const Cross c = cross(x, a.vocab, r, false, bound, s);
  const int token = tie_index(x, a.vocab, c.key, c.tie, s);
  if (threadIdx.x == 0) {
    a.token[row] = token;
    if (a.logprob) {
      const double d = c.key == r.kmax ? 0.0 : ((double)key_logit(c.key) - (double)key_logit(r.kmax)) * r.inv_t;
      a.logprob[row] = (float)(d - log((double)total / kUnit));
    }
  }
}

template <typename T>
int launch_sample(const SampleArgs &a, cudaStream_t st) {
  const cudaError_t e = launch_pdl(sample_kernel<T>, dim3((unsigned)a.rows), dim3(kThreads), 0, st, a);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_sample(const void *logits, int logits_dtype, int rows, int vocab, long long row_stride,
                          const float *u, const float *temperature, float temperature_all, const int32_t *top_k,
                          int top_k_all, const float *top_p, float top_p_all, const float *min_p, float min_p_all,
                          int32_t *token, float *logprob, tsb_stream_t stream) {
  if (!logits || !u || !token) return TSB_EINVAL;
  if (rows <= 0 || vocab <= 0 || (rows > 1 && row_stride < vocab)) return TSB_EINVAL;
  if (vocab > kMaxVocab) return TSB_EUNSUPPORTED;
  SampleArgs a;
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
  a.rows = rows;
  a.vocab = vocab;
  a.row_stride = row_stride;
  a.token = token;
  a.logprob = logprob;
  switch (logits_dtype) {
    case TSB_MASK_BF16: return aligned(logits, 2) ? launch_sample<__nv_bfloat16>(a, (cudaStream_t)stream) : TSB_EINVAL;
    case TSB_MASK_F16: return aligned(logits, 2) ? launch_sample<__half>(a, (cudaStream_t)stream) : TSB_EINVAL;
    case TSB_MASK_F32: return aligned(logits, 4) ? launch_sample<float>(a, (cudaStream_t)stream) : TSB_EINVAL;
    default: return TSB_EUNSUPPORTED;
  }
}
