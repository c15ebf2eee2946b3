// What follows a verify pass on the device: the walk down each request's draft
// tree along the sampled tokens, and the compaction of the caches along it.
//
// The walk (the reference decodes the accepted path on the host,
// mlx-tree-spec src/mlx_tree_spec/tree_verify.py:499-516 takes it as `nodes`):
//   cur = 0; while some node c > cur has parents[c] == cur and
//   tokens[c] == samples[cur] >= 0: cur = the lowest such c.
// One warp per request holds the whole tree (T <= 64, two nodes per lane); a
// step is two ballots, so the call is a launch plus at most T such steps (2.6 us for 4
// trees of 16 nodes and for 64 of 64; a step of ~40 cycles hardly shows).
#include "sm100.cuh"

namespace tsb {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kAcceptWarps = 4;  // requests per CTA

__global__ void __launch_bounds__(kAcceptWarps * 32)
tree_accept_kernel(const int32_t *__restrict__ tokens, const int32_t *__restrict__ parents,
                   const int32_t *__restrict__ samples, int B, int T, int32_t *__restrict__ path,
                   int32_t *__restrict__ n_keep, int32_t *__restrict__ next) {
  griddep_wait();  // programmatic dependent: the samples are the previous kernel's
  griddep_launch_dependents();
  const int b = blockIdx.x * kAcceptWarps + threadIdx.x / 32, lane = threadIdx.x % 32;
  if (b >= B) return;
  const size_t row = (size_t)b * T;
  int tok[2], par[2], smp[2], out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = lane + 32 * h;
    const bool in = i < T;
    tok[h] = in ? tokens[row + i] : -1;
    par[h] = in ? parents[row + i] : -1;
    smp[h] = in ? samples[row + i] : -1;
    out[h] = -1;
  }
  int cur = 0, n = 0, want = -1;
  for (int step = 0; step < T; ++step) {  // every step moves to a later node: at most T steps
    if (lane == (n & 31)) {
      if (n < 32) out[0] = cur; else out[1] = cur;
    }
    ++n;
    const int s0 = __shfl_sync(0xffffffffu, smp[0], cur & 31), s1 = __shfl_sync(0xffffffffu, smp[1], cur & 31);
    want = cur < 32 ? s0 : s1;
    const bool h0 = want >= 0 && lane > cur && par[0] == cur && tok[0] == want;
    const bool h1 = want >= 0 && lane + 32 > cur && par[1] == cur && tok[1] == want;
    const unsigned m0 = __ballot_sync(0xffffffffu, h0), m1 = __ballot_sync(0xffffffffu, h1);
    if (!(m0 | m1)) break;
    cur = m0 ? __ffs(m0) - 1 : __ffs(m1) + 31;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (lane + 32 * h < T) path[row + lane + 32 * h] = out[h];
  if (lane == 0) {
    n_keep[b] = n;
    next[b] = want;
  }
}

// ---------------------------------------------------------------- compaction
// One warp per (layer, request, KV head, K or V). Rows base + path[i] move to
// base + i, base = lengths[b] - T. The path increases, so path[i] >= i and the
// rows written by one chunk of U rows are never read by a later one; within a
// chunk every load comes before any store. Rows that stay (path[i] == i) are
// not touched. Bound by latency: an accepted path is a few rows of 256-512 B (4.2 us for
// 8 layers of bf16 caches, 4 requests and 4 heads; 6.2 us for 6 layers of MLX 8-bit ones,
// 32 requests). One launch serves up to 48 layers.
constexpr int kMaxPathLayers = 48;

struct PathPlanes {
  void *k, *v, *ks, *kb, *vs, *vb;
};

struct PathArgs {
  PathPlanes layer[kMaxPathLayers];
  const int32_t *lengths, *path, *n_keep;
  int32_t *new_lengths;
  int kv_format, layers, B, T, Hkv, cap;
};

// Copies rows [0, n) of `vec` elements per row along the path, LPR lanes per row.
template <typename V, int VEC, int U>
TSB_HD void move_rows(V *rows, int p0, int p1, int n, int lane) {
  constexpr int RPI = 32 / VEC;  // rows per warp instruction
  const int col = lane % VEC, sub = lane / VEC;
  for (int c = 0; c < n; c += U * RPI) {
    V v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = c + u * RPI + sub;
      const int a = __shfl_sync(0xffffffffu, p0, i & 31), b = __shfl_sync(0xffffffffu, p1, i & 31);
      const int src = i < 32 ? a : b;
      if (i < n && src != i) v[u] = rows[(size_t)src * VEC + col];
    }
    __syncwarp();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = c + u * RPI + sub;
      const int a = __shfl_sync(0xffffffffu, p0, i & 31), b = __shfl_sync(0xffffffffu, p1, i & 31);
      const int src = i < 32 ? a : b;
      if (i < n && src != i) rows[(size_t)i * VEC + col] = v[u];
    }
    __syncwarp();
  }
}

constexpr int kPathWarps = 4;

__global__ void __launch_bounds__(kPathWarps * 32) kv_commit_paths_kernel(const __grid_constant__ PathArgs a) {
  griddep_wait();  // programmatic dependent: lengths and paths are the previous kernels'
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int item = blockIdx.x * kPathWarps + threadIdx.x / 32;
  const int per_layer = a.B * a.Hkv * 2;
  if (item >= a.layers * per_layer) return;
  const int layer = item / per_layer, rem = item % per_layer;
  const int b = rem / (2 * a.Hkv), head = rem % (2 * a.Hkv) / 2;
  const bool isv = rem & 1;
  const int len = a.lengths[b];
  const bool fits = len >= a.T && len <= a.cap;  // else the request is left as it is
  const int32_t *path = a.path + (size_t)b * a.T;
  const int limit = fits ? min(max(a.n_keep[b], 0), a.T) : 0;
  const int p0 = lane < limit ? path[lane] : -1;
  const int p1 = lane + 32 < limit ? path[lane + 32] : -1;
  // the path ends at its first entry that is no tree node or does not increase
  const int before0 = __shfl_up_sync(0xffffffffu, p0, 1), last0 = __shfl_sync(0xffffffffu, p0, 31);
  const int before1 = __shfl_up_sync(0xffffffffu, p1, 1);
  const bool ok0 = p0 >= 0 && p0 < a.T && (lane == 0 || p0 > before0);
  const bool ok1 = p1 >= 0 && p1 < a.T && p1 > (lane == 0 ? last0 : before1);
  const unsigned bad0 = ~__ballot_sync(0xffffffffu, ok0), bad1 = ~__ballot_sync(0xffffffffu, ok1);
  const int n = bad0 ? __ffs(bad0) - 1 : (bad1 ? __ffs(bad1) + 31 : 64);
  if (layer == 0 && head == 0 && !isv && lane == 0 && a.new_lengths) a.new_lengths[b] = fits ? len - a.T + n : len;
  if (n == 0) return;
  const size_t row0 = ((size_t)b * a.Hkv + head) * a.cap + (len - a.T);
  const PathPlanes &pl = a.layer[layer];
  uint4 *data = static_cast<uint4 *>(isv ? pl.v : pl.k);
  if (a.kv_format == TSB_KV_BF16) {
    move_rows<uint4, 32, 4>(data + row0 * 32, p0, p1, n, lane);
    return;
  }
  move_rows<uint4, 16, 2>(data + row0 * 16, p0, p1, n, lane);
  if (a.kv_format == TSB_KV_REF_Q8_ROW) {
    move_rows<float, 1, 2>(static_cast<float *>(isv ? pl.vs : pl.ks) + row0, p0, p1, n, lane);
  } else {
    move_rows<uint2, 1, 2>(static_cast<uint2 *>(isv ? pl.vs : pl.ks) + row0, p0, p1, n, lane);
    move_rows<uint2, 1, 2>(static_cast<uint2 *>(isv ? pl.vb : pl.kb) + row0, p0, p1, n, lane);
  }
}

}  // namespace
}  // namespace tsb

using namespace tsb;

extern "C" int tsb_tree_accept(const int32_t *tokens, const int32_t *parents, const int32_t *samples, int B, int T,
                               int32_t *path, int32_t *n_keep, int32_t *next, tsb_stream_t stream) {
  if (!tokens || !parents || !samples || !path || !n_keep || !next) return TSB_EINVAL;
  if (B <= 0 || T <= 0) return TSB_EINVAL;
  if (T > kMaxNodes) return TSB_EUNSUPPORTED;
  const cudaError_t e = launch_pdl(tree_accept_kernel, dim3((B - 1) / kAcceptWarps + 1), dim3(kAcceptWarps * 32), 0,
                                   (cudaStream_t)stream, tokens, parents, samples, B, T, path, n_keep, next);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}

extern "C" int tsb_kv_commit_paths(int kv_format, int layers, void *const *k, void *const *k_scales,
                                   void *const *k_biases, void *const *v, void *const *v_scales, void *const *v_biases,
                                   int B, int Hkv, int D, int kv_capacity, int T, const int32_t *lengths,
                                   const int32_t *path, const int32_t *n_keep, int32_t *new_lengths,
                                   tsb_stream_t stream) {
  if (!k || !v || !lengths || !path || !n_keep) return TSB_EINVAL;
  if (layers <= 0 || B <= 0 || Hkv <= 0 || kv_capacity <= 0 || T <= 0) return TSB_EINVAL;
  if (new_lengths == lengths || new_lengths == n_keep) return TSB_EINVAL;  // other warps still read them
  if (D != 256 || T > kMaxNodes || layers > kMaxPathLayers) return TSB_EUNSUPPORTED;
  if (kv_format < 0 || kv_format > 2) return TSB_EUNSUPPORTED;
  if ((long long)layers * B * Hkv * 2 > 0x7ffffff0LL) return TSB_EUNSUPPORTED;
  PathArgs a = {};
  for (int l = 0; l < layers; ++l) {
    PathPlanes &p = a.layer[l];
    p = PathPlanes{k[l], v[l], nullptr, nullptr, nullptr, nullptr};
    if (!p.k || !p.v || !aligned(p.k, 16) || !aligned(p.v, 16)) return TSB_EINVAL;
    if (kv_format != TSB_KV_BF16) {
      const size_t al = kv_format == TSB_KV_REF_Q8_ROW ? 4 : 8;
      if (!k_scales || !v_scales) return TSB_EINVAL;
      p.ks = k_scales[l];
      p.vs = v_scales[l];
      if (!p.ks || !p.vs || !aligned(p.ks, al) || !aligned(p.vs, al)) return TSB_EINVAL;
    }
    if (kv_format == TSB_KV_MLX_Q8_G64) {
      if (!k_biases || !v_biases) return TSB_EINVAL;
      p.kb = k_biases[l];
      p.vb = v_biases[l];
      if (!p.kb || !p.vb || !aligned(p.kb, 8) || !aligned(p.vb, 8)) return TSB_EINVAL;
    }
  }
  a.lengths = lengths;
  a.path = path;
  a.n_keep = n_keep;
  a.new_lengths = new_lengths;
  a.kv_format = kv_format;
  a.layers = layers;
  a.B = B;
  a.T = T;
  a.Hkv = Hkv;
  a.cap = kv_capacity;
  const int items = layers * B * Hkv * 2;
  const cudaError_t e = launch_pdl(kv_commit_paths_kernel, dim3((items - 1) / kPathWarps + 1), dim3(kPathWarps * 32), 0,
                                   (cudaStream_t)stream, a);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}
