// Tree attention for a batch that shares a long prefix. Each node attends to
// the rows of one prefix cache, which every request sees, and to its own
// request's rows: out = softmax(scale q k) v over both, with the tree rule of
// tsb_tree_attn on the last `tail` own rows.
//
// The prefix is computed once for all: a KV head's query rows of the WHOLE
// batch (row = (request, head of the group, node)) are packed into blocks of
// 256, so each block of rows reads the prefix once instead of once per request.
// A unit is (KV head, row block) over the prefix or (request, KV head, row
// block) over that request's own rows; it is cut along the keys into segments.
// A pair of CTAs on two SMs works off a list of segments: prefix segments of
// equal length, laid out so that neighbouring pairs read the same keys at the
// same time (the row blocks of a head share them through L2), then as many chunks
// of own rows as even the pairs out. Own lengths are read on the device, so the
// list is made there too. A segment leaves normalised partials with (max, sum);
// a combine kernel merges those of each row. (One list of tiles per row block, its
// requests' own rows behind the prefix in the same segments, does without the own
// segments' ~10,000 cycles each, but masks other requests' rows in every own tile and
// starts later: 12 x 32 nodes over 32K rows 246 us against 216, after an idle time.)
//
// Measured (24 query and 4 KV heads; calls one after the other, and a replayed graph): 12
// requests x 32 nodes over 32K shared rows + 1K own 251 and 248 us, 1.27 PFLOP/s, 0.92 of
// what a large matrix product sustains at the clock that the power limit leaves (1.43
// GHz); 216 and 213 us in the first milliseconds after an idle time, 1.47 PFLOP/s, 0.89 of such
// a product's burst. 8 x 16 over 8K + 512: 35 and 35 us; 4 x 1 over 1K + 64: 22 (the host's
// time) and 12 us, two dependent launches around a tile or two; 5 x 32 over 32K in 8 bits 158
// and 155 us, after an idle time 136 and 133, 34 of them the conversion.
//
// With many packed rows the work is bound by the tensor cores: 64 keys x 128 rows
// are ~1024 cycles of MMA per SM. One SM by itself cannot feed them: a tile's 64 KB of
// K and V, written to shared memory once and read once at 128 B per cycle, take those
// 1024 cycles too (measured ~1400-1800 per tile that way, with the softmax's P on
// top). So two CTAs share each tile (cta_group::2, M = 256): each loads half of it,
// 32 of the keys and 128 of the value columns, and the MMAs read both halves.
//   warp 0       TMA of this CTA's half of K tiles of 64 keys (int8 rows: their scales, too)
//   warp 1       (CTA 0) S_g = Q K_g^T  (M=256, N=64, K=256; Q in TMEM)
//   warp 2       (CTA 0) O += P_g V_g   (M=256, N=256, K=64; P in shared memory)
//                An MMA with N=64 takes one thread longer to issue than the tensor
//                cores to run, so S and P V have an issuer each.
//   warp 3       TMA of this CTA's half of V tiles
//   warps 4-11   softmax of this CTA's 128 rows, a thread per row (= TMEM lane): warps
//                4-7 have the even tiles, 8-11 the odd ones, so that the exponentials
//                of one tile overlap the loads and stores of the other. The running
//                maximum is a reference that both use; it moves only when a score
//                exceeds it by 2^8. A token passes between the two warps of a row block
//                from tile to tile: its holder looks at the reference and may move it.
// TMEM (512 columns): O [0, 256), Q [256, 384), S0 [384, 448), S1 [448, 512). P_g goes to
// shared memory (two buffers), so S_{g+2} waits only until S_g has been read.
// g counts a pair's tiles over all its segments.
//
// 8-bit caches are converted to bf16 in the workspace first: each row block would
// convert every tile again in here, which held a tile to 2.1 us where bf16 takes 1 (5 x 32
// nodes over 32K rows: 264 us in all against 135, both after an idle time). With a single row block
// (B G T <= 256) no tile would be converted twice; the copy is made there too, and was not
// measured against converting in here.
// MLX: the values. int8 rows: the codes, exact in bf16, with the row scales applied in
// float32 to scores and weights.
//
// Rows at or past a cache's valid rows never reach the output, whatever they hold
// (even NaN): their scores are masked and their V rows are zero in shared memory.
#include <algorithm>
#include <atomic>

#include "attn_tile.cuh"

namespace tsb {

namespace {

constexpr int SH_KT = 64;                    // keys per tile
constexpr int SH_D = 256;
constexpr int SH_ROWS = 256;                 // query rows of a pair, 128 per CTA
constexpr int SH_KBOX = SH_KT / 2 * 128;     // 64-wide D box of 32 keys (bytes)
constexpr int SH_VBOX = SH_KT * 128;         // 64-wide D box of 64 keys
constexpr int SH_K_BYTES = 4 * SH_KBOX;      // a CTA's half of a K tile: 32 keys
constexpr int SH_V_BYTES = 2 * SH_VBOX;      // a CTA's half of a V tile: 128 columns
constexpr int SH_P_BYTES = 128 * 128;        // P of a tile: 128 rows of 64 bf16
constexpr uint32_t SH_O = 0, SH_Q = 256, SH_S0 = 384;
constexpr float SH_RESCALE_LOG2 = 8.f;
constexpr int SH_NK = 5, SH_NV = 5;          // tiles in flight
constexpr int SH_NSC = 8;                    // row-scale ring (tiles)
constexpr int SH_SOFT0 = 4, SH_NSOFT = 8;    // softmax warps
constexpr int SH_MAX_SPLITS = 64;            // key splits of a prefix unit
constexpr int SH_MAX_CHUNKS = 16;            // chunks of a request's own rows
constexpr int SH_MIN_CHUNK = 4;              // tiles
// What a segment costs beside its tiles, in tiles of ~1060 cycles: Q in and partials out
// (~10,000 cycles measured); of own rows the node masks and a cold walk besides.
constexpr int SH_SEG_COST = 10, SH_OWN_SEG_COST = 12;

template <bool SCALED>
struct ShCfg {
  static constexpr int SC_BYTES = SCALED ? SH_NSC * 2 * SH_KT * 4 : 0;
  static constexpr int NBARS = 2 * SH_NK + 2 * SH_NV + 12 + (SCALED ? 2 * SH_NSC : 0);
  static constexpr int CTRL = 6144;  // barriers, TMEM address, schedule, masks of each warp pair, row exchange
  static constexpr int THREADS = 384;
  static constexpr size_t SMEM =
      (size_t)SH_NK * SH_K_BYTES + (size_t)SH_NV * SH_V_BYTES + 2 * SH_P_BYTES + SC_BYTES + CTRL + 1024;
  static_assert((NBARS + 4) * 8 + 4 * 64 * (8 + 4) + 3 * 128 * 4 <= CTRL, "control block");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// One cache of bf16 rows as the kernel reads it (through tensor maps).
struct ShSource {
  const float *ks, *vs;  // row scales (int8 rows), in the cache's own layout
  int sc_cap;            // its rows per (request, head)
  int cap;               // rows per (request, head) of what the tensor maps cover
  int rows;              // valid rows: the prefix's, or the most any request has
};

struct ShArgs {
  ShSource src[2];  // prefix, own
  const uint16_t *q;
  long long q_sb, q_sh, q_st;  // element strides of q [B, Hq, T, D]
  const int32_t *parents;
  const unsigned long long *bits;
  const int32_t *lengths;
  int B, T, Hq, Hkv, tail;
  int rb_p, rb_o;   // row blocks of a KV head's prefix rows / of a request's rows
  int splits, tps;  // prefix: key splits, tiles per split
  int items, more;  // prefix segments: Hkv * splits * rb_p; how many pairs have one more than the others
  int chunk;        // own: tiles per chunk
  int chunks;       // the most chunks a request has
  float scale_log2;
  float *part_o;   // [splits + chunks][B*Hq*T][D]
  float *part_ml;  // [splits + chunks][B*Hq*T][2]
};

TSB_HD int own_rows_of(const int32_t *lengths, int b, int most) {
  return lengths ? min(max(lengths[b], 0), most) : most;
}
TSB_HD int ceil_to(int a, int b) { return (a + b - 1) / b; }

// Deals `total` own chunks of cost c to pairs of which `more` have a prefix segment (cost
// seg) more than the others: either all to those others, or as many as even them out, and
// then the same number to each. `few`: the chunks of the pairs without the extra segment.
struct ShDeal {
  long long few, level;  // level: the longest pair's load beyond the segments that all have
};
__host__ __device__ inline ShDeal deal_chunks(long long total, int pairs, int more, long long seg, long long c) {
  const int less = pairs - more;  // never 0
  const long long k = (total + less - 1) / less, alone = k * c > seg || !more ? k * c : seg;
  if (!more || k * c <= seg) return {total, alone};
  const long long f = seg / c, r = (total - less * f + pairs - 1) / pairs;  // r >= 1
  if (alone <= seg + r * c) return {total, alone};
  const long long few = less * (f + r);
  return {few < total ? few : total, seg + r * c};
}

// A pair's share of the own chunks: `left` chunks from (b, u, ch) on; len = b's rows.
struct ShShare {
  int b, u, ch, left, len;
};

struct ShSegment {
  bool own;
  int b, kh, rb;       // unit
  int j0, nt;          // tiles
  int slot, slots;     // the partial it writes, and further slots it covers (marked empty)
  int n_kv, tail_lo;   // keys, and where the tree rule begins
};

// Walks a pair's segments; every role does so by itself. The share of the own chunks
// is looked at when the prefix segments are done: it is found meanwhile.
struct ShWalk {
  const ShArgs &a;
  const ShShare *share;
  uint64_t *ready;
  int item, step, len;
  bool waiting;
  ShShare w;
  TSB_HD ShWalk(const ShArgs &args, const ShShare *sh, uint64_t *bar, int pair, int pairs)
      : a(args), share(sh), ready(bar), item(pair), step(pairs), len(0), waiting(true), w{0, 0, 0, 0, 0} {}
  TSB_HD bool next(ShSegment &s) {
    if (item < a.items) {
      s.own = false;
      s.rb = item % a.rb_p;
      const int split = item / a.rb_p % a.splits;
      s.kh = item / a.rb_p / a.splits;
      s.b = 0;
      s.n_kv = s.tail_lo = a.src[0].rows;
      s.j0 = split * a.tps;
      s.nt = min(a.tps, ceil_to(s.n_kv, SH_KT) - s.j0);
      s.slot = split;
      s.slots = 1;
      item += step;
      return true;
    }
    if (waiting) {
      waiting = false;
      if (mbar_wait(ready, 0)) w = *share;
      len = w.len;
    }
    while (w.left > 0) {
      const int tiles = ceil_to(len, SH_KT), n = ceil_to(tiles, a.chunk);
      if (w.ch >= n) {  // this unit has no more: on to the next one that has rows
        w.ch = 0;
        if (n == 0 || ++w.u == a.Hkv * a.rb_o) {
          w.u = 0;
          ++w.b;
          len = own_rows_of(a.lengths, w.b, a.src[1].rows);
        }
        continue;
      }
      const int take = min(w.left, n - w.ch);
      s.own = true;
      s.b = w.b;
      s.kh = w.u / a.rb_o;
      s.rb = w.u % a.rb_o;
      s.n_kv = len;
      s.tail_lo = len - a.tail;  // may be negative: fewer own rows than tree rows
      s.j0 = w.ch * a.chunk;
      s.nt = min(take * a.chunk, tiles - s.j0);
      s.slot = a.splits + w.ch;
      s.slots = take;
      w.ch += take;
      w.left -= take;
      return true;
    }
    return false;
  }
};

// ---------------------------------------------------------------- pairs of CTAs
// Address of this CTA's shared-memory object in CTA `rank` of the cluster.
TSB_HD uint32_t cluster_addr(const void *p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
// Arrivals on a barrier of either CTA. What they announce is read by MMAs alone
// (tiles, P and O), behind the writer's own proxy and tcgen05 fences, so the barrier
// need not order ordinary accesses across the cluster: a cluster-scope release per
// arrival cost ~500 cycles, twice a tile.
TSB_HD void cluster_arrive_on(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
TSB_HD void cluster_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
TSB_HD void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Tiled load into this CTA's shared memory that completes on a barrier of either CTA.
TSB_HD void tma_load_2d_pair(void *dst, const void *tmap, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
TSB_HD void pair_tmem_alloc(uint32_t *dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
TSB_HD void pair_tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// D (+)= A B over both CTAs: each has its 128 rows of A and D, and half of B's columns.
TSB_HD void pair_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
TSB_HD void pair_mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on bar in both CTAs once every MMA issued so far by this thread completes.
TSB_HD void pair_commit(uint64_t *bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}

TSB_HD void cp_async4(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
// Arrive on bar when this thread's cp.async copies issued so far have landed
// (counts as one of the barrier's expected arrivals).
TSB_HD void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
TSB_HD void named_barrier_arrive(int id, int count) {
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(count) : "memory");
}

template <bool SCALED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(ShCfg<SCALED>::THREADS, 1)
tree_attn_shared_kernel(const __grid_constant__ CUtensorMap tmap_kp, const __grid_constant__ CUtensorMap tmap_vp,
                        const __grid_constant__ CUtensorMap tmap_ko, const __grid_constant__ CUtensorMap tmap_vo,
                        const __grid_constant__ ShArgs a) {
  using C = ShCfg<SCALED>;
  constexpr int NK = SH_NK, NV = SH_NV;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sK = smem;
  unsigned char *sV = sK + NK * SH_K_BYTES;
  unsigned char *sP = sV + NV * SH_V_BYTES;
  float *sSc = reinterpret_cast<float *>(sP + 2 * SH_P_BYTES);  // [SH_NSC][2][64]: key, then value scales
  uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(sSc) + C::SC_BYTES);
  // in CTA 0, both CTAs arrive: tiles loaded, scores read, P written, Q written, O read
  uint64_t *k_full = bars, *v_full = k_full + NK, *s_free = v_full + NV, *p_full = s_free + 2;
  uint64_t *q_full = p_full + 2, *o_free = q_full + 1;
  // in both CTAs: commits of the MMAs
  uint64_t *k_free = o_free + 1, *v_free = k_free + NK, *s_full = v_free + NV, *pv_done = s_full + 2;
  uint64_t *v_last = pv_done + 2;                       // a CTA's own: a V tile with rows past the end
  uint64_t *share_ready = v_last + 1;
  uint64_t *sc_full = share_ready + 1, *sc_free = sc_full + SH_NSC;  // row scales
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::NBARS);
  ShShare *sShare = reinterpret_cast<ShShare *>(tmem_slot + 1);
  unsigned long long *sBits = reinterpret_cast<unsigned long long *>(bars + C::NBARS + 4);  // [4][T <= 64]
  int32_t *sPar = reinterpret_cast<int32_t *>(sBits + 4 * 64);                                   // [4][T <= 64]
  float *sRow = reinterpret_cast<float *>(sPar + 4 * 64);                                        // [2][128]
  float *sRef = sRow + 2 * 128;                                                                  // [128]

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], 2); mbar_init(&k_free[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], 2); mbar_init(&v_free[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], SH_NSOFT);  // four warps of each CTA have a tile
      mbar_init(&p_full[i], SH_NSOFT);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(q_full, 2 * SH_NSOFT);
    mbar_init(o_free, 2 * SH_NSOFT);
    mbar_init(v_last, 1);
    mbar_init(share_ready, 1);
    if (SCALED)
      for (int i = 0; i < SH_NSC; ++i) { mbar_init(&sc_full[i], 32); mbar_init(&sc_free[i], SH_NSOFT / 2); }
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 0) pair_tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the other CTA's barriers are ready
  tc_fence_after();
  griddep_wait();  // programmatic dependent: q, the caches and the lengths are the previous kernels'
  const uint32_t tmem = *tmem_slot;
  ShWalk walk(a, sShare, share_ready, pair, pairs);
  ShSegment sg = {};
  const int G = a.Hq / a.Hkv, R = G * a.T;

  if (warp == 0) {
    // ---------------- K producer: keys 32 rank .. 32 rank + 31 of each tile, and (int8 rows)
    // the row scales of all its keys and values
    int g = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const CUtensorMap *map = sg.own ? &tmap_ko : &tmap_kp;
      const ShSource &src = a.src[sg.own];
      const int row0 = (sg.b * a.Hkv + sg.kh) * src.cap + sg.j0 * SH_KT + rank * (SH_KT / 2);
      const size_t sc0 = (size_t)(sg.b * a.Hkv + sg.kh) * (size_t)src.sc_cap;
      for (int j = 0; j < sg.nt; ++j, ++g) {
        const int st = g % NK;
        if (g >= NK && !warp_wait(&k_free[st], ((g / NK) - 1) & 1)) { ok = false; break; }
        if (elect_one()) {
          const uint32_t full = cluster_addr(&k_full[st], 0);
          cluster_expect_tx(full, SH_K_BYTES);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            tma_load_2d_pair(sK + st * SH_K_BYTES + d * SH_KBOX, map, d * 64, row0 + j * SH_KT, full);
        }
        __syncwarp();
        if (SCALED) {
          const int sc = g % SH_NSC;
          if (g >= SH_NSC && !warp_wait(&sc_free[sc], ((g / SH_NSC) - 1) & 1)) { ++g; ok = false; break; }
          float *dst = sSc + sc * 2 * SH_KT;
          for (int r = lane; r < SH_KT; r += 32) {
            const int key = (sg.j0 + j) * SH_KT + r;
            if (key < sg.n_kv) {
              cp_async4(dst + r, src.ks + sc0 + key);
              cp_async4(dst + SH_KT + r, src.vs + sc0 + key);
            } else {
              dst[r] = dst[SH_KT + r] = 0.f;
            }
          }
          cp_async_arrive(&sc_full[sc]);
        }
      }
    }
    // Before the CTA may exit: its tiles have been used, and the commits that say so
    // have arrived. After a failure, at least the loads have landed (both CTAs' in CTA 0).
    for (int i = (g > NK ? g - NK : 0); i < g; ++i) ok = ok && warp_wait(&k_free[i % NK], (i / NK) & 1);
    if (!ok && rank == 0)
      for (int i = (g > NK ? g - NK : 0); i < g; ++i) mbar_drain(&k_full[i % NK], (i / NK) & 1);
    if (SCALED) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == 3) {
    // ---------------- V producer: columns 128 rank .. 128 rank + 127 of each tile
    int g = 0, lasts = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const CUtensorMap *map = sg.own ? &tmap_vo : &tmap_vp;
      const int row0 = (sg.b * a.Hkv + sg.kh) * a.src[sg.own].cap + sg.j0 * SH_KT;
      for (int j = 0; j < sg.nt; ++j, ++g) {
        const int st = g % NV;
        if (g >= NV && !warp_wait(&v_free[st], ((g / NV) - 1) & 1)) { ok = false; break; }
        const uint32_t full = cluster_addr(&v_full[st], 0);
        unsigned char *dst = sV + st * SH_V_BYTES;
        const int first = sg.n_kv - (sg.j0 + j) * SH_KT;  // rows past the keys from here on
        if (first >= SH_KT) {
          if (elect_one()) {
            cluster_expect_tx(full, SH_V_BYTES);
#pragma unroll
            for (int d = 0; d < 2; ++d)
              tma_load_2d_pair(dst + d * SH_VBOX, map, rank * 128 + d * 64, row0 + j * SH_KT, full);
          }
        } else {
          // the tile holds whatever follows row n_kv; zero those rows before the MMA
          // reads them (their weights are 0, but 0 * NaN would not be 0)
          if (elect_one()) {
            mbar_arrive_expect_tx(v_last, SH_V_BYTES);
#pragma unroll
            for (int d = 0; d < 2; ++d)
              tma_load_2d(dst + d * SH_VBOX, map, rank * 128 + d * 64, row0 + j * SH_KT, v_last);
          }
          __syncwarp();
          ok = warp_wait(v_last, lasts & 1);
          ++lasts;
          for (int i = lane; i < (SH_KT - first) * 16; i += 32) {
            const int r = first + (i >> 4), c = i & 15;
            *reinterpret_cast<uint4 *>(dst + (c >> 3) * SH_VBOX + r * 128 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) cluster_arrive_on(full);
        }
        __syncwarp();
      }
    }
    for (int i = (g > NV ? g - NV : 0); i < g; ++i) ok = ok && warp_wait(&v_free[i % NV], (i / NV) & 1);
    if (!ok && rank == 0)
      for (int i = (g > NV ? g - NV : 0); i < g; ++i) mbar_drain(&v_full[i % NV], (i / NV) & 1);
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- S = Q K^T
      const uint32_t idesc = idesc_bf16_f32(SH_ROWS, SH_KT);
      int g = 0, seg = 0;
      bool ok = true;
      while (ok && walk.next(sg)) {
        ok = warp_wait(q_full, seg & 1);
        ++seg;
        for (int j = 0; j < sg.nt && ok; ++j, ++g) {
          const int s = g % NK, sb = g & 1;
          ok = warp_wait(&k_full[s], (g / NK) & 1);
          if (ok && g >= 2) ok = warp_wait(&s_free[sb], ((g >> 1) - 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t kb = smem_addr(sK + s * SH_K_BYTES);
#pragma unroll
            for (int kk = 0; kk < 16; ++kk)
              pair_mma_ts(tmem + SH_S0 + sb * 64, tmem + SH_Q + kk * 8,
                          desc_kmajor_sw128(kb + (kk >> 2) * SH_KBOX + (kk & 3) * 32), idesc, kk > 0 ? 1u : 0u);
            pair_commit(&s_full[sb]);
            pair_commit(&k_free[s]);
          }
          __syncwarp();
        }
      }
    }
  } else if (warp == 2) {
    // ---------------- this pair's share of the own chunks. A lane adds up a run of requests.
    {
      const int per = ceil_to(a.B, 32);
      const int b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B);
      const int units = a.Hkv * a.rb_o;
      auto chunks_of = [&](int b) {
        return ceil_to(ceil_to(own_rows_of(a.lengths, b, a.src[1].rows), SH_KT), a.chunk) * units;
      };
      int mine = 0;
      if (a.src[1].rows > 0)
        for (int b = b0; b < b1; ++b) mine += chunks_of(b);
      int up = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
      }
      const int before = up - mine, total = __shfl_sync(0xffffffffu, up, 31);
      const int more = a.more, less = pairs - more;
      const long long few = deal_chunks(total, pairs, more, a.tps + SH_SEG_COST, a.chunk + SH_OWN_SEG_COST).few;
      auto start = [&](int i) -> int {
        return i < more ? (int)((total - few) * i / more) : (int)((total - few) + (less ? few * (i - more) / less : 0));
      };
      const int w0 = start(pair), w1 = start(pair + 1);
      if (lane == 0) *sShare = ShShare{0, 0, 0, 0, 0};
      __syncwarp();
      if (w1 > w0 && w0 >= before && w0 < before + mine) {
        int at = w0 - before, b = b0, n = chunks_of(b);
        while (at >= n) {
          at -= n;
          n = chunks_of(++b);
        }
        n /= units;
        *sShare = ShShare{b, at / n, at % n, w1 - w0, own_rows_of(a.lengths, b, a.src[1].rows)};
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(share_ready);
    }
    if (rank == 0) {
      // ---------------- O += P V
      const uint32_t idesc = idesc_bf16_f32(SH_ROWS, SH_D) | (1u << 16);  // B (V) MN-major
      int g = 0, seg = 0;
      bool ok = true;
      while (ok && walk.next(sg)) {
        if (seg > 0) ok = warp_wait(o_free, (seg - 1) & 1);  // the last segment's O has been read
        ++seg;
        for (int j = 0; j < sg.nt && ok; ++j, ++g) {
          const int s = g % NV, pb = g & 1;
          ok = warp_wait(&v_full[s], (g / NV) & 1);
          if (ok) ok = warp_wait(&p_full[pb], (g >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t vb = smem_addr(sV + s * SH_V_BYTES), pa = smem_addr(sP + pb * SH_P_BYTES);
#pragma unroll
            for (int kk = 0; kk < SH_KT / 16; ++kk)
              pair_mma_ss(tmem + SH_O, desc_kmajor_sw128(pa + kk * 32), desc_mnmajor_sw128(vb + kk * 2048, SH_VBOX),
                          idesc, (j > 0 || kk > 0) ? 1u : 0u);
            pair_commit(&v_free[s]);
            pair_commit(&pv_done[pb]);
          }
          __syncwarp();
        }
      }
    }
  } else {
    // ---------------- softmax / epilogue
    const int odd = (warp - SH_SOFT0) >> 2, q = warp & 3;  // this warp's tiles, and its 32 rows
    const int r = q * 32 + lane;
    const int bar_rows = 1 + q;                                 // both warps of the rows
    const int bar_take = 5 + 4 * odd + q, bar_pass = 5 + 4 * (odd ^ 1) + q;  // the token
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16);
    const float sl2 = a.scale_log2;
    const size_t rows_all = (size_t)a.B * a.Hq * a.T;
    const uint32_t q_full0 = cluster_addr(q_full, 0), o_free0 = cluster_addr(o_free, 0);
    const uint32_t s_free0 = cluster_addr(&s_free[odd], 0), p_full0 = cluster_addr(&p_full[odd], 0);
    int g = 0;
    // A wait that ran out (never in a healthy run) is not followed by others, but the
    // barriers among the warps go on: nobody waits for a warp that has left.
    bool ok = true;
    // the row of a segment that this thread has
    int rq = 0, head = 0, node = 0;
    bool row_valid = false;
    auto place = [&](const ShSegment &s) {
      const int gr = s.rb * SH_ROWS + rank * 128 + r;
      row_valid = gr < (s.own ? R : a.B * R);
      rq = row_valid && !s.own ? gr / R : s.b;
      const int rr = row_valid ? (s.own ? gr : gr % R) : 0;
      head = s.kh * G + rr / a.T;
      node = rr % a.T;
    };
    // A warp's own 32 rows of its P buffer, 4 KB: nobody else touches them, and between
    // segments (after the last P V) no MMA reads them. Rows of 128 bytes pass through it
    // on their way between memory, where eight lanes have 16 bytes each of a row, and
    // TMEM, where a lane has a row: a lane reading its own row alone took ~8000 cycles
    // a segment for Q and as many for O.
    unsigned char *const stage = sP + odd * SH_P_BYTES + q * 4096;
    const int s_row = lane >> 3, s_ch = lane & 7;  // this lane's row (of four at a time) and 16-byte chunk
    auto stage_at = [&](int row, int ch) { return reinterpret_cast<uint4 *>(stage + row * 128 + ((ch ^ (row & 7)) << 4)); };
    // Q row -> TMEM lane r, columns SH_Q + d/2 (the A-operand layout of a K-major
    // M=128 tile), half of D per warp. All S of the segment before are complete.
    int masks_of = -1;  // the request whose node masks are in sBits
    float m_l = -INFINITY, l = 0.f;  // the sum over this warp's tiles, relative to the reference m_l
    bool had = false, had_rows = false;  // the segment before: its partial is still to be written
    int had_slots = 0;
    size_t had_row = 0;
    bool had_valid = false;
    for (;;) {
      const bool more = walk.next(sg);
      float sum = 0.f, m_ref = -INFINITY;
      if (had) {
        // All S of the segment before are complete once P V of its last tile is. A warp
        // follows its own buffer's barriers phase by phase; the other buffer's are looked
        // at only when the phase before is known to be over.
        const int last = g - 1;
        if (last >= 1) ok = ok && warp_wait(&pv_done[(last - 1) & 1], ((last - 1) >> 1) & 1);
        ok = ok && warp_wait(&pv_done[last & 1], (last >> 1) & 1);
        tc_fence_after();
        named_barrier_sync(bar_rows, 64);  // the last tile has settled the reference
        m_ref = sRef[r];
        sRow[odd * 128 + r] = l * (m_l == -INFINITY ? 0.f : ex2(m_l - m_ref));
        named_barrier_sync(bar_rows, 64);
        sum = sRow[r] + sRow[128 + r];
        named_barrier_sync(bar_rows, 64);
      }
      // ---- the next segment's Q: its S can start
      bool any_row = false;
      if (more) {
        place(sg);
        any_row = __any_sync(0xffffffffu, row_valid);
        if (any_row) {  // else whatever Q is in TMEM: nobody reads what comes of it
          const long long off = row_valid ? rq * a.q_sb + head * a.q_sh + node * a.q_st + odd * 128 : -1ll;
          uint4 qv[2][8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const long long o = __shfl_sync(0xffffffffu, off, i * 4 + s_row);
#pragma unroll
            for (int bx = 0; bx < 2; ++bx)
              qv[bx][i] = o >= 0 ? __ldg(reinterpret_cast<const uint4 *>(a.q + o + bx * 64) + s_ch) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int bx = 0; bx < 2; ++bx) {
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) *stage_at(i * 4 + s_row, s_ch) = qv[bx][i];
            __syncwarp();
            uint32_t w[32];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const uint4 u = *stage_at(lane, c);
              w[4 * c] = u.x; w[4 * c + 1] = u.y; w[4 * c + 2] = u.z; w[4 * c + 3] = u.w;
            }
            tmem_st32(lane_base + SH_Q + odd * 64 + bx * 32, w);
          }
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cluster_arrive_on(q_full0);
      }
      // ---- the partial of the segment before, normalised
      if (had) {
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        const long long off = had_valid ? (long long)(had_row * SH_D + odd * 128) : -1ll;
#pragma unroll 1
        for (int c = 0; c < SH_D / 2 && had_rows; c += 32) {
          uint32_t o[32];
          tmem_ld32(lane_base + SH_O + odd * 128 + c, o);
          tmem_wait_ld();
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float4 f = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                                   __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
            *reinterpret_cast<float4 *>(stage_at(lane, e)) = f;
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const long long at = __shfl_sync(0xffffffffu, off, i * 4 + s_row);
            const uint4 u = *stage_at(i * 4 + s_row, s_ch);
            if (at >= 0) *(reinterpret_cast<uint4 *>(a.part_o + at + c) + s_ch) = u;
          }
        }
        tc_fence_before();
        __syncwarp();  // the stage is P's again
        if (lane == 0) cluster_arrive_on(o_free0);
        if (had_valid && odd == 0) {
          float2 *ml = reinterpret_cast<float2 *>(a.part_ml);
          ml[had_row] = make_float2(m_ref, sum);  // sum 0: nothing visible, the partial counts for nothing
          for (int s = 1; s < had_slots; ++s) ml[had_row + s * rows_all] = make_float2(-INFINITY, 0.f);
        }
      }
      if (!more) break;
      had = true;
      had_rows = any_row;
      had_valid = row_valid;
      had_slots = sg.slots;
      had_row = (size_t)sg.slot * rows_all + ((size_t)rq * a.Hq + head) * a.T + node;
      if (sg.own && masks_of != sg.b) {  // node masks, from the parent array or given; the rows' two warps have their own
        masks_of = sg.b;
        const int st = odd * 32 + lane;
        named_barrier_sync(bar_rows, 64);  // the last request's have been read
        if (st < a.T) sPar[q * 64 + st] = a.parents ? a.parents[(size_t)sg.b * a.T + st] : 0;
        named_barrier_sync(bar_rows, 64);
        if (st < a.T) {
          unsigned long long mk = 0;
          if (a.parents) {
            int j = st;
            bool okp = true;
            for (int steps = 0; steps <= a.T && j != -1; ++steps) {
              mk |= 1ull << j;
              const int pj = sPar[q * 64 + j];
              if (!(pj == -1 || (pj >= 0 && pj < j))) { okp = false; break; }
              j = pj;
            }
            if (!okp) mk = 0;
          } else {
            mk = a.bits[(size_t)sg.b * a.T + st];
          }
          sBits[q * 64 + st] = mk;
        }
        named_barrier_sync(bar_rows, 64);
      }
      const unsigned long long mybits = sg.own ? sBits[q * 64 + node] : 0ull;
      m_l = -INFINITY;
      l = 0.f;
      const int g0 = g, g1 = g + sg.nt;
      for (g = g0 + ((g0 & 1) ^ odd); g < g1; g += 2) {
        const int j = g - g0;
        ok = ok && warp_wait(&s_full[odd], (g >> 1) & 1);
        tc_fence_after();
        uint32_t sr[64];
        {
          uint32_t (&lo)[32] = *reinterpret_cast<uint32_t (*)[32]>(&sr[0]);
          uint32_t (&hi)[32] = *reinterpret_cast<uint32_t (*)[32]>(&sr[32]);
          tmem_ld32(lane_base + SH_S0 + odd * 64, lo);
          tmem_ld32(lane_base + SH_S0 + odd * 64 + 32, hi);
        }
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) cluster_arrive_on(s_free0);
        const float *ksc = sSc + (g % SH_NSC) * 2 * SH_KT;  // key, then value scales
        if (SCALED) {
          ok = ok && warp_wait(&sc_full[g % SH_NSC], (g / SH_NSC) & 1);
#pragma unroll
          for (int e = 0; e < 64; e += 4) {
            const float4 k4 = *reinterpret_cast<const float4 *>(ksc + e);
            sr[e] = __float_as_uint(__uint_as_float(sr[e]) * k4.x);
            sr[e + 1] = __float_as_uint(__uint_as_float(sr[e + 1]) * k4.y);
            sr[e + 2] = __float_as_uint(__uint_as_float(sr[e + 2]) * k4.z);
            sr[e + 3] = __float_as_uint(__uint_as_float(sr[e + 3]) * k4.w);
          }
        }
        // mask (only the tail and the last tile need it), then the maximum of the raw
        // scores in eight independent chains; the scale is applied in the exp
        const int key0 = (sg.j0 + j) * SH_KT;
        if ((key0 + SH_KT > sg.tail_lo) || (key0 + SH_KT > sg.n_kv)) {
          const int before = sg.tail_lo - key0, keys = sg.n_kv - key0;  // keys of the tile before the tree, and in all
          unsigned long long vis = before >= 64   ? ~0ull
                                   : before > 0   ? (mybits << before) | ((1ull << before) - 1)
                                   : before > -64 ? mybits >> -before
                                                  : 0ull;
          if (keys < 64) vis &= (1ull << keys) - 1;  // at least one key
          const uint32_t v2[2] = {(uint32_t)vis, (uint32_t)(vis >> 32)};
#pragma unroll
          for (int e = 0; e < 64; ++e)
            if (!(v2[e >> 5] >> (e & 31) & 1u)) sr[e] = __float_as_uint(-INFINITY);
        }
        float mx[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) mx[c] = __uint_as_float(sr[c]);
#pragma unroll
        for (int e = 8; e < 64; ++e) mx[e & 7] = fmaxf(mx[e & 7], __uint_as_float(sr[e]));
        const float tmax = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                 fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * sl2;  // scale > 0
        // the token: tile g - 1 has settled the reference
        if (j > 0) named_barrier_sync(bar_take, 64);
        const float m_old = j > 0 ? sRef[r] : -INFINITY;
        const bool grow = tmax > m_old + SH_RESCALE_LOG2;
        const float m = grow ? tmax : m_old;
        const bool moves = __any_sync(0xffffffffu, grow);
        if (moves || j == 0) sRef[r] = m;
        if (j + 1 < sg.nt) named_barrier_arrive(bar_pass, 64);
        if (g >= 2) ok = ok && warp_wait(&pv_done[odd], ((g >> 1) - 1) & 1);  // P_{g-2} has been read
        if (moves && j > 0) {
          // O holds earlier tiles: wait for P V_{g-1} (and all before), then scale O in place
          ok = ok && warp_wait(&pv_done[odd ^ 1], ((g - 1) >> 1) & 1);
          tc_fence_after();
          const float alpha = (m_old == -INFINITY) ? 0.f : ex2(m_old - m);
#pragma unroll 1
          for (int c = 0; c < SH_D; c += 32) {
            uint32_t o[32];
            tmem_ld32(lane_base + SH_O + c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(lane_base + SH_O + c, o);
          }
          tmem_wait_st();
        }
        if (m != m_l) {  // the reference has moved since this warp's last tile
          l *= m_l == -INFINITY ? 0.f : ex2(m_l - m);
          m_l = m;
        }
        const float nbase = (m == -INFINITY) ? 0.f : -m;
        // P_g: row r of a K-major, 128-byte-swizzled tile
        unsigned char *prow = sP + odd * SH_P_BYTES + r * 128;
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          uint32_t pk[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 8 * c + 2 * e;
            const float p0 = ex2(__fmaf_rn(__uint_as_float(sr[i]), sl2, nbase));
            const float p1 = ex2(__fmaf_rn(__uint_as_float(sr[i + 1]), sl2, nbase));
            ps[e] += p0 + p1;
            if (SCALED) {
              // the value rows' scales weight P; the running sum keeps the plain weights
              const float2 v2 = *reinterpret_cast<const float2 *>(ksc + SH_KT + i);
              pk[e] = pack_bf16x2(p0 * v2.x, p1 * v2.y);
            } else {
              pk[e] = pack_bf16x2(p0, p1);
            }
          }
          *reinterpret_cast<uint4 *>(prow + ((c ^ (r & 7)) << 4)) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
        }
        l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        fence_proxy_async_smem();
        tc_fence_before();  // a rescaled O, too
        __syncwarp();
        if (lane == 0) {
          cluster_arrive_on(p_full0);
          if (SCALED) mbar_arrive(&sc_free[g % SH_NSC]);
        }
      }
      g = g1;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the other CTA has no use for this one's shared memory any more
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    pair_tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- 8-bit caches
// The valid rows of an 8-bit cache as bf16 rows [heads][rows][D]: MLX values
// bf16(fmaf(code, s, b)), or the int8 codes themselves. 16 lanes have a row (272 or 256
// bytes read and 512 written): 4 x 32K rows of K and V, 205 MB, in 34.3 us. Of the bytes
// written 59 MB stay in L2, and what goes through DRAM, 148 MB, is 54% of its rate: memory is
// not shown to be the limit. All loads stand before the first use, a lane's 32 bytes go
// out in one store (64-row blocks, 16-byte stores and late scale loads: 43.5 us).
constexpr int SH_CV_ROWS = 32;  // rows of a CTA

struct ShConvert {
  struct Cache {
    const unsigned char *src[2];      // K, V codes
    const uint2 *scale[2], *bias[2];  // MLX: four bf16 per row
    uint16_t *dst[2];
    int cap, rows;          // rows of a head in the source, and (at most) in the copy
    int blocks;
  } cache[2];               // prefix, own
  const int32_t *lengths;   // own rows of each request, or NULL
  int hkv;
};

template <bool MLX>
__global__ void __launch_bounds__(256) tree_attn_shared_convert_kernel(const __grid_constant__ ShConvert a) {
  griddep_wait();  // programmatic dependent: the caches are the previous kernels'
  griddep_launch_dependents();
  // blocks of the prefix, then of the own rows: (head, K or V, run of rows)
  const int own = (int)blockIdx.x >= a.cache[0].blocks;
  const ShConvert::Cache &c = a.cache[own];
  const int block = blockIdx.x - (own ? a.cache[0].blocks : 0), runs = ceil_to(c.rows, SH_CV_ROWS);
  const int head = block / (2 * runs), v = block / runs & 1;
  const int n = own ? own_rows_of(a.lengths, head / a.hkv, c.rows) : c.rows;
  const int row0 = block % runs * SH_CV_ROWS;
  if (row0 >= n) return;
  const int c16 = threadIdx.x & 15;
  uint4 w[SH_CV_ROWS / 16];
  uint16_t sc[SH_CV_ROWS / 16], bi[SH_CV_ROWS / 16];
#pragma unroll
  for (int i = 0; i < SH_CV_ROWS / 16; ++i) {  // all loads before the first use
    const int row = row0 + i * 16 + (threadIdx.x >> 4);
    const size_t at = (size_t)head * c.cap + min(row, n - 1);
    w[i] = ldg_nc_v4(c.src[v] + at * SH_D + c16 * 16);
    if (MLX) {
      sc[i] = __ldg(reinterpret_cast<const uint16_t *>(c.scale[v] + at) + (c16 >> 2));
      bi[i] = __ldg(reinterpret_cast<const uint16_t *>(c.bias[v] + at) + (c16 >> 2));
    }
  }
#pragma unroll
  for (int i = 0; i < SH_CV_ROWS / 16; ++i) {
    const int row = row0 + i * 16 + (threadIdx.x >> 4);
    if (row >= n) break;
    uint4 lo, hi;
    if (MLX) {
      const float s = bf16_bits_to_float(sc[i]), b = bf16_bits_to_float(bi[i]);
      lo = dequant8_mlx(make_uint2(w[i].x, w[i].y), s, b);
      hi = dequant8_mlx(make_uint2(w[i].z, w[i].w), s, b);
    } else {
      lo = convert8_s8(make_uint2(w[i].x, w[i].y));
      hi = convert8_s8(make_uint2(w[i].z, w[i].w));
    }
    uint16_t *dst = c.dst[v] + ((size_t)head * c.rows + row) * SH_D + c16 * 16;
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst), "r"(lo.x), "r"(lo.y), "r"(lo.z),
                 "r"(lo.w), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w)
                 : "memory");
  }
}

template <bool MLX>
int launch_convert(const ShConvert &a, cudaStream_t st) {
  const int blocks = a.cache[0].blocks + a.cache[1].blocks;
  if (blocks == 0) return TSB_OK;
  const cudaError_t e = launch_pdl(tree_attn_shared_convert_kernel<MLX>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}

// ---------------------------------------------------------------- combine
// out = sum_s w_s o_s, w_s = l_s 2^(m_s - m) / sum, over the prefix's splits and the
// chunks that the request's length has. Partials with l = 0 count for nothing. A warp
// per row, eight of the 256 columns per lane. Bound by latency: a round trip to L2 for
// the weights, with the first partials' loads beside it, and one for every four more
// partials (3.5 us for 96 rows, 4.5 us for 24 heads of 8 x 16 nodes, 5 partials each).
constexpr int SH_CB_WARPS = 4;

__global__ void __launch_bounds__(SH_CB_WARPS * 32)
tree_attn_shared_combine_kernel(const float *__restrict__ part_o, const float *__restrict__ part_ml, int splits,
                                const int32_t *__restrict__ lengths, int own_rows, int chunk_rows, int rows_per_b,
                                int rows, uint16_t *__restrict__ out, float *__restrict__ lse, float *__restrict__ sums) {
  griddep_wait();  // programmatic dependent: the partials are the attention kernel's
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int row = blockIdx.x * SH_CB_WARPS + threadIdx.x / 32;
  if (row >= rows) return;
  const int slots = splits + ceil_to(own_rows_of(lengths, row / rows_per_b, own_rows), chunk_rows);
  const float2 *ml = reinterpret_cast<const float2 *>(part_ml) + row;
  float m = -INFINITY, den = 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < slots; s0 += 32) {
    const int n = min(32, slots - s0);
    const float2 v = lane < n ? ml[(size_t)(s0 + lane) * rows] : make_float2(-INFINITY, 0.f);
    float4 x[4], y[4];  // four partials' loads in flight
    auto fetch = [&](int s) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 *src = reinterpret_cast<const float4 *>(part_o + ((size_t)(s0 + min(s + i, n - 1)) * rows + row) * SH_D) + lane;
        x[i] = __ldg(src);
        y[i] = __ldg(src + 32);
      }
    };
    fetch(0);  // beside the weights, which may turn out to be 0
    float top = v.y != 0.f ? v.x : -INFINITY;  // a sum of NaN stays one
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(top, m);
    const float w = v.y != 0.f ? v.y * exp2f(v.x - top) : 0.f;
    const float before = m == -INFINITY ? 0.f : exp2f(m - top);
    m = top;
    float part = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    den = fmaf(den, before, part);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] *= before;
    for (int s = 0; s < n; s += 4) {
      if (s > 0) fetch(s);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ws = __shfl_sync(0xffffffffu, w, (s + i) & 31);
        if (s + i >= n || ws == 0.f) continue;  // a partial of no weight may hold anything
        acc[0] = fmaf(ws, x[i].x, acc[0]); acc[1] = fmaf(ws, x[i].y, acc[1]);
        acc[2] = fmaf(ws, x[i].z, acc[2]); acc[3] = fmaf(ws, x[i].w, acc[3]);
        acc[4] = fmaf(ws, y[i].x, acc[4]); acc[5] = fmaf(ws, y[i].y, acc[5]);
        acc[6] = fmaf(ws, y[i].z, acc[6]); acc[7] = fmaf(ws, y[i].w, acc[7]);
      }
    }
  }
  const float inv = den != 0.f ? 1.f / den : 0.f;
  uint2 *dst = reinterpret_cast<uint2 *>(out + (size_t)row * SH_D) + lane;
  dst[0] = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  dst[32] = make_uint2(pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  if (sums && lane == 0) sums[row] = 1.f;
  if (lse && lane == 0) lse[row] = den != 0.f ? (m + log2f(den)) * 0.69314718055994531f : -INFINITY;
}

// ---------------------------------------------------------------- plan
struct ShPlan {
  int rb_p, rb_o, splits, tps, items, chunk, chunks, pairs;
};

ShPlan plan_shared(int B, int T, int Hq, int Hkv, int P, int own_rows) {
  ShPlan p = {};
  const int pairs = std::max(1, sm_count() / 2), R = (Hq / Hkv) * T;
  p.rb_p = (int)(((long long)B * R + SH_ROWS - 1) / SH_ROWS);
  p.rb_o = (R + SH_ROWS - 1) / SH_ROWS;
  // The number of key splits of the prefix and the chunks of the own rows with the
  // shortest longest pair, were all requests as long as the longest. A prefix in one
  // round that leaves pairs to the own rows beats one that fills all pairs evenly
  // (8 x 16 nodes over 8K + 512 rows: 37 us with 48 segments of 32 tiles on 74 pairs,
  // 41 with 72 of 22 and the own rows behind them).
  const int tiles = (P + SH_KT - 1) / SH_KT, own_tiles = (own_rows + SH_KT - 1) / SH_KT;
  const long long units = tiles > 0 ? (long long)Hkv * p.rb_p : 0;
  const long long own_units = own_tiles > 0 ? (long long)B * Hkv * p.rb_o : 0;
  p.chunk = std::max(1, own_tiles);
  int s_most = std::min(SH_MAX_SPLITS, std::max(1, tiles / 2));
  if (units > 0) s_most = (int)std::min<long long>(s_most, 1 + 4LL * pairs / units);  // at most four rounds
  long long best = -1;
  for (int s = 1; s <= s_most; ++s) {
    const int tps = (tiles + s - 1) / s, n = tps ? (tiles + tps - 1) / tps : 0;
    const long long rounds = units * n / pairs, seg = tps + SH_SEG_COST;
    const int more = (int)(units * n % pairs);
    for (int ch = 1; ch <= SH_MAX_CHUNKS && (ch == 1 || own_tiles >= ch * SH_MIN_CHUNK); ch *= 2) {
      const int chunk = std::max(1, (own_tiles + ch - 1) / ch), chunks = (own_tiles + chunk - 1) / chunk;
      const long long cost = rounds * seg + deal_chunks(own_units * chunks, pairs, more, seg, chunk + SH_OWN_SEG_COST).level;
      if (best < 0 || cost < best) {
        best = cost;
        p.splits = n;
        p.tps = tps;
        p.chunk = chunk;
        p.chunks = chunks;
      }
    }
  }
  p.items = (int)std::min(units * p.splits, 0x7fffffffLL);
  p.pairs = (int)std::min<long long>(pairs, (long long)p.items + own_units * p.chunks);
  return p;
}

bool sizes_ok(int B, int T, int Hq, int Hkv, int P, int own_rows) {
  return B > 0 && T > 0 && Hq > 0 && Hkv > 0 && P >= 0 && own_rows >= 0 && (long long)B * Hq * T <= (1 << 22);
}

// Bytes of the workspace's parts: partials, then (8-bit formats) the bf16 copies.
size_t partial_bytes(const ShPlan &p, int B, int T, int Hq) {
  const size_t n = (size_t)(p.splits + p.chunks) * B * Hq * T * (SH_D + 2) * sizeof(float);
  return (n + 255) & ~size_t(255);
}
size_t copy_bytes(int B, int Hkv, int P, int own_rows) {  // of K or of V
  return ((size_t)Hkv * P + (size_t)B * Hkv * own_rows) * SH_D * 2;
}

template <bool SCALED>
int launch_attn(const CUtensorMap *maps, const ShArgs &a, int pairs, cudaStream_t st) {
  using C = ShCfg<SCALED>;
  static std::atomic<unsigned long long> ready{0};  // devices on which the attribute is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return TSB_ECUDA;
  const unsigned long long bit = 1ull << (dev & 63);
  if (dev > 63 || !(ready.load(std::memory_order_relaxed) & bit)) {
    if (cudaFuncSetAttribute(tree_attn_shared_kernel<SCALED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)C::SMEM) != cudaSuccess)
      return TSB_ECUDA;
    ready.fetch_or(bit, std::memory_order_relaxed);
  }
  const cudaError_t e = launch_pdl(tree_attn_shared_kernel<SCALED>, dim3((unsigned)pairs * 2), dim3(C::THREADS),
                                   (size_t)C::SMEM, st, maps[0], maps[1], maps[2], maps[3], a);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}

// Checks one cache's planes; `used` false: the cache has no rows and is not read.
int check_source(int fmt, const tsb_kv_t *c, bool used) {
  if (!used) return TSB_OK;
  if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return TSB_EINVAL;
  if (fmt == TSB_KV_BF16) return TSB_OK;
  const size_t al = fmt == TSB_KV_MLX_Q8_G64 ? 8 : 4;
  if (!c->k_scales || !c->v_scales || !aligned(c->k_scales, al) || !aligned(c->v_scales, al)) return TSB_EINVAL;
  if (fmt == TSB_KV_MLX_Q8_G64 &&
      (!c->k_biases || !c->v_biases || !aligned(c->k_biases, al) || !aligned(c->v_biases, al)))
    return TSB_EINVAL;
  return TSB_OK;
}

}  // namespace

unsigned int status_attn_shared(bool reset) {
  unsigned int v = 0;
  cudaMemcpyFromSymbol(&v, g_device_status, sizeof(v));
  if (reset && v) {
    const unsigned int z = 0;
    cudaMemcpyToSymbol(g_device_status, &z, sizeof(z));
  }
  return v;
}

}  // namespace tsb

using namespace tsb;

extern "C" size_t tsb_tree_attn_shared_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int P, int own_rows,
                                                       int kv_format) {
  (void)D;
  if (!sizes_ok(B, T, Hq, Hkv, P, own_rows) || Hq % Hkv) return 0;
  const size_t n = partial_bytes(plan_shared(B, T, Hq, Hkv, P, own_rows), B, T, Hq);
  return kv_format == TSB_KV_BF16 ? n : n + 2 * copy_bytes(B, Hkv, P, own_rows);
}

extern "C" int tsb_tree_attn_shared(const void *q, long long q_stride_b, long long q_stride_h, long long q_stride_t,
                                    int kv_format, const tsb_kv_t *prefix, const tsb_kv_t *own, const int32_t *lengths,
                                    const int32_t *parents, const uint64_t *bits, int B, int T, int Hq, int Hkv, int D,
                                    int tail, float scale, void *out, float *lse, float *sums, void *ws, size_t ws_bytes,
                                    tsb_stream_t stream) {
  if (!q || !prefix || !own || !out) return TSB_EINVAL;
  const int P = prefix->rows, own_rows = own->rows;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || P < 0 || own_rows < 0) return TSB_EINVAL;
  if (prefix->capacity < P || own->capacity < own_rows) return TSB_EINVAL;
  if (!sizes_ok(B, T, Hq, Hkv, P, own_rows)) return TSB_EUNSUPPORTED;
  if (D != SH_D || Hq % Hkv || T > 64) return TSB_EUNSUPPORTED;
  if (!parents && !bits) return TSB_EINVAL;
  if (parents) tail = T;
  if (tail < 0 || tail > 64) return TSB_EUNSUPPORTED;
  if (kv_format < 0 || kv_format > 2) return TSB_EUNSUPPORTED;
  if (!(scale > 0.f)) return TSB_EUNSUPPORTED;  // the kernel takes row maxima of unscaled scores
  if (!aligned(q, 16) || q_stride_b % 8 || q_stride_h % 8 || q_stride_t % 8) return TSB_EINVAL;
  if (!aligned(out, 16) || !aligned(lse, 4) || !aligned(sums, 4)) return TSB_EINVAL;
  const tsb_kv_t *srcs[2] = {prefix, own};
  for (int i = 0; i < 2; ++i) {
    const int st = check_source(kv_format, srcs[i], srcs[i]->rows > 0);
    if (st != TSB_OK) return st;
  }
  if ((long long)Hkv * prefix->capacity > 0x7fffffc0LL || (long long)B * Hkv * own->capacity > 0x7fffffc0LL)
    return TSB_EUNSUPPORTED;  // tensor-map row coordinates are 32-bit
  const ShPlan p = plan_shared(B, T, Hq, Hkv, P, own_rows);
  const size_t part = partial_bytes(p, B, T, Hq);
  const size_t need = tsb_tree_attn_shared_workspace_bytes(B, T, Hq, Hkv, D, P, own_rows, kv_format);
  if (need && (!ws || ws_bytes < need)) return TSB_EWORKSPACE;
  if (!aligned(ws, 32)) return TSB_EINVAL;

  const size_t rows = (size_t)B * Hq * T;
  cudaStream_t stm = (cudaStream_t)stream;
  ShArgs a = {};
  CUtensorMap maps[4] = {};
  // the bf16 rows to attend to: the caches themselves, or copies of them
  char *copy = (char *)ws + part;
  ShConvert cv = {};
  cv.lengths = lengths;
  cv.hkv = Hkv;
  for (int i = 0; i < 2; ++i) {
    const tsb_kv_t *c = srcs[i];
    if (!c->rows) continue;
    const int requests = i ? B : 1;
    const void *kv[2] = {c->k, c->v}, *scales[2] = {c->k_scales, c->v_scales}, *biases[2] = {c->k_biases, c->v_biases};
    int cap = c->capacity;
    if (kv_format != TSB_KV_BF16) {
      ShConvert::Cache &to = cv.cache[i];
      to.cap = cap;
      to.rows = cap = c->rows;
      const long long blocks = 2LL * requests * Hkv * ((c->rows + SH_CV_ROWS - 1) / SH_CV_ROWS);
      if (blocks > 0x3fffffffLL) return TSB_EUNSUPPORTED;
      to.blocks = (int)blocks;
      for (int v = 0; v < 2; ++v) {
        to.src[v] = (const unsigned char *)kv[v];
        to.scale[v] = (const uint2 *)scales[v];
        to.bias[v] = (const uint2 *)biases[v];
        to.dst[v] = (uint16_t *)copy;
        kv[v] = copy;
        copy += (size_t)requests * Hkv * to.rows * SH_D * 2;
      }
    }
    a.src[i] = ShSource{(const float *)c->k_scales, (const float *)c->v_scales, c->capacity, cap, c->rows};
    for (int v = 0; v < 2; ++v)
      if (make_tmap_2d(&maps[2 * i + v], kv[v], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, SH_D,
                       (uint64_t)requests * Hkv * cap, SH_D * 2, 64, v ? SH_KT : SH_KT / 2,
                       CU_TENSOR_MAP_SWIZZLE_128B) != TSB_OK)
        return TSB_ECUDA;
  }
  if (kv_format != TSB_KV_BF16) {
    const int e = kv_format == TSB_KV_MLX_Q8_G64 ? launch_convert<true>(cv, stm) : launch_convert<false>(cv, stm);
    if (e != TSB_OK) return e;
  }
  a.q = (const uint16_t *)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_st = q_stride_t;
  a.parents = parents;
  a.bits = (const unsigned long long *)bits;
  a.lengths = lengths;
  a.B = B; a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.tail = tail;
  a.rb_p = p.rb_p; a.rb_o = p.rb_o;
  a.splits = p.splits; a.tps = p.tps; a.items = p.items;
  a.more = p.pairs ? p.items % p.pairs : 0;
  a.chunk = p.chunk; a.chunks = p.chunks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = (float *)ws;
  a.part_ml = a.part_o + (size_t)(p.splits + p.chunks) * rows * SH_D;
  if (p.pairs > 0) {
    const int e = kv_format == TSB_KV_REF_Q8_ROW ? launch_attn<true>(maps, a, p.pairs, stm)
                                                 : launch_attn<false>(maps, a, p.pairs, stm);
    if (e != TSB_OK) return e;
  }
  const cudaError_t e =
      launch_pdl(tree_attn_shared_combine_kernel, dim3((unsigned)((rows + SH_CB_WARPS - 1) / SH_CB_WARPS)),
                 dim3(SH_CB_WARPS * 32), 0, stm, (const float *)a.part_o, (const float *)a.part_ml, p.splits, lengths,
                 own_rows, p.chunk * SH_KT, Hq * T, (int)rows, (uint16_t *)out, lse, sums);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}
