// Tree attention for a batch that shares a long prefix. Each node attends to
// the P rows of one prefix cache, which every request sees, and to its own
// request's rows: out = softmax(scale q k) v over both, with the tree rule of
// tsb_tree_attn on the last `tail` own rows.
//
// The prefix is computed once for all: a KV head's query rows of the WHOLE
// batch (row = (request, head of the group, node)) are packed into blocks of
// 128, so each block of rows reads the prefix once instead of once per request.
// A work unit is (KV head, row block) over the prefix or (request, KV head, row
// block) over that request's own rows, and a CTA takes one key split of a unit.
// Every split leaves normalised partials with (max, sum), and a combine kernel
// merges a row's prefix and own partials.
//
// The roles and the TMEM plan inside a CTA are those of attn_tc.cu: TMA or
// converter warps fill K and V tiles of 64 keys, warp 1 issues S = Q K^T (Q in
// TMEM) and O += P V (P in TMEM), four softmax warps own a query row per
// thread. Unlike there, Q is gathered row by row from q's strides (a packed
// block spans requests), and 8-byte cp.async copies bring MLX scales and biases,
// so a cache of any capacity works. Own lengths are read on the device.
#include <algorithm>

#include "attn_tile.cuh"

namespace tsb {

namespace {

constexpr int SH_KT = 64;                  // keys per tile
constexpr int SH_D = 256;
constexpr int SH_KVBOX = SH_KT * 128;      // one 64-wide D box of 64 keys (bytes)
constexpr int SH_KV_BYTES = 4 * SH_KVBOX;  // 32 KB per bf16 K or V tile
constexpr uint32_t SH_O = 0, SH_Q = 256, SH_S0 = 384;
constexpr float SH_RESCALE_LOG2 = 8.f;
constexpr int SH_RAW_CODES = SH_KT * SH_D;  // 16 KB: one tile of 8-bit codes
constexpr int SH_NSC = 8;                   // row-scale ring of the reference format (tiles)
constexpr int SH_NCONV = 8;                 // converter warps (8-bit formats)
constexpr int SH_MAX_SPLITS = 64;           // key splits of a unit

template <int FMT>
struct ShCfg {
  static constexpr bool Q8 = FMT != TSB_KV_BF16;
  static constexpr bool MLX = FMT == TSB_KV_MLX_Q8_G64;
  static constexpr bool REF = FMT == TSB_KV_REF_Q8_ROW;
  static constexpr int NK = Q8 ? 2 : 3;  // bf16 K tiles in flight
  static constexpr int NV = Q8 ? 2 : 3;  // bf16 V tiles in flight
  static constexpr int NR = Q8 ? 5 : 0;  // raw 8-bit tiles in flight
  // raw stage: codes [64][256] u8, then (MLX) scales [64][4] and biases [64][4] bf16
  static constexpr int RAW_STAGE = MLX ? SH_RAW_CODES + 2 * SH_KT * 8 : SH_RAW_CODES;
  static constexpr int SC_BYTES = REF ? SH_NSC * 2 * SH_KT * 4 : 0;
  static constexpr int NBARS = 1 + 2 * NK + 2 * NV + 8 + 2 * NR + (REF ? SH_NSC : 0);
  static constexpr int CTRL = 2048;  // barriers, TMEM address, masks, parents
  static constexpr int THREADS = Q8 ? (6 + SH_NCONV) * 32 : 224;
  static constexpr size_t SMEM = (size_t)(NK + NV) * SH_KV_BYTES + (size_t)NR * RAW_STAGE + SC_BYTES + CTRL + 1024;
  static_assert((NBARS + 1) * 8 + 64 * 8 + 64 * 4 <= CTRL, "control block");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// One cache as the kernel reads it.
struct ShSource {
  const unsigned char *kc, *vc;   // 8-bit codes, D bytes per row
  const void *ks, *kb, *vs, *vb;  // MLX: bf16 [rows][4]; reference: float [rows] (ks, vs)
  int cap;                        // rows per (request, head)
  int rows;                       // valid rows: the prefix's, or the most any request has
};

struct ShArgs {
  ShSource src[2];  // prefix, own
  const uint16_t *q;
  long long q_sb, q_sh, q_st;  // element strides of q [B, Hq, T, D]
  const int32_t *parents;
  const unsigned long long *bits;
  const int32_t *lengths;
  int B, T, Hq, Hkv, tail;
  int rb_p, rb_o;          // row blocks of a prefix unit set / of a request's unit set
  int splits_p, splits_o;  // key splits
  int tps_p, tps_o;        // tiles per split
  int ctas_p;              // CTAs of prefix units; the others are own units
  float scale_log2;
  float *part_o;   // [splits_p + splits_o][B*Hq*T][D]
  float *part_ml;  // [splits_p + splits_o][B*Hq*T][2]
};

TSB_HD void cp_async8(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
// Arrive on bar when this thread's cp.async copies issued so far have landed
// (counts as one of the barrier's expected arrivals).
TSB_HD void cp_async_arrive(uint64_t *bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

template <int FMT>
__global__ void __launch_bounds__(ShCfg<FMT>::THREADS, 1)
tree_attn_shared_kernel(const __grid_constant__ CUtensorMap tmap_kp, const __grid_constant__ CUtensorMap tmap_vp,
                        const __grid_constant__ CUtensorMap tmap_ko, const __grid_constant__ CUtensorMap tmap_vo,
                        const __grid_constant__ ShArgs a) {
  using C = ShCfg<FMT>;
  constexpr int NK = C::NK, NV = C::NV, NR = C::NR;
  extern __shared__ unsigned char smem_raw[];
  unsigned char *smem =
      reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char *sK = smem;
  unsigned char *sV = sK + NK * SH_KV_BYTES;
  unsigned char *sRaw = sV + NV * SH_KV_BYTES;
  float *sSc = reinterpret_cast<float *>(sRaw + NR * C::RAW_STAGE);
  uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<unsigned char *>(sSc) + C::SC_BYTES);
  uint64_t *q_done = bars;
  uint64_t *k_full = bars + 1, *k_free = k_full + NK;
  uint64_t *v_full = k_free + NK, *v_free = v_full + NV;
  uint64_t *s_full = v_free + NV, *s_free = s_full + 2;
  uint64_t *p_full = s_free + 2, *p_free = p_full + 2;
  uint64_t *raw_full = p_free + 2, *raw_free = raw_full + NR;  // 8-bit formats
  uint64_t *sc_full = raw_free + NR;                            // reference format, [SH_NSC]
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + C::NBARS);
  unsigned long long *sBits = reinterpret_cast<unsigned long long *>(bars + C::NBARS + 1);  // [T <= 64]
  int32_t *sPar = reinterpret_cast<int32_t *>(sBits + 64);                                 // [T <= 64]

  griddep_wait();  // programmatic dependent: q, the caches and the lengths are the previous kernels'
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int G = a.Hq / a.Hkv, R = G * a.T;
  // ---- this CTA's unit
  const bool own = (int)blockIdx.x >= a.ctas_p;
  int unit = own ? blockIdx.x - a.ctas_p : blockIdx.x;
  const int splits = own ? a.splits_o : a.splits_p;
  const int split = unit % splits;
  unit /= splits;
  const int rbs = own ? a.rb_o : a.rb_p;
  const int rb = unit % rbs;
  unit /= rbs;
  const int kh = unit % a.Hkv;
  const int b = own ? unit / a.Hkv : 0;  // prefix units span the batch
  const ShSource &src = a.src[own];
  const int n_kv = own && a.lengths ? min(max(a.lengths[b], 0), src.rows) : src.rows;
  const int tail_lo = own ? n_kv - a.tail : n_kv;  // may be negative: fewer own rows than tree rows
  const int n_rows = own ? R : a.B * R;
  const int tps = own ? a.tps_o : a.tps_p;
  const int n_tiles_total = (n_kv + SH_KT - 1) / SH_KT;
  const int j_begin = split * tps;
  const int nt = max(0, min(n_tiles_total, j_begin + tps) - j_begin);
  const CUtensorMap &tmap_k = own ? tmap_ko : tmap_kp;
  const CUtensorMap &tmap_v = own ? tmap_vo : tmap_vp;
  const size_t kv_row0 = ((size_t)b * a.Hkv + kh) * (size_t)src.cap;

  if (threadIdx.x == 0) {
    // bf16 tiles are filled by a TMA transaction, 8-bit ones by the converter warps
    const uint32_t fill = C::Q8 ? SH_NCONV : 1;
    mbar_init(q_done, 4);
    for (int i = 0; i < NK; ++i) { mbar_init(&k_full[i], fill); mbar_init(&k_free[i], 1); }
    for (int i = 0; i < NV; ++i) { mbar_init(&v_full[i], fill); mbar_init(&v_free[i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_free[i], 4);
      mbar_init(&p_full[i], 4);
      mbar_init(&p_free[i], 1);
    }
    // raw tiles: the bulk copy's expect, and (MLX) 32 lanes' scale copies
    for (int i = 0; i < NR; ++i) { mbar_init(&raw_full[i], C::MLX ? 33 : 1); mbar_init(&raw_free[i], SH_NCONV); }
    if (C::REF)
      for (int i = 0; i < SH_NSC; ++i) mbar_init(&sc_full[i], SH_NCONV);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if constexpr (!C::Q8) {
      // ---------------- K producer
      if (elect_one()) {
        tma_prefetch_desc(&tmap_k);
        int j = 0;
        for (; j < nt; ++j) {
          const int key0 = (int)kv_row0 + (j_begin + j) * SH_KT;
          const int st = j % NK;
          if (j >= NK && !mbar_wait(&k_free[st], ((j / NK) - 1) & 1)) break;
          mbar_arrive_expect_tx(&k_full[st], SH_KV_BYTES);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            tma_load_2d(sK + st * SH_KV_BYTES + d * SH_KVBOX, &tmap_k, d * 64, key0, &k_full[st]);
        }
        // drain: the issued loads have landed before the CTA can exit
        for (int i = (j > NK ? j - NK : 0); i < j; ++i) mbar_drain(&k_full[i % NK], (i / NK) & 1);
      }
    } else {
      // ---------------- raw 8-bit tiles, rows [key0, min(key0 + 64, cap)) of this head's cache
      int seq = 0;
      auto load_raw = [&](bool isv, int j) -> bool {
        const int rs = seq % NR;
        if (seq >= NR && !warp_wait(&raw_free[rs], ((seq / NR) - 1) & 1)) return false;
        const int key0 = (j_begin + j) * SH_KT;
        const int rows = min(SH_KT, src.cap - key0);
        const size_t r0 = kv_row0 + key0;
        unsigned char *dst = sRaw + rs * C::RAW_STAGE;
        if (lane == 0) {
          mbar_arrive_expect_tx(&raw_full[rs], (uint32_t)rows * SH_D);
          bulk_load(dst, (isv ? src.vc : src.kc) + r0 * SH_D, (uint32_t)rows * SH_D, &raw_full[rs]);
        }
        if (C::MLX) {
          const uint2 *sc = reinterpret_cast<const uint2 *>(isv ? src.vs : src.ks) + r0;
          const uint2 *bi = reinterpret_cast<const uint2 *>(isv ? src.vb : src.kb) + r0;
          for (int r = lane; r < rows; r += 32) {
            cp_async8(dst + SH_RAW_CODES + r * 8, sc + r);
            cp_async8(dst + SH_RAW_CODES + SH_KT * 8 + r * 8, bi + r);
          }
          cp_async_arrive(&raw_full[rs]);
        }
        ++seq;
        return true;
      };
      bool ok = true;
      for (int j = 0; j < nt && ok; ++j) {
        if (j == 0) ok = load_raw(false, 0);
        if (ok && j + 1 < nt) ok = load_raw(false, j + 1);
        if (ok) ok = load_raw(true, j);
      }
      for (int i = (seq > NR ? seq - NR : 0); i < seq; ++i) mbar_drain(&raw_full[i % NR], (i / NR) & 1);
      __syncwarp();
    }
  } else if (warp >= 6) {
    if constexpr (!C::Q8) {
      // ---------------- V producer (warp 6)
      if (elect_one()) {
        tma_prefetch_desc(&tmap_v);
        int j = 0;
        for (; j < nt; ++j) {
          const int key0 = (int)kv_row0 + (j_begin + j) * SH_KT;
          const int st = j % NV;
          if (j >= NV && !mbar_wait(&v_free[st], ((j / NV) - 1) & 1)) break;
          mbar_arrive_expect_tx(&v_full[st], SH_KV_BYTES);
#pragma unroll
          for (int d = 0; d < 4; ++d)
            tma_load_2d(sV + st * SH_KV_BYTES + d * SH_KVBOX, &tmap_v, d * 64, key0, &v_full[st]);
        }
        for (int i = (j > NV ? j - NV : 0); i < j; ++i) mbar_drain(&v_full[i % NV], (i / NV) & 1);
      }
    } else {
      // ---------------- converters: raw tile -> swizzled bf16 tile. Lane l of
      // warp w writes 16-byte chunk l&7 of D box l>>3 (the MLX group) of rows
      // (w - 6) + 8 i: eight lanes fill one 128-byte row of a box.
      const int r_lo = warp - 6;
      const int grp = lane >> 3, ch = lane & 7;
      const int ct = threadIdx.x - 192;
      int seq = 0;
      auto convert = [&](bool isv, int j) -> bool {
        const int rs = seq % NR;
        uint64_t *full;
        unsigned char *dst;
        if (!isv) {
          const int st = j % NK;
          if (j >= NK && !warp_wait(&k_free[st], ((j / NK) - 1) & 1)) return false;
          dst = sK + st * SH_KV_BYTES;
          full = &k_full[st];
        } else {
          const int st = j % NV;
          if (j >= NV && !warp_wait(&v_free[st], ((j / NV) - 1) & 1)) return false;
          dst = sV + st * SH_KV_BYTES;
          full = &v_full[st];
        }
        const int key0 = (j_begin + j) * SH_KT;
        const int nvalid = n_kv - key0;  // rows below this are keys
        // reference format: the tile's key (threads 0-63) and value (64-127) row scales
        float rsc = 0.f;
        if (C::REF && !isv && ct < 2 * SH_KT) {
          const int r = ct & 63;
          if (r < nvalid) rsc = reinterpret_cast<const float *>(ct < 64 ? src.ks : src.vs)[kv_row0 + key0 + r];
        }
        if (!warp_wait(&raw_full[rs], (seq / NR) & 1)) return false;
        const unsigned char *raw = sRaw + rs * C::RAW_STAGE;
        const uint16_t *rsb = reinterpret_cast<const uint16_t *>(raw + SH_RAW_CODES);
        constexpr int CB = 4, ROWS = SH_KT / SH_NCONV;
        static_assert(SH_KT % SH_NCONV == 0 && ROWS % CB == 0, "converter rows");
        // batches of CB rows, loads first; rolled, as the instruction cache also
        // holds the softmax loop of the same sub-partition
#pragma unroll 1
        for (int h = 0; h < ROWS / CB; ++h) {
          uint2 w[CB];
          uint32_t sb[CB], bb[CB];
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            const int r = r_lo + SH_NCONV * (CB * h + i);
            w[i] = make_uint2(0u, 0u);
            sb[i] = 0u;
            bb[i] = 0u;
            if (r < nvalid) {
              w[i] = *reinterpret_cast<const uint2 *>(raw + r * SH_D + lane * 8);
              if (C::MLX) {
                sb[i] = rsb[r * 4 + grp];
                bb[i] = rsb[SH_KT * 4 + r * 4 + grp];
              }
            }
          }
#pragma unroll
          for (int i = 0; i < CB; ++i) {
            const int r = r_lo + SH_NCONV * (CB * h + i);
            uint4 o = make_uint4(0u, 0u, 0u, 0u);
            if (r < nvalid) {
              if (C::MLX)
                o = dequant8_mlx(w[i], __uint_as_float(sb[i] << 16), __uint_as_float(bb[i] << 16));
              else
                o = convert8_s8(w[i]);
            }
            *reinterpret_cast<uint4 *>(dst + grp * SH_KVBOX + r * 128 + ((ch ^ (r & 7)) << 4)) = o;
          }
        }
        if (C::REF && !isv && ct < 2 * SH_KT) sSc[(j % SH_NSC) * 2 * SH_KT + ct] = rsc;
        fence_proxy_async_smem();  // generic writes -> MMA reads; raw slot reads -> refill
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&raw_free[rs]);
          mbar_arrive(full);
          if (C::REF && !isv) mbar_arrive(&sc_full[j % SH_NSC]);
        }
        ++seq;
        return true;
      };
      bool ok = true;
      for (int j = 0; j < nt && ok; ++j) {
        if (j == 0) ok = convert(false, 0);
        if (ok && j + 1 < nt) ok = convert(false, j + 1);
        if (ok) ok = convert(true, j);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer
    const uint32_t idesc_s = idesc_bf16_f32(128, SH_KT);
    const uint32_t idesc_o = idesc_bf16_f32(128, SH_D) | (1u << 16);  // B (V) MN-major
    bool ok = warp_wait(q_done, 0);
    auto issue_s = [&](int j) -> bool {
      const int s = j % NK, sb = j & 1;
      if (!warp_wait(&k_full[s], (j / NK) & 1)) return false;
      if (j >= 2 && !warp_wait(&s_free[sb], ((j >> 1) - 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t kb = smem_addr(sK + s * SH_KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) {
          const uint32_t off_k = (kk >> 2) * SH_KVBOX + (kk & 3) * 32;
          mma_ts_f16(tmem + SH_S0 + sb * 64, tmem + SH_Q + kk * 8, desc_kmajor_sw128(kb + off_k), idesc_s,
                     kk > 0 ? 1u : 0u);
        }
        mma_commit(&s_full[sb]);
        mma_commit(&k_free[s]);
      }
      __syncwarp();
      return true;
    };
    auto issue_pv = [&](int j) -> bool {
      const int s = j % NV, pb = j & 1;
      if (!warp_wait(&v_full[s], (j / NV) & 1)) return false;
      if (!warp_wait(&p_full[pb], (j >> 1) & 1)) return false;
      tc_fence_after();
      if (!C::Q8) {
        // bf16: the TMA tile holds whatever follows row n_kv; zero those V rows
        // (their weights are 0, but 0 * NaN would not be 0)
        const int first = n_kv - (j_begin + j) * SH_KT;
        if (first < SH_KT) {
          unsigned char *vt = sV + s * SH_KV_BYTES;
          for (int i = lane; i < (SH_KT - first) * 32; i += 32) {
            const int r = first + (i >> 5), c = i & 31;
            *reinterpret_cast<uint4 *>(vt + (c >> 3) * SH_KVBOX + r * 128 + ((c & 7) << 4)) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
          __syncwarp();
        }
      }
      if (elect_one()) {
        const uint32_t vb = smem_addr(sV + s * SH_KV_BYTES);
#pragma unroll
        for (int kk = 0; kk < SH_KT / 16; ++kk) {
          mma_ts_f16(tmem + SH_O, tmem + SH_S0 + pb * 64 + kk * 8, desc_mnmajor_sw128(vb + kk * 2048, SH_KVBOX),
                     idesc_o, (j > 0 || kk > 0) ? 1u : 0u);
        }
        mma_commit(&v_free[s]);
        mma_commit(&p_free[pb]);  // completes after this and every earlier MMA
      }
      __syncwarp();
      return true;
    };
    if (ok && nt > 0) ok = issue_s(0);
    for (int j = 0; j < nt && ok; ++j) {
      if (j + 1 < nt) ok = issue_s(j + 1);
      if (ok) ok = issue_pv(j);
    }
  } else if (warp >= 2 && warp <= 5) {
    // ---------------- softmax / epilogue (thread = query row = TMEM lane)
    if (own) {  // node masks, from the parent array or given
      const int st = threadIdx.x - 64;  // 0..127
      if (st < a.T) sPar[st] = a.parents ? a.parents[(size_t)b * a.T + st] : 0;
      named_barrier_sync(1, 128);
      if (st < a.T) {
        unsigned long long m = 0;
        if (a.parents) {
          int j = st;
          bool okp = true;
          for (int steps = 0; steps <= a.T && j != -1; ++steps) {
            m |= 1ull << j;
            const int pj = sPar[j];
            if (!(pj == -1 || (pj >= 0 && pj < j))) { okp = false; break; }
            j = pj;
          }
          if (!okp) m = 0;
        } else {
          m = a.bits[(size_t)b * a.T + st];
        }
        sBits[st] = m;
      }
      named_barrier_sync(1, 128);
    }
    const int q = warp & 3;
    const int r = q * 32 + lane;
    const int gr = rb * 128 + r;
    const bool row_valid = gr < n_rows;
    // the row's request, head and node
    const int rq = row_valid ? (own ? b : gr / R) : 0;
    const int rr = row_valid ? (own ? gr : gr % R) : 0;
    const int hl = rr / a.T, node = rr % a.T;
    const int head = kh * G + hl;
    const unsigned long long mybits = own ? sBits[node] : 0ull;
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16);
    const float sl2 = a.scale_log2;
    float m = -INFINITY, l = 0.f;  // running max (log2 domain) and sum
    if (nt > 0) {
      // Q row -> TMEM lane r, columns SH_Q + d/2 (the A-operand layout of a K-major M=128 tile)
      const uint4 *qrow = reinterpret_cast<const uint4 *>(a.q + rq * a.q_sb + head * a.q_sh + node * a.q_st);
#pragma unroll 1
      for (int bx = 0; bx < 4; ++bx) {
        uint32_t qv[32];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint4 u = row_valid ? __ldg(qrow + bx * 8 + c) : make_uint4(0u, 0u, 0u, 0u);
          qv[4 * c] = u.x; qv[4 * c + 1] = u.y; qv[4 * c + 2] = u.z; qv[4 * c + 3] = u.w;
        }
        tmem_st32(lane_base + SH_Q + bx * 32, qv);
      }
      tmem_wait_st();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(q_done);
    bool ok = true;
    for (int j = 0; j < nt && ok; ++j) {
      const int sb = j & 1;
      ok = warp_wait(&s_full[sb], (j >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      uint32_t sr[64];
      {
        uint32_t (&lo)[32] = *reinterpret_cast<uint32_t (*)[32]>(&sr[0]);
        uint32_t (&hi)[32] = *reinterpret_cast<uint32_t (*)[32]>(&sr[32]);
        tmem_ld32(lane_base + SH_S0 + sb * 64, lo);
        tmem_ld32(lane_base + SH_S0 + sb * 64 + 32, hi);
      }
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&s_free[sb]);
      const float *ksc = sSc + (j % SH_NSC) * 2 * SH_KT;  // reference format: key, then value scales
      if (C::REF) {
        ok = warp_wait(&sc_full[j % SH_NSC], (j / SH_NSC) & 1);
        if (!ok) break;
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          const float4 k4 = *reinterpret_cast<const float4 *>(ksc + e);
          sr[e] = __float_as_uint(__uint_as_float(sr[e]) * k4.x);
          sr[e + 1] = __float_as_uint(__uint_as_float(sr[e + 1]) * k4.y);
          sr[e + 2] = __float_as_uint(__uint_as_float(sr[e + 2]) * k4.z);
          sr[e + 3] = __float_as_uint(__uint_as_float(sr[e + 3]) * k4.w);
        }
      }
      // mask (only the tail and the last tile need it), then the tile max of the
      // raw scores in eight independent chains; the scale is applied in the exp
      const int key0 = (j_begin + j) * SH_KT;
      if ((key0 + SH_KT > tail_lo) || (key0 + SH_KT > n_kv)) {
#pragma unroll
        for (int e = 0; e < 64; ++e) {
          const int key = key0 + e;
          bool vis = key < n_kv;
          if (vis && key >= tail_lo) vis = (mybits >> (key - tail_lo)) & 1ull;
          if (!vis) sr[e] = __float_as_uint(-INFINITY);
        }
      }
      float mx8[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) mx8[c] = __uint_as_float(sr[c]);
#pragma unroll
      for (int e = 8; e < 64; ++e) mx8[e & 7] = fmaxf(mx8[e & 7], __uint_as_float(sr[e]));
      const float traw = fmaxf(fmaxf(fmaxf(mx8[0], mx8[1]), fmaxf(mx8[2], mx8[3])),
                               fmaxf(fmaxf(mx8[4], mx8[5]), fmaxf(mx8[6], mx8[7])));
      const float tmax = traw * sl2;  // scale > 0: max commutes with it
      // P V_{j-2} is done (S_j, written after it, is complete); waiting here
      // keeps every p_free wait below at most one phase behind.
      if (j >= 2) {
        ok = warp_wait(&p_free[sb], ((j >> 1) - 1) & 1);
        if (!ok) break;
      }
      // lazy rescale: move the reference max only when it grows by > 2^8
      const bool grow = tmax > m + SH_RESCALE_LOG2;
      if (__any_sync(0xffffffffu, grow)) {
        const float m_new = grow ? tmax : m;
        const float alpha = (m == -INFINITY) ? 0.f : ex2(m - m_new);
        if (j > 0) {  // O holds earlier tiles: wait for P V_{j-1} (and all before), then scale O in place
          ok = warp_wait(&p_free[sb ^ 1], ((j - 1) >> 1) & 1);
          if (!ok) break;
          tc_fence_after();
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
        l *= alpha;
        m = m_new;
      }
      const float nbase = (m == -INFINITY) ? 0.f : -m;
      uint32_t pk[32];
      float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        const float p0 = ex2(__fmaf_rn(__uint_as_float(sr[2 * e]), sl2, nbase));
        const float p1 = ex2(__fmaf_rn(__uint_as_float(sr[2 * e + 1]), sl2, nbase));
        ps[e & 3] += p0 + p1;
        if (C::REF) {
          // the value rows' scales weight P; the running sum keeps the plain weights
          const float2 v2 = *reinterpret_cast<const float2 *>(ksc + SH_KT + 2 * e);
          pk[e] = pack_bf16x2(p0 * v2.x, p1 * v2.y);
        } else {
          pk[e] = pack_bf16x2(p0, p1);
        }
      }
      l += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      // P_j into TMEM, over the scores it was made from
      tc_fence_after();
      tmem_st32(lane_base + SH_S0 + sb * 64, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[sb]);
    }
    // ---------------- epilogue: normalised partials and (max, sum)
    const size_t orow = ((size_t)rq * a.Hq + head) * a.T + node;
    const size_t prow = (size_t)(own ? a.splits_p + split : split) * a.B * a.Hq * a.T + orow;
    if (ok && nt > 0 && warp_wait(&p_free[(nt - 1) & 1], ((nt - 1) >> 1) & 1)) {
      tc_fence_after();
      const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < SH_D; c += 32) {
        uint32_t o[32];
        tmem_ld32(lane_base + SH_O + c, o);
        tmem_wait_ld();
        if (!row_valid) continue;
        float4 *dst = reinterpret_cast<float4 *>(a.part_o + prow * SH_D + c);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          dst[e] = make_float4(__uint_as_float(o[4 * e]) * inv, __uint_as_float(o[4 * e + 1]) * inv,
                               __uint_as_float(o[4 * e + 2]) * inv, __uint_as_float(o[4 * e + 3]) * inv);
      }
    }
    if (row_valid) {
      a.part_ml[prow * 2 + 0] = m;
      a.part_ml[prow * 2 + 1] = l;  // 0: nothing visible, the partial is not read
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- combine
// out = sum_s w_s o_s, w_s = l_s 2^(m_s - m) / sum. Partials of empty splits
// (l = 0) are not read. A warp per row: lane = 8 of the 256 columns.
constexpr int SH_CB_WARPS = 4;

__global__ void __launch_bounds__(SH_CB_WARPS * 32)
tree_attn_shared_combine_kernel(const float *__restrict__ part_o, const float *__restrict__ part_ml, int slots,
                                int rows, uint16_t *__restrict__ out, float *__restrict__ lse) {
  griddep_wait();  // programmatic dependent: the partials are the attention kernel's
  griddep_launch_dependents();
  const int lane = threadIdx.x % 32;
  const int row = blockIdx.x * SH_CB_WARPS + threadIdx.x / 32;
  if (row >= rows) return;
  const float2 *ml = reinterpret_cast<const float2 *>(part_ml) + row;
  float m = -INFINITY;
  for (int s = lane; s < slots; s += 32) {
    const float2 v = ml[(size_t)s * rows];
    if (v.y > 0.f) m = fmaxf(m, v.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float den = 0.f;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < slots; s0 += 32) {
    float w = 0.f;
    if (s0 + lane < slots) {
      const float2 v = ml[(size_t)(s0 + lane) * rows];
      if (v.y > 0.f) w = v.y * exp2f(v.x - m);
    }
    float part = w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
    den += part;
    for (int s = 0; s < min(32, slots - s0); ++s) {
      const float ws = __shfl_sync(0xffffffffu, w, s);
      if (ws == 0.f) continue;
      const float4 *src = reinterpret_cast<const float4 *>(part_o + ((size_t)(s0 + s) * rows + row) * SH_D) + lane;
      const float4 x = src[0], y = src[32];
      acc[0] = fmaf(ws, x.x, acc[0]); acc[1] = fmaf(ws, x.y, acc[1]);
      acc[2] = fmaf(ws, x.z, acc[2]); acc[3] = fmaf(ws, x.w, acc[3]);
      acc[4] = fmaf(ws, y.x, acc[4]); acc[5] = fmaf(ws, y.y, acc[5]);
      acc[6] = fmaf(ws, y.z, acc[6]); acc[7] = fmaf(ws, y.w, acc[7]);
    }
  }
  const float inv = den > 0.f ? 1.f / den : 0.f;
  uint2 *dst = reinterpret_cast<uint2 *>(out + (size_t)row * SH_D) + lane;
  dst[0] = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  dst[32] = make_uint2(pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
  if (lse && lane == 0) lse[row] = den > 0.f ? (m + log2f(den)) * 0.69314718055994531f : -INFINITY;
}

struct ShPlan {
  int rb_p, rb_o, splits_p, splits_o, tps_p, tps_o;
};

int split_tiles(int tiles, int units, int &tps) {
  if (tiles <= 0) { tps = 0; return 0; }
  int s = sm_count() / units;
  s = std::min(std::min(s, tiles / 4), SH_MAX_SPLITS);
  s = std::max(s, 1);
  tps = (tiles + s - 1) / s;
  return (tiles + tps - 1) / tps;
}

ShPlan plan_shared(int B, int T, int Hq, int Hkv, int P, int own_rows) {
  ShPlan p;
  const int R = (Hq / Hkv) * T;
  p.rb_p = (int)(((long long)B * R + 127) / 128);
  p.rb_o = (R + 127) / 128;
  p.splits_p = split_tiles((P + SH_KT - 1) / SH_KT, Hkv * p.rb_p, p.tps_p);
  p.splits_o = split_tiles((own_rows + SH_KT - 1) / SH_KT, B * Hkv * p.rb_o, p.tps_o);
  return p;
}

bool sizes_ok(int B, int T, int Hq, int Hkv, int P, int own_rows) {
  return B > 0 && T > 0 && Hq > 0 && Hkv > 0 && P >= 0 && own_rows >= 0 && (long long)B * Hq * T <= (1 << 24);
}

template <int FMT>
int launch_fmt(const CUtensorMap *maps, const ShArgs &a, int ctas, cudaStream_t st) {
  using C = ShCfg<FMT>;
  if (cudaFuncSetAttribute(tree_attn_shared_kernel<FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM) !=
      cudaSuccess)
    return TSB_ECUDA;
  const cudaError_t e = launch_pdl(tree_attn_shared_kernel<FMT>, dim3((unsigned)ctas), dim3(C::THREADS),
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

extern "C" size_t tsb_tree_attn_shared_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int P, int own_rows) {
  (void)D;
  if (!sizes_ok(B, T, Hq, Hkv, P, own_rows) || Hq % Hkv) return 0;
  const ShPlan p = plan_shared(B, T, Hq, Hkv, P, own_rows);
  return (size_t)(p.splits_p + p.splits_o) * B * Hq * T * (SH_D + 2) * sizeof(float);
}

extern "C" int tsb_tree_attn_shared(const void *q, long long q_stride_b, long long q_stride_h, long long q_stride_t,
                                    int kv_format, const tsb_kv_t *prefix, const tsb_kv_t *own, const int32_t *lengths,
                                    const int32_t *parents, const uint64_t *bits, int B, int T, int Hq, int Hkv, int D,
                                    int tail, float scale, void *out, float *lse, void *ws, size_t ws_bytes,
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
  if (!aligned(out, 16) || !aligned(lse, 4)) return TSB_EINVAL;
  int st = check_source(kv_format, prefix, P > 0);
  if (st == TSB_OK) st = check_source(kv_format, own, own_rows > 0);
  if (st != TSB_OK) return st;
  if ((long long)Hkv * prefix->capacity > 0x7fffffc0LL || (long long)B * Hkv * own->capacity > 0x7fffffc0LL)
    return TSB_EUNSUPPORTED;  // tensor-map row coordinates are 32-bit
  const size_t need = tsb_tree_attn_shared_workspace_bytes(B, T, Hq, Hkv, D, P, own_rows);
  if (need && (!ws || ws_bytes < need)) return TSB_EWORKSPACE;
  if (!aligned(ws, 16)) return TSB_EINVAL;

  const ShPlan p = plan_shared(B, T, Hq, Hkv, P, own_rows);
  const size_t rows = (size_t)B * Hq * T;
  const int slots = p.splits_p + p.splits_o;
  ShArgs a = {};
  const tsb_kv_t *srcs[2] = {prefix, own};
  for (int i = 0; i < 2; ++i)
    a.src[i] = ShSource{reinterpret_cast<const unsigned char *>(srcs[i]->k),
                        reinterpret_cast<const unsigned char *>(srcs[i]->v), srcs[i]->k_scales, srcs[i]->k_biases,
                        srcs[i]->v_scales, srcs[i]->v_biases, srcs[i]->capacity, srcs[i]->rows};
  a.q = (const uint16_t *)q;
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.q_st = q_stride_t;
  a.parents = parents;
  a.bits = (const unsigned long long *)bits;
  a.lengths = lengths;
  a.B = B; a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.tail = tail;
  a.rb_p = p.rb_p; a.rb_o = p.rb_o;
  a.splits_p = p.splits_p; a.splits_o = p.splits_o;
  a.tps_p = p.tps_p; a.tps_o = p.tps_o;
  a.ctas_p = Hkv * p.rb_p * p.splits_p;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.part_o = (float *)ws;
  a.part_ml = a.part_o + (size_t)slots * rows * SH_D;
  const long long ctas = (long long)a.ctas_p + (long long)B * Hkv * p.rb_o * p.splits_o;
  if (ctas > 0x7fffffffLL) return TSB_EUNSUPPORTED;
  cudaStream_t stm = (cudaStream_t)stream;
  if (ctas > 0) {
    CUtensorMap maps[4] = {};
    if (kv_format == TSB_KV_BF16) {
      for (int i = 0; i < 2; ++i) {
        if (!(i ? own_rows : P)) continue;
        const uint64_t n = (uint64_t)(i ? B : 1) * Hkv * srcs[i]->capacity;
        for (int v = 0; v < 2; ++v)
          if (make_tmap_2d(&maps[2 * i + v], v ? srcs[i]->v : srcs[i]->k, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, SH_D, n,
                           SH_D * 2, 64, SH_KT, CU_TENSOR_MAP_SWIZZLE_128B) != TSB_OK)
            return TSB_ECUDA;
      }
    }
    int e;
    if (kv_format == TSB_KV_BF16) e = launch_fmt<TSB_KV_BF16>(maps, a, (int)ctas, stm);
    else if (kv_format == TSB_KV_MLX_Q8_G64) e = launch_fmt<TSB_KV_MLX_Q8_G64>(maps, a, (int)ctas, stm);
    else e = launch_fmt<TSB_KV_REF_Q8_ROW>(maps, a, (int)ctas, stm);
    if (e != TSB_OK) return e;
  }
  const cudaError_t e =
      launch_pdl(tree_attn_shared_combine_kernel, dim3((unsigned)((rows + SH_CB_WARPS - 1) / SH_CB_WARPS)),
                 dim3(SH_CB_WARPS * 32), 0, stm, (const float *)a.part_o, (const float *)a.part_ml, slots, (int)rows,
                 (uint16_t *)out, lse);
  return e == cudaSuccess ? TSB_OK : TSB_ECUDA;
}
