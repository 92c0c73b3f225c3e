// Attention over a sliding window with visible first tokens, forward, on tcgen05: for a training step or a prompt
// (contiguous keys), for the drafted tokens of a serving step (a tree of them over a paged or contiguous cache) and for
// single next tokens.
//
//   o_i = sum_j p_ij v_j,   p_i = softmax over the keys that row i sees of  scale * q_i.k_j   (plus, where a head has a sink
//   logit, one key of that logit and value 0)
//
// Row i stands at position P_i and sees key j when j <= P_i, j is a valid key, and P_i - j < window or j < ns; drafted node n
// stands at prefix + (number of its ancestors) and sees of the other nodes only those in its 64-bit word.
//
// Work of a CTA: a 128-row tile (window_attn.h: g heads x 128 / g queries) against tiles of 64 keys.
//
//   S = Q.K^T       tcgen05.mma 128 x n x 16, fp32 in TMEM (n = the tile's keys, rounded up to 16: the few first tokens and the
//                   last tile cost what they hold)
//   P = exp2(S c - m)   one row per thread, its scores in registers, P written back over S in TMEM as bf16.  P's rounding (half
//                   a step, 2^-8) is that of the product's operand type; the row's sum is of the unrounded values in fp32.
//   O += P.V        A from TMEM (from shared memory, P and its reads would cost half as much shared-memory bandwidth again as
//                   the K, V and Q reads that already take most of it), V read MN-major in place, accumulator resident in TMEM
//
// The reference m need not be the maximum: bf16 and fp32 share the exponent range, so P, its sum and O keep their precision at any m
// that neither overflows nor loses the largest terms.  m is the maximum of the first tile with a key, and moves (O rescaled in
// TMEM) when a tile's sum comes out above 2^40; terms 2^126 below m are nothing beside the first tile's, which reach 1.  So the common
// tile needs no maximum at all.
//
// Two CTAs share an SM (8 warps, half the TMEM and 113 KB of shared memory each): one's products run under the other's
// exponentials, and its start and end under the other's tiles.  Against one CTA an SM with two row tiles that shared the key tiles,
// this fetches every key tile twice from L2 and still gains where the tiles are many (2 x 4096 queries, 16 heads over 4 of 128, a window of 1024: 104 -> 94 us),
// and more where they are few (128 single tokens over a window of 1024: 50 -> 37 us).  Tiles of 64 keys leave room for two score
// buffers, so that the next scores run under this tile's exponentials: with one buffer of 128 every tile waited for its product and
// the next scores, 2000 of 5200 clocks.
//
// With <= 32 (64) rows the tile holds them four (two) times in its TMEM lane quarters and each copy takes a quarter (half) of a tile's
// keys, because a warp can only read its own quarter of the lanes: otherwise one warp would do all the exponentials.
//
// Few row tiles are split over the key axis as well (grid): up to 8 splits of up to 64 rows are a cluster, which joins
// their partial results through shared memory; others go through global memory and window_combine_kernel (a cluster of 128-row tiles
// took 16.1 us where this took 12.7: 60 nodes over 1024 keys).
//
// Rows of V that no row may see (past a sequence's end, padding, pages handed on to others) may hold anything, NaN included:
// the products' warp zeroes them in shared memory before they are multiplied with P's zeros.
//
// Every wait is bounded (sm100.cuh).
#include <cstring>
#include <type_traits>

#include "window_attn.h"

namespace cmb {

constexpr float WA_FAR = 1099511627776.f;   // 2^40: a tile's row sum above which the reference moves
constexpr int WA_CTL = 1024;             // barriers and looked-up pages

struct WindowParams {
  int S, T, H, Hk, g;                    // queries, keys per sequence (cache capacity), heads
  int box_q;                             // queries in a row tile's TMA box
  int Dv;
  float scale_log2;                      // softmax scale * log2(e)
  int window, ns;
  int cached;                            // 0: row i at T - S + i, lengths = valid keys (or null); 1: lengths = prefix
  const int* lengths;
  const unsigned long long* tree;        // cached: [.., S] words, null = a chain
  int tree_sb;
  const int* table;                      // null = contiguous
  int table_w, page, num_pages, box_k;   // box_k: key rows per TMA box; tiles start at its multiples when paged
  WaSinks sinks;
  __nv_bfloat16* out;
  long long o_sb, o_ss, o_sh;
  float* lse;                            // [B, H, S] natural log, +inf where a row sees nothing; may be null
  int splits, joined;                    // joined: a row's splits are a cluster, which joins them through shared memory
  float* ws_o;                           // [B, S, H, splits, Dv], not joined
  float2* ws_ml;                         // [B, S, H, splits] (max, sum)
  int* status;
};

template <int DB, int COPIES>
struct WindowCfg {
  static constexpr int BN = 64;                          // keys of a tile
  static constexpr int BUFS = 2;                         // score buffers
  static constexpr int COPY_ROWS = 128 / COPIES;
  static constexpr int TN = BN / COPIES;                 // keys of a tile that a softmax thread takes, in chunks of CW
  static constexpr int CW = TN < 32 ? TN : 32, CH = TN / CW;
  // warps: 0-3 softmax, then the producer of keys, scores, products, producer of values
  static constexpr int W_K = 4, W_S = 5, W_P = 6, W_V = 7, THREADS = 256, CTAS = 2;      // CTAs of an SM
  static constexpr int KBLK = BN * 128;                  // bytes of a [BN keys x 64 columns] block
  static constexpr int Q_BYTES = DB * WA_BLK;
  static constexpr int NK = DB == 2 ? 3 : 6, NV = DB == 2 ? 2 : 6;
  static constexpr int STAGE = DB * KBLK;
  static constexpr int SMEM_BYTES = Q_BYTES + (NK + NV) * STAGE + WA_CTL;
  static constexpr int PART_PITCH = DB * 64 + 4;         // floats; rows 16 bytes apart in banks
  static_assert((SMEM_BYTES + 1024) * CTAS <= 233472 && (9 + 2 * NK + 2 * NV) * 8 + 8 <= 512, "shared memory");
  static_assert(128 * PART_PITCH * 4 <= (NK + NV) * STAGE, "partial results reuse the rings");
  // TMEM: O, then the score buffers; P is written over the scores
  static constexpr int S_COL = 128, TMEM_COLS = 256;
};

// One row's place in the problem.
struct WindowRow {
  int s, h;                    // query, head
  bool ok;                     // sees anything at all by construction (in range, not padding)
  int p, plim, lo;             // position; last key seen by position; first key of its window
  unsigned long long nodes;    // drafted nodes it sees
};

__device__ __forceinline__ WindowRow window_row(const WindowParams& p, int r, int s0, int hk, int b, int klim, int prefix) {
  WindowRow w;
  const int ql = r / p.g;
  w.s = s0 + ql;
  w.h = hk * p.g + (r - ql * p.g);
  w.ok = ql < p.box_q && w.s < p.S;
  w.nodes = 0ull;
  w.p = p.cached ? prefix + w.s : p.T - p.S + w.s;
  w.plim = min(w.p, klim - 1);
  if (w.ok && p.tree != nullptr) {
    const unsigned long long* tree = p.tree + static_cast<long long>(b) * p.tree_sb;
    const unsigned long long places = p.S < 64 ? (1ull << p.S) - 1ull : ~0ull;      // bits past the last node say nothing
    const unsigned long long word = tree[w.s] & places;
    const int depth = __popcll(word) - 1;
    w.ok = word != 0ull;
    w.p = prefix + depth;
    w.plim = prefix - 1;
    w.nodes = word;
    if (p.window <= depth) {                 // the window ends inside the drafted nodes
      unsigned long long left = w.nodes;
      while (left) {
        const int m = __ffsll(static_cast<long long>(left)) - 1;
        left &= left - 1ull;
        const int dm = __popcll(tree[m] & places) - 1;
        if (!(depth - dm < p.window || prefix + dm < p.ns)) w.nodes &= ~(1ull << m);
      }
    }
  }
  w.lo = w.p - p.window + 1;
  return w;
}
__device__ __forceinline__ unsigned window_word(const WindowParams& p, const WindowRow& w, int j0, int k1, int prefix) {
  unsigned bits = wa_mask_word(j0, w.plim, w.lo, p.ns, k1);
  if (p.tree != nullptr) {
    const int d = j0 - prefix;
    if (d > -32 && d < 64) bits |= static_cast<unsigned>(d >= 0 ? w.nodes >> d : w.nodes << (-d));
    bits &= wa_low_bits(k1 - j0);
  }
  return w.ok ? bits : 0u;
}

template <int DB, int COPIES>
__global__ void __launch_bounds__(WindowCfg<DB, COPIES>::THREADS, WindowCfg<DB, COPIES>::CTAS)
window_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                  const __grid_constant__ CUtensorMap tmV, const WindowParams p) {
  using Cfg = WindowCfg<DB, COPIES>;
  constexpr int NK = Cfg::NK, NV = Cfg::NV, BN = Cfg::BN, BUFS = Cfg::BUFS;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {   // swizzled TMA / MMA tiles need 1024-byte aligned buffers
    if (threadIdx.x == 0 && p.status != nullptr && atomicCAS(p.status, 0, ST_BAD_ARGUMENT) == 0) p.status[1] = -1024;
    return;
  }
  uint8_t* qs = smem;
  uint8_t* ks = qs + Cfg::Q_BYTES;
  uint8_t* vs = ks + NK * Cfg::STAGE;
  uint8_t* ctl = vs + NV * Cfg::STAGE;
  // at the end, when the queries and the rings have been read:
  float2* xml = reinterpret_cast<float2*>(qs);           // [128] (reference, sum) of every row and copy
  float2* fml = xml + 128;                               // [128] of every row, for the cluster's other splits
  float* part = reinterpret_cast<float*>(ks);            // [128][PART_PITCH]
  uint64_t* q_full = reinterpret_cast<uint64_t*>(ctl);
  uint64_t* k_full = q_full + 1;           // [NK]
  uint64_t* k_empty = k_full + NK;         // [NK]
  uint64_t* v_full = k_empty + NK;         // [NV] landed
  uint64_t* v_empty = v_full + NV;         // [NV]
  uint64_t* s_full = v_empty + NV;         // [buffer]
  uint64_t* p_full = s_full + BUFS;        // [buffer] P written
  uint64_t* pv_done = p_full + BUFS;       // [buffer] P read, O added to
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(pv_done + BUFS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z / p.splits, split = blockIdx.z - b * p.splits;
  const int hk = blockIdx.y;
  const int xt = static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x);   // longest rows first
  int* status = p.status;

  // rows and keys of this CTA
  const int s_first = xt * p.box_q;
  const int s_last = min(p.S, s_first + p.box_q) - 1;
  int prefix = 0, klim, pmin, pmax;
  if (p.cached) {
    prefix = max(0, min(p.lengths[b], p.T - p.S));                 // out-of-range prefixes are reported below
    klim = prefix + p.S;
    pmin = p.tree != nullptr ? prefix : prefix + s_first;
    pmax = p.tree != nullptr ? prefix + p.S - 1 : prefix + s_last;
  } else {
    klim = p.lengths != nullptr ? max(0, min(p.lengths[b], p.T)) : p.T;
    pmin = p.T - p.S + s_first;
    pmax = p.T - p.S + s_last;
  }
  const WaRange<BN> R(pmin, pmax, klim, p.window, p.ns, p.table != nullptr ? p.box_k : 1);
  const int per = (R.n_t + p.splits - 1) / p.splits;
  const int t0 = min(R.n_t, split * per), t1 = min(R.n_t, t0 + per);
  const int NT = t1 - t0;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
    mbar_init(q_full, 1);
    for (int i = 0; i < NK; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < NV; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    *abort_flag = 0;
    fence_mbar_init();
    if (p.lengths != nullptr && status != nullptr) {   // a length that the cache cannot hold
      const int n = p.lengths[b];
      if ((n < 0 || n > (p.cached ? p.T - p.S : p.T)) && atomicCAS(status, 0, ST_BAD_ARGUMENT) == 0) {
        status[1] = b;
        status[2] = n;
      }
    }
  }
  if (warp == Cfg::W_K) {
    tmem_alloc(tmem_slot, Cfg::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // a row's end: its head's sink logit joins (reference, sum), and what O is multiplied with
  auto finish = [&](int h, float& m, float& l) {
    float f = 1.f;
    if (p.sinks.p != nullptr) {
      const float s2 = p.sinks.log2_at(h), top = fmaxf(m, s2);
      if (s2 != -INFINITY) {                 // (a logit of -inf is no key: a row that sees nothing keeps its sum of 0)
        f = m == -INFINITY ? 0.f : exp2f(m - top);
        l = l * f + exp2f(s2 - top);
        m = top;
      }
    }
    return l > 0.f ? f / l : (l == l ? 0.f : l);
  };
  auto put_lse = [&](int s, int h, float m, float l) {
    p.lse[(static_cast<long long>(b) * p.H + h) * p.S + s] = l == 0.f ? INFINITY : (m + log2f(l)) * 0.6931471805599453f;
  };
  auto put_row = [&](int s, int h, int col, float m, float l, const float (&f8)[8]) {
    const float inv = finish(h, m, l);
    uint4 v;
    v.x = pack_bf16x2(f8[0] * inv, f8[1] * inv);
    v.y = pack_bf16x2(f8[2] * inv, f8[3] * inv);
    v.z = pack_bf16x2(f8[4] * inv, f8[5] * inv);
    v.w = pack_bf16x2(f8[6] * inv, f8[7] * inv);
    *reinterpret_cast<uint4*>(p.out + b * p.o_sb + s * p.o_ss + h * p.o_sh + col) = v;
    if (p.lse != nullptr && col == 0) put_lse(s, h, m, l);
  };
  if (warp >= Cfg::W_K) {
  if (warp == Cfg::W_K || warp == Cfg::W_V) {
    // ---------------------------------------------------------------- TMA producers of keys (and queries) and of values: one thread
    // of the warp issues (copies issued lane by lane cost 500 clocks each, and one thread for both was the bound of short
    // windows), all look up pages, 32 boxes at a time and a batch ahead
    if (NT > 0) {
      const bool is_k = warp == Cfg::W_K;
      const CUtensorMap* map = is_k ? &tmK : &tmV;
      uint8_t* ring = is_k ? ks : vs;
      uint64_t *full = is_k ? k_full : v_full, *empty = is_k ? k_empty : v_empty;
      int* pages = reinterpret_cast<int*>(ctl + (is_k ? 512 : 768));     // [2 batches][32 boxes]
      const int box_log = __ffs(p.box_k) - 1, box_bytes = p.box_k * 128;     // (a power of two)
      const int per_tile = BN >> box_log, batch = 32 / per_tile;    // boxes of a tile, tiles of a batch of lookups
      const bool paged = p.table != nullptr;
      auto look_up = [&](int i0) {           // the page of this lane's box, of the batch that begins at tile i0
        const int i = i0 + lane / per_tile;
        if (!paged || i >= t1) return 0;
        const WaTile<BN> t(R, i);
        const int j = t.k0 + (lane % per_tile) * p.box_k;
        return j < t.k1() ? p.table[static_cast<long long>(b) * p.table_w + j / p.page] : 0;
      };
      int next = look_up(t0);
      if (is_k && elect_one()) {
        mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(p.box_q * p.g * 128) * COPIES * DB);
        for (int t = 0; t < COPIES; ++t)
          for (int kb = 0; kb < DB; ++kb)
            tma_load_5d(qs + kb * WA_BLK + t * Cfg::COPY_ROWS * 128, &tmQ, q_full, kb * 64, 0, s_first, hk, b);
      }
      WaTile<BN> t(R, t0);
      const int stages = is_k ? NK : NV;
      int kst = 0, kph = 1, row = paged ? t.k0 % p.page : t.k0;     // stage, its phase, row in the page
      for (int i0 = t0, odd = 0; i0 < t1; i0 += batch, odd ^= 32) {
        if (paged) {
          if (next < 0 || next >= p.num_pages) {     // reported, and read as page 0: the copies stay inside the pool
            if (status != nullptr && atomicCAS(status, 0, ST_BAD_ARGUMENT) == 0) {
              status[1] = b;
              status[2] = i0 + lane / per_tile;
              status[3] = next;
            }
            next = 0;
          }
          pages[odd + lane] = next;
          __syncwarp();
          next = look_up(i0 + batch);
        }
        bool ok = true;
        if (elect_one()) {             // (always the same thread)
          const int* page = pages + odd;
          for (int i = i0; i < t1 && i < i0 + batch && ok; ++i) {
            const int boxes = (t.keys() + p.box_k - 1) >> box_log;
            ok = wa_wait(&empty[kst], kph, abort_flag, status, ST_TIMEOUT_EMPTY);
            if (ok) {
              mbar_arrive_expect_tx(&full[kst], static_cast<uint32_t>(boxes * box_bytes) * DB);
              uint8_t* dst = ring + kst * Cfg::STAGE;
              for (int m = 0; m < boxes; ++m) {
                const int outer = paged ? page[m] : b;
#pragma unroll
                for (int kb = 0; kb < DB; ++kb) tma_load_4d(dst + kb * Cfg::KBLK, map, &full[kst], kb * 64, row, hk, outer);
                dst += box_bytes;
                row += p.box_k;
                if (paged && row == p.page) row = 0;
              }
            }
            if (++kst == stages) {
              kst = 0;
              kph ^= 1;
            }
            t.next();
            if (t.left == 0) row = paged ? t.k0 % p.page : t.k0;    // the window's first tile
            page += per_tile;
          }
        }
        if (!__all_sync(0xffffffffu, ok)) break;
      }
    }
  } else if (warp == Cfg::W_S) {
    // ---------------------------------------------------------------- scores (one thread issues).  Scores and products have a thread
    // each: one for both would hold a finished P back behind the scores of two tiles later, because an issuing thread advances no
    // faster than the tensor pipe takes its instructions.
    if (NT > 0 && elect_one()) {
      // one descriptor each, advanced by adding to its address field (16-byte units)
      const uint64_t q_desc = make_smem_desc_sw128(smem_u32(qs), 16, 1024), k_desc = make_smem_desc_sw128(smem_u32(ks), 16, 1024);
      bool ok = wa_wait(q_full, 0, abort_flag, status, ST_TIMEOUT_FULL);
      WaTile<BN> t(R, t0);
      for (int c = 0, stage = 0, phase = 0; c < NT && ok; ++c) {
        const int buf = c & 1;
        const uint32_t idesc_s = make_idesc(128, (t.keys() + 15) & ~15, 1, 1, 0, 0);
        const uint64_t kd = k_desc + static_cast<uint32_t>(stage * (Cfg::STAGE >> 4));
        const uint32_t d = tmem_base + Cfg::S_COL + buf * 64;
        // the scores take the place of an earlier tile's P, once the product has read it
        if (c >= 2 && !wa_wait(&pv_done[buf], ((c >> 1) - 1) & 1, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) break;
        if (!wa_wait(&k_full[stage], phase, abort_flag, status, ST_TIMEOUT_FULL)) break;
        tc_fence_after();
#pragma unroll
        for (int kb = 0; kb < DB; ++kb)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(d, q_desc + ((kb * WA_BLK + k * 32) >> 4), kd + ((kb * Cfg::KBLK + k * 32) >> 4), idesc_s, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit(&k_empty[stage]);
        umma_commit(&s_full[buf]);
        t.next();
        if (++stage == NK) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
  } else {
    // ---------------------------------------------------------------- products: the warp zeroes the rows of V that nobody sees, one
    // thread issues
    constexpr uint32_t idesc_o = make_idesc(128, DB * 64, 1, 1, 0, 1);
    const uint64_t v_desc = make_smem_desc_sw128(smem_u32(vs), Cfg::KBLK, 1024);
    unsigned long long nodes_any = ~0ull;
    if (p.tree != nullptr) {       // which drafted places hold a node
      nodes_any = 0ull;
      const unsigned long long* tree = p.tree + static_cast<long long>(b) * p.tree_sb;
      for (int m = 0; m < p.S; ++m) nodes_any |= tree[m];
    }
    WaTile<BN> t(R, t0);
    for (int c = 0, stage = 0, phase = 0; c < NT; ++c) {
      if (!wa_warp_wait(&v_full[stage], phase, abort_flag, status, ST_TIMEOUT_FULL)) break;
      const int k1 = t.k1();
      const bool tail = k1 - t.k0 < BN, head = t.in_window() && t.k0 < R.wtrue;
      const bool drafted = p.tree != nullptr && k1 > prefix;
      if (tail || head || drafted) {
        for (int r = lane; r < BN; r += 32) {
          const int j = t.k0 + r;
          const bool seen = j < k1 && (j >= R.wtrue || j < p.ns) &&
                            (!drafted || j < prefix || (j - prefix < 64 && ((nodes_any >> (j - prefix)) & 1ull)));
          if (!seen) {
#pragma unroll
            for (int kb = 0; kb < DB; ++kb)
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<uint4*>(vs + stage * Cfg::STAGE + kb * Cfg::KBLK + r * 128 + e * 16) = make_uint4(0, 0, 0, 0);
          }
        }
        fence_proxy_async_smem();
      }
      __syncwarp();
      bool ok = true;
      if (elect_one()) {           // (always the same thread)
        const int buf = c & 1;
        const int k16 = (t.keys() + 15) >> 4;
        const uint64_t vd = v_desc + static_cast<uint32_t>(stage * (Cfg::STAGE >> 4));
        const uint32_t a = tmem_base + Cfg::S_COL + buf * 64;
        ok = wa_wait(&p_full[buf], (c >> 1) & 1, abort_flag, status, ST_TIMEOUT_TMEM_FULL);
        if (ok) {
          tc_fence_after();
          umma_f16_ts(tmem_base, a, vd, idesc_o, c > 0 ? 1u : 0u);
          if (k16 == BN / 16) {
#pragma unroll
            for (int k = 1; k < BN / 16; ++k) umma_f16_ts(tmem_base, a + k * 8, vd + ((k * 2048) >> 4), idesc_o, 1u);
          } else {
            for (int k = 1; k < k16; ++k) umma_f16_ts(tmem_base, a + k * 8, vd + ((k * 2048) >> 4), idesc_o, 1u);
          }
          umma_commit(&v_empty[stage]);
          umma_commit(&pv_done[buf]);
        }
      }
      if (!__all_sync(0xffffffffu, ok)) break;
      t.next();
      if (++stage == NV) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  } else {
    // ---------------------------------------------------------------- softmax and epilogue
    const int quarter = warp, row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_base = tmem_base + lane_addr + Cfg::S_COL, o_addr = tmem_base + lane_addr;
    const int copy = row / Cfg::COPY_ROWS;
    const int rr = row - copy * Cfg::COPY_ROWS;         // row within the tile
    const WindowRow w = window_row(p, rr, s_first, hk, b, klim, prefix);
    constexpr int CW = Cfg::CW, CH = Cfg::CH;
    const int first_key = copy * Cfg::TN;    // of a tile's keys, this thread's TN begin here
    const bool warp_ok = __any_sync(0xffffffffu, w.ok);
    // what every row of the warp sees (rows that are not ok are never read): most tiles need no mask
    const int all_upto = __reduce_min_sync(0xffffffffu, w.ok ? w.plim : 0x7fffffff);
    const int all_from = __reduce_max_sync(0xffffffffu, w.ok ? w.lo : -0x7fffffff);
    float m_ref = -INFINITY, l_sum = 0.f;
    bool ok = true;
    int c = 0;
    {
      auto scores_in = [&](int at) {         // tile `at`: are its scores there?
        return wa_warp_wait(&s_full[at % BUFS], (at / BUFS) & 1, abort_flag, status, ST_TIMEOUT_TMEM_FULL);
      };
      uint32_t x[CH][CW];                    // the scores of this thread's chunks
      // (a short tile's last columns hold anything and are masked; wide: more keys than the first chunk's)
      auto load = [&](int at, bool wide) {
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          if (e > 0 && !wide) continue;
          const uint32_t a = s_base + (at % BUFS) * 64 + first_key + e * CW;
          if constexpr (CW == 32) tmem_ld_x32(a, x[e]);
          else tmem_ld_x16(a, x[e]);
        }
      };
      for (int i = t0; i < t1 && !warp_ok; ++i, ++c) {    // no rows: this warp only keeps step
        if (!scores_in(c)) {
          ok = false;
          break;
        }
        wa_warp_arrive(&p_full[c % BUFS]);
      }
      WaTile<BN> t(R, t0);
      bool wide = CH == 1 || t.keys() > CW;
      if (warp_ok && t0 < t1) {
        ok = scores_in(0);
        tc_fence_after();
        if (ok) load(0, wide);
        tmem_wait_ld();
      }
      for (int i = t0; i < t1 && warp_ok && ok; ++i, ++c) {
        const int buf = c % BUFS;
        const uint32_t s_addr = s_base + buf * 64;
        const int k1 = t.k1();
        const bool whole = k1 - t.k0 == BN && k1 - 1 <= all_upto && (t.k0 >= all_from || k1 <= p.ns);
        if (!whole) {                        // what is masked may be NaN: selected, not added to
#pragma unroll
          for (int e = 0; e < CH; ++e) {
            const unsigned word = window_word(p, w, t.k0 + first_key + e * CW, k1, prefix);
#pragma unroll
            for (int i2 = 0; i2 < CW; ++i2) x[e][i2] = (word >> i2) & 1u ? x[e][i2] : 0xff800000u;
          }
        }
        const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
        float2 acc[2];
        auto probs = [&](int e, float2 neg_m) {
          // P of a chunk takes half its scores' columns, all read by now (the row's lane is this thread's)
          uint32_t w16[CW / 2];
#pragma unroll
          for (int i2 = 0; i2 < CW / 2; ++i2) {
            float2 v = fma2(make_float2(__uint_as_float(x[e][2 * i2]), __uint_as_float(x[e][2 * i2 + 1])), c2, neg_m);
            v.x = exp2f(v.x);
            v.y = exp2f(v.y);
            acc[i2 & 1] = add2(acc[i2 & 1], v);
            w16[i2] = pack_bf16x2(v.x, v.y);
          }
          const uint32_t a = s_addr + (first_key + e * CW) / 2;
          if constexpr (CW == 32) tmem_st_x16(a, w16);
          else tmem_st_x8(a, w16);
        };
        auto tile_sum = [&] {
          // a row without a key yet: exp2(-inf - 0) = 0
          const float2 neg_m = m_ref == -INFINITY ? make_float2(0.f, 0.f) : make_float2(-m_ref, -m_ref);
          acc[0] = acc[1] = make_float2(0.f, 0.f);
#pragma unroll
          for (int e = 0; e < CH; ++e)
            if (e == 0 || wide) probs(e, neg_m);
          return (acc[0].x + acc[0].y) + (acc[1].x + acc[1].y);
        };
        // P, with a reference that rises to the row's largest score so far
        auto lift = [&] {
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int e = 0; e < CH; ++e)
#pragma unroll
            for (int i2 = 0; i2 < CW && (e == 0 || wide); ++i2) m4[i2 & 3] = fmaxf(m4[i2 & 3], __uint_as_float(x[e][i2]));
          const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
          float alpha = 1.f;
          if (mx > m_ref) {
            alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mx);
            m_ref = mx;
            l_sum *= alpha;
          }
          if (c > 0) {
            // O is rescaled when the previous tile's product has completed
            if (!wa_warp_wait(&pv_done[buf ^ 1], ((c - 1) / BUFS) & 1, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int cc = 0; cc < DB * 2; ++cc) {
              uint32_t o[32];
              tmem_ld_x32(o_addr + cc * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tmem_st_x32(o_addr + cc * 32, o);
            }
          }
          return true;
        };
        const bool first_keys = __any_sync(0xffffffffu, w.ok && m_ref == -INFINITY);     // a row without a reference yet
        float sum = 0.f;
        if constexpr (COPIES > 1) {          // few tiles: the first one counts
          bool seek = first_keys;
          for (int pass = 0;; ++pass) {
            if (seek && !(ok = lift())) break;
            sum = tile_sum();
            seek = pass == 0 && __any_sync(0xffffffffu, w.ok && !(sum < WA_FAR));
            if (!seek) break;
          }
        } else {                             // many: the loop without the maximum is straight
          sum = tile_sum();
          if (first_keys || __any_sync(0xffffffffu, w.ok && !(sum < WA_FAR))) {
            ok = lift();
            sum = tile_sum();
          }
        }
        if (!ok) break;
        l_sum += sum;
        const bool more = i + 1 < t1;
        t.next();
        const bool wide_n = CH == 1 || t.keys() > CW;
        if constexpr (COPIES > 1) {          // the other copies' keys count nothing here
          const uint32_t z[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
#pragma unroll
          for (int ch = 0; ch < 4; ++ch)
            if (ch * 16 / Cfg::TN != copy) tmem_st_x8(s_addr + ch * 8, z);
        }
        tmem_wait_st();
        tc_fence_before();
        wa_warp_arrive(&p_full[buf]);
        if (more) {
          if (!scores_in(c + 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          load(c + 1, wide_n);
        }
        tmem_wait_ld();
        wide = wide_n;
      }
      // (the product before the last completes before it: one thread issued both)
      if (c > 0 && ok)
        ok = wa_warp_wait(&pv_done[(c - 1) % BUFS], ((c - 1) / BUFS) & 1, abort_flag, status, ST_TIMEOUT_TMEM_FULL);
      tc_fence_after();
    }
    if (!w.ok) {                             // its scores were never masked: what its query holds (NaN, too) ends here
      m_ref = -INFINITY;
      l_sum = 0.f;
    }
    if constexpr (COPIES == 1) {
      // -------------------------------------------------------------- a thread holds a row; it leaves through the rings, which are
      // free: the last product has completed, and the products read every tile that was fetched
      if (ok) {
        float inv = 1.f;
        const bool in = rr / p.g < p.box_q && w.s < p.S;       // a padding node's row is written too (zeros)
        const long long idx = ((static_cast<long long>(b) * p.S + w.s) * p.H + w.h) * p.splits + split;
        if (p.splits == 1) {
          float l = l_sum;
          inv = in ? finish(w.h, m_ref, l) : 0.f;
          if (p.lse != nullptr && in) put_lse(w.s, w.h, m_ref, l);
        } else if (in) {
          p.ws_ml[idx] = make_float2(m_ref, l_sum);
        }
        const bool any = __any_sync(0xffffffffu, w.ok) && c > 0, have = any && w.ok;
        float* mine = part + row * Cfg::PART_PITCH;
#pragma unroll
        for (int cc = 0; cc < DB * 2; ++cc) {
          uint32_t o[32];
          if (any) {
            tmem_ld_x32(o_addr + cc * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = have ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
          if (p.splits == 1) {
#pragma unroll
            for (int ch = 0; ch < 4; ++ch) {
              uint32_t v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = pack_bf16x2(__uint_as_float(o[8 * ch + 2 * e]), __uint_as_float(o[8 * ch + 2 * e + 1]));
              reinterpret_cast<uint4*>(mine)[cc * 4 + ch] = make_uint4(v[0], v[1], v[2], v[3]);
            }
          } else {
#pragma unroll
            for (int ch = 0; ch < 8; ++ch)
              reinterpret_cast<uint4*>(mine)[cc * 8 + ch] = make_uint4(o[4 * ch], o[4 * ch + 1], o[4 * ch + 2], o[4 * ch + 3]);
          }
        }
        if (p.splits == 1)
          wa_write_rows(reinterpret_cast<const uint8_t*>(part + quarter * 32 * Cfg::PART_PITCH), Cfg::PART_PITCH * 4, p.Dv / 8,
                        p.out + b * p.o_sb + w.s * p.o_ss + w.h * p.o_sh, in);
        else
          wa_write_rows(reinterpret_cast<const uint8_t*>(part + quarter * 32 * Cfg::PART_PITCH), Cfg::PART_PITCH * 4, p.Dv / 4,
                        p.ws_o + idx * p.Dv, in);
      }
    } else {
      // -------------------------------------------------------------- join the copies, then write
      // The rings are free: the last product has completed, and the products read every tile that was fetched.
      if (c == 0) m_ref = -INFINITY;
      xml[row] = make_float2(m_ref, l_sum);
      if (named_bar_and(1, 128, ok)) {
        float top = -INFINITY;
        for (int q = 0; q < COPIES; ++q) top = fmaxf(top, xml[q * Cfg::COPY_ROWS + rr].x);
        const float wt = m_ref > -INFINITY ? exp2f(m_ref - top) : (l_sum == l_sum ? 0.f : l_sum);
        float* mine = part + row * Cfg::PART_PITCH;
#pragma unroll
        for (int cc = 0; cc < DB * 2; ++cc) {
          uint32_t o[32];
          const bool any = __any_sync(0xffffffffu, wt != 0.f);
          if (any) {
            tmem_ld_x32(o_addr + cc * 32, o);
            tmem_wait_ld();
          }
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) {
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
            if (wt != 0.f)
              v = make_float4(__uint_as_float(o[4 * ch]) * wt, __uint_as_float(o[4 * ch + 1]) * wt,
                              __uint_as_float(o[4 * ch + 2]) * wt, __uint_as_float(o[4 * ch + 3]) * wt);
            *reinterpret_cast<float4*>(mine + cc * 32 + ch * 4) = v;
          }
        }
      }
      if (named_bar_and(1, 128, ok)) {
        const int vec = p.Dv / 8;                                  // 16-byte output pieces of a row
        const int rows = min(p.box_q, p.S - s_first) * p.g;
        for (int it = threadIdx.x; it < rows * vec; it += 128) {
          const int r = it / vec, col = (it - r * vec) * 8;
          float top = -INFINITY, l = 0.f, f8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          for (int q = 0; q < COPIES; ++q) top = fmaxf(top, xml[q * Cfg::COPY_ROWS + r].x);
          for (int q = 0; q < COPIES; ++q) {
            const int pr = q * Cfg::COPY_ROWS + r;
            const float2 ml = xml[pr];
            l += ml.x > -INFINITY ? ml.y * exp2f(ml.x - top) : (ml.y == ml.y ? 0.f : ml.y);
            const float4 a = *reinterpret_cast<const float4*>(part + pr * Cfg::PART_PITCH + col);
            const float4 d = *reinterpret_cast<const float4*>(part + pr * Cfg::PART_PITCH + col + 4);
            f8[0] += a.x; f8[1] += a.y; f8[2] += a.z; f8[3] += a.w;
            f8[4] += d.x; f8[5] += d.y; f8[6] += d.z; f8[7] += d.w;
          }
          const int ql = r / p.g, s = s_first + ql, h = hk * p.g + (r - ql * p.g);
          if (p.splits == 1) {
            put_row(s, h, col, top, l, f8);
          } else if (p.joined) {             // in place: no other thread reads these columns of the row
            float4* dst = reinterpret_cast<float4*>(part + r * Cfg::PART_PITCH + col);
            dst[0] = make_float4(f8[0], f8[1], f8[2], f8[3]);
            dst[1] = make_float4(f8[4], f8[5], f8[6], f8[7]);
            if (col == 0) fml[r] = make_float2(top, l);
          } else {
            const long long idx = ((static_cast<long long>(b) * p.S + s) * p.H + h) * p.splits + split;
            float4* dst = reinterpret_cast<float4*>(p.ws_o + idx * p.Dv + col);
            dst[0] = make_float4(f8[0], f8[1], f8[2], f8[3]);
            dst[1] = make_float4(f8[4], f8[5], f8[6], f8[7]);
            if (col == 0) p.ws_ml[idx] = make_float2(top, l);
          }
        }
      }
    }
  }

  if (COPIES > 1 && p.joined) {
    // ---------------------------------------------------------------- the cluster joins its splits, each CTA some pieces of the rows
    __syncwarp();
    cluster_sync_all();
    const int vec = p.Dv / 8;
    const int items = min(p.box_q, p.S - s_first) * p.g * vec;
    for (int it = split * Cfg::THREADS + static_cast<int>(threadIdx.x); it < items; it += p.splits * Cfg::THREADS) {
      const int r = it / vec, col = (it - r * vec) * 8;
      float2 ml[8];
      float4 a[8], d[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        ml[q] = make_float2(-INFINITY, 0.f);
        a[q] = d[q] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (q < p.splits) {
          const float* at = wa_peer(part + r * Cfg::PART_PITCH + col, q);
          ml[q] = *reinterpret_cast<const float2*>(wa_peer(reinterpret_cast<float*>(fml + r), q));
          a[q] = *reinterpret_cast<const float4*>(at);
          d[q] = *reinterpret_cast<const float4*>(at + 4);
        }
      }
      float top = -INFINITY, l = 0.f, f8[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 8; ++q) top = fmaxf(top, ml[q].x);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const float wt = ml[q].x > -INFINITY ? exp2f(ml[q].x - top) : (ml[q].y == ml[q].y ? 0.f : ml[q].y);
        if (wt != 0.f) {
          l = fmaf(ml[q].y, wt, l);
          f8[0] = fmaf(a[q].x, wt, f8[0]); f8[1] = fmaf(a[q].y, wt, f8[1]);
          f8[2] = fmaf(a[q].z, wt, f8[2]); f8[3] = fmaf(a[q].w, wt, f8[3]);
          f8[4] = fmaf(d[q].x, wt, f8[4]); f8[5] = fmaf(d[q].y, wt, f8[5]);
          f8[6] = fmaf(d[q].z, wt, f8[6]); f8[7] = fmaf(d[q].w, wt, f8[7]);
        }
      }
      const int ql = r / p.g;
      put_row(s_first + ql, hk * p.g + (r - ql * p.g), col, top, l, f8);
    }
    cluster_sync_all();          // no CTA's shared memory goes before the others have read it
  }

  // ---------------------------------------------------------------- teardown
  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);   // bounded grace period for copies / MMAs still in flight
  }
  tc_fence_before();
  __syncthreads();
  if (warp == Cfg::W_K) {
    tc_fence_after();
    tmem_dealloc(tmem_base, Cfg::TMEM_COLS);
  }
}

// Joins the splits of a row (sequence, query, head): a block of four warps that share them, four output columns per lane (61 nodes,
// 16 heads, 37 splits: 5.2 us; 13.8 us with one warp).
struct CombineParams {
  int S, H, splits, Dv;
  long long rows;
  const float* ws_o;
  const float2* ws_ml;
  WaSinks sinks;
  __nv_bfloat16* out;
  long long o_sb, o_ss, o_sh;
  float* lse;
};
__global__ void __launch_bounds__(128) window_combine_kernel(const CombineParams p) {
  __shared__ float4 parts[3][32];
  const int warp = threadIdx.x >> 5;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 31;
  const int h = static_cast<int>(row % p.H);
  const long long bs = row / p.H;
  const int s = static_cast<int>(bs % p.S);
  const long long b = bs / p.S;
  // lane i holds the (max, sum) of splits i and i + 32, then their weights; the partial outputs are fetched eight at a time
  const float2* ml = p.ws_ml + row * p.splits;
  const float2 none = make_float2(-INFINITY, 0.f);
  const float2 v0 = lane < p.splits ? ml[lane] : none, v1 = lane + 32 < p.splits ? ml[lane + 32] : none;
  float top = warp_max(fmaxf(v0.x, v1.x));
  const float w0 = v0.x > -INFINITY ? exp2f(v0.x - top) : (v0.y == v0.y ? 0.f : v0.y);
  const float w1 = v1.x > -INFINITY ? exp2f(v1.x - top) : (v1.y == v1.y ? 0.f : v1.y);
  float l = warp_sum((w0 != 0.f ? w0 * v0.y : 0.f) + (w1 != 0.f ? w1 * v1.y : 0.f));
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool in = lane * 4 < p.Dv;
  const float* src = p.ws_o + row * p.splits * p.Dv + lane * 4;
  for (int i0 = 8 * warp; i0 < p.splits; i0 += 32) {
    float4 a[8];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = i0 + i;
      w[i] = __shfl_sync(0xffffffffu, at < 32 ? w0 : w1, at & 31);
      a[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (in && at < p.splits && w[i] != 0.f) a[i] = *reinterpret_cast<const float4*>(src + static_cast<long long>(at) * p.Dv);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      o.x = fmaf(a[i].x, w[i], o.x);
      o.y = fmaf(a[i].y, w[i], o.y);
      o.z = fmaf(a[i].z, w[i], o.z);
      o.w = fmaf(a[i].w, w[i], o.w);
    }
  }
  if (warp > 0) parts[warp - 1][lane] = o;
  __syncthreads();
  if (warp > 0) return;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const float4 a = parts[i][lane];
    o.x += a.x; o.y += a.y; o.z += a.z; o.w += a.w;
  }
  float f = 1.f;
  if (p.sinks.p != nullptr) {
    const float s2 = p.sinks.log2_at(h);
    const float t2 = fmaxf(top, s2);
    if (s2 != -INFINITY) {
      f = top == -INFINITY ? 0.f : exp2f(top - t2);
      l = l * f + exp2f(s2 - t2);
      top = t2;
    }
  }
  const float inv = l > 0.f ? f / l : (l == l ? 0.f : l);
  if (lane * 4 < p.Dv)
    *reinterpret_cast<uint2*>(p.out + b * p.o_sb + s * p.o_ss + h * p.o_sh + lane * 4) =
        make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
  if (p.lse != nullptr && lane == 0) p.lse[(b * p.H + h) * p.S + s] = l == 0.f ? INFINITY : (top + log2f(l)) * 0.6931471805599453f;
}

}  // namespace cmb

namespace cmb_host {

int make_tmap_rows(CUtensorMap* out, const void* base, int D, long long rows, int heads, long long outer, long long s_row,
                   long long s_head, long long s_outer, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return 101;
  bind_context_once();
  if (reinterpret_cast<uintptr_t>(base) & 15) return 102;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads),
                        static_cast<cuuint64_t>(outer)};
  // the stride of a dimension of size 1 is never used, but has to be a positive multiple of 16 bytes
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(rows > 1 ? s_row : 8) * 2, static_cast<cuuint64_t>(heads > 1 ? s_head : 8) * 2,
                           static_cast<cuuint64_t>(outer > 1 ? s_outer : 8) * 2};
  for (int i = 0; i < 3; ++i)
    if (strides[i] == 0 || (strides[i] & 15) || strides[i] >= (1ull << 40)) return 105;
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + static_cast<int>(r);
}

int make_tmap_grouped(CUtensorMap* out, const void* base, int D, int S, int Hk, int g, int Bn, long long s_row, long long s_head,
                      long long s_batch, int box_q) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return 101;
  bind_context_once();
  if (reinterpret_cast<uintptr_t>(base) & 15) return 102;
  cuuint64_t dims[5] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(g), static_cast<cuuint64_t>(S),
                        static_cast<cuuint64_t>(Hk), static_cast<cuuint64_t>(Bn)};
  cuuint64_t strides[4] = {static_cast<cuuint64_t>(g > 1 ? s_head : 8) * 2, static_cast<cuuint64_t>(S > 1 ? s_row : 8) * 2,
                           static_cast<cuuint64_t>(Hk > 1 ? s_head * g : 8) * 2, static_cast<cuuint64_t>(Bn > 1 ? s_batch : 8) * 2};
  for (int i = 0; i < 4; ++i)
    if (strides[i] == 0 || (strides[i] & 15) || strides[i] >= (1ull << 40)) return 105;
  cuuint32_t box[5] = {64, static_cast<cuuint32_t>(g), static_cast<cuuint32_t>(box_q), 1, 1};
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : 1000 + static_cast<int>(r);
}

}  // namespace cmb_host

namespace {

template <int DB, int COPIES>
int launch_window_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const cmb::WindowParams& p, int B,
                      cudaStream_t stream) {
  using Cfg = cmb::WindowCfg<DB, COPIES>;
  auto kern = cmb::window_fwd_kernel<DB, COPIES>;
  static std::atomic<unsigned long long> attr_done{0};
  if (cmb_host::set_smem_limit_once_per_device(attr_done, reinterpret_cast<const void*>(kern), Cfg::SMEM_BYTES)) return 103;
  dim3 grid((p.S + p.box_q - 1) / p.box_q, p.Hk, B * p.splits);
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(Cfg::THREADS);
  config.dynamicSmemBytes = Cfg::SMEM_BYTES;
  config.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim = {1, 1, static_cast<unsigned>(p.splits)};
  config.attrs = &cluster;
  config.numAttrs = p.joined ? 1 : 0;
  return cudaLaunchKernelEx(&config, kern, tq, tk, tv, p) == cudaSuccess ? 0 : 104;
}

}  // namespace

// One call: what its tensors look like, then where they are (host memory, both).
struct cmb_window_call {
  int B, S, T, H, Hk, Dq, Dv, window, ns, cached, tree_sb, table_w, page, num_pages, box_k, splits, sinks_bf16, pad;
  long long q_sb, q_ss, q_sh, k_outer, k_row, k_head, v_outer, v_row, v_head, o_sb, o_ss, o_sh;
  double scale;
};
struct cmb_window_ptrs {
  const void *q, *k, *v, *lengths, *tree, *table, *sinks;
  void *out, *lse, *ws_o, *ws_ml, *status;
};
// q [B,S,H,Dq]; k / v rows [outer, rows, Hk, Dq | Dv] with outer = B (contiguous, rows = T) or pages of a pool (table
// [B, table_w], rows = page size); bf16 with unit inner stride.  Dq, Dv <= 128 and multiples of 8; H / Hk <= 128.  ws_o / ws_ml
// are needed for more than 8 splits, and for 2 or more where S H / Hk > 64.  Returns 0, 1 for arguments that the kernel does not cover.
extern "C" int cmb_window_fwd(const cmb_window_call* call, const cmb_window_ptrs* at, void* stream) {
  const cmb_window_call& a = *call;
  cmb::WindowParams p{};
  const int B = a.B, Dq = a.Dq;
  p.S = a.S; p.T = a.T; p.H = a.H; p.Hk = a.Hk; p.Dv = a.Dv;
  p.window = a.window; p.ns = a.ns; p.cached = a.cached;
  p.tree = static_cast<const unsigned long long*>(at->tree); p.tree_sb = a.tree_sb;
  p.table = static_cast<const int*>(at->table); p.table_w = a.table_w; p.page = a.page; p.num_pages = a.num_pages; p.box_k = a.box_k;
  p.splits = a.splits;
  p.lengths = static_cast<const int*>(at->lengths);
  p.sinks.p = at->sinks; p.sinks.bf16 = a.sinks_bf16;
  if (B <= 0 || p.S <= 0 || p.Hk <= 0 || p.H <= 0 || p.H % p.Hk || p.T < 0 || p.splits < 1 || p.splits > 64) return 1;
  p.g = p.H / p.Hk;
  if (p.g > 128 || p.Hk > 65535 || static_cast<long long>(B) * p.splits > 65535) return 1;
  if (Dq <= 0 || Dq > 128 || Dq % 8 || p.Dv <= 0 || p.Dv > 128 || p.Dv % 8) return 1;
  if (p.window < 1 || p.window > cmb::WA_NO_WINDOW || p.ns < 0 || !(a.scale > 0.)) return 1;
  if (p.cached && (p.lengths == nullptr || p.T < p.S)) return 1;
  if (!p.cached && (p.tree != nullptr || p.table != nullptr || p.T < p.S)) return 1;
  if (p.tree != nullptr && p.S > 64) return 1;
  if (p.box_k != 8 && p.box_k != 16 && p.box_k != 32 && p.box_k != 64) return 1;
  if (p.table != nullptr && (p.page <= 0 || p.page % p.box_k || p.num_pages <= 0 || p.table_w <= 0 ||
                             static_cast<long long>(p.table_w) * p.page < p.T))
    return 1;
  const long long rows = static_cast<long long>(p.S) * p.g;
  p.joined = p.splits > 1 && p.splits <= 8 && rows <= 64;
  if (p.splits > 1 && !p.joined && (at->ws_o == nullptr || at->ws_ml == nullptr)) return 1;
  if ((a.o_sb | a.o_ss | a.o_sh) & 7 || (reinterpret_cast<uintptr_t>(at->out) & 15)) return 1;
  p.box_q = 128 / p.g < p.S ? 128 / p.g : p.S;
  const int copies = rows <= 32 ? 4 : (rows <= 64 ? 2 : 1);
  p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.out = static_cast<__nv_bfloat16*>(at->out); p.o_sb = a.o_sb; p.o_ss = a.o_ss; p.o_sh = a.o_sh;
  p.lse = static_cast<float*>(at->lse);
  p.ws_o = static_cast<float*>(at->ws_o); p.ws_ml = static_cast<float2*>(at->ws_ml);
  p.status = static_cast<int*>(at->status);
  CUtensorMap tq, tk, tv;
  int rc = cmb_host::make_tmap_grouped(&tq, at->q, Dq, p.S, p.Hk, p.g, B, a.q_ss, a.q_sh, a.q_sb, p.box_q);
  if (rc) return rc;
  const long long krows = p.table != nullptr ? p.page : p.T, outer = p.table != nullptr ? p.num_pages : B;
  rc = cmb_host::make_tmap_rows(&tk, at->k, Dq, krows, p.Hk, outer, a.k_row, a.k_head, a.k_outer, p.box_k);
  if (rc) return rc + 10000;
  rc = cmb_host::make_tmap_rows(&tv, at->v, p.Dv, krows, p.Hk, outer, a.v_row, a.v_head, a.v_outer, p.box_k);
  if (rc) return rc + 20000;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool wide = Dq > 64 || p.Dv > 64;
  auto launch = [&](auto db) {
    constexpr int DB = decltype(db)::value;
    switch (copies) {
      case 1: return launch_window_fwd<DB, 1>(tq, tk, tv, p, B, st);
      case 2: return launch_window_fwd<DB, 2>(tq, tk, tv, p, B, st);
      default: return launch_window_fwd<DB, 4>(tq, tk, tv, p, B, st);
    }
  };
  rc = wide ? launch(std::integral_constant<int, 2>{}) : launch(std::integral_constant<int, 1>{});
  if (rc || p.splits == 1 || p.joined) return rc;
  cmb::CombineParams c{};
  c.S = p.S; c.H = p.H; c.splits = p.splits; c.Dv = p.Dv;
  c.rows = static_cast<long long>(B) * p.S * p.H;
  c.ws_o = p.ws_o; c.ws_ml = p.ws_ml; c.sinks = p.sinks;
  c.out = p.out; c.o_sb = p.o_sb; c.o_ss = p.o_ss; c.o_sh = p.o_sh; c.lse = p.lse;
  if (c.rows > 0x7fffffffll) return 1;
  cmb::window_combine_kernel<<<static_cast<unsigned>(c.rows), 128, 0, st>>>(c);
  return cudaGetLastError() == cudaSuccess ? 0 : 104;
}
