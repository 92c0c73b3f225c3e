// Backward of windowed attention (window_attn.cu) on tcgen05: three launches (and a join where the first tokens' keys were
// split), no atomics and no S x T tensor.
//
//   delta_i = do_i . o_i                                     window_stats_kernel
//   P = exp2(S c - lse2),  dS = P o (dO V^T - delta)         recomputed in both of:
//   DKV  CTA = 128 keys of one (sequence, key head); streams the rows that may see them, 64 at a time (64 / g queries x g heads,
//        so a group's heads are summed on chip).  Lanes are keys:  S^T = K Q^T,  dP^T = V dO^T  ->  dV += P^T dO,  dK += dS^T Q
//   DQ   CTA = 128 rows (128 / g queries x g heads); streams the keys that they see, 64 at a time.  Lanes are rows:
//        S = Q K^T,  dP = dO V^T  ->  dQ += dS K
//
// The sinks' gradient, -sum_i p_i,sink (do_i . o_i), would feel the rounding of o to bf16 (the sum has few outputs and both signs), so
// DQ adds up do_i . o_i = sum_j p_ij dP_ij itself, in fp32, where sinks are trained.
//
// dK and dQ carry the softmax scale once, at the end.  P and dS are rounded to bf16 (half a step, 2^-8: the operand type of the
// gradient products) and written back over S and dP in TMEM, where they are the A operands; dQ, dK, dV accumulate there in fp32.
// One thread issues every product in order; two warp groups take alternate sub-tiles, so that one's exponentials run under
// the other's products.  64-wide sub-tiles, because two of {S, dP} and the accumulators have to fit the 512 TMEM columns.
//
// The first tokens are seen by every later row: their key tiles would run S / (64 / g) sub-tiles where another runs about
// (window + 128) / (64 / g).  Their rows are split over CTAs, fp32 partial results are summed in a fixed order by window_join_kernel.
//
// DKV goes first, and DQ's blocks start beside its last ones (a programmatic launch; the two need nothing of each other): DKV has few
// long blocks, 256 where 2 x 4096 queries meet 4 key heads, which keep 148 SMs busy for 86% of two waves.  Forward and backward of
// that call, 16 heads of 128, a window of 1024: 414 -> 388 us; 16384 queries, a window of 2048: 1414 -> 1255 us.
//
// What bounds it: inside a sub-tile the products, 1304 of its 1640 clocks in DKV and 1044 of 1430 in DQ, because those of N = 64 with
// both operands in shared memory run at 70% of the full rate.  Over the whole kernels the pipe multiplies 43% (37%) of the time: the rest is
// that rate, the hand-overs, the blocks' starts and ends, and SMs on which a DQ block that is done waits for the last DKV block.
//
// A key that no row sees may hold anything: K rows of no row of the tile are zeroed in shared memory before dQ's product.
#include "window_attn.h"

namespace cmb {

enum : int { WB_DQ = 0, WB_DKV = 1 };
constexpr int WB_THREADS = 352;            // warps 0-3 / 4-7 elements, 8 TMA, 9 MMA, 10 helper
constexpr int WB_SUB = 64;
constexpr int WB_SBLK = WB_SUB * 128;      // bytes of a [64 rows x 64 bf16] block
constexpr int WB_NS = 4;                   // sub-tiles in flight

struct WindowBwdParams {
  int S, T, H, Hk, g, Dq, Dv;
  int box_q;                               // queries of a 128-row tile (DQ)
  int sub_q;                               // queries of a 64-row sub-tile (DKV)
  float scale, scale_log2;
  int window, ns;
  const int* lengths;
  float2* stats;                           // [B, Hk, S * g] (lse * log2 e, delta) of packed rows; lse = +inf: sees nothing
  __nv_bfloat16 *dq, *dk, *dv;             // DQ's, DKV's results
  long long dq_sb, dq_ss, dq_sh, dk_sb, dk_ss, dk_sh, dv_sb, dv_ss, dv_sh;
  int sink_tiles, sink_splits;             // DKV: the first sink_tiles key tiles are split
  float* part;                             // [B, Hk, sink_tiles, sink_splits, 128, Dq + Dv]
  WaSinks sinks;                           // for SINKS
  float* sink_part;                        // [H, B * row tiles]
  int* status;
};

template <int DB>
struct WindowBwdCfg {
  static constexpr int R_BYTES = 2 * DB * WA_BLK;               // resident pair of operands
  static constexpr int STAGE = 2 * DB * WB_SBLK;
  static constexpr int CTL = 1024 + WB_NS * WB_SUB * 8;        // barriers; row statistics of the stages, then the rows' sums (SINKS)
  static constexpr int SMEM_BYTES = R_BYTES + WB_NS * STAGE + CTL;
  static constexpr int X_COL = 0;                               // buffer i: S at 128 i, dP at 128 i + 64
  static constexpr int O1_COL = 256, O2_COL = 384;
  static_assert(SMEM_BYTES <= 232448, "shared memory");
};

template <int MODE, int DB, bool SINKS>
__global__ void __launch_bounds__(WB_THREADS, 1)
window_bwd_kernel(const __grid_constant__ CUtensorMap tmR1, const __grid_constant__ CUtensorMap tmR2,
                  const __grid_constant__ CUtensorMap tmT1, const __grid_constant__ CUtensorMap tmT2, const WindowBwdParams p) {
  using Cfg = WindowBwdCfg<DB>;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0 && p.status != nullptr && atomicCAS(p.status, 0, ST_BAD_ARGUMENT) == 0) p.status[1] = -1024;
    return;
  }
  uint8_t* r1s = smem;
  uint8_t* r2s = r1s + DB * WA_BLK;
  uint8_t* ts = r2s + DB * WA_BLK;
  uint8_t* ctl = ts + WB_NS * Cfg::STAGE;
  uint64_t* r_full = reinterpret_cast<uint64_t*>(ctl);
  uint64_t* t_full = r_full + 1;             // [WB_NS] landed
  uint64_t* t_ready = t_full + WB_NS;        // [WB_NS] cleaned, row statistics fetched
  uint64_t* t_empty = t_ready + WB_NS;       // [WB_NS] gradient products done
  uint64_t* x_full = t_empty + WB_NS;        // [2] scores
  uint64_t* a_full = x_full + 2;             // [2] P, dS written
  uint64_t* all_done = a_full + 2;           // every product
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(all_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float2* aux = reinterpret_cast<float2*>(ctl + 1024);          // [WB_NS][64]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hk = blockIdx.y, b = blockIdx.z;
  const int off = p.T - p.S;                                    // position of query 0
  const int klim = p.lengths != nullptr ? max(0, min(p.lengths[b], p.T)) : p.T;
  int* status = p.status;

  // ---- what this CTA holds and what it streams
  int row0, n_first, NT, split = -1, key_tile = 0;
  const int xr = static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x);
  const int s_first = MODE == WB_DQ ? xr * p.box_q : 0;         // DQ: the last queries first (without a window they see most)
  const WaRange<64> R(off + s_first, off + min(p.S, s_first + p.box_q) - 1, klim, p.window, p.ns, 1);
  const int used = p.sub_q * p.g;                               // rows of a sub-tile (DKV)
  if (MODE == WB_DQ) {
    row0 = s_first;
    n_first = 0;
    NT = R.n_t;
  } else {
    int part = 0, parts = 1;
    const int x = blockIdx.x, n_split = p.sink_tiles * p.sink_splits;
    if (x < n_split) {
      key_tile = x / p.sink_splits;
      part = x - key_tile * p.sink_splits;
      parts = p.sink_splits;
      split = p.sink_splits > 1 ? part : -1;
    } else {
      key_tile = p.sink_tiles + (x - n_split);
    }
    row0 = key_tile * 128;
    const int k_last = min(row0 + 127, klim - 1);
    const int q_lo = max(0, row0 - off);
    const int q_hi = row0 < p.ns ? p.S : min(p.S, k_last - off + p.window);      // exclusive
    const bool any = k_last >= row0 && q_hi > q_lo;
    const int sub_lo = q_lo / p.sub_q, sub_n = any ? (q_hi + p.sub_q - 1) / p.sub_q - sub_lo : 0;
    const int per = (sub_n + parts - 1) / parts;
    n_first = sub_lo + min(sub_n, part * per);
    NT = min(sub_n, (part + 1) * per) - min(sub_n, part * per);
  }

  if (MODE == WB_DKV) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // DQ's blocks may follow on idle SMs
  if (threadIdx.x == 0) {
    mbar_init(r_full, 1);
    for (int i = 0; i < WB_NS; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_ready[i], 1);
      mbar_init(&t_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&x_full[i], 1);
      mbar_init(&a_full[i], 4);
    }
    mbar_init(all_done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmR1);
    tma_prefetch_desc(&tmR2);
    tma_prefetch_desc(&tmT1);
    tma_prefetch_desc(&tmT2);
  }
  if (MODE == WB_DKV && used < WB_SUB) {     // rows of a sub-tile that no copy fills are multiplied with zeros: no NaN there
    const int rows = WB_SUB - used;
    for (int i = threadIdx.x; i < WB_NS * 2 * DB * rows * 8; i += WB_THREADS) {
      const int c = i & 7, r = (i >> 3) % rows, blk = (i >> 3) / rows;
      *reinterpret_cast<uint4*>(ts + blk * WB_SBLK + (used + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
    fence_proxy_async_smem();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (warp == 8) {
    // ---------------------------------------------------------------- TMA producer
    if (NT > 0 && elect_one()) {
      const uint32_t r_bytes = (MODE == WB_DQ ? p.box_q * p.g : 128) * 128;
      mbar_arrive_expect_tx(r_full, 2 * DB * r_bytes);
      for (int kb = 0; kb < DB; ++kb) {
        if (MODE == WB_DQ) {
          tma_load_5d(r1s + kb * WA_BLK, &tmR1, r_full, kb * 64, 0, row0, hk, b);
          tma_load_5d(r2s + kb * WA_BLK, &tmR2, r_full, kb * 64, 0, row0, hk, b);
        } else {
          tma_load_4d(r1s + kb * WA_BLK, &tmR1, r_full, kb * 64, row0, hk, b);
          tma_load_4d(r2s + kb * WA_BLK, &tmR2, r_full, kb * 64, row0, hk, b);
        }
      }
      const uint32_t t_bytes = (MODE == WB_DQ ? WB_SUB : used) * 128;
      for (int n = 0; n < NT; ++n) {
        const int st = n % WB_NS;
        if (!wa_wait(&t_empty[st], ((n / WB_NS) & 1) ^ 1, abort_flag, status, ST_TIMEOUT_EMPTY)) break;
        mbar_arrive_expect_tx(&t_full[st], 2 * DB * t_bytes);
        uint8_t* t1 = ts + st * Cfg::STAGE;
        uint8_t* t2 = t1 + DB * WB_SBLK;
        for (int kb = 0; kb < DB; ++kb) {
          if (MODE == WB_DQ) {
            const int k0 = WaTile<64>(R, n).k0;
            tma_load_4d(t1 + kb * WB_SBLK, &tmT1, &t_full[st], kb * 64, k0, hk, b);
            tma_load_4d(t2 + kb * WB_SBLK, &tmT2, &t_full[st], kb * 64, k0, hk, b);
          } else {
            tma_load_5d(t1 + kb * WB_SBLK, &tmT1, &t_full[st], kb * 64, 0, (n_first + n) * p.sub_q, hk, b);
            tma_load_5d(t2 + kb * WB_SBLK, &tmT2, &t_full[st], kb * 64, 0, (n_first + n) * p.sub_q, hk, b);
          }
        }
      }
    }
  } else if (warp == 10) {
    // ---------------------------------------------------------------- helper: row statistics, keys that nobody sees
    const long long rows = static_cast<long long>(p.S) * p.g;
    const float2* stats = p.stats + (static_cast<long long>(b) * p.Hk + hk) * rows;
    for (int n = 0; n < NT; ++n) {
      const int st = n % WB_NS;
      float2 v[2];
      if (MODE == WB_DKV) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int c = lane + 32 * i;
          const long long r = static_cast<long long>(n_first + n) * used + c;
          v[i] = c < used && r < rows ? stats[r] : make_float2(INFINITY, 0.f);
        }
      }
      if (!wa_warp_wait(&t_full[st], (n / WB_NS) & 1, abort_flag, status, ST_TIMEOUT_FULL)) break;
      if (MODE == WB_DKV) {
        aux[st * WB_SUB + lane] = v[0];
        aux[st * WB_SUB + 32 + lane] = v[1];
      } else {
        const WaTile<64> t(R, n);
        if (t.keys() < WB_SUB) {
          for (int r = t.keys() + (lane >> 3); r < WB_SUB; r += 4)
#pragma unroll
            for (int kb = 0; kb < DB; ++kb)
              *reinterpret_cast<uint4*>(ts + st * Cfg::STAGE + kb * WB_SBLK + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
      }
      wa_warp_arrive(&t_ready[st]);
    }
  } else if (warp == 9) {
    // ---------------------------------------------------------------- MMA issuer (one thread)
    if (NT > 0 && elect_one()) {
      constexpr uint32_t idesc_x = make_idesc(128, WB_SUB, 1, 1, 0, 0);
      constexpr uint32_t idesc_g = make_idesc(128, DB * 64, 1, 1, 0, 1);
      // descriptors are advanced by adding to their address field (16-byte units)
      const uint64_t r1d = make_smem_desc_sw128(smem_u32(r1s), 16, 1024), r2d = make_smem_desc_sw128(smem_u32(r2s), 16, 1024);
      const uint64_t td = make_smem_desc_sw128(smem_u32(ts), 16, 1024), gd = make_smem_desc_sw128(smem_u32(ts), WB_SBLK, 1024);
      bool ok = wa_wait(r_full, 0, abort_flag, status, ST_TIMEOUT_FULL);
      auto issue_scores = [&](int n) {
        const int st = n % WB_NS, buf = n & 1;
        if (!wa_wait(&t_ready[st], (n / WB_NS) & 1, abort_flag, status, ST_TIMEOUT_FULL)) return false;
        // the buffer holds P and dS of sub-tile n - 2 until its gradient products have read them
        if (n >= 2 && !wa_wait(&t_empty[(n - 2) % WB_NS], ((n - 2) / WB_NS) & 1, abort_flag, status, ST_TIMEOUT_TMEM_EMPTY)) return false;
        tc_fence_after();
        const uint32_t x = tmem_base + Cfg::X_COL + buf * 128;
        const uint64_t t1 = td + static_cast<uint32_t>(st * (Cfg::STAGE >> 4)), t2 = t1 + ((DB * WB_SBLK) >> 4);
#pragma unroll
        for (int kb = 0; kb < DB; ++kb)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(x, r1d + ((kb * WA_BLK + k * 32) >> 4), t1 + ((kb * WB_SBLK + k * 32) >> 4), idesc_x, (kb > 0 || k > 0) ? 1u : 0u);
#pragma unroll
        for (int kb = 0; kb < DB; ++kb)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(x + 64, r2d + ((kb * WA_BLK + k * 32) >> 4), t2 + ((kb * WB_SBLK + k * 32) >> 4), idesc_x, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit(&x_full[buf]);
        return true;
      };
      if (ok) ok = issue_scores(0);
      for (int n = 0; n < NT && ok; ++n) {
        if (n + 1 < NT && !issue_scores(n + 1)) break;
        const int st = n % WB_NS, buf = n & 1;
        if (!wa_wait(&a_full[buf], (n >> 1) & 1, abort_flag, status, ST_TIMEOUT_TMEM_FULL)) break;
        tc_fence_after();
        const uint32_t x = tmem_base + Cfg::X_COL + buf * 128;
        const uint64_t t1 = gd + static_cast<uint32_t>(st * (Cfg::STAGE >> 4)), t2 = t1 + ((DB * WB_SBLK) >> 4);
#pragma unroll
        for (int k = 0; k < WB_SUB / 16; ++k) {
          if (MODE == WB_DKV) umma_f16_ts(tmem_base + Cfg::O2_COL, x + k * 8, t2 + ((k * 2048) >> 4), idesc_g, (n > 0 || k > 0) ? 1u : 0u);
          umma_f16_ts(tmem_base + Cfg::O1_COL, x + 64 + k * 8, t1 + ((k * 2048) >> 4), idesc_g, (n > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(&t_empty[st]);
        if (n == NT - 1) umma_commit(all_done);
      }
    }
  } else {
    // ---------------------------------------------------------------- P, dS and the epilogue
    const int st_id = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t x_addr = tmem_base + lane_addr + Cfg::X_COL + st_id * 128;
    // DQ: this thread's row;  DKV: its key
    const int ql = row / p.g, qi = row0 + ql;
    const int head = hk * p.g + (row - ql * p.g);
    const bool row_ok = MODE == WB_DQ ? (ql < p.box_q && qi < p.S) : (row0 + row < klim);
    float lse2 = INFINITY, delta = 0.f;
    if (MODE == WB_DQ && row_ok) {
      const float2 v = p.stats[(static_cast<long long>(b) * p.Hk + hk) * p.S * p.g + static_cast<long long>(qi) * p.g + (row - ql * p.g)];
      lse2 = v.x;
      delta = v.y;
    }
    const float2 c2 = make_float2(p.scale_log2, p.scale_log2);
    bool ok = true;
    float row_dot = 0.f;                   // SINKS: sum_j p_ij dP_ij over this warp group's keys
    for (int n = st_id; n < NT; n += 2) {
      const int st = n % WB_NS;
      unsigned words[2] = {0u, 0u};
      if (row_ok) {
        if (MODE == WB_DQ) {
          const WaTile<64> t(R, n);
          const int pos = off + qi;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            words[i] = wa_mask_word(t.k0 + 32 * i, min(pos, klim - 1), pos - p.window + 1, p.ns, t.k1());
        } else {     // the columns [lo, hi) of this key: rows at or behind it, inside its window
          const int j = row0 + row, q0 = (n_first + n) * p.sub_q;
          const int first = min(max(j - off - q0, 0), p.sub_q);
          const int last = j < p.ns ? p.sub_q : min(max(j - off - q0 + p.window, 0), p.sub_q);
          const int lo = first * p.g, hi = min(last, p.S - q0) * p.g;
#pragma unroll
          for (int i = 0; i < 2; ++i) words[i] = wa_low_bits(hi - 32 * i) & ~wa_low_bits(lo - 32 * i);
        }
      }
      // (the row statistics came before the scores: their barrier is waited for so that this warp sees them)
      if (!wa_warp_wait(&x_full[st_id], (n >> 1) & 1, abort_flag, status, ST_TIMEOUT_TMEM_FULL) ||
          (MODE == WB_DKV && !wa_warp_wait(&t_ready[st], (n / WB_NS) & 1, abort_flag, status, ST_TIMEOUT_FULL))) {
        ok = false;
        break;
      }
      tc_fence_after();
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t x1[32], x2[32], pw[16], dw[16];
        tmem_ld_x32(x_addr + 32 * i, x1);
        tmem_ld_x32(x_addr + 64 + 32 * i, x2);
        tmem_wait_ld();
        const bool full = __all_sync(0xffffffffu, words[i] == 0xffffffffu);
        const float4* a4 = reinterpret_cast<const float4*>(aux + st * WB_SUB + 32 * i);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float4 a;
          if (MODE == WB_DKV) a = a4[e];
          else a = make_float4(lse2, delta, lse2, delta);
          float2 pr = fma2(make_float2(__uint_as_float(x1[2 * e]), __uint_as_float(x1[2 * e + 1])), c2, make_float2(-a.x, -a.z));
          pr.x = exp2f(pr.x);
          pr.y = exp2f(pr.y);
          float2 d = mul2(pr, add2(make_float2(__uint_as_float(x2[2 * e]), __uint_as_float(x2[2 * e + 1])), make_float2(-a.y, -a.w)));
          if (!full) {      // selected, not multiplied: what is masked may be NaN
            const bool v0 = (words[i] >> (2 * e)) & 1u, v1 = (words[i] >> (2 * e + 1)) & 1u;
            pr.x = v0 ? pr.x : 0.f;
            d.x = v0 ? d.x : 0.f;
            pr.y = v1 ? pr.y : 0.f;
            d.y = v1 ? d.y : 0.f;
          }
          if (SINKS) row_dot += fmaf(pr.x, delta, d.x) + fmaf(pr.y, delta, d.y);
          if (MODE == WB_DKV) pw[e] = pack_bf16x2(pr.x, pr.y);
          dw[e] = pack_bf16x2(d.x, d.y);
        }
        if (MODE == WB_DKV) tmem_st_x16(x_addr + 16 * i, pw);
        tmem_st_x16(x_addr + 64 + 16 * i, dw);
      }
      tmem_wait_st();
      tc_fence_before();
      wa_warp_arrive(&a_full[st_id]);
    }
    if (NT > 0 && ok) ok = wa_warp_wait(all_done, 0, abort_flag, status, ST_TIMEOUT_TMEM_FULL);
    tc_fence_after();
    if (SINKS) {
      // -exp(sink - lse) do.o, summed over the tile's queries for each head
      float* red = reinterpret_cast<float*>(aux);      // [2][128]
      red[st_id * 128 + row] = row_ok ? -exp2f(p.sinks.log2_at(head) - lse2) * row_dot : 0.f;
      if (named_bar_and(1, 256, ok) && threadIdx.x < p.g) {
        float t = 0.f;
        for (int i = threadIdx.x; i < p.box_q * p.g; i += p.g) t += red[i] + red[128 + i];
        p.sink_part[(static_cast<long long>(hk * p.g + threadIdx.x) * gridDim.z + b) * gridDim.x + blockIdx.x] = t;
      }
    }
    if (ok) {
      // DQ: each warp group half of dq's columns;  DKV: dk by the first, dv by the second
      const bool second = MODE == WB_DKV && st_id == 1;
      const int col0 = MODE == WB_DQ ? st_id * DB * 32 : 0;
      constexpr int CHUNKS = MODE == WB_DQ ? DB : 2 * DB;
      const int D = second ? p.Dv : p.Dq;
      const float mul = second ? 1.f : p.scale;
      const bool in = MODE == WB_DQ ? row_ok : row0 + row < p.T;
      __nv_bfloat16* dst = MODE == WB_DQ ? p.dq + b * p.dq_sb + qi * p.dq_ss + head * p.dq_sh + col0
                           : second      ? p.dv + b * p.dv_sb + (row0 + row) * p.dv_ss + hk * p.dv_sh
                                         : p.dk + b * p.dk_sb + (row0 + row) * p.dk_ss + hk * p.dk_sh;
      float* fdst = nullptr;
      if (MODE == WB_DKV && split >= 0)
        fdst = p.part + ((((static_cast<long long>(b) * p.Hk + hk) * p.sink_tiles + key_tile) * p.sink_splits + split) * 128 + row) *
                            (p.Dq + p.Dv) + (second ? p.Dq : 0);
      // through the operands' shared memory, which is free: every product has completed
      constexpr int PITCH = CHUNKS * (MODE == WB_DQ ? 64 : 128) + 16;
      static_assert(8 * 32 * PITCH <= Cfg::R_BYTES + WB_NS * Cfg::STAGE, "rows reuse the operands");
      uint8_t* stage = smem + warp * 32 * PITCH;
      uint4* mine = reinterpret_cast<uint4*>(stage + lane * PITCH);
#pragma unroll
      for (int c = 0; c < CHUNKS; ++c) {
        uint32_t o[32];
        if (NT > 0) {
          tmem_ld_x32(tmem_base + lane_addr + (second ? Cfg::O2_COL : Cfg::O1_COL) + col0 + c * 32, o);
          tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) o[e] = NT > 0 ? __float_as_uint(__uint_as_float(o[e]) * mul) : 0u;
        if (MODE == WB_DKV && fdst != nullptr) {
#pragma unroll
          for (int ch = 0; ch < 8; ++ch) mine[c * 8 + ch] = make_uint4(o[4 * ch], o[4 * ch + 1], o[4 * ch + 2], o[4 * ch + 3]);
        } else {
#pragma unroll
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = pack_bf16x2(__uint_as_float(o[8 * ch + 2 * e]), __uint_as_float(o[8 * ch + 2 * e + 1]));
            mine[c * 4 + ch] = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
      const int cols = min(D - col0, CHUNKS * 32);
      if (MODE == WB_DKV && fdst != nullptr) wa_write_rows(stage, PITCH, cols / 4, fdst, in);
      else wa_write_rows(stage, PITCH, cols / 8, dst, in);
    }
  }

  __syncwarp();
  if (*abort_flag) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
  // Done is done for DKV too: what follows reads both.  This wait comes when the TMEM is back, because a DKV block that shares the SM
  // may still be waiting for it (every block of this DKV is on an SM by now, so the wait needs nothing that this block holds).
  if (MODE == WB_DQ) asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Row statistics for the kernel above: stats[b, hk, s, hg] = (lse log2 e, do.o).  16 lanes to a row (8 columns each).
struct StatsParams {
  int B, S, T, H, g, Dq, Dv, window, ns;
  float scale_log2;
  const int* lengths;
  const __nv_bfloat16 *q, *k, *v;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  const __nv_bfloat16* o;
  const __nv_bfloat16* d;
  long long o_sb, o_ss, o_sh, d_sb, d_ss, d_sh;
  const float* lse;                        // [B, H, S]
  float2* stats;
};
constexpr int WS_ROWS = 64;                // queries of a block (one head)
// Rows that see few keys have an o as large as single values, and dP - delta cancels: there o's rounding would be most of dS's error,
// and delta is sum_j p_ij dP_ij in fp32.  o's rounding (half a step, 2^-8) is 1 / sqrt(keys) of dP's size: with more than 16 keys it
// adds less than a tenth to what dS's own rounding costs.
constexpr int WS_FEW = 16;
__global__ void __launch_bounds__(256, 3) window_stats_kernel(const StatsParams p) {
  const int h = blockIdx.y, b = blockIdx.z, hk = h / p.g, hg = h - hk * p.g, Hk = p.H / p.g;
  const int sub = threadIdx.x >> 4, l16 = threadIdx.x & 15;
  const int s0 = blockIdx.x * WS_ROWS;
  const int klim = p.lengths != nullptr ? max(0, min(p.lengths[b], p.T)) : p.T;
  uint4 a[4], c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = s0 + i * 16 + sub;
    a[i] = c[i] = make_uint4(0, 0, 0, 0);
    if (s < p.S && l16 * 8 < p.Dv) {
      a[i] = *reinterpret_cast<const uint4*>(p.o + b * p.o_sb + s * p.o_ss + h * p.o_sh + l16 * 8);
      c[i] = *reinterpret_cast<const uint4*>(p.d + b * p.d_sb + s * p.d_ss + h * p.d_sh + l16 * 8);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int s = s0 + i * 16 + sub;
    float fa[8], fc[8], sum = 0.f;
    unpack8_bf16(a[i], fa);
    unpack8_bf16(c[i], fc);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fmaf(fa[e], fc[e], sum);
#pragma unroll
    for (int m = 8; m > 0; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    if (s < p.S && l16 == 0) {
      const float lse = p.lse[(static_cast<long long>(b) * p.H + h) * p.S + s];
      p.stats[((static_cast<long long>(b) * Hk + hk) * p.S + s) * p.g + hg] = make_float2(lse * 1.4426950408889634f, sum);
    }
  }
  if (klim == p.T && min(p.T - p.S + s0 + 1, p.window) > WS_FEW) return;       // no such row in most blocks
  // the rows that see few keys, once more: four keys' loads at a time, sums handed round so that lane e + 4 i gets key e's
#pragma unroll 1
  for (int s = s0 + sub; s < min(s0 + WS_ROWS, p.S); s += 16) {
    const int pos = p.T - p.S + s, lo = max(0, pos - p.window + 1);
    const int n1 = min(min(p.ns, lo), klim), n = n1 + max(0, min(pos, klim - 1) - lo + 1);      // keys it sees: first tokens, all
    if (n > WS_FEW) continue;
    const unsigned half = 0xffffu << (16 * (sub & 1));
    const bool in_q = l16 * 8 < p.Dq, in_v = l16 * 8 < p.Dv;
    const float lse2 = p.lse[(static_cast<long long>(b) * p.H + h) * p.S + s] * 1.4426950408889634f;
    uint4 xq = make_uint4(0, 0, 0, 0), xd = xq;
    if (in_q) xq = *reinterpret_cast<const uint4*>(p.q + b * p.q_sb + s * p.q_ss + h * p.q_sh + l16 * 8);
    if (in_v) xd = *reinterpret_cast<const uint4*>(p.d + b * p.d_sb + s * p.d_ss + h * p.d_sh + l16 * 8);
    float fq[8], fd[8], sum = 0.f;
    unpack8_bf16(xq, fq);
    unpack8_bf16(xd, fd);
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 4) {
      uint4 xk[4], xv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e;
        const long long j = i < n1 ? i : lo + (i - n1);
        xk[e] = xv[e] = make_uint4(0, 0, 0, 0);
        if (i < n && in_q) xk[e] = *reinterpret_cast<const uint4*>(p.k + b * p.k_sb + j * p.k_ss + hk * p.k_sh + l16 * 8);
        if (i < n && in_v) xv[e] = *reinterpret_cast<const uint4*>(p.v + b * p.v_sb + j * p.v_ss + hk * p.v_sh + l16 * 8);
      }
      float x[4], dp[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float fk[8], fv[8];
        unpack8_bf16(xk[e], fk);
        unpack8_bf16(xv[e], fv);
        x[e] = dp[e] = 0.f;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          x[e] = fmaf(fq[u], fk[u], x[e]);
          dp[e] = fmaf(fd[u], fv[u], dp[e]);
        }
      }
      auto spread = [&](float (&y)[4]) {
        const bool b0 = l16 & 1, b1 = l16 & 2;
        const float s0 = __shfl_xor_sync(half, b0 ? y[0] : y[1], 1), s1 = __shfl_xor_sync(half, b0 ? y[2] : y[3], 1);
        const float u0 = (b0 ? y[1] : y[0]) + s0, u1 = (b0 ? y[3] : y[2]) + s1;
        float t = (b1 ? u1 : u0) + __shfl_xor_sync(half, b1 ? u0 : u1, 2);
        t += __shfl_xor_sync(half, t, 4);
        return t + __shfl_xor_sync(half, t, 8);
      };
      const float tx = spread(x), td = spread(dp);
      if (i0 + (l16 & 3) < n) sum = fmaf(exp2f(fmaf(tx, p.scale_log2, -lse2)), td, sum);
    }
    sum += __shfl_xor_sync(half, sum, 1);
    sum += __shfl_xor_sync(half, sum, 2);
    if (l16 == 0) p.stats[((static_cast<long long>(b) * Hk + hk) * p.S + s) * p.g + hg].y = sum;
  }
}

// Sums the split key tiles' partial gradients in order: a thread per (sequence, key head, key, 4 columns).
struct JoinParams {
  int T, Hk, Dq, Dv, tiles, splits;
  const float* part;
  __nv_bfloat16 *dk, *dv;
  long long k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;
  long long n;
};
__global__ void __launch_bounds__(256) window_join_kernel(const JoinParams p) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= p.n) return;
  const int vec = (p.Dq + p.Dv) / 4;
  const int col = static_cast<int>(i % vec) * 4;
  long long r = i / vec;
  const int key = static_cast<int>(r % (p.tiles * 128));
  r /= p.tiles * 128;
  const int hk = static_cast<int>(r % p.Hk);
  const long long b = r / p.Hk;
  if (key >= p.T) return;
  const float* src = p.part + ((((b * p.Hk + hk) * p.tiles + key / 128) * p.splits) * 128 + key % 128) * (p.Dq + p.Dv) + col;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int q = 0; q < p.splits; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(src + static_cast<long long>(q) * 128 * (p.Dq + p.Dv));
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  __nv_bfloat16* dst = col < p.Dq ? p.dk + b * p.k_sb + key * p.k_ss + hk * p.k_sh + col
                                  : p.dv + b * p.v_sb + key * p.v_ss + hk * p.v_sh + (col - p.Dq);
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
}

// The sinks' gradient: a warp per head sums its row tiles in a fixed order.
__global__ void __launch_bounds__(32) window_sinks_kernel(const float* part, int n, void* out, int bf16) {
  const float* src = part + static_cast<long long>(blockIdx.x) * n;
  float s = 0.f;
  for (int i = threadIdx.x; i < n; i += 32) s += src[i];
  s = warp_sum(s);
  if (threadIdx.x == 0) {
    if (bf16) static_cast<__nv_bfloat16*>(out)[blockIdx.x] = __float2bfloat16(s);
    else static_cast<float*>(out)[blockIdx.x] = s;
  }
}

}  // namespace cmb

namespace {

template <int MODE, int DB, bool SINKS = false>
int launch_window_bwd(const CUtensorMap (&m)[4], const cmb::WindowBwdParams& p, int gx, int B, cudaStream_t stream, bool beside = false) {
  using Cfg = cmb::WindowBwdCfg<DB>;
  auto kern = cmb::window_bwd_kernel<MODE, DB, SINKS>;
  static std::atomic<unsigned long long> attr_done{0};
  if (cmb_host::set_smem_limit_once_per_device(attr_done, reinterpret_cast<const void*>(kern), Cfg::SMEM_BYTES)) return 103;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(gx, p.Hk, B);
  config.blockDim = dim3(cmb::WB_THREADS);
  config.dynamicSmemBytes = Cfg::SMEM_BYTES;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&config, kern, m[0], m[1], m[2], m[3], p) == cudaSuccess ? 0 : 104;
}

}  // namespace

// One call: what its tensors look like, then where they are (host memory, both).
struct cmb_window_bwd_call {
  int B, S, T, H, Hk, Dq, Dv, window, ns, sink_tiles, sink_splits, sinks_bf16;
  long long q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh, do_sb, do_ss, do_sh;
  long long dq_sb, dq_ss, dq_sh, dk_sb, dk_ss, dk_sh, dv_sb, dv_ss, dv_sh;
  double scale;
};
struct cmb_window_bwd_ptrs {
  const void *q, *k, *v, *o, *dO, *lengths, *sinks, *lse;
  void *dq, *dk, *dv, *dsinks, *stats, *sink_part, *part, *status;
};
// Backward of cmb_window_fwd's contiguous form.  o (the forward's output), dO [B,S,H,Dv]; lse [B,H,S]; dq [B,S,H,Dq],
// dk [B,T,Hk,Dq], dv [B,T,Hk,Dv] bf16 (every element written; dq, or dk and dv together, may be null), dsinks [H] of the sinks' type
// or null.  stats: scratch of 2 B S H floats; sink_part (with dsinks and dq): [H, B * ceil(S / min(S, 128 / (H / Hk)))] floats;
// part: B Hk sink_tiles sink_splits 128 (Dq + Dv) floats where sink_splits > 1.  H / Hk <= 64.
extern "C" int cmb_window_bwd(const cmb_window_bwd_call* call, const cmb_window_bwd_ptrs* at, void* stream) {
  const cmb_window_bwd_call& a = *call;
  const int B = a.B, S = a.S, T = a.T, H = a.H, Hk = a.Hk, Dq = a.Dq, Dv = a.Dv;
  if (B <= 0 || B > 65535 || S <= 0 || T < S || Hk <= 0 || Hk > 65535 || H <= 0 || H > 65535 || H % Hk || H / Hk > 64) return 1;
  if (Dq <= 0 || Dq > 128 || Dq % 8 || Dv <= 0 || Dv > 128 || Dv % 8) return 1;
  if (a.window < 1 || a.window > cmb::WA_NO_WINDOW || a.ns < 0 || !(a.scale > 0.)) return 1;
  if ((a.o_sb | a.o_ss | a.o_sh | a.do_sb | a.do_ss | a.do_sh | a.dq_sb | a.dq_ss | a.dq_sh | a.dk_sb | a.dk_ss | a.dk_sh | a.dv_sb |
       a.dv_ss | a.dv_sh) & 7)
    return 1;
  if (at->dsinks != nullptr && (at->sinks == nullptr || at->dq == nullptr || at->sink_part == nullptr)) return 1;
  const int key_tiles = (T + 127) / 128;
  cmb::WindowBwdParams p{};
  p.S = S; p.T = T; p.H = H; p.Hk = Hk; p.g = H / Hk; p.Dq = Dq; p.Dv = Dv;
  p.box_q = 128 / p.g < S ? 128 / p.g : S;
  p.sub_q = cmb::WB_SUB / p.g;
  p.scale = static_cast<float>(a.scale); p.scale_log2 = static_cast<float>(a.scale * 1.4426950408889634);
  p.window = a.window; p.ns = a.ns; p.lengths = static_cast<const int*>(at->lengths);
  p.stats = static_cast<float2*>(at->stats);
  p.sink_tiles = a.sink_tiles; p.sink_splits = a.sink_splits; p.part = static_cast<float*>(at->part);
  p.status = static_cast<int*>(at->status);
  if (p.sink_tiles < 0 || p.sink_tiles > key_tiles || p.sink_splits < 1 || (p.sink_splits > 1 && at->dk != nullptr && p.part == nullptr))
    return 1;
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  cmb::StatsParams sp{};
  sp.B = B; sp.S = S; sp.T = T; sp.H = H; sp.g = p.g; sp.Dq = Dq; sp.Dv = Dv; sp.window = p.window; sp.ns = p.ns;
  sp.scale_log2 = p.scale_log2; sp.lengths = p.lengths;
  sp.q = static_cast<const __nv_bfloat16*>(at->q); sp.q_sb = a.q_sb; sp.q_ss = a.q_ss; sp.q_sh = a.q_sh;
  sp.k = static_cast<const __nv_bfloat16*>(at->k); sp.k_sb = a.k_sb; sp.k_ss = a.k_ss; sp.k_sh = a.k_sh;
  sp.v = static_cast<const __nv_bfloat16*>(at->v); sp.v_sb = a.v_sb; sp.v_ss = a.v_ss; sp.v_sh = a.v_sh;
  sp.o = static_cast<const __nv_bfloat16*>(at->o); sp.o_sb = a.o_sb; sp.o_ss = a.o_ss; sp.o_sh = a.o_sh;
  sp.d = static_cast<const __nv_bfloat16*>(at->dO); sp.d_sb = a.do_sb; sp.d_ss = a.do_ss; sp.d_sh = a.do_sh;
  sp.lse = static_cast<const float*>(at->lse); sp.stats = p.stats;
  cmb::window_stats_kernel<<<dim3((S + cmb::WS_ROWS - 1) / cmb::WS_ROWS, H, B), 256, 0, st>>>(sp);
  if (cudaGetLastError() != cudaSuccess) return 104;

  const bool wide = Dq > 64 || Dv > 64;
  auto maps = [&](CUtensorMap& mq, CUtensorMap& mo, CUtensorMap& mk, CUtensorMap& mv, int box_q, int box_k) {
    int rc = cmb_host::make_tmap_grouped(&mq, at->q, Dq, S, Hk, p.g, B, a.q_ss, a.q_sh, a.q_sb, box_q);
    if (!rc) rc = cmb_host::make_tmap_grouped(&mo, at->dO, Dv, S, Hk, p.g, B, a.do_ss, a.do_sh, a.do_sb, box_q);
    if (!rc) rc = cmb_host::make_tmap_rows(&mk, at->k, Dq, T, Hk, B, a.k_ss, a.k_sh, a.k_sb, box_k);
    if (!rc) rc = cmb_host::make_tmap_rows(&mv, at->v, Dv, T, Hk, B, a.v_ss, a.v_sh, a.v_sb, box_k);
    return rc;
  };
  CUtensorMap mq, mo, mk, mv;
  if (at->dk != nullptr) {
    if (int rc = maps(mq, mo, mk, mv, p.sub_q, 128)) return rc;
    p.dk = static_cast<__nv_bfloat16*>(at->dk); p.dk_sb = a.dk_sb; p.dk_ss = a.dk_ss; p.dk_sh = a.dk_sh;
    p.dv = static_cast<__nv_bfloat16*>(at->dv); p.dv_sb = a.dv_sb; p.dv_ss = a.dv_ss; p.dv_sh = a.dv_sh;
    const CUtensorMap m[4] = {mk, mv, mq, mo};
    const int gx = key_tiles + p.sink_tiles * (p.sink_splits - 1);
    const int rc = wide ? launch_window_bwd<cmb::WB_DKV, 2>(m, p, gx, B, st) : launch_window_bwd<cmb::WB_DKV, 1>(m, p, gx, B, st);
    if (rc) return rc + 10000;
  }
  if (at->dq != nullptr) {
    if (int rc = maps(mq, mo, mk, mv, p.box_q, cmb::WB_SUB)) return rc;
    p.dq = static_cast<__nv_bfloat16*>(at->dq); p.dq_sb = a.dq_sb; p.dq_ss = a.dq_ss; p.dq_sh = a.dq_sh;
    const CUtensorMap m[4] = {mq, mo, mk, mv};
    const int gx = (S + p.box_q - 1) / p.box_q;
    int rc;
    if (at->dsinks != nullptr) {
      p.sinks.p = at->sinks; p.sinks.bf16 = a.sinks_bf16; p.sink_part = static_cast<float*>(at->sink_part);
      rc = wide ? launch_window_bwd<cmb::WB_DQ, 2, true>(m, p, gx, B, st, at->dk != nullptr) : launch_window_bwd<cmb::WB_DQ, 1, true>(m, p, gx, B, st, at->dk != nullptr);
      if (rc) return rc + 20000;
      cmb::window_sinks_kernel<<<H, 32, 0, st>>>(p.sink_part, B * gx, at->dsinks, a.sinks_bf16);
      if (cudaGetLastError() != cudaSuccess) return 104;
    } else {
      rc = wide ? launch_window_bwd<cmb::WB_DQ, 2>(m, p, gx, B, st, at->dk != nullptr) : launch_window_bwd<cmb::WB_DQ, 1>(m, p, gx, B, st, at->dk != nullptr);
      if (rc) return rc + 20000;
    }
  }
  if (at->dk != nullptr && p.sink_splits > 1 && p.sink_tiles > 0) {
    cmb::JoinParams j{};
    j.T = T; j.Hk = Hk; j.Dq = Dq; j.Dv = Dv; j.tiles = p.sink_tiles; j.splits = p.sink_splits; j.part = p.part;
    j.dk = p.dk; j.k_sb = p.dk_sb; j.k_ss = p.dk_ss; j.k_sh = p.dk_sh;
    j.dv = p.dv; j.v_sb = p.dv_sb; j.v_ss = p.dv_ss; j.v_sh = p.dv_sh;
    j.n = static_cast<long long>(B) * Hk * p.sink_tiles * 128 * ((Dq + Dv) / 4);
    if ((j.n + 255) / 256 > 0x7fffffffll) return 1;
    cmb::window_join_kernel<<<static_cast<unsigned>((j.n + 255) / 256), 256, 0, st>>>(j);
    if (cudaGetLastError() != cudaSuccess) return 104;
  }
  return 0;
}
