// Shared by the forward and backward kernels of windowed attention (window_attn.cu, window_attn_bwd.cu): which keys a query
// sees, and how query rows are packed into tiles.
//
// A row tile holds 128 / g consecutive queries of one key/value head, each with the g query heads that share that head
// (row = query * g + head of the group): grouped heads read a key tile once, and for g > 1 a tile spans few positions, so
// little of a window's edge is masked work.
#pragma once
#include "sm100.cuh"

namespace cmb {

constexpr int WA_BLK = 128 * 128;            // bytes of one [128 rows x 64 bf16] block
constexpr int WA_NO_WINDOW = 1 << 30;

// Sink logits, fp32 or bf16, in log2 units.
struct WaSinks {
  const void* p;                             // [H] or null
  int bf16;
  __device__ __forceinline__ float log2_at(int h) const {
    const float v = bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[h]) : static_cast<const float*>(p)[h];
    return v * 1.4426950408889634f;
  }
};

// The key tiles of a block of rows whose positions lie in [pmin, pmax]: the visible first tokens [0, send), then the window
// [wlo, kend), BN keys a tile.  Keys of the two ranges are disjoint.
template <int BN>
struct WaRange {
  int wtrue;         // first key inside any row's window
  int wlo;           // where the window's tiles start (wtrue rounded down to a whole box of rows)
  int send, kend, n_s, n_t;
  __host__ __device__ WaRange(int pmin, int pmax, int klim, int window, int ns, int align) {
    wtrue = pmin - window + 1;
    if (wtrue < 0) wtrue = 0;
    wlo = wtrue - wtrue % align;
    kend = pmax + 1 < klim ? pmax + 1 : klim;
    if (kend < 0) kend = 0;
    send = ns < wlo ? ns : wlo;
    if (send > klim) send = klim;
    if (send < 0) send = 0;
    n_s = (send + BN - 1) / BN;
    n_t = n_s + (kend > wlo ? (kend - wlo + BN - 1) / BN : 0);
  }
};
// One tile, keys [k0, k1), and the way to the next: a few dependent instructions a step, because the issuing threads walk alone.
template <int BN>
struct WaTile {
  int k0, end;       // end of the range that the tile is in
  int left, wlo, kend;    // tiles of the first range from this one on (<= 0: in the window)
  __host__ __device__ WaTile(const WaRange<BN>& r, int i) : left(r.n_s - i), wlo(r.wlo), kend(r.kend) {
    k0 = left > 0 ? BN * i : r.wlo + BN * (i - r.n_s);
    end = left > 0 ? r.send : r.kend;
  }
  __host__ __device__ int keys() const { return end - k0 < BN ? end - k0 : BN; }
  __host__ __device__ int k1() const { return k0 + keys(); }
  __host__ __device__ bool in_window() const { return left <= 0; }
  __host__ __device__ void next() {
    k0 += BN;
    if (--left == 0) {
      k0 = wlo;
      end = kend;
    }
  }
};

// Bits of the 32 keys j0 .. j0 + 31 that a row sees: j <= plim, and j >= lo (its window) or j < ns (a visible first token),
// and j < k1 (the tile's end; may exceed j0 + 31).
__device__ __forceinline__ unsigned wa_low_bits(int n) {   // the n lowest bits, any n
  return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u);
}
__device__ __forceinline__ unsigned wa_mask_word(int j0, int plim, int lo, int ns, int k1) {
  const unsigned upto = wa_low_bits(min(plim + 1, k1) - j0);
  return upto & (~wa_low_bits(lo - j0) | wa_low_bits(ns - j0));
}

// D[tmem] (+)= A[tmem] * B[smem]; bf16 inputs (A two to a 32-bit column), fp32 accumulate. One thread issues.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// Barrier over `threads` threads that ORs a predicate.
__device__ __forceinline__ bool named_bar_or(int id, int threads, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(out)
      : "r"(id), "r"(threads), "r"(static_cast<uint32_t>(pred))
      : "memory");
  return out != 0;
}
// Waits.  A role's thread is chosen with elect_one(): the compiler then knows that one thread runs, and a product issues in the 33
// to 65 clocks that it takes (44 at the least behind `lane == 0`) and a wait on a completed barrier in 70 clocks (205).  A whole
// warp waits through one of its threads, because 32 polls of a barrier take their turns (140 clocks on a completed one).
__device__ __forceinline__ bool wa_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  return mbar_try_wait(bar, parity) || mbar_wait(bar, parity, abort_flag, status, code);
}
__device__ __forceinline__ bool wa_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  bool ok = true;
  if (elect_one()) ok = wa_wait(bar, parity, abort_flag, status, code);
  ok = __all_sync(0xffffffffu, ok);
  __syncwarp();
  return ok;
}
// Writes the warp's 32 rows of `vec` 16-byte pieces, staged in shared memory `pitch` bytes apart, each to its lane's `to` (rows of lanes
// that are not `in` are left out): whole lines, where every lane writing its own row leaves half of each sector to a second write.
__device__ __forceinline__ void wa_write_rows(const uint8_t* rows, int pitch, int vec, void* to, bool in) {
  if (vec <= 0) return;
  __syncwarp();
  const int lane = threadIdx.x & 31;
  const unsigned rows_in = __ballot_sync(0xffffffffu, in);
  const int row_step = 32 / vec, piece_step = 32 - row_step * vec;
  int r = lane / vec, piece = lane - r * vec;
  for (int e0 = 0; e0 < vec; e0 += 4) {          // (four loads, then their stores)
    uint4 v[4];
    uint4* at[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      at[e] = reinterpret_cast<uint4*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), r & 31)) + piece;
      if (e0 + e >= vec || !((rows_in >> (r & 31)) & 1u)) at[e] = nullptr;
      else v[e] = *reinterpret_cast<const uint4*>(rows + r * pitch + piece * 16);
      r += row_step;
      piece += piece_step;
      if (piece >= vec) {
        piece -= vec;
        ++r;
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (at[e] != nullptr) *at[e] = v[e];
  }
}
__device__ __forceinline__ float* wa_peer(float* mine, int rank) {      // the same place in a cluster CTA's shared memory
  float* at;
  asm("mapa.u64 %0, %1, %2;" : "=l"(at) : "l"(mine), "r"(rank));
  return at;
}
__device__ __forceinline__ void wa_warp_arrive(uint64_t* bar) {      // one arrival for the warp's work so far
  __syncwarp();
  if (elect_one()) mbar_arrive(bar);
}
// Two fp32 operations of one instruction (a pair of registers each).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ void tma_load_5d(void* smem_dst, const CUtensorMap* m, uint64_t* bar, int c0, int c1, int c2, int c3,
                                            int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3),
      "r"(c4)
      : "memory");
}

}  // namespace cmb

namespace cmb_host {

// Key / value rows: [outer, rows, heads, D] with unit inner stride and any other strides that are multiples of 8 elements
// (outer = batch of a contiguous cache, or page of a pool); box of `box_rows` rows x 64 columns.  Columns past D read as 0.
int make_tmap_rows(CUtensorMap* out, const void* base, int D, long long rows, int heads, long long outer, long long s_row,
                   long long s_head, long long s_outer, int box_rows);
// Query-side rows [B, S, H = Hk * g, D] as (D, g, S, Hk, B); box of `box_q` queries x g heads x 64 columns.
int make_tmap_grouped(CUtensorMap* out, const void* base, int D, int S, int Hk, int g, int Bn, long long s_row, long long s_head,
                      long long s_batch, int box_q);

}  // namespace cmb_host
