// Attention over whole prompts with grouped K / V heads: packed sequences of different
// lengths, causal (aligned to the end of the keys) or full, bf16 / f16 in and out, fp32
// accumulation, natural-log lse.  No counterpart in the reference's kernels.
//
//   x_ij = scale q_i.k_j over the keys j <= i + nk - nq of row i's sequence (all keys if not
//   causal);  o_i = sum_j e^(x_ij - lse_i) v_j,  lse_i = log sum_j e^x_ij.
//   A row that sees no key: o = 0, lse = -inf.
//
// One pass over the keys with the running maximum and sum of a softmax (one thread per row).
// A work item is one K / V head and up to two 128-row query tiles; the rows of a tile are
// (token, head of the group) pairs, so all query heads of a group share each K / V tile and
// the keys of a tile's last token bound its key range.  One block per SM, 384 threads:
//   warps 0-3, 4-7  softmax, output and lse of query tile 0 and 1 (thread = row = TMEM lane)
//   warp 8          TMA: query tiles, K and V tiles into one ring of slots
//   warp 9          TMEM and the MMA-issuing thread
//   warp 10         scheduler: next work items (the grid holds one block per item; a running
//                   block cancels blocks that have not started and takes their items), the
//                   longest key ranges first
//   warp 11         repairs V tiles that reach past what some row sees: a NaN or infinity there
//                   would reach that row as 0 * v.  Such values are taken out of the tile; the
//                   rows that do see them add them in the epilogue.
// The two query tiles take turns on the tensor cores: QK_0(j+1) is issued behind PV_0(j), so
// one tile's products run while the other's exponentials do.  S and P of a tile share 128 TMEM
// columns (P overwrites S), O takes D; a row's O is rescaled only when its maximum has grown
// by more than 2^8 (2^7 for f16; fp32 sums lose nothing by waiting).  A weight is rounded once, to V's type, for
// the product (both operands of an MMA have one type, and a second product with what is left would add
// half of the step's tensor time, which bounds it); the row's sum takes the unrounded ones.  o is within
// u sum_j p_j |v_j| of the 32-bit form, u = 2^-8 or 2^-11.
// Where few rows meet many keys, an item's key range is cut into parts that a second kernel joins
// (16 tokens on 30000 keys, 32 heads on 8: 345 us in one part, 48 us in 18).
//
// Measured (B200): one prompt of 16384 tokens, 16 heads on 2, D = 128, in 0.79-0.81 ms = 1360-1390
// TFLOP/s alone (1690 is a cuBLAS burst), 0.94 ms = 1170 TFLOP/s back to back at the 1 kW power cap
// (1410 is cuBLAS there); nine prompts of 1 to 2047 tokens, 32 heads on 8, in 128-132 us = 960-990
// TFLOP/s.  A
// step (two 128 x 128 tiles) takes ~3100 cycles: 2048 are the tensor cores' (66 % active), 1792 the
// exponential unit's (58 %); the rest is the chain of a tile, scores -> maximum -> exponentials ->
// weights -> product -> next scores, which two tiles in turns do not hide in full.  What was tried
// against it and was slower or no better: a thread for half a row (with an exchange of the maxima),
// weights against the maximum of the tile before, one issuing thread for each tile (they fall into
// step and fight for the exponential unit), more of the exponentials on the FMA pipe.
#include "gqa_items.cuh"
#include "gqa_softmax.cuh"
#include "tc.cuh"

namespace mzb {
namespace gqa {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

template <int D>
struct PCfg {
  static constexpr int DB = (D + 63) / 64;  // 64-channel column blocks (D = 96: the last half is zero fill)
  static constexpr int Q_BYTES = DB * 128 * 128;
  static constexpr int SLOT = DB * BN * 128;
  static constexpr int NS = DB == 1 ? 8 : 4;  // ring slots (K and V tiles alternate)
  static constexpr int STAGE = 2 * Q_BYTES + NS * SLOT;  // output staging: 4 KB for each softmax warp
  static constexpr int TILES = STAGE + 8 * 4096;
  static constexpr int SMEM = TILES + 1024;
  // TMEM columns.  D = 64 has room for P beside S: S is free for the next QK^T as soon as the softmax
  // has read it, so the products leave the softmax's chain (SEP).  Else P takes S's place, 64 keys
  // in the front of each half of it, and QK_t(j+1) follows PV_t(j).
  static constexpr bool SEP = D == 64;
  static constexpr int S_COL = 0;                           // + 128 t
  static constexpr int P_COL = SEP ? 256 : 0, P_TILE = SEP ? 64 : 128, P_HALF = SEP ? 32 : 64;
  static constexpr int O_COL = SEP ? 384 : 256, O_TILE = SEP ? 64 : 128;
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct PrefillArgs : ItemArgs {
  const void* v;
  void* o;
  float* lse;
  int64_t sv_t, sv_h;
  int Hq, Hkv, g, neg;  // g = Hq / Hkv
  float sl;             // |scale| log2 e
  int* err;
  float *plse, *po;     // of cut key ranges: [splits, Tq * Hq], [splits, Tq * Hq, D]
};

enum PBar { P_QF = 0, P_QE = 2, P_SF = 4, P_PF = 6, P_OF = 10, P_OE = 12, P_ITF = 14, P_ITE = 16, P_CLC = 18, P_ASK = 19,
            P_KF = 20, P_KE = P_KF + 8, P_VOK = P_KE + 8, P_SE = P_VOK + 8, P_PE = P_SE + 2, P_NBAR = P_PE + 2 };
constexpr int ITEM_READERS = 8 + 3;  // softmax warps, TMA, MMA, repair

__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Maxima that a NaN passes through.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// 2^x of a pair on the FMA pipe, 0 for x <= -127 (a masked -inf): x = n + f with f in
// [-1/2, 1/2] (adding 1.5 2^23 rounds to nearest), 2^f by the degree-4 polynomial of least
// maximal relative error (2.6e-6, found by Remez exchange), times 2^n built in the exponent field.
__device__ __forceinline__ float2 poly_exp2(uint64_t x2) {
  const float2 xc = unpack_f32x2(x2);
  const uint64_t x = pack_f32x2(fmaxf(xc.x, -127.0f), fmaxf(xc.y, -127.0f));
  const uint64_t t = add_f32x2(x, pack_f32x2(12582912.0f, 12582912.0f));
  const uint64_t r = add_f32x2(t, pack_f32x2(-12582912.0f, -12582912.0f));
  const uint64_t f = ffma_f32x2(r, pack_f32x2(-1.0f, -1.0f), x);
  uint64_t p = ffma_f32x2(f, pack_f32x2(9.570101911e-03f, 9.570101911e-03f),
                          pack_f32x2(5.591786032e-02f, 5.591786032e-02f));
  p = ffma_f32x2(p, f, pack_f32x2(2.402474483e-01f, 2.402474483e-01f));
  p = ffma_f32x2(p, f, pack_f32x2(6.931218147e-01f, 6.931218147e-01f));
  p = ffma_f32x2(p, f, pack_f32x2(9.999992614e-01f, 9.999992614e-01f));
  const float2 tn = unpack_f32x2(t);
  return unpack_f32x2(mul_f32x2(p, pack_f32x2(__uint_as_float((__float_as_uint(tn.x) << 23) + 0x3f800000u),
                                              __uint_as_float((__float_as_uint(tn.y) << 23) + 0x3f800000u))));
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == MZB_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// Larger magnitude of the halves of m and w; a NaN passes through.
template <int DT>
__device__ __forceinline__ uint32_t maxabs2(uint32_t m, uint32_t w) {
  if constexpr (DT == MZB_BF16) {
    const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&m),
                                         __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&w)));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
// Bits set where a 16-bit half of w is NaN or infinite (exponent all ones).
template <int DT>
__device__ __forceinline__ uint32_t nonfinite2(uint32_t w) {
  constexpr uint32_t E = DT == MZB_BF16 ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}

// ---------------------------------------------------------------- kernel

// CUT: items may be parts of a key range (compiled apart: its registers and branches would cost the
// calls without parts 2-4 %).
template <int DT, int D, bool CUT>
__global__ void __launch_bounds__(384, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                   const __grid_constant__ CUtensorMap tv, const __grid_constant__ PrefillArgs a) {
  using C = PCfg<D>;
  using T = typename Elem<DT>::T;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* qs = smem;
  uint8_t* ring = smem + 2 * C::Q_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::TILES);
  Item* items = reinterpret_cast<Item*>(smem + C::TILES + 8 * P_NBAR + 16);  // [2]
  uint4* clc = reinterpret_cast<uint4*>(smem + C::TILES + 512);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::TILES + 544);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::TILES + 548);
  volatile int* bad_v = reinterpret_cast<volatile int*>(smem + C::TILES + 552);  // [4] by item number
  static_assert(8 * P_NBAR + 16 + 2 * sizeof(Item) <= 512, "misc layout");
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) atomicExch(a.err, MZB_ERR_ALIGN);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < P_NBAR; ++i) {
      uint32_t c = 1;
      if ((i >= P_PF && i < P_PF + 4) || i == P_SE || i == P_SE + 1) c = 4;
      if (i == P_OE || i == P_OE + 1) c = 4;
      if (i == P_ITE || i == P_ITE + 1) c = ITEM_READERS;
      if (i >= P_KE && i < P_KE + 8) c = 2;  // the last product that reads the slot; the repair warp
      tc::mbar_init(&bars[i], c);
    }
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (warp == 9) tc::tmem_alloc(tmem_slot, 512);
  if (warp == 8 && lane == 0) {
    tc::prefetch_tmap(&tq);
    tc::prefetch_tmap(&tk);
    tc::prefetch_tmap(&tv);
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  if constexpr (CUT) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // a wait that the whole warp agrees on; false: it (or another role) gave up
  auto wait_all = [&](int bar, uint32_t parity, int code) -> bool {
    const bool got = !*abort_flag && tc::mbar_wait(&bars[bar], parity, a.err, code);
    if (__all_sync(0xffffffffu, got)) return true;
    *abort_flag = 1;
    return false;
  };
  // next item: every reader copies it and lets the slot go (the whole warp calls)
  int itn = 0;
  auto next_item = [&](Item& m) -> bool {
    const int s = itn & 1;
    if (!wait_all(P_ITF + s, (itn >> 1) & 1, 401)) return false;
    m = items[s];
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(&bars[P_ITE + s]);
    ++itn;
    return !m.done;
  };
  Item m;

  // registers: 384 x 168 at launch (the host checks it) = 256 x 208 (softmax) + 128 x 88
  if (warp < 8) {
    // ---------------------------------------------------------------- softmax, output
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, sw = warp & 3, r = sw * 32 + lane;
    const uint32_t scol = tc::taddr(tmem, sw * 32, C::S_COL + 128 * t), ocol = tc::taddr(tmem, sw * 32, C::O_COL + C::O_TILE * t);
    const uint32_t pcol = tc::taddr(tmem, sw * 32, C::P_COL + C::P_TILE * t);
    const int rtok = r / a.g, rhead = r % a.g;
    uint32_t ns = 0, no = 0;
    while (next_item(m)) {
      const int par = (itn - 1) & 3;
      const int tok = m.tok0 + t * a.ntok + rtok, i = m.i0 + t * a.ntok + rtok;
      const bool row_ok = rtok < a.ntok && tok < m.tok_end;
      const int lim = row_ok ? max(0, min(m.nk, i + m.shift)) : 0x3fffffff;  // keys that this row sees
      const int n = t ? m.n1 : m.n0;
      float ms = 0.0f, mx = -INFINITY, lsum = 0.0f;  // the weights' reference, running maximum (log2 domain), sum
      bool ok = true;
      for (int j = 0; j < n; ++j, ++ns) {
        if (!__all_sync(0xffffffffu, tc::mbar_wait(&bars[P_SF + t], ns & 1, a.err, 409))) {
          *abort_flag = 1;
          ok = false;
          break;
        }
        tc::fence_after_sync();
        const int vis = lim - j * BN;  // columns below this are seen
        if (!__all_sync(0xffffffffu, vis >= BN)) {
          // masked scores to -inf where they lie (a rolled loop: tiles like this are few, and long
          // unrolled code that runs once an item is fetched anew each time)
#pragma unroll 1
          for (int c0 = 0; c0 < BN; c0 += 32) {
            if (__all_sync(0xffffffffu, vis >= c0 + 32)) continue;
            uint32_t x[32];
            tc::tmem_ld32(scol + c0, x);
            tc::tmem_wait_ld();
            tc::reg_after_wait(x);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e >= vis - c0) x[e] = 0xff800000u;
            tc::tmem_st32(scol + c0, x);
          }
          tc::tmem_wait_st();
        }
        uint32_t sv[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) tc::tmem_ld32(scol + 32 * q, sv[q]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int q = 0; q < 4; ++q) tc::reg_after_wait(sv[q]);
        if constexpr (C::SEP) {  // the next scores may come
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&bars[P_SE + t]);
        }
        float m4[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          m4[q] = max3(__uint_as_float(sv[q][0]), __uint_as_float(sv[q][1]), __uint_as_float(sv[q][2]));
#pragma unroll
          for (int e = 3; e < 31; e += 2) m4[q] = max3(m4[q], __uint_as_float(sv[q][e]), __uint_as_float(sv[q][e + 1]));
          m4[q] = max2(m4[q], __uint_as_float(sv[q][31]));
        }
        // a NaN or +infinite score makes the row NaN: through the maximum, since the polynomial
        // exponential does not carry one
        float mt = max2(max2(m4[0], m4[1]), max2(m4[2], m4[3])) * a.sl;
        mt = mt < INFINITY ? mt : NAN;
        const bool need = !(mt <= mx + Running<DT>::GROW);
        bool behind = C::SEP && j > 0;  // the previous PV may still read P and add to O
        auto after_pv = [&]() {
          if (!behind) return true;
          behind = false;
          const bool got = wait_all(P_PE + t, (ns - 1) & 1, 416);
          tc::fence_after_sync();
          return got;
        };
        if (__any_sync(0xffffffffu, need)) {
          if (!after_pv()) { ok = false; break; }
          const float mn = need ? mt : mx;
          const float alpha = need ? fast_exp2(Running<DT>::relative(mx) - Running<DT>::relative(mn)) : 1.0f;
          mx = mn;
          lsum *= alpha;
          ms = Running<DT>::reference(mx);
          if (j > 0) {  // (not SEP: S_FULL was committed behind the previous PV, so O is complete)
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              uint32_t ov[32];
              tc::tmem_ld32(ocol + c0, ov);
              tc::tmem_wait_ld();
              tc::reg_after_wait(ov);
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tc::tmem_st32(ocol + c0, ov);
            }
          }
        }
        const uint64_t sl2 = pack_f32x2(a.sl, a.sl), nm2 = pack_f32x2(-ms, -ms);
        uint64_t acc[2] = {0, 0};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const uint64_t x = ffma_f32x2(pack_f32x2(__uint_as_float(sv[q][2 * e]), __uint_as_float(sv[q][2 * e + 1])), sl2, nm2);
            float2 p;
            // one pair in eight on the FMA pipe.  With 0, 1/8, 1/4, 3/8, 1/2 of them: a prompt of 16384, 16 heads on 2, D = 128
            // 814, 803, 818, 818, 877 us; D = 96 746, 745, 790, 746, 806; two f16 chunks, 24 on 4, D = 64 100, 97, 100, 103, 110
            if (e % 8 == 7) {
              p = poly_exp2(x);
            } else {
              const float2 xf = unpack_f32x2(x);
              p = make_float2(fast_exp2(xf.x), fast_exp2(xf.y));
            }
            acc[e & 1] = add_f32x2(acc[e & 1], pack_f32x2(p.x, p.y));
            pk[e] = pack2<DT>(p.x, p.y);
          }
          if (q == 0 && !after_pv()) { ok = false; break; }
          tc::tmem_st16(pcol + C::P_HALF * (q >> 1) + 16 * (q & 1), pk);
          if (q & 1) {  // 64 keys' weights: their product can start
            tc::tmem_wait_st();
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bars[P_PF + 2 * t + (q >> 1)]);
          }
        }
        if (!ok) break;
        const float2 s0 = unpack_f32x2(add_f32x2(acc[0], acc[1]));
        lsum += s0.x + s0.y;
      }
      if (!ok) break;
      const int64_t row = (int64_t)tok * a.Hq + m.hk * a.g + rhead;
      const bool cut = CUT && m.of > 1;  // into the workspace, in 32 bits
      float* prow = cut ? a.po + ((int64_t)m.part * a.Tq * a.Hq + row) * D : nullptr;
      float* lse_at = cut ? a.plse + (int64_t)m.part * a.Tq * a.Hq + row : a.lse + row;
      if (n == 0) {  // no row of this tile sees a key
        if (row_ok && cut) {
          *lse_at = -INFINITY;  // the part's output is not read
        } else if (row_ok) {
          uint4* mine = reinterpret_cast<uint4*>(static_cast<T*>(a.o) + row * D);
#pragma unroll 1
          for (int c = 0; c < D / 8; ++c) mine[c] = make_uint4(0, 0, 0, 0);
          a.lse[row] = -INFINITY;
        }
        continue;
      }
      if (!wait_all(P_OF + t, no & 1, 410)) break;
      ++no;
      tc::fence_after_sync();
      const bool bad = bad_v[par] != 0;
      const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;  // a row without keys or with scores of -inf alone: O is 0
      // through shared memory, 32 channels at a time, so that a store covers 64 bytes of each of eight
      // rows (a thread storing its own row touches 32 lines an instruction: ~4000 cycles an item);
      // the 16-byte pieces of a row at its place mod 8 keep both directions free of conflicts
      uint8_t* stage = smem + C::STAGE + warp * 4096;
      T* orow[4];  // this lane's rows of the four stores of a block: 8 i + lane / 4
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const int64_t at = __shfl_sync(0xffffffffu, row_ok ? row : -1, 8 * i4 + (lane >> 2));
        orow[i4] = at < 0 ? nullptr : static_cast<T*>(a.o) + at * D + 8 * (lane & 3);
      }
      uint8_t* st_at = stage + lane * 64;
      const uint8_t* ld_at = stage + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) * 16);
      const uint64_t inv2 = pack_f32x2(inv, inv);
      constexpr int CB = D % 64 ? 1 : 2;  // blocks of 32 channels in flight
      if (CUT && cut) {  // the part's numbers in fp32, the same way: 128 bytes of four rows a store
        int at[8];  // this lane's rows of a block's stores: 4 i + lane / 8
#pragma unroll
        for (int i = 0; i < 8; ++i) at[i] = __shfl_sync(0xffffffffu, row_ok ? int(row) : -1, 4 * i + (lane >> 3));
        float* part = prow - row * D + 4 * (lane & 7);
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          uint32_t ov[32];
          tc::tmem_ld32(ocol + c0, ov);
          tc::tmem_wait_ld();
          tc::reg_after_wait(ov);
#pragma unroll
          for (int c = 0; c < 8; ++c)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((c ^ (lane & 7)) * 16)) =
                make_float4(__uint_as_float(ov[4 * c]) * inv, __uint_as_float(ov[4 * c + 1]) * inv,
                            __uint_as_float(ov[4 * c + 2]) * inv, __uint_as_float(ov[4 * c + 3]) * inv);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            const float4 x = *reinterpret_cast<const float4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) * 16));
            if (at[i] >= 0) *reinterpret_cast<float4*>(part + (int64_t)at[i] * D + c0) = x;
          }
          __syncwarp();
        }
      }
#pragma unroll 1
      for (int c0 = cut ? D : 0; c0 < D; c0 += 32 * CB) {
        uint32_t ov[CB][32];
#pragma unroll
        for (int b = 0; b < CB; ++b) tc::tmem_ld32(ocol + c0 + 32 * b, ov[b]);
        tc::tmem_wait_ld();
#pragma unroll
        for (int b = 0; b < CB; ++b) {
          tc::reg_after_wait(ov[b]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 x = unpack_f32x2(mul_f32x2(
                  pack_f32x2(__uint_as_float(ov[b][8 * c + 2 * e]), __uint_as_float(ov[b][8 * c + 2 * e + 1])), inv2));
              w[e] = pack2<DT>(x.x, x.y);
            }
            *reinterpret_cast<uint4*>(st_at + 2048 * b + ((c ^ ((lane >> 1) & 3)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        __syncwarp();
        uint4 x[CB][4];
#pragma unroll
        for (int b = 0; b < CB; ++b)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) x[b][i4] = *reinterpret_cast<const uint4*>(ld_at + 2048 * b + 512 * i4);
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4)
          if (orow[i4]) {
#pragma unroll
            for (int b = 0; b < CB; ++b) *reinterpret_cast<uint4*>(orow[i4] + c0 + 32 * b) = x[b][i4];
          }
        __syncwarp();
      }
      if (bad && row_ok) {  // values taken out of the repaired tiles, for the rows that see them
        T* mine = static_cast<T*>(a.o) + row * D;
#pragma unroll 1
        for (int k = m.jfix * BN; k < lim; ++k) {
          const T* vr = static_cast<const T*>(a.v) + (int64_t)(m.k0 + k) * a.sv_t + m.hk * a.sv_h;
#pragma unroll 1
          for (int e = 0; e < D; ++e) {
            const float x = Elem<DT>::load(vr[e]);
            if (isfinite(x)) continue;
            if (cut) prow[e] += x; else mine[e] = Elem<DT>::store(Elem<DT>::load(mine[e]) + x);
          }
        }
      }
      if (row_ok) *lse_at = lim > 0 ? (Running<DT>::relative(mx) + log2f(lsum)) * LN2 : -INFINITY;
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bars[P_OE + t]);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8) {
      // ---------------------------------------------------------------- TMA
      uint32_t g = 0, nq[2] = {0, 0};
      const uint32_t qbytes = uint32_t(C::DB) * 128 * a.g * a.ntok;
      while (next_item(m)) {
        if (tc::elect_one()) {
        const int n = max(m.n0, m.n1);
        bool ok = true;
        auto load_q = [&](int t) {
          if ((t ? m.n1 : m.n0) == 0) return;
          if (!tc::mbar_wait(&bars[P_QE + t], (nq[t] & 1) ^ 1, a.err, 402)) { ok = false; return; }
          ++nq[t];
          tc::mbar_expect_tx(&bars[P_QF + t], qbytes);
#pragma unroll
          for (int cb = 0; cb < C::DB; ++cb)
            tc::tma_load_3d(qs + t * C::Q_BYTES + cb * 128 * 128, &tq, &bars[P_QF + t], cb * 64, m.hk * a.g,
                            m.tok0 + t * a.ntok);
        };
        auto load_kv = [&](const CUtensorMap* map, int j) {
          const uint32_t s = g % C::NS;
          if (!tc::mbar_wait(&bars[P_KE + s], ((g / C::NS) & 1) ^ 1, a.err, 403)) { ok = false; return; }
          tc::mbar_expect_tx(&bars[P_KF + s], C::SLOT);
#pragma unroll
          for (int cb = 0; cb < C::DB; ++cb)
            tc::tma_load_3d(ring + s * C::SLOT + cb * BN * 128, map, &bars[P_KF + s], cb * 64, m.hk, m.k0 + j * BN);
          ++g;
        };
        const int ask = max(0, n - 3);  // the next item is bound late, or the last blocks' shares are uneven
        load_q(0);
        for (int j = 0; j < n && ok; ++j) {
          load_kv(&tk, j);
          if (j == 0 && ok) load_q(1);
          if (ok) load_kv(&tv, j);
          if (j == ask) tc::mbar_arrive(&bars[P_ASK]);
        }
        if (n == 0) tc::mbar_arrive(&bars[P_ASK]);
        if (!ok) *abort_flag = 1;
        }
        __syncwarp();
      }
      // a wait gave up: no copy is left in flight when the block ends (the ring's slots, from the one that is next, and
      // the query tiles; of a barrier that was not used yet phase -1 has passed)
      if (*abort_flag && tc::elect_one()) {
#pragma unroll 1
        for (uint32_t x = 0; x < C::NS + 2; ++x) {
          const uint32_t fills = x < C::NS ? (g + x) / C::NS : x == C::NS ? nq[0] : nq[1];
          tc::mbar_wait(&bars[x < C::NS ? P_KF + (g + x) % C::NS : P_QF + x - C::NS], (fills & 1) ^ 1, a.err, 418);
        }
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------------- MMA issue
      const uint32_t fmt = DT == MZB_BF16 ? 1 : 0;
      // a negative scale: the scores of -q (negate-A bit), so that larger is always more
      const uint32_t idesc_qk = tc::make_idesc(128, BN, fmt, fmt) | (a.neg ? 1u << 13 : 0u);
      const uint32_t idesc_pv = tc::make_idesc(128, D, fmt, fmt, false, true);
      const uint32_t q_base = smem_u32(qs), r_base = smem_u32(ring);
      uint32_t g = 0, nq[2] = {0, 0}, np[2] = {0, 0}, se[2] = {0, 0}, vok = 0;
      bool k_seen[2];
      while (next_item(m)) {
        if (tc::elect_one()) {
        const int nt[2] = {m.n0, m.n1}, n = max(m.n0, m.n1);
        bool ok = true;
        auto full = [&](uint32_t gg) {
          if (!tc::mbar_wait(&bars[P_KF + gg % C::NS], (gg / C::NS) & 1, a.err, 404)) ok = false;
        };
        auto qk = [&](int t, int j, uint32_t gk) {  // S_t = Q_t K_j^T
          const uint64_t qd = tc::make_sdesc<128>(q_base + t * C::Q_BYTES, 16, 1024);
          const uint64_t kd = tc::make_sdesc<128>(r_base + (gk % C::NS) * C::SLOT, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int cb = kk >> 2, off = (kk & 3) * 32;
            tc::mma_ss<0>(tmem + C::S_COL + 128 * t, tc::sdesc_add(qd, cb * 128 * 128 + off),
                          tc::sdesc_add(kd, cb * BN * 128 + off), idesc_qk, kk > 0);
          }
          tc::mma_commit(&bars[P_SF + t]);
          if (j == nt[t] - 1) tc::mma_commit(&bars[P_QE + t]);
        };
        auto pv = [&](int t, int j, uint32_t gv) {  // O_t += P_t V_j, 64 keys as their weights come
          if (ok && j == 0 && !tc::mbar_wait(&bars[P_OE + t], ((nq[t] - 1) & 1) ^ 1, a.err, 407)) ok = false;
          const uint64_t vd = tc::make_sdesc<128>(r_base + (gv % C::NS) * C::SLOT, BN * 128, 1024);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (ok && !tc::mbar_wait(&bars[P_PF + 2 * t + h], np[t] & 1, a.err, 408)) ok = false;
            if (!ok) continue;
            tc::fence_after_sync();
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              tc::mma_ts(tmem + C::O_COL + C::O_TILE * t, tmem + C::P_COL + C::P_TILE * t + C::P_HALF * h + 8 * kk,
                         tc::sdesc_add(vd, (4 * h + kk) * 16 * 128), idesc_pv, (j > 0 || h > 0 || kk > 0) ? 1u : 0u);
          }
          if (!ok) return;
          ++np[t];
          if constexpr (C::SEP) tc::mma_commit(&bars[P_PE + t]);
          if (j == nt[t] - 1) tc::mma_commit(&bars[P_OF + t]);
        };
        int v_seen = -1;
        auto full_v = [&](int j, uint32_t gv) {  // V_j is there, and repaired where it has to be
          if (v_seen == j) return;
          v_seen = j;
          full(gv);
          const uint32_t sv = gv % C::NS;
          if (ok && j >= m.jfix) {
            if (!tc::mbar_wait(&bars[P_VOK + sv], (vok >> sv) & 1, a.err, 406)) ok = false;
            vok ^= 1u << sv;
          }
        };
        // slots of this item: K_j at g + 2 j, V_j at g + 2 j + 1
        if (n > 0) {
          full(g);
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (ok && nt[t] > 0) {
              if (!tc::mbar_wait(&bars[P_QF + t], nq[t]++ & 1, a.err, 405)) ok = false;
              tc::fence_after_sync();
              if (ok) qk(t, 0, g);
            }
          if (ok) tc::mma_commit(&bars[P_KE + g % C::NS]);
        }
        if constexpr (C::SEP) {
          // in the order of events when tile 1 is half a step behind: QK_0(j+1), PV_1(j-1), QK_1(j+1), PV_0(j)
          auto next_qk = [&](int t, int j) {  // QK_t(j+1), once the softmax has read S_t(j)
            if (!ok || j + 1 >= nt[t]) return;
            if (!tc::mbar_wait(&bars[P_SE + t], se[t]++ & 1, a.err, 417)) ok = false;
            if (!k_seen[j & 1]) {
              full(g + 2 * j + 2);
              k_seen[j & 1] = true;
            }
            tc::fence_after_sync();
            if (ok) qk(t, j + 1, g + 2 * j + 2);
          };
          for (int j = 0; j <= n && ok; ++j) {
            k_seen[j & 1] = false;
            next_qk(0, j);
            if (j > 0) {
              if (ok && j - 1 < nt[1]) {
                full_v(j - 1, g + 2 * j - 1);
                pv(1, j - 1, g + 2 * j - 1);
              }
              if (ok) tc::mma_commit(&bars[P_KE + (g + 2 * j - 1) % C::NS]);
            }
            next_qk(1, j);
            if (ok && j + 1 < n) tc::mma_commit(&bars[P_KE + (g + 2 * j + 2) % C::NS]);
            if (ok && j < nt[0]) {
              full_v(j, g + 2 * j + 1);
              pv(0, j, g + 2 * j + 1);
            }
          }
          // the softmax's last read of a tile's S is behind its last QK^T; its arrival is still to be counted
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (nt[t] > 0) ++se[t];
        } else {
          for (int j = 0; j < n && ok; ++j) {
            const uint32_t gv = g + 2 * j + 1, gk = gv + 1;
            bool have_k = false;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (!ok || j >= nt[t]) continue;
              full_v(j, gv);
              pv(t, j, gv);
              if (ok && j + 1 < nt[t]) {
                if (!have_k) {
                  full(gk);
                  tc::fence_after_sync();
                  have_k = true;
                }
                if (ok) qk(t, j + 1, gk);
              }
            }
            if (ok) {
              tc::mma_commit(&bars[P_KE + gv % C::NS]);
              if (j + 1 < n) tc::mma_commit(&bars[P_KE + gk % C::NS]);
            }
          }
        }
        g += 2 * n;
        if (!ok) *abort_flag = 1;
        }
        __syncwarp();
      }
      // nor a product when the TMEM is freed
      if (*abort_flag && tc::elect_one()) {
        uint64_t* last = reinterpret_cast<uint64_t*>(smem + C::TILES + 568);
        tc::mbar_init(last, 1);
        tc::fence_barrier_init();
        tc::mma_commit(last);
        tc::mbar_wait(last, 0, a.err, 419);
      }
    } else if (warp == 10) {
      // ---------------------------------------------------------------- scheduler
      Finder f;
      f.init(a, lane);
      uint32_t idx = blockIdx.x;
      int k = 0;
      uint32_t tries = 0;
      bool more = true;
      while (more) {
        int pair = 0;
        const uint32_t item = CUT ? idx / uint32_t(a.splits) : idx, part = CUT ? idx % uint32_t(a.splits) : 0;
        int who = f.find(a, int(item / uint32_t(a.Hkv)), lane, pair);
        int of = 1;
        if (CUT && who >= 0) {
          of = __shfl_sync(0xffffffffu, parts_of(a, f.of(a, who), pair), who % 32);
          if (int(part) >= of) who = -1;
        }
        if (who >= 0) {
          const int s = k & 1;
          if (!wait_all(P_ITE + s, ((k >> 1) & 1) ^ 1, 411)) break;
          if (lane == who % 32) {
            fill(a, f.of(a, who), pair, int(item % uint32_t(a.Hkv)), int(part), of, &items[s]);
            tc::mbar_arrive(&bars[P_ITF + s]);
          }
          if (!wait_all(P_ASK, k & 1, 415)) break;
          ++k;
        }
        if (lane == 0) {
          tc::mbar_expect_tx(&bars[P_CLC], 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                           smem_u32(clc)),
                       "r"(smem_u32(&bars[P_CLC]))
                       : "memory");
        }
        if (!wait_all(P_CLC, tries & 1, 412)) break;
        ++tries;
        uint32_t got, x;
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b128 h;\n\t.reg .b32 y, z, w;\n\t"
            "ld.shared.b128 h, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t"
            "mov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, h;\n\t}"
            : "=r"(got), "=r"(x)
            : "r"(smem_u32(clc))
            : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the next answer is written behind this read
        __syncwarp();
        more = got != 0;
        idx = x;
      }
      const int s = k & 1;
      if (wait_all(P_ITE + s, ((k >> 1) & 1) ^ 1, 413) && lane == 0) {
        items[s].done = 1;
        tc::mbar_arrive(&bars[P_ITF + s]);
      }
    } else {
      // ---------------------------------------------------------------- V repair
      uint32_t g = 0;
      while (next_item(m)) {
        const int n = max(m.n0, m.n1), par = (itn - 1) & 3;
        int found = 0;
        if (lane == 0) bad_v[par] = 0;
        __syncwarp();
        // every fill of the ring passes here, so that this warp is neither ahead of the barriers'
        // phases nor lapped by them
        for (int f = 0; f < 2 * n; ++f, ++g) {
          const uint32_t s = g % C::NS;
          if (!wait_all(P_KF + s, (g / C::NS) & 1, 414)) break;
          if (!(f & 1) || (f >> 1) < m.jfix) {
            if (lane == 0) tc::mbar_arrive(&bars[P_KE + s]);
            continue;
          }
          // rows from the first one that the first token does not see; behind the last key of the
          // packed tensor the copy has filled in zeros
          const int r0 = max(0, m.lim0 - (f >> 1) * BN), r1 = min(BN, int(a.Tk) - m.k0 - (f >> 1) * BN);
          uint8_t* tile = ring + s * C::SLOT + (lane & 7) * 16;
          const int x1 = r1 * C::DB;  // 128-byte row pieces, four a step
          uint32_t top = 0;           // largest magnitudes of this lane's halves; NaN passes
#pragma unroll 1
          for (int x0 = r0 * C::DB + (lane >> 3); x0 < x1; x0 += 4 * 8) {
            uint4 w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const int x = min(x0 + 4 * e, x1 - 1);
              w[e] = *reinterpret_cast<const uint4*>(tile + (x % C::DB) * (BN * 128) + (x / C::DB) * 128);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) top = maxabs2<DT>(maxabs2<DT>(maxabs2<DT>(maxabs2<DT>(top, w[e].x), w[e].y), w[e].z), w[e].w);
          }
          if (__any_sync(0xffffffffu, nonfinite2<DT>(top) != 0)) {
            found = 1;
#pragma unroll 1
            for (int x = r0 * C::DB + (lane >> 3); x < x1; x += 4) {
              uint4* at = reinterpret_cast<uint4*>(tile + (x % C::DB) * (BN * 128) + (x / C::DB) * 128);
              const uint4 w = *at;
              *at = make_uint4(w.x & ~nonfinite2<DT>(w.x), w.y & ~nonfinite2<DT>(w.y), w.z & ~nonfinite2<DT>(w.z),
                               w.w & ~nonfinite2<DT>(w.w));
            }
          }
          if (found && lane == 0) bad_v[par] = 1;
          tc::fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tc::mbar_arrive(&bars[P_VOK + s]);
            tc::mbar_arrive(&bars[P_KE + s]);
          }
        }
      }
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  if (warp == 9) {
    tc::fence_after_sync();
    tc::tmem_free(tmem, 512);
  }
}

// The parts of a cut key range, in their order: a warp per row, or eight that share a row's parts where there
// may be 32 and more.  With a warp a row and shared, the whole call: 16 tokens of 16 heads on one behind 30000 keys (117
// parts) 64 us and 32; 64 tokens of 32 on 8 behind 16000 (18 parts of 2048 rows) 40 and 45; 128 of 16 on 2 behind
// 8000 (18 of 2048) 34 and 39.  (The number of rows counts too: 18 parts of 512 rows take 50 and 45.)
constexpr int SHARE_FROM = 32;
template <int DT, int D>
__global__ void __launch_bounds__(256) prefill_join_kernel(const __grid_constant__ PrefillArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int C = D / 32;
  __shared__ float shared_acc[8][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int share = a.splits >= SHARE_FROM ? 8 : 1, sub = warp & (share - 1);  // warps of a row, this one's place
  const int64_t rows = a.Tq * a.Hq, row = (int64_t)blockIdx.x * (8 / share) + (share == 8 ? 0 : warp);
  // the count from the offsets, as the items have it: it needs no word of the kernel before, whose rows may be
  // fewer than these (padding behind the last sequence) or, behind a wait that gave up, unwritten
  const int n = row < rows ? parts_of_token(a, int(row / a.Hq), lane) : 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (n <= 1) return;  // (with shared rows: the whole block)
  float top = -INFINITY, sum = 0.0f;
  for (int i = lane; i < n; i += 32) {
    const float x = a.plse[i * rows + row];
    top = fmaxf(top, x);
    if (x != x) sum = x;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int i = lane; i < n; i += 32) sum += exp2f((a.plse[i * rows + row] - ref) * LOG2E);
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.0f;
#pragma unroll 4
  for (int i = sub; i < n; i += share) {
    const float x = a.plse[i * rows + row];
    if (x == -INFINITY) continue;  // a part without keys for this row has no output
    const float w = exp2f((x - ref) * LOG2E);
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] += w * a.po[(i * rows + row) * D + lane + 32 * c];
  }
  if (share > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) shared_acc[warp][lane + 32 * c] = acc[c];
    __syncthreads();
    if (sub) return;
#pragma unroll
    for (int c = 0; c < C; ++c)
      for (int w = 1; w < 8; ++w) acc[c] += shared_acc[w][lane + 32 * c];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int c = 0; c < C; ++c) static_cast<T*>(a.o)[row * D + lane + 32 * c] = Elem<DT>::store(acc[c] * inv);
  if (lane == 0) a.lse[row] = sum == 0.0f ? -INFINITY : ref + logf(sum);
}

// Query tile pairs that Tq tokens in `seqs` sequences have at most: all of them one token longer than whole pairs.
int64_t most_pairs(int64_t Tq, int64_t seqs, int g) {
  const int64_t c = 2 * (128 / g);
  return (Tq + (seqs < Tq ? seqs : Tq) * (c - 1)) / c;
}

// Parts of a key range: only where the items would leave more than half of the SMs without work.
int split_count(int64_t Tq, int64_t Tk, int B, int Hq, int Hkv) {
  const int64_t items = most_pairs(Tq, B, Hq / Hkv) * Hkv, most = (Tk + BN - 1) / BN / MIN_PART;
  const int64_t n = num_sms() / items;
  return int(n < 2 || most < 2 ? 1 : n < most ? n : most);
}

template <int DT, int D>
int launch(const void* q, const void* k, PrefillArgs a, int64_t sq_t, int64_t sq_h, int64_t sk_t, int64_t sk_h,
           cudaStream_t st) {
  using C = PCfg<D>;
  CUtensorMap m[3];
  const void* base[3] = {q, k, a.v};
  const int64_t str[3][2] = {{sq_h, sq_t}, {sk_h, sk_t}, {a.sv_h, a.sv_t}};
  const int64_t heads[3] = {a.Hq, a.Hkv, a.Hkv}, toks[3] = {a.Tq, a.Tk, a.Tk};
  for (int i = 0; i < 3; ++i) {
    if (i > 0 && a.Tk == 0) {  // no keys at all: nothing is loaded through these
      m[i] = m[0];
      continue;
    }
    const uint64_t dims[3] = {uint64_t(D), uint64_t(heads[i]), uint64_t(toks[i])};
    // the stride of a dimension of size 1 is never used: any legal one
    const uint64_t s[2] = {heads[i] > 1 ? uint64_t(str[i][0]) * 2 : uint64_t(D) * 2,
                           toks[i] > 1 ? uint64_t(str[i][1]) * 2 : uint64_t(D) * 2};
    const uint32_t box[3] = {64, i ? 1u : uint32_t(a.g), i ? uint32_t(BN) : uint32_t(a.ntok)};
    if (int r = encode_tmap(&m[i], DT == MZB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                            base[i], dims, s, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return r;
  }
  auto kern = a.splits > 1 ? prefill_kernel<DT, D, true> : prefill_kernel<DT, D, false>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
    return launch_status("gqa_prefill(smem attr)");
  // the softmax warps' larger share of the registers would be waited for without end if the kernel
  // were built with fewer at launch
  static const int regs = [] {
    cudaFuncAttributes x, y;
    return cudaFuncGetAttributes(&x, prefill_kernel<DT, D, true>) == cudaSuccess &&
                   cudaFuncGetAttributes(&y, prefill_kernel<DT, D, false>) == cudaSuccess
               ? (x.numRegs < y.numRegs ? x.numRegs : y.numRegs) : 0;
  }();
  MZB_REQUIRE(regs * 384 >= 256 * 208 + 128 * 88, MZB_ERR_LAUNCH, "gqa_prefill: built with %d registers a thread", regs);
  const int64_t blocks = most_pairs(a.Tq, int64_t(a.B) + 1, a.g) * a.Hkv * a.splits;  // (the padding is one more sequence)
  MZB_REQUIRE(blocks < (int64_t(1) << 31), MZB_ERR_SHAPE, "gqa_prefill: too large");
  kern<<<unsigned(blocks), 384, C::SMEM, st>>>(m[0], m[1], m[2], a);
  if (int r = launch_status("gqa_prefill")) return r;
  if (a.splits == 1) return MZB_OK;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(a.splits >= SHARE_FROM ? a.Tq * a.Hq : (a.Tq * a.Hq + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, prefill_join_kernel<DT, D>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("gqa_prefill(join): launch failed: %s", cudaGetErrorString(e));
    return MZB_ERR_LAUNCH;
  }
  return MZB_OK;
}

}  // namespace gqa
}  // namespace mzb

using namespace mzb;

extern "C" int64_t mzb_gqa_prefill_ws(int64_t Tq, int64_t Tk, int B, int Hq, int Hkv, int D) {
  if (Tq <= 0 || Tk <= 0 || B <= 0 || Hkv <= 0 || Hq < Hkv || Hq % Hkv || Hq / Hkv > 128) return 0;
  const int n = gqa::split_count(Tq, Tk, B, Hq, Hkv);
  return n == 1 ? 0 : ((Tq * Hq * n + 3) & ~int64_t(3)) + n * Tq * Hq * D;
}

extern "C" int mzb_gqa_prefill(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k,
                               void* o, float* lse, float* ws, int64_t Tq, int64_t Tk, int B, int Hq, int Hkv, int D, int dtype,
                               int64_t sq_t, int64_t sq_h, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h,
                               int causal, float softmax_scale, int* err, void* stream) {
  MZB_REQUIRE(Tq >= 0 && Tk >= 0 && B >= 1 && Tq < (int64_t(1) << 29) && Tk < (int64_t(1) << 29), MZB_ERR_SHAPE,
              "gqa_prefill: bad sizes Tq=%lld Tk=%lld B=%d", (long long)Tq, (long long)Tk, B);
  MZB_REQUIRE(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 128, MZB_ERR_SHAPE,
              "gqa_prefill: query heads must be a multiple (at most 128) of the K/V heads, got %d and %d", Hq, Hkv);
  MZB_REQUIRE(D == 64 || D == 96 || D == 128, MZB_ERR_UNSUPPORTED, "gqa_prefill: unsupported head dim %d", D);
  MZB_REQUIRE(dtype == MZB_BF16 || dtype == MZB_F16, MZB_ERR_UNSUPPORTED, "gqa_prefill: unsupported dtype %d", dtype);
  MZB_REQUIRE(err != nullptr, MZB_ERR_SHAPE, "gqa_prefill: needs an error word");
  MZB_REQUIRE(reinterpret_cast<uintptr_t>(o) % 16 == 0, MZB_ERR_ALIGN, "gqa_prefill: o must be 16-byte aligned");
  if (Tq == 0) return MZB_OK;
  gqa::PrefillArgs a{};
  a.v = v; a.cu_q = cu_q; a.cu_k = cu_k; a.o = o; a.lse = lse;
  a.Tq = Tq; a.Tk = Tk; a.sv_t = sv_t; a.sv_h = sv_h;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.g = Hq / Hkv; a.ntok = 128 / a.g; a.causal = causal;
  a.neg = softmax_scale < 0;
  a.sl = (softmax_scale < 0 ? -softmax_scale : softmax_scale) * gqa::LOG2E;
  if (a.sl < 1e-37f) a.sl = 1e-37f;  // scale 0: all weights still 1, and a masked -inf stays -inf
  a.err = err;
  a.splits = gqa::split_count(Tq, Tk, B, Hq, Hkv);
  MZB_REQUIRE(a.splits == 1 || ws != nullptr, MZB_ERR_SHAPE, "gqa_prefill: needs a workspace");
  a.plse = ws;
  a.po = ws + ((Tq * Hq * a.splits + 3) & ~int64_t(3));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define MZB_GO(DT, DD) gqa::launch<DT, DD>(q, k, a, sq_t, sq_h, sk_t, sk_h, st)
  if (dtype == MZB_BF16) return D == 64 ? MZB_GO(MZB_BF16, 64) : D == 96 ? MZB_GO(MZB_BF16, 96) : MZB_GO(MZB_BF16, 128);
  return D == 64 ? MZB_GO(MZB_F16, 64) : D == 96 ? MZB_GO(MZB_F16, 96) : MZB_GO(MZB_F16, 128);
#undef MZB_GO
}
