// Attention of one new token per sequence over a paged K / V cache with grouped heads, bf16 /
// f16 in and out, fp32 accumulation, natural-log lse.  No counterpart in the reference.
//
//   key t < len[b] of sequence b is slot t % page of page table[b, t / page];
//   o = softmax(scale q K^T) V; a sequence of length 0: o = 0, lse = -inf.
//
// The live part of the cache is read once and everything else is small, so the kernel is
// built to keep HBM busy.  The keys of every (sequence, K / V head) are cut into tiles of 128,
// the tiles of all of them form one list, and each of one block per SM takes an equal run of
// it, whatever the lengths: a warp walks the page tables and feeds a ring of shared-memory
// stages (K and V of one tile each, ~200 KB in flight per SM) by TMA, eight warps do the
// products, S^T = K Q^T and O^T = V^T P^T: keys and channels are the 16 rows of mma.sync tiles, the query heads
// of a group their 8 columns, so that a small group wastes little (heads as rows: 349 us in the place of the
// batch's 323 when they were compared, back to back, where the power cap bound it).  The tensor pipe is 15 % busy
// while the bytes come: larger tensor instructions would gain nothing up to 16 heads a group.
// A (sequence, head) that lies in several blocks' runs leaves its (maximum, sum, output) parts in
// a workspace; a second kernel, started early and waiting, joins them in a fixed order.
//
// Measured (B200, 32 heads on 8, D = 128, bf16): 64 sequences of 512 to 16384 keys (2.2 GB) in 329 us
// a pass (6.8 TB/s; a copy's rate is 6.54); one of 131001 keys (0.54 GB) in 88 us with 5 of join; 256 of 300 keys, where
// merging a sequence's results costs half as much as its bytes, 73 us (4.4 TB/s).  64 heads on one K / V head are
// bound by products and exponentials (183 us for 0.54 GB).  Small calls are
// bound by latency: ~4 us from the start to the first tile (lengths, page ids, the copy: three
// dependent trips to memory), 6.1 us in all for 77 keys.
#include <type_traits>

#include "gqa_softmax.cuh"
#include "tc.cuh"

namespace mzb {
namespace gqad {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int TK = 128, TK_LOG = 7;  // keys per tile
constexpr int MIN_TILES = 2;         // a block's run is at least this long
constexpr int MAX_BLOCKS = 160;
constexpr int MAX_STAGES = 12;
constexpr int THREADS = 384;         // eight warps for the products, four for the loads (one of them works)
constexpr int PRODUCT_REGS = 208, LOAD_REGS = 88;
constexpr int MERGE_BYTES = 16384;   // the eight warps' results of a few rows at a time

struct DecodeArgs {
  const void* q;
  const int32_t *table, *lens;
  void* o;
  float* lse;
  float* ws;
  int64_t P, sq_b, sq_h;
  int B, Hq, Hkv, g, W, page, page_log, stages, blocks;
  float sl;                                    // scale * log2 e
  int* err;
  bool whole;  // runs end where a (sequence, head) does: no parts, no second kernel
  bool q16;    // query rows in 16-byte pieces
};

// ws: int [MAX_BLOCKS] (the (sequence, head) that a block begins and leaves to others; -1: none), int [B * Hkv]
// (the block that ends such a one), then for each of 2 * MAX_BLOCKS parts: float2 [g] (reference or -inf, sum), float [g][D].
__device__ __forceinline__ int* ws_open(const DecodeArgs& a) { return reinterpret_cast<int*>(a.ws); }
__device__ __forceinline__ int* ws_last(const DecodeArgs& a) { return reinterpret_cast<int*>(a.ws) + MAX_BLOCKS; }
__host__ __device__ inline int64_t ws_head(int B, int Hkv) { return (MAX_BLOCKS + (int64_t)B * Hkv + 3) & ~int64_t(3); }
__device__ __forceinline__ float* ws_part(const DecodeArgs& a, int part, int D) {
  return a.ws + ws_head(a.B, a.Hkv) + (int64_t)part * a.g * (D + 2);
}

// What the loading warp tells the computing ones about a stage.
struct __align__(16) Meta {
  int b, hk;
  uint16_t keys, flags;  // keys of the tile that exist; FIRST / LAST tile of the block's segment
  int part;              // -1: the segment is the whole (sequence, head), else its part number
};
constexpr int FIRST = 1, LAST = 2, END = 4;

template <int D>
struct DCfg {
  static constexpr int DB = (D + 63) / 64;
  static constexpr int K_BYTES = DB * TK * 128;
  static constexpr int STAGE = 2 * K_BYTES;
  static constexpr int QROW = D * 2 + 16;        // bytes from query row to row: no two of eight on the same banks
  static constexpr int ROWS = D == 64 ? 8 : 4;   // rows of a merging pass
};

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (DT == MZB_BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// An 8 x 8 matrix of 16-bit numbers, a row in four lanes, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
template <int DT>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
  if constexpr (DT == MZB_BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// The barrier's phase waits for this thread's copies so far, too.
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// All lanes wait for a phase; nobody waits on once a wait of the block has run out of time.
__device__ __forceinline__ bool wait_stage(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
  bool got = tc::mbar_try_wait(bar, parity);
  if (__all_sync(0xffffffffu, got)) return true;
  if (!got) got = !*abort_flag && tc::mbar_wait(bar, parity, err, code);
  return __all_sync(0xffffffffu, got);
}

// The eight product warps meet: whether one of them has given up (they leave through here only, all of them at one
// meeting, so that none is left behind at a barrier).
__device__ __forceinline__ bool meet(bool gave_up) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"(uint32_t(gave_up)) : "memory");
  return any != 0;
}

__device__ __forceinline__ int len_of(const DecodeArgs& a, int b) { return max(0, min(a.lens[b], a.W * a.page)); }

// MT: head tiles of 8 NH heads.  A warp has one of them and, 32 at a time, its share of the key tile.  With one head
// tile four warps share a key tile and the other four have the next one: a warp's chain of products and
// exponentials (~1 us) is spread over two tiles' time.
template <int DT, int D, int MT, int NH>
__global__ void __launch_bounds__(THREADS, 1)
    decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                  const __grid_constant__ DecodeArgs a) {
  using C = DCfg<D>;
  using T = typename Elem<DT>::T;
  constexpr int GROUPS = MT == 1 ? 2 : 1;       // warps 0-3 and 4-7 take tiles in turn
  constexpr int KP = 8 / MT / GROUPS;           // warps that share a tile's keys
  constexpr int STEPS = TK / KP / 32;           // 32-key steps of a warp per tile
  constexpr int PARTS = 8 / MT;                 // partial results of a head tile to merge
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  __shared__ Meta meta[MAX_STAGES];
  __shared__ float sm_m[8][16], sm_l[8][16];
  __shared__ int abort_s;
  volatile int* abort_flag = &abort_s;
  float* merge = reinterpret_cast<float*>(smem + a.stages * C::STAGE);  // [8 warps][ROWS][D]
  uint8_t* q_rows = smem + a.stages * C::STAGE + MERGE_BYTES;           // up to 16 heads: [stages][g] rows of QROW bytes
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023) {
    if (threadIdx.x == 0) atomicExch(a.err, MZB_ERR_ALIGN);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 8);  // every warp lets every stage go, so none is lapped by the ring
    }
    abort_s = 0;
    tc::fence_barrier_init();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __syncthreads();

  if (warp >= 8) {
    // ---------------------------------------------------------------- loads (one warp of four)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(LOAD_REGS));
    if (warp > 8) return;
    if (lane == 0) {
      tc::prefetch_tmap(&tk);
      tc::prefetch_tmap(&tv);
    }
    // this block's run of tiles: first (sequence, head, tile) and how many.  A lane keeps the length of
    // one sequence of the 32 from `base_b`: every look at a length is a shuffle, not another load.
    if (lane == 0 && !a.whole) ws_open(a)[blockIdx.x] = -1;
    int b = 0, hk = 0, t0 = 0, base_b = 0, my_len = 0;
    int64_t left = 0;
    auto load_lens = [&](int from) {
      base_b = from;
      my_len = from + lane < a.B ? len_of(a, from + lane) : 0;
    };
    auto len_at = [&](int x) {  // (the whole warp; x only grows)
      if (x >= base_b + 32) load_lens(x);
      return __shfl_sync(0xffffffffu, my_len, x - base_b);
    };
    auto tiles_of = [](int len) { return (len + TK - 1) / TK; };
    if (a.whole) {
      const int64_t rows = (int64_t)a.B * a.Hkv, lo = rows * blockIdx.x / a.blocks, hi = rows * (blockIdx.x + 1) / a.blocks;
      b = int(lo / a.Hkv);
      hk = int(lo % a.Hkv);
      for (int64_t b0 = b; b0 * a.Hkv < hi; b0 += 32) {
        load_lens(int(b0));
        const int64_t mine = max(lo, (b0 + lane) * a.Hkv), end = min(hi, (b0 + lane + 1) * a.Hkv);
        left += __reduce_add_sync(0xffffffffu, mine < end ? int(end - mine) * tiles_of(my_len) : 0);
      }
      load_lens(b);
      while (left > 0 && len_at(b) == 0) {
        ++b;
        hk = 0;
      }
    } else {
      int64_t total = 0;
      for (int b0 = 0; b0 < a.B; b0 += 32) {
        load_lens(b0);
        const int64_t n = __reduce_add_sync(0xffffffffu, tiles_of(my_len));
        total += n;
      }
      total *= a.Hkv;
      const int64_t per = max((int64_t)MIN_TILES, (total + a.blocks - 1) / a.blocks), lo = per * blockIdx.x;
      left = min(per, total - lo);
      if (left > 0) {
        int64_t at = 0;
        for (int b0 = 0;; b0 += 32) {
          if (b0 != base_b) load_lens(b0);
          const int64_t n = (int64_t)tiles_of(my_len) * a.Hkv;
          int64_t inc = n;
#pragma unroll
          for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, inc, d);
            if (lane >= d) inc += y;
          }
          const unsigned hit = __ballot_sync(0xffffffffu, lo < at + inc);
          if (hit) {
            const int l = __ffs(hit) - 1;
            b = b0 + l;
            const int64_t in = lo - at - __shfl_sync(0xffffffffu, inc - n, l);
            const int tiles = __shfl_sync(0xffffffffu, tiles_of(my_len), l);
            hk = int(in / tiles);
            t0 = int(in % tiles);
            break;
          }
          at += __shfl_sync(0xffffffffu, inc, 31);
        }
      }
    }
    // rows of a TMA box, boxes of a tile (per K / V and column block), as powers of two: a division by a
    // number of the launch costs ~80 cycles, and five of them a tile made this loop the limit
    const int rows_log = min(a.page_log, TK_LOG), rows = 1 << rows_log, tile_log = TK_LOG - rows_log;
    int s = 0;
    uint32_t phase = 0;
    bool ok = true;
    while (left > 0 && ok && b < a.B) {
      const int len = len_at(b), tiles = tiles_of(len);
      const int n = int(min((int64_t)(tiles - t0), left));  // this block's segment: tiles t0 .. t0 + n
      const bool begins = t0 == 0, ends = t0 + n == tiles;
      const int part = begins && ends ? -1 : begins ? 2 * (int)blockIdx.x + 1 : 2 * (int)blockIdx.x;
      if (lane == 0 && part >= 0) {
        const int64_t row = (int64_t)b * a.Hkv + hk;
        if (begins) ws_open(a)[blockIdx.x] = int(row);
        if (ends) ws_last(a)[row] = blockIdx.x;
      }
      // page ids of 32 boxes at a time, one per lane, the next ones in flight meanwhile
      const int32_t* row = a.table + (int64_t)b * a.W;
      const int box0 = t0 << tile_log, boxes = (len + rows - 1) >> rows_log;  // boxes with live keys
      auto ids = [&](int x) {  // box x of the sequence
        return x < boxes ? row[x >> (a.page_log - rows_log)] : 0;
      };
      // an id outside the pool is an error, and some page is read in its place; looked at when the ids are needed, so
      // that the next ones stay in flight
      auto checked = [&](int p) {
        if (p < 0 || p >= a.P) atomicCAS(a.err, 0, MZB_ERR_PAGES);
        return max(0, min(p, int(a.P - 1)));
      };
      int cur = ids(box0 + lane), nxt = ids(box0 + 32 + lane), base = box0;
      cur = checked(cur);
      for (int i = 0; i < n; ++i) {
        const int t = t0 + i, keys = min(TK, len - t * TK), live = (keys + rows - 1) >> rows_log;
        if ((t << tile_log) - base >= 32) {
          base += 32;
          cur = checked(nxt);
          nxt = ids(base + 32 + lane);
        }
        ok = wait_stage(&empty[s], phase ^ 1, abort_flag, a.err, 421);
        if (!ok) break;
        if (MT * NH <= 2 && i == 0) {  // the segment's query rows come with its first tile
          const T* q = static_cast<const T*>(a.q) + (int64_t)b * a.sq_b + (int64_t)hk * a.g * a.sq_h;
          const uint32_t to = smem_u32(q_rows) + s * a.g * C::QROW;
          auto rows_by = [&](auto piece) {
            constexpr int BYTES = decltype(piece)::value, N = D * 2 / BYTES;
            for (int x = lane; x < a.g * N; x += 32)
              copy_async<BYTES>(to + x / N * C::QROW + x % N * BYTES, q + (int64_t)(x / N) * a.sq_h + x % N * (BYTES / 2));
          };
          if (a.q16) rows_by(std::integral_constant<int, 16>());
          else rows_by(std::integral_constant<int, 4>());
          copies_arrive(&full[s]);
          __syncwarp();
        }
        // page ids of the tile's boxes, then all copies by one elected lane (behind a condition that
        // differs by lane each copy's operands are made uniform in a loop: ~700 ns a tile)
        int pid[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) pid[x] = __shfl_sync(0xffffffffu, cur, min((t << tile_log) + x - base, 31));
        if (tc::elect_one()) {
          meta[s] = Meta{b, hk, uint16_t(keys), uint16_t((i == 0 ? FIRST : 0) | (i == n - 1 ? LAST : 0)), part};
          tc::mbar_expect_tx(&full[s], uint32_t(live) * rows * 128 * C::DB * 2);
          uint8_t* to = smem + s * C::STAGE;
          const int slot = (t * TK) & (a.page - 1);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            if (x < live) {
#pragma unroll
              for (int cb = 0; cb < C::DB; ++cb) {
                tma_load_4d(to + cb * TK * 128 + x * rows * 128, &tk, &full[s], cb * 64, slot, hk, pid[x]);
                tma_load_4d(to + C::K_BYTES + cb * TK * 128 + x * rows * 128, &tv, &full[s], cb * 64, slot, hk, pid[x]);
              }
            }
        }
        __syncwarp();
        if (++s == a.stages) {
          s = 0;
          phase ^= 1;
        }
      }
      left -= n;
      t0 = 0;
      if (++hk == a.Hkv) {
        hk = 0;
        ++b;
        while (left > 0 && b < a.B && len_at(b) == 0) ++b;
      }
    }
    // the end, as a stage without data
    if (ok && wait_stage(&empty[s], phase ^ 1, abort_flag, a.err, 422)) {
      if (lane == 0) {
        meta[s].flags = END;
        tc::mbar_arrive(&full[s]);
      }
    } else {
      *abort_flag = 1;
      // no copy is left in flight when the block ends: stages below s were last filled in this round of the ring, the
      // others in the one before (never: the barrier's phase -1, which has passed)
      for (int x = 0; x < a.stages; ++x) tc::mbar_wait(&full[x], x < s ? phase : phase ^ 1, a.err, 424);
    }
  } else {
    // ---------------------------------------------------------------- products
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(PRODUCT_REGS));
    // sequences without keys
    for (int b = blockIdx.x; b < a.B; b += gridDim.x)
      if (a.lens[b] <= 0 || a.W == 0) {
        for (int x = threadIdx.x; x < a.Hq * D / 8; x += 256)
          reinterpret_cast<uint4*>(static_cast<T*>(a.o) + (int64_t)b * a.Hq * D)[x] = make_uint4(0, 0, 0, 0);
        for (int x = threadIdx.x; x < a.Hq; x += 256) a.lse[(int64_t)b * a.Hq + x] = -INFINITY;
      }
    const int mt = warp % MT, kp = warp / MT % KP, turn = warp / (8 / GROUPS);
    const int r0 = lane >> 2, c0 = (lane & 3) * 2;
    constexpr int HT = 8 * NH;  // heads of a tile
    uint32_t qf[NH][D / 16][2];                  // (channels) x (heads)
    float o[D / 16][NH][4], m[NH][2], l[NH][2];  // channels r0, r0 + 8 of 16 x heads c0, c0 + 1 of 8
    auto clear = [&]() {
#pragma unroll
      for (int n = 0; n < NH; ++n) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][n][e] = 0.0f;
        m[n][0] = m[n][1] = -INFINITY;
        l[n][0] = l[n][1] = 0.0f;
      }
    };
    clear();
    // ldmatrix rows of this lane.  K: (keys 0-7, 8-15) x (channels 0-7, 8-15), the keys first; V transposed:
    // (keys 0-7, 8-15) x (channels 0-7, 8-15), the channels first
    const int krow = lane & 15, kch = lane >> 4;
    const int vrow = (lane & 7) + ((lane >> 4) << 3), vch = (lane >> 3) & 1;
    int s = -1, nth = 1;
    uint32_t phase = 0;
    while (true) {
      nth ^= 1;
      if (++s == a.stages) {
        s = 0;
        phase ^= 1;
      }
      const bool got = wait_stage(&full[s], phase, abort_flag, a.err, 423);
      if (!got) *abort_flag = 1;
      const Meta w = meta[s];
      if (!got || (w.flags & END)) {
        meet(!got);
        break;
      }
      if (w.flags & FIRST) {  // this group's query rows
        if constexpr (MT * HT <= 16) {  // (rows behind the last repeat it: their results go nowhere)
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            const uint32_t from = smem_u32(q_rows) + (s * a.g + min(mt * HT + 8 * n + (lane & 7), a.g - 1)) * C::QROW + (lane >> 3) * 16;
#pragma unroll
            for (int kk = 0; kk < D / 16; kk += 2) {
              uint32_t x[4];
              ldsm4<false>(x, from + kk * 32);
              qf[n][kk][0] = x[0];
              qf[n][kk][1] = x[1];
              qf[n][kk + 1][0] = x[2];
              qf[n][kk + 1][1] = x[3];
            }
          }
        } else {
          const T* q = static_cast<const T*>(a.q) + (int64_t)w.b * a.sq_b;
#pragma unroll
          for (int n = 0; n < NH; ++n) {
            const int h = mt * HT + 8 * n + r0;
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                qf[n][kk][j] = h < a.g ? *reinterpret_cast<const uint32_t*>(q + (int64_t)(w.hk * a.g + h) * a.sq_h + 16 * kk + 8 * j + c0)
                                       : 0u;
          }
        }
      }
      if (GROUPS == 1 || nth == turn) {
        const uint32_t kt = smem_u32(smem + s * C::STAGE), vt = kt + C::K_BYTES;
#pragma unroll 1
        for (int st = 0; st < STEPS; ++st) {
          const int key0 = (kp * STEPS + st) * 32;
          if (key0 >= w.keys) break;
          float sc[2][NH][4] = {};  // keys r0, r0 + 8 of 16 x heads c0, c0 + 1 of 8
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const int ch = 2 * kk + kch;  // 16-byte piece
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              uint32_t ak[4];
              const int kr = key0 + 16 * x + krow;
              ldsm4<false>(ak, kt + (ch >> 3) * (TK * 128) + kr * 128 + (((ch & 7) ^ (kr & 7)) * 16));
#pragma unroll
              for (int n = 0; n < NH; ++n) mma16816<DT>(sc[x][n], ak, qf[n][kk][0], qf[n][kk][1]);
            }
          }
          const int vis = w.keys - key0;  // keys of these 32 that exist
          float top[NH][2];
#pragma unroll
          for (int n = 0; n < NH; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float t = -INFINITY;
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  float& y = sc[x][n][2 * r + e];
                  y *= a.sl;
                  if (16 * x + 8 * r + r0 >= vis) y = -INFINITY;
                  t = fmaxf(t, y);
                }
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
              top[n][e] = t;
            }
          // O and the sums are rescaled only when a maximum has grown by more than 2^GROW
          bool grown = false;
#pragma unroll
          for (int n = 0; n < NH; ++n) grown |= top[n][0] > m[n][0] + Running<DT>::GROW || top[n][1] > m[n][1] + Running<DT>::GROW;
          if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              float al[2];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float mn = fmaxf(m[n][e], top[n][e]);
                al[e] = mn == -INFINITY ? 1.0f : fast_exp2(Running<DT>::relative(m[n][e]) - Running<DT>::relative(mn));
                m[n][e] = mn;
                l[n][e] *= al[e];
              }
#pragma unroll
              for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][n][e] *= al[e & 1];
            }
          }
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int seen = vis - 16 * x;
            if (seen <= 0) break;
            // the weights as a sum of two numbers of the type (16 bits and more), turned to (keys) x (heads)
            uint32_t ph[NH][2], pl[NH][2];
#pragma unroll
            for (int n = 0; n < NH; ++n) {
              const float ms[2] = {Running<DT>::reference(m[n][0]), Running<DT>::reference(m[n][1])};
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float p0 = fast_exp2(sc[x][n][2 * r] - ms[0]), p1 = fast_exp2(sc[x][n][2 * r + 1] - ms[1]);
                l[n][0] += p0;
                l[n][1] += p1;
                const uint32_t h2 = pack2<DT>(p0, p1);
                const float2 f = unpack2<DT>(h2);
                ph[n][r] = transpose8(h2);
                pl[n][r] = transpose8(pack2<DT>(p0 - f.x, p1 - f.y));
              }
            }
            const bool tail = seen < 16;
            const uint32_t k01 = tail ? (c0 < seen ? 0xffffu : 0u) | (c0 + 1 < seen ? 0xffff0000u : 0u) : ~0u;
            const uint32_t k89 = tail ? (c0 + 8 < seen ? 0xffffu : 0u) | (c0 + 9 < seen ? 0xffff0000u : 0u) : ~0u;
            const int vr = key0 + 16 * x + vrow;
#pragma unroll
            for (int i = 0; i < D / 16; i += 2) {
              uint32_t av[2][4];
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int ch = 2 * (i + j) + vch;
                ldsm4<true>(av[j], vt + (ch >> 3) * (TK * 128) + vr * 128 + (((ch & 7) ^ (vr & 7)) * 16));
                if (tail) {  // what lies behind the sequence's end must not meet its zero weights
                  av[j][0] &= k01;
                  av[j][1] &= k01;
                  av[j][2] &= k89;
                  av[j][3] &= k89;
                }
              }
#pragma unroll
              for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma16816<DT>(o[i + j][n], av[j], ph[n][0], ph[n][1]);
#pragma unroll
              for (int n = 0; n < NH; ++n)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma16816<DT>(o[i + j][n], av[j], pl[n][0], pl[n][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&empty[s]);
      if (w.flags & LAST) {
        // ------------------------------------------------------------ merge the warps' results
#pragma unroll
        for (int n = 0; n < NH; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
        if (meet(false)) break;  // (and what the last merge wrote has been read)
        // a few heads of a tile at a time (the ring needs the shared memory more); channels are exchanged in
        // eights by the head's number, so that the heads of a store lie on different banks
        const int gr = min(a.g, HT);
#pragma unroll 1
        for (int at = 0; at < gr; at += C::ROWS) {
          if (at) tc::bar_sync(1, 256);  // what the last pass wrote has been read
          if (at == 0 && r0 == 0)
#pragma unroll
            for (int n = 0; n < NH; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                sm_m[warp][8 * n + c0 + e] = Running<DT>::relative(m[n][e]);
                sm_l[warp][8 * n + c0 + e] = l[n][e];
              }
          const int mine = c0 + (at & 8) - at;  // this thread's heads of the pass: this one and the next
          if (mine >= 0 && mine < C::ROWS) {
            float* to = merge + (warp * C::ROWS + mine) * D;
            const int flip = (mine >> 1 & 3) * 8;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                to[(e & 1) * D + ((16 * i + 8 * (e >> 1) + r0) ^ flip)] = at < 8 ? o[i][0][e] : o[i][NH - 1][e];
          }
          tc::bar_sync(1, 256);
          constexpr int LANES = D == 64 ? 16 : 32;  // of a row, four channels each
          const int d = (threadIdx.x % LANES) * 4;
#pragma unroll 1
          for (int x = threadIdx.x / LANES; x < MT * C::ROWS; x += 256 / LANES) {
            const int tile = x / C::ROWS, r = at + x % C::ROWS, h = tile * HT + r;
            if (h >= a.g || d >= D) continue;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < PARTS; ++i) mx = fmaxf(mx, sm_m[i * MT + tile][r]);
            const float ms = mx == -INFINITY ? 0.0f : mx;
            float ls = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) {
              const int wp = i * MT + tile;
              const float al = fast_exp2(sm_m[wp][r] - ms);
              const float4 v = *reinterpret_cast<const float4*>(merge + (wp * C::ROWS + (r - at)) * D + (d ^ (((r - at) >> 1 & 3) * 8)));
              ls += sm_l[wp][r] * al;
              acc.x += v.x * al;
              acc.y += v.y * al;
              acc.z += v.z * al;
              acc.w += v.w * al;
            }
            if (w.part < 0) {
              const int64_t row = (int64_t)w.b * a.Hq + w.hk * a.g + h;
              const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;  // 0: scores of -inf alone
              *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + row * D + d) =
                  make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
              if (d == 0) a.lse[row] = (mx + log2f(ls)) * LN2;
            } else {
              float* to = ws_part(a, w.part, D);
              float2* y = reinterpret_cast<float2*>(to + 2 * a.g + h * D + d);
              y[0] = make_float2(acc.x, acc.y);
              y[1] = make_float2(acc.z, acc.w);
              if (d == 0) *reinterpret_cast<float2*>(to + 2 * h) = make_float2(mx, ls);
            }
          }
        }
        clear();
      }
    }
  }
}

// One block per query head of a (sequence, head) that lies in several blocks' runs (each run leaves at
// most one to the next, so the grid is runs x group): its warps share the parts, whose weights each lane
// finds for up to 5 of them first.
template <int DT, int D>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ DecodeArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int PER = MAX_BLOCKS / 32, C4 = D / 4;  // parts of a lane, four-channel pieces of a row
  __shared__ float weight[MAX_BLOCKS];
  __shared__ float4 sum[4][C4];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int first = blockIdx.x / a.g, h = blockIdx.x % a.g;
  const int of = ws_open(a)[first];  // sequence * Hkv + head
  if (of < 0 || of >= a.B * a.Hkv) return;
  const int64_t row = (int64_t)of * a.g + h;
  const int n = max(1, min(ws_last(a)[of], a.blocks - 1) - first + 1);
  auto part = [&](int i) { return ws_part(a, i == 0 ? 2 * first + 1 : 2 * (first + i), D); };
  // the first eight parts of each warp are on their way while the weights are found
  constexpr int AHEAD = 8;
  float2 va[AHEAD], vb[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (lane < C4 && warp + 4 * i < n) {
      const float* p = part(warp + 4 * i) + 2 * a.g + h * D + 4 * lane;
      va[i] = *reinterpret_cast<const float2*>(p);
      vb[i] = *reinterpret_cast<const float2*>(p + 2);
    }
  // every warp for itself: the same numbers in the same order
  float2 ml[PER];
  float mx = -INFINITY, ls = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    ml[i] = make_float2(-INFINITY, 0.0f);
    if (lane + 32 * i < n) ml[i] = *reinterpret_cast<const float2*>(part(lane + 32 * i) + 2 * h);
    mx = fmaxf(mx, ml[i].x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
  const float ms = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float al = fast_exp2(ml[i].x - ms);
    ls += ml[i].y * al;
    if (warp == 0 && lane + 32 * i < n) weight[lane + 32 * i] = al;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, d);
  __syncthreads();
  if (lane < C4) {
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (warp + 4 * i < n) {
        const float al = weight[warp + 4 * i];
        acc.x += va[i].x * al;
        acc.y += va[i].y * al;
        acc.z += vb[i].x * al;
        acc.w += vb[i].y * al;
      }
#pragma unroll 4
    for (int i = warp + 4 * AHEAD; i < n; i += 4) {
      const float* p = part(i) + 2 * a.g + h * D + 4 * lane;
      const float2 x = *reinterpret_cast<const float2*>(p), y = *reinterpret_cast<const float2*>(p + 2);
      const float al = weight[i];
      acc.x += x.x * al;
      acc.y += x.y * al;
      acc.z += y.x * al;
      acc.w += y.y * al;
    }
    sum[warp][lane] = acc;
  }
  __syncthreads();
  if (threadIdx.x < C4) {
    const float inv = ls == 0.0f ? 0.0f : 1.0f / ls;
    float4 t = sum[0][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) {
      t.x += sum[w][lane].x;
      t.y += sum[w][lane].y;
      t.z += sum[w][lane].z;
      t.w += sum[w][lane].w;
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + row * D + 4 * lane) =
        make_uint2(pack2<DT>(t.x * inv, t.y * inv), pack2<DT>(t.z * inv, t.w * inv));
    if (lane == 0) a.lse[row] = (mx + log2f(ls)) * LN2;
  }
}

int block_count() { return num_sms() < MAX_BLOCKS ? num_sms() : MAX_BLOCKS; }

// Tables of at most MIN_TILES tiles: whole (sequence, head)s to a block, nothing to join: 64 sequences of one key on
// 8 heads 17.5 -> 15.4 us with the launches, 256 of 256 keys 66.6 -> 65.5.  Longer ones in runs of equal length.
bool short_table(int W, int page) { return (int64_t)W * page <= MIN_TILES * TK; }

template <int DT, int D, int MT, int NH>
int launch(const void* k, const void* v, DecodeArgs a, const int64_t* sk, const int64_t* sv, cudaStream_t st) {
  using C = DCfg<D>;
  CUtensorMap m[2];
  for (int i = 0; i < 2; ++i) {
    const int64_t* s = i ? sv : sk;  // page, head, token
    const uint64_t dims[4] = {uint64_t(D), uint64_t(a.page), uint64_t(a.Hkv), uint64_t(a.P)};
    // the stride of a dimension of size 1 is never used: any legal one
    const uint64_t str[3] = {uint64_t(s[2]) * 2, a.Hkv > 1 ? uint64_t(s[1]) * 2 : uint64_t(D) * 2,
                             a.P > 1 ? uint64_t(s[0]) * 2 : uint64_t(D) * 2};
    const uint32_t box[4] = {64, uint32_t(a.page < TK ? a.page : TK), 1, 1};
    if (int r = encode_tmap(&m[i], DT == MZB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                            i ? v : k, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B))
      return r;
  }
  const int budget = 227 * 1024 - 3072 - MERGE_BYTES;  // 3 KB: the static arrays
  const int q_bytes = MT * NH <= 2 ? a.g * C::QROW : 0;  // of a stage
  a.stages = budget / (C::STAGE + q_bytes) < MAX_STAGES ? budget / (C::STAGE + q_bytes) : MAX_STAGES;
  a.whole = short_table(a.W, a.page);
  a.blocks = block_count();
  if (a.whole && (int64_t)a.B * a.Hkv < a.blocks) a.blocks = a.B * a.Hkv;
  auto kern = decode_kernel<DT, D, MT, NH>;
  const int smem = a.stages * (C::STAGE + q_bytes) + MERGE_BYTES;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return launch_status("gqa_decode(smem attr)");
  // the product warps' share is drawn from what the block is launched with: less would wait for ever
  static const int regs = [] {
    cudaFuncAttributes x;
    return cudaFuncGetAttributes(&x, decode_kernel<DT, D, MT, NH>) == cudaSuccess ? x.numRegs : 0;
  }();
  MZB_REQUIRE(regs * THREADS >= 256 * PRODUCT_REGS + (THREADS - 256) * LOAD_REGS, MZB_ERR_LAUNCH,
              "gqa_decode: built with %d registers a thread", regs);
  kern<<<a.blocks, THREADS, smem, st>>>(m[0], m[1], a);
  if (int r = launch_status("gqa_decode")) return r;
  if (a.whole) return MZB_OK;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(unsigned(a.blocks * a.g));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, join_kernel<DT, D>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("gqa_decode(join): launch failed: %s", cudaGetErrorString(e));
    return MZB_ERR_LAUNCH;
  }
  return MZB_OK;
}

}  // namespace gqad
}  // namespace mzb

using namespace mzb;

extern "C" int64_t mzb_gqa_decode_ws(int B, int Hq, int Hkv, int D, int W, int page) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || gqad::short_table(W, page)) return 0;
  return gqad::ws_head(B, Hkv) + 2 * (int64_t)gqad::block_count() * (Hq / Hkv) * (D + 2);
}

extern "C" int mzb_gqa_decode(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                              const int32_t* seq_lens, void* o, float* lse, float* ws, int B, int Hq, int Hkv, int D,
                              int dtype, int page, int64_t P, int W, int64_t sq_b, int64_t sq_h, int64_t sk_p,
                              int64_t sk_h, int64_t sk_t, int64_t sv_p, int64_t sv_h, int64_t sv_t,
                              float softmax_scale, int* err, void* stream) {
  MZB_REQUIRE(B >= 0 && P >= 1 && P < (int64_t(1) << 31) && W >= 0 && (int64_t)W * page < (int64_t(1) << 31),
              MZB_ERR_SHAPE, "gqa_decode: bad sizes B=%d pages=%lld table width=%d page=%d", B, (long long)P, W, page);
  MZB_REQUIRE(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 128 && (int64_t)B * Hq < (int64_t(1) << 31), MZB_ERR_SHAPE,
              "gqa_decode: query heads must be a multiple (at most 128) of the K/V heads, got %d and %d", Hq, Hkv);
  MZB_REQUIRE(D == 64 || D == 96 || D == 128, MZB_ERR_UNSUPPORTED, "gqa_decode: unsupported head dim %d", D);
  MZB_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, MZB_ERR_UNSUPPORTED,
              "gqa_decode: unsupported page size %d (16, 32, 64 or 128 tokens)", page);
  MZB_REQUIRE(dtype == MZB_BF16 || dtype == MZB_F16, MZB_ERR_UNSUPPORTED, "gqa_decode: unsupported dtype %d", dtype);
  MZB_REQUIRE(err != nullptr, MZB_ERR_SHAPE, "gqa_decode: needs an error word");
  MZB_REQUIRE(reinterpret_cast<uintptr_t>(q) % 4 == 0 && reinterpret_cast<uintptr_t>(o) % 16 == 0 && sq_b % 2 == 0 && sq_h % 2 == 0,
              MZB_ERR_ALIGN, "gqa_decode: q rows must be 4-byte and o 16-byte aligned");
  MZB_REQUIRE(ws != nullptr || B == 0 || gqad::short_table(W, page), MZB_ERR_SHAPE, "gqa_decode: needs a workspace");
  if (B == 0) return MZB_OK;
  gqad::DecodeArgs a{};
  a.q = q; a.table = page_table; a.lens = seq_lens; a.o = o; a.lse = lse; a.ws = ws;
  a.P = P; a.sq_b = sq_b; a.sq_h = sq_h;
  a.B = B; a.Hq = Hq; a.Hkv = Hkv; a.g = Hq / Hkv; a.W = W; a.page = page;
  a.page_log = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  a.sl = softmax_scale * gqad::LOG2E;
  a.err = err;
  a.q16 = reinterpret_cast<uintptr_t>(q) % 16 == 0 && sq_b % 8 == 0 && sq_h % 8 == 0;
  const int64_t sk[3] = {sk_p, sk_h, sk_t}, sv[3] = {sv_p, sv_h, sv_t};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // up to 16 heads in tiles of 8 (9 to 16 as one of 16: 200 sequences of 500 keys, 64 heads on 4, 68.6 us against
  // 62.3), more in tiles of 16, which read K and V half as often (64 on 1: 189 us against 222)
#define MZB_GO(DT, DD)                                                                              \
  (a.g <= 8 ? gqad::launch<DT, DD, 1, 1>(k_pages, v_pages, a, sk, sv, st)                           \
   : a.g <= 16 ? gqad::launch<DT, DD, 2, 1>(k_pages, v_pages, a, sk, sv, st)                        \
   : a.g <= 32 ? gqad::launch<DT, DD, 2, 2>(k_pages, v_pages, a, sk, sv, st)                        \
   : a.g <= 64 ? gqad::launch<DT, DD, 4, 2>(k_pages, v_pages, a, sk, sv, st)                        \
               : gqad::launch<DT, DD, 8, 2>(k_pages, v_pages, a, sk, sv, st))
  if (dtype == MZB_BF16) return D == 64 ? MZB_GO(MZB_BF16, 64) : D == 96 ? MZB_GO(MZB_BF16, 96) : MZB_GO(MZB_BF16, 128);
  return D == 64 ? MZB_GO(MZB_F16, 64) : D == 96 ? MZB_GO(MZB_F16, 96) : MZB_GO(MZB_F16, 128);
#undef MZB_GO
}
