// Work items of the prefill kernel: what a block number stands for (sequence, pair of query tiles,
// part of its key range) and how many parts a row's key range has.  Arithmetic on the offsets and
// warp collectives only, so that the tests run it on the host, a fiber for each lane.
#pragma once

#include <stdint.h>

namespace mzb {
namespace gqa {

constexpr int BN = 128;  // keys per tile
// key tiles of a part at least (a part costs a block's start and its share of the join): 16 tokens of 16 heads on
// one behind 4000 keys take 32 us with parts of six, 24 of two
constexpr int MIN_PART = 2;

struct ItemArgs {
  const int32_t *cu_q, *cu_k;
  int64_t Tq, Tk;
  int B, ntok, causal;  // ntok: tokens per query tile
  int splits;           // a call with few work items cuts the longer key ranges into up to `splits` (1: none) parts
};

// One work item, in shared memory.  Of a part, k0, nk and shift are those of its keys alone.
struct Item {
  int tok0, tok_end;  // first packed token, end of the sequence
  int i0, shift;      // tok0's place in its sequence; keys seen by place i: min(nk, i + shift) (not causal: nk)
  int k0, nk, hk;     // first packed key, keys, K / V head
  int n0, n1;         // key tiles of the query tiles
  int part, of;       // which part of how many
  int lim0, jfix;     // keys that tok0 sees (the fewest); V tiles from jfix on reach past them
  int done;
};

__device__ __forceinline__ int least(int x, int y) { return x < y ? x : y; }
__device__ __forceinline__ int most(int x, int y) { return x > y ? x : y; }
__device__ __forceinline__ int clip(int x, int lo, int hi) { return most(lo, least(x, hi)); }

struct Seq {
  int q0, nq, k0, nk;
};
// Sequence b.  Whatever the offsets hold, its rows stay inside the tensors.
__device__ __forceinline__ Seq seq_at(const ItemArgs& a, int b) {
  const int qa = a.cu_q[b], qb = a.cu_q[b + 1], ka = a.cu_k[b], kb = a.cu_k[b + 1];
  Seq s;
  s.q0 = clip(qa, 0, int(a.Tq));
  s.nq = most(0, clip(qb, 0, int(a.Tq)) - s.q0);  // (clipped on both sides: -2^31 - q0 would wrap)
  s.k0 = clip(ka, 0, int(a.Tk));
  s.nk = most(0, clip(kb, 0, int(a.Tk)) - s.k0);
  return s;
}
// keys that place i of a sequence sees; key tiles of query tile t of the pair at i0
__device__ __forceinline__ int sees(const ItemArgs& a, const Seq& s, int i) {
  return a.causal ? clip(i + s.nk - s.nq + 1, 0, s.nk) : s.nk;
}
__device__ __forceinline__ int tiles(const ItemArgs& a, const Seq& s, int i0, int t) {
  const int first = i0 + t * a.ntok, last = least(first + a.ntok, s.nq) - 1;
  return last >= first ? (sees(a, s, last) + BN - 1) / BN : 0;
}
__device__ __forceinline__ int parts_of(const ItemArgs& a, const Seq& s, int pair) {
  const int i0 = pair * 2 * a.ntok;
  return most(1, least(a.splits, most(tiles(a, s, i0, 0), tiles(a, s, i0, 1)) / MIN_PART));
}

// Parts of the key range of a packed token (the whole warp calls); 1 for a token of no sequence.
__device__ __forceinline__ int parts_of_token(const ItemArgs& a, int tok, int lane) {
  int lo = 0, hi = a.B;  // the last sequence that starts at or before it, 32 probes at a time
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, at = lo + lane * step;
    const unsigned m = __ballot_sync(0xffffffffu, at < hi && a.cu_q[at < hi ? at : lo] <= tok);
    const int last = m ? 31 - __clz(m) : 0;
    lo = lo + last * step;
    hi = least(hi, lo + step);
  }
  const Seq s = seq_at(a, lo);
  return tok >= s.q0 && tok < s.q0 + s.nq ? parts_of(a, s, (tok - s.q0) / (2 * a.ntok)) : 1;
}

// By one lane: the item, or part `part` of it.
__device__ __forceinline__ void fill(const ItemArgs& a, const Seq& s, int pair, int hk, int part, int of, Item* m) {
  const int i0 = pair * 2 * a.ntok, t0 = tiles(a, s, i0, 0), t1 = tiles(a, s, i0, 1), n = most(t0, t1);
  // (an item without parts: plain numbers, no division)
  const int j0 = of == 1 ? 0 : int((int64_t)n * part / of), j1 = of == 1 ? n : int((int64_t)n * (part + 1) / of);
  m->tok0 = s.q0 + i0;
  m->tok_end = s.q0 + s.nq;
  m->i0 = i0;
  m->shift = a.causal ? s.nk - s.nq + 1 - j0 * BN : 0x3fffffff;
  m->k0 = s.k0 + j0 * BN;
  m->nk = least(s.nk, j1 * BN) - j0 * BN;
  m->hk = hk;
  m->n0 = most(0, least(t0, j1) - j0);
  m->n1 = most(0, least(t1, j1) - j0);
  m->lim0 = clip(sees(a, s, i0) - j0 * BN, 0, m->nk);
  m->jfix = m->lim0 / BN;
  m->part = part;
  m->of = of;
  m->done = 0;
}

// Item number -> (sequence, pair within it), by the scheduler warp.  Up to 32 sequences (a lane
// for each): by descending end of the pair's key range, so that the longest items come first and
// the last blocks' shares are even; more: sequence after sequence, the last pair first, from a
// cursor, which a number behind it sets back (a block's numbers mostly grow, but nothing promises it).  Rows behind the last sequence (a padded batch) come
// last, as the pairs of one more sequence, which has no keys.
struct Finder {
  static constexpr int PAD = 32;
  Seq mine;    // this lane's sequence (of 32 from cur_b)
  int n;       // its pairs
  int behind;  // end of the last sequence
  int low, top, total, cur_b, cur_at;

  // the sequence of find's answer, in its lane (the padding: in lane 0)
  __device__ Seq of(const ItemArgs& a, int who) const {
    const int end = clip(behind, 0, int(a.Tq));
    return who == PAD ? Seq{end, int(a.Tq) - end, 0, 0} : mine;
  }
  __device__ void load(const ItemArgs& a, int lane) {
    const int b = cur_b + lane;
    mine = Seq{0, 0, 0, 0};
    n = 0;
    if (b < a.B) {
      mine = seq_at(a, b);
      n = (mine.nq + 2 * a.ntok - 1) / (2 * a.ntok);
    }
    total = __reduce_add_sync(0xffffffffu, n);
    low = __reduce_min_sync(0xffffffffu, n ? end_of(a, 0) : 0x7fffffff);
    top = __reduce_max_sync(0xffffffffu, n ? end_of(a, n - 1) : -0x7fffffff);
  }
  // a pair's key range ends here (or at the sequence's end)
  __device__ int end_of(const ItemArgs& a, int pair) const { return mine.nk - mine.nq + (pair + 1) * 2 * a.ntok; }
  __device__ void init(const ItemArgs& a, int lane) {
    behind = a.cu_q[a.B];
    cur_b = cur_at = 0;
    load(a, lane);
  }
  // pairs that end at x or later
  __device__ int above(const ItemArgs& a, int x) const {
    const int before = most(0, x - end_of(a, 0) + 2 * a.ntok - 1) / (2 * a.ntok);
    return __reduce_add_sync(0xffffffffu, most(0, n - before));
  }
  // -> the lane of the sequence, PAD, or -1 behind the last item
  __device__ int find(const ItemArgs& a, int idx, int lane, int& pair) {
    if (idx < cur_at) {
      cur_b = cur_at = 0;
      load(a, lane);
    }
    while (idx >= cur_at + total) {
      if (cur_b + 32 >= a.B) {
        pair = idx - cur_at - total;
        return pair * int64_t(2 * a.ntok) < a.Tq - clip(behind, 0, int(a.Tq)) ? PAD : -1;
      }
      cur_at += total;
      cur_b += 32;
      load(a, lane);
    }
    const int r = idx - cur_at;
    if (a.B > 32) {
      int inc = n;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
      }
      const int l = __ffs(__ballot_sync(0xffffffffu, r < inc)) - 1;
      pair = __shfl_sync(0xffffffffu, inc, l) - 1 - r;
      return l;
    }
    int lo = low, hi = top + 1;  // above(lo) > r >= above(hi)
    while (hi - lo > 1) {
      const int mid = lo + (hi - lo) / 2;
      if (above(a, mid) > r) lo = mid; else hi = mid;
    }
    // the sequences that have a pair with this end, at most one each
    const int off = lo - end_of(a, 0), at = off >= 0 && off % (2 * a.ntok) == 0 ? off / (2 * a.ntok) : n;
    const unsigned have = __ballot_sync(0xffffffffu, at < n);
    const int rank = r - above(a, hi);
    const int l = __ffs(__ballot_sync(0xffffffffu, at < n && __popc(have & ((1u << lane) - 1)) == rank)) - 1;
    pair = __shfl_sync(0xffffffffu, at, most(l, 0));
    return l;
  }
};

}  // namespace gqa
}  // namespace mzb
