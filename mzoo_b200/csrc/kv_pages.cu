// Pages of a K / V cache: writing new rows into their pages, taking, sharing (fork),
// releasing and compacting pages.  No counterpart in the reference.
//
// The state is on the device and is changed on the caller's stream, so a serving step needs
// no host read: page_table int32 [S, W] (-1 = no page), seq_lens int32 [S], refs int32 [P]
// (how many tables name the page; 0 = free).  New pages are always the lowest free ids, in
// the order of the sequences that ask, so equal inputs give equal tables.  What cannot be
// done (a position past the table, a page id outside the pool, no free page) is left out and
// recorded in the error word, the first cause staying: MZB_ERR_TABLE, MZB_ERR_PAGES, MZB_ERR_NO_PAGE.
//
// Rows and pages move at HBM's rate (B200: 19700 rows of 2 x 2 KB written in 30 us = 5.4 TB/s of reads
// and writes, 2048 moves of 2 x 64 KB in 86 us = 6.2 TB/s); the planning kernels are chains of dependent
// look-ups in small tables (a fork of 8 sequences into 64: 10 us; compaction of 8192 pages: 9 us), so
// they are one block, or one cluster where the table's cells are many.
#include "tc.cuh"

namespace mzb {
namespace pages {

constexpr int NT = 1024;  // threads of the single-block planning kernels

// ---------------------------------------------------------------- block-wide helpers

// Exclusive prefix sum of one value per thread over a block of NT threads, and the total.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();  // the previous call's readers are done with warp_sums
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += y;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[31];
  return x - v + (warp ? warp_sums[warp - 1] : 0);
}

constexpr int PT = 8;  // consecutive elements of a thread in the scans

__device__ __forceinline__ void load_refs(const int32_t* refs, int64_t p0, int64_t P, int32_t none, int32_t (&r)[PT]) {
  if (p0 + PT <= P && (reinterpret_cast<uintptr_t>(refs) & 15) == 0) {
#pragma unroll
    for (int e = 0; e < PT; e += 4) {
      const int4 x = __ldcg(reinterpret_cast<const int4*>(refs + p0 + e));
      r[e] = x.x;
      r[e + 1] = x.y;
      r[e + 2] = x.z;
      r[e + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < PT; ++e) r[e] = p0 + e < P ? __ldcg(refs + p0 + e) : none;
  }
}

// The lowest `want` free pages, ascending, into list; returns how many there are (<= want).
__device__ int lowest_free(const int32_t* refs, int64_t P, int want, int32_t* list, int* warp_sums) {
  int found = 0;
  for (int64_t c0 = 0; c0 < P && found < want; c0 += NT * PT) {
    const int64_t p0 = c0 + threadIdx.x * PT;
    int32_t r[PT];
    load_refs(refs, p0, P, 1, r);
    int f = 0, total;
#pragma unroll
    for (int e = 0; e < PT; ++e) f += r[e] == 0;
    int at = found + block_scan(f, warp_sums, total);
#pragma unroll
    for (int e = 0; e < PT; ++e)
      if (r[e] == 0 && at < want) list[at++] = int32_t(p0 + e);
    found += total;
  }
  __syncthreads();
  return min(found, want);
}

__device__ __forceinline__ void report(int* err, int code) { atomicCAS(err, 0, code); }

// ---------------------------------------------------------------- append

struct AppendArgs {
  const uint8_t *k, *v;
  uint8_t *kp, *vp;
  const int32_t *table, *starts, *cu;
  int64_t T, P, sk_t, sk_h, sv_t, sv_h, kp_p, kp_h, kp_t, vp_p, vp_h, vp_t;  // byte strides
  int B, H, chunks, W, page, tok;                                          // chunks: 16-byte pieces of a row
  int* err;
};

constexpr int AP_TOK = 8, AP_IN_FLIGHT = 4;  // tokens of a block, K and V pieces of a thread

// A copy: bound by HBM.  The rows are requested before their places are known, so that the
// search for the sequence and the table's look-up (three dependent loads) pass while they are
// on their way.
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
  __shared__ int64_t kdst[AP_TOK], vdst[AP_TOK];
  const int64_t t0 = (int64_t)blockIdx.x * a.tok;
  const int nt = int(min((int64_t)a.tok, a.T - t0)), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = a.H * a.chunks, n = nt * per;
  uint4 kv[AP_IN_FLIGHT], vv[AP_IN_FLIGHT];
  auto request = [&](int x0) {
#pragma unroll
    for (int i = 0; i < AP_IN_FLIGHT; ++i) {
      const int x = x0 + 256 * i;
      if (x < n) {
        const int t = x / per, y = x % per, h = y / a.chunks, c = y % a.chunks;
        kv[i] = __ldcs(reinterpret_cast<const uint4*>(a.k + (t0 + t) * a.sk_t + h * a.sk_h + c * 16));
        vv[i] = __ldcs(reinterpret_cast<const uint4*>(a.v + (t0 + t) * a.sv_t + h * a.sv_h + c * 16));
      }
    }
  };
  request(threadIdx.x);
  if (warp < nt) {  // a warp for each token
    const int64_t t = t0 + warp;
    int b = int(t);
    int64_t i = 0;
    bool ok = true;
    if (a.cu) {
      int lo = 0, hi = a.B;  // the last sequence that starts at or before t, 32 probes at a time
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned m = __ballot_sync(0xffffffffu, at < hi && a.cu[at < hi ? at : lo] <= t);
        const int last = m ? 31 - __clz(m) : 0;
        lo = lo + last * step;
        hi = min(hi, lo + step);
      }
      b = lo;
      const int q0 = a.cu[b], q1 = a.cu[b + 1];
      i = t - q0;
      ok = i >= 0 && t < q1;
    }
    if (lane == 0) {
      int64_t d = -1, e = -1;
      if (ok) {
        const int64_t pos = (int64_t)a.starts[b] + i, j = pos / a.page;
        const bool there = pos >= 0 && j < a.W;
        if (there) {
          const int64_t p = a.table[(int64_t)b * a.W + j];
          if (p >= 0 && p < a.P) {
            d = p * a.kp_p + (pos % a.page) * a.kp_t;
            e = p * a.vp_p + (pos % a.page) * a.vp_t;
          }
        }
        if (d < 0) report(a.err, there ? MZB_ERR_PAGES : MZB_ERR_TABLE);
      }
      kdst[warp] = d;
      vdst[warp] = e;
    }
  }
  __syncthreads();
  for (int x0 = threadIdx.x; x0 < n; x0 += 256 * AP_IN_FLIGHT) {
    if (x0 >= 256 * AP_IN_FLIGHT) request(x0);
#pragma unroll
    for (int i = 0; i < AP_IN_FLIGHT; ++i) {
      const int x = x0 + 256 * i;
      if (x < n) {
        const int t = x / per, y = x % per, h = y / a.chunks, c = y % a.chunks;
        if (kdst[t] >= 0) {
          *reinterpret_cast<uint4*>(a.kp + kdst[t] + h * a.kp_h + c * 16) = kv[i];
          *reinterpret_cast<uint4*>(a.vp + vdst[t] + h * a.vp_h + c * 16) = vv[i];
        }
      }
    }
  }
}

// ---------------------------------------------------------------- reserve

// One block: needs per sequence, their prefix sum, the lowest free pages, the table entries.  A sequence whose sum
// passes the number of free pages gets none, and so does every one behind it: no one is passed over.
__global__ void __launch_bounds__(NT) reserve_kernel(int32_t* table, int32_t* lens, int32_t* refs,
                                                     const int32_t* n_new, int32_t* starts, int32_t* list, int B,
                                                     int W, int64_t P, int page, int* err) {
  __shared__ int ws[32];
  int base = 0;
  // pass 0 counts what is wanted, pass 1 gives it out
  int have = 0;
  for (int pass = 0; pass < 2; ++pass) {
    int run = 0;
    for (int b0 = 0; b0 < B; b0 += NT) {
      const int b = b0 + threadIdx.x;
      int need = 0, j0 = 0, j1 = 0;
      int64_t len = 0, to = 0;
      bool ok = false;
      if (b < B) {
        len = lens[b];
        to = len + n_new[b];
        ok = len >= 0 && n_new[b] >= 0 && to <= (int64_t)W * page;
        if (ok) {
          j0 = int((len + page - 1) / page);
          j1 = int((to + page - 1) / page);
          for (int j = j0; j < j1; ++j) need += table[(int64_t)b * W + j] < 0;
        }
      }
      int total;
      const int at = run + block_scan(need, ws, total);
      run += total;
      if (pass == 1 && b < B) {
        starts[b] = int32_t(len);
        if (ok && (need == 0 || at + need <= have)) {
          int r = at;
          for (int j = j0; j < j1; ++j)
            if (table[(int64_t)b * W + j] < 0) {
              const int32_t p = list[r++];
              table[(int64_t)b * W + j] = p;
              refs[p] = 1;
            }
          lens[b] = int32_t(to);
        } else {
          report(err, ok ? MZB_ERR_NO_PAGE : MZB_ERR_TABLE);
        }
      }
      __syncthreads();
    }
    if (pass == 0) {
      base = run;
      have = lowest_free(refs, P, int(min((int64_t)base, P)), list, ws);
    }
  }
}

// ---------------------------------------------------------------- free

// Exchanging the table entry for -1 makes a sequence named twice harmless.
__global__ void __launch_bounds__(256) free_kernel(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* seqs,
                                                   int64_t n, int64_t S, int W, int64_t P, int* err) {
  const int64_t i = blockIdx.y + (int64_t)gridDim.y * blockIdx.z;
  if (i >= n) return;
  const int64_t s = seqs[i];
  if (s < 0 || s >= S) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report(err, MZB_ERR_PAGES);
    return;
  }
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j == 0) lens[s] = 0;
  if (j >= W) return;
  const int p = atomicExch(&table[s * W + j], -1);
  if (p >= 0 && p < P) atomicSub(&refs[p], 1);
}

// ---------------------------------------------------------------- fork

// One cluster of FORK_CTAS blocks, which share the table's cells and meet at cluster barriers
// (a release / acquire of global memory too).  ws: pairs_src [n], pairs_dst [n], list [n], mark [S].
constexpr int FORK_CTAS = 8;

__global__ void __cluster_dims__(FORK_CTAS, 1, 1) __launch_bounds__(NT)
    fork_kernel(int32_t* table, int32_t* lens, int32_t* refs, const int32_t* src, const int32_t* dst, int n, int32_t* ws,
                int64_t S, int W, int64_t P, int page, int* err) {
  __shared__ int wsum[32];
  int32_t *ps = ws, *pd = ws + n, *list = ws + 2 * (int64_t)n, *mark = ws + 3 * (int64_t)n;
  const int tid = blockIdx.x * NT + threadIdx.x;
  constexpr int ALL = FORK_CTAS * NT;
  auto in = [&](int64_t s) { return s >= 0 && s < S; };
  // a pair is taken if both names are in the table, dst is named once and is no one's src
  for (int i = tid; i < n; i += ALL) {
    const int s = src[i], d = dst[i];
    if (in(s)) mark[s] = 0;
    if (in(d)) mark[d] = 0;
  }
  tc::cluster_sync();
  for (int i = tid; i < n; i += ALL) {
    const int s = src[i], d = dst[i];
    if (in(s)) atomicOr(&mark[s], 1 << 30);
    if (in(d)) atomicAdd(&mark[d], 1);
  }
  tc::cluster_sync();
  // full pages of pair i, -1: not taken
  auto full_of = [&](int i) {
    const int64_t s = src[i], d = dst[i];
    if (!in(s) || !in(d)) return -1;
    const int len = lens[s], m = __ldcg(&mark[d]);
    return m == 1 && len >= 0 && len <= (int64_t)W * page ? len / page : -1;
  };
  // a warp for each pair: what dst held is released, src's full pages are shared.  The counts of a page
  // only add up, and no source row is written, so the order does not matter.
  for (int i = tid >> 5; i < n; i += ALL / 32) {
    const int full = full_of(i);
    if (full < 0) continue;
    int32_t* to = table + (int64_t)dst[i] * W;
    const int32_t* from = table + (int64_t)src[i] * W;
    for (int j0 = threadIdx.x & 31; j0 < W; j0 += 32 * 8) {
      int was[8], now[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = j0 + 32 * e;
        was[e] = j < W ? to[j] : -1;
        now[e] = j < full ? from[j] : -1;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int j = j0 + 32 * e;
        if (j >= W) continue;
        const bool share = now[e] >= 0 && now[e] < P;
        if (j < full && !share) report(err, MZB_ERR_PAGES);
        if (was[e] != -1 || share) to[j] = share ? now[e] : -1;
        if (was[e] >= 0 && was[e] < P) atomicSub(&refs[was[e]], 1);
        if (share) atomicAdd(&refs[now[e]], 1);
      }
    }
  }
  tc::cluster_sync();
  if (blockIdx.x) return;
  int want = 0;
  for (int i0 = 0; i0 < n; i0 += NT) {  // ranks of the copies that need a page of their own
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < n) {
      ps[i] = pd[i] = -1;
      const int full = full_of(i);
      if (full < 0) {
        report(err, MZB_ERR_PAGES);
      } else if (lens[src[i]] % page) {
        const int p = table[(int64_t)src[i] * W + full];
        if (p >= 0 && p < P) {
          need = 1;
          ps[i] = p;
        } else {
          report(err, MZB_ERR_PAGES);
        }
      }
    }
    int total;
    const int at = want + block_scan(need, wsum, total);
    if (i < n && need) pd[i] = at;
    want += total;
  }
  __syncthreads();
  const int have = lowest_free(refs, P, want, list, wsum);
  for (int i = threadIdx.x; i < n; i += NT) {
    const int full = full_of(i);
    if (full < 0) continue;
    const int64_t d = dst[i];
    const int len = lens[src[i]];
    int32_t got = len;
    if (len % page) {
      const int32_t p = pd[i] >= 0 && pd[i] < have ? list[pd[i]] : -1;
      if (p >= 0) {
        table[d * W + full] = p;
        refs[p] = 1;
      } else {  // no page for the last tokens: the copy ends at its last full page
        if (pd[i] >= 0) report(err, MZB_ERR_NO_PAGE);
        got = full * page;
        ps[i] = -1;
      }
      pd[i] = p;
    }
    lens[d] = got;
  }
}

// ---------------------------------------------------------------- compact

// One block.  The i-th live page at an index >= n moves to the i-th hole below n (n = number
// of live pages), so the pages that move and the holes are disjoint and the copies need no
// order.  to [P]: where a page is afterwards (-1: free); (from, hole) lists of m = count[0] moves.
__global__ void __launch_bounds__(NT) compact_plan_kernel(const int32_t* refs, int32_t* new_refs, int32_t* to,
                                                          int32_t* from_list, int32_t* hole_list, int32_t* count,
                                                          int64_t P) {
  __shared__ int ws[32];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  int n, mine = 0;
  int32_t first[PT];  // the first chunk stays in registers
  load_refs(refs, threadIdx.x * PT, P, 0, first);
#pragma unroll
  for (int e = 0; e < PT; ++e) mine += first[e] > 0;
  for (int64_t p0 = (NT + threadIdx.x) * PT; p0 < P; p0 += NT * PT) {
    int32_t r[PT];
    load_refs(refs, p0, P, 0, r);
#pragma unroll
    for (int e = 0; e < PT; ++e) mine += r[e] > 0;
  }
  block_scan(mine, ws, n);
  int holes = 0, moved = 0;
  for (int64_t c0 = 0; c0 < P; c0 += NT * PT) {
    const int64_t p0 = c0 + threadIdx.x * PT;
    int32_t r[PT], goes[PT], left[PT];
    if (c0 == 0) {
#pragma unroll
      for (int e = 0; e < PT; ++e) r[e] = first[e];
    } else {
      load_refs(refs, p0, P, 0, r);
    }
    int hm = 0, total;  // holes in the low half, moves in the high half: at most NT * PT each
#pragma unroll
    for (int e = 0; e < PT; ++e) hm += p0 + e < n ? (r[e] <= 0) : (r[e] > 0) << 16;
    const int at = block_scan(hm, ws, total);
    int ah = holes + (at & 0xffff), am = moved + (at >> 16);
    holes += total & 0xffff;
    moved += total >> 16;
#pragma unroll
    for (int e = 0; e < PT; ++e) {
      const int64_t p = p0 + e;
      if (p < n) {
        if (r[e] <= 0) hole_list[ah++] = int32_t(p);
      } else if (r[e] > 0) {
        from_list[am++] = int32_t(p);
      }
      goes[e] = r[e] > 0 ? int32_t(p) : -1;
      left[e] = p < n && r[e] > 0 ? r[e] : 0;
    }
    if (p0 + PT <= P && ((reinterpret_cast<uintptr_t>(to) | reinterpret_cast<uintptr_t>(new_refs)) & 15) == 0) {
#pragma unroll
      for (int e = 0; e < PT; e += 4) {
        *reinterpret_cast<int4*>(to + p0 + e) = make_int4(goes[e], goes[e + 1], goes[e + 2], goes[e + 3]);
        *reinterpret_cast<int4*>(new_refs + p0 + e) = make_int4(left[e], left[e + 1], left[e + 2], left[e + 3]);
      }
    } else {
      for (int e = 0; e < PT && p0 + e < P; ++e) {
        to[p0 + e] = goes[e];
        new_refs[p0 + e] = left[e];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < moved; i += NT) {
    const int f = from_list[i], h = hole_list[i];
    to[f] = h;
    new_refs[h] = refs[f];
  }
  if (threadIdx.x == 0) count[0] = moved;
}

// ---------------------------------------------------------------- copying pages

constexpr int MAX_POOLS = 64;
constexpr int CHUNK = 16384;  // bytes of a page that one block step copies: 256 threads x 4 x 16
constexpr int COPY_BLOCKS = 32;  // blocks per SM at most: 8 resident ones that stay take 5 % longer, more empty ones cost too

struct CopyArgs {
  uint8_t* pool[MAX_POOLS];
  int64_t stride[MAX_POOLS];  // bytes from page to page
  int64_t bytes[MAX_POOLS];   // bytes of a page
  const int32_t *src, *dst;   // src or dst -1: no copy
  const int32_t* count;       // device count of pairs (null: n)
  int64_t n, P;
  int n_pools, chunks;  // chunks of the largest page
  int* err;
  // a page table to rewrite with a map of the pages (null: none)
  const int32_t *table, *to;
  int32_t* new_table;
  int64_t entries;
};

__global__ void __launch_bounds__(256) copy_kernel(const __grid_constant__ CopyArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");  // behind the kernel that made the lists
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * 256) {
    const int p = a.table[i];
    int q = -1;
    if (p >= 0) {
      q = p < a.P ? a.to[p] : -1;
      if (q < 0) report(a.err, MZB_ERR_PAGES);  // a table names a free page or none of the pool's
    }
    a.new_table[i] = q;
  }
  const int64_t n = a.count ? min((int64_t)*a.count, a.n) : a.n;
  const int64_t per = (int64_t)a.n_pools * a.chunks;
  for (int64_t w = blockIdx.x; w < n * per; w += gridDim.x) {
    const int64_t i = w / per;
    const int pool = int(w % per) / a.chunks, c = int(w % per) % a.chunks;
    const int64_t s = a.src[i], d = a.dst[i];
    if (s < 0 && d < 0) continue;
    if (s < 0 || d < 0 || s >= a.P || d >= a.P) {
      if (threadIdx.x == 0) report(a.err, MZB_ERR_PAGES);
      continue;
    }
    const int64_t off = (int64_t)c * CHUNK, left = a.bytes[pool] - off;
    const uint4* from = reinterpret_cast<const uint4*>(a.pool[pool] + s * a.stride[pool] + off);
    uint4* to = reinterpret_cast<uint4*>(a.pool[pool] + d * a.stride[pool] + off);
    uint4 v[CHUNK / 4096];
    if (left >= CHUNK) {
#pragma unroll
      for (int q = 0; q < CHUNK / 4096; ++q) v[q] = from[threadIdx.x + 256 * q];
#pragma unroll
      for (int q = 0; q < CHUNK / 4096; ++q) to[threadIdx.x + 256 * q] = v[q];
    } else {
#pragma unroll
      for (int q = 0; q < CHUNK / 4096; ++q)
        if ((int64_t)(threadIdx.x + 256 * q) * 16 < left) v[q] = from[threadIdx.x + 256 * q];
#pragma unroll
      for (int q = 0; q < CHUNK / 4096; ++q)
        if ((int64_t)(threadIdx.x + 256 * q) * 16 < left) to[threadIdx.x + 256 * q] = v[q];
    }
  }
}

// One launch for up to MAX_POOLS pools, allowed to start while the kernel before it runs.
int copy_pages(const int64_t* pools, int n_pools, CopyArgs a, const char* what, cudaStream_t st) {
  for (int i = 0; i < n_pools; ++i)
    MZB_REQUIRE(pools[3 * i] % 16 == 0 && pools[3 * i + 1] >= 16 && pools[3 * i + 1] % 16 == 0 && pools[3 * i + 2] % 16 == 0,
                MZB_ERR_ALIGN, "%s: pool %d: pages must be 16-byte aligned and multiples of 16 bytes", what, i);
  for (int p0 = 0; p0 < n_pools || (p0 == 0 && a.entries); p0 += MAX_POOLS) {
    a.n_pools = n_pools - p0 < MAX_POOLS ? n_pools - p0 : MAX_POOLS;
    int64_t most = 16;
    for (int i = 0; i < a.n_pools; ++i) {
      const int64_t* x = pools + 3 * (p0 + i);
      a.pool[i] = reinterpret_cast<uint8_t*>(x[0]);
      a.bytes[i] = x[1];
      a.stride[i] = x[2];
      most = most > a.bytes[i] ? most : a.bytes[i];
    }
    a.chunks = int((most + CHUNK - 1) / CHUNK);
    const int64_t work = a.n * a.n_pools * a.chunks, rows = (a.entries + 255) / 256, cap = COPY_BLOCKS * num_sms();
    const int64_t want = work > rows ? work : rows;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(unsigned(want < 1 ? 1 : want < cap ? want : cap));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, copy_kernel, a);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("%s: launch failed: %s", what, cudaGetErrorString(e));
      return MZB_ERR_LAUNCH;
    }
    a.entries = 0;
  }
  return MZB_OK;
}

}  // namespace pages
}  // namespace mzb

using namespace mzb;

#define MZB_POOL_SIZES(what, P, W, page)                                                                            \
  MZB_REQUIRE((P) >= 1 && (P) < (int64_t(1) << 31) && (W) >= 1 && (page) >= 1 &&                                    \
                  (int64_t)(W) * (page) < (int64_t(1) << 31),                                                       \
              MZB_ERR_SHAPE, what ": bad sizes pages=%lld table width=%d page=%d", (long long)(P), int(W), int(page)); \
  MZB_REQUIRE(err != nullptr, MZB_ERR_SHAPE, what ": needs an error word")

extern "C" int mzb_kv_append(const void* k, const void* v, void* k_pages, void* v_pages, const int32_t* page_table,
                             const int32_t* starts, const int32_t* cu, int64_t T, int B, int Hkv, int row_bytes,
                             int page, int64_t P, int W, int elem_bytes, const int64_t* strides, int* err,
                          void* stream) {
  MZB_POOL_SIZES("kv_append", P, W, page);
  MZB_REQUIRE(T >= 0 && B >= 1 && Hkv >= 1 && (cu != nullptr || T == B), MZB_ERR_SHAPE,
              "kv_append: bad sizes T=%lld B=%d Hkv=%d", (long long)T, B, Hkv);
  MZB_REQUIRE(row_bytes >= 16 && row_bytes % 16 == 0, MZB_ERR_ALIGN, "kv_append: rows of %d bytes (a multiple of 16)",
              row_bytes);
  for (const void* p : {k, v, (const void*)k_pages, (const void*)v_pages})
    MZB_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, MZB_ERR_ALIGN, "kv_append: pointers must be 16-byte aligned");
  MZB_REQUIRE(elem_bytes >= 1 && elem_bytes <= 16, MZB_ERR_UNSUPPORTED, "kv_append: elements of %d bytes", elem_bytes);
  int64_t sb[10];
  for (int i = 0; i < 10; ++i) {
    sb[i] = strides[i] * elem_bytes;
    // the stride of a single head, slot or page is never used
    const bool one = (i == 1 || i == 3 || i == 5 || i == 8) ? Hkv == 1 : (i == 4 || i == 7) ? P == 1 : (i == 6 || i == 9) ? page == 1 : T == 1;
    if (one) sb[i] = 0;
    MZB_REQUIRE(sb[i] % 16 == 0, MZB_ERR_ALIGN, "kv_append: strides must be multiples of 16 bytes");
  }
  if (T == 0) return MZB_OK;
  // tokens of a block (8 heads of 256 bytes, with 1, 4, 8): 592 rows 4.6, 4.9, 5.4 us; 2368 rows 12.3, 6.8, 7.2; 4736 rows
  // 21.4, 11.0, 9.6; one head: 64 rows 4.0, 3.6, 3.6, 592 4.2, 3.9, 4.0, 2368 11.4, 4.2, 4.3, 4736 19.9, 6.6, 4.4
  const int tok = T <= 4 * num_sms() ? 1 : T <= 16 * num_sms() ? 4 : pages::AP_TOK;
  pages::AppendArgs a{static_cast<const uint8_t*>(k), static_cast<const uint8_t*>(v), static_cast<uint8_t*>(k_pages),
                      static_cast<uint8_t*>(v_pages), page_table, starts, cu, T, P, sb[0], sb[1],
                      sb[2], sb[3], sb[4], sb[5], sb[6], sb[7], sb[8], sb[9],
                      B, Hkv, row_bytes / 16, W, page, tok, err};
  pages::append_kernel<<<unsigned((T + tok - 1) / tok), 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status("kv_append");
}

extern "C" int mzb_kv_reserve(int32_t* page_table, int32_t* seq_lens, int32_t* refs, const int32_t* n_new,
                              int32_t* starts, int32_t* ws, int B, int W, int64_t P, int page, int* err,
                              void* stream) {
  MZB_POOL_SIZES("kv_reserve", P, W, page);
  MZB_REQUIRE(B >= 0, MZB_ERR_SHAPE, "kv_reserve: bad B=%d", B);
  if (B == 0) return MZB_OK;
  pages::reserve_kernel<<<1, pages::NT, 0, static_cast<cudaStream_t>(stream)>>>(page_table, seq_lens, refs, n_new,
                                                                                starts, ws, B, W, P, page, err);
  return launch_status("kv_reserve");
}

extern "C" int mzb_kv_free(int32_t* page_table, int32_t* seq_lens, int32_t* refs, const int32_t* seqs, int64_t n,
                           int64_t S, int W, int64_t P, int* err, void* stream) {
  MZB_POOL_SIZES("kv_free", P, W, 1);
  MZB_REQUIRE(n >= 0 && n < (int64_t(1) << 31) && S >= 1, MZB_ERR_SHAPE, "kv_free: bad sizes n=%lld S=%lld",
              (long long)n, (long long)S);
  if (n == 0) return MZB_OK;
  const unsigned ny = unsigned(n < 65535 ? n : 65535), nz = unsigned((n + ny - 1) / ny);
  pages::free_kernel<<<dim3(unsigned((W + 255) / 256), ny, nz), 256, 0, static_cast<cudaStream_t>(stream)>>>(
      page_table, seq_lens, refs, seqs, n, S, W, P, err);
  return launch_status("kv_free");
}

extern "C" int mzb_kv_fork(int32_t* page_table, int32_t* seq_lens, int32_t* refs, const int32_t* src,
                           const int32_t* dst, int n, int32_t* ws, int64_t S, int W, int64_t P, int page,
                           const int64_t* pools, int n_pools, int* err, void* stream) {
  MZB_POOL_SIZES("kv_fork", P, W, page);
  MZB_REQUIRE(n >= 0 && S >= 1 && S < (int64_t(1) << 31) && n_pools >= 0, MZB_ERR_SHAPE, "kv_fork: bad sizes n=%d S=%lld", n,
              (long long)S);
  if (n == 0) return MZB_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  pages::fork_kernel<<<pages::FORK_CTAS, pages::NT, 0, st>>>(page_table, seq_lens, refs, src, dst, n, ws, S, W, P, page, err);
  if (int r = launch_status("kv_fork")) return r;
  pages::CopyArgs a{};
  a.src = ws; a.dst = ws + n; a.n = n; a.P = P; a.err = err;
  return pages::copy_pages(pools, n_pools, a, "kv_fork(copy)", st);
}

extern "C" int mzb_kv_compact(const int32_t* page_table, const int32_t* refs, int32_t* new_table, int32_t* new_refs,
                              int32_t* ws, int64_t entries, int64_t P, const int64_t* pools, int n_pools, int* err,
                              void* stream) {
  MZB_POOL_SIZES("kv_compact", P, 1, 1);
  MZB_REQUIRE(entries >= 0 && n_pools >= 0, MZB_ERR_SHAPE, "kv_compact: bad table size %lld", (long long)entries);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int32_t *from = ws, *hole = ws + P, *to = ws + 2 * P, *count = ws + 3 * P;
  pages::compact_plan_kernel<<<1, pages::NT, 0, st>>>(refs, new_refs, to, from, hole, count, P);
  if (int r = launch_status("kv_compact")) return r;
  pages::CopyArgs a{};
  a.src = from; a.dst = hole; a.count = count; a.n = P / 2; a.P = P; a.err = err;
  a.table = page_table; a.to = to; a.new_table = new_table; a.entries = entries;
  return pages::copy_pages(pools, n_pools, a, "kv_compact(copy)", st);
}

extern "C" int mzb_kv_copy_pages(const int64_t* pools, int n_pools, const int32_t* src, const int32_t* dst, int64_t n,
                                 int64_t P, int* err, void* stream) {
  MZB_POOL_SIZES("kv_copy_pages", P, 1, 1);
  MZB_REQUIRE(n >= 0 && n_pools >= 0, MZB_ERR_SHAPE, "kv_copy_pages: bad sizes n=%lld pools=%d", (long long)n, n_pools);
  if (n == 0) return MZB_OK;
  pages::CopyArgs a{};
  a.src = src; a.dst = dst; a.n = n; a.P = P; a.err = err;
  return pages::copy_pages(pools, n_pools, a, "kv_copy_pages", static_cast<cudaStream_t>(stream));
}
