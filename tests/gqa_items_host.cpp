// Runs csrc/gqa_items.cuh on the host: a warp is 32 fibers that meet at every collective.
// stdin:  B ntok causal splits Tq Tk seed, then cu_q and cu_k (B + 1 numbers each); seed < 0: block
//         numbers ascending, else in an order drawn from it
// stdout: "item who tok0 tok_end k0 nk n0 n1 part of" for each item that some block number stands for, then
//         "token parts" for each token
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <ucontext.h>

#include <algorithm>
#include <functional>
#include <random>
#include <vector>

#define __device__
#define __forceinline__ inline

namespace {
ucontext_t lanes[32], home;
std::vector<char> stacks[32];
int now, vals[32];
bool done[32];
std::function<void(int)> body;

void meet() { swapcontext(&lanes[now], &home); }  // until all lanes are here
void lane_main() {
  const int l = now;
  body(l);
  done[l] = true;
  swapcontext(&lanes[l], &home);
}
void warp(std::function<void(int)> f) {
  body = f;
  for (int l = 0; l < 32; ++l) {
    getcontext(&lanes[l]);
    stacks[l].resize(1 << 16);
    lanes[l].uc_stack.ss_sp = stacks[l].data();
    lanes[l].uc_stack.ss_size = stacks[l].size();
    lanes[l].uc_link = nullptr;
    done[l] = false;
    makecontext(&lanes[l], lane_main, 0);
  }
  while (true) {
    for (now = 0; now < 32; ++now)
      if (!done[now]) swapcontext(&home, &lanes[now]);
    int n = 0;
    for (bool d : done) n += d;
    if (n == 32) return;
    if (n) { fprintf(stderr, "lanes parted\n"); exit(2); }
  }
}
template <class F>
int exchange(int v, F f) {
  const int l = now;
  vals[l] = v;
  meet();
  const int r = f(l);
  meet();
  return r;
}
int __shfl_sync(unsigned, int v, int src) { return exchange(v, [=](int) { return vals[src & 31]; }); }
int __shfl_up_sync(unsigned, int v, int d) { return exchange(v, [=](int l) { return vals[l < d ? l : l - d]; }); }
unsigned __ballot_sync(unsigned, bool v) {
  return exchange(v, [](int) { unsigned m = 0; for (int i = 0; i < 32; ++i) m |= unsigned(vals[i] != 0) << i; return int(m); });
}
int __reduce_add_sync(unsigned, int v) { return exchange(v, [](int) { int s = 0; for (int x : vals) s += x; return s; }); }
int __reduce_min_sync(unsigned, int v) { return exchange(v, [](int) { return *std::min_element(vals, vals + 32); }); }
int __reduce_max_sync(unsigned, int v) { return exchange(v, [](int) { return *std::max_element(vals, vals + 32); }); }
int __ffs(unsigned x) { return x ? __builtin_ctz(x) + 1 : 0; }
int __clz(unsigned x) { return x ? __builtin_clz(x) : 32; }
int __popc(unsigned x) { return __builtin_popcount(x); }
}  // namespace

#include "gqa_items.cuh"

using namespace mzb::gqa;

int main() {
  int B, ntok, causal, splits, seed;
  long long Tq, Tk;
  if (scanf("%d %d %d %d %lld %lld %d", &B, &ntok, &causal, &splits, &Tq, &Tk, &seed) != 7) return 1;
  std::vector<int32_t> cq(B + 1), ck(B + 1);
  for (auto* v : {&cq, &ck})
    for (int& x : *v)
      if (scanf("%d", &x) != 1) return 1;
  ItemArgs a{cq.data(), ck.data(), Tq, Tk, B, ntok, causal, splits};
  const int64_t c = 2 * ntok, seqs = std::min<int64_t>(B + 1, Tq), grid = (Tq + seqs * (c - 1)) / c * splits;
  std::vector<int> order(grid);
  for (int i = 0; i < grid; ++i) order[i] = i;
  if (seed >= 0) std::shuffle(order.begin(), order.end(), std::mt19937(seed));
  Item item;
  warp([&](int lane) {
    Finder f;
    f.init(a, lane);
    for (int idx : order) {
      int pair = 0, who = f.find(a, idx / splits, lane, pair), of = 1;
      if (who < 0) continue;
      of = __shfl_sync(~0u, parts_of(a, f.of(a, who), pair), who % 32);
      if (idx % splits >= of) continue;
      if (lane == who % 32) {
        fill(a, f.of(a, who), pair, 0, idx % splits, of, &item);
        printf("item %d %d %d %d %d %d %d %d %d\n", who, item.tok0, item.tok_end, item.k0, item.nk, item.n0, item.n1, item.part, item.of);
      }
    }
    for (int t = 0; t < Tq; ++t) {
      const int n = parts_of_token(a, t, lane);
      if (lane == 0) printf("token %d\n", n);
    }
  });
}
