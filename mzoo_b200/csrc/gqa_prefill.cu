// Attention over whole prompts with grouped K / V heads: packed sequences of different
// lengths, causal (aligned to the end of the keys) or full, bf16 / f16 in and out, fp32
// accumulation, natural-log lse.  No counterpart in the reference's kernels.
//
//   x_ij = scale q_i.k_j over the keys j <= i + nk - nq of row i's sequence (all keys if not
//   causal);  o_i = sum_j e^(x_ij - lse_i) v_j,  lse_i = log sum_j e^x_ij.
//   A row that sees no key: o = 0, lse = -inf.
//
// One warp per (token, head) row with an online softmax, D / 32 channels per lane.
#include "common.cuh"

namespace mzb {
namespace gqa {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct PrefillArgs {
  const void *q, *k, *v;
  const int32_t *cu_q, *cu_k;
  void* o;
  float* lse;
  int64_t Tq, Tk, sq_t, sq_h, sk_t, sk_h, sv_t, sv_h;
  int B, Hq, Hkv, causal;
  float scale;
};

template <int DT, int D>
__global__ void __launch_bounds__(256) prefill_kernel(PrefillArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int C = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= a.Tq * a.Hq) return;
  const int64_t t = row / a.Hq;
  const int h = int(row % a.Hq), hk = h / (a.Hq / a.Hkv);
  int lo = 0, hi = a.B;  // the last sequence that starts at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  const int64_t k0 = max((int64_t)0, min((int64_t)a.cu_k[lo], a.Tk)), k1 = max(k0, min((int64_t)a.cu_k[lo + 1], a.Tk));
  const int64_t nk = k1 - k0, nq = a.cu_q[lo + 1] - a.cu_q[lo];
  int64_t n = a.causal ? min(nk, t - a.cu_q[lo] + nk - nq + 1) : nk;
  if (t < a.cu_q[lo] || t >= a.cu_q[lo + 1]) n = 0;
  float qv[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    qv[c] = E::load(static_cast<const T*>(a.q)[t * a.sq_t + h * a.sq_h + lane + 32 * c]);
    acc[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = 0; j < n; ++j) {
    const T* kr = static_cast<const T*>(a.k) + (k0 + j) * a.sk_t + hk * a.sk_h;
    const T* vr = static_cast<const T*>(a.v) + (k0 + j) * a.sv_t + hk * a.sv_h;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += qv[c] * E::load(kr[lane + 32 * c]);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale * LOG2E;
    const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.0f : mn;
    const float al = exp2f(m - ms), p = exp2f(s - ms);
    l = l * al + p;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = acc[c] * al + p * E::load(vr[lane + 32 * c]);
    m = mn;
  }
  const float inv = n > 0 ? 1.0f / l : 0.0f;
#pragma unroll
  for (int c = 0; c < C; ++c) static_cast<T*>(a.o)[row * D + lane + 32 * c] = E::store(acc[c] * inv);
  if (lane == 0) a.lse[row] = n > 0 ? (m + log2f(l)) * LN2 : -INFINITY;
}

template <int DT, int D>
int launch(const PrefillArgs& a, cudaStream_t st) {
  prefill_kernel<DT, D><<<unsigned((a.Tq * a.Hq + 7) / 8), 256, 0, st>>>(a);
  return launch_status("gqa_prefill");
}

}  // namespace gqa
}  // namespace mzb

using namespace mzb;

extern "C" int mzb_gqa_prefill(const void* q, const void* k, const void* v, const int32_t* cu_q, const int32_t* cu_k,
                               void* o, float* lse, int64_t Tq, int64_t Tk, int B, int Hq, int Hkv, int D, int dtype,
                               int64_t sq_t, int64_t sq_h, int64_t sk_t, int64_t sk_h, int64_t sv_t, int64_t sv_h,
                               int causal, float softmax_scale, int* err, void* stream) {
  MZB_REQUIRE(Tq >= 0 && Tk >= 0 && B >= 1 && Tq < (int64_t(1) << 31) && Tk < (int64_t(1) << 31), MZB_ERR_SHAPE,
              "gqa_prefill: bad sizes Tq=%lld Tk=%lld B=%d", (long long)Tq, (long long)Tk, B);
  MZB_REQUIRE(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 128, MZB_ERR_SHAPE,
              "gqa_prefill: query heads must be a multiple (at most 128) of the K/V heads, got %d and %d", Hq, Hkv);
  MZB_REQUIRE(D == 64 || D == 96 || D == 128, MZB_ERR_UNSUPPORTED, "gqa_prefill: unsupported head dim %d", D);
  MZB_REQUIRE(dtype == MZB_BF16 || dtype == MZB_F16, MZB_ERR_UNSUPPORTED, "gqa_prefill: unsupported dtype %d", dtype);
  MZB_REQUIRE(err != nullptr, MZB_ERR_SHAPE, "gqa_prefill: needs an error word");
  if (Tq == 0) return MZB_OK;
  gqa::PrefillArgs a{q, k, v, cu_q, cu_k, o, lse, Tq, Tk, sq_t, sq_h, sk_t, sk_h, sv_t, sv_h, B, Hq, Hkv, causal,
                     softmax_scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MZB_BF16)
    return D == 64 ? gqa::launch<MZB_BF16, 64>(a, st) : D == 96 ? gqa::launch<MZB_BF16, 96>(a, st)
                                                                : gqa::launch<MZB_BF16, 128>(a, st);
  return D == 64 ? gqa::launch<MZB_F16, 64>(a, st) : D == 96 ? gqa::launch<MZB_F16, 96>(a, st)
                                                             : gqa::launch<MZB_F16, 128>(a, st);
}
