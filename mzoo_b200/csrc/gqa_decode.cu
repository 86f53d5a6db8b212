// Attention of one new token per sequence over a paged K / V cache with grouped heads, bf16 /
// f16 in and out, fp32 accumulation, natural-log lse.  No counterpart in the reference.
//
//   key t < len[b] of sequence b is slot t % page of page table[b, t / page];
//   o = softmax(scale q K^T) V; a sequence of length 0: o = 0, lse = -inf.
//
// One block of 8 warps per (sequence, head): the warps share the keys and are joined.
#include "common.cuh"

namespace mzb {
namespace gqa {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct DecodeArgs {
  const void *q, *k, *v;
  const int32_t *table, *lens;
  void* o;
  float* lse;
  int64_t P, sq_b, sq_h, sk_p, sk_h, sk_t, sv_p, sv_h, sv_t;
  int B, Hq, Hkv, W, page;
  float scale;
};

template <int DT, int D>
__global__ void __launch_bounds__(256) decode_kernel(DecodeArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int C = D / 32;
  __shared__ float sm[8], sl[8], so[8][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, hk = h / (a.Hq / a.Hkv);
  const int64_t n = max((int64_t)0, min((int64_t)a.lens[b], (int64_t)a.W * a.page));
  float qv[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    qv[c] = E::load(static_cast<const T*>(a.q)[b * a.sq_b + h * a.sq_h + lane + 32 * c]);
    acc[c] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = warp; j < n; j += 8) {
    const int64_t p = min(max((int64_t)a.table[(int64_t)b * a.W + j / a.page], (int64_t)0), a.P - 1), r = j % a.page;
    const T* kr = static_cast<const T*>(a.k) + p * a.sk_p + hk * a.sk_h + r * a.sk_t;
    const T* vr = static_cast<const T*>(a.v) + p * a.sv_p + hk * a.sv_h + r * a.sv_t;
    float s = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) s += qv[c] * E::load(kr[lane + 32 * c]);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale * LOG2E;
    const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.0f : mn;
    const float al = exp2f(m - ms), pr = exp2f(s - ms);
    l = l * al + pr;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = acc[c] * al + pr * E::load(vr[lane + 32 * c]);
    m = mn;
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int c = 0; c < C; ++c) so[warp][lane + 32 * c] = acc[c];
  __syncthreads();
  if (warp) return;
  float mt = -INFINITY, lt = 0.0f;
  for (int w = 0; w < 8; ++w) mt = fmaxf(mt, sm[w]);
  const float ms = mt == -INFINITY ? 0.0f : mt;
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.0f;
  for (int w = 0; w < 8; ++w) {
    const float al = exp2f(sm[w] - ms);
    lt += sl[w] * al;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] += so[w][lane + 32 * c] * al;
  }
  const float inv = n > 0 ? 1.0f / lt : 0.0f;
  const int64_t row = (int64_t)b * a.Hq + h;
#pragma unroll
  for (int c = 0; c < C; ++c) static_cast<T*>(a.o)[row * D + lane + 32 * c] = E::store(acc[c] * inv);
  if (lane == 0) a.lse[row] = n > 0 ? (mt + log2f(lt)) * LN2 : -INFINITY;
}

template <int DT, int D>
int launch(const DecodeArgs& a, cudaStream_t st) {
  decode_kernel<DT, D><<<unsigned(a.B) * a.Hq, 256, 0, st>>>(a);
  return launch_status("gqa_decode");
}

}  // namespace gqa
}  // namespace mzb

using namespace mzb;

extern "C" int64_t mzb_gqa_decode_ws(int B, int Hq, int Hkv, int D, int W, int page) { return 0; }

extern "C" int mzb_gqa_decode(const void* q, const void* k_pages, const void* v_pages, const int32_t* page_table,
                              const int32_t* seq_lens, void* o, float* lse, float* ws, int B, int Hq, int Hkv, int D,
                              int dtype, int page, int64_t P, int W, int64_t sq_b, int64_t sq_h, int64_t sk_p,
                              int64_t sk_h, int64_t sk_t, int64_t sv_p, int64_t sv_h, int64_t sv_t,
                              float softmax_scale, int* err, void* stream) {
  MZB_REQUIRE(B >= 0 && P >= 1 && P < (int64_t(1) << 31) && W >= 0 && (int64_t)W * page < (int64_t(1) << 31),
              MZB_ERR_SHAPE, "gqa_decode: bad sizes B=%d pages=%lld table width=%d page=%d", B, (long long)P, W, page);
  MZB_REQUIRE(Hkv >= 1 && Hq >= 1 && Hq % Hkv == 0 && Hq / Hkv <= 128, MZB_ERR_SHAPE,
              "gqa_decode: query heads must be a multiple (at most 128) of the K/V heads, got %d and %d", Hq, Hkv);
  MZB_REQUIRE(D == 64 || D == 96 || D == 128, MZB_ERR_UNSUPPORTED, "gqa_decode: unsupported head dim %d", D);
  MZB_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, MZB_ERR_UNSUPPORTED,
              "gqa_decode: unsupported page size %d (16, 32, 64 or 128 tokens)", page);
  MZB_REQUIRE(dtype == MZB_BF16 || dtype == MZB_F16, MZB_ERR_UNSUPPORTED, "gqa_decode: unsupported dtype %d", dtype);
  MZB_REQUIRE(err != nullptr, MZB_ERR_SHAPE, "gqa_decode: needs an error word");
  if (B == 0) return MZB_OK;
  gqa::DecodeArgs a{q, k_pages, v_pages, page_table, seq_lens, o, lse, P, sq_b, sq_h, sk_p, sk_h, sk_t, sv_p, sv_h,
                    sv_t, B, Hq, Hkv, W, page, softmax_scale};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == MZB_BF16)
    return D == 64 ? gqa::launch<MZB_BF16, 64>(a, st) : D == 96 ? gqa::launch<MZB_BF16, 96>(a, st)
                                                                : gqa::launch<MZB_BF16, 128>(a, st);
  return D == 64 ? gqa::launch<MZB_F16, 64>(a, st) : D == 96 ? gqa::launch<MZB_F16, 96>(a, st)
                                                             : gqa::launch<MZB_F16, 128>(a, st);
}
