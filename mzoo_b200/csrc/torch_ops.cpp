// The serving-step ops of torch.library (`mzb::gqa_*`, `mzb::kv_*`) as C++ kernels over the C ABI:
// allocation, current stream, one C call.  Through ctypes and the dispatcher's way back into
// Python such a call takes ~16 us of the host, more than the smallest decode step takes on the
// device; here ~6.  Schemas and fake implementations are declared in ops.py.  What a kernel would read
// wrongly or outside its memory (device, type, shape, strides) is refused here, since an op can be called
// without the wrappers (gqa_attn.py, kv_pages.py) and their messages; sizes are the C ABI's to check.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <array>
#include <atomic>

#include "../../include/mzb200.h"

namespace {

using at::Tensor;

// A non-zero status becomes a RuntimeError whose last word is the status; ops.py turns it into
// the exception that the other ops raise.
void ok(int status, const char* what) {
  if (status != MZB_OK) TORCH_CHECK(false, what, ": ", mzb_last_error(), " [mzb status ", status, "]");
}

int code_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return MZB_F32;
    case at::kBFloat16: return MZB_BF16;
    case at::kHalf: return MZB_F16;
    default: return -1;
  }
}

// A refusal, as the C ABI's: ops.py raises it as an AssertionError.
#define MZB_NEED(cond, what) TORCH_CHECK(cond, what, " [mzb status ", MZB_ERR_SHAPE, "]")

// A dense int32 tensor of `dim` dimensions on the device of `on`.
void ints_on(const Tensor& t, const Tensor& on, int dim, const char* what) {
  MZB_NEED(t.is_cuda() && t.get_device() == on.get_device() && t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous(), what);
}
// `t` like `on` in type and device, of `dim` dimensions with dense rows.
void rows_on(const Tensor& t, const Tensor& on, int dim, const char* what) {
  MZB_NEED(t.is_cuda() && t.get_device() == on.get_device() && t.scalar_type() == on.scalar_type() && t.dim() == dim &&
               (t.numel() == 0 || t.size(dim - 1) == 1 || t.stride(dim - 1) == 1),
           what);
}
// Page table [S, W], lengths [S] and reference counts.
void state_on(const Tensor& table, const Tensor& lens, const Tensor& refs, const char* what) {
  ints_on(table, table, 2, what);
  ints_on(lens, table, 1, what);
  ints_on(refs, table, 1, what);
  MZB_NEED(lens.size(0) == table.size(0), what);
}

struct Call {  // the tensor's device and that device's current stream
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit Call(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

template <class T = int32_t>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}

// The error word of a launch: the given one, or (none given: the usual case, and graphs that were traced) the
// device's persistent one, which Python keeps and check_errors() reads.
using Err = std::optional<Tensor>;
using WordOf = int64_t (*)(int);  // address of a device's persistent error word
WordOf word_of = nullptr;
int* word(const Err& err, const Tensor& on) {
  if (err.has_value()) return static_cast<int*>(err->data_ptr());
  static std::array<std::atomic<int*>, 64> known{};
  const int i = int(on.get_device());
  TORCH_CHECK(i >= 0 && i < int(known.size()) && word_of, "no error word for device ", i);
  int* w = known[i].load(std::memory_order_acquire);
  if (!w) {
    w = reinterpret_cast<int*>(word_of(i));
    TORCH_CHECK(w, "no error word for device ", i);
    known[i].store(w, std::memory_order_release);
  }
  return w;
}

Tensor floats(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }
Tensor ints(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kInt)); }

// (address, bytes of a page, bytes from page to page) of each pool; pages dense and apart
std::vector<int64_t> pool_array(at::TensorList pools, const Tensor& on, int64_t P, const char* what) {
  std::vector<int64_t> x;
  x.reserve(3 * pools.size());
  for (const Tensor& p : pools) {
    MZB_NEED(p.is_cuda() && p.get_device() == on.get_device() && p.dim() >= 2 && p.size(0) == P, what);
    int64_t n = 1;
    for (int64_t i = p.dim() - 1; i > 0; --i) {
      MZB_NEED(p.size(i) == 1 || p.stride(i) == n, what);
      n *= p.size(i);
    }
    MZB_NEED(P == 1 || p.stride(0) >= n, what);
    const int64_t size = p.element_size();
    x.insert(x.end(), {reinterpret_cast<int64_t>(p.data_ptr()), p.numel() / std::max<int64_t>(1, p.size(0)) * size, p.stride(0) * size});
  }
  return x;
}

std::tuple<Tensor, Tensor> gqa_prefill(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q,
                                       const Tensor& cu_k, const Err& err, bool causal, double scale) {
  const char* what = "gqa_prefill: q, k and v must be [tokens, heads, D] of one type, cu_q and cu_k dense int32 [B + 1], all on one device";
  rows_on(q, q, 3, what);
  rows_on(k, q, 3, what);
  rows_on(v, q, 3, what);
  ints_on(cu_q, q, 1, what);
  ints_on(cu_k, q, 1, what);
  MZB_NEED(k.size(2) == q.size(2) && v.sizes() == k.sizes() && cu_q.numel() >= 2 && cu_k.numel() == cu_q.numel(), what);
  Call c(q);
  const int64_t Tq = q.size(0), Tk = k.size(0), Hq = q.size(1), Hkv = k.size(1), D = q.size(2), B = cu_q.numel() - 1;
  Tensor o = at::empty({Tq, Hq, D}, q.options()), lse = at::empty({Tq, Hq}, q.options().dtype(at::kFloat)), ws;
  const int64_t n = mzb_gqa_prefill_ws(Tq, Tk, int(B), int(Hq), int(Hkv), int(D));
  if (n) ws = floats(n, q);
  ok(mzb_gqa_prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(cu_q), ptr(cu_k), o.data_ptr(), ptr<float>(lse),
                     n ? ptr<float>(ws) : nullptr, Tq, Tk, int(B), int(Hq), int(Hkv), int(D), code_of(q), q.stride(0),
                     q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1), causal, float(scale), word(err, q),
                     c.stream),
     "mzb_gqa_prefill");
  return {o, lse};
}

std::tuple<Tensor, Tensor> gqa_decode(const Tensor& q, const Tensor& k_pages, const Tensor& v_pages,
                                      const Tensor& page_table, const Tensor& seq_lens, const Err& err, double scale) {
  const char* what = "gqa_decode: q [B, heads, D] and the pools [pages, heads, page, D] must have one type, page_table [B, W] and "
                     "seq_lens [B] be dense int32, all on one device";
  rows_on(q, q, 3, what);
  rows_on(k_pages, q, 4, what);
  rows_on(v_pages, q, 4, what);
  ints_on(page_table, q, 2, what);
  ints_on(seq_lens, q, 1, what);
  MZB_NEED(k_pages.size(3) == q.size(2) && v_pages.sizes() == k_pages.sizes() && page_table.size(0) == q.size(0) &&
               seq_lens.size(0) == q.size(0),
           what);
  Call c(q);
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2), P = k_pages.size(0), Hkv = k_pages.size(1),
                page = k_pages.size(2), W = page_table.size(1);
  Tensor o = at::empty({B, Hq, D}, q.options()), lse = at::empty({B, Hq}, q.options().dtype(at::kFloat)), ws;
  const int64_t n = mzb_gqa_decode_ws(int(B), int(Hq), int(Hkv), int(D), int(W), int(page));
  if (n) ws = floats(n, q);
  ok(mzb_gqa_decode(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), ptr(page_table), ptr(seq_lens), o.data_ptr(),
                    ptr<float>(lse), n ? ptr<float>(ws) : nullptr, int(B), int(Hq), int(Hkv), int(D), code_of(q),
                    int(page), P, int(W), q.stride(0), q.stride(1), k_pages.stride(0), k_pages.stride(1),
                    k_pages.stride(2), v_pages.stride(0), v_pages.stride(1), v_pages.stride(2), float(scale), word(err, q),
                    c.stream),
     "mzb_gqa_decode");
  return {o, lse};
}

void kv_append(const Tensor& k, const Tensor& v, Tensor k_pages, Tensor v_pages, const Tensor& page_table,
               const Tensor& starts, const std::optional<Tensor>& cu, const Err& err) {
  const char* what = "kv_append: k and v [tokens, heads, D] and the pools [pages, heads, page, D] must have one type, page_table [B, W], "
                     "starts [B] and cu [B + 1] be dense int32, all on one device";
  rows_on(k, k, 3, what);
  rows_on(v, k, 3, what);
  rows_on(k_pages, k, 4, what);
  rows_on(v_pages, k, 4, what);
  ints_on(page_table, k, 2, what);
  ints_on(starts, k, 1, what);
  if (cu) ints_on(*cu, k, 1, what);
  MZB_NEED(v.sizes() == k.sizes() && v_pages.sizes() == k_pages.sizes() && k_pages.size(1) == k.size(1) && k_pages.size(3) == k.size(2) &&
               page_table.size(0) == starts.size(0) && (cu ? cu->size(0) == starts.size(0) + 1 : k.size(0) == starts.size(0)),
           what);
  Call c(k);
  const int size = int(k.element_size());
  const int64_t strides[10] = {k.stride(0),       k.stride(1),       v.stride(0),       v.stride(1),       k_pages.stride(0),
                               k_pages.stride(1), k_pages.stride(2), v_pages.stride(0), v_pages.stride(1), v_pages.stride(2)};
  ok(mzb_kv_append(k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), ptr(page_table), ptr(starts),
                   cu ? ptr(*cu) : nullptr, k.size(0), int(starts.numel()), int(k.size(1)), int(k.size(2)) * size,
                   int(k_pages.size(2)), k_pages.size(0), int(page_table.size(1)), size, strides, word(err, k), c.stream),
     "mzb_kv_append");
}

Tensor kv_reserve(Tensor page_table, Tensor seq_lens, Tensor refs, const Tensor& n_new, const Err& err, int64_t page) {
  const char* what = "kv_reserve: page_table [S, W], seq_lens [S], refs and n_new [S] must be dense int32 tensors on one device";
  state_on(page_table, seq_lens, refs, what);
  ints_on(n_new, page_table, 1, what);
  MZB_NEED(n_new.size(0) == seq_lens.size(0), what);
  Call c(page_table);
  Tensor starts = at::empty_like(seq_lens), ws = ints(refs.numel(), refs);
  ok(mzb_kv_reserve(ptr(page_table), ptr(seq_lens), ptr(refs), ptr(n_new), ptr(starts), ptr(ws), int(page_table.size(0)),
                    int(page_table.size(1)), refs.numel(), int(page), word(err, page_table), c.stream),
     "mzb_kv_reserve");
  return starts;
}

void kv_free(Tensor page_table, Tensor seq_lens, Tensor refs, const Tensor& seqs, const Err& err) {
  const char* what = "kv_free: page_table [S, W], seq_lens [S], refs and seqs must be dense int32 tensors on one device";
  state_on(page_table, seq_lens, refs, what);
  ints_on(seqs, page_table, 1, what);
  Call c(page_table);
  ok(mzb_kv_free(ptr(page_table), ptr(seq_lens), ptr(refs), ptr(seqs), seqs.numel(), page_table.size(0),
                 int(page_table.size(1)), refs.numel(), word(err, page_table), c.stream),
     "mzb_kv_free");
}

void kv_copy_pages(at::TensorList pools, const Tensor& src, const Tensor& dst, const Err& err) {
  const char* what = "kv_copy_pages: pools must be [pages, ...] with dense pages apart, src and dst dense int32 of one length, all on one device";
  MZB_NEED(!pools.empty() && pools[0].dim() >= 2, what);
  ints_on(src, src, 1, what);
  ints_on(dst, src, 1, what);
  MZB_NEED(dst.size(0) == src.size(0), what);
  Call c(src);
  const std::vector<int64_t> x = pool_array(pools, src, pools[0].size(0), what);
  ok(mzb_kv_copy_pages(x.data(), int(pools.size()), ptr(src), ptr(dst), src.numel(), pools[0].size(0), word(err, src), c.stream),
     "mzb_kv_copy_pages");
}

void kv_fork(at::TensorList pools, Tensor page_table, Tensor seq_lens, Tensor refs, const Tensor& src, const Tensor& dst,
             const Err& err, int64_t page) {
  const char* what = "kv_fork: pools must be [pages, ...] with dense pages apart, page_table [S, W], seq_lens [S], refs [pages], src and dst "
                     "dense int32, all on one device";
  state_on(page_table, seq_lens, refs, what);
  ints_on(src, page_table, 1, what);
  ints_on(dst, page_table, 1, what);
  MZB_NEED(dst.size(0) == src.size(0), what);
  Call c(page_table);
  const int64_t n = src.numel(), S = page_table.size(0);
  Tensor ws = ints(3 * n + S, refs);
  const std::vector<int64_t> x = pool_array(pools, refs, refs.numel(), what);
  ok(mzb_kv_fork(ptr(page_table), ptr(seq_lens), ptr(refs), ptr(src), ptr(dst), int(n), ptr(ws), S,
                 int(page_table.size(1)), refs.numel(), int(page), x.data(), int(pools.size()), word(err, page_table), c.stream),
     "mzb_kv_fork");
}

std::tuple<Tensor, Tensor> kv_compact(at::TensorList pools, const Tensor& page_table, const Tensor& refs, const Err& err) {
  const char* what = "kv_compact: pools must be [pages, ...] with dense pages apart, page_table [S, W] and refs [pages] dense int32, all on one device";
  ints_on(page_table, page_table, 2, what);
  ints_on(refs, page_table, 1, what);
  Call c(page_table);
  const int64_t P = refs.numel();
  Tensor ws = ints(3 * P + 1, refs), table = at::empty_like(page_table), new_refs = at::empty_like(refs);
  const std::vector<int64_t> x = pool_array(pools, refs, P, what);
  ok(mzb_kv_compact(ptr(page_table), ptr(refs), ptr(table), ptr(new_refs), ptr(ws), page_table.numel(), P, x.data(),
                    int(pools.size()), word(err, page_table), c.stream),
     "mzb_kv_compact");
  return {table, new_refs};
}

}  // namespace

// Called once by the Python side with its keeper of error words (not a static initialiser, whose exception at a stale build's
// other schema would end the process): 0, or -1 with the reason in msg.
extern "C" __attribute__((visibility("default"))) int mzb_torch_init(int64_t (*word)(int), char* msg, size_t size) {
  try {
    word_of = word;
    static torch::Library m(torch::Library::IMPL, "mzb", c10::DispatchKey::CUDA, __FILE__, __LINE__);
    m.impl("gqa_prefill", &gqa_prefill);
    m.impl("gqa_decode", &gqa_decode);
    m.impl("kv_append", &kv_append);
    m.impl("kv_reserve", &kv_reserve);
    m.impl("kv_free", &kv_free);
    m.impl("kv_copy_pages", &kv_copy_pages);
    m.impl("kv_fork", &kv_fork);
    m.impl("kv_compact", &kv_compact);
    return 0;
  } catch (const std::exception& e) {
    snprintf(msg, size, "%s", e.what());
    return -1;
  }
}
