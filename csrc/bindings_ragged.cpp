// PyTorch bindings of the ragged-batch operators (ragged.h). Arguments are
// checked here, on the host and without a synchronisation: a wrong type,
// device, shape or size raises ValueError before anything is launched. Rows
// that the kernels cannot load as they lie (a head dim that is not
// contiguous, rows off a 16-byte boundary) are copied first. Numbers enter
// messages through std::to_string: an integer streamed into c10's message
// builder crashes where the extension carries its own copy of the C++ runtime.

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>

#include "ragged.h"

namespace afd {

namespace {

using OptTensor = c10::optional<at::Tensor>;

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check_rc(int rc, const char* what) {
  TORCH_CHECK(rc == 0, std::string(what) + " failed with code " + std::to_string(rc) +
                           (rc > 4000 ? std::string(" (") +
                                            cudaGetErrorString((cudaError_t)(rc - 4000)) + ")"
                                      : std::string()));
}

int elem16(const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, what,
              " must be bf16 or fp16");
  return t.scalar_type() == at::kBFloat16 ? kElemBf16 : kElemF16;
}

void check_like(const at::Tensor& t, const at::Tensor& like, const char* what) {
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == like.scalar_type(), what,
              " must be on the queries' device and of their type");
}

int num_sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// Zeroed counters that the kernels leave zeroed: one buffer for each stream
// (calls on one stream follow one another), kept for good. Inside a stream
// capture the call gets zeros of its own, set again at every replay, so that
// graphs may be replayed on any stream.
at::Tensor zeroed_counters(const at::Tensor& like, int64_t n) {
  const auto opt = at::TensorOptions().device(like.device()).dtype(at::kInt);
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return at::zeros({n}, opt);
  static std::mutex mu;
  static auto* pool = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
  std::lock_guard<std::mutex> lock(mu);
  at::Tensor& t = (*pool)[{like.device().index(), stream()}];
  if (!t.defined() || t.numel() < n) t = at::zeros({std::max<int64_t>(n, 4096)}, opt);
  return t;
}

// Workspace that no call expects anything in: one buffer for each stream, which
// grows (at most about 40 MB: the split forms of few rows alone use it) and is kept,
// 0.8 us less on the host than an allocation a call. A capture gets its own.
at::Tensor scratch(const at::Tensor& like, int64_t bytes) {
  const auto opt = at::TensorOptions().device(like.device()).dtype(at::kByte);
  if (at::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None)
    return at::empty({bytes}, opt);
  static std::mutex mu;
  static auto* pool = new std::map<std::pair<int, cudaStream_t>, at::Tensor>();
  std::lock_guard<std::mutex> lock(mu);
  at::Tensor& t = (*pool)[{like.device().index(), stream()}];
  if (!t.defined() || t.numel() < bytes) t = at::empty({bytes}, opt);
  return t;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// A contiguous copy at an aligned address, or `t` itself where `ok`.
at::Tensor loadable(const at::Tensor& t, bool ok) {
  return ok || t.numel() == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// [rows, heads, D] with contiguous heads and 16-byte aligned rows that do not
// overlap: a tensor map gets their distance, so rows expanded from one are copied.
at::Tensor take_rows(const at::Tensor& t, const char* what) {
  TORCH_CHECK_VALUE(t.is_cuda(), what, " must be a CUDA tensor");
  TORCH_CHECK_VALUE(t.dim() == 3, what, " must be [rows, heads, head_dim]");
  TORCH_CHECK_VALUE(t.size(2) == 64 || t.size(2) == 128, what, ": head_dim must be 64 or 128");
  TORCH_CHECK_VALUE(t.size(0) < (1ll << 31), what, ": too many rows");
  return loadable(t, t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2)) &&
                         (t.size(0) == 1 ||
                          (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1) * t.size(2))) &&
                         aligned16(t.data_ptr()));
}

// Elements between the rows of what take_rows gave; a single row has any stride.
int64_t row_of(const at::Tensor& t) {
  return t.size(0) == 1 ? t.size(1) * t.size(2) : t.stride(0);
}

void check_ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* what) {
  TORCH_CHECK_VALUE(t.device() == like.device() && t.scalar_type() == at::kInt && t.is_contiguous() &&
                  t.dim() == 1 && t.numel() == n,
              what, " must be a contiguous int32 tensor of ", std::to_string(n), " on the same device");
}

int* status_ptr(const OptTensor& s, const at::Tensor& like) {
  if (!s.has_value() || !s->defined()) return nullptr;
  TORCH_CHECK_VALUE(s->device() == like.device() && s->scalar_type() == at::kInt &&
                        s->numel() >= 2 && s->is_contiguous(),
                    "status must be a contiguous int32 tensor of 2 on the same device");
  return s->data_ptr<int>();
}

// Checks the pool against nkv heads of D and fills the struct's pool fields.
template <typename Args>
void take_pool(Args& a, const at::Tensor& k_pages, const at::Tensor& v_pages,
               const at::Tensor& like) {
  check_like(k_pages, like, "k_pages");
  check_like(v_pages, like, "v_pages");
  TORCH_CHECK_VALUE(k_pages.dim() == 4 && v_pages.sizes() == k_pages.sizes() &&
                  v_pages.strides() == k_pages.strides(),
              "k_pages and v_pages must be [pages, kv heads, page_size, head_dim], laid out alike");
  const int64_t page = k_pages.size(2), D = k_pages.size(3);
  TORCH_CHECK_VALUE(D == 64 || D == 128, "head_dim must be 64 or 128");
  TORCH_CHECK_VALUE(page >= 16 && page % 16 == 0 && page <= 4096,
              "page_size must be a multiple of 16, at most 4096");
  TORCH_CHECK_VALUE(k_pages.numel() == 0 ||
                  (k_pages.stride(3) == 1 && k_pages.stride(2) == D &&
                   (k_pages.size(1) == 1 || k_pages.stride(1) == page * D) &&
                   k_pages.stride(0) % 8 == 0 && k_pages.stride(0) >= k_pages.size(1) * page * D &&
                   aligned16(k_pages.data_ptr()) && aligned16(v_pages.data_ptr())),
              "each page must be contiguous and 16-byte aligned");
  TORCH_CHECK_VALUE(k_pages.size(0) >= 1 && k_pages.size(0) < (1ll << 31), "the pool has no page");
  a.page_stride = k_pages.stride(0);
  a.num_pages = (int)k_pages.size(0);
  a.page_size = (int)page;
}

float scale_of(c10::optional<double> scale, int D) {
  TORCH_CHECK_VALUE(!scale.has_value() || ((float)*scale > 0 && std::isfinite((float)*scale)),
                    "scale must be positive, in 32 bits");
  return scale.has_value() ? (float)*scale : 1.f / std::sqrt((float)D);
}

void check_heads(int64_t nq, int64_t nkv) {
  TORCH_CHECK_VALUE(nkv >= 1 && nq >= 1 && nq % nkv == 0, "query heads (", std::to_string(nq),
                    ") must be a multiple of the kv heads (", std::to_string(nkv), ")");
}

template <typename Args>
void take_table(Args& a, const at::Tensor& table, int64_t n, const at::Tensor& like) {
  TORCH_CHECK_VALUE(table.device() == like.device() && table.scalar_type() == at::kInt &&
                  table.dim() == 2 && table.size(0) == n && table.size(1) >= 1 &&
                  (n == 0 || table.size(1) == 1 || table.stride(1) == 1),
              "page_table must be an int32 [", std::to_string(n), ", pages] on the same device with unit stride");
  // positions are ints, and the kernels look a few thousand ahead of the last one
  TORCH_CHECK_VALUE(table.size(1) * a.page_size < (1ll << 30) &&
                        (n <= 1 || table.stride(0) < (1ll << 31)),
                    "page_table spans too many positions");
  a.page_table = table.data_ptr<int>();
  a.table_row = (int)table.stride(0);
  a.max_pages = (int)table.size(1);
}

at::Tensor paged_decode_attention(const at::Tensor& q_in, const at::Tensor& k_pages,
                                  const at::Tensor& v_pages, const at::Tensor& page_table,
                                  const at::Tensor& seq_lens, c10::optional<double> scale,
                                  const OptTensor& status) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = take_rows(q_in, "q");
  PagedDecodeArgs a{};
  a.elem = elem16(q, "q");
  take_pool(a, k_pages, v_pages, q);
  a.B = (int)q.size(0);
  a.nq = (int)q.size(1);
  a.nkv = (int)k_pages.size(1);
  a.D = (int)q.size(2);
  TORCH_CHECK_VALUE(k_pages.size(3) == a.D, "q and the pages differ in head_dim");
  check_heads(a.nq, a.nkv);
  take_table(a, page_table, a.B, q);
  check_ints(seq_lens, q, a.B, "seq_lens");
  at::Tensor out = at::empty({a.B, (int64_t)a.nq * a.D}, q.options());
  a.q = q.data_ptr();
  a.q_row = row_of(q);
  a.k_pages = k_pages.data_ptr();
  a.v_pages = v_pages.data_ptr();
  a.seq_lens = seq_lens.data_ptr<int>();
  a.out = out.data_ptr();
  a.scale = scale_of(scale, a.D);
  a.status = status_ptr(status, q);
  const int sms = num_sms();
  TORCH_CHECK_VALUE((double)a.B * (a.max_pages * (a.page_size / 16.0) + 4) * a.nkv *
                            ((a.nq / a.nkv + 15) / 16) < 2147483648.0 - 65536.0 * sms,
                    "the page table spans too many positions in all");
  const at::Tensor parts = scratch(q, paged_decode_part_bytes(a.nq, a.nkv, a.D, sms));
  const at::Tensor counters = zeroed_counters(q, paged_decode_counters(sms));
  a.parts = parts.data_ptr();
  a.counters = counters.data_ptr<int>();
  check_rc(launch_paged_decode(a, sms, stream()), "paged_decode_attention");
  return out;
}

at::Tensor packed_common(PackedAttnArgs& a, const at::Tensor& q, const at::Tensor& cu_q,
                         c10::optional<double> scale, const OptTensor& status, int64_t nkv) {
  a.elem = elem16(q, "q");
  a.T = (int)q.size(0);
  a.nq = (int)q.size(1);
  a.nkv = (int)nkv;
  a.D = (int)q.size(2);
  check_heads(a.nq, a.nkv);
  TORCH_CHECK_VALUE(a.nq / a.nkv <= 128, "at most 128 query heads per kv head");
  TORCH_CHECK_VALUE(cu_q.dim() == 1 && cu_q.numel() >= 1, "cu_seqlens must hold n + 1 offsets");
  check_ints(cu_q, q, cu_q.numel(), "cu_seqlens");
  a.n_seqs = (int)cu_q.numel() - 1;
  at::Tensor out = at::empty({a.T, (int64_t)a.nq * a.D}, q.options());
  a.q = q.data_ptr();
  a.q_row = row_of(q);
  a.cu_q = cu_q.data_ptr<int>();
  a.out = out.data_ptr();
  a.scale = scale_of(scale, a.D);
  a.status = status_ptr(status, q);
  return out;
}

void run_packed(PackedAttnArgs& a, const at::Tensor& q, int64_t most_keys, const char* what) {
  const int sms = num_sms();
  const at::Tensor counter = zeroed_counters(q, 1);
  a.counter = counter.data_ptr<int>();
  a.splits = packed_attention_splits(a.T, a.n_seqs, a.nq, a.nkv, most_keys, sms);
  at::Tensor parts;
  if (a.splits > 1)
    parts = scratch(q, packed_attention_part_bytes((int64_t)a.T * a.nq, a.D, a.splits));
  check_rc(launch_packed_attention(a, a.splits > 1 ? parts.data_ptr() : nullptr, sms, stream()),
           what);
}

at::Tensor packed_attention(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in,
                            const at::Tensor& cu_q, const OptTensor& cu_k_in,
                            c10::optional<double> scale, const OptTensor& status) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = take_rows(q_in, "q"), k = take_rows(k_in, "k"), v = take_rows(v_in, "v");
  check_like(k, q, "k");
  check_like(v, q, "v");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(2) == q.size(2),
              "k and v must be [rows, kv heads, head_dim] with the queries' head_dim");
  PackedAttnArgs a{};
  at::Tensor out = packed_common(a, q, cu_q, scale, status, k.size(1));
  const at::Tensor& cu_k = cu_k_in.has_value() ? *cu_k_in : cu_q;
  TORCH_CHECK_VALUE(cu_k_in.has_value() || k.size(0) == q.size(0),
                    "k has other rows than q: give cu_seqlens_k");
  check_ints(cu_k, q, cu_q.numel(), "cu_seqlens_k");
  a.k = k.data_ptr();
  a.v = v.data_ptr();
  a.k_row = row_of(k);
  a.v_row = row_of(v);
  a.Tk = (int)k.size(0);
  a.cu_k = cu_k.data_ptr<int>();
  run_packed(a, q, a.Tk, "packed_attention");
  return out;
}

at::Tensor paged_prefill_attention(const at::Tensor& q_in, const at::Tensor& k_pages,
                                   const at::Tensor& v_pages, const at::Tensor& page_table,
                                   const at::Tensor& seq_lens, const at::Tensor& cu_q,
                                   c10::optional<double> scale, const OptTensor& status) {
  TORCH_CHECK_VALUE(q_in.is_cuda(), "q must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(q_in.device());
  const at::Tensor q = take_rows(q_in, "q");
  PackedAttnArgs a{};
  a.paged = 1;
  take_pool(a, k_pages, v_pages, q);
  TORCH_CHECK_VALUE(k_pages.size(3) == q.size(2), "q and the pages differ in head_dim");
  at::Tensor out = packed_common(a, q, cu_q, scale, status, k_pages.size(1));
  take_table(a, page_table, a.n_seqs, q);
  check_ints(seq_lens, q, a.n_seqs, "seq_lens");
  a.k_pages = k_pages.data_ptr();
  a.v_pages = v_pages.data_ptr();
  a.seq_lens = seq_lens.data_ptr<int>();
  run_packed(a, q, (int64_t)a.max_pages * a.page_size, "paged_prefill_attention");
  return out;
}

// q [T, nq, D], and k [T, nkv, D] where there is no pool to store it to.
std::tuple<at::Tensor, at::Tensor> norm_rope(const at::Tensor& qkv_in, const at::Tensor& q_norm,
                                             const at::Tensor& k_norm, const at::Tensor& rope,
                                             const at::Tensor& positions, int64_t nq, int64_t nkv,
                                             double eps, const OptTensor& k_pages,
                                             const OptTensor& v_pages, const OptTensor& slots,
                                             const OptTensor& status) {
  TORCH_CHECK_VALUE(qkv_in.is_cuda() && qkv_in.dim() == 2,
                    "qkv must be a CUDA tensor [tokens, width]");
  const c10::cuda::CUDAGuard guard(qkv_in.device());
  const at::Tensor qkv = loadable(qkv_in, qkv_in.stride(1) == 1 && qkv_in.stride(0) % 8 == 0 &&
                                              qkv_in.stride(0) >= 0 &&
                                              aligned16(qkv_in.data_ptr()));
  NormRopeArgs a{};
  a.elem = elem16(qkv, "qkv");
  check_heads(nq, nkv);
  const int64_t T = qkv.size(0), D = q_norm.numel();
  TORCH_CHECK_VALUE(D == 64 || D == 128, "head_dim must be 64 or 128");
  TORCH_CHECK_VALUE(T < (1ll << 31) && qkv.size(1) == (nq + 2 * nkv) * D, "qkv must be [tokens, ",
                    std::to_string((nq + 2 * nkv) * D), "]");
  check_like(q_norm, qkv, "q_norm");
  check_like(k_norm, qkv, "k_norm");
  TORCH_CHECK_VALUE(q_norm.is_contiguous() && k_norm.is_contiguous() && k_norm.numel() == D &&
                  aligned16(q_norm.data_ptr()) && aligned16(k_norm.data_ptr()),
              "q_norm and k_norm must be contiguous, aligned and of head_dim values");
  TORCH_CHECK_VALUE(rope.device() == qkv.device() && rope.scalar_type() == at::kFloat &&
                  rope.dim() == 2 && rope.size(1) == D && rope.size(0) >= 1 &&
                  rope.size(0) < (1ll << 31) && rope.is_contiguous() && aligned16(rope.data_ptr()),
              "rope must be a contiguous fp32 table [positions, head_dim]");
  check_ints(positions, qkv, T, "positions");
  at::Tensor q_out = at::empty({T, nq, D}, qkv.options()), k_out;
  a.T = (int)T;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.D = (int)D;
  if (k_pages.has_value()) {
    TORCH_CHECK_VALUE(v_pages.has_value() && slots.has_value(),
                "the pool needs v_pages and slots");
    take_pool(a, *k_pages, *v_pages, qkv);
    TORCH_CHECK_VALUE(k_pages->size(1) == nkv && k_pages->size(3) == D,
                "the pages' heads differ from qkv's");
    TORCH_CHECK_VALUE(slots->device() == qkv.device() && slots->scalar_type() == at::kLong &&
                    slots->is_contiguous() && slots->numel() == T,
                "slots must be a contiguous int64 tensor, one per token");
    a.k_pages = k_pages->data_ptr();
    a.v_pages = v_pages->data_ptr();
    a.slots = slots->data_ptr<int64_t>();
  } else {
    k_out = at::empty({T, nkv, D}, qkv.options());
    a.k_out = k_out.data_ptr();
  }
  a.qkv = qkv.data_ptr();
  a.qkv_row = qkv.stride(0);
  a.q_norm = q_norm.data_ptr();
  a.k_norm = k_norm.data_ptr();
  a.rope = rope.data_ptr<float>();
  a.max_pos = (int)rope.size(0);
  a.positions = positions.data_ptr<int>();
  a.q_out = q_out.data_ptr();
  a.eps = (float)eps;
  a.status = status_ptr(status, qkv);
  check_rc(launch_norm_rope(a, stream()), "norm_rope");
  return {q_out, k_out};
}

// (logprob [R], entropy [R], top_ids [R, top_k], top_logprobs [R, top_k])
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs(
    const at::Tensor& logits_in, const at::Tensor& ids, int64_t top_k) {
  TORCH_CHECK_VALUE(logits_in.is_cuda() && logits_in.dim() == 2,
                    "logits must be a CUDA tensor [rows, vocab]");
  const c10::cuda::CUDAGuard guard(logits_in.device());
  const auto t = logits_in.scalar_type();
  TORCH_CHECK_VALUE(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat,
                    "logits must be bf16, fp16 or fp32");
  const int64_t R = logits_in.size(0), V = logits_in.size(1);
  TORCH_CHECK_VALUE(V >= 1 && V <= kMaxLogprobVocab && R < (1ll << 31),
                    "logits must hold 1 to " + std::to_string(kMaxLogprobVocab) + " values a row");
  TORCH_CHECK_VALUE(ids.device() == logits_in.device() && ids.scalar_type() == at::kLong &&
                        ids.is_contiguous() && ids.numel() == R,
                    "ids must be a contiguous int64 tensor, one per row");
  TORCH_CHECK_VALUE(top_k >= 0 && top_k <= kMaxTopLogprobs && top_k <= V,
                    "top_k must be at most ", std::to_string(kMaxTopLogprobs), " and the vocabulary");
  const at::Tensor logits = loadable(logits_in, V == 1 || logits_in.stride(1) == 1);
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logprob = at::empty({R}, f32), entropy = at::empty({R}, f32);
  at::Tensor top_ids = at::empty({R, top_k}, ids.options());
  at::Tensor top_logprobs = at::empty({R, top_k}, f32);
  TokenLogprobsArgs a{};
  a.elem = t == at::kBFloat16 ? kElemBf16 : t == at::kHalf ? kElemF16 : kElemF32;
  a.logits = logits.data_ptr();
  a.row = logits.stride(0);
  a.ids = ids.data_ptr<int64_t>();
  a.logprob = logprob.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.top_ids = top_ids.data_ptr<int64_t>();
  a.top_logprobs = top_logprobs.data_ptr<float>();
  a.R = (int)R;
  a.V = (int)V;
  a.top_k = (int)top_k;
  const int splits = token_logprobs_splits(a.R, a.V, num_sms());
  at::Tensor ws, counters;
  if (splits > 1) {
    ws = scratch(logits, (int64_t)token_logprobs_workspace(a.R, a.V, splits));
    counters = zeroed_counters(logits, R);
    a.counters = counters.data_ptr<int>();
  }
  check_rc(launch_token_logprobs(a, splits, splits > 1 ? ws.data_ptr() : nullptr, stream()),
           "token_logprobs");
  return {logprob, entropy, top_ids, top_logprobs};
}

}  // namespace

void bind_ragged(pybind11::module& m) {
  m.def("paged_decode_attention", &paged_decode_attention);
  m.def("packed_attention", &packed_attention);
  m.def("paged_prefill_attention", &paged_prefill_attention);
  m.def("norm_rope", &norm_rope);
  m.def("token_logprobs", &token_logprobs);
}

}  // namespace afd
