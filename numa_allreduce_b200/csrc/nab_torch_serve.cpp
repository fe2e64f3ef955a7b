// Python bindings of the paged-cache decode operators and the token
// log-probabilities: functions of the extension module itself (PyInit__C),
// not torch.ops. An eager decode step calls them once or twice per layer, on few
// tokens, and is bound by the host then: the dispatcher's parsing and boxing of 4 to 13
// arguments took 2.4 us of a call of 8.8 (8 tokens: pages 8.8 -> 5.9 us, append
// 8.3 -> 4.6, attention 8.5 -> 5.2, log-probabilities 8.9 -> 6.1, with the check below
// in place of a look into os.environ, 0.6 us).
//
// Every argument is checked here before anything is launched. A bad one is
// refused with its name whatever device it lies on, and so are tensors that
// share memory with one that the call writes; tensors on a device other than
// CUDA are refused last, and so is one that asks for a derivative. There is no
// dispatcher to take a fake, batched or wrapped tensor elsewhere: these are
// refused. The GIL is released during the call.
#include <Python.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/torch.h>

#include <climits>
#include <cmath>
#include <cstdlib>
#include <initializer_list>
#include <optional>
#include <tuple>
#include <utility>

#include "nab_common.h"
#include "nab_logprobs.h"
#include "nab_paged.h"

namespace {

using OptTensor = std::optional<at::Tensor>;
using Named = std::pair<const char*, const at::Tensor*>;

// The last check of every op: no derivative asked for, and one CUDA device for all.
void check_devices(const char* op, std::initializer_list<Named> tensors) {
  const at::Tensor& first = *tensors.begin()->second;
  for (const auto& [name, t] : tensors) {
    if (t == nullptr) continue;
    TORCH_CHECK(!(at::GradMode::is_enabled() && t->requires_grad()), op, ": ", name,
                " requires a gradient; this operator has none (use torch.no_grad())");
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), op, ": ", name,
                " carries a forward-mode tangent; this operator has no derivative");
  }
  for (const auto& [name, t] : tensors) {
    if (t == nullptr) continue;
    TORCH_CHECK(t->is_cuda(), op, ": ", name, " must be a CUDA tensor");
    TORCH_CHECK(t->device() == first.device(), op, ": ", name, " is on ", t->device(), ", ", tensors.begin()->first,
                " on ", first.device());
  }
}

// The bytes of a tensor whose first dimension may have its rows apart and whose other ones are contiguous.
struct Extent {
  const char* name;
  uintptr_t at = 0;
  int64_t rows = 0, width = 0, step = 0;  // bytes but for `rows`
  Extent(const char* n, const at::Tensor* t) : name(n) {
    if (t == nullptr || t->numel() == 0) return;
    at = reinterpret_cast<uintptr_t>(t->const_data_ptr());
    const int64_t e = t->element_size();
    if (t->is_contiguous()) {
      rows = 1;
      width = t->numel() * e;
    } else {
      rows = t->size(0);
      width = t->numel() / rows * e;
      step = t->stride(0) * e;
    }
  }
};

// Whether a row of `a` shares bytes with `b`, which is one block.
bool touches(const Extent& a, const Extent& b) {
  if (a.at == 0 || b.at == 0) return false;
  const int64_t lo = static_cast<int64_t>(b.at - a.at), hi = lo + b.width;  // b's bytes, counted from a's first
  if (a.step == 0) return lo < a.width && hi > 0;
  // the first row that ends behind b's first byte
  const int64_t r = lo < a.width ? 0 : (lo - a.width) / a.step + 1;
  return r < a.rows && r * a.step < hi;
}

// No tensor that the call writes shares memory with another one of the call. Of two tensors with rows apart only one
// may be given here as written.
void check_apart(const char* op, std::initializer_list<Extent> written, std::initializer_list<Extent> read) {
  const auto check = [op](const Extent& w, const Extent& r) {
    TORCH_CHECK(!(w.rows > 1 ? touches(w, r) : touches(r, w)), op, ": ", w.name, " and ", r.name,
                " overlap in memory");
  };
  for (const Extent* w = written.begin(); w != written.end(); ++w) {
    for (const Extent* v = w + 1; v != written.end(); ++v) check(*w, *v);
    for (const Extent& r : read) check(*w, r);
  }
}

void check_vector(const char* op, const char* name, const at::Tensor& t, at::ScalarType type, int64_t n) {
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous() && t.scalar_type() == type, op, ": ", name,
              " must be a contiguous ", type, " tensor of ", n, " elements");
}

int half_dtype(const char* op, const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, op, ": ", name,
              " must be bfloat16 or float16, got ", t.scalar_type());
  return t.scalar_type() == at::kHalf ? nab::kF16 : nab::kBF16;
}

bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0; }

// k_pages and v_pages: [pages, kv heads, P, D]
void check_pages(const char* op, const at::Tensor& k, const at::Tensor& v, at::ScalarType type) {
  TORCH_CHECK(k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes(), op,
              ": k_pages and v_pages must be contiguous [pages, kv_heads, page_size, head_dim] of one shape");
  TORCH_CHECK(k.scalar_type() == type && v.scalar_type() == type, op, ": k_pages and v_pages must be ", type);
  TORCH_CHECK(k.size(0) >= 1 && k.size(1) >= 1, op, ": no pages");
  TORCH_CHECK(k.size(2) >= 16 && k.size(2) % 16 == 0, op, ": page_size must be a multiple of 16, got ", k.size(2));
  TORCH_CHECK(k.size(3) == 64 || k.size(3) == 128, op, ": head_dim must be 64 or 128, got ", k.size(3));
  TORCH_CHECK(k.size(0) * k.size(1) * k.size(2) < INT_MAX, op, ": too many page rows");
  TORCH_CHECK(aligned16(k) && aligned16(v), op, ": k_pages and v_pages must be 16-byte aligned");
  check_apart(op, {{"k_pages", &k}}, {{"v_pages", &v}});
}

// An uninitialised tensor on the device of `like` (the call's device guard is set): the allocator without the
// dispatcher, which is what a call of a few microseconds has to save.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

// Outputs of one call in one allocation, each 16-byte aligned: of 4 to 6 small tensors that saves 1 to 2 us.
class Outputs {
 public:
  explicit Outputs(const at::Tensor& like) : like_(like) {}
  void add(at::IntArrayRef sizes, at::ScalarType type) {
    parts_[n_++] = {c10::SmallVector<int64_t, 2>(sizes.begin(), sizes.end()), type, bytes_};
    bytes_ += (c10::multiply_integers(sizes) * static_cast<int64_t>(c10::elementSize(type)) + 15) / 16 * 16;
  }
  void make() { storage_ = fresh({bytes_}, at::kByte, like_).storage(); }
  at::Tensor operator[](int i) const {
    const Part& p = parts_[i];
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(
        c10::Storage(storage_), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(p.type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(p.sizes);
    t.unsafeGetTensorImpl()->set_storage_offset(p.offset / static_cast<int64_t>(c10::elementSize(p.type)));
    return t;
  }

 private:
  struct Part {
    c10::SmallVector<int64_t, 2> sizes;
    at::ScalarType type = at::kByte;
    int64_t offset = 0;
  };
  at::Tensor like_;
  Part parts_[6];
  int n_ = 0;
  int64_t bytes_ = 0;
  c10::Storage storage_;
};

int sms_of(const at::Tensor& t) { return at::cuda::getDeviceProperties(t.device().index())->multiProcessorCount; }

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> assign_pages(const at::Tensor& cached,
                                                                        const OptTensor& query_start,
                                                                        at::Tensor& block_tables,
                                                                        const at::Tensor& free_pages,
                                                                        const at::Tensor& taken, int64_t page_size,
                                                                        int64_t num_tokens) {
  constexpr const char* op = "assign_pages";
  TORCH_CHECK(cached.dim() == 1 && cached.size(0) >= 1 && cached.size(0) <= nab::kMaxPagedRequests, op,
              ": cached must hold 1 to ", nab::kMaxPagedRequests, " requests");
  const int64_t B = cached.size(0);
  check_vector(op, "cached", cached, at::kInt, B);
  if (query_start) check_vector(op, "query_start", *query_start, at::kInt, B + 1);
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == B && block_tables.scalar_type() == at::kInt &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1) &&
                  (B == 1 || block_tables.stride(0) >= block_tables.size(1)),
              op, ": block_tables must be int32 [", B, ", pages], each row contiguous and apart from the others");
  // the kernel's indices run a grid's width past these
  TORCH_CHECK(block_tables.size(1) * B <= (1 << 30), op, ": block_tables is too large");
  TORCH_CHECK(free_pages.dim() == 1 && free_pages.is_contiguous() && free_pages.scalar_type() == at::kInt &&
                  free_pages.size(0) < INT_MAX,
              op, ": free_pages must be a contiguous int32 vector");
  check_vector(op, "taken", taken, at::kInt, 1);
  TORCH_CHECK(page_size >= 16 && page_size % 16 == 0 && page_size <= (1 << 20), op,
              ": page_size must be a multiple of 16, got ", page_size);
  TORCH_CHECK(num_tokens >= 0 && num_tokens <= (1 << 30), op, ": bad num_tokens ", num_tokens);
  TORCH_CHECK(query_start || num_tokens >= B, op, ": num_tokens must be at least the ", B, " requests");
  const at::Tensor* starts = query_start ? &*query_start : nullptr;
  check_apart(op, {{"block_tables", &block_tables}},
              {{"cached", &cached}, {"query_start", starts}, {"free_pages", &free_pages}, {"taken", &taken}});
  check_devices(op, {{"cached", &cached},
                     {"query_start", starts},
                     {"block_tables", &block_tables},
                     {"free_pages", &free_pages},
                     {"taken", &taken}});
  const at::cuda::CUDAGuard guard(cached.device());
  Outputs outputs(cached);
  outputs.add({num_tokens}, at::kInt);
  outputs.add({num_tokens}, at::kLong);
  outputs.add({B}, at::kInt);
  outputs.add({1}, at::kInt);
  outputs.make();
  at::Tensor positions = outputs[0], slots = outputs[1], lengths = outputs[2], taken_out = outputs[3];
  nab::AssignPagesArgs a{};
  a.cached = cached.const_data_ptr<int>();
  a.starts = starts ? starts->const_data_ptr<int>() : nullptr;
  a.tables = block_tables.mutable_data_ptr<int>();
  a.table_stride = B == 1 ? 0 : block_tables.stride(0);
  a.free_pages = free_pages.const_data_ptr<int>();
  a.taken = taken.const_data_ptr<int>();
  a.positions = positions.mutable_data_ptr<int>();
  a.slots = slots.mutable_data_ptr<int64_t>();
  a.lengths = lengths.mutable_data_ptr<int>();
  a.taken_out = taken_out.mutable_data_ptr<int>();
  a.B = static_cast<int>(B);
  a.M = static_cast<int>(block_tables.size(1));
  a.F = static_cast<int>(free_pages.size(0));
  a.T = static_cast<int>(num_tokens);
  a.P = static_cast<int>(page_size);
  nab::assign_pages(at::cuda::getCurrentCUDAStream().stream(), a, sms_of(cached));
  return {positions, slots, lengths, taken_out};
}

// out: null for a new tensor (and in paged_attention: no scale for 1 / sqrt(head_dim))
at::Tensor rope_append_paged(const at::Tensor& qkv, const at::Tensor& cos, const at::Tensor& sin,
                                const at::Tensor& positions, const at::Tensor& slots, at::Tensor& k_pages,
                                at::Tensor& v_pages, int64_t q_heads, const OptTensor& q_norm, const OptTensor& k_norm,
                                double eps, bool interleaved, const at::Tensor* given) {
  constexpr const char* op = "rope_append_paged";
  const int dtype = half_dtype(op, qkv, "qkv");
  check_pages(op, k_pages, v_pages, qkv.scalar_type());
  const int64_t Hkv = k_pages.size(1), P = k_pages.size(2), D = k_pages.size(3), Hq = q_heads;
  TORCH_CHECK(Hq >= 1 && Hq < (1 << 20) && Hq % Hkv == 0, op, ": ", Hq, " query heads do not divide over ", Hkv,
              " kv heads");
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(1) == (Hq + 2 * Hkv) * D && qkv.stride(1) == 1, op, ": qkv must be [tokens, ",
              (Hq + 2 * Hkv) * D, "] with contiguous rows");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(given == nullptr || (given->dim() == 3 && given->size(0) == T && given->size(1) == Hq &&
                                   given->size(2) == D && given->is_contiguous() &&
                                   given->scalar_type() == qkv.scalar_type() && aligned16(*given)),
              op, ": out must be contiguous [", T, ", ", Hq, ", ", D, "] of qkv's type");
  TORCH_CHECK(aligned16(qkv) && (T <= 1 || qkv.stride(0) % 8 == 0), op, ": the rows of qkv must be 16-byte aligned");
  TORCH_CHECK(cos.dim() == 2 && cos.is_contiguous() && sin.is_contiguous() && sin.sizes() == cos.sizes() &&
                  cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat && cos.size(0) >= 1,
              op, ": cos and sin must be contiguous float32 [positions, rotary_dim / 2]");
  const int64_t R = 2 * cos.size(1);
  TORCH_CHECK(R % 16 == 0 && R >= 16 && R <= D, op, ": rotary_dim must be a multiple of 16 up to head_dim, got ", R);
  TORCH_CHECK(cos.size(0) < INT_MAX && aligned16(cos) && aligned16(sin), op, ": cos and sin must be 16-byte aligned");
  check_vector(op, "positions", positions, at::kInt, T);
  check_vector(op, "slots", slots, at::kLong, T);
  for (const auto& [name, w] : {std::pair<const char*, const OptTensor*>{"q_norm", &q_norm}, {"k_norm", &k_norm}}) {
    if (!*w) continue;
    check_vector(op, name, **w, qkv.scalar_type(), D);
    TORCH_CHECK(aligned16(**w), op, ": ", name, " must be 16-byte aligned");
  }
  const at::Tensor *qw = q_norm ? &*q_norm : nullptr, *kw = k_norm ? &*k_norm : nullptr;
  check_apart(op, {{"k_pages", &k_pages}, {"v_pages", &v_pages}, {"out", given}},
              {{"qkv", &qkv},
               {"cos", &cos},
               {"sin", &sin},
               {"positions", &positions},
               {"slots", &slots},
               {"q_norm", qw},
               {"k_norm", kw}});
  check_devices(op, {{"qkv", &qkv},
                     {"cos", &cos},
                     {"sin", &sin},
                     {"positions", &positions},
                     {"slots", &slots},
                     {"k_pages", &k_pages},
                     {"v_pages", &v_pages},
                     {"q_norm", qw},
                     {"k_norm", kw},
                     {"out", given}});
  const at::cuda::CUDAGuard guard(qkv.device());
  at::Tensor out = given ? *given : fresh({T, Hq, D}, qkv.scalar_type(), qkv);
  nab::RopeAppendArgs a{};
  a.qkv = qkv.const_data_ptr();
  a.qkv_stride = qkv.stride(0);
  a.cos_t = cos.const_data_ptr<float>();
  a.sin_t = sin.const_data_ptr<float>();
  a.positions = positions.const_data_ptr<int>();
  a.slots = slots.const_data_ptr<int64_t>();
  a.q_norm = qw ? qw->const_data_ptr() : nullptr;
  a.k_norm = kw ? kw->const_data_ptr() : nullptr;
  a.q_out = out.mutable_data_ptr();
  a.k_pages = k_pages.mutable_data_ptr();
  a.v_pages = v_pages.mutable_data_ptr();
  a.T = T;
  a.num_slots = k_pages.size(0) * P;
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.R = static_cast<int>(R);
  a.P = static_cast<int>(P);
  a.max_pos = static_cast<int>(cos.size(0));
  a.eps = static_cast<float>(eps);
  nab::rope_append_paged(at::cuda::getCurrentCUDAStream().stream(), a, dtype, interleaved, sms_of(qkv));
  return out;
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& k_pages, const at::Tensor& v_pages,
                              const at::Tensor& block_tables, const at::Tensor& lengths,
                              std::optional<double> scale,
                              const at::Tensor* given) {
  constexpr const char* op = "paged_attention";
  const int dtype = half_dtype(op, q, "q");
  check_pages(op, k_pages, v_pages, q.scalar_type());
  const int64_t Hkv = k_pages.size(1), P = k_pages.size(2), D = k_pages.size(3);
  TORCH_CHECK(q.dim() == 3 && q.size(1) >= 1 && q.size(2) == D, op, ": q must be [requests, q_heads, ", D, "]");
  const int64_t B = q.size(0), Hq = q.size(1);
  TORCH_CHECK(Hq % Hkv == 0, op, ": ", Hq, " query heads do not divide over ", Hkv, " kv heads");
  TORCH_CHECK(q.stride(2) == 1 && (Hq == 1 || q.stride(1) == D) && aligned16(q) &&
                  (B <= 1 || (q.stride(0) >= Hq * D && q.stride(0) % D == 0)),
              op, ": the heads of q must be contiguous and 16-byte aligned, its rows a multiple of head_dim apart");
  TORCH_CHECK(given == nullptr || (given->sizes() == q.sizes() && given->is_contiguous() &&
                                   given->scalar_type() == q.scalar_type() && aligned16(*given)),
              op, ": out must be contiguous, of q's shape and type");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == B && block_tables.scalar_type() == at::kInt &&
                  (block_tables.size(1) <= 1 || block_tables.stride(1) == 1),
              op, ": block_tables must be int32 [", B, ", pages] with contiguous rows");
  TORCH_CHECK(block_tables.size(1) * P <= INT_MAX - 127, op, ": block_tables is too wide");  // and a tile fits 32 bits
  check_vector(op, "lengths", lengths, at::kInt, B);
  check_apart(op, {{"out", given}},
              {{"q", &q},
               {"k_pages", &k_pages},
               {"v_pages", &v_pages},
               {"block_tables", &block_tables},
               {"lengths", &lengths}});
  check_devices(op, {{"q", &q},
                     {"k_pages", &k_pages},
                     {"v_pages", &v_pages},
                     {"block_tables", &block_tables},
                     {"lengths", &lengths},
                     {"out", given}});
  const at::cuda::CUDAGuard guard(q.device());
  at::Tensor out = given ? *given : fresh({B, Hq, D}, q.scalar_type(), q);
  if (B == 0) return out;
  const int sms = sms_of(q);
  nab::PagedAttnArgs a{};
  a.q = q.const_data_ptr();
  a.q_stride = q.stride(0);
  a.k_pages = k_pages.const_data_ptr();
  a.v_pages = v_pages.const_data_ptr();
  a.tables = block_tables.const_data_ptr<int>();
  a.table_stride = block_tables.stride(0);
  a.lengths = lengths.const_data_ptr<int>();
  a.out = out.mutable_data_ptr();
  a.num_pages = k_pages.size(0);
  a.B = static_cast<int>(B);
  a.M = static_cast<int>(block_tables.size(1));
  a.P = static_cast<int>(P);
  a.Hq = static_cast<int>(Hq);
  a.Hkv = static_cast<int>(Hkv);
  a.D = static_cast<int>(D);
  a.scale = static_cast<float>(scale.value_or(1.0 / std::sqrt(static_cast<double>(D))));
  // of this call alone: two streams or graphs never share it
  const at::Tensor ws = fresh({nab::paged_attention_ws_floats(a.B, a.M, a.P, a.Hq, a.Hkv, a.D, sms)}, at::kFloat, q);
  a.ws = ws.mutable_data_ptr<float>();
  nab::paged_attention(at::cuda::getCurrentCUDAStream().stream(), a, dtype, sms);
  return out;
}

using LogprobsResult = std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>;

LogprobsResult token_logprobs(const at::Tensor& logits, const at::Tensor& tokens, int64_t top_k,
                              int64_t vocab_start) {
  constexpr const char* op = "token_logprobs";
  TORCH_CHECK(logits.dim() == 2 && logits.size(1) >= 1 && (logits.size(1) == 1 || logits.stride(1) == 1), op,
              ": logits must be [rows, vocabulary] with contiguous rows");
  const int64_t rows = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V < (1 << 30), op, ": the vocabulary is too large");
  int dtype = nab::kF32;
  if (logits.scalar_type() != at::kFloat) {
    TORCH_CHECK(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf, op,
                ": logits must be float32, float16 or bfloat16, got ", logits.scalar_type());
    dtype = logits.scalar_type() == at::kHalf ? nab::kF16 : nab::kBF16;
  }
  check_vector(op, "tokens", tokens, at::kLong, rows);
  TORCH_CHECK(top_k >= 0 && top_k <= nab::kMaxTopK && top_k <= V, op, ": top_k must be from 0 to ", nab::kMaxTopK,
              " and at most the vocabulary, got ", top_k);
  TORCH_CHECK(vocab_start >= 0, op, ": vocab_start must not be negative");
  check_devices(op, {{"logits", &logits}, {"tokens", &tokens}});
  const at::cuda::CUDAGuard guard(logits.device());
  Outputs outputs(logits);
  for (int i = 0; i < 3; ++i) outputs.add({rows}, at::kFloat);
  outputs.add({rows, top_k}, at::kFloat);
  outputs.add({rows, top_k}, at::kLong);
  outputs.add({rows, top_k}, at::kFloat);
  outputs.make();
  at::Tensor logprob = outputs[0], entropy = outputs[1], lse = outputs[2], top_logprobs = outputs[3];
  at::Tensor top_tokens = outputs[4], top_logits = outputs[5];
  nab::LogprobsArgs a{};
  a.logits = logits.const_data_ptr();
  a.stride = logits.stride(0);
  a.tokens = tokens.const_data_ptr<int64_t>();
  a.vocab_start = vocab_start;
  a.logprob = logprob.mutable_data_ptr<float>();
  a.entropy = entropy.mutable_data_ptr<float>();
  a.lse = lse.mutable_data_ptr<float>();
  a.top_logprobs = top_logprobs.mutable_data_ptr<float>();
  a.top_tokens = top_tokens.mutable_data_ptr<int64_t>();
  a.top_logits = top_logits.mutable_data_ptr<float>();
  a.rows = rows;
  a.V = static_cast<int>(V);
  a.top_k = static_cast<int>(top_k);
  nab::token_logprobs(at::cuda::getCurrentCUDAStream().stream(), a, dtype, sms_of(logits));
  return {logprob, entropy, lse, top_logprobs, top_tokens, top_logits};
}

// ------------------------------------------------------ Python side --
// Whether the tensor's bytes are its values: not a fake, traced, batched or wrapped one, which the dispatcher would have
// taken elsewhere, nor one with a negation or conjugation pending.
bool plain(const at::Tensor& t) {
  using K = c10::DispatchKey;
  constexpr c10::DispatchKeySet other({K::Python, K::Functionalize, K::FuncTorchBatched, K::FuncTorchGradWrapper,
                                       K::BatchedNestedTensor, K::Negative, K::Conjugate, K::ZeroTensor});
  return !t.key_set().has_any(other) && t.layout() == at::kStrided && !t.is_meta() && t.has_storage();
}

// The positional arguments of a call, taken one after the other.
class Args {
 public:
  Args(const char* op, PyObject* const* args, Py_ssize_t n, Py_ssize_t wanted) : op_(op), args_(args) {
    TORCH_CHECK_TYPE(n == wanted, op, " takes ", wanted, " arguments, got ", n);
  }
  const at::Tensor& tensor(const char* name) {
    PyObject* o = args_[i_++];
    TORCH_CHECK_TYPE(THPVariable_Check(o), op_, ": ", name, " must be a tensor, got ", Py_TYPE(o)->tp_name);
    const at::Tensor& t = THPVariable_Unpack(o);
    TORCH_CHECK(t.defined() && plain(t), op_, ": ", name, " must be a plain tensor, got ", Py_TYPE(o)->tp_name, " of ",
                t.layout(), " layout, keys ", t.key_set());
    return t;
  }
  OptTensor optional_tensor(const char* name) {
    if (args_[i_] == Py_None) {
      ++i_;
      return std::nullopt;
    }
    return tensor(name);
  }
  int64_t integer(const char* name) {
    PyObject* o = args_[i_++];
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) refuse(name, "a 64-bit integer", o);
    return v;
  }
  std::optional<double> optional_number(const char* name) {
    if (args_[i_] == Py_None) {
      ++i_;
      return std::nullopt;
    }
    return number(name);
  }
  double number(const char* name) {
    PyObject* o = args_[i_++];
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) refuse(name, "a number", o);
    return v;
  }
  bool truth() {
    const int v = PyObject_IsTrue(args_[i_++]);
    if (v < 0) throw python_error();
    return v != 0;
  }

 private:
  void refuse(const char* name, const char* what, PyObject* o) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, op_, ": ", name, " must be ", what, ", got ", Py_TYPE(o)->tp_name);
  }
  const char* op_;
  PyObject* const* args_;
  Py_ssize_t i_ = 0;
};

// Runs f without the GIL, as an event that profilers see, with its inputs.
template <typename F, typename... Inputs>
auto without_gil(const char* name, F&& f, const Inputs&... inputs) {
  struct Released {
    PyThreadState* state = PyEval_SaveThread();
    ~Released() { PyEval_RestoreThread(state); }
  } released;
  const auto values = [&] { return std::vector<c10::IValue>{c10::IValue(inputs)...}; };  // made when one is listening
  RECORD_FUNCTION(name, values());
  return f();
}

template <typename... T>
PyObject* tuple_of(const std::tuple<T...>& tensors) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (r == nullptr) throw python_error();
  Py_ssize_t i = 0;
  std::apply([&](const auto&... t) { (PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t)), ...); }, tensors);
  return r;
}

PyObject* py_assign_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("assign_pages", args, n, 7);
  const at::Tensor& cached = a.tensor("cached");
  const OptTensor query_start = a.optional_tensor("query_start");
  at::Tensor block_tables = a.tensor("block_tables");
  const at::Tensor &free_pages = a.tensor("free_pages"), &taken = a.tensor("taken");
  const int64_t page_size = a.integer("page_size"), num_tokens = a.integer("num_tokens");
  return tuple_of(without_gil("nab::assign_pages", [&] {
    return assign_pages(cached, query_start, block_tables, free_pages, taken, page_size, num_tokens);
  }, cached, query_start, block_tables, free_pages, taken, page_size, num_tokens));
  END_HANDLE_TH_ERRORS
}

PyObject* py_rope_append_paged(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("rope_append_paged", args, n, 13);
  const at::Tensor &qkv = a.tensor("qkv"), &cos = a.tensor("cos"), &sin = a.tensor("sin");
  const at::Tensor &positions = a.tensor("positions"), &slots = a.tensor("slots");
  at::Tensor k_pages = a.tensor("k_pages"), v_pages = a.tensor("v_pages");
  const int64_t q_heads = a.integer("q_heads");
  const OptTensor q_norm = a.optional_tensor("q_norm"), k_norm = a.optional_tensor("k_norm");
  const double eps = a.number("eps");
  const bool interleaved = a.truth();
  const OptTensor out = a.optional_tensor("out");
  return THPVariable_Wrap(without_gil("nab::rope_append_paged", [&] {
    return rope_append_paged(qkv, cos, sin, positions, slots, k_pages, v_pages, q_heads, q_norm, k_norm, eps,
                             interleaved, out ? &*out : nullptr);
  }, qkv, cos, sin, positions, slots, k_pages, v_pages, q_heads, q_norm, k_norm, eps, interleaved, out));
  END_HANDLE_TH_ERRORS
}

PyObject* py_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("paged_attention", args, n, 7);
  const at::Tensor &q = a.tensor("q"), &k_pages = a.tensor("k_pages"), &v_pages = a.tensor("v_pages");
  const at::Tensor &block_tables = a.tensor("block_tables"), &lengths = a.tensor("lengths");
  const std::optional<double> scale = a.optional_number("scale");
  const OptTensor out = a.optional_tensor("out");
  return THPVariable_Wrap(without_gil("nab::paged_attention", [&] {
    return paged_attention(q, k_pages, v_pages, block_tables, lengths, scale, out ? &*out : nullptr);
  }, q, k_pages, v_pages, block_tables, lengths, scale, out));
  END_HANDLE_TH_ERRORS
}

PyObject* py_token_logprobs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Args a("token_logprobs", args, n, 4);
  const at::Tensor &logits = a.tensor("logits"), &tokens = a.tensor("tokens");
  const int64_t top_k = a.integer("top_k"), vocab_start = a.integer("vocab_start");
  return tuple_of(without_gil("nab::token_logprobs",
                              [&] { return token_logprobs(logits, tokens, top_k, vocab_start); }, logits, tokens, top_k,
                              vocab_start));
  END_HANDLE_TH_ERRORS
}

// Whether NAB_CHECK asks for a check after every launch (os.environ's changes reach getenv).
PyObject* py_check_requested(PyObject*, PyObject*) {
  const char* v = std::getenv("NAB_CHECK");
  if (v == nullptr || *v == '\0') Py_RETURN_FALSE;
  Py_RETURN_TRUE;  // any value: the caller reads it
}

template <typename F>
PyCFunction method(F* f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef kMethods[] = {
    {"assign_pages", method(py_assign_pages), METH_FASTCALL,
     "assign_pages(cached, query_start, block_tables, free_pages, taken, page_size, num_tokens)"},
    {"rope_append_paged", method(py_rope_append_paged), METH_FASTCALL,
     "rope_append_paged(qkv, cos, sin, positions, slots, k_pages, v_pages, q_heads, q_norm, k_norm, eps, interleaved, "
     "out)"},
    {"paged_attention", method(py_paged_attention), METH_FASTCALL,
     "paged_attention(q, k_pages, v_pages, block_tables, lengths, scale, out)"},
    {"token_logprobs", method(py_token_logprobs), METH_FASTCALL, "token_logprobs(logits, tokens, top_k, vocab_start)"},
    {"check_requested", method(py_check_requested), METH_NOARGS, "whether NAB_CHECK is set"},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_C", "Serving operators; the other ops are torch.ops.nab.*", -1,
                       kMethods,              nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__C() { return PyModule_Create(&kModule); }
