// Python bindings of the serving operators: rotary positions, attention over a shared prefix, rules
// on logits.  Arguments are checked here; outputs and workspaces come from the caching allocator on
// the current stream, per call, so calls on several streams or in several captured graphs share none.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <string>
#include <vector>

#include "kernels.h"
#include "serving.h"

int* pra_attention_status_word(const torch::Device& dev);

namespace {

using torch::Tensor;
using OptTensor = c10::optional<torch::Tensor>;

// Numbers in error messages (streaming an integer goes through the process's locale facets, which
// another library's copy of the C++ runtime can leave unusable).
std::string num(int64_t v) { return std::to_string(v); }

inline cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

void check(cudaError_t e, const char* what) {
  TORCH_CHECK(e == cudaSuccess, "pra_ops.", what, " failed: ", cudaGetErrorString(e));
}

int dtype_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return PRA_BF16;
    case at::kHalf: return PRA_FP16;
    case at::kFloat: return PRA_FP32;
    default: break;
  }
  TORCH_CHECK(false, name, " has dtype ", t.scalar_type(), ", expected bf16, fp16 or fp32");
  return -1;
}

// A tensor of the call: on the device of the first one.
void same(const Tensor& t, const Tensor& first, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == first.device(), name, " must be on ", first.device(), ", it is on ", t.device());
}

void typed(const Tensor& t, at::ScalarType dt, const Tensor& first, const char* name) {
  same(t, first, name);
  TORCH_CHECK(t.scalar_type() == dt, name, " has dtype ", t.scalar_type(), ", expected ", dt);
}

// A contiguous vector with one entry per row.
template <typename T>
const T* per_row(const OptTensor& t, at::ScalarType dt, const Tensor& first, int64_t rows, const char* name) {
  if (!t.has_value()) return nullptr;
  typed(*t, dt, first, name);
  TORCH_CHECK(t->dim() == 1 && t->size(0) == rows && t->is_contiguous(), name, " must be a contiguous vector of ", num(rows),
              " entries");
  return static_cast<const T*>(t->data_ptr());
}

// ---------------------------------------------------------------- rotary
void rotary_tables(RotaryArgs& a, const Tensor& cos_t, const Tensor& sin_t, const Tensor& first, int64_t head_dim,
                   bool interleaved) {
  typed(cos_t, at::kFloat, first, "cos");
  typed(sin_t, at::kFloat, first, "sin");
  TORCH_CHECK(cos_t.dim() == 2 && cos_t.is_contiguous() && sin_t.is_contiguous() && cos_t.sizes() == sin_t.sizes(),
              "cos and sin must be contiguous [positions, rotary_dim / 2] tables of one shape");
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.max_pos = cos_t.size(0);
  TORCH_CHECK(a.max_pos > 0, "cos and sin hold no positions");
  a.rot = (int)(2 * cos_t.size(1));
  TORCH_CHECK(head_dim > 0 && head_dim % 2 == 0 && head_dim <= 4096, "head_dim must be even and at most 4096");
  TORCH_CHECK(a.rot >= 2 && a.rot <= head_dim, "the table rotates ", num(a.rot), " elements of a head of ",
              num(head_dim));
  a.head_dim = (int)head_dim;
  a.interleaved = interleaved;
}

void rotary_positions(RotaryArgs& a, const Tensor& positions, const Tensor& first) {
  same(positions, first, "positions");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
              "positions must be int32 or int64");
  TORCH_CHECK(positions.is_contiguous(), "positions must be contiguous");
  a.pos = positions.data_ptr();
  a.pos64 = positions.scalar_type() == at::kLong;
}

// The one stride with which the leading dimensions of [..., heads, head_dim] walk its tokens in order; -1: there is
// none.  Dimensions of size 1 are never walked: their strides say nothing.
int64_t token_stride(at::IntArrayRef sizes, at::IntArrayRef strides) {
  int64_t stride = 0, next = -1;  // the innermost walked dimension's stride; what the dimension around it has to have
  for (int64_t d = (int64_t)sizes.size() - 3; d >= 0; --d) {
    if (sizes[d] == 1) continue;
    if (next < 0) stride = strides[d];
    else if (strides[d] != next) return -1;
    next = strides[d] * sizes[d];
  }
  return stride;
}

// The segment of x [..., heads, head_dim] (read in place where its tokens have one stride) and its new output.
Tensor rotary_segment(RotarySegment& s, Tensor& x, int64_t head_dim) {
  TORCH_CHECK(x.dim() >= 2 && x.size(-1) == head_dim, "queries and keys must be [..., heads, head_dim] of one head_dim");
  auto out = torch::empty(x.sizes(), x.options());
  const int64_t heads = x.size(-2);
  TORCH_CHECK(heads <= 4096, "at most 4096 heads");
  const int64_t token = token_stride(x.sizes(), x.strides());
  const bool strided = (x.stride(-1) == 1 && token >= 0) || x.numel() == 0;
  if (!strided) x = x.contiguous();
  s.src = x.data_ptr();
  s.src_token = strided && x.numel() > 0 ? token : heads * head_dim;
  s.src_head = x.stride(-2);
  s.dst = out.data_ptr();
  s.dst_token = heads * head_dim;
  s.dst_head = head_dim;
  s.heads = (int)heads;
  s.rotate = 1;
  return out;
}

std::vector<OptTensor> rotate(Tensor q, OptTensor k, const Tensor& positions, const Tensor& cos_t, const Tensor& sin_t,
                              bool interleaved, bool inverse) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  const int dtype = dtype_code(q, "q");
  TORCH_CHECK(q.dim() >= 2, "q must be [..., heads, head_dim]");
  RotaryArgs a{};
  rotary_tables(a, cos_t, sin_t, q, q.size(-1), interleaved);
  rotary_positions(a, positions, q);
  a.inverse = inverse;
  a.tokens = positions.numel();
  TORCH_CHECK(q.dim() == positions.dim() + 2 && q.sizes().slice(0, q.dim() - 2) == positions.sizes(),
              "positions must have the leading dimensions of q");
  std::vector<OptTensor> result;
  result.emplace_back(rotary_segment(a.seg[0], q, a.head_dim));
  if (k.has_value()) {
    typed(*k, q.scalar_type(), q, "k");
    TORCH_CHECK(k->dim() == q.dim() && k->sizes().slice(0, q.dim() - 2) == positions.sizes(),
                "k must have the leading dimensions of q");
    result.emplace_back(rotary_segment(a.seg[1], *k, a.head_dim));
  } else {
    result.emplace_back(c10::nullopt);
  }
  if (a.seg[0].heads + a.seg[1].heads > 0) check(pra_rotary(a, dtype, stream()), "rotary");
  return result;
}

std::vector<OptTensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& cos_t,
                              const Tensor& sin_t, bool interleaved, bool inverse);

// The rotation is linear in (q, k): its backward is the transposed rotation, differentiable again.
struct Rotary : torch::autograd::Function<Rotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const OptTensor& k,
                                                const Tensor& positions, const Tensor& cos_t, const Tensor& sin_t,
                                                bool interleaved, bool inverse) {
    at::AutoDispatchBelowADInplaceOrView guard;
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions, cos_t, sin_t});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    auto y = rotate(q, k, positions, cos_t, sin_t, interleaved, inverse);
    if (!k.has_value()) return {*y[0]};
    return {*y[0], *y[1]};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["interleaved"].toBool(), inverse = ctx->saved_data["inverse"].toBool();
    torch::autograd::variable_list dx(7);
    const bool dq = dy[0].defined(), dk = dy.size() > 1 && dy[1].defined();
    if (dq || dk) {  // where only one of the two took part, it goes alone
      const auto r = rotary(dq ? dy[0] : dy[1], dq && dk ? OptTensor(dy[1]) : OptTensor(), saved[0], saved[1], saved[2],
                            interleaved, !inverse);
      dx[dq ? 0 : 1] = *r[0];
      if (dq && dk) dx[1] = *r[1];
    }
    return dx;
  }
};

std::vector<OptTensor> rotary(const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& cos_t,
                              const Tensor& sin_t, bool interleaved, bool inverse) {
  const auto dual = [](const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); };
  TORCH_CHECK(!dual(q) && !(k.has_value() && dual(*k)) && !dual(cos_t) && !dual(sin_t),
              "rotary has no forward-mode derivatives (the map is linear: rotate the tangents)");
  TORCH_CHECK(!torch::GradMode::is_enabled() || !(cos_t.requires_grad() || sin_t.requires_grad()),
              "rotary has no gradients for its table: detach cos and sin");
  if (!torch::GradMode::is_enabled() || !(q.requires_grad() || (k.has_value() && k->requires_grad())))
    return rotate(q, k, positions, cos_t, sin_t, interleaved, inverse);
  auto y = Rotary::apply(q, k, positions, cos_t, sin_t, interleaved, inverse);
  if (!k.has_value()) return {y[0], c10::nullopt};
  return {y[0], y[1]};
}

Tensor rotary_cache(Tensor qkv, int64_t heads, int64_t kv_heads, int64_t head_dim, Tensor positions, Tensor cos_t,
                    Tensor sin_t, bool interleaved, Tensor k_cache, Tensor v_cache, Tensor slots) {
  TORCH_CHECK(qkv.is_cuda(), "qkv must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(qkv.device());
  const int dtype = dtype_code(qkv, "qkv");
  TORCH_CHECK(heads >= 0 && kv_heads > 0 && heads <= 4096 && kv_heads <= 4096, "1 to 4096 heads");
  RotaryArgs a{};
  rotary_tables(a, cos_t, sin_t, qkv, head_dim, interleaved);
  rotary_positions(a, positions, qkv);
  TORCH_CHECK(qkv.dim() == 2 && qkv.stride(1) == 1 && qkv.size(1) >= (heads + 2 * kv_heads) * head_dim,
              "qkv must be [tokens, >= (heads + 2 kv_heads) * head_dim] with contiguous rows");
  a.tokens = qkv.size(0);
  TORCH_CHECK(positions.numel() == a.tokens, "one position per token");
  a.slots = per_row<int>(slots, at::kInt, qkv, a.tokens, "slots");
  for (const Tensor* c : {&k_cache, &v_cache}) {
    typed(*c, qkv.scalar_type(), qkv, "the caches");
    TORCH_CHECK(c->dim() == 2 && c->stride(1) == 1 && c->size(1) >= kv_heads * head_dim && c->size(0) == k_cache.size(0),
                "the caches must be [rows, >= kv_heads * head_dim] with contiguous rows");
    TORCH_CHECK(c->size(0) <= 1 || c->stride(0) >= kv_heads * head_dim, "cache rows overlap");
  }
  a.slot_rows = k_cache.size(0);
  auto q = torch::empty({a.tokens, heads * head_dim}, qkv.options());
  const int64_t size = qkv.element_size(), ld = qkv.stride(0);
  char* base = static_cast<char*>(qkv.data_ptr());
  a.seg[0] = {base, q.data_ptr(), ld, head_dim, heads * head_dim, head_dim, (int)heads, 1, 0};
  a.seg[1] = {base + heads * head_dim * size, k_cache.data_ptr(), ld, head_dim, k_cache.stride(0), head_dim, (int)kv_heads, 1, 1};
  a.seg[2] = {base + (heads + kv_heads) * head_dim * size, v_cache.data_ptr(), ld, head_dim, v_cache.stride(0), head_dim, (int)kv_heads, 0, 1};
  check(pra_rotary(a, dtype, stream()), "rotary_cache");
  return q;
}

// ---------------------------------------------------------------- rules on logits
struct Rules {
  OptTensor ids, hist_len, prompt_len, repetition, presence, frequency, bias_ids, bias_values, mask, mask_rows;
};

LogitsArgs rules_args(const Tensor& logits, const Rules& r, int64_t vocab_start) {
  TORCH_CHECK(logits.dim() == 2 && (logits.stride(1) == 1 || logits.size(1) <= 1), "logits must be [B, V] with contiguous rows");
  LogitsArgs a{};
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(B <= 65535, "at most 65535 rows of logits");
  TORCH_CHECK(V > 0, "logits need at least one column");
  TORCH_CHECK(vocab_start >= 0 && vocab_start % 8 == 0, "vocab_start must be a multiple of 8");
  TORCH_CHECK(vocab_start + V <= INT32_MAX - 64, "token ids must fit 31 bits");
  a.logits = logits.data_ptr();
  a.in_stride = logits.stride(0);
  a.B = (int)B;
  a.V = (int)V;
  a.vocab_start = (int)vocab_start;
  TORCH_CHECK(r.ids.has_value() == r.hist_len.has_value(), "a history is ids and lengths");
  if (r.ids.has_value()) {
    typed(*r.ids, at::kInt, logits, "history ids");
    TORCH_CHECK(r.ids->dim() == 2 && r.ids->size(0) == B && (r.ids->stride(1) == 1 || r.ids->size(1) <= 1),
                "history ids must be [B, capacity] with contiguous rows");
    TORCH_CHECK(r.ids->size(1) < PRA_RULES_MAX_HISTORY, "a history holds fewer than ", num(PRA_RULES_MAX_HISTORY), " ids");
    a.ids = r.ids->data_ptr<int>();
    a.ids_stride = r.ids->stride(0);
    a.capacity = (int)r.ids->size(1);
    a.hist_len = const_cast<int*>(per_row<int>(r.hist_len, at::kInt, logits, B, "history lengths"));
    a.prompt_len = per_row<int>(r.prompt_len, at::kInt, logits, B, "prompt lengths");
    a.repetition = per_row<float>(r.repetition, at::kFloat, logits, B, "repetition");
    a.presence = per_row<float>(r.presence, at::kFloat, logits, B, "presence");
    a.frequency = per_row<float>(r.frequency, at::kFloat, logits, B, "frequency");
  }
  TORCH_CHECK(r.bias_ids.has_value() == r.bias_values.has_value(), "biases are ids and values");
  if (r.bias_ids.has_value() && r.bias_ids->numel() > 0) {
    typed(*r.bias_ids, at::kInt, logits, "bias ids");
    typed(*r.bias_values, at::kFloat, logits, "bias values");
    TORCH_CHECK(r.bias_ids->dim() == 2 && r.bias_ids->size(0) == B && r.bias_ids->sizes() == r.bias_values->sizes() &&
                    r.bias_ids->is_contiguous() && r.bias_values->is_contiguous(),
                "bias ids and values must be contiguous [B, n]");
    TORCH_CHECK(r.bias_ids->size(1) <= PRA_RULES_MAX_BIASES, "at most ", num(PRA_RULES_MAX_BIASES), " biases a row");
    a.bias_ids = r.bias_ids->data_ptr<int>();
    a.bias_values = r.bias_values->data_ptr<float>();
    a.n_bias = (int)r.bias_ids->size(1);
  }
  if (r.mask.has_value()) {
    typed(*r.mask, at::kInt, logits, "mask");
    TORCH_CHECK(r.mask->dim() == 2 && r.mask->is_contiguous() && r.mask->size(1) * 32 >= vocab_start + V,
                "mask must be contiguous [masks, >= ceil(vocabulary / 32)] int32 words");
    TORCH_CHECK(r.mask_rows.has_value() || r.mask->size(0) == B, "one mask per row, or mask_rows");
    a.mask = reinterpret_cast<const uint32_t*>(r.mask->data_ptr<int>());
    a.mask_count = (int)r.mask->size(0);
    a.mask_words = r.mask->size(1);
    a.mask_rows = per_row<int>(r.mask_rows, at::kInt, logits, B, "mask_rows");
  } else {
    TORCH_CHECK(!r.mask_rows.has_value(), "mask_rows without a mask");
  }
  TORCH_CHECK((a.ids == nullptr && a.bias_ids == nullptr) || V <= PRA_RULES_MAX_VOCAB, "a history or biases need at most ",
              num(PRA_RULES_MAX_VOCAB), " columns");
  return a;
}

Tensor process_logits(Tensor logits, OptTensor out_in, OptTensor ids, OptTensor hist_len, OptTensor prompt_len,
                      OptTensor repetition, OptTensor presence, OptTensor frequency, OptTensor bias_ids,
                      OptTensor bias_values, OptTensor mask, OptTensor mask_rows, int64_t vocab_start) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(logits.device());
  const int dtype = dtype_code(logits, "logits");
  LogitsArgs a = rules_args(logits, {ids, hist_len, prompt_len, repetition, presence, frequency, bias_ids, bias_values, mask, mask_rows}, vocab_start);
  Tensor out;
  if (out_in.has_value()) {
    out = *out_in;
    typed(out, logits.scalar_type(), logits, "out");
    TORCH_CHECK(out.sizes() == logits.sizes() && (out.stride(1) == 1 || out.size(1) <= 1), "out must be shaped as logits");
    TORCH_CHECK(out.size(0) <= 1 || out.stride(0) >= out.size(1), "rows of out overlap");
    const auto extent = [](const Tensor& t) { return ((t.size(0) - 1) * t.stride(0) + t.size(1)) * t.element_size(); };
    const char* x = static_cast<const char*>(logits.data_ptr());
    const char* y = static_cast<const char*>(out.data_ptr());
    TORCH_CHECK(logits.size(0) == 0 || (x == y && (out.size(0) == 1 || out.stride(0) == logits.stride(0))) ||
                    x + extent(logits) <= y || y + extent(out) <= x,
                "out must be logits itself or not overlap it");
  } else {
    out = torch::empty(logits.sizes(), logits.options());
  }
  a.out = out.data_ptr();
  a.out_stride = out.stride(0);
  check(pra_logits_rules(a, dtype, stream()), "process_logits");
  return out;
}

std::vector<Tensor> choose_tokens(Tensor logits, OptTensor ids, OptTensor hist_len, OptTensor prompt_len,
                                  OptTensor repetition, OptTensor presence, OptTensor frequency, OptTensor bias_ids,
                                  OptTensor bias_values, OptTensor mask, OptTensor mask_rows, int64_t vocab_start,
                                  bool append) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(logits.device());
  const int dtype = dtype_code(logits, "logits");
  LogitsArgs a = rules_args(logits, {ids, hist_len, prompt_len, repetition, presence, frequency, bias_ids, bias_values, mask, mask_rows}, vocab_start);
  TORCH_CHECK(!append || ids.has_value(), "append needs a history");
  TORCH_CHECK(!append || ids->size(0) <= 1 || ids->stride(0) >= ids->size(1), "rows of an appended history overlap");
  auto token = torch::empty({logits.size(0)}, logits.options().dtype(at::kLong));
  auto value = torch::empty({logits.size(0)}, logits.options().dtype(at::kFloat));
  a.token = token.data_ptr<int64_t>();
  a.value = value.data_ptr<float>();
  if (append) a.append_ids = const_cast<int*>(a.ids);
  check(pra_logits_rules(a, dtype, stream()), "choose_tokens");
  return {token, value};
}

// ---------------------------------------------------------------- attention over a shared prefix
// Rows of 16-byte pieces that the tensor-memory accelerator can address.
void rows_ok(const Tensor& t, int64_t width, const char* name) {
  TORCH_CHECK(t.stride(-1) == 1 && t.size(-1) >= width, name, " needs contiguous rows of at least ", num(width), " elements");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name, " must start on a 16-byte boundary");
  for (int64_t d = 0; d + 1 < t.dim(); ++d)
    TORCH_CHECK(t.size(d) <= 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0), name, " needs strides that are multiples of 16 bytes");
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// > 0: launches from here on give up in front of a CTA's copy of that number, as if its wait had run out (set by tests
// of that way).
int give_up = 0;

// {out [like q], lse [B, H, T] or none}, or with `partials` {unnormalised o [B * T, H, 1, D], (max, sum)
// [B * T, H, 1, 2]}.
std::vector<OptTensor> prefix_attention(Tensor q, Tensor pk, Tensor pv, Tensor k, Tensor v, Tensor lengths,
                                               int64_t heads, int64_t kv_heads, int64_t head_dim,
                                               OptTensor prefix_lengths, double scale, bool return_lse,
                                               bool partials) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  c10::cuda::CUDAGuard guard(q.device());
  TORCH_CHECK(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
  TORCH_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
  TORCH_CHECK(std::isfinite((float)scale) && (float)scale > 0, "scale must be positive, in 32 bits");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16, "q has dtype ", q.scalar_type(), ", expected bf16");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == heads * head_dim, "q must be [B, T, heads * head_dim]");
  rows_ok(q, heads * head_dim, "q");
  const int64_t width = kv_heads * head_dim;
  for (const Tensor* t : {&pk, &pv, &k, &v}) typed(*t, at::kBFloat16, q, "keys and values");
  TORCH_CHECK(pk.dim() == 2 && pv.dim() == 2 && pk.size(0) == pv.size(0), "prefix keys and values must be [P, kv_heads * head_dim]");
  TORCH_CHECK(k.dim() == 3 && v.dim() == 3 && k.size(0) == q.size(0) && v.size(0) == q.size(0) && k.size(1) == v.size(1),
              "own keys and values must be [B, capacity, kv_heads * head_dim]");
  const int64_t B = q.size(0), T = q.size(1), G = heads / kv_heads;
  TORCH_CHECK(pk.size(0) < (1 << 30) && k.size(1) < (1 << 30) && B * T * G < (1 << 30) && B * kv_heads < (1 << 24),
              "too many keys or queries");
  if (pk.size(0) > 0) rows_ok(pk, width, "prefix keys"), rows_ok(pv, width, "prefix values");
  if (k.size(1) > 0 && B > 0) {
    rows_ok(k, width, "own keys"), rows_ok(v, width, "own values");
    // tensor maps are specified with outer strides that are multiples of the inner ones
    for (const Tensor* t : {&k, &v})
      TORCH_CHECK(B == 1 || k.size(1) == 1 || t->stride(0) % t->stride(1) == 0,
                  "the batch stride of own keys and values must be a multiple of their row stride");
  }
  PrefixAttnArgs a{};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_batch = q.stride(0);
  a.q_token = q.stride(1);
  a.pk = reinterpret_cast<const __nv_bfloat16*>(pk.data_ptr());
  a.pv = reinterpret_cast<const __nv_bfloat16*>(pv.data_ptr());
  a.P = (int)pk.size(0);
  // the stride of a single row is never walked, but the tensor maps want a real one
  a.pk_row = pk.size(0) > 1 ? pk.stride(0) : width;
  a.pv_row = pv.size(0) > 1 ? pv.stride(0) : width;
  a.prefix_len = per_row<int>(prefix_lengths, at::kInt, q, B, "prefix_lengths");
  a.k = reinterpret_cast<const __nv_bfloat16*>(k.data_ptr());
  a.v = reinterpret_cast<const __nv_bfloat16*>(v.data_ptr());
  a.cap = (int)k.size(1);
  // (and of a single own row the batch stride is a multiple)
  a.k_row = k.size(1) > 1 ? k.stride(1) : B > 1 ? k.stride(0) : width;
  a.v_row = v.size(1) > 1 ? v.stride(1) : B > 1 ? v.stride(0) : width;
  a.k_batch = B > 1 ? k.stride(0) : a.cap * a.k_row;
  a.v_batch = B > 1 ? v.stride(0) : a.cap * a.v_row;
  a.len = per_row<int>(lengths, at::kInt, q, B, "lengths");
  a.B = (int)B;
  a.T = (int)T;
  a.H = (int)heads;
  a.Hkv = (int)kv_heads;
  a.D = (int)head_dim;
  a.scale = (float)scale;
  a.status = pra_attention_status_word(q.device());
  a.give_up = give_up;
  const auto fo = q.options().dtype(at::kFloat);
  // One allocation for the call's parts: n slots of sums and (max, sum) pairs for each of the queries, and `more`
  // floats.
  Tensor work;
  const auto workspace = [&](int64_t n, int64_t more, int64_t queries) {
    const int64_t own = (queries * n * (head_dim + 2) + 3) / 4 * 4;  // what follows: 16-byte aligned
    work = torch::empty({own + more}, fo);
    a.n_slots = (int)n;
    a.part_o = n > 0 ? work.data_ptr<float>() : nullptr;
    a.part_ml = n > 0 ? a.part_o + queries * n * head_dim : nullptr;
    return work.data_ptr<float>() + own;
  };
  // The joined partial that a call for partials returns.
  Tensor joined_o, joined_ml;
  const auto joined = [&]() -> std::vector<OptTensor> {
    joined_o = torch::empty({B * T, heads, 1, head_dim}, fo);
    joined_ml = torch::empty({B * T, heads, 1, 2}, fo);
    return {joined_o, joined_ml};
  };
  Tensor out;
  if (!partials) out = torch::empty({B, T, heads * head_dim}, q.options());
  std::vector<OptTensor> result{out, c10::nullopt};
  float* lse = nullptr;
  if (return_lse && !partials) {
    auto l = torch::empty({B, heads, T}, q.options().dtype(at::kFloat));
    lse = l.data_ptr<float>();
    result[1] = l;
  }
  if (B == 0 || T == 0 || (a.P == 0 && a.cap == 0)) {
    if (partials) {
      auto r = joined();
      joined_o.zero_();
      joined_ml.zero_();
      joined_ml.select(-1, 0).fill_(-INFINITY);
      return r;
    }
    out.zero_();
    if (return_lse) result[1]->fill_(-INFINITY);
    return result;
  }
  if (!partials) a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.lse = lse;
  const int prefix_blocks = ceil_div(a.P, 128), own_blocks = ceil_div(a.cap, 128);
  // Up to `most` parts of a tile's blocks.  In us: 2 (1.6) per block of a part, and each part costs the merge 0.1, more
  // than 30 of them another 3 (a second round).  One row behind 32K with 2 KV heads: 64 parts 22.8 us, all 148 that
  // run at once 27.4; 2 x 4 drafts behind 6,877 keys, head dim 64: 24 parts 17.7 us, 54 23.4.
  const auto best_splits = [head_dim](int blocks, int most) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= std::min(blocks, most); ++s) {
      const double us = (head_dim == 128 ? 2.0 : 1.6) * ceil_div(blocks, s) + 0.1 * s + (s > 30 ? 3 : 0);
      if (us < least) {
        least = us;
        best = s;
      }
    }
    return best;
  };
  const auto splits_for = [&](const PrefixAttnArgs& p, int blocks) {
    int tiles, slots;
    pra_prefix_attention_shape(p, &tiles, &slots);
    return best_splits(blocks, slots / tiles);
  };
  PrefixMergeArgs m{};
  m.B = a.B;
  m.T = a.T;
  m.H = a.H;
  m.Hkv = a.Hkv;
  m.D = a.D;
  const auto merge = [&]() -> std::vector<OptTensor> {
    m.part_o = a.part_o;
    m.part_ml = a.part_ml;
    m.n_slots = a.part_o != nullptr ? a.n_slots : 0;
    auto r = partials ? joined() : result;
    if (partials) {
      m.joined_o = joined_o.data_ptr<float>();
      m.joined_ml = joined_ml.data_ptr<float>();
    } else {
      m.out = a.out;
      m.lse = lse;
    }
    check(pra_prefix_merge(m, stream()), "shared_prefix_attention");
    return r;
  };
  const int64_t rows = T * G;  // query rows of a (batch row, KV head)
  const bool few = rows <= PRA_OWN_ROWS && a.cap > 0;
  // A batch row with 256 or more query rows of a KV head (or the only batch row) fills its tiles: prefix and own
  // keys in one walk.  Else the prefix is walked once for the query rows of the whole batch, and the own
  // keys on their own.
  if (a.cap == 0 || rows >= 256 || (B == 1 && a.P > 0) || (a.P == 0 && !few)) {
    a.packed = a.cap == 0;
    a.use_prefix = a.P > 0;
    a.use_own = a.cap > 0;
    const int blocks = prefix_blocks + own_blocks;
    a.splits = splits_for(a, blocks);
    std::vector<OptTensor> r = result;
    int tiles, slots, tile_rows;
    pra_prefix_attention_shape(a, &tiles, &slots, &tile_rows);
    if (a.splits == 1 && tiles % slots != 0 && prefix_blocks >= own_blocks && !partials) {
      // The tiles behind the last full wave are split among all SMs (where their keys are mostly the prefix, alike
      // for all: causal tiles of all lengths fill the last wave anyway, 4,096 queries without a prefix took 3%
      // longer).  In blocks of 128 keys: a CTA takes 5 more than its keys, the join 2 and what it writes and reads.
      // 3, 4 and 5 x 512 queries behind 16K (192, 256 and 320 tiles on 148 SMs) 544 -> 405, 485 -> 480 and
      // 731 -> 571 us.
      const int behind = tiles % slots;
      double best = blocks + 5;
      for (int s = 2; s <= std::min(16, blocks); ++s) {
        const double cost = ceil_div((int64_t)behind * s, slots) * (ceil_div(blocks, s) + 5.0) + 2 +
                            behind * s * (tile_rows * head_dim / 32768.0) * 0.014;
        if (cost < best) {
          best = cost;
          a.splits = s;
        }
      }
      a.whole = a.splits > 1 ? tiles - behind : 0;
      if (a.whole > 0) {
        m.tile0 = a.whole;
        m.tiles = behind;
        m.tile_rows = tile_rows;
        m.packed = a.packed;
      }
    }
    if (a.splits > 1) {
      if (a.whole > 0) workspace(a.splits, 0, (int64_t)m.tiles * tile_rows);
      else workspace(a.splits, 0, B * T * heads);
    } else if (partials) {
      r = joined();
      a.part_o = joined_o.data_ptr<float>();
      a.part_ml = joined_ml.data_ptr<float>();
      a.n_slots = 1;
    }
    check(pra_prefix_attention(a, stream()), "shared_prefix_attention");
    return a.splits > 1 ? merge() : r;
  }
  PrefixAttnArgs own = a;
  if (a.P > 0) {
    a.packed = a.use_prefix = 1;
    a.splits = splits_for(a, prefix_blocks);
  }
  if (few) {
    // Both parts at once where that is shorter.  The lengths are not known here: half of the capacity (64 rows of 64 to
    // 150 own keys behind 8K take 30 us at a capacity of 160, 35 at 1,280 and 39 from 4,096 on).
    // Times in us as measured, for head dim 128 (64), with two own CTAs on an SM; of 10 to 16 query rows of head dim 128
    // one fits, and the own part then is the longer one (64 x 2 drafts behind 4K 33 us, 64 x 3 60).
    int own_ctas = INT32_MAX;
    if (a.P > 0) {
      int tiles, slots;
      pra_prefix_attention_shape(a, &tiles, &slots);
      const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
      const bool wide = head_dim == 128;
      const double own_kb = 2e-3 * B * a.cap * width;
      if (slots == sms) {
        // Two tiles a CTA: the prefix part is bound by its products and the own part by HBM, each takes its SMs.
        // A prefix CTA takes 13 (4) + 1.85 (1.6) per block; an SM of own CTAs 0.34 (0.26) per block of 64 keys, two
        // more of them per item, up to HBM's rate, behind which more SMs help little.  64 rows behind 8K with
        // 64 to 1,024 own keys 68 -> 46 us, 128 rows behind 32K 140 -> 107 us.
        const auto prefix_us = [&](int splits) { return (wide ? 13 : 4) + (wide ? 1.85 : 1.6) * ceil_div(prefix_blocks, splits); };
        const double block_kb = 0.256 * head_dim, blocks = (double)B * kv_heads * (a.cap / 128.0 + 2.5);
        const auto own_us = [&](int s) {
          const double rate = s * block_kb / (wide ? 0.34 : 0.26);
          return 6 + blocks * block_kb / (rate < 5800 ? rate : 5800 + 0.25 * (rate - 5800));
        };
        double best = prefix_us(a.splits) + 4 + own_kb / 6000;
        int splits = 0;
        for (int s = std::min(prefix_blocks, (sms - 4) / tiles); s >= 1 && sms - s * tiles <= sms * 3 / 4; --s) {
          const double us = std::max(prefix_us(s), own_us(sms - s * tiles));
          if (us < best) {
            best = us;
            splits = s;
          }
        }
        if (splits > 0) {
          a.splits = splits;
          own_ctas = 2 * (sms - splits * tiles);
        }
      } else if (tiles <= sms) {
        // One tile a CTA: a CTA of each part fits on an SM.
        // A prefix CTA takes 8 + 2 (1.6) per block, two of them on an SM 2.9 (2).
        const int splits = best_splits(prefix_blocks, sms / tiles);
        const auto prefix_us = [&](int s, double per_block) { return 8 + per_block * ceil_div(prefix_blocks, s); };
        const double both = std::max(prefix_us(splits, wide ? 2.0 : 1.6), 6 + own_kb / 6000);
        const double after =
            prefix_us(a.splits, a.splits > splits ? (wide ? 2.9 : 2.0) : (wide ? 2.0 : 1.6)) + 4 + own_kb / 6000;
        if (both < after) {
          a.splits = splits;
          own_ctas = sms;
        }
      }
    }
    OwnAttnArgs o{};
    o.q = a.q;
    o.q_batch = a.q_batch;
    o.q_token = a.q_token;
    o.k = a.k;
    o.v = a.v;
    o.k_batch = a.k_batch;
    o.k_row = a.k_row;
    o.v_batch = a.v_batch;
    o.v_row = a.v_row;
    o.cap = a.cap;
    o.len = a.len;
    o.B = a.B;
    o.T = a.T;
    o.H = a.H;
    o.Hkv = a.Hkv;
    o.D = a.D;
    o.scale = a.scale;
    o.status = a.status;
    o.give_up = a.give_up;
    o.after_prefix = a.P > 0;
    o.ctas = pra_own_attention_ctas(o);
    o.ctas = std::min(o.ctas, own_ctas);
    // behind the slots: the pieces' sums, their (max, sum) pairs, the items' first and last CTAs
    const int64_t items = B * kv_heads, pieces = (items + o.ctas) * rows;
    o.piece_o = workspace(a.P > 0 ? a.splits : 0, pieces * (head_dim + 2) + 2 * items, B * T * heads);
    o.piece_ml = o.piece_o + pieces * head_dim;
    o.first = reinterpret_cast<int*>(o.piece_ml + pieces * 2);
    o.last = o.first + items;
    m.piece_o = o.piece_o;
    m.piece_ml = o.piece_ml;
    m.first = o.first;
    m.last = o.last;
    if (a.P > 0) check(pra_prefix_attention(a, stream()), "shared_prefix_attention");
    check(pra_own_attention(o, stream()), "shared_prefix_attention");
    return merge();
  }
  own.use_own = 1;
  own.splits = splits_for(own, own_blocks);
  workspace(a.splits + own.splits, 0, B * T * heads);
  own.part_o = a.part_o;
  own.part_ml = a.part_ml;
  own.n_slots = a.n_slots;
  own.slot0 = a.splits;
  own.after_prefix = 1;
  check(pra_prefix_attention(a, stream()), "shared_prefix_attention");
  check(pra_prefix_attention(own, stream()), "shared_prefix_attention");
  return merge();
}

// {out [B, T, H * D] bf16, lse [B, H, T] or none} of one or two sets of partials [B * T, H, n, D].
std::vector<OptTensor> merge_attention_partials(Tensor part_o, Tensor part_ml, OptTensor more_o, OptTensor more_ml,
                                                int64_t batch, bool return_lse) {
  TORCH_CHECK(part_o.is_cuda(), "partials must be CUDA tensors");
  c10::cuda::CUDAGuard guard(part_o.device());
  TORCH_CHECK(more_o.has_value() == more_ml.has_value(), "partials are sums and (max, sum) pairs");
  const auto set = [&](const Tensor& o, const Tensor& ml) {
    typed(o, at::kFloat, part_o, "partials");
    typed(ml, at::kFloat, part_o, "partials");
    TORCH_CHECK(o.dim() == 4 && ml.dim() == 4 && o.is_contiguous() && ml.is_contiguous() && ml.size(3) == 2 &&
                    o.sizes().slice(0, 3) == ml.sizes().slice(0, 3) && o.size(0) == part_o.size(0) &&
                    o.size(1) == part_o.size(1) && o.size(3) == part_o.size(3),
                "partials must be contiguous [B * T, H, n, D] and [B * T, H, n, 2]");
    TORCH_CHECK(reinterpret_cast<uintptr_t>(o.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(ml.data_ptr()) % 8 == 0,
                "partials must start on a 16-byte boundary");
  };
  set(part_o, part_ml);
  const int64_t rows = part_o.size(0), H = part_o.size(1), D = part_o.size(3);
  TORCH_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128");
  TORCH_CHECK(batch > 0 ? rows % batch == 0 : rows == 0, "the partials hold whole batch rows");
  PrefixMergeArgs m{};
  m.part_o = part_o.data_ptr<float>();
  m.part_ml = part_ml.data_ptr<float>();
  m.n_slots = (int)part_o.size(2);
  if (more_o.has_value()) {
    set(*more_o, *more_ml);
    m.more_o = more_o->data_ptr<float>();
    m.more_ml = more_ml->data_ptr<float>();
    m.n_more = (int)more_o->size(2);
  }
  m.B = (int)batch;
  m.T = batch > 0 ? (int)(rows / batch) : 0;
  m.H = m.Hkv = (int)H;
  m.D = (int)D;
  auto out = torch::empty({batch, m.T, H * D}, part_o.options().dtype(at::kBFloat16));
  m.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  std::vector<OptTensor> result{out, c10::nullopt};
  if (return_lse) {
    auto l = torch::empty({batch, H, m.T}, part_o.options());
    m.lse = l.data_ptr<float>();
    result[1] = l;
  }
  check(pra_prefix_merge(m, stream()), "merge_attention_partials");
  return result;
}

}  // namespace

void pra_bind_serving_ops(pybind11::module_& m) {
  m.def("rotary", &rotary);
  m.def("rotary_cache", &rotary_cache);
  m.def("token_stride", [](const std::vector<int64_t>& sizes, const std::vector<int64_t>& strides) { return token_stride(sizes, strides); });
  m.def("process_logits", &process_logits);
  m.def("choose_tokens", &choose_tokens);
  m.def("shared_prefix_attention", &prefix_attention);
  m.def("merge_attention_partials", &merge_attention_partials);
  m.def("prefix_attention_give_up", [](int64_t copy) { give_up = (int)copy; });
}
