// torch_binding.cpp -- the PyTorch side of bfa_rope, bfa_tree_fwd,
// bfa_verify_tree and bfa_cache_append: checks of arguments, outputs and
// workspaces from torch's allocator, the current stream, autograd of the
// rotation. Compiled into bfa_torch.so, which calls libbfa.so through its C ABI
// alone.
//
// These calls run once or more per layer of a decoding step whose kernels take
// a few microseconds. The same checks and argument blocks written in Python
// made a call 16 to 33 us of host time, several times what the kernels take; from
// here one takes 6 to 7, the attention, with four tensor maps and two launches, 12.
//
// A failed check raises what the attention functions raise: AssertionError for
// shapes that do not fit together, ValueError for arguments that make no
// sense, RuntimeError for dtypes and devices.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>
#include <initializer_list>
#include <optional>
#include <sstream>
#include <string>
#include <tuple>

#include "bfa.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  const py::gil_scoped_acquire gil;  // autograd runs a backward without it
  PyErr_SetString(type, msg.c_str());
  throw py::error_already_set();
}
// The message is only formed where the check fails.
#define BFA_ASSERT(cond, ...) \
  if (C10_UNLIKELY(!(cond))) raise(PyExc_AssertionError, c10::str(__VA_ARGS__))
#define BFA_VALUE(cond, ...) \
  if (C10_UNLIKELY(!(cond))) raise(PyExc_ValueError, c10::str(__VA_ARGS__))
#define BFA_RUNTIME(cond, ...) \
  if (C10_UNLIKELY(!(cond))) raise(PyExc_RuntimeError, c10::str(__VA_ARGS__))

void require_cuda(const char* what, const Tensor& t, const at::Device& dev) {
  BFA_RUNTIME(t.is_cuda(), what, " (B200 build) needs CUDA tensors; there is no CPU path");
  BFA_RUNTIME(t.device() == dev, what, ": tensors on ", dev.str(), " and ", t.device().str(), "; they must share a device");
}
const at::Device first_device(const char* what, const Tensor& t) {
  BFA_RUNTIME(t.is_cuda(), what, " (B200 build) needs CUDA tensors; there is no CPU path");
  return t.device();
}

// A tangent of forward-mode differentiation would be lost: the outputs are new
// tensors that know nothing of it.
void refuse_tangents(const char* what, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs)
    BFA_RUNTIME(!(t->defined() && t->_fw_grad(/*level=*/0).defined()), what, " has no forward-mode derivative (an input carries a tangent)");
}

// Operators without a backward: a gradient that an input wants would be lost.
void refuse_gradients(const char* what, std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : inputs)
    BFA_RUNTIME(!(t->defined() && t->requires_grad()), what, " has no backward; call it under torch.no_grad()");
}

// Written in place: autograd finds out from the version that a tensor it saved
// has changed. (Inference tensors have none.)
void note_written(const Tensor& t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int64_t dtype_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return BFA_DTYPE_F32;
    case at::kHalf: return BFA_DTYPE_F16;
    case at::kBFloat16: return BFA_DTYPE_BF16;
    default: break;
  }
  raise(PyExc_RuntimeError, c10::str("unsupported dtype ", t.scalar_type(), " (need float32, float16 or bfloat16)"));
}

int64_t int_bytes(const Tensor& t, const char* what) {
  BFA_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, what, " must be int32 or int64, got ", t.scalar_type());
  return t.scalar_type() == at::kInt ? 4 : 8;
}

bfa_tensor flat(const Tensor& t) {
  bfa_tensor r;
  r.data = t.data_ptr();
  for (int i = 0; i < 4; ++i) r.stride[i] = t.stride(i);
  return r;
}

// The device's status word, owned by bfa_lib (one int32 per device).
int32_t* status_word(const at::Device& dev) {
  static int32_t* words[64] = {};
  const int i = dev.index();
  if (i < 64 && words[i]) return words[i];
  const py::gil_scoped_acquire gil;
  const auto at = py::module_::import("bfa_lib").attr("status_ptr")(i).cast<uintptr_t>();
  if (i < 64) words[i] = reinterpret_cast<int32_t*>(at);
  return reinterpret_cast<int32_t*>(at);
}

void check(int rc) {
  if (C10_LIKELY(rc == BFA_OK)) return;
  std::string msg = bfa_strerror(rc);
  if (rc == BFA_ERR_CUDA && bfa_last_error()[0]) msg += std::string(" (") + bfa_last_error() + ")";
  raise(PyExc_RuntimeError, msg);
}

void* stream_of(const at::Device& dev) { return at::cuda::getCurrentCUDAStream(dev.index()).stream(); }

std::string shape_of(const Tensor& t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}

// ------------------------------------------------------------------ rotary
void rope_launch(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions, const Tensor& offsets,
                 bool interleaved, bool inverse, const Tensor& qo, const Tensor& ko) {
  const Tensor& some = q.defined() ? q : k;
  const at::Device dev = some.device();
  bfa_rope_args a{};
  a.batch = some.size(0);
  a.heads_q = q.defined() ? q.size(1) : 0;
  a.heads_k = k.defined() ? k.size(1) : 0;
  a.seqlen = some.size(2);
  a.head_dim = some.size(3);
  a.rotary_dim = 2 * cos.size(1);
  a.dtype = dtype_of(some);
  a.interleaved = interleaved;
  a.inverse = inverse;
  if (q.defined()) a.q = flat(q), a.q_out = flat(qo);
  if (k.defined()) a.k = flat(k), a.k_out = flat(ko);
  a.cos = cos.data_ptr<float>();
  a.sin = sin.data_ptr<float>();
  a.table_rows = cos.size(0);
  a.table_stride = cos.stride(0);
  if (positions.defined()) {
    a.positions = positions.data_ptr();
    a.positions_bytes = int_bytes(positions, "positions");
    a.positions_stride[1] = positions.stride(-1);
    a.positions_stride[0] = positions.dim() == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
  }
  if (offsets.defined()) {
    a.offsets = offsets.data_ptr();
    a.offsets_bytes = int_bytes(offsets, "offsets");
  }
  const c10::cuda::CUDAGuard guard(dev);
  a.status = status_word(dev);
  check(bfa_rope(&a, stream_of(dev)));
}

Tensor like(const Tensor& t) { return t.defined() ? at::empty_like(t) : Tensor(); }

// The gradient of a rotation is the transposed rotation of the gradients, so
// only the table and the positions are saved; the backward is the same
// function with `inverse` turned, and differentiable in its turn.
std::tuple<Tensor, Tensor> rope_apply(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                                      const Tensor& offsets, bool interleaved, bool inverse);

struct RotaryEmbedding : torch::autograd::Function<RotaryEmbedding> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const OptTensor& q, const OptTensor& k,
                                                const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                                                const OptTensor& offsets, bool interleaved, bool inverse) {
    const Tensor qt = q.value_or(Tensor()), kt = k.value_or(Tensor()), pt = positions.value_or(Tensor()), ot = offsets.value_or(Tensor());
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({cos, sin, pt, ot});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["inverse"] = inverse;
    ctx->saved_data["q"] = qt.defined();
    // An input that needs no gradient gets none, and its output wants none.
    const bool need_q = qt.defined() && qt.requires_grad(), need_k = kt.defined() && kt.requires_grad();
    ctx->saved_data["need_q"] = need_q;
    ctx->saved_data["need_k"] = need_k;
    const Tensor qo = like(qt), ko = like(kt);
    rope_launch(qt, kt, cos, sin, pt, ot, interleaved, inverse, qo, ko);
    torch::autograd::variable_list out, constant;
    if (qo.defined()) out.push_back(qo);
    if (ko.defined()) out.push_back(ko);
    if (qo.defined() && !need_q) constant.push_back(qo);
    if (ko.defined() && !need_k) constant.push_back(ko);
    ctx->mark_non_differentiable(constant);
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const bool has_q = ctx->saved_data["q"].toBool();
    const Tensor dq = ctx->saved_data["need_q"].toBool() ? grads[0] : Tensor();
    const Tensor dk = ctx->saved_data["need_k"].toBool() ? grads[has_q ? 1 : 0] : Tensor();
    Tensor gq, gk;
    if (dq.defined() || dk.defined())
      std::tie(gq, gk) = rope_apply(dq, dk, saved[0], saved[1], saved[2], saved[3], ctx->saved_data["interleaved"].toBool(),
                                    !ctx->saved_data["inverse"].toBool());
    return {gq, gk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> rope_apply(const Tensor& q, const Tensor& k, const Tensor& cos, const Tensor& sin, const Tensor& positions,
                                      const Tensor& offsets, bool interleaved, bool inverse) {
  const bool grads = at::GradMode::is_enabled() && ((q.defined() && q.requires_grad()) || (k.defined() && k.requires_grad()));
  if (!grads) {
    const Tensor qo = like(q), ko = like(k);
    rope_launch(q, k, cos, sin, positions, offsets, interleaved, inverse, qo, ko);
    return {qo, ko};
  }
  auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  auto out = RotaryEmbedding::apply(opt(q), opt(k), cos, sin, opt(positions), opt(offsets), interleaved, inverse);
  return {q.defined() ? out[0] : Tensor(), k.defined() ? out.back() : Tensor()};
}

// Whether two tensors of one shape are the same elements (strides of dims of
// length 1 do not count).
bool same_elements(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr()) return false;
  for (int i = 0; i < 4; ++i)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}
// Whether they are known to share memory (ATen's rule, which leaves views that
// interleave in one buffer to the caller, plus equal addresses).
bool share_memory(const Tensor& a, const Tensor& b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const auto status = at::get_overlap_status(a, b);
  return status == at::MemOverlapStatus::Full || status == at::MemOverlapStatus::Partial || a.data_ptr() == b.data_ptr();
}

using QkPair = std::tuple<OptTensor, OptTensor>;

QkPair rotary_embedding(const OptTensor& query, const OptTensor& key, const Tensor& cos, const Tensor& sin, const OptTensor& positions,
                        const OptTensor& offsets, bool interleaved, const std::optional<QkPair>& out) {
  const char* what = "rotary_embedding";
  const Tensor q = query.value_or(Tensor()), k = key.value_or(Tensor());
  const Tensor pos = positions.value_or(Tensor()), off = offsets.value_or(Tensor());
  BFA_VALUE(q.defined() || k.defined(), "rotary_embedding needs query or key");
  const Tensor& first = q.defined() ? q : k;
  BFA_ASSERT(first.dim() == 4, "query and key are [B, H, S, D]");
  const int64_t B = first.size(0), S = first.size(2), D = first.size(3);
  if (q.defined() && k.defined()) {
    BFA_ASSERT(k.dim() == 4 && k.size(0) == B && k.size(2) == S && k.size(3) == D,
               "query and key must agree in batch, length and head dim");
    BFA_RUNTIME(k.scalar_type() == q.scalar_type(), "query and key must have one dtype");
  }
  refuse_tangents(what, {&q, &k, &cos, &sin});
  const at::Device dev = first_device(what, first);
  for (const Tensor* t : {&k, &cos, &sin, &pos, &off})
    if (t->defined()) require_cuda(what, *t, dev);
  BFA_VALUE(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin must be fp32");
  BFA_VALUE(cos.dim() == 2 && cos.sizes() == sin.sizes() && cos.strides() == sin.strides() && (cos.size(1) <= 1 || cos.stride(1) == 1),
            "cos and sin must be [positions, rotary_dim / 2] of one layout with unit inner stride");
  BFA_ASSERT(cos.size(1) > 0 && 2 * cos.size(1) <= D, "rotary_dim must be in 2..head_dim");
  BFA_VALUE(!cos.requires_grad() && !sin.requires_grad(), "the rotary table is not differentiable here");
  if (pos.defined()) {
    BFA_VALUE((pos.dim() == 1 && pos.size(0) == S) || (pos.dim() == 2 && (pos.size(0) == B || pos.size(0) == 1) && pos.size(1) == S),
              "positions must be [", S, "] or [", B, ", ", S, "], got ", shape_of(pos));
    int_bytes(pos, "positions");
  }
  if (off.defined()) {
    BFA_VALUE(off.dim() == 1 && off.size(0) == B && (B <= 1 || off.stride(0) == 1), "offsets must be a contiguous [", B, "], got ",
              shape_of(off));
    int_bytes(off, "offsets");
  }
  auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  if (out) {
    const Tensor qo = std::get<0>(*out).value_or(Tensor()), ko = std::get<1>(*out).value_or(Tensor());
    for (const Tensor* t : {&q, &k, &qo, &ko})
      BFA_VALUE(!(at::GradMode::is_enabled() && t->defined() && t->requires_grad()), "out= is not differentiable; call it under torch.no_grad()");
    refuse_tangents(what, {&qo, &ko});
    auto fits = [](const Tensor& t, const Tensor& o) {
      return t.defined() == o.defined() &&
             (!t.defined() || (o.sizes() == t.sizes() && o.scalar_type() == t.scalar_type() && o.device() == t.device()));
    };
    BFA_VALUE(fits(q, qo), "out for query must match it in shape, dtype and device");
    BFA_VALUE(fits(k, ko), "out for key must match it in shape, dtype and device");
    for (const Tensor* t : {&qo, &ko})
      BFA_VALUE(!t->defined() || at::has_internal_overlap(*t) != at::MemOverlap::Yes, "out has elements that share memory");
    // The heads are turned side by side, in no order: a result may lie where its
    // own input does and nowhere else among what the call reads and writes.
    auto apart = [](const Tensor& a, const Tensor& b) { return !a.defined() || !b.defined() || !share_memory(a, b); };
    BFA_VALUE((!q.defined() || same_elements(q, qo) || apart(q, qo)) && (!k.defined() || same_elements(k, ko) || apart(k, ko)) &&
                  apart(qo, k) && apart(ko, q) && apart(qo, ko),
              "out may be the inputs themselves, but not overlap them, or itself, in another way");
    rope_launch(q, k, cos, sin, pos, off, interleaved, false, qo, ko);
    note_written(qo), note_written(ko);
    return {std::get<0>(*out), std::get<1>(*out)};
  }
  Tensor qo, ko;
  std::tie(qo, ko) = rope_apply(q, k, cos, sin, pos, off, interleaved, false);
  return {opt(qo), opt(ko)};
}

// ------------------------------------------------------------------ cache and tree
struct Cache {
  Tensor k_pages, v_pages, table, lens;
};

void check_cache(const char* what, const Cache& c, int64_t B, int64_t Hkv, int64_t D, at::ScalarType dt, const at::Device& dev) {
  BFA_VALUE(c.k_pages.dim() == 4 && c.v_pages.sizes() == c.k_pages.sizes() && c.k_pages.size(1) == Hkv && c.k_pages.size(3) == D, what,
            ": pages must be two [num_pages, ", Hkv, ", page_size, ", D, "] tensors, got ", shape_of(c.k_pages), " and ",
            shape_of(c.v_pages));
  BFA_RUNTIME(c.k_pages.scalar_type() == dt && c.v_pages.scalar_type() == dt, what, ": pages must have the dtype of the new tokens, ", dt);
  BFA_VALUE(D <= 1 || (c.k_pages.stride(3) == 1 && c.v_pages.stride(3) == 1), what, ": pages need a unit innermost stride");
  BFA_VALUE(c.table.scalar_type() == at::kInt && c.table.dim() == 2 && c.table.size(0) == B &&
                (c.table.size(1) <= 1 || c.table.stride(1) == 1),
            what, ": page_table must be int32 [", B, ", max_pages] with unit inner stride");
  BFA_VALUE(c.lens.scalar_type() == at::kInt && c.lens.dim() == 1 && c.lens.size(0) == B && (B <= 1 || c.lens.stride(0) == 1), what,
            ": lens must be a contiguous int32 [", B, "]");
  for (const Tensor* t : {&c.k_pages, &c.v_pages, &c.table, &c.lens}) require_cuda(what, *t, dev);
}

// The tree's pointer and row stride; none is a chain.
std::pair<const int32_t*, int64_t> check_parents(const char* what, const OptTensor& parents, int64_t B, int64_t N, const at::Device& dev) {
  if (!parents) return {nullptr, 0};
  const Tensor& t = *parents;
  const bool shape = (t.dim() == 1 && t.size(0) == N) || (t.dim() == 2 && (t.size(0) == B || t.size(0) == 1) && t.size(1) == N);
  BFA_VALUE(t.scalar_type() == at::kInt && shape && (N <= 1 || t.stride(-1) == 1), what, ": parents must be int32 [", N, "] or [", B, ", ",
            N, "] with unit inner stride, got ", t.scalar_type(), " ", shape_of(t));
  require_cuda(what, t, dev);
  return {t.data_ptr<int32_t>(), t.dim() == 2 && t.size(0) > 1 ? t.stride(0) : 0};
}

// Rows of head_dim elements are read in place; other layouts are copied.
Tensor rows(const Tensor& t) { return t.stride(3) == 1 || t.size(3) == 1 ? t : t.contiguous(); }

constexpr int64_t kMaxNodes = 64;

std::tuple<Tensor, OptTensor> tree_attention(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& k_pages,
                                             const Tensor& v_pages, const Tensor& table, const Tensor& lens, const OptTensor& parents,
                                             std::optional<double> scale, int64_t sliding_window, double soft_cap,
                                             const OptTensor& alibi_slope, bool return_lse) {
  const char* what = "tree_attention";
  BFA_ASSERT(query.dim() == 4 && key.dim() == 4 && value.dim() == 4, "query, key and value are [B, H, N, D]");
  const int64_t B = query.size(0), Hq = query.size(1), N = query.size(2), D = query.size(3), Hkv = key.size(1);
  BFA_ASSERT(key.size(0) == B && key.size(2) == N && key.size(3) == D && value.sizes() == key.sizes(),
             "key and value must be [B, Hkv, N, D] of the query's B, N, D");
  BFA_ASSERT(Hkv > 0 && Hq % Hkv == 0, "Hq must be divisible by Hkv");
  BFA_VALUE(N >= 1 && N <= kMaxNodes, "a tree has 1 to ", kMaxNodes, " nodes, got ", N);
  BFA_VALUE(sliding_window >= 0 && soft_cap >= 0, "sliding_window and soft_cap must be >= 0");
  const at::ScalarType dt = query.scalar_type();
  BFA_RUNTIME(key.scalar_type() == dt && value.scalar_type() == dt, "query, key and value must have one dtype");
  refuse_tangents(what, {&query, &key, &value, &k_pages, &v_pages});
  if (alibi_slope) refuse_tangents(what, {&*alibi_slope});
  const at::Device dev = first_device(what, query);
  require_cuda(what, key, dev);
  require_cuda(what, value, dev);
  refuse_gradients(what, {&query, &key, &value, &k_pages, &v_pages});
  if (alibi_slope) refuse_gradients(what, {&*alibi_slope});
  check_cache(what, {k_pages, v_pages, table, lens}, B, Hkv, D, dt, dev);
  const auto up = check_parents(what, parents, B, N, dev);
  Tensor slopes;
  if (alibi_slope) {
    slopes = alibi_slope->to(dev, at::kFloat).reshape({-1}).contiguous();
    BFA_RUNTIME(slopes.numel() == Hq, "alibi_slope must have one slope per query head (", Hq, "), got ", slopes.numel());
  }
  const Tensor q = rows(query), k = rows(key), v = rows(value);
  bfa_tree_args a{};
  a.batch = B, a.heads_q = Hq, a.heads_kv = Hkv, a.nodes = N, a.head_dim = D;
  a.dtype = dtype_of(query);
  a.num_pages = k_pages.size(0), a.page_size = k_pages.size(2), a.max_pages = table.size(1);
  a.sliding_window = sliding_window;
  a.scale = scale ? *scale : 1.0 / std::sqrt((double)D);
  a.soft_cap = soft_cap;
  a.alibi_slopes = slopes.defined() ? slopes.data_ptr<float>() : nullptr;
  a.q = flat(q), a.k = flat(k), a.v = flat(v);
  a.k_pages = flat(k_pages), a.v_pages = flat(v_pages);
  a.page_table = table.data_ptr<int32_t>(), a.page_table_stride = table.stride(0);
  a.lens = lens.data_ptr<int32_t>();
  a.parents = up.first, a.parents_stride = up.second;
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor o = at::empty({B, Hq, N, D}, query.options().requires_grad(false));
  OptTensor lse;
  if (return_lse) lse = at::empty({B, Hq, N}, o.options().dtype(at::kFloat));
  a.o = flat(o);
  a.lse = lse ? lse->data_ptr<float>() : nullptr;
  a.status = status_word(dev);
  // Scratch of the partial results, from torch's caching allocator: the library allocates nothing.
  a.workspace_bytes = (int64_t)bfa_tree_workspace_bytes(&a);
  const Tensor ws = at::empty({a.workspace_bytes}, o.options().dtype(at::kByte));
  a.workspace = ws.data_ptr();
  check(bfa_tree_fwd(&a, stream_of(dev)));
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> verify_tree(const Tensor& target_probs, const Tensor& draft_tokens, const OptTensor& parents,
                                               const Tensor& uniforms, const Tensor& noise, const OptTensor& draft_probs) {
  const char* what = "verify_tree";
  BFA_ASSERT(target_probs.dim() == 3, "target_probs is [B, N, V]");
  const int64_t B = target_probs.size(0), N = target_probs.size(1), V = target_probs.size(2);
  BFA_VALUE(N >= 1 && N <= kMaxNodes, "a tree has 1 to ", kMaxNodes, " nodes, got ", N);
  BFA_VALUE(V >= 1, "the vocabulary is empty");
  auto is = [](const Tensor& t, int64_t a, int64_t b) { return t.dim() == 2 && t.size(0) == a && t.size(1) == b; };
  BFA_VALUE(is(draft_tokens, B, N), "draft_tokens must be [", B, ", ", N, "], got ", shape_of(draft_tokens));
  const int64_t token_bytes = int_bytes(draft_tokens, "draft_tokens");
  BFA_VALUE(uniforms.scalar_type() == at::kFloat && is(uniforms, B, N) && noise.scalar_type() == at::kFloat && is(noise, B, V),
            "uniforms must be fp32 [", B, ", ", N, "] and noise fp32 [", B, ", ", V, "]");
  BFA_VALUE(!draft_probs || (draft_probs->sizes() == target_probs.sizes() && draft_probs->scalar_type() == target_probs.scalar_type()),
            "draft_probs must match target_probs in shape and dtype");
  const at::Device dev = first_device(what, target_probs);
  for (const Tensor* t : {&draft_tokens, &uniforms, &noise}) require_cuda(what, *t, dev);
  if (draft_probs) require_cuda(what, *draft_probs, dev);
  const auto up = check_parents(what, parents, B, N, dev);
  auto unit = [](const Tensor& t) { return t.stride(-1) == 1 || t.size(-1) == 1 ? t : t.contiguous(); };
  const Tensor p = unit(target_probs), tokens = unit(draft_tokens), u = unit(uniforms), e = unit(noise);
  const Tensor q = draft_probs ? unit(*draft_probs) : Tensor();
  bfa_verify_args a{};
  a.batch = B, a.nodes = N, a.vocab = V;
  a.dtype = dtype_of(p);
  a.target = p.data_ptr(), a.target_stride[0] = p.stride(0), a.target_stride[1] = p.stride(1);
  if (q.defined()) a.draft = q.data_ptr(), a.draft_stride[0] = q.stride(0), a.draft_stride[1] = q.stride(1);
  a.tokens = tokens.data_ptr(), a.tokens_bytes = token_bytes, a.tokens_stride = tokens.stride(0);
  a.parents = up.first, a.parents_stride = up.second;
  a.uniforms = u.data_ptr<float>(), a.uniforms_stride = u.stride(0);
  a.noise = e.data_ptr<float>(), a.noise_stride = e.stride(0);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = at::empty({B * (N + 2)}, p.options().dtype(at::kInt).requires_grad(false));
  a.path = out.data_ptr<int32_t>(), a.count = a.path + B * N, a.next_token = a.count + B;
  a.status = status_word(dev);
  check(bfa_verify_tree(&a, stream_of(dev)));
  return {out.as_strided({B, N}, {N, 1}), out.as_strided({B}, {1}, B * N), out.as_strided({B}, {1}, B * (N + 1))};
}

Tensor cache_append(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens, const Tensor& key,
                    const Tensor& value, const OptTensor& take, const OptTensor& count) {
  const char* what = "cache_append";
  BFA_ASSERT(key.dim() == 4 && value.sizes() == key.sizes(), "key and value are [B, Hkv, S, D]");
  const int64_t B = key.size(0), Hkv = key.size(1), S = key.size(2), D = key.size(3);
  BFA_RUNTIME(value.scalar_type() == key.scalar_type(), "key and value must have one dtype");
  refuse_tangents(what, {&key, &value, &k_pages, &v_pages});
  const at::Device dev = first_device(what, key);
  require_cuda(what, value, dev);
  refuse_gradients(what, {&key, &value, &k_pages, &v_pages});
  check_cache(what, {k_pages, v_pages, table, lens}, B, Hkv, D, key.scalar_type(), dev);
  bfa_append_args a{};
  if (take) {
    BFA_VALUE(take->scalar_type() == at::kInt && take->dim() == 2 && take->size(0) == B && take->size(1) == S &&
                  (S <= 1 || take->stride(1) == 1),
              "take must be int32 [", B, ", ", S, "] with unit inner stride");
    require_cuda(what, *take, dev);
    a.take = take->data_ptr<int32_t>(), a.take_stride = take->stride(0);
  }
  if (count) {
    BFA_VALUE(count->scalar_type() == at::kInt && count->dim() == 1 && count->size(0) == B && (B <= 1 || count->stride(0) == 1),
              "count must be a contiguous int32 [", B, "]");
    require_cuda(what, *count, dev);
    a.count = count->data_ptr<int32_t>();
  }
  a.batch = B, a.heads_kv = Hkv, a.tokens = S, a.head_dim = D;
  a.dtype = dtype_of(key);
  a.num_pages = k_pages.size(0), a.page_size = k_pages.size(2), a.max_pages = table.size(1);
  a.k = flat(key), a.v = flat(value), a.k_pages = flat(k_pages), a.v_pages = flat(v_pages);
  a.page_table = table.data_ptr<int32_t>(), a.page_table_stride = table.stride(0);
  a.lens = lens.data_ptr<int32_t>();
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor out = at::empty({B}, lens.options());
  a.lens_out = out.data_ptr<int32_t>();
  a.status = status_word(dev);
  check(bfa_cache_append(&a, stream_of(dev)));
  note_written(k_pages), note_written(v_pages);
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("rotary_embedding", &rotary_embedding);
  m.def("tree_attention", &tree_attention);
  m.def("verify_tree", &verify_tree);
  m.def("cache_append", &cache_append);
}
