// Calls of the operators on a paged K/V cache (rotary positions, append, attention, eviction) for torch tensors: argument
// checks, outputs and workspaces from torch's allocator, torch's current stream of the tensors' device, and the gradient of the
// rotary turn, on top of the C ABI. Native for the same reason as torch_calls.cc: a decoding step's kernels take 3 to 15 us, and
// a call's way through Python, ctypes and the allocator would take longer.
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pycfunction_helpers.h>

#include <array>
#include <cmath>

#include "fa2_b200.h"

namespace {

using at::Tensor;

#define VALUE_CHECK(cond, ...) \
  if (!(cond)) C10_THROW_ERROR(ValueError, c10::str(__VA_ARGS__))
#define TYPE_CHECK(cond, ...) \
  if (!(cond)) C10_THROW_ERROR(TypeError, c10::str(__VA_ARGS__))

Tensor empty(at::IntArrayRef shape, c10::ScalarType type, c10::Device dev) {
  return Tensor(at::detail::empty_cuda(shape, type, dev, std::nullopt));
}

void check(int rc) {
  if (rc == FA2_OK) return;
  if (rc == FA2_E_TYPE) C10_THROW_ERROR(TypeError, fa2_last_error());
  if (rc == FA2_E_VALUE) C10_THROW_ERROR(ValueError, fa2_last_error());
  TORCH_CHECK(false, fa2_last_error());
}

int32_t int32_of(int64_t x, const char* name) {
  VALUE_CHECK(x >= INT32_MIN && x <= INT32_MAX, name, " must fit int32, got ", x);
  return static_cast<int32_t>(x);
}

// On a CUDA device, the call's when that is known.
void on_device(const Tensor& t, const char* name, const char* op, const Tensor* like = nullptr) {
  if (!t.is_cuda()) C10_THROW_ERROR(NotImplementedError, c10::str(op, ": no CPU implementation; ", name, " must be on a CUDA device"));
  VALUE_CHECK(t.layout() == c10::kStrided, op, ": ", name, " must be strided");
  if (like != nullptr) VALUE_CHECK(t.device() == like->device(), op, ": ", name, " must be on ", like->device(), ", is on ", t.device());
}

int dtype_code(const Tensor& t, const char* name) {
  const auto dt = t.scalar_type();
  TYPE_CHECK(dt == at::kHalf || dt == at::kBFloat16, name, " must be float16 or bfloat16, got ", dt);
  return dt == at::kBFloat16 ? FA2_BF16 : FA2_F16;
}

// These calls record no operations: a tracer would see constants, a transform's wrappers have no storage of their own, and
// forward-mode tangents would be lost.
void refuse_transforms(const char* op, std::initializer_list<const Tensor*> inputs) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), op, " cannot be traced");
  TORCH_CHECK(!c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode), op,
              " has no rules for function transforms");
  for (const Tensor* t : inputs)
    if (t->defined() && t->_fw_grad(0).defined()) C10_THROW_ERROR(NotImplementedError, c10::str(op, " has no jvp (forward-mode derivative)"));
}
void refuse_gradients(const char* op, std::initializer_list<const Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->defined() || !t->requires_grad(), op, " has no gradient: call it under torch.no_grad(), or detach its inputs");
}

// What a call has written to.
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A view whose last stride is 1, and no negative bit.
Tensor rows(Tensor t) {
  if (t.is_neg()) t = t.resolve_neg();
  return t.stride(-1) != 1 && t.size(-1) > 1 ? t.clone(at::MemoryFormat::Contiguous) : t;
}

// {batch, row, head} of [B, S, H, D], or of [T, H, D] as a batch of one; of a dimension of length 1 the stride is 0.
void strides_of(const Tensor& t, int64_t out[3]) {
  const int d = static_cast<int>(t.dim());
  out[0] = 0;
  for (int i = 0; i < d - 1; ++i) out[i + (d == 3)] = t.size(i) > 1 ? t.stride(i) : 0;
}

bool addressable(const Tensor& t) {
  if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && (t.stride(i) % 8 != 0 || t.stride(i) < 0)) return false;
  return t.stride(-1) == 1 || t.size(-1) == 1;
}

// ---------------------------------------------------------------- rotary positions
struct Turn {
  std::array<int32_t, 4> sections{};
  int axes = 0;
  int64_t pairs = 0;
  bool interleaved_axes = false, interleaved_pairs = false;
};

// The rotary part of a call: q and k (either may be undefined) are checked and laid out, q_out and k_out allocated where asked
// for. Returns whether there is anything to do. `k_out`: null where the keys go elsewhere.
bool turn_args(const char* op, Tensor& q, Tensor& k, Tensor& positions, Tensor& inv_freq, const Turn& turn, Tensor* q_out, Tensor* k_out,
               fa2_rotary_args& a) {
  Tensor& x = q.defined() ? q : k;
  for (auto [t, name] : {std::pair<Tensor*, const char*>{&q, "q"}, {&k, "k"}}) {
    if (!t->defined()) continue;
    on_device(*t, name, op, &x);
    dtype_code(*t, name);
    VALUE_CHECK(t->dim() == 3 || t->dim() == 4, op, ": ", name, " must be [B, S, H, D] or [T, H, D]");
    *t = rows(*t);
  }
  const int dt = dtype_code(x, "q");
  const auto last = x.dim() - 1;
  const int64_t batch = x.dim() == 4 ? x.size(0) : 1, seqlen = x.size(last - 2);
  if (q.defined() && k.defined()) {
    TYPE_CHECK(k.scalar_type() == q.scalar_type(), op, ": q and k must share dtype");
    VALUE_CHECK(k.dim() == q.dim() && k.size(last) == q.size(last) && k.sizes().slice(0, last - 1) == q.sizes().slice(0, last - 1), op,
                ": k must have q's tokens and head dim, got ", q.sizes(), " and ", k.sizes());
  }
  on_device(positions, "positions", op, &x);
  on_device(inv_freq, "inv_freq", op, &x);
  const auto pt = positions.scalar_type();
  TYPE_CHECK(pt == at::kInt || pt == at::kLong, op, ": positions must be int32 or int64, got ", pt);
  TYPE_CHECK(inv_freq.scalar_type() == at::kFloat, op, ": inv_freq must be float32");
  VALUE_CHECK(positions.dim() == x.dim() - 1 && positions.size(0) == turn.axes && positions.size(-1) == seqlen &&
                  (x.dim() == 3 || positions.size(1) == batch),
              op, ": positions must be [", turn.axes, x.dim() == 4 ? ", B, S" : ", T", "] for the tokens of q and k, got ", positions.sizes());
  VALUE_CHECK(inv_freq.dim() == 1 && inv_freq.size(0) == turn.pairs, op, ": inv_freq must have one frequency for each of the ", turn.pairs,
              " pairs of the sections, got ", inv_freq.sizes());
  inv_freq = inv_freq.contiguous();
  a.size = sizeof(a);
  a.dtype = dt;
  a.batch = int32_of(batch, "batch");
  a.seqlen = int32_of(seqlen, "seqlen");
  a.head_dim = int32_of(x.size(last), "head dim");
  a.axes = turn.axes;
  for (int i = 0; i < 4; ++i) a.sections[i] = turn.sections[i];
  a.interleaved_axes = turn.interleaved_axes;
  a.interleaved_pairs = turn.interleaved_pairs;
  a.positions = positions.data_ptr();
  a.position_bits = pt == at::kLong ? 64 : 32;
  a.position_stride[0] = positions.stride(0);
  a.position_stride[1] = x.dim() == 4 ? positions.stride(1) : 0;
  a.position_stride[2] = positions.stride(-1);
  a.inv_freq = static_cast<const float*>(inv_freq.data_ptr());
  if (q.defined()) {
    a.heads = int32_of(q.size(last - 1), "heads");
    *q_out = empty(q.sizes(), q.scalar_type(), q.device());
    a.q = q.data_ptr();
    a.q_out = q_out->data_ptr();
    strides_of(q, a.q_stride);
    strides_of(*q_out, a.q_out_stride);
  }
  if (k.defined()) {
    a.heads_k = int32_of(k.size(last - 1), "heads");
    a.k = k.data_ptr();
    strides_of(k, a.k_stride);
    if (k_out != nullptr) {
      *k_out = empty(k.sizes(), k.scalar_type(), k.device());
      a.k_out = k_out->data_ptr();
      strides_of(*k_out, a.k_out_stride);
    }
  }
  return x.numel() > 0;
}

std::optional<Tensor> some(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

class RotaryAxes : public torch::autograd::Function<RotaryAxes> {
 public:
  // Outputs: those of q and of k that there are. (An input that is not there has to be an empty optional here.)
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const std::optional<Tensor>& q_in,
                                                const std::optional<Tensor>& k_in, Tensor positions, Tensor inv_freq, const Turn& turn, bool inverse) {
    Tensor q = q_in.value_or(Tensor()), k = k_in.value_or(Tensor()), q_out, k_out;
    {
      const c10::cuda::CUDAGuard guard((q.defined() ? q : k).device());
      fa2_rotary_args a{};
      const bool any = turn_args("rotary_axes_func", q, k, positions, inv_freq, turn, &q_out, &k_out, a);
      a.inverse = inverse;
      // An empty call launches nothing, but its other arguments are checked.
      if (!any) a.q = a.k = nullptr;
      check(fa2_rotary(&a, c10::cuda::getCurrentCUDAStream(guard.current_device().index()).stream()));
    }
    if (ctx != nullptr) {
      ctx->save_for_backward({positions, inv_freq});
      std::vector<int64_t> d(turn.sections.begin(), turn.sections.begin() + turn.axes);
      d.insert(d.end(), {turn.interleaved_axes, turn.interleaved_pairs, inverse, q.defined(), k.defined()});
      ctx->saved_data["turn"] = std::move(d);
    }
    torch::autograd::variable_list out;
    if (q_out.defined()) out.push_back(q_out);
    if (k_out.defined()) out.push_back(k_out);
    return out;
  }
  // The turn back, which is this function again: it has gradients of its own.
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto d = ctx->saved_data["turn"].toIntVector();
    Turn turn;
    turn.axes = static_cast<int>(d.size()) - 5;
    for (int i = 0; i < turn.axes; ++i) turn.pairs += turn.sections[i] = static_cast<int32_t>(d[i]);
    const int64_t* rest = d.data() + turn.axes;
    turn.interleaved_axes = rest[0];
    turn.interleaved_pairs = rest[1];
    const bool inverse = rest[2], has_q = rest[3], has_k = rest[4];
    Tensor dq, dk;
    if (has_q && ctx->needs_input_grad(0)) dq = grads[0];
    if (has_k && ctx->needs_input_grad(has_q)) dk = grads[has_q];
    torch::autograd::variable_list result(6);
    if (!dq.defined() && !dk.defined()) return result;
    auto turned = at::GradMode::is_enabled() ? apply(some(dq), some(dk), saved[0], saved[1], turn, !inverse)
                                             : forward(nullptr, some(dq), some(dk), saved[0], saved[1], turn, !inverse);
    if (dq.defined()) result[0] = turned.front();
    if (dk.defined()) result[1] = turned.back();
    return result;
  }
};

// ---------------------------------------------------------------- the cache
int32_t* int_rows(const Tensor& t, const char* name, const char* op, const Tensor& like) {
  on_device(t, name, op, &like);
  TYPE_CHECK(t.scalar_type() == at::kInt, op, ": ", name, " must be int32");
  return static_cast<int32_t*>(t.data_ptr());
}

void vector_arg(const Tensor& t, int64_t n, const char* name, const char* op) {
  VALUE_CHECK(t.dim() == 1 && t.size(0) == n && t.is_contiguous(), op, ": ", name, " must be a contiguous vector of ", n, " entries, got ", t.sizes());
}

void table_arg(const Tensor& t, const char* name, const char* op) {
  VALUE_CHECK(t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1), op, ": ", name, " must be [B, pages] with unit last stride, got ", t.sizes());
  VALUE_CHECK(t.size(1) > 0, op, ": ", name, " must have room for a page");
}

void cache_args(const char* op, const Tensor& k, const Tensor& v, const Tensor& mass, const Tensor& table, const Tensor& seqlens,
                fa2_paged_cache& c) {
  on_device(k, "k_cache", op);
  on_device(v, "v_cache", op, &k);
  VALUE_CHECK(k.dim() == 4 && v.sizes() == k.sizes(), op, ": k_cache and v_cache must both be [pages, page_size, Hk, D], got ", k.sizes(), " and ",
              v.sizes());
  c.size = sizeof(c);
  c.dtype = dtype_code(k, "k_cache");
  TYPE_CHECK(v.scalar_type() == k.scalar_type(), op, ": k_cache and v_cache must share dtype");
  VALUE_CHECK(k.numel() > 0, op, ": the cache is empty");
  VALUE_CHECK((k.stride(3) == 1 || k.size(3) == 1) && (v.stride(3) == 1 || v.size(3) == 1) && !k.is_neg() && !v.is_neg(), op,
              ": k_cache and v_cache must have unit last stride");
  c.block_table = int_rows(table, "block_table", op, k);
  table_arg(table, "block_table", op);
  c.block_table_stride = table.stride(0);
  c.seqlens_k = int_rows(seqlens, "seqlens_k", op, k);
  vector_arg(seqlens, table.size(0), "seqlens_k", op);
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  strides_of(k, c.k_stride);
  strides_of(v, c.v_stride);
  c.num_pages = int32_of(k.size(0), "pages");
  c.page_size = int32_of(k.size(1), "page_size");
  c.max_pages = int32_of(table.size(1), "pages of a sequence");
  c.batch = int32_of(table.size(0), "batch");
  c.heads_k = int32_of(k.size(2), "heads");
  c.head_dim = int32_of(k.size(3), "head dim");
  if (mass.defined()) {
    on_device(mass, "attn_mass", op, &k);
    TYPE_CHECK(mass.scalar_type() == at::kFloat, op, ": attn_mass must be float32");
    VALUE_CHECK(mass.dim() == 3 && mass.size(0) == k.size(0) && mass.size(1) == k.size(2) && mass.size(2) == k.size(1) && mass.is_contiguous(), op,
                ": attn_mass must be contiguous [pages, Hk, page_size], got ", mass.sizes());
    c.attn_mass = static_cast<float*>(mass.data_ptr());
  }
}

// Two elements of what is written must not share an address.
void check_written(const Tensor& t, const char* name, const char* op) {
  VALUE_CHECK(at::has_internal_overlap(t) != at::MemOverlap::Yes, op, ": elements of ", name, " share addresses");
}

Tensor append(Tensor q, Tensor k, Tensor v, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& seqlens, Tensor positions,
              Tensor inv_freq, const Turn& turn, const Tensor& cu_seqlens, const Tensor& seqlens_new, const Tensor& mass) {
  const char* op = "paged_append";
  refuse_transforms(op, {&q, &k, &v, &k_cache, &v_cache, &mass});
  refuse_gradients(op, {&q, &k, &v, &k_cache, &v_cache, &mass});
  fa2_paged_cache c{};
  cache_args(op, k_cache, v_cache, mass, table, seqlens, c);
  check_written(k_cache, "k_cache", op);
  check_written(v_cache, "v_cache", op);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  on_device(k, "k", op, &k_cache);
  on_device(v, "v", op, &k_cache);
  if (q.defined()) on_device(q, "q", op, &k_cache);
  TYPE_CHECK(v.scalar_type() == k.scalar_type() && k.scalar_type() == k_cache.scalar_type(), op, ": k, v and the cache must share dtype");
  VALUE_CHECK(v.sizes() == k.sizes(), op, ": v must have k's shape, got ", k.sizes(), " and ", v.sizes());
  fa2_rotary_args a{};
  Tensor q_out;
  // Tokens that lie in the pools themselves: a row may be written before it has been read.
  for (Tensor* t : {&q, &k, &v})
    for (const Tensor* pool : {&k_cache, &v_cache})
      if (t->defined() && t->is_alias_of(*pool) && at::get_overlap_status(*t, *pool) != at::MemOverlapStatus::No) {
        *t = t->clone(at::MemoryFormat::Contiguous);
        break;
      }
  const bool any = turn_args(op, q, k, positions, inv_freq, turn, &q_out, nullptr, a);
  v = rows(v);
  VALUE_CHECK(a.heads_k == c.heads_k && a.head_dim == c.head_dim, op, ": k must have the cache's heads and head dim, got ", k.sizes(), " and ",
              k_cache.sizes());
  fa2_paged_append_args p{};
  p.size = sizeof(p);
  if (k.dim() == 3) {
    VALUE_CHECK(cu_seqlens.defined() && !seqlens_new.defined(), op, ": packed tokens [T, H, D] need cu_seqlens, and take no seqlens_new");
    p.cu_seqlens = int_rows(cu_seqlens, "cu_seqlens", op, k);
    vector_arg(cu_seqlens, table.size(0) + 1, "cu_seqlens", op);
  } else {
    VALUE_CHECK(!cu_seqlens.defined(), op, ": cu_seqlens is for packed tokens [T, H, D]");
    VALUE_CHECK(k.size(0) == table.size(0), op, ": the new tokens must have the block table's batch, got ", k.size(0), " and ", table.size(0));
    if (seqlens_new.defined()) {
      p.seqlens_new = int_rows(seqlens_new, "seqlens_new", op, k);
      vector_arg(seqlens_new, table.size(0), "seqlens_new", op);
    }
  }
  if (!any || table.size(0) == 0) return q_out;
  p.turn = &a;
  p.cache = &c;
  p.v = v.data_ptr();
  strides_of(v, p.v_stride);
  check(fa2_paged_append(&p, c10::cuda::getCurrentCUDAStream(guard.current_device().index()).stream()));
  written(k_cache);
  written(v_cache);
  if (mass.defined()) written(mass);
  return q_out;
}

std::pair<Tensor, Tensor> fwd(Tensor q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& table, const Tensor& seqlens, Tensor out,
                              const Tensor& mass, std::optional<double> scale, int64_t window, double softcap, std::optional<int64_t> max_seqlen_k) {
  const char* op = "paged_fwd";
  refuse_transforms(op, {&q, &k_cache, &v_cache, &mass, &out});
  refuse_gradients(op, {&q, &k_cache, &v_cache, &mass, &out});
  fa2_paged_cache c{};
  cache_args(op, k_cache, v_cache, mass, table, seqlens, c);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  on_device(q, "q", op, &k_cache);
  TYPE_CHECK(q.scalar_type() == k_cache.scalar_type(), op, ": q and the cache must share dtype");
  VALUE_CHECK(q.dim() == 4 && q.size(0) == table.size(0) && q.size(3) == k_cache.size(3), op,
              ": q must be [B, Sq, H, D] with the block table's batch and the cache's head dim, got ", q.sizes());
  if (out.defined()) {
    on_device(out, "out", op, &k_cache);
    VALUE_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && !out.is_neg(), op, ": out must match q's shape and dtype");
    check_written(out, "out", op);
  }
  if (q.is_neg()) q = q.resolve_neg();
  if (!addressable(q)) q = q.clone(at::MemoryFormat::Contiguous);
  // An output that the kernel cannot write, or that shares memory with what it reads, is computed aside.
  bool aside = !out.defined() || !addressable(out);
  if (!aside)
    for (const Tensor* t : std::initializer_list<const Tensor*>{&q, &k_cache, &v_cache, &table, &seqlens, &mass})
      aside = aside || (t->defined() && at::get_overlap_status(out, *t) != at::MemOverlapStatus::No);
  Tensor to = aside ? empty(q.sizes(), q.scalar_type(), q.device()) : out;
  Tensor lse = empty({q.size(0), q.size(2), q.size(1)}, at::kFloat, q.device());
  if (q.numel() > 0) {
    fa2_paged_fwd_args a{};
    a.size = sizeof(a);
    a.cache = &c;
    a.q = q.data_ptr();
    a.out = to.data_ptr();
    a.lse = static_cast<float*>(lse.data_ptr());
    strides_of(q, a.q_stride);
    strides_of(to, a.o_stride);
    a.seqlen_q = int32_of(q.size(1), "seqlen_q");
    a.heads = int32_of(q.size(2), "heads");
    a.softmax_scale = static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(q.size(3))));
    a.window_left = int32_of(window, "window_size_left");
    a.softcap = static_cast<float>(softcap);
    if (max_seqlen_k) {
      VALUE_CHECK(*max_seqlen_k > 0, op, ": max_seqlen_k must be positive, got ", *max_seqlen_k);
      a.max_seqlen_k = int32_of(*max_seqlen_k, "max_seqlen_k");
    }
    const int64_t need = fa2_paged_fwd_workspace_bytes(&a);
    const Tensor workspace = empty({need}, at::kByte, q.device());
    check(fa2_paged_fwd(&a, workspace.data_ptr(), need, c10::cuda::getCurrentCUDAStream(guard.current_device().index()).stream()));
    if (mass.defined()) written(mass);
  }
  if (out.defined()) {
    if (aside) out.copy_(to);
    else written(out);
    to = out;
  }
  return {to, lse};
}

std::pair<Tensor, Tensor> evict(const Tensor& k_cache, const Tensor& v_cache, const Tensor& mass, const Tensor& table, const Tensor& seqlens,
                                const Tensor& dst_table, int64_t budget, int64_t recent) {
  const char* op = "paged_evict";
  refuse_transforms(op, {&k_cache, &v_cache, &mass});
  refuse_gradients(op, {&k_cache, &v_cache, &mass});
  fa2_paged_cache c{};
  cache_args(op, k_cache, v_cache, mass, table, seqlens, c);
  check_written(k_cache, "k_cache", op);
  check_written(v_cache, "v_cache", op);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  fa2_paged_evict_args a{};
  a.size = sizeof(a);
  a.cache = &c;
  a.dst_block_table = int_rows(dst_table, "dst_block_table", op, k_cache);
  table_arg(dst_table, "dst_block_table", op);
  VALUE_CHECK(dst_table.size(0) == table.size(0), op, ": dst_block_table must have block_table's batch");
  a.dst_block_table_stride = dst_table.stride(0);
  a.dst_max_pages = int32_of(dst_table.size(1), "pages of a sequence");
  a.budget = int32_of(budget, "budget");
  a.recent = int32_of(recent, "recent");
  VALUE_CHECK(a.budget > 0 && a.recent >= 0 && a.recent <= a.budget, op, ": budget must be positive and recent in 0..=budget, got ", budget, " and ",
              recent);
  Tensor seqlens_out = empty({table.size(0)}, at::kInt, k_cache.device());
  Tensor kept = empty({table.size(0), k_cache.size(2), budget}, at::kInt, k_cache.device());
  if (table.size(0) == 0) return {seqlens_out, kept};
  a.seqlens_out = static_cast<int32_t*>(seqlens_out.data_ptr());
  a.kept = static_cast<int32_t*>(kept.data_ptr());
  check(fa2_paged_evict(&a, c10::cuda::getCurrentCUDAStream(guard.current_device().index()).stream()));
  written(k_cache);
  written(v_cache);
  written(mass);
  return {seqlens_out, kept};
}

// ---------------------------------------------------------------- Python arguments
Tensor tensor_arg(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return Tensor();
  TYPE_CHECK(THPVariable_CheckExact(o), name, " must be a torch.Tensor, got ", Py_TYPE(o)->tp_name);
  return THPVariable_Unpack(o);
}
int64_t int_arg(PyObject* o, const char* name) {
  TYPE_CHECK(PyIndex_Check(o) && !PyBool_Check(o), name, " must be an int, got ", Py_TYPE(o)->tp_name);
  const Py_ssize_t x = PyNumber_AsSsize_t(o, PyExc_ValueError);
  if (x == -1 && PyErr_Occurred()) throw python_error();
  return x;
}
double float_arg(PyObject* o, const char* name) {
  TYPE_CHECK((PyFloat_Check(o) || PyLong_Check(o)) && !PyBool_Check(o), name, " must be a float, got ", Py_TYPE(o)->tp_name);
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw python_error();
  return x;
}
bool bool_arg(PyObject* o, const char* name) {
  TYPE_CHECK(PyBool_Check(o), name, " must be a bool, got ", Py_TYPE(o)->tp_name);
  return o == Py_True;
}
// sections, interleaved_axes, interleaved_pairs
Turn turn_arg(PyObject* const* a) {
  Turn t;
  TYPE_CHECK(PyTuple_Check(a[0]) || PyList_Check(a[0]), "sections must be a tuple of ints, got ", Py_TYPE(a[0])->tp_name);
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(a[0]);
  VALUE_CHECK(n >= 1 && n <= 4, "sections must name 1 to 4 axes, got ", n);
  t.axes = static_cast<int>(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const int64_t s = int_arg(PySequence_Fast_GET_ITEM(a[0], i), "sections");
    VALUE_CHECK(s >= 0 && s <= 128, "a section must have 0 to 128 pairs, got ", s);
    t.sections[i] = static_cast<int32_t>(s);
    t.pairs += s;
  }
  t.interleaved_axes = bool_arg(a[1], "interleaved_axes");
  t.interleaved_pairs = bool_arg(a[2], "interleaved_pairs");
  return t;
}

// Allocations and launches can block: other Python threads run meanwhile.
struct WithoutPython {
  PyThreadState* const state = PyEval_SaveThread();
  ~WithoutPython() { PyEval_RestoreThread(state); }
};

PyObject* object(const Tensor& t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject* pair_of(const Tensor& a, const Tensor& b) {
  PyObject* t = PyTuple_New(2);
  if (t == nullptr) return nullptr;
  PyTuple_SET_ITEM(t, 0, object(a));
  PyTuple_SET_ITEM(t, 1, object(b));
  return t;
}
void count(Py_ssize_t n, Py_ssize_t wanted) { TYPE_CHECK(n == wanted, "expected ", wanted, " arguments, got ", n); }

// rotary(q, k, positions, inv_freq, sections, interleaved_axes, interleaved_pairs) -> (q_out, k_out)
PyObject* py_rotary(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  const Tensor q = tensor_arg(args[0], "q", true), k = tensor_arg(args[1], "k", true);
  const Tensor positions = tensor_arg(args[2], "positions"), inv_freq = tensor_arg(args[3], "inv_freq");
  const Turn turn = turn_arg(args + 4);
  VALUE_CHECK(q.defined() || k.defined(), "rotary_axes_func: q and k are both None");
  for (const Tensor* t : {&q, &k})
    if (t->defined()) on_device(*t, "q and k", "rotary_axes_func");
  refuse_transforms("rotary_axes_func", {&q, &k, &inv_freq});
  if (at::GradMode::is_enabled()) TORCH_CHECK(!inv_freq.requires_grad(), "rotary_axes_func has no gradient for inv_freq: detach it");
  torch::autograd::variable_list out;
  {
    const WithoutPython unlocked;
    if (at::GradMode::is_enabled() && ((q.defined() && q.requires_grad()) || (k.defined() && k.requires_grad())))
      out = RotaryAxes::apply(some(q), some(k), positions, inv_freq, turn, false);
    else
      out = RotaryAxes::forward(nullptr, some(q), some(k), positions, inv_freq, turn, false);
  }
  return pair_of(q.defined() ? out.front() : Tensor(), k.defined() ? out.back() : Tensor());
  END_HANDLE_TH_ERRORS
}

// append(q, k, v, k_cache, v_cache, block_table, seqlens_k, positions, inv_freq, sections, interleaved_axes, interleaved_pairs,
// cu_seqlens, seqlens_new, attn_mass) -> q_out
PyObject* py_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 15);
  const Tensor q = tensor_arg(args[0], "q", true), k = tensor_arg(args[1], "k"), v = tensor_arg(args[2], "v");
  const Tensor k_cache = tensor_arg(args[3], "k_cache"), v_cache = tensor_arg(args[4], "v_cache");
  const Tensor table = tensor_arg(args[5], "block_table"), seqlens = tensor_arg(args[6], "seqlens_k");
  const Tensor positions = tensor_arg(args[7], "positions"), inv_freq = tensor_arg(args[8], "inv_freq");
  const Turn turn = turn_arg(args + 9);
  const Tensor cu = tensor_arg(args[12], "cu_seqlens", true), fresh = tensor_arg(args[13], "seqlens_new", true);
  const Tensor mass = tensor_arg(args[14], "attn_mass", true);
  Tensor out;
  {
    const WithoutPython unlocked;
    out = append(q, k, v, k_cache, v_cache, table, seqlens, positions, inv_freq, turn, cu, fresh, mass);
  }
  return object(out);
  END_HANDLE_TH_ERRORS
}

// fwd(q, k_cache, v_cache, block_table, seqlens_k, out, attn_mass, softmax_scale, window_size_left, softcap, max_seqlen_k) -> (out, lse)
PyObject* py_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 11);
  const Tensor q = tensor_arg(args[0], "q"), k_cache = tensor_arg(args[1], "k_cache"), v_cache = tensor_arg(args[2], "v_cache");
  const Tensor table = tensor_arg(args[3], "block_table"), seqlens = tensor_arg(args[4], "seqlens_k");
  const Tensor out = tensor_arg(args[5], "out", true), mass = tensor_arg(args[6], "attn_mass", true);
  std::optional<double> scale;
  if (args[7] != Py_None) scale = float_arg(args[7], "softmax_scale");
  const int64_t window = int_arg(args[8], "window_size_left");
  const double softcap = float_arg(args[9], "softcap");
  std::optional<int64_t> most;
  if (args[10] != Py_None) most = int_arg(args[10], "max_seqlen_k");
  std::pair<Tensor, Tensor> r;
  {
    const WithoutPython unlocked;
    r = fwd(q, k_cache, v_cache, table, seqlens, out, mass, scale, window, softcap, most);
  }
  return pair_of(r.first, r.second);
  END_HANDLE_TH_ERRORS
}

// evict(k_cache, v_cache, attn_mass, block_table, seqlens_k, dst_block_table, budget, recent) -> (seqlens, kept)
PyObject* py_evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 8);
  const Tensor k_cache = tensor_arg(args[0], "k_cache"), v_cache = tensor_arg(args[1], "v_cache"), mass = tensor_arg(args[2], "attn_mass");
  const Tensor table = tensor_arg(args[3], "block_table"), seqlens = tensor_arg(args[4], "seqlens_k"), to = tensor_arg(args[5], "dst_block_table");
  const int64_t budget = int_arg(args[6], "budget"), recent = int_arg(args[7], "recent");
  std::pair<Tensor, Tensor> r;
  {
    const WithoutPython unlocked;
    r = evict(k_cache, v_cache, mass, table, seqlens, to, budget, recent);
  }
  return pair_of(r.first, r.second);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"rotary", castPyCFunctionFast(py_rotary), METH_FASTCALL, nullptr},
    {"append", castPyCFunctionFast(py_append), METH_FASTCALL, nullptr},
    {"fwd", castPyCFunctionFast(py_fwd), METH_FASTCALL, nullptr},
    {"evict", castPyCFunctionFast(py_evict), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fa2_paged", "Operators on a paged K/V cache, on torch tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fa2_paged() { return PyModule_Create(&module); }
