// Binding of the decode-step operators for torch tensors: checks arguments, takes the current stream of
// the tensors' device, allocates outputs and scratch from torch's allocator and calls the C ABI.
//
// The other operators go through ctypes, where checking eight tensors in Python and converting twenty
// arguments takes 10 us and more.  A decode step's kernels take 3 to 10 us, so that these calls would be
// bound by the host; the same work takes about 1 us here.  Nothing is computed in this file.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <cstdio>
#include <stdexcept>

#include "../../include/b200moe.h"

namespace {

using at::Tensor;

[[noreturn]] void refuse(const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof(text), fmt, ap);
  va_end(ap);
  throw std::runtime_error(text);
}

void check_status(int rc, const char* name) {
  if (rc != B200MOE_OK) refuse("%s: %s (status %d)", name, b200moe_last_error(), rc);
}

// The arguments of one call, by position.
struct Args {
  const char* name;
  PyObject* const* v;

  const Tensor& tensor(int i, const char* what) const {
    if (!THPVariable_Check(v[i])) refuse("%s: %s must be a tensor, got %s", name, what, Py_TYPE(v[i])->tp_name);
    return THPVariable_Unpack(v[i]);
  }
  int64_t integer(int i, const char* what, int64_t lo, int64_t hi) const {
    const int64_t n = PyLong_AsLongLong(v[i]);
    if (n == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      refuse("%s: %s must be an integer", name, what);
    }
    if (n < lo || n > hi) refuse("%s: %s=%lld is out of range", name, what, static_cast<long long>(n));
    return n;
  }
  double number(int i, const char* what) const {
    const double x = PyFloat_AsDouble(v[i]);
    if (x == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      refuse("%s: %s must be a number", name, what);
    }
    return x;
  }
};

constexpr int64_t kInt = 0x7fffffff;

void on_cuda(const char* name, const char* what, const Tensor& t) {
  if (!t.is_cuda()) refuse("%s: %s must be on a CUDA device; there is no CPU implementation", name, what);
}
void on_device(const char* name, const char* what, const Tensor& t, const Tensor& like) {
  on_cuda(name, what, t);
  if (t.get_device() != like.get_device())
    refuse("%s: tensors are on different devices (%s on cuda:%d, others on cuda:%d)", name, what,
           static_cast<int>(t.get_device()), static_cast<int>(like.get_device()));
}
void contiguous(const char* name, const char* what, const Tensor& t) {
  if (!t.is_contiguous()) refuse("%s: %s must be contiguous", name, what);
}
void of_type(const char* name, const char* what, const Tensor& t, at::ScalarType type) {
  if (t.scalar_type() != type)
    refuse("%s: %s must be %s, got %s", name, what, c10::toString(type), c10::toString(t.scalar_type()));
}
// A contiguous tensor of `type` on the device of `like`.
void plain(const char* name, const char* what, const Tensor& t, const Tensor& like, at::ScalarType type) {
  on_device(name, what, t, like);
  of_type(name, what, t, type);
  contiguous(name, what, t);
}

int float_tag(const char* name, const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return B200MOE_F32;
    case at::kHalf: return B200MOE_F16;
    case at::kBFloat16: return B200MOE_BF16;
    default: refuse("%s: unsupported dtype %s", name, c10::toString(t.scalar_type()));
  }
}

const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }
int32_t* i32_out(const Tensor& t) { return static_cast<int32_t*>(t.mutable_data_ptr()); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Row stride of a two-dimensional table whose rows are contiguous.
int64_t table_stride(const char* name, const Tensor& t) {
  const int64_t width = t.size(1);
  if (width > 1 && t.stride(1) != 1) refuse("%s: the entries of a block_table row must be contiguous", name);
  return t.size(0) > 1 ? t.stride(0) : width;
}

// Caches and scales of the 8-bit paged cache.
struct Codes {
  const Tensor &k, &v, &ks, &vs;
  int64_t blocks, block_size, heads, dim;

  Codes(const char* name, const Tensor& k_, const Tensor& v_, const Tensor& ks_, const Tensor& vs_)
      : k(k_), v(v_), ks(ks_), vs(vs_) {
    on_cuda(name, "K_cache", k);
    if (k.dim() != 4 || v.sizes() != k.sizes())
      refuse("%s: caches must both be [blocks, block_size, kv_heads, head_dim]", name);
    plain(name, "K_cache", k, k, at::kFloat8_e4m3fn);
    plain(name, "V_cache", v, k, at::kFloat8_e4m3fn);
    plain(name, "K_scale", ks, k, at::kFloat);
    plain(name, "V_scale", vs, k, at::kFloat);
    blocks = k.size(0); block_size = k.size(1); heads = k.size(2); dim = k.size(3);
    for (const Tensor* s : {&ks, &vs})
      if (s->dim() != 2 || s->size(0) != blocks || s->size(1) != heads)
        refuse("%s: scales must be float32 [blocks, kv_heads] = [%lld, %lld]", name, (long long)blocks, (long long)heads);
    if (block_size > kInt || heads > kInt || dim > kInt) refuse("%s: caches are too large", name);
  }
};

// Rows [n, heads, dim] whose heads are contiguous; returns the row stride in elements.
int64_t row_stride(const char* name, const char* what, const Tensor& t) {
  const int64_t n = t.size(0), heads = t.size(1), dim = t.size(2);
  if ((dim > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != dim))
    refuse("%s: the heads of a row of %s must be contiguous", name, what);
  return n > 1 ? t.stride(0) : heads * dim;
}

void paged_schedule(const Args& a) {
  const char* name = a.name;
  const Tensor& ctx = a.tensor(0, "context_lens");
  const Tensor& fresh = a.tensor(1, "new_lens");
  const Tensor& table = a.tensor(2, "block_table");
  const Tensor& stack = a.tensor(3, "free_blocks");
  const Tensor& count = a.tensor(4, "free_count");
  const int64_t block_size = a.integer(5, "block_size", 1, kInt);
  const Tensor& seq = a.tensor(6, "seq_lens");
  const Tensor& cu = a.tensor(7, "cu_seqlens");
  const Tensor& slots = a.tensor(8, "slot_mapping");
  const Tensor* positions = a.v[9] == Py_None ? nullptr : &a.tensor(9, "positions");
  const Tensor& count_out = a.tensor(10, "free_count_out");
  const Tensor& refused = a.tensor(11, "num_refused");
  on_cuda(name, "context_lens", ctx);
  plain(name, "context_lens", ctx, ctx, at::kInt);
  plain(name, "new_lens", fresh, ctx, at::kInt);
  on_device(name, "block_table", table, ctx);
  of_type(name, "block_table", table, at::kInt);
  plain(name, "free_blocks", stack, ctx, at::kInt);
  plain(name, "free_count", count, ctx, at::kInt);
  plain(name, "seq_lens", seq, ctx, at::kInt);
  plain(name, "cu_seqlens", cu, ctx, at::kInt);
  plain(name, "slot_mapping", slots, ctx, at::kInt);
  plain(name, "free_count_out", count_out, ctx, at::kInt);
  plain(name, "num_refused", refused, ctx, at::kInt);
  if (table.dim() != 2) refuse("%s: block_table must be [requests, max_blocks]", name);
  const int64_t requests = table.size(0), width = table.size(1), rows = slots.numel();
  if (ctx.numel() != requests || fresh.numel() != requests || seq.numel() != requests || cu.numel() != requests + 1)
    refuse("%s: context_lens, new_lens and seq_lens must hold %lld elements and cu_seqlens one more", name,
           (long long)requests);
  if (count.numel() != 1 || count_out.numel() != 1 || refused.numel() != 1)
    refuse("%s: free_count, free_count_out and num_refused hold one element", name);
  if (positions) {
    plain(name, "positions", *positions, ctx, at::kLong);
    if (positions->numel() != rows) refuse("%s: positions must have one entry per row of slot_mapping", name);
  }
  const c10::cuda::CUDAGuard guard(ctx.device());
  check_status(b200moe_paged_schedule(
      i32(ctx), i32(fresh), i32_out(table), i32_out(stack), i32(count), requests, width, table_stride(name, table),
      static_cast<int>(block_size), stack.numel(), rows, i32_out(seq), i32_out(cu), i32_out(slots),
      positions ? static_cast<int64_t*>(positions->mutable_data_ptr()) : nullptr, i32_out(count_out), i32_out(refused),
      stream_of(ctx)), name);
}

void paged_store_kvcache_fp8(const Args& a) {
  const char* name = a.name;
  const Tensor& key = a.tensor(0, "K");
  const Tensor& value = a.tensor(1, "V");
  const Codes c(name, a.tensor(2, "K_cache"), a.tensor(3, "V_cache"), a.tensor(4, "K_scale"), a.tensor(5, "V_scale"));
  const Tensor& slots = a.tensor(6, "slot_mapping");
  if (key.dim() != 3 || value.sizes() != key.sizes() || key.size(1) != c.heads || key.size(2) != c.dim)
    refuse("%s: K and V must both be [tokens, %lld, %lld]", name, (long long)c.heads, (long long)c.dim);
  on_device(name, "K", key, c.k);
  on_device(name, "V", value, c.k);
  if (key.scalar_type() != value.scalar_type()) refuse("%s: K and V must share a dtype", name);
  plain(name, "slot_mapping", slots, c.k, at::kInt);
  if (slots.numel() != key.size(0)) refuse("%s: slot_mapping must have one entry per token", name);
  const c10::cuda::CUDAGuard guard(c.k.device());
  check_status(b200moe_paged_store_kvcache_fp8(
      key.const_data_ptr(), value.const_data_ptr(), c.k.mutable_data_ptr(), c.v.mutable_data_ptr(),
      static_cast<float*>(c.ks.mutable_data_ptr()), static_cast<float*>(c.vs.mutable_data_ptr()), i32(slots),
      float_tag(name, key), key.size(0), static_cast<int>(c.heads), static_cast<int>(c.dim),
      row_stride(name, "K", key), row_stride(name, "V", value), c.blocks, static_cast<int>(c.block_size),
      stream_of(c.k)), name);
}

Tensor paged_attn_varlen_fp8(const Args& a) {
  const char* name = a.name;
  const Tensor& q = a.tensor(0, "Q");
  const Codes c(name, a.tensor(1, "K_cache"), a.tensor(2, "V_cache"), a.tensor(3, "K_scale"), a.tensor(4, "V_scale"));
  const int64_t max_len = a.integer(5, "max_seqlen_k", -kInt, INT64_MAX);
  const Tensor& lens = a.tensor(6, "context_lens");
  const Tensor& table = a.tensor(7, "block_table");
  const double scale = a.number(8, "softmax_scale");
  int64_t splits = a.integer(9, "num_splits", -kInt, kInt);
  on_device(name, "Q", q, c.k);
  if (q.dim() != 3 || q.size(2) != c.dim) refuse("%s: Q must be [batch, heads, %lld]", name, (long long)c.dim);
  const int64_t batch = q.size(0), heads = q.size(1);
  plain(name, "context_lens", lens, c.k, at::kInt);
  on_device(name, "block_table", table, c.k);
  of_type(name, "block_table", table, at::kInt);
  if (table.dim() != 2 || table.size(0) != batch || lens.numel() != batch)
    refuse("%s: block_table must be [batch, max_blocks] and context_lens [batch]", name);
  const int64_t width = table.size(1);
  if (batch > kInt || heads > kInt || width > kInt) refuse("%s: tensors are too large", name);
  const int tag = float_tag(name, q);
  const int64_t q_stride = row_stride(name, "Q", q), t_stride = table_stride(name, table);
  const c10::cuda::CUDAGuard guard(c.k.device());
  if (splits <= 0) {
    int64_t longest = width * c.block_size;
    if (max_len > 0 && max_len < longest) longest = max_len;
    splits = b200moe_paged_attn_fp8_num_splits(static_cast<int>(batch), static_cast<int>(heads),
                                               static_cast<int>(c.heads), longest);
  }
  Tensor out = at::empty({batch, heads, c.dim}, q.options());
  const size_t bytes = b200moe_paged_attn_fp8_workspace_bytes(static_cast<int>(batch), static_cast<int>(heads),
                                                              static_cast<int>(c.heads), static_cast<int>(splits));
  Tensor ws;
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  check_status(b200moe_paged_attn_varlen_fp8(
      q.const_data_ptr(), c.k.const_data_ptr(), c.v.const_data_ptr(), static_cast<const float*>(c.ks.const_data_ptr()),
      static_cast<const float*>(c.vs.const_data_ptr()), out.mutable_data_ptr(), i32(table), i32(lens), tag,
      static_cast<int>(batch), static_cast<int>(heads), static_cast<int>(c.heads), static_cast<int>(c.dim), q_stride,
      c.blocks, static_cast<int>(c.block_size), static_cast<int>(width), t_stride, static_cast<float>(scale),
      static_cast<int>(splits), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream_of(c.k)), name);
  return out;
}

void moe_few_tokens(const Args& a) {
  const char* name = a.name;
  const Tensor& out = a.tensor(0, "output");
  const Tensor& x = a.tensor(1, "hidden_states");
  const Tensor& logits = a.tensor(2, "gating_output");
  const Tensor& w13 = a.tensor(3, "w13");
  const Tensor& w2 = a.tensor(4, "w2");
  const int64_t renormalize = a.integer(5, "renormalize", 0, 1);
  on_cuda(name, "hidden_states", x);
  plain(name, "hidden_states", x, x, at::kBFloat16);
  plain(name, "output", out, x, at::kBFloat16);
  plain(name, "w13", w13, x, at::kBFloat16);
  plain(name, "w2", w2, x, at::kBFloat16);
  on_device(name, "gating_output", logits, x);
  contiguous(name, "gating_output", logits);
  const int tag = float_tag(name, logits);
  if (x.dim() != 2 || w13.dim() != 3 || w2.dim() != 3 || logits.dim() != 2)
    refuse("%s: expected hidden_states [T, H], gating_output [T, E], w13 [E, 2 * I, H] and w2 [E, H, I]", name);
  const int64_t tokens = x.size(0), hidden = x.size(1), experts = w13.size(0), inter = w2.size(2);
  if (out.sizes() != x.sizes() || logits.size(0) != tokens || logits.size(1) != experts || w13.size(1) != 2 * inter ||
      w13.size(2) != hidden || w2.size(0) != experts || w2.size(1) != hidden || experts > kInt)
    refuse("%s: shapes of output, hidden_states, gating_output, w13 and w2 do not match", name);
  const c10::cuda::CUDAGuard guard(x.device());
  const size_t bytes = b200moe_few_tokens_workspace_bytes(tokens, inter);
  Tensor ws;
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
  check_status(b200moe_few_tokens(x.const_data_ptr(), logits.const_data_ptr(), tag, w13.const_data_ptr(),
                                  w2.const_data_ptr(), out.mutable_data_ptr(), tokens, static_cast<int>(experts), 2, hidden,
                                  inter, static_cast<int>(renormalize), bytes ? ws.mutable_data_ptr() : nullptr, bytes,
                                  stream_of(x)), name);
}

PyObject* wrap(Tensor t) { return THPVariable_Wrap(std::move(t)); }

// One Python function: a fixed number of positional arguments.
#define B200MOE_FUNCTION(FN, COUNT, BODY)                                                        \
  PyObject* py_##FN(PyObject*, PyObject* const* args, Py_ssize_t n) {                            \
    HANDLE_TH_ERRORS                                                                             \
    if (n != COUNT) refuse(#FN ": %d arguments expected, got %d", COUNT, static_cast<int>(n));   \
    const Args a{#FN, args};                                                                     \
    BODY                                                                                         \
    END_HANDLE_TH_ERRORS                                                                         \
  }
B200MOE_FUNCTION(paged_schedule, 12, paged_schedule(a); Py_RETURN_NONE;)
B200MOE_FUNCTION(paged_store_kvcache_fp8, 7, paged_store_kvcache_fp8(a); Py_RETURN_NONE;)
B200MOE_FUNCTION(paged_attn_varlen_fp8, 10, return wrap(paged_attn_varlen_fp8(a));)
B200MOE_FUNCTION(moe_few_tokens, 6, moe_few_tokens(a); Py_RETURN_NONE;)
#undef B200MOE_FUNCTION

#define B200MOE_METHOD(FN) \
  {#FN, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_##FN)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {B200MOE_METHOD(paged_schedule), B200MOE_METHOD(paged_store_kvcache_fp8),
                         B200MOE_METHOD(paged_attn_varlen_fp8), B200MOE_METHOD(moe_few_tokens),
                         {nullptr, nullptr, 0, nullptr}};
#undef B200MOE_METHOD

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" PyObject* PyInit__binding() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", B200MOE_BUILT_FOR) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
