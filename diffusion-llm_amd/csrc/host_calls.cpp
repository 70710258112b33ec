// host_calls.cpp - the Python calls of the kernels, prepared natively: a CPython
// extension (lib/bd3_host.so) that takes torch tensors, makes them readable for
// the kernels, allocates outputs and workspaces and calls the C ABI of
// libbd3attn.so on the tensors' current stream.
//
// Why: prepared in Python (attribute reads, torch.empty, slices of the cache and
// of the modulation vectors, ctypes argument conversion) a call cost more host
// time than most of the kernels it launches take. Host time per call, launches
// included: attention_inputs with a cache 16.0 -> 7.7 us, decode of a 16-token
// block (two launches) 16.4 -> 8.2, ln_modulate 12.9 -> 5.0, with the residual
// 17.8 -> 6.2, gate_residual 11.4 -> 4.7, the sampling draw 10.8 -> 5.5 (now two
// launches), training forward + backward 128 -> 87 (67 of it autograd's own).
//
// The C ABI's addresses come from the caller (bind), which loads the library, so
// the library path and a missing library behave as there. Argument errors raise
// AssertionError with the same texts as the Python checks and the library's
// messages, runtime errors RuntimeError. Every function drops the GIL once its
// arguments are unpacked: a launch can wait for a full queue.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <string>
#include <type_traits>

#include "bd3attn.h"

namespace {

using at::Tensor;

constexpr int kHeadDim = 64;
const float kScale = 1.0f / std::sqrt((float)kHeadDim);

// The C ABI, bound by name.
struct Library {
  decltype(&bd3_last_error) last_error;
  decltype(&bd3_attn_fwd) attn_fwd;
  decltype(&bd3_attn_bwd_workspace_bytes) attn_bwd_workspace_bytes;
  decltype(&bd3_attn_bwd) attn_bwd;
  decltype(&bd3_decode) decode;
  decltype(&bd3_decode_splitkv) decode_splitkv;
  decltype(&bd3_decode_workspace_bytes) decode_workspace_bytes;
  decltype(&bd3_qkv_rope) qkv_rope;
  decltype(&bd3_subs_sample_ws) subs_sample_ws;
  decltype(&bd3_subs_sample_workspace_bytes) subs_sample_workspace_bytes;
  decltype(&bd3_paged_attn_pool_workspace_bytes) paged_attn_workspace_bytes;
  decltype(&bd3_paged_attn_pool) paged_attn;
  decltype(&bd3_paged_qkv_rope) paged_qkv_rope;
  decltype(&bd3_paged_qkv_rope8) paged_qkv_rope8;
  decltype(&bd3_page_values) page_values;
  decltype(&bd3_page_bounds) page_bounds;
  decltype(&bd3_select_pages_workspace_bytes) select_pages_workspace_bytes;
  decltype(&bd3_select_pages) select_pages;
  decltype(&bd3_adjust_logits) adjust_logits;
  decltype(&bd3_ln_modulate) ln_modulate;
  decltype(&bd3_gate_residual) gate_residual;
  decltype(&bd3_gate_residual_ln_modulate) gate_residual_ln_modulate;
} g_lib = {};

// A Python exception to raise: its type (PyExc_...) and text.
struct Refused {
  PyObject* type;
  std::string text;
};

void require(bool ok, const char* text) {
  if (!ok) throw Refused{PyExc_AssertionError, text};
}

// Status of a C-ABI call, as kernels._native.check maps it.
void check(int status) {
  if (status == BD3_OK) return;
  const char* m = g_lib.last_error();
  const std::string text = m ? m : "";
  if (status == BD3_EINVAL) throw Refused{PyExc_AssertionError, text};
  throw Refused{PyExc_RuntimeError, "libbd3attn: " + text};
}

struct NoGil {
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// Runs f and turns what it throws into a Python exception.
template <class F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// Argument readers: positional only, in the order of the Python wrappers.
struct Args {
  PyObject* const* a;
  Py_ssize_t n, at = 0;
  Args(PyObject* const* args, Py_ssize_t count, Py_ssize_t want) : a(args), n(count) {
    if (count != want) throw Refused{PyExc_TypeError, "wrong number of arguments"};
  }
  Tensor tensor() {
    PyObject* o = a[at++];
    if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, "expected a tensor"};
    return THPVariable_Unpack(o);
  }
  Tensor maybe_tensor() {  // undefined for None
    if (a[at] == Py_None) {
      ++at;
      return Tensor();
    }
    return tensor();
  }
  int64_t integer() {
    const long long v = PyLong_AsLongLong(a[at++]);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  int32_t int32() {
    const int64_t v = integer();
    if (v < INT32_MIN || v > INT32_MAX) throw Refused{PyExc_OverflowError, "argument does not fit 32 bits"};
    return (int32_t)v;
  }
  uint64_t unsigned64() {  // modulo 2^64, any integer, as ctypes takes it (a seed or counter set by the caller)
    const unsigned long long v = PyLong_AsUnsignedLongLongMask(a[at++]);
    if (v == (unsigned long long)-1 && PyErr_Occurred()) throw python_error();
    return v;
  }
  double real() {
    const double v = PyFloat_AsDouble(a[at++]);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
  }
};

template <class... T>
PyObject* pack(const T&... t) {
  PyObject* r = PyTuple_New(sizeof...(T));
  if (r == nullptr) return nullptr;
  Py_ssize_t i = 0;
  (PyTuple_SET_ITEM(r, i++, THPVariable_Wrap(t)), ...);
  return r;
}

// The kernels read 16-byte vectors of rows in place: 16-byte aligned base,
// last stride 1, other strides multiples of 8 elements. Anything else is
// copied (kernels._native.as_kernel_input).
bool vec_ready(const Tensor& t) {
  if (t.dim() == 0 || t.stride(-1) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.stride(i) % 8 != 0) return false;
  return true;
}

Tensor ready(const Tensor& t) { return vec_ready(t) ? t : t.contiguous(); }

// (b, h, s) element strides of 4-D tensors, in order.
template <class... T>
std::array<int64_t, 3 * sizeof...(T)> strides(const T&... ts) {
  std::array<int64_t, 3 * sizeof...(T)> s;
  size_t i = 0;
  auto add = [&](const Tensor& t) {
    require(t.dim() == 4 && t.stride(-1) == 1, "tensors must be 4-D with last stride 1");
    for (int d = 0; d < 3; ++d) s[i++] = t.stride(d);
  };
  (add(ts), ...);
  return s;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

// The kernels read the operands' addresses as they are: refuses any that is not
// on the first one's GPU (an undefined one is an absent optional argument).
template <class... T>
void on_one_gpu(const Tensor& first, const T&... others) {
  require(first.is_cuda(), "inputs must be on CUDA");
  require((... && (!others.defined() || others.device() == first.device())), "inputs must be on one device");
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(bytes, 1)}, like.options().dtype(at::kByte));
}

int32_t dim32(const Tensor& t, int64_t d) { return (int32_t)t.size(d); }

// attn_fwd(q, k, v, block_size) -> (q, k, v, O, L): the tensors as the kernel read them.
PyObject* attn_fwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 4);
    Tensor q = a.tensor(), k = a.tensor(), v = a.tensor();
    const int32_t bs = a.int32();
    Tensor o, lse;
    on_one_gpu(q, k, v);
    {
      NoGil nogil;
      const c10::DeviceGuard device(q.device());
      q = ready(q);
      k = ready(k);
      v = ready(v);
      o = at::empty(q.sizes(), q.options());
      lse = at::empty({q.size(0), q.size(1), q.size(2)}, q.options().dtype(at::kFloat));
      const auto st = strides(q, k, v, o);
      check(g_lib.attn_fwd(ptr(q), ptr(k), ptr(v), ptr(o), static_cast<float*>(ptr(lse)), dim32(q, 0), dim32(q, 1),
                           dim32(q, 2) / 2, dim32(q, 3), bs, st.data(), kScale, stream_of(q)));
    }
    return pack(q, k, v, o, lse);
  });
}

// attn_bwd(q, k, v, O, L, dO, block_size) -> (dQ, dK, dV)
PyObject* attn_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 7);
    Tensor q = a.tensor(), k = a.tensor(), v = a.tensor(), o = a.tensor(), lse = a.tensor(), dout = a.tensor();
    const int32_t bs = a.int32();
    Tensor dq, dk, dv;
    on_one_gpu(q, k, v, o, lse, dout);
    {
      NoGil nogil;
      const c10::DeviceGuard device(q.device());
      q = ready(q);
      k = ready(k);
      v = ready(v);
      o = ready(o);
      lse = lse.contiguous();
      dout = ready(dout.to(q.scalar_type()));
      dq = at::empty(q.sizes(), q.options());
      dk = at::empty(q.sizes(), q.options());
      dv = at::empty(q.sizes(), q.options());
      const int32_t B = dim32(q, 0), H = dim32(q, 1), half = dim32(q, 2) / 2, D = dim32(q, 3);
      const size_t bytes = g_lib.attn_bwd_workspace_bytes(B, H, half, D);
      const Tensor ws = workspace(bytes, q);
      const auto st = strides(q, k, v, o, dout, dq, dk, dv);
      check(g_lib.attn_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(dout), static_cast<const float*>(ptr(lse)), ptr(dq),
                           ptr(dk), ptr(dv), ptr(ws), bytes, B, H, half, D, bs, st.data(), kScale, stream_of(q)));
    }
    return pack(dq, dk, dv);
  });
}

// decode(q, k, v, block_size, n_splits[, token_major]) -> O; n_splits 0:
// bd3_decode's own count; token_major: O is a (b, h, s, d) view of (b, s, h, d)
// memory, so that a caller's transpose + reshape to (b, s, h * d) copies nothing
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, n == 6 ? 6 : 5);
    Tensor q = a.tensor(), k = a.tensor(), v = a.tensor();
    const int32_t bs = a.int32(), splits = a.int32();
    const bool token_major = n == 6 && a.int32() != 0;
    Tensor o;
    on_one_gpu(q, k, v);
    {
      NoGil nogil;
      const c10::DeviceGuard device(q.device());
      q = ready(q);
      k = ready(k);
      v = ready(v);
      const int32_t B = dim32(q, 0), H = dim32(q, 1), L = dim32(q, 2), D = dim32(q, 3), kv = dim32(k, 2);
      o = token_major ? at::empty({B, L, H, D}, q.options()).transpose(1, 2) : at::empty(q.sizes(), q.options());
      const size_t bytes = g_lib.decode_workspace_bytes(B, H, L, kv, D, splits);
      const Tensor ws = bytes ? workspace(bytes, q) : Tensor();
      const auto st = strides(q, k, v, o);
      if (splits == 0)
        check(g_lib.decode(ptr(q), ptr(k), ptr(v), ptr(o), B, H, L, kv, D, bs, st.data(), kScale, ptr(ws), bytes,
                           stream_of(q)));
      else
        check(g_lib.decode_splitkv(ptr(q), ptr(k), ptr(v), ptr(o), B, H, L, kv, D, bs, splits, st.data(), kScale,
                                   ptr(ws), bytes, stream_of(q)));
    }
    return THPVariable_Wrap(o);
  });
}

// qkv_rope(qkv, heads, sin, cos, positions or None, pos0, k_buf, v_buf, len) -> (q, k_all, v_all):
// k and v go to slots len .. len + seq - 1 of the buffers (batch, heads, capacity,
// 64), k_all / v_all are their first len + seq tokens; without buffers
// (None) to new tensors.
PyObject* qkv_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 9);
    Tensor qkv = a.tensor();
    const int64_t heads = a.integer();
    Tensor sin = a.tensor(), cos = a.tensor(), positions = a.maybe_tensor();
    const int32_t pos0 = a.int32();
    Tensor k = a.maybe_tensor(), v = a.maybe_tensor();
    const int64_t len = a.integer();
    Tensor q, k_all, v_all;
    on_one_gpu(qkv, sin, cos, k, v);
    {
      NoGil nogil;
      const c10::DeviceGuard device(qkv.device());
      qkv = ready(qkv);
      sin = sin.contiguous();
      cos = cos.contiguous();
      if (positions.defined()) positions = positions.to(qkv.device(), at::kLong).contiguous();
      const int64_t B = qkv.size(0), S = qkv.size(1);
      q = at::empty({B, heads, S, kHeadDim}, qkv.options());
      Tensor k_out, v_out;
      if (k.defined()) {
        k_out = k.narrow(2, len, S);
        v_out = v.narrow(2, len, S);
      } else {
        k_out = at::empty_like(q);
        v_out = at::empty_like(q);
      }
      const int64_t xs[2] = {qkv.stride(0), qkv.stride(1)};
      const auto st = strides(q, k_out, v_out);
      check(g_lib.qkv_rope(ptr(qkv), xs, (int32_t)B, (int32_t)S, (int32_t)heads, kHeadDim,
                           static_cast<const int64_t*>(ptr(positions)), pos0, static_cast<const float*>(ptr(sin)),
                           static_cast<const float*>(ptr(cos)), dim32(sin, 0), ptr(q), ptr(k_out), ptr(v_out),
                           st.data(), stream_of(qkv)));
      k_all = k.defined() ? k.narrow(2, 0, len + S) : k_out;
      v_all = v.defined() ? v.narrow(2, 0, len + S) : v_out;
    }
    return pack(q, k_all, v_all);
  });
}

// subs_sample(logits, block, mask_index, keep, u or None, seed, offset) -> the next block
PyObject* subs_sample(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 7);
    const Tensor logits = a.tensor(), block = a.tensor();
    const int32_t mask = a.int32();
    const double keep = a.real();
    Tensor u = a.maybe_tensor();
    const uint64_t seed = a.unsigned64(), offset = a.unsigned64();
    Tensor out;
    on_one_gpu(logits, u);
    {
      NoGil nogil;
      const c10::DeviceGuard device(logits.device());
      const int64_t rows = block.numel(), vocab = logits.size(-1);
      Tensor lg = logits.reshape({rows, vocab});
      if (lg.stride(-1) != 1) lg = lg.contiguous();
      const Tensor xt = block.reshape({rows}).to(logits.device(), at::kLong).contiguous();
      out = at::empty_like(xt);
      if (u.defined()) u = u.reshape({rows, vocab}).contiguous();
      const size_t bytes = g_lib.subs_sample_workspace_bytes((int32_t)rows, (int32_t)vocab);
      const Tensor ws = bytes ? workspace(bytes, lg) : Tensor();
      check(g_lib.subs_sample_ws(ptr(lg), lg.stride(0), lg.scalar_type() == at::kFloat, static_cast<int64_t*>(ptr(xt)),
                                 static_cast<int64_t*>(ptr(out)), (int32_t)rows, (int32_t)vocab, mask, keep,
                                 static_cast<const double*>(ptr(u)), seed, offset, ptr(ws), bytes, stream_of(lg)));
      out = out.view(block.sizes());
    }
    return THPVariable_Wrap(out);
  });
}

int32_t is_f32(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return 1;
  if (t.scalar_type() == at::kBFloat16) return 0;
  throw Refused{PyExc_KeyError, std::string("bf16 or fp32 tensors only, got ") + c10::toString(t.scalar_type())};
}

// The pages of a pool and, of an 8-bit one, their scales.
int32_t pool_type(const Tensor& pages) {
  if (pages.scalar_type() == at::kBFloat16) return BD3_POOL_BF16;
  if (pages.scalar_type() == at::kChar) return BD3_POOL_INT8;
  require(pages.scalar_type() == at::kFloat8_e4m3fn, "bf16 inputs only (pages may be int8 or float8_e4m3fn, with scales)");
  return BD3_POOL_E4M3;
}

bool pages_ready(const Tensor& t) {
  if (!vec_ready(t)) return false;
  for (int64_t i = 0; i < 3; ++i)
    if (t.stride(i) * t.element_size() % 16 != 0) return false;
  return true;
}

void check_scales(const Tensor& pages, const Tensor& scales) {
  require(scales.defined() == (pool_type(pages) != BD3_POOL_BF16), "8-bit pages need scales, bf16 pages take none");
  if (!scales.defined()) return;
  on_one_gpu(pages, scales);
  require(scales.scalar_type() == at::kFloat && scales.dim() == 3 && scales.size(0) == pages.size(0) &&
              scales.size(1) == pages.size(1) && scales.size(2) == pages.size(2) / 16 && scales.is_contiguous(),
          "scales must be contiguous float32 (pages, kv_heads, page_size / 16)");
}

const float* scales_p(const Tensor& t) { return t.defined() ? static_cast<const float*>(t.data_ptr()) : nullptr; }

// The arrays that describe a ragged batch.
struct BatchArrays {
  Tensor table, starts, lens;
  int32_t seqs, width;
  BatchArrays(Args& a) : table(a.tensor()), starts(a.tensor()), lens(a.tensor()) {}
  void check(const Tensor& first) {
    on_one_gpu(first, table, starts, lens);
    require(table.scalar_type() == at::kInt && starts.scalar_type() == at::kInt && lens.scalar_type() == at::kInt,
            "page_table, q_starts and kv_lens must be int32");
    require(table.dim() == 2 && (table.size(1) == 1 || table.stride(1) == 1),
            "page_table must be (seqs, width) with last stride 1");
    require(starts.dim() == 1 && lens.dim() == 1 && starts.size(0) == table.size(0) + 1 &&
                lens.size(0) == table.size(0) && starts.is_contiguous() && lens.is_contiguous(),
            "q_starts must be (seqs + 1) and kv_lens (seqs), contiguous");
    require(table.size(0) <= INT32_MAX - 1 && table.size(1) <= INT32_MAX, "batch or pool too large");
    seqs = dim32(table, 0);
    width = dim32(table, 1);
  }
  const int32_t* table_p() const { return static_cast<const int32_t*>(ptr(table)); }
  const int32_t* starts_p() const { return static_cast<const int32_t*>(ptr(starts)); }
  const int32_t* lens_p() const { return static_cast<const int32_t*>(ptr(lens)); }
};

// The tensors that describe a ragged batch and its pool, checked (the kernels take
// their addresses and sizes as they are).
struct PagedPool {
  Tensor k, v;
  int32_t pages, kv_heads, page, type;
  PagedPool(Args& a) : k(a.tensor()), v(a.tensor()) {}
};
struct PagedBatch : PagedPool, BatchArrays {
  PagedBatch(Args& a) : PagedPool(a), BatchArrays(a) {}
  void check(const Tensor& first, int64_t heads) {
    on_one_gpu(first, k, v, table, starts, lens);
    type = pool_type(k);
    require(v.scalar_type() == k.scalar_type(), "k_pages and v_pages must have one dtype");
    require(k.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == kHeadDim,
            "k_pages and v_pages must be (pages, kv_heads, page_size, 64)");
    require(pages_ready(k) && pages_ready(v), "k_pages and v_pages must have 16-byte aligned rows (they are not copied)");
    require(k.size(1) >= 1 && heads % k.size(1) == 0, "heads must be a multiple of k_pages' kv_heads");
    BatchArrays::check(first);
    require(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX, "batch or pool too large");
    pages = dim32(k, 0);
    kv_heads = dim32(k, 1);
    page = k.size(2) <= INT32_MAX ? dim32(k, 2) : 0;
  }
};

// Written tensors: no element twice (an expanded one would be a race).
bool writable(const Tensor& t) { return at::has_internal_overlap(t) != at::MemOverlap::Yes; }

// A written tensor apart from all that the same launch reads or writes elsewhere, as far
// as that can be told (dense tensors; woven views are the caller's to keep apart).
// Absent and empty ones are.
bool apart_from(const Tensor& written, const Tensor& other) {
  if (!written.defined() || !other.defined() || written.storage().data() == nullptr ||
      written.storage().data() != other.storage().data() || written.numel() == 0 || other.numel() == 0)
    return true;
  const auto s = at::get_overlap_status(written, other);
  return s != at::MemOverlapStatus::Full && s != at::MemOverlapStatus::Partial && written.data_ptr() != other.data_ptr();
}
template <class... T>
bool apart(const Tensor& written, const T&... others) {
  return (... && apart_from(written, others));
}

// Every element of one at the address of the other's (of the same sizes): strides of
// dimensions of one do not matter.
bool same_memory(const Tensor& a, const Tensor& b) {
  if (a.data_ptr() != b.data_ptr()) return false;
  for (int64_t i = 0; i < a.dim(); ++i)
    if (a.size(i) != 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// Packed tokens, readable for the kernels. A single one counts as contiguous whatever
// its stride is, and contiguous() hands it back; in ordinary use it is a row of a wider
// tensor.
Tensor ready_tokens(const Tensor& t) {
  const Tensor c = ready(t);
  return vec_ready(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}

// (tokens, heads, 64) result: the caller's, or a new one.
Tensor token_rows(const Tensor& out, int64_t tokens, int64_t heads, const Tensor& like) {
  if (!out.defined()) return at::empty({tokens, heads, kHeadDim}, like.options());
  require(out.dim() == 3 && out.size(0) == tokens && out.size(1) == heads && out.size(2) == kHeadDim &&
              out.scalar_type() == at::kBFloat16 && out.device() == like.device() && vec_ready(out) && writable(out),
          "out must be a (tokens, heads, 64) bf16 tensor with 16-byte aligned rows");
  return out;
}

// paged_attention(q, k_pages, v_pages, page_table, q_starts, kv_lens, block_size, max_q, max_kv, total_kv,
// out or None, k_scales or None, v_scales or None, columns or None) -> O; max_kv, total_kv < 0: the table's,
// seqs * max_kv
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 14);
    Tensor q = a.tensor();
    PagedBatch b(a);
    const int32_t bs = a.int32(), max_q = a.int32();
    int32_t max_kv = a.int32();
    int64_t total = a.integer();
    Tensor out = a.maybe_tensor();
    const Tensor k_scales = a.maybe_tensor(), v_scales = a.maybe_tensor();
    Tensor columns = a.maybe_tensor();
    require(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.size(2) == kHeadDim,
            "q must be a (tokens, heads, 64) bf16 tensor");
    require(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX, "q is too large");
    b.check(q, q.size(1));
    check_scales(b.k, k_scales);
    check_scales(b.v, v_scales);
    if (columns.defined()) {
      on_one_gpu(q, columns);
      require(columns.dim() == 3 && columns.scalar_type() == at::kInt && columns.size(0) == q.size(0) &&
                  columns.size(1) == b.kv_heads && columns.size(2) >= 1 && columns.size(2) <= INT32_MAX &&
                  (columns.size(2) == 1 || columns.stride(2) == 1),
              "columns must be int32 (tokens, kv_heads, top) with last stride 1");
    }
    {
      NoGil nogil;
      const c10::DeviceGuard device(q.device());
      q = ready_tokens(q);
      const int32_t T = dim32(q, 0), H = dim32(q, 1), top = columns.defined() ? dim32(columns, 2) : 0;
      out = token_rows(out, T, H, q);
      require(apart(out, q, b.k, b.v, b.table, b.starts, b.lens, k_scales, v_scales, columns), "out must not overlap an input");
      if (max_kv < 0) max_kv = (int32_t)std::min<int64_t>((int64_t)b.width * b.page, INT32_MAX);
      if (total < 0) total = (int64_t)b.seqs * max_kv;
      const size_t bytes =
          g_lib.paged_attn_workspace_bytes(b.type, b.seqs, T, H, b.kv_heads, b.page, max_q, max_kv, total, bs, top);
      const Tensor ws = bytes ? workspace(bytes, q) : Tensor();
      const int64_t st[13] = {q.stride(0),   q.stride(1),   b.k.stride(0), b.k.stride(1),   b.k.stride(2),
                              b.v.stride(0), b.v.stride(1), b.v.stride(2), out.stride(0),   out.stride(1),
                              b.table.stride(0), top ? columns.stride(0) : 0, top ? columns.stride(1) : 0};
      check(g_lib.paged_attn(ptr(q), ptr(b.k), ptr(b.v), scales_p(k_scales), scales_p(v_scales), b.type, ptr(out),
                             b.table_p(), b.starts_p(), b.lens_p(), static_cast<const int32_t*>(ptr(columns)), top, b.seqs,
                             T, H, b.kv_heads, kHeadDim, b.pages, b.page, b.width, max_q, max_kv, total, bs, st, kScale,
                             ptr(ws), bytes, stream_of(q)));
    }
    return THPVariable_Wrap(out);
  });
}

// paged_attention_inputs(qkv, heads, sin, cos, k_pages, v_pages, page_table, q_starts, kv_lens, out or None,
// k_scales or None, v_scales or None) -> q
PyObject* paged_attention_inputs(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 12);
    Tensor qkv = a.tensor();
    const int32_t heads = a.int32();
    Tensor sin = a.tensor(), cos = a.tensor();
    PagedBatch b(a);
    Tensor out = a.maybe_tensor();
    const Tensor k_scales = a.maybe_tensor(), v_scales = a.maybe_tensor();
    require(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16, "qkv must be a (tokens, width) bf16 tensor");
    require(heads >= 1, "n_heads must be >= 1");
    b.check(qkv, heads);
    on_one_gpu(qkv, sin, cos);
    check_scales(b.k, k_scales);
    check_scales(b.v, v_scales);
    require(writable(b.k) && writable(b.v), "k_pages and v_pages are written: no element may occur twice");
    require(qkv.size(1) == ((int64_t)heads + 2 * (int64_t)b.kv_heads) * kHeadDim,
            "projection width must be (n_heads + 2 * kv_heads) * 64");
    require(qkv.size(0) <= INT32_MAX, "qkv is too large");
    require(sin.dim() == 2 && sin.sizes() == cos.sizes() && sin.size(1) == kHeadDim / 2 &&
                sin.scalar_type() == at::kFloat && cos.scalar_type() == at::kFloat && sin.size(0) <= INT32_MAX,
            "RoPE tables must be (max_seq_len, 32) float32");
    {
      NoGil nogil;
      const c10::DeviceGuard device(qkv.device());
      qkv = ready_tokens(qkv);
      sin = ready(sin.contiguous());
      cos = ready(cos.contiguous());
      out = token_rows(out, qkv.size(0), heads, qkv);
      require(qkv.numel() == 0 || (apart(out, qkv, b.k, b.v) && apart(b.k, qkv, b.v) && apart(b.v, qkv)),
              "qkv, out, k_pages and v_pages must not overlap");
      for (const Tensor* t : {&out, &b.k, &b.v})
        require(apart(*t, sin, cos, b.table, b.starts, b.lens), "out and the pages must not overlap an input");
      const int64_t st[10] = {qkv.stride(0), out.stride(0), out.stride(1), b.k.stride(0), b.k.stride(1), b.k.stride(2),
                              b.v.stride(0), b.v.stride(1), b.v.stride(2), b.table.stride(0)};
      if (b.type == BD3_POOL_BF16) {
        check(g_lib.paged_qkv_rope(ptr(qkv), static_cast<const float*>(ptr(sin)), static_cast<const float*>(ptr(cos)),
                                   dim32(sin, 0), ptr(out), ptr(b.k), ptr(b.v), b.table_p(), b.starts_p(), b.lens_p(),
                                   b.seqs, dim32(qkv, 0), heads, b.kv_heads, kHeadDim, b.pages, b.page, b.width, st,
                                   stream_of(qkv)));
      } else {
        for (const Tensor* t : {&k_scales, &v_scales})
          require(apart(*t, qkv, out, b.k, b.v, sin, cos, b.table, b.starts, b.lens), "the scales must not overlap another argument");
        require(apart(k_scales, v_scales), "the scales must not overlap another argument");
        check(g_lib.paged_qkv_rope8(ptr(qkv), static_cast<const float*>(ptr(sin)), static_cast<const float*>(ptr(cos)),
                                    dim32(sin, 0), ptr(out), ptr(b.k), ptr(b.v), static_cast<float*>(ptr(k_scales)),
                                    static_cast<float*>(ptr(v_scales)), b.type, b.table_p(), b.starts_p(), b.lens_p(),
                                    b.seqs, dim32(qkv, 0), heads, b.kv_heads, kHeadDim, b.pages, b.page, b.width, st,
                                    stream_of(qkv)));
      }
    }
    return THPVariable_Wrap(out);
  });
}

// page_values(k_pages, v_pages, k_scales, v_scales) -> (k, v) bf16
PyObject* page_values(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 4);
    const Tensor k = a.tensor(), v = a.tensor(), k_scales = a.tensor(), v_scales = a.tensor();
    on_one_gpu(k, v);
    const int32_t type = pool_type(k);
    require(type != BD3_POOL_BF16, "k_pages and v_pages must be int8 or float8_e4m3fn");
    require(v.scalar_type() == k.scalar_type(), "k_pages and v_pages must have one dtype");
    require(k.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == kHeadDim,
            "k_pages and v_pages must be (pages, kv_heads, page_size, 64)");
    require(pages_ready(k) && pages_ready(v), "k_pages and v_pages must have 16-byte aligned rows (they are not copied)");
    require(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX, "pool too large");
    check_scales(k, k_scales);
    check_scales(v, v_scales);
    Tensor k_out, v_out;
    {
      NoGil nogil;
      const c10::DeviceGuard device(k.device());
      k_out = at::empty(k.sizes(), k.options().dtype(at::kBFloat16));
      v_out = at::empty(k.sizes(), k.options().dtype(at::kBFloat16));
      const int64_t st[6] = {k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2)};
      check(g_lib.page_values(ptr(k), ptr(v), scales_p(k_scales), scales_p(v_scales), type, ptr(k_out), ptr(v_out),
                              dim32(k, 0), dim32(k, 1), dim32(k, 2), kHeadDim, st, stream_of(k)));
    }
    return pack(k_out, v_out);
  });
}

void check_bounds(const Tensor& bounds, int64_t pages, int64_t kv_heads) {
  require(bounds.dim() == 4 && bounds.scalar_type() == at::kBFloat16 && (pages < 0 || bounds.size(0) == pages) &&
              (kv_heads < 0 || bounds.size(1) == kv_heads) && bounds.size(2) == 2 && bounds.size(3) == kHeadDim &&
              bounds.is_contiguous() && vec_ready(bounds),
          "bounds must be contiguous bf16 (pages, kv_heads, 2, 64)");
}

// page_bounds(k_pages, bounds, page_table, q_starts, kv_lens, tokens, k_scales or None) -> bounds
PyObject* page_bounds(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 7);
    const Tensor k = a.tensor(), bounds = a.tensor();
    BatchArrays b(a);
    const int32_t tokens = a.int32();
    const Tensor k_scales = a.maybe_tensor();
    on_one_gpu(k, bounds);
    b.check(k);
    const int32_t type = pool_type(k);
    require(k.dim() == 4 && k.size(3) == kHeadDim && k.size(1) >= 1, "k_pages must be (pages, kv_heads, page_size, 64)");
    require(pages_ready(k), "k_pages must have 16-byte aligned rows (they are not copied)");
    require(k.size(0) <= INT32_MAX && k.size(1) <= INT32_MAX && k.size(2) <= INT32_MAX, "pool too large");
    check_scales(k, k_scales);
    check_bounds(bounds, k.size(0), k.size(1));
    {
      NoGil nogil;
      const c10::DeviceGuard device(k.device());
      require(apart(bounds, k, b.table, b.starts, b.lens, k_scales), "bounds must not overlap an input");
      const int64_t st[4] = {k.stride(0), k.stride(1), k.stride(2), b.table.stride(0)};
      check(g_lib.page_bounds(ptr(k), scales_p(k_scales), type, ptr(bounds), b.table_p(), b.starts_p(), b.lens_p(), b.seqs,
                              tokens, dim32(k, 1), kHeadDim, dim32(k, 0), dim32(k, 2), b.width, st, stream_of(k)));
    }
    return THPVariable_Wrap(bounds);
  });
}

// select_pages(q, bounds, page_table, q_starts, kv_lens, block_size, page_size, top, max_q, max_kv, first, recent,
// out or None) -> columns; max_kv < 0: the table's
PyObject* select_pages(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 13);
    Tensor q = a.tensor();
    const Tensor bounds = a.tensor();
    BatchArrays b(a);
    const int32_t bs = a.int32(), page = a.int32(), top = a.int32(), max_q = a.int32();
    int32_t max_kv = a.int32();
    const int32_t first = a.int32(), recent = a.int32();
    Tensor out = a.maybe_tensor();
    require(q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.size(2) == kHeadDim,
            "q must be a (tokens, heads, 64) bf16 tensor");
    require(q.size(0) <= INT32_MAX && q.size(1) <= INT32_MAX, "q is too large");
    on_one_gpu(q, bounds);
    b.check(q);
    check_bounds(bounds, -1, -1);
    require(bounds.size(0) <= INT32_MAX && bounds.size(1) >= 1 && q.size(1) % bounds.size(1) == 0,
            "heads must be a multiple of the bounds' kv_heads");
    require(page >= 1, "page_size must be a power of two in [16, 1024]");
    {
      NoGil nogil;
      const c10::DeviceGuard device(q.device());
      q = ready_tokens(q);
      const int32_t T = dim32(q, 0), H = dim32(q, 1), KH = dim32(bounds, 1);
      require(top >= 1, "top must be >= 1");
      if (!out.defined()) out = at::empty({T, KH, top}, q.options().dtype(at::kInt));
      require(out.dim() == 3 && out.size(0) == T && out.size(1) == KH && out.size(2) == top && out.scalar_type() == at::kInt &&
                  out.device() == q.device() && out.is_contiguous(),
              "out must be contiguous int32 (tokens, kv_heads, top)");
      require(apart(out, q, bounds, b.table, b.starts, b.lens), "out must not overlap an input");
      if (max_kv < 0) max_kv = (int32_t)std::min<int64_t>((int64_t)b.width * page, INT32_MAX);
      const size_t bytes = g_lib.select_pages_workspace_bytes(b.seqs, T, KH, page, std::max(max_kv, 1), bs);
      const Tensor ws = bytes ? workspace(bytes, q) : Tensor();
      const int64_t st[3] = {q.stride(0), q.stride(1), b.table.stride(0)};
      check(g_lib.select_pages(ptr(q), ptr(bounds), b.table_p(), b.starts_p(), b.lens_p(), static_cast<int32_t*>(ptr(out)),
                               b.seqs, T, H, KH, kHeadDim, dim32(bounds, 0), page, b.width, max_q, max_kv, bs, top, first,
                               recent, st, ptr(ws), bytes, stream_of(q)));
    }
    return THPVariable_Wrap(out);
  });
}

// A penalty: one number, or a (batch) float32 tensor.
struct Penalty {
  float one;
  Tensor each;
  Penalty(Args& a, float neutral) : one(neutral) {
    if (THPVariable_Check(a.a[a.at]))
      each = a.tensor();
    else
      one = (float)a.real();
  }
  const float* p() const { return static_cast<const float*>(ptr(each)); }
};

// adjust_logits(logits (batch, rows, vocab), tokens or None, lengths or None, repetition, frequency, presence, bias or
// None, allowed or None, fill, out or None) -> out
PyObject* adjust_logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 10);
    Tensor x = a.tensor(), tokens = a.maybe_tensor(), lengths = a.maybe_tensor();
    Penalty rep(a, 1.f), freq(a, 0.f), pres(a, 0.f);
    Tensor bias = a.maybe_tensor(), allowed = a.maybe_tensor();
    const double fill = a.real();
    Tensor out = a.maybe_tensor();
    on_one_gpu(x, tokens, lengths, rep.each, freq.each, pres.each, bias, allowed, out);
    require(x.dim() == 3, "logits must be (batch, rows, vocab)");
    const int64_t B = x.size(0), R = x.size(1), V = x.size(2);
    require(B <= INT32_MAX && R <= INT32_MAX && V <= INT32_MAX && V >= 1, "logits are too large");
    const int32_t fp32 = is_f32(x);
    int64_t history = 0;
    if (tokens.defined()) {
      require(tokens.dim() == 2 && tokens.size(0) == B && tokens.scalar_type() == at::kLong,
              "tokens must be (batch, history) int64");
      history = tokens.size(1);
      require(history <= INT32_MAX, "the history is too long");
    }
    if (lengths.defined())
      require(tokens.defined() && lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == at::kInt,
              "lengths must be (batch) int32, with tokens");
    for (Penalty* p : {&rep, &freq, &pres})
      if (p->each.defined())
        require(p->each.dim() == 1 && p->each.size(0) == B && p->each.scalar_type() == at::kFloat,
                "a penalty must be a number or a (batch) float32 tensor");
    if (bias.defined())
      require(bias.scalar_type() == at::kFloat && bias.size(-1) == V && bias.dim() <= 2 &&
                  (bias.dim() == 1 || bias.size(0) == B),
              "bias must be (vocab) or (batch, vocab) float32");
    if (allowed.defined())
      require(allowed.scalar_type() == at::kInt && allowed.dim() >= 1 && allowed.dim() <= 3 &&
                  allowed.size(-1) == (V + 31) / 32 && (allowed.dim() == 1 || allowed.size(0) == B) &&
                  (allowed.dim() < 3 || allowed.size(1) == R),
              "allowed must be int32 words, (ceil(vocab / 32)) for all, each sequence or each row");
    {
      NoGil nogil;
      const c10::DeviceGuard device(x.device());
      if (x.stride(2) != 1 && V > 1) x = x.contiguous();
      auto rows = [](Tensor& t) {
        if (t.defined() && t.dim() > 0 && t.stride(-1) != 1) t = t.contiguous();
      };
      rows(tokens);
      rows(bias);
      rows(allowed);
      if (lengths.defined()) lengths = lengths.contiguous();
      for (Penalty* p : {&rep, &freq, &pres})
        if (p->each.defined()) p->each = p->each.contiguous();
      if (!out.defined()) out = at::empty({B, R, V}, x.options());
      require(out.scalar_type() == x.scalar_type() && out.sizes() == x.sizes() && (V == 1 || out.stride(2) == 1) &&
                  writable(out),
              "out must have the logits' shape and dtype, with last stride 1");
      require(same_memory(out, x) || at::get_overlap_status(out, x) != at::MemOverlapStatus::Partial,
              "out must be the logits themselves or not overlap them");
      require(apart(out, tokens, lengths, rep.each, freq.each, pres.each, bias, allowed),
              "out must not overlap an input other than the logits");
      const float penalties[3] = {rep.one, freq.one, pres.one};
      const int64_t st[8] = {x.stride(0),
                             x.stride(1),
                             out.stride(0),
                             out.stride(1),
                             tokens.defined() ? tokens.stride(0) : 0,
                             bias.defined() && bias.dim() == 2 ? bias.stride(0) : 0,
                             allowed.defined() && allowed.dim() > 1 ? allowed.stride(0) : 0,
                             allowed.defined() && allowed.dim() > 2 ? allowed.stride(1) : 0};
      check(g_lib.adjust_logits(ptr(x), fp32, ptr(out), (int32_t)B, (int32_t)R, (int32_t)V,
                                static_cast<const int64_t*>(ptr(tokens)), (int32_t)history,
                                static_cast<const int32_t*>(ptr(lengths)), penalties, rep.p(), freq.p(), pres.p(),
                                static_cast<const float*>(ptr(bias)), static_cast<const int32_t*>(ptr(allowed)),
                                (float)fill, st, stream_of(x)));
    }
    return THPVariable_Wrap(out);
  });
}

// A (batch, d) or (batch, 1, d) modulation vector as (batch, d).
Tensor vec(Tensor t) {
  if (t.dim() == 3) {
    require(t.size(1) == 1, "modulation vectors broadcast over the sequence");
    t = t.select(1, 0);
  }
  return ready(t);
}

bool is_bd(const Tensor& t, int64_t B, int64_t D) { return t.dim() == 2 && t.size(0) == B && t.size(1) == D; }

at::ScalarType float_type(bool f32) { return f32 ? at::kFloat : at::kBFloat16; }

// ln_modulate(x, weight, shift, scale, eps, out_fp32): out_fp32 -1 keeps the eager dtype
PyObject* ln_modulate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 6);
    Tensor x = a.tensor(), w = a.tensor(), shift = a.tensor(), scale = a.tensor();
    const double eps = a.real();
    const int64_t want = a.integer();
    Tensor out;
    on_one_gpu(x, w, shift, scale);
    {
      NoGil nogil;
      const c10::DeviceGuard device(x.device());
      const int64_t B = x.size(0), S = x.size(1), D = x.size(2);
      x = ready(x);
      w = ready(w);
      shift = vec(shift);
      scale = vec(scale);
      require(shift.scalar_type() == scale.scalar_type() && is_bd(shift, B, D) && is_bd(scale, B, D),
              "shift and scale must be (batch, d_model) of one dtype");
      const int32_t xf = is_f32(x), mf = is_f32(shift);
      out = at::empty({B, S, D}, x.options().dtype(float_type(want < 0 ? xf || mf : want != 0)));
      const int64_t st[5] = {x.stride(0), x.stride(1), shift.stride(0), out.stride(0), out.stride(1)};
      check(g_lib.ln_modulate(ptr(x), xf, ptr(w), is_f32(w), ptr(shift), ptr(scale), mf, ptr(out), is_f32(out),
                              (int32_t)B, (int32_t)S, (int32_t)D, st, (float)eps, stream_of(x)));
    }
    return THPVariable_Wrap(out);
  });
}

// gate_residual(x, gate, y, out or None)
PyObject* gate_residual(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 4);
    Tensor x = a.tensor(), gate = a.tensor(), y = a.tensor(), out = a.maybe_tensor();
    on_one_gpu(x, gate, y, out);
    {
      NoGil nogil;
      const c10::DeviceGuard device(x.device());
      const int64_t B = x.size(0), S = x.size(1), D = x.size(2);
      x = ready(x);
      y = ready(y);
      gate = vec(gate);
      const int32_t xf = is_f32(x), gf = is_f32(gate), yf = is_f32(y);
      const at::ScalarType type = float_type(xf || gf || yf);
      if (!out.defined()) out = at::empty({B, S, D}, x.options().dtype(type));
      require(out.scalar_type() == type && out.sizes() == x.sizes(), "out must have the result's shape and dtype");
      const int64_t st[7] = {x.stride(0), x.stride(1),   gate.stride(0), y.stride(0),
                             y.stride(1), out.stride(0), out.stride(1)};
      check(g_lib.gate_residual(ptr(x), xf, ptr(gate), gf, ptr(y), yf, ptr(out), (int32_t)B, (int32_t)S, (int32_t)D,
                                st, stream_of(x)));
    }
    return THPVariable_Wrap(out);
  });
}

// gate_residual_ln_modulate(x, gate, y, weight, shift, scale, eps, out_fp32, x_out or None) -> (x_out, out)
PyObject* gate_residual_ln_modulate(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded([&] {
    Args a(args, n, 9);
    Tensor x = a.tensor(), gate = a.tensor(), y = a.tensor(), w = a.tensor(), shift = a.tensor(), scale = a.tensor();
    const double eps = a.real();
    const int64_t want = a.integer();
    Tensor x_out = a.maybe_tensor(), out;
    on_one_gpu(x, gate, y, w, shift, scale, x_out);
    {
      NoGil nogil;
      const c10::DeviceGuard device(x.device());
      const int64_t B = x.size(0), S = x.size(1), D = x.size(2);
      x = ready(x);
      y = ready(y);
      w = ready(w);
      gate = vec(gate);
      shift = vec(shift);
      scale = vec(scale);
      require(gate.scalar_type() == shift.scalar_type() && shift.scalar_type() == scale.scalar_type() &&
                  is_bd(gate, B, D) && is_bd(shift, B, D) && is_bd(scale, B, D),
              "gate, shift and scale must be (batch, d_model) of one dtype");
      if (gate.stride(0) != shift.stride(0) || shift.stride(0) != scale.stride(0)) {  // one batch stride for the three
        gate = gate.contiguous();
        shift = shift.contiguous();
        scale = scale.contiguous();
      }
      const int32_t xf = is_f32(x), mf = is_f32(gate), yf = is_f32(y);
      const bool rf = xf || mf || yf;
      if (!x_out.defined()) x_out = at::empty({B, S, D}, x.options().dtype(float_type(rf)));
      require(x_out.scalar_type() == float_type(rf) && x_out.sizes() == x.sizes(),
              "x_out must have the residual's shape and dtype");
      out = at::empty({B, S, D}, x.options().dtype(float_type(want < 0 ? rf || mf : want != 0)));
      const int64_t st[9] = {x.stride(0),     x.stride(1),     gate.stride(0), y.stride(0),  y.stride(1),
                             x_out.stride(0), x_out.stride(1), out.stride(0),  out.stride(1)};
      check(g_lib.gate_residual_ln_modulate(ptr(x), xf, ptr(gate), ptr(y), yf, ptr(x_out), ptr(w), is_f32(w),
                                            ptr(shift), ptr(scale), mf, ptr(out), is_f32(out), (int32_t)B, (int32_t)S,
                                            (int32_t)D, st, (float)eps, stream_of(x)));
    }
    return pack(x_out, out);
  });
}

// bind({"bd3_...": address}): the C ABI of the loaded library.
PyObject* bind(PyObject*, PyObject* dict) {
  return guarded([&]() -> PyObject* {
    if (!PyDict_Check(dict)) throw Refused{PyExc_TypeError, "bind takes a dict of addresses"};
    auto set = [&](const char* name, auto& fn) {
      PyObject* o = PyDict_GetItemString(dict, name);
      void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
      if (p == nullptr) throw Refused{PyExc_KeyError, std::string("no address for ") + name};
      fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(p);
    };
    Library l = {};
    set("bd3_last_error", l.last_error);
    set("bd3_attn_fwd", l.attn_fwd);
    set("bd3_attn_bwd_workspace_bytes", l.attn_bwd_workspace_bytes);
    set("bd3_attn_bwd", l.attn_bwd);
    set("bd3_decode", l.decode);
    set("bd3_decode_splitkv", l.decode_splitkv);
    set("bd3_decode_workspace_bytes", l.decode_workspace_bytes);
    set("bd3_qkv_rope", l.qkv_rope);
    set("bd3_subs_sample_ws", l.subs_sample_ws);
    set("bd3_subs_sample_workspace_bytes", l.subs_sample_workspace_bytes);
    set("bd3_paged_attn_pool_workspace_bytes", l.paged_attn_workspace_bytes);
    set("bd3_paged_attn_pool", l.paged_attn);
    set("bd3_paged_qkv_rope", l.paged_qkv_rope);
    set("bd3_paged_qkv_rope8", l.paged_qkv_rope8);
    set("bd3_page_values", l.page_values);
    set("bd3_page_bounds", l.page_bounds);
    set("bd3_select_pages_workspace_bytes", l.select_pages_workspace_bytes);
    set("bd3_select_pages", l.select_pages);
    set("bd3_adjust_logits", l.adjust_logits);
    set("bd3_ln_modulate", l.ln_modulate);
    set("bd3_gate_residual", l.gate_residual);
    set("bd3_gate_residual_ln_modulate", l.gate_residual_ln_modulate);
    g_lib = l;
    Py_RETURN_NONE;
  });
}

#define BD3_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {
    {"bind", bind, METH_O, nullptr},
    BD3_FAST(attn_fwd),
    BD3_FAST(attn_bwd),
    BD3_FAST(decode),
    BD3_FAST(qkv_rope),
    BD3_FAST(subs_sample),
    BD3_FAST(paged_attention),
    BD3_FAST(paged_attention_inputs),
    BD3_FAST(page_values),
    BD3_FAST(page_bounds),
    BD3_FAST(select_pages),
    BD3_FAST(adjust_logits),
    BD3_FAST(ln_modulate),
    BD3_FAST(gate_residual),
    BD3_FAST(gate_residual_ln_modulate),
    {nullptr, nullptr, 0, nullptr},
};
#undef BD3_FAST

PyModuleDef module = {PyModuleDef_HEAD_INIT, "bd3_host", "Native preparation of the kernels' Python calls.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_bd3_host(void) { return PyModule_Create(&module); }
