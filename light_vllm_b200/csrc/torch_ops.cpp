// CPython module light_vllm_b200._torch_ops: the 8-bit cache's and the draft
// verification's calls straight from torch tensors.
//
// A call of these operators takes up to fifteen tensors; reading their shapes,
// types and addresses one attribute at a time from Python costs about 20 us, four
// times what the launch itself does.  Each function here checks the usual case
// (the types, shapes, strides and devices that need no copy), allocates the
// outputs through torch, finds the workspace of the current stream and calls the
// C entry point.  Anything else -- a malformed argument, rows that need a copy,
// another device than the current one, a workspace that does not exist yet, a
// stream under capture (its graph's workspace is its own) --
// returns None with nothing done, and the Python wrapper (kv8.py,
// speculative.py), which knows every rule and message, takes the call.  A status
// other than 0 of the entry point is returned as an int.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <map>
#include <utility>

#include "../../include/lvb200.h"

namespace {

decltype(&lvb_kv8_append_strided) g_append;
decltype(&lvb_kv8_read_blocks) g_read;
decltype(&lvb_kv8_attention_strided) g_attention;
decltype(&lvb_kv8_attention_workspace_bytes) g_attention_bytes;
decltype(&lvb_verify_drafts) g_verify;
decltype(&lvb_verify_drafts_workspace_bytes) g_verify_bytes;
decltype(&lvb_stream_capture_id) g_capture;

// Scratch of each (operator, device, stream), given by the Python side, which keeps it alive.
struct Scratch {
  void *ptr;
  size_t bytes;
};
std::map<std::pair<int, std::pair<int, uintptr_t>>, Scratch> g_scratch;
enum { kAttentionScratch = 0, kVerifyScratch = 1 };

bool scratch(int op, int device, cudaStream_t stream, size_t need, Scratch &out) {
  out = {nullptr, 0};
  if (need == 0) return true;
  if (g_capture(reinterpret_cast<lvb_stream_t>(stream)) != 0) return false;
  const auto it = g_scratch.find({op, {device, reinterpret_cast<uintptr_t>(stream)}});
  if (it == g_scratch.end() || it->second.bytes < need) return false;
  out = it->second;
  return true;
}

const at::Tensor *tensor(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool i32(const at::Tensor &t, int device) {
  return t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == device && t.is_contiguous();
}

template <typename T>
T *data(const at::Tensor &t) {
  return static_cast<T *>(t.data_ptr());
}

// One layer of the cache.
struct Layer {
  const at::Tensor *t[4];
  int64_t blocks, hkv, bs, d;
  int code, device;
};

bool layer(PyObject *const *args, Layer &l) {
  for (int i = 0; i < 4; ++i)
    if (!(l.t[i] = tensor(args[i]))) return false;
  const at::Tensor &k = *l.t[0], &v = *l.t[1];
  if (!k.is_cuda() || k.dim() != 4 || v.scalar_type() != k.scalar_type() || v.sizes() != k.sizes()) return false;
  if (k.scalar_type() == at::kChar)
    l.code = LVB_KV8_INT8;
  else if (k.scalar_type() == at::kFloat8_e4m3fn)
    l.code = LVB_KV8_E4M3;
  else
    return false;
  l.device = k.get_device();
  l.blocks = k.size(0), l.hkv = k.size(1), l.bs = k.size(2), l.d = k.size(3);
  for (int i = 0; i < 4; ++i)
    if (!l.t[i]->is_cuda() || l.t[i]->get_device() != l.device || !l.t[i]->is_contiguous()) return false;
  for (int i = 2; i < 4; ++i)
    if (l.t[i]->scalar_type() != at::kFloat || l.t[i]->dim() != 2 || l.t[i]->size(0) != l.blocks || l.t[i]->size(1) != l.hkv)
      return false;
  return l.device == c10::cuda::current_device();
}

// The step's metadata: tables, computed, query_start, max_query_len, max_seq_len.
struct Step {
  const at::Tensor *tables, *computed, *start;
  int64_t n, max_query, max_seq;
};

bool whole(PyObject *o, int64_t &v) {
  if (!PyLong_Check(o)) return false;
  v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return true;
}

bool step(PyObject *const *args, int device, Step &s) {
  s.tables = tensor(args[0]), s.computed = tensor(args[1]), s.start = tensor(args[2]);
  if (!s.tables || !s.computed || !s.start || !i32(*s.computed, device) || !i32(*s.start, device)) return false;
  const at::Tensor &t = *s.tables;
  if (t.scalar_type() != at::kInt || !t.is_cuda() || t.get_device() != device || t.dim() != 2 || s.computed->dim() != 1 ||
      s.start->dim() != 1)
    return false;
  s.n = s.computed->size(0);
  return s.n > 0 && t.size(0) == s.n && s.start->size(0) == s.n + 1 && (t.size(1) <= 1 || t.stride(1) == 1) &&
         whole(args[3], s.max_query) && whole(args[4], s.max_seq);
}

// [tokens, heads, d] rows of the model's type with dense heads.
bool rows(const at::Tensor *t, int64_t tokens, int64_t heads, int64_t d, at::ScalarType type, int device) {
  if (!t || t->dim() != 3 || t->scalar_type() != type || !t->is_cuda() || t->get_device() != device) return false;
  if (t->size(0) != tokens || (heads >= 0 && t->size(1) != heads) || t->size(2) != d) return false;
  return t->stride(2) == 1 && (t->size(1) <= 1 || t->stride(1) == d) && (tokens == 1 || t->stride(0) >= t->size(1) * d);
}

// Elements from token to token; a single one's stride means nothing.
int64_t token_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); }

// A new tensor on the current device, from torch's caching allocator without
// the dispatcher (about 1 us less than at::empty).
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type) {
  return at::Tensor(at::detail::empty_generic(size, c10::cuda::CUDACachingAllocator::get(),
                                              c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt));
}

// Whether rows may be read and written 16 bytes at a time.
bool aligned(const at::Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && token_stride(t) % 8 == 0; }

int act_of(const at::Tensor &t) {
  return t.scalar_type() == at::kHalf ? LVB_DTYPE_F16 : t.scalar_type() == at::kBFloat16 ? LVB_DTYPE_BF16 : -1;
}

lvb_stream_t handle(cudaStream_t s) { return reinterpret_cast<lvb_stream_t>(s); }

PyObject *status_or(int status, const at::Tensor &out) {
  return status == LVB_OK ? THPVariable_Wrap(out) : PyLong_FromLong(status);
}

PyObject *pair_or(int status, const at::Tensor &a, const at::Tensor &b) {
  if (status != LVB_OK) return PyLong_FromLong(status);
  PyObject *x = THPVariable_Wrap(a), *y = x ? THPVariable_Wrap(b) : nullptr;
  PyObject *both = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return both;
}

// kv8_attention(query, keys, values, key_scales, value_scales, tables,
// computed, query_start, max_query_len, max_seq_len, scale, out)
PyObject *attention(PyObject *const *args) {
  Layer l;
  Step s;
  const at::Tensor *q = tensor(args[0]);
  if (!q || q->dim() != 3 || !layer(args + 1, l) || !step(args + 5, l.device, s)) Py_RETURN_NONE;
  const int act = act_of(*q);
  const int64_t tokens = q->size(0), hq = q->size(1);
  if (act < 0 || tokens == 0 || hq == 0 || l.hkv == 0 || hq % l.hkv || !rows(q, tokens, hq, l.d, q->scalar_type(), l.device) ||
      !aligned(*q))
    Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(args[10]);
  if (scale == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  const at::Tensor *given = args[11] == Py_None ? nullptr : tensor(args[11]);
  if (args[11] != Py_None && (!rows(given, tokens, hq, l.d, q->scalar_type(), l.device) || !aligned(*given))) Py_RETURN_NONE;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(l.device)).stream();
  Scratch ws;
  if (!scratch(kAttentionScratch, l.device, stream, g_attention_bytes(s.n, hq, l.hkv, l.d, s.max_query, s.max_seq), ws))
    Py_RETURN_NONE;
  const at::Tensor out = given ? *given : fresh({tokens, hq, l.d}, q->scalar_type());
  const int status = g_attention(
      data<uint16_t>(*q), token_stride(*q), data<void>(*l.t[0]), data<void>(*l.t[1]), data<float>(*l.t[2]),
      data<float>(*l.t[3]), data<uint16_t>(out), token_stride(out), data<int32_t>(*s.tables), s.tables->size(1), s.tables->stride(0),
      data<int32_t>(*s.computed), data<int32_t>(*s.start), s.n, tokens, s.max_query, s.max_seq, hq, l.hkv, l.d, l.bs,
      l.blocks, static_cast<float>(scale), act, l.code, ws.ptr, ws.bytes, handle(stream));
  if (status == LVB_OK && given) {
    Py_INCREF(args[11]);
    return args[11];
  }
  return status_or(status, out);
}

// kv8_append(query, key, value, keys, values, key_scales, value_scales,
// tables, computed, query_start, max_query_len, max_seq_len, positions, cos,
// sin, query_out)
PyObject *append(PyObject *const *args) {
  Layer l;
  Step s;
  const at::Tensor *key = tensor(args[1]), *value = tensor(args[2]), *query = nullptr, *given = nullptr;
  if (!key || key->dim() != 3 || !layer(args + 3, l) || !step(args + 7, l.device, s)) Py_RETURN_NONE;
  const int act = act_of(*key);
  const int64_t tokens = key->size(0);
  const at::ScalarType type = key->scalar_type();
  if (act < 0 || tokens == 0 || !rows(key, tokens, l.hkv, l.d, type, l.device) ||
      !rows(value, tokens, l.hkv, l.d, type, l.device))
    Py_RETURN_NONE;
  const at::Tensor *pos = nullptr, *cos = nullptr, *sin = nullptr;
  if (args[12] != Py_None) {
    pos = tensor(args[12]), cos = tensor(args[13]), sin = tensor(args[14]);
    if (!pos || !cos || !sin || !i32(*pos, l.device) || pos->dim() != 1 || pos->size(0) != tokens || cos->dim() != 2 ||
        cos->size(1) != l.d || cos->sizes() != sin->sizes())
      Py_RETURN_NONE;
    for (const at::Tensor *t : {cos, sin})
      if (t->scalar_type() != type || !t->is_cuda() || t->get_device() != l.device || !t->is_contiguous()) Py_RETURN_NONE;
  }
  int64_t hq = 0;
  if (args[0] != Py_None) {
    query = tensor(args[0]);
    if (!query || query->dim() != 3 || !pos || query->size(1) == 0) Py_RETURN_NONE;
    hq = query->size(1);
    if (!rows(query, tokens, hq, l.d, type, l.device)) Py_RETURN_NONE;
    if (args[15] != Py_None && !rows(given = tensor(args[15]), tokens, hq, l.d, type, l.device)) Py_RETURN_NONE;
  } else if (args[15] != Py_None) {
    Py_RETURN_NONE;
  }
  at::Tensor out;
  if (query) out = given ? *given : fresh({tokens, hq, l.d}, type);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(l.device)).stream();
  const int status = g_append(
      query ? data<uint16_t>(*query) : nullptr, query ? token_stride(*query) : 0, query ? data<uint16_t>(out) : nullptr,
      query ? token_stride(out) : 0, data<uint16_t>(*key), token_stride(*key), data<uint16_t>(*value), token_stride(*value),
      pos ? data<int32_t>(*pos) : nullptr, cos ? data<uint16_t>(*cos) : nullptr, sin ? data<uint16_t>(*sin) : nullptr,
      cos ? cos->size(0) : 0, data<void>(*l.t[0]), data<void>(*l.t[1]), data<float>(*l.t[2]), data<float>(*l.t[3]),
      data<int32_t>(*s.tables), s.tables->size(1), s.tables->stride(0), data<int32_t>(*s.computed), data<int32_t>(*s.start), s.n, tokens,
      s.max_query, hq, l.hkv, l.d, l.bs, l.blocks, act, l.code, handle(stream));
  if (status != LVB_OK) return PyLong_FromLong(status);
  if (given) {
    Py_INCREF(args[15]);
    return args[15];
  }
  if (query) return THPVariable_Wrap(out);
  Py_RETURN_TRUE;  // done, nothing to return
}

// kv8_read_blocks(keys, values, key_scales, value_scales, ids, bf16)
PyObject *read_blocks(PyObject *const *args) {
  Layer l;
  const at::Tensor *ids = tensor(args[4]);
  if (!layer(args, l) || !ids || !i32(*ids, l.device) || ids->dim() != 1 || ids->size(0) == 0) Py_RETURN_NONE;
  const bool bf16 = args[5] == Py_True;
  const int64_t n = ids->size(0);
  const at::ScalarType type = bf16 ? at::kBFloat16 : at::kHalf;
  const at::Tensor keys = fresh({n, l.hkv, l.bs, l.d}, type), values = fresh({n, l.hkv, l.bs, l.d}, type);
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(l.device)).stream();
  const int status = g_read(data<void>(*l.t[0]), data<void>(*l.t[1]), data<float>(*l.t[2]), data<float>(*l.t[3]),
                            data<int32_t>(*ids), n, data<uint16_t>(keys), data<uint16_t>(values), l.hkv, l.d, l.bs,
                            l.blocks, bf16 ? LVB_DTYPE_BF16 : LVB_DTYPE_F16, l.code, handle(stream));
  return pair_or(status, keys, values);
}

bool probs(const at::Tensor *t, int64_t n, int64_t vocab, int device) {
  return t && t->dim() == 2 && t->scalar_type() == at::kFloat && t->is_cuda() && t->get_device() == device &&
         t->size(0) == n && t->size(1) == vocab && t->stride(1) == 1 && (n <= 1 || t->stride(0) >= vocab);
}

bool vec(const at::Tensor *t, at::ScalarType type, int64_t n, int device) {
  return t && t->dim() == 1 && t->scalar_type() == type && t->is_cuda() && t->get_device() == device && t->size(0) == n &&
         t->is_contiguous();
}

// verify_drafts(target_probs, draft_tokens, accept_uniform, sample_uniform,
// query_start, max_query_len, draft_probs)
PyObject *verify(PyObject *const *args) {
  const at::Tensor *target = tensor(args[0]), *tokens = tensor(args[1]), *accept = tensor(args[2]), *sample = tensor(args[3]),
                   *start = tensor(args[4]), *draft = nullptr;
  int64_t width;
  if (!target || target->dim() != 2 || !target->is_cuda() || !tokens || tokens->dim() != 1 || !start || start->dim() != 1 ||
      start->size(0) < 2 || !whole(args[5], width) || width < 0)
    Py_RETURN_NONE;
  const int device = target->get_device();
  const int64_t rows = target->size(0), vocab = target->size(1), n = start->size(0) - 1, drafts = tokens->size(0);
  if (device != c10::cuda::current_device() || vocab == 0 || rows != drafts + n || !probs(target, rows, vocab, device) ||
      !vec(tokens, at::kLong, drafts, device) || !vec(accept, at::kFloat, drafts, device) ||
      !vec(sample, at::kFloat, n, device) || !vec(start, at::kInt, n + 1, device))
    Py_RETURN_NONE;
  if (args[6] != Py_None && !probs(draft = tensor(args[6]), drafts, vocab, device)) Py_RETURN_NONE;
  const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
  Scratch ws;
  if (!scratch(kVerifyScratch, device, stream, g_verify_bytes(n, vocab), ws)) Py_RETURN_NONE;
  const at::Tensor out = fresh({n, width}, at::kLong), accepted = fresh({n}, at::kInt);
  const bool use = draft && drafts > 0;
  const int status = g_verify(data<float>(*target), rows > 1 ? target->stride(0) : vocab, use ? data<float>(*draft) : nullptr,
                              use ? (drafts > 1 ? draft->stride(0) : vocab) : 0, data<int64_t>(*tokens),
                              data<float>(*accept), data<float>(*sample), data<int32_t>(*start), data<int64_t>(out),
                              data<int32_t>(accepted), n, rows, width, vocab, ws.ptr, ws.bytes, handle(stream));
  return pair_or(status, out, accepted);
}

template <PyObject *(*F)(PyObject *const *), int kArgs>
PyObject *entry(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", kArgs, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// bind(append, read_blocks, attention, attention_bytes, verify, verify_bytes, capture): library entry points
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long p[7];
  if (!PyArg_ParseTuple(args, "KKKKKKK", p, p + 1, p + 2, p + 3, p + 4, p + 5, p + 6)) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(p[0]);
  g_read = reinterpret_cast<decltype(g_read)>(p[1]);
  g_attention = reinterpret_cast<decltype(g_attention)>(p[2]);
  g_attention_bytes = reinterpret_cast<decltype(g_attention_bytes)>(p[3]);
  g_verify = reinterpret_cast<decltype(g_verify)>(p[4]);
  g_verify_bytes = reinterpret_cast<decltype(g_verify_bytes)>(p[5]);
  g_capture = reinterpret_cast<decltype(g_capture)>(p[6]);
  Py_RETURN_NONE;
}

// set_scratch(op, device, stream, address, bytes)
PyObject *set_scratch(PyObject *, PyObject *args) {
  int op, device;
  unsigned long long stream, ptr;
  Py_ssize_t bytes;
  if (!PyArg_ParseTuple(args, "iiKKn", &op, &device, &stream, &ptr, &bytes)) return nullptr;
  try {
    g_scratch[{op, {device, static_cast<uintptr_t>(stream)}}] = {reinterpret_cast<void *>(static_cast<uintptr_t>(ptr)),
                                                                static_cast<size_t>(bytes)};
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
  Py_RETURN_NONE;
}

template <PyObject *(*F)(PyObject *const *), int kArgs>
PyMethodDef method(const char *name, const char *doc) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(&entry<F, kArgs>)), METH_FASTCALL, doc};
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, "library entry points"},
    {"set_scratch", set_scratch, METH_VARARGS, "set_scratch(op, device, stream, address, bytes)"},
    method<attention, 12>("kv8_attention", "output, None (not the usual case) or a status"),
    method<append, 16>("kv8_append", "rotated queries or True, None (not the usual case) or a status"),
    method<read_blocks, 6>("kv8_read_blocks", "(keys, values), None or a status"),
    method<verify, 7>("verify_drafts", "(tokens, accepted), None or a status"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", "Operator calls straight from torch tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&module); }
