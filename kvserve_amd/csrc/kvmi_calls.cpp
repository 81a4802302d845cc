// Python entry to the decode-instance operators for calls that are not checked: the arguments
// are taken apart here instead of in Python (4 us a call instead of 13, where the kernels
// themselves take 3 to 10).
//
// Each function returns True if the call was enqueued.  It returns False, with nothing done, for
// every argument that is not plainly right: the caller's own checks then name the mistake, or
// serve what is rare (a current device that is not the tensors', a query to be copied).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

#include "../../include/kvserve_amd.h"

namespace {

// What a call has gathered: the device that all its tensors must be on.
struct Args {
  c10::Device device{c10::DeviceType::CPU};
  bool ok = true;

  const at::Tensor* any(PyObject* o) {
    if (!THPVariable_Check(o)) {
      ok = false;
      return nullptr;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) ok = false;
    if (device.type() == c10::DeviceType::CPU)
      device = t.device();
    else if (t.device() != device)
      ok = false;
    return ok ? &t : nullptr;
  }
  // A contiguous tensor of this type; sizes of -1 are any.
  template <class T>
  T* flat(PyObject* o, at::ScalarType type, int64_t n0, int64_t n1 = -2) {
    const at::Tensor* t = any(o);
    if (!t) return nullptr;
    const int64_t dim = n1 == -2 ? 1 : 2;
    if (t->scalar_type() != type || t->dim() != dim || !t->is_contiguous() || (n0 >= 0 && t->size(0) != n0) ||
        (dim == 2 && n1 >= 0 && t->size(1) != n1)) {
      ok = false;
      return nullptr;
    }
    return static_cast<T*>(t->data_ptr());
  }
  int32_t* err(PyObject* o) { return o == Py_None ? nullptr : flat<int32_t>(o, at::kInt, 1); }
  bool integer(PyObject* o, int32_t* to) {
    if (!PyLong_CheckExact(o)) return ok = false;
    int over = 0;
    const long v = PyLong_AsLongAndOverflow(o, &over);
    if (over || v < 0 || v > 0x7fffffffL) return ok = false;
    *to = (int32_t)v;
    return true;
  }
  // Cache [2, P, S, H, D] or [P, 2, S, H, D].
  at::ScalarType cache(PyObject* o, kvmi_cache* c) {
    const at::Tensor* t = any(o);
    if (!t || t->dim() != 5 || t->element_size() != 2 || !t->is_contiguous() || t->numel() == 0 ||
        (t->size(0) != 2 && t->size(1) != 2)) {
      ok = false;
      return at::kByte;
    }
    const int64_t S = t->size(2), H = t->size(3), D = t->size(4), row = S * H * D;
    const bool first = t->size(0) == 2;
    const int64_t blocks = first ? t->size(1) : t->size(0);
    if (blocks > 0x7fffffff || row > 0x7fffffff) ok = false;
    *c = kvmi_cache{t->data_ptr(), first ? blocks * row : row, first ? row : 2 * row, (int32_t)blocks, (int32_t)S,
                    (int32_t)H,    (int32_t)D};
    return t->scalar_type();
  }
  // The current stream of the tensors' device, if that is the current device.
  bool stream(kvmi_stream_t* s) {
    int current = -1;
    if (!ok || hipGetDevice(&current) != hipSuccess || current != device.index()) return false;
    *s = c10::hip::getCurrentHIPStream(device.index()).stream();
    return true;
  }
};

PyObject* answer(bool done) { return PyBool_FromLong(done); }

// Other threads run while a call is enqueued (it waits where the stream is full).
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
template <class F>
PyObject* enqueue(F f) {
  int rc;
  {
    Unlocked unlocked;
    rc = f();
  }
  return answer(rc == KVMI_OK);
}

// write_kv(key, value, cache, slots, err)
PyObject* write_kv(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 5) return answer(false);
  Args a;
  kvmi_cache c;
  const at::ScalarType type = a.cache(in[2], &c);
  const at::Tensor *k = a.any(in[0]), *v = a.any(in[1]);
  if (!a.ok) return answer(false);
  for (const at::Tensor* t : {k, v})
    if (t->scalar_type() != type || t->dim() != 3 || t->size(0) != k->size(0) || t->size(1) != c.num_heads ||
        t->size(2) != c.head_dim || t->stride(2) != 1)
      return answer(false);
  const int64_t tokens = k->size(0);
  const int64_t* slots = a.flat<int64_t>(in[3], at::kLong, tokens);
  int32_t* err = a.err(in[4]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  return enqueue([&] {
    return kvmi_write_kv(&c, k->data_ptr(), v->data_ptr(), k->stride(0), k->stride(1), v->stride(0), v->stride(1),
                         slots, tokens, err, st);
  });
} catch (...) {
  return answer(false);
}

// build_block_tables(lengths, new_lengths, tables, free, state, block_size, max_tokens, out, ticket, err),
// `out` a tuple of tables, lengths, state, slots, starts
PyObject* build_block_tables(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 10 || !PyTuple_Check(in[7]) || PyTuple_GET_SIZE(in[7]) != 5) return answer(false);
  Args a;
  kvmi_tables_args t;
  std::memset(&t, 0, sizeof(t));
  a.integer(in[5], &t.block_size);
  a.integer(in[6], &t.max_tokens);
  const at::Tensor *now = a.any(in[0]), *tables = a.any(in[2]), *ring = a.any(in[3]);
  if (!a.ok || tables->dim() != 2) return answer(false);
  const int64_t R = now->numel(), C = tables->size(1), N = ring->numel();
  if (R < 1 || R > 0x7fffffff || C > 0x7fffffff || N > 0x7fffffff) return answer(false);
  t.requests = (int32_t)R;
  t.columns = (int32_t)C;
  t.ring = (int32_t)N;
  t.lengths = a.flat<int32_t>(in[0], at::kInt, R);
  t.new_lengths = a.flat<int32_t>(in[1], at::kInt, R);
  t.tables = a.flat<int32_t>(in[2], at::kInt, R, C);
  t.free_blocks = a.flat<int32_t>(in[3], at::kInt, N);
  t.state = a.flat<int32_t>(in[4], at::kInt, 2);
  PyObject* const out = in[7];
  t.out_tables = a.flat<int32_t>(PyTuple_GET_ITEM(out, 0), at::kInt, R, C);
  t.out_lengths = a.flat<int32_t>(PyTuple_GET_ITEM(out, 1), at::kInt, R);
  t.out_state = a.flat<int32_t>(PyTuple_GET_ITEM(out, 2), at::kInt, 2);
  t.slots = a.flat<int64_t>(PyTuple_GET_ITEM(out, 3), at::kLong, t.max_tokens);
  t.starts = a.flat<int32_t>(PyTuple_GET_ITEM(out, 4), at::kInt, R + 1);
  t.ticket = in[8] == Py_None ? nullptr : a.flat<int32_t>(in[8], at::kInt, 1);
  t.err = a.err(in[9]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  return enqueue([&] { return kvmi_build_tables(&t, st); });
} catch (...) {
  return answer(false);
}

// tree_attention(query, cache, tables, lengths, starts, max_query, max_length, mask, scale, out, err)
PyObject* tree_attention(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 11) return answer(false);
  Args a;
  kvmi_attention_args t;
  std::memset(&t, 0, sizeof(t));
  const at::ScalarType type = a.cache(in[1], &t.cache);
  const at::Tensor *q = a.any(in[0]), *out = a.any(in[9]), *lengths = a.any(in[3]), *tables = a.any(in[2]);
  if (!a.ok || (type != at::kBFloat16 && type != at::kHalf) || q->scalar_type() != type || q->dim() != 3 ||
      q->size(2) != t.cache.head_dim || q->stride(2) != 1 || out->scalar_type() != type || !out->is_contiguous() ||
      out->sizes() != q->sizes() || tables->dim() != 2)
    return answer(false);
  const int64_t tokens = q->size(0), heads = q->size(1), R = lengths->numel(), C = tables->size(1);
  if (tokens < 1 || tokens > 0x7fffffff || heads > 0x7fffffff || R < 1 || R > 0x7fffffff || C > 0x7fffffff)
    return answer(false);
  t.dtype = type == at::kHalf ? KVMI_DTYPE_FP16 : KVMI_DTYPE_BF16;
  t.requests = (int32_t)R;
  t.columns = (int32_t)C;
  t.total_queries = (int32_t)tokens;
  t.query_heads = (int32_t)heads;
  t.query = q->data_ptr();
  t.out = out->data_ptr();
  t.query_token_stride = q->stride(0);
  t.query_head_stride = q->stride(1);
  t.tables = a.flat<int32_t>(in[2], at::kInt, R, C);
  t.lengths = a.flat<int32_t>(in[3], at::kInt, R);
  t.starts = a.flat<int32_t>(in[4], at::kInt, R + 1);
  if (!a.integer(in[5], &t.max_query)) return answer(false);
  if (t.max_query > t.total_queries) t.max_query = t.total_queries;
  if (in[6] == Py_None) {
    const int64_t most = C * t.cache.block_size;
    t.max_length = most > 0x7fffffff ? 0x7fffffff : (int32_t)most;
  } else if (!a.integer(in[6], &t.max_length)) {
    return answer(false);
  }
  if (in[7] != Py_None) {
    t.mask = a.flat<uint64_t>(in[7], at::kLong, tokens, -1);
    if (!a.ok) return answer(false);
    const int64_t words = THPVariable_Unpack(in[7]).size(1);
    if (words > 0x7fffffff || words * 64 < t.max_query) return answer(false);
    t.mask_words = (int32_t)words;
  }
  if (in[8] == Py_None)
    t.scale = (float)(1.0 / std::sqrt((double)t.cache.head_dim));
  else if (PyFloat_CheckExact(in[8]))
    t.scale = (float)PyFloat_AS_DOUBLE(in[8]);
  else
    return answer(false);
  t.err = a.err(in[10]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  const int64_t space = kvmi_attention_workspace_bytes(&t);
  if (space < 0) return answer(false);
  at::Tensor parts;
  if (space) {
    parts = at::empty({space}, q->options().dtype(at::kByte).requires_grad(false));
    t.workspace = parts.data_ptr();
    t.workspace_bytes = space;
  }
  return enqueue([&] { return kvmi_tree_attention(&t, st); });
} catch (...) {
  return answer(false);
}

// keep_drafts(cache struct's address, bases, tables, lengths, accepted, out, err)
PyObject* keep_drafts(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 7 || !PyLong_CheckExact(in[0])) return answer(false);
  const kvmi_cache* c = static_cast<const kvmi_cache*>(PyLong_AsVoidPtr(in[0]));
  if (!c) {
    PyErr_Clear();
    return answer(false);
  }
  Args a;
  const at::Tensor *bases = a.any(in[1]), *lengths = a.any(in[3]), *tables = a.any(in[2]), *path = a.any(in[4]);
  if (!a.ok || tables->dim() != 2 || path->dim() != 2) return answer(false);
  const int64_t R = lengths->numel(), C = tables->size(1), W = path->size(1), L = bases->numel();
  if (R < 1 || R > 0x7fffffff || C > 0x7fffffff || W > 1024 || L > 65535) return answer(false);
  const int64_t* at_bases = a.flat<int64_t>(in[1], at::kLong, L);
  const int32_t* tab = a.flat<int32_t>(in[2], at::kInt, R, C);
  const int32_t* now = a.flat<int32_t>(in[3], at::kInt, R);
  const int32_t* acc = a.flat<int32_t>(in[4], at::kInt, R, W);
  int32_t* out = a.flat<int32_t>(in[5], at::kInt, R);
  int32_t* err = a.err(in[6]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  return enqueue([&] {
    return kvmi_keep_drafts(c, (void* const*)at_bases, (int32_t)L, tab, (int32_t)C, now, acc, (int32_t)R, (int32_t)W,
                            out, err, st);
  });
} catch (...) {
  return answer(false);
}

// fork_block_tables(lengths, parents, new_lengths, tables, shares, free, state, block_size, max_tokens, out,
// workspace, err), `out` a tuple of tables, lengths, shares, state, slots, starts, copies
PyObject* fork_block_tables(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 12 || !PyTuple_Check(in[9]) || PyTuple_GET_SIZE(in[9]) != 7) return answer(false);
  Args a;
  kvmi_fork_args t;
  std::memset(&t, 0, sizeof(t));
  a.integer(in[7], &t.block_size);
  a.integer(in[8], &t.max_tokens);
  const at::Tensor *now = a.any(in[0]), *tables = a.any(in[3]), *shares = a.any(in[4]), *space = a.any(in[10]);
  if (!a.ok || tables->dim() != 2) return answer(false);
  const int64_t R = now->numel(), C = tables->size(1), N = shares->numel();
  if (R < 1 || R > 0x7fffffff || C > 0x7fffffff || N > 0x7fffffff) return answer(false);
  t.rows = (int32_t)R;
  t.columns = (int32_t)C;
  t.blocks = (int32_t)N;
  t.lengths = a.flat<int32_t>(in[0], at::kInt, R);
  if (in[1] != Py_None) t.parents = a.flat<int32_t>(in[1], at::kInt, R);
  if (PyLong_CheckExact(in[2]))
    a.integer(in[2], &t.grow);
  else
    t.new_lengths = a.flat<int32_t>(in[2], at::kInt, R);
  t.tables = a.flat<int32_t>(in[3], at::kInt, R, C);
  t.shares = a.flat<int32_t>(in[4], at::kInt, N);
  t.free_blocks = a.flat<int32_t>(in[5], at::kInt, N);
  t.state = a.flat<int32_t>(in[6], at::kInt, 2);
  PyObject* const out = in[9];
  t.out_tables = a.flat<int32_t>(PyTuple_GET_ITEM(out, 0), at::kInt, R, C);
  t.out_lengths = a.flat<int32_t>(PyTuple_GET_ITEM(out, 1), at::kInt, R);
  t.out_shares = a.flat<int32_t>(PyTuple_GET_ITEM(out, 2), at::kInt, N);
  t.out_state = a.flat<int32_t>(PyTuple_GET_ITEM(out, 3), at::kInt, 2);
  t.slots = a.flat<int64_t>(PyTuple_GET_ITEM(out, 4), at::kLong, t.max_tokens);
  t.starts = a.flat<int32_t>(PyTuple_GET_ITEM(out, 5), at::kInt, R + 1);
  t.copies = a.flat<int32_t>(PyTuple_GET_ITEM(out, 6), at::kInt, R, 3);
  t.workspace = a.flat<int32_t>(in[10], at::kInt, -1);
  t.workspace_bytes = space->numel() * 4;
  t.err = a.err(in[11]);
  kvmi_stream_t st;
  if (!a.stream(&st) || kvmi_fork_workspace_bytes(t.blocks, t.rows, t.columns) != t.workspace_bytes) return answer(false);
  return enqueue([&] { return kvmi_fork_tables(&t, st); });
} catch (...) {
  return answer(false);
}

// copy_blocks(cache struct's address, bases, copies, err)
PyObject* copy_blocks(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 4 || !PyLong_CheckExact(in[0])) return answer(false);
  const kvmi_cache* c = static_cast<const kvmi_cache*>(PyLong_AsVoidPtr(in[0]));
  if (!c) {
    PyErr_Clear();
    return answer(false);
  }
  Args a;
  const at::Tensor *bases = a.any(in[1]), *copies = a.any(in[2]);
  if (!a.ok || copies->dim() != 2) return answer(false);
  const int64_t L = bases->numel(), rows = copies->size(0);
  if (L > 32767 || rows < 1 || rows > 0x7fffffff) return answer(false);
  const int64_t* at_bases = a.flat<int64_t>(in[1], at::kLong, L);
  const int32_t* list = a.flat<int32_t>(in[2], at::kInt, rows, 3);
  int32_t* err = a.err(in[3]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  return enqueue([&] { return kvmi_copy_blocks(c, (void* const*)at_bases, (int32_t)L, list, (int32_t)rows, err, st); });
} catch (...) {
  return answer(false);
}

// compact_block_tables(lengths, tables, shares, free, state, block_size, out, workspace, err), `out` a
// tuple of tables, shares, free, state, copies
PyObject* compact_block_tables(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 9 || !PyTuple_Check(in[6]) || PyTuple_GET_SIZE(in[6]) != 5) return answer(false);
  Args a;
  kvmi_compact_args t;
  std::memset(&t, 0, sizeof(t));
  a.integer(in[5], &t.block_size);
  const at::Tensor *now = a.any(in[0]), *tables = a.any(in[1]), *shares = a.any(in[2]), *space = a.any(in[7]);
  if (!a.ok || tables->dim() != 2) return answer(false);
  const int64_t R = now->numel(), C = tables->size(1), N = shares->numel();
  if (R < 1 || R > 0x7fffffff || C > 0x7fffffff || N < 1 || N > 0x7fffffff) return answer(false);
  t.rows = (int32_t)R;
  t.columns = (int32_t)C;
  t.blocks = (int32_t)N;
  t.lengths = a.flat<int32_t>(in[0], at::kInt, R);
  t.tables = a.flat<int32_t>(in[1], at::kInt, R, C);
  t.shares = a.flat<int32_t>(in[2], at::kInt, N);
  t.free_blocks = a.flat<int32_t>(in[3], at::kInt, N);
  t.state = a.flat<int32_t>(in[4], at::kInt, 2);
  PyObject* const out = in[6];
  t.out_tables = a.flat<int32_t>(PyTuple_GET_ITEM(out, 0), at::kInt, R, C);
  t.out_shares = a.flat<int32_t>(PyTuple_GET_ITEM(out, 1), at::kInt, N);
  t.out_free = a.flat<int32_t>(PyTuple_GET_ITEM(out, 2), at::kInt, N);
  t.out_state = a.flat<int32_t>(PyTuple_GET_ITEM(out, 3), at::kInt, 2);
  t.copies = a.flat<int32_t>(PyTuple_GET_ITEM(out, 4), at::kInt, N / 2, 3);
  t.workspace = a.flat<int32_t>(in[7], at::kInt, -1);
  t.workspace_bytes = space->numel() * 4;
  t.err = a.err(in[8]);
  kvmi_stream_t st;
  if (!a.stream(&st) || kvmi_compact_workspace_bytes(t.blocks) != t.workspace_bytes) return answer(false);
  return enqueue([&] { return kvmi_compact_tables(&t, st); });
} catch (...) {
  return answer(false);
}

// select_beams(logits, scores, beams, count, end_token, out, err), `out` a tuple of parents, tokens,
// scores, all_parents, all_tokens, all_scores
PyObject* select_beams(PyObject*, PyObject* const* in, Py_ssize_t n) try {
  if (n != 7 || !PyTuple_Check(in[5]) || PyTuple_GET_SIZE(in[5]) != 6) return answer(false);
  Args a;
  kvmi_select_args t;
  std::memset(&t, 0, sizeof(t));
  a.integer(in[2], &t.beams);
  a.integer(in[3], &t.count);
  t.end_token = -1;
  if (in[4] != Py_None) a.integer(in[4], &t.end_token);
  const at::Tensor* logits = a.any(in[0]);
  if (!a.ok || t.beams < 1 || logits->dim() != 2) return answer(false);
  const int64_t rows = logits->size(0), V = logits->size(1), R = rows / t.beams;
  if (rows < 1 || rows > 65535 || rows % t.beams || V < 1 || V > 0x7fffffff || (logits->stride(1) != 1 && V > 1))
    return answer(false);
  switch (logits->scalar_type()) {
    case at::kBFloat16: t.dtype = KVMI_DTYPE_BF16; break;
    case at::kHalf: t.dtype = KVMI_DTYPE_FP16; break;
    case at::kFloat: t.dtype = KVMI_DTYPE_FP32; break;
    default: return answer(false);
  }
  t.requests = (int32_t)R;
  t.vocab = (int32_t)V;
  t.logits = logits->data_ptr();
  t.row_stride = logits->stride(0);
  t.scores = a.flat<float>(in[1], at::kFloat, rows);
  PyObject* const out = in[5];
  t.parents = a.flat<int32_t>(PyTuple_GET_ITEM(out, 0), at::kInt, rows);
  t.tokens = a.flat<int32_t>(PyTuple_GET_ITEM(out, 1), at::kInt, rows);
  t.next_scores = a.flat<float>(PyTuple_GET_ITEM(out, 2), at::kFloat, rows);
  t.all_parents = a.flat<int32_t>(PyTuple_GET_ITEM(out, 3), at::kInt, R, t.count);
  t.all_tokens = a.flat<int32_t>(PyTuple_GET_ITEM(out, 4), at::kInt, R, t.count);
  t.all_scores = a.flat<float>(PyTuple_GET_ITEM(out, 5), at::kFloat, R, t.count);
  t.err = a.err(in[6]);
  kvmi_stream_t st;
  if (!a.stream(&st)) return answer(false);
  const int64_t space = kvmi_select_workspace_bytes(&t);
  if (space < 0) return answer(false);
  at::Tensor parts = at::empty({space}, logits->options().dtype(at::kByte).requires_grad(false));
  t.workspace = parts.data_ptr();
  t.workspace_bytes = space;
  return enqueue([&] { return kvmi_select_beams(&t, st); });
} catch (...) {
  return answer(false);
}

PyMethodDef kMethods[] = {
    {"write_kv", (PyCFunction)(void (*)(void))write_kv, METH_FASTCALL, nullptr},
    {"build_block_tables", (PyCFunction)(void (*)(void))build_block_tables, METH_FASTCALL, nullptr},
    {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
    {"keep_drafts", (PyCFunction)(void (*)(void))keep_drafts, METH_FASTCALL, nullptr},
    {"fork_block_tables", (PyCFunction)(void (*)(void))fork_block_tables, METH_FASTCALL, nullptr},
    {"copy_blocks", (PyCFunction)(void (*)(void))copy_blocks, METH_FASTCALL, nullptr},
    {"compact_block_tables", (PyCFunction)(void (*)(void))compact_block_tables, METH_FASTCALL, nullptr},
    {"select_beams", (PyCFunction)(void (*)(void))select_beams, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() { return PyModule_Create(&kModule); }
