// Calls of the operators around a step, checked and launched without Python's part of it: a small step's kernels take 3 to 8 us,
// and reading a dozen tensors' types, shapes, strides and addresses one Python attribute after another takes as long.
//
// Every function takes (device, stream, operands ...), returns True where the call was accepted and launched, and False where
// anything is not as it should be; the Python wrapper then looks for itself, says what it was and raises.  So the wrapper's
// checks are the ones that count, and what is accepted here is never more than what they accept.
//
// A Python extension module (host code; tensors are read through torch's own headers), bound to the entry points of the
// libraries by their addresses.

#include <ATen/ops/empty.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>

#include "fp4_attention_api.h"
#include "serving_api.h"

namespace {

using at::Tensor;
constexpr int64_t k31 = 0x7fffffff;

struct NotAccepted {};
void need(bool ok) {
  if (!ok) throw NotAccepted{};
}

const Tensor& tensor(PyObject* o) {
  need(THPVariable_Check(o));
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  need(PyLong_Check(o));
  int overflow = 0;
  const long long v = PyLong_AsLongLongAndOverflow(o, &overflow);
  need(overflow == 0);
  return v;
}
double real(PyObject* o) {
  need(PyFloat_CheckExact(o));
  return PyFloat_AS_DOUBLE(o);
}

int code_of(const Tensor& t) {  // the libraries' numbers of their types
  const auto type = t.scalar_type();
  need(type == at::kFloat || type == at::kBFloat16);
  return type == at::kFloat ? 0 : 1;
}
bool on(const Tensor& t, int device) { return t.is_cuda() && t.get_device() == device && t.layout() == at::kStrided; }

// A contiguous vector of `n` elements (any number: -1); its address.
template <typename T = int>
T* vector(const Tensor& t, int device, int64_t n, at::ScalarType type = at::kInt) {
  need(t.scalar_type() == type && on(t, device) && t.dim() == 1 && (n < 0 || t.size(0) == n) && t.size(0) <= k31 && t.is_contiguous());
  return static_cast<T*>(t.data_ptr());
}

// Bytes of memory: `rows` runs of `width` bytes, `stride` apart.
struct Area {
  uintptr_t lo;
  int64_t rows, width, stride;
  uintptr_t end() const { return lo + (uintptr_t)((rows - 1) * stride + width); }
};
Area area(const Tensor& t) { return {reinterpret_cast<uintptr_t>(t.data_ptr()), 1, t.numel() * (int64_t)t.element_size(), 0}; }
Area area(const Tensor& t, int64_t width) {  // the first `width` elements of every row
  const int64_t item = (int64_t)t.element_size();
  return {reinterpret_cast<uintptr_t>(t.data_ptr()), t.size(0), width * item, t.stride(0) * item};
}
// Whether two areas share a byte.  Windows of columns of one buffer, side by side, do not; rows of different strides that lie in
// one another's range count as if they did.
bool meet(const Area& a, const Area& b) {
  if (a.rows == 0 || b.rows == 0 || a.width == 0 || b.width == 0 || a.end() <= b.lo || b.end() <= a.lo) return false;
  if (a.stride == b.stride && a.rows > 1 && b.rows > 1 && a.stride > 0) {
    const int64_t apart = (int64_t)(b.lo - a.lo) % a.stride, offset = apart < 0 ? apart + a.stride : apart;
    return offset < a.width || offset + b.width > a.stride;
  }
  return true;
}

struct Bound {
  decltype(&ls_step_tables) step_tables;
  decltype(&ls_fp4_write) fp4_write;
  decltype(&ls_fp4_read) fp4_read;
  decltype(&ls_token_logprobs) token_logprobs;
  decltype(&ls_logprobs_scratch_bytes) logprobs_scratch;
  int64_t max_requests, max_top, max_vocab;
  PyTypeObject* pages;  // the type of a pool of pages in 4 bits
  struct {
    decltype(&ls_fp4_attention) run;
    decltype(&ls_fp4_attention_scratch_bytes) scratch;
  } attention[9];  // by head size / 32
} bound;

template <typename F>
void bind(F& to, PyObject* address) {
  to = reinterpret_cast<F>(integer(address));
}

// The body's calls and checks; whatever goes wrong is for Python to say.
template <typename F>
PyObject* accepted(Py_ssize_t given, Py_ssize_t wanted, F body) {
  bool ok = false;
  if (given == wanted) {
    try {
      ok = body() == 0;
    } catch (const NotAccepted&) {
    } catch (const std::exception&) {
    }
    PyErr_Clear();
  }
  return PyBool_FromLong(ok);
}
template <typename F>
int without_gil(F call) {
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = call();
  Py_END_ALLOW_THREADS
  return code;
}

PyObject* bind_serving(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return accepted(n, 9, [&] {
    need(PyType_Check(x[8]));
    bind(bound.step_tables, x[0]);
    bind(bound.fp4_write, x[1]);
    bind(bound.fp4_read, x[2]);
    bind(bound.token_logprobs, x[3]);
    bind(bound.logprobs_scratch, x[4]);
    bound.max_requests = integer(x[5]);
    bound.max_top = integer(x[6]);
    bound.max_vocab = integer(x[7]);
    Py_INCREF(x[8]);
    bound.pages = reinterpret_cast<PyTypeObject*>(x[8]);
    return 0;
  });
}

PyObject* bind_attention(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return accepted(n, 3, [&] {
    const int64_t d = integer(x[0]);
    need(d % 32 == 0 && d >= 32 && d <= 256);
    bind(bound.attention[d / 32].run, x[1]);
    bind(bound.attention[d / 32].scratch, x[2]);
    return 0;
  });
}

PyObject* step_tables(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return accepted(n, 14, [&] {
    need(bound.step_tables != nullptr);
    const int device = (int)integer(x[0]);
    void* stream = reinterpret_cast<void*>(integer(x[1]));
    const Tensor &lengths = tensor(x[2]), &table = tensor(x[4]), &slots = tensor(x[8]), &free_pages = tensor(x[6]);
    const int64_t requests = lengths.numel(), tokens = slots.numel(), page_size = integer(x[5]), free_count = free_pages.numel();
    need(requests <= bound.max_requests);
    struct Range {
      uintptr_t lo;
      int64_t bytes;
      bool output;
    } ranges[12];
    int used = 0;
    const auto taken = [&](PyObject* o, int64_t count, bool output) {
      const Tensor& t = tensor(o);
      int* p = vector(t, device, count);
      if (t.numel() > 0) ranges[used++] = {reinterpret_cast<uintptr_t>(p), 4 * t.numel(), output};
      return p;
    };
    const int* held = taken(x[2], requests, false);
    const int* news = taken(x[3], requests, false);
    const int* free_list = taken(x[6], -1, false);
    const int* cursor = taken(x[7], 1, false);
    int* slot = taken(x[8], tokens, true);
    int* tok_seq = taken(x[9], tokens, true);
    int* tok_pos = taken(x[10], tokens, true);
    int* offsets = taken(x[11], requests + 1, true);
    int* new_lengths = taken(x[12], requests, true);
    int* progress = taken(x[13], 2, true);
    need(table.scalar_type() == at::kInt && on(table, device) && table.dim() == 2 && table.size(0) == requests && table.size(1) >= 1 &&
         table.is_contiguous());
    const int64_t columns = table.size(1);
    need(page_size >= 4 && page_size <= k31 && (page_size & (page_size - 1)) == 0 && columns <= k31 / page_size);
    int* pages = static_cast<int*>(table.data_ptr());
    if (requests > 0) ranges[used++] = {reinterpret_cast<uintptr_t>(pages), 4 * requests * columns, true};
    // an output may lie in no other operand: in the order of their addresses each begins behind all before
    std::sort(ranges, ranges + used, [](const Range& a, const Range& b) {
      return a.lo != b.lo ? a.lo < b.lo : a.bytes != b.bytes ? a.bytes < b.bytes : a.output < b.output;
    });
    uintptr_t end = 0, written = 0;
    for (int i = 0; i < used; ++i) {
      need(ranges[i].lo >= (ranges[i].output ? end : written));
      end = std::max(end, ranges[i].lo + (uintptr_t)ranges[i].bytes);
      if (ranges[i].output) written = ranges[i].lo + (uintptr_t)ranges[i].bytes;
    }
    return without_gil([&] {
      return bound.step_tables(held, news, (int)requests, pages, (int)columns, (int)page_size, free_list, (int)free_count, cursor, slot,
                               tok_seq, tok_pos, (int)tokens, offsets, new_lengths, progress, stream);
    });
  });
}

struct Pool {  // a pool of pages in 4 bits, checked
  int64_t pages, heads, page_size, dim;
  void* data[4];
  Area areas[4];
  Pool(PyObject* o, int device) {
    need(bound.pages != nullptr && PyObject_TypeCheck(o, bound.pages) && PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4);
    const Tensor& codes = tensor(PyTuple_GET_ITEM(o, 0));
    need(codes.dim() == 4);
    pages = codes.size(0);
    heads = codes.size(1);
    page_size = codes.size(2);
    dim = 2 * codes.size(3);
    need(pages >= 1 && pages <= k31 && heads >= 1 && page_size >= 4 && page_size <= k31 && (page_size & (page_size - 1)) == 0 &&
         dim % 32 == 0 && dim >= 32 && dim <= 256);
    const int64_t shapes[4][6] = {{pages, heads, page_size, dim / 2, 0, 0}, {pages, heads, page_size, dim / 32, 0, 0},
                                  {pages, heads, page_size / 4, dim / 8, 4, 4}, {pages, heads, page_size / 4, dim / 32, 4, 0}};
    const int dims[4] = {4, 4, 6, 5};
    for (int i = 0; i < 4; ++i) {
      const Tensor& t = tensor(PyTuple_GET_ITEM(o, i));
      need(t.scalar_type() == at::kByte && on(t, device) && t.dim() == dims[i] && t.is_contiguous());
      for (int k = 0; k < dims[i]; ++k) need(t.size(k) == shapes[i][k]);
      data[i] = t.data_ptr();
      areas[i] = area(t);
      need((reinterpret_cast<uintptr_t>(data[i]) & 15) == 0);
    }
  }
};

PyObject* fp4_rows(PyObject* const* x, Py_ssize_t n, bool write) {
  return accepted(n, 6, [&] {
    need((write ? bound.fp4_write != nullptr : bound.fp4_read != nullptr));
    const int device = (int)integer(x[0]);
    void* stream = reinterpret_cast<void*>(integer(x[1]));
    const Tensor &k = tensor(x[2]), &v = tensor(x[3]), &slots = tensor(x[4]);
    const Pool pool(x[5], device);
    const int64_t tokens = slots.numel(), width = pool.heads * pool.dim;
    need(pool.pages <= k31 / pool.page_size && pool.heads <= 65536);
    const int* slot = vector(slots, device, tokens);
    const int code = code_of(k);
    for (const Tensor* t : {&k, &v})
      need(t->scalar_type() == k.scalar_type() && on(*t, device) && t->dim() == 2 && t->size(0) == tokens && t->size(1) == width &&
           t->stride(1) == 1 && t->stride(0) >= 0);
    void *kp = k.data_ptr(), *vp = v.data_ptr();
    const int64_t ldk = k.stride(0), ldv = v.stride(0);
    if (tokens == 0) return 0;
    if (write) {
      const Area others[3] = {area(k, width), area(v, width), area(slots)};
      for (int i = 0; i < 4; ++i) {
        for (int j = 0; j < i; ++j) need(!meet(pool.areas[i], pool.areas[j]));
        for (const Area& x : others) need(!meet(pool.areas[i], x));
      }
    } else {
      const Area keys = area(k, width), values = area(v, width), ids = area(slots);
      need((tokens <= 1 || (ldk >= width && ldv >= width)) && !meet(keys, values) && !meet(keys, ids) && !meet(values, ids));
      for (const Area& held : pool.areas) need(!meet(keys, held) && !meet(values, held));
    }
    return without_gil([&] {
      return write ? bound.fp4_write(code, kp, ldk, vp, ldv, slot, (int)tokens, (int)pool.heads, (int)pool.dim, pool.data[0], pool.data[1],
                                     pool.data[2], pool.data[3], (int)pool.pages, (int)pool.page_size, stream)
                   : bound.fp4_read(code, kp, ldk, vp, ldv, slot, (int)tokens, (int)pool.heads, (int)pool.dim, pool.data[0], pool.data[1],
                                    pool.data[2], pool.data[3], (int)pool.pages, (int)pool.page_size, stream);
    });
  });
}
PyObject* fp4_write(PyObject*, PyObject* const* x, Py_ssize_t n) { return fp4_rows(x, n, true); }
PyObject* fp4_read(PyObject*, PyObject* const* x, Py_ssize_t n) { return fp4_rows(x, n, false); }

// Memory of one call (of its stream, or of the graph's own memory while one is captured).
Tensor call_scratch(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, at::TensorOptions().dtype(at::kByte).device(like.device())) : Tensor();
}

PyObject* fp4_attention(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return accepted(n, 15, [&] {
    const int device = (int)integer(x[0]);
    void* stream = reinterpret_cast<void*>(integer(x[1]));
    const Tensor &q = tensor(x[2]), &table = tensor(x[7]), &offsets = tensor(x[8]), &lengths = tensor(x[9]), &out = tensor(x[12]);
    const int64_t nq = integer(x[3]), nkv = integer(x[4]), d = integer(x[5]);
    const Pool pool(x[6], device);
    int64_t most = integer(x[10]), longest = integer(x[11]), window = integer(x[14]);
    const double scale = real(x[13]);
    need(pool.dim == d && pool.heads == nkv && nkv <= 1024 && nq >= nkv && nq <= k31 / d && nq % nkv == 0);
    const auto& entry = bound.attention[d / 32];
    need(entry.run != nullptr);
    const int code = code_of(q);
    for (const Tensor* t : {&q, &out})
      need(t->scalar_type() == q.scalar_type() && on(*t, device) && t->dim() == 2 && t->stride(1) == 1 && t->size(1) >= nq * d);
    const int64_t rows = q.size(0), ldq = q.stride(0), ldo = out.stride(0);
    need(out.size(0) == rows && rows <= k31 && ldq >= 0 && ldo >= 0 && (rows <= 1 || ldo >= nq * d));
    need(table.scalar_type() == at::kInt && on(table, device) && table.dim() == 2 && table.is_contiguous() && table.size(1) >= 1);
    const int64_t requests = table.size(0), columns = table.size(1);
    const int* offset = vector(offsets, device, requests + 1);
    const int* length = vector(lengths, device, requests);
    need(requests <= 65535 && columns <= k31 && most >= 0 && longest >= 0 && longest <= columns * pool.page_size && window >= 0 &&
         scale >= -1e30 && scale <= 1e30);
    void *qp = q.data_ptr(), *op = out.data_ptr();
    const Area to = area(out, nq * d);
    need(!meet(to, area(q, nq * d)) && !meet(to, area(table)) && !meet(to, area(offsets)) && !meet(to, area(lengths)));
    for (const Area& held : pool.areas) need(!meet(to, held));
    most = std::min(most, rows);
    if (most == 0 || requests == 0) return 0;
    need(longest <= k31);
    if (window >= longest) window = 0;  // every row sees all keys before it
    const int group = (int)(nq / nkv);
    const int64_t bytes = entry.scratch(code, (int)rows, (int)requests, (int)nkv, group, (int)most, (int)longest, (int)window);
    const Tensor scratch = call_scratch(bytes, q);
    void* memory = bytes > 0 ? scratch.data_ptr() : nullptr;
    return without_gil([&] {
      return entry.run(code, qp, ldq, op, ldo, (int)rows, pool.data[0], pool.data[1], pool.data[2], pool.data[3], (int)pool.pages,
                       (int)pool.page_size, (int)nkv, group, static_cast<const int*>(table.data_ptr()), (int)columns, offset, length,
                       (int)requests, (int)most, (int)longest, (float)scale, (int)window, memory, bytes, stream);
    });
  });
}

PyObject* token_logprobs(PyObject*, PyObject* const* x, Py_ssize_t n) {
  return accepted(n, 9, [&] {
    need(bound.token_logprobs != nullptr);
    const int device = (int)integer(x[0]);
    void* stream = reinterpret_cast<void*>(integer(x[1]));
    const Tensor &logits = tensor(x[2]), &ids = tensor(x[7]), &theirs = tensor(x[8]);
    const int code = code_of(logits);
    need(on(logits, device) && logits.dim() == 2 && logits.stride(1) == 1 && logits.stride(0) >= 0);
    const int64_t rows = logits.size(0), vocab = logits.size(1), ld = logits.stride(0);
    const int* tokens = vector(tensor(x[3]), device, rows);
    float* logprob = vector<float>(tensor(x[4]), device, rows, at::kFloat);
    float* entropy = vector<float>(tensor(x[5]), device, rows, at::kFloat);
    int* rank = vector(tensor(x[6]), device, rows);
    need(ids.scalar_type() == at::kInt && theirs.scalar_type() == at::kFloat);
    for (const Tensor* t : {&ids, &theirs})
      need(on(*t, device) && t->dim() == 2 && t->size(0) == rows && t->size(1) == ids.size(1) && t->is_contiguous());
    const int64_t top = ids.size(1);
    need(top <= bound.max_top && top <= vocab);
    if (rows == 0) return 0;
    need(vocab >= 1 && vocab <= bound.max_vocab);
    const Area outs[5] = {area(tensor(x[4])), area(tensor(x[5])), area(tensor(x[6])), area(ids), area(theirs)};
    const Area ins[2] = {area(logits, vocab), area(tensor(x[3]))};
    for (int i = 0; i < 5; ++i) {
      for (int j = 0; j < i; ++j) need(!meet(outs[i], outs[j]));
      for (const Area& in : ins) need(!meet(outs[i], in));
    }
    const int64_t bytes = bound.logprobs_scratch((int)rows, (int)vocab);
    const Tensor scratch = call_scratch(bytes, logits);
    void* memory = bytes > 0 ? scratch.data_ptr() : nullptr;
    return without_gil([&] {
      return bound.token_logprobs(code, logits.data_ptr(), ld, tokens, (int)rows, (int)vocab, (int)top, logprob, entropy, rank,
                                  static_cast<int*>(ids.data_ptr()), static_cast<float*>(theirs.data_ptr()), memory, bytes, stream);
    });
  });
}

#define LS_FAST(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {LS_FAST(bind_serving), LS_FAST(bind_attention), LS_FAST(step_tables),    LS_FAST(fp4_write),
                         LS_FAST(fp4_read),     LS_FAST(fp4_attention),  LS_FAST(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "lockstep_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_lockstep_calls() { return PyModule_Create(&module); }
