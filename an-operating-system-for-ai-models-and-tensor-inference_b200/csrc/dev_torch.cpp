// myos.dev's calls on torch tensors: the checks of tensors (device, type, shape,
// strides) and the C ABI call behind them, as a CPython extension.
//
// A serving step makes these calls once per layer and token, each a few
// microseconds of device time. Asking a dozen tensors the same questions from
// Python took 12 us a call (7 us of it the questions, 1.6 us ctypes).
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <string>

#include "../../include/myos_cuda.h"

namespace {

using at::Tensor;
using c10::ScalarType;

PyObject* g_error = nullptr;  // myos._lib.MyosError

struct Refusal {
  int code;
  std::string why;
};
struct PyFailed {};  // a Python exception is set

[[noreturn]] void refuse(int code, std::string why) { throw Refusal{code, std::move(why)}; }

// ------------------------------------------------------------------ arguments
// Positional and keyword arguments into out[0 .. n), by the names' order.
void parse(const char* fn, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames,
           const char* const* names, int n, int required, PyObject** out) {
  for (int i = 0; i < n; ++i) out[i] = nullptr;
  if (nargs > n) {
    PyErr_Format(PyExc_TypeError, "%s() takes at most %d arguments (%zd given)", fn, n, nargs);
    throw PyFailed{};
  }
  for (Py_ssize_t i = 0; i < nargs; ++i) out[i] = args[i];
  const Py_ssize_t nk = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
  for (Py_ssize_t k = 0; k < nk; ++k) {
    PyObject* name = PyTuple_GET_ITEM(kwnames, k);
    int at = -1;
    for (int i = 0; i < n && at < 0; ++i)
      if (PyUnicode_CompareWithASCIIString(name, names[i]) == 0) at = i;
    if (at < 0 || out[at]) {
      PyErr_Format(PyExc_TypeError, at < 0 ? "%s() got an unexpected argument '%U'"
                                           : "%s() got two values for argument '%U'",
                   fn, name);
      throw PyFailed{};
    }
    out[at] = args[nargs + k];
  }
  for (int i = 0; i < n; ++i) {
    if (i < required && !out[i]) {
      PyErr_Format(PyExc_TypeError, "%s() misses argument '%s'", fn, names[i]);
      throw PyFailed{};
    }
    if (out[i] == Py_None) out[i] = nullptr;
  }
}

uint32_t u32(PyObject* o, const char* what) {
  const long long v = o ? PyLong_AsLongLong(o) : 0;
  if (v == -1 && PyErr_Occurred()) throw PyFailed{};
  if (v < 0 || v > 0xffffffffll) refuse(MYOS_ERR_ARG, std::string(what) + ": out of range");
  return (uint32_t)v;
}

float f32(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyFailed{};
  return (float)v;
}

std::string shape_text(c10::IntArrayRef s) {
  std::string t = "[";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + "]";
}

// The tensors of one call, all on the first one's device.
struct Call {
  int dev;

  static const Tensor& cuda(PyObject* o, const char* what) {
    if (!o || !THPVariable_Check(o)) refuse(MYOS_ERR_ARG, std::string(what) + ": not a CUDA tensor");
    const Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.layout() != c10::kStrided)
      refuse(MYOS_ERR_ARG, std::string(what) + ": not a CUDA tensor");
    return t;
  }
  Call(PyObject* first, const char* what) : dev(cuda(first, what).get_device()) {}

  const Tensor& get(PyObject* o, const char* what, std::initializer_list<ScalarType> types) const {
    const Tensor& t = cuda(o, what);
    if (t.get_device() != dev)
      refuse(MYOS_ERR_ARG, std::string(what) + ": on cuda:" + std::to_string(t.get_device()) +
                               ", not cuda:" + std::to_string(dev));
    bool ok = false;
    for (ScalarType k : types) ok |= t.scalar_type() == k;
    if (!ok) refuse(MYOS_ERR_ARG, std::string(what) + ": dtype " + c10::toString(t.scalar_type()));
    return t;
  }
  // n contiguous values (n < 0: any number); null stays null.
  void* vec(PyObject* o, const char* what, std::initializer_list<ScalarType> types, int64_t n) const {
    if (!o) return nullptr;
    const Tensor& t = get(o, what, types);
    if (n >= 0 && t.numel() != n)
      refuse(MYOS_ERR_SHAPE, std::string(what) + ": " + std::to_string(n) + " values wanted, got " +
                                 shape_text(t.sizes()));
    if (!t.is_contiguous()) refuse(MYOS_ERR_ARG, std::string(what) + ": not contiguous");
    return t.data_ptr();
  }
  // A tensor of this shape whose rows are contiguous, and the elements from row
  // to row (a single row has no stride of its own).
  void* rows(PyObject* o, const char* what, std::initializer_list<ScalarType> types,
             c10::IntArrayRef shape, size_t* stride) const {
    const Tensor& t = get(o, what, types);
    if (t.sizes() != shape)
      refuse(MYOS_ERR_SHAPE, std::string(what) + ": " + shape_text(shape) + " wanted, got " +
                                 shape_text(t.sizes()));
    int64_t row = 1;
    bool packed = true;
    for (size_t i = shape.size() - 1; i > 0; --i) {
      packed &= shape[i] <= 1 || t.stride(i) == row;
      row *= shape[i];
    }
    if (!packed || (shape[0] > 1 && t.stride(0) < 0))
      refuse(MYOS_ERR_ARG, std::string(what) + ": the values of a row are not contiguous");
    *stride = (size_t)(shape[0] > 1 ? t.stride(0) : row);
    return t.data_ptr();
  }
};

constexpr ScalarType kF32 = ScalarType::Float, kI32 = ScalarType::Int, kI64 = ScalarType::Long,
                     kBF16 = ScalarType::BFloat16, kU8 = ScalarType::Byte,
                     kU32 = ScalarType::UInt32, kI8 = ScalarType::Char;

int32_t dtype_of(const Tensor& t) { return t.scalar_type() == kF32 ? MYOS_F32 : MYOS_BF16; }

void* stream_of(PyObject* o, int dev) {
  if (!o) return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
  PyObject* raw = PyLong_Check(o) ? Py_NewRef(o) : PyObject_GetAttrString(o, "cuda_stream");
  if (!raw) throw PyFailed{};
  void* s = PyLong_AsVoidPtr(raw);
  Py_DECREF(raw);
  if (!s && PyErr_Occurred()) throw PyFailed{};
  return s;
}

// The C call on the tensors' device.
template <class F>
void run(const char* fn, int dev, F&& call) {
  int st;
  if (c10::cuda::current_device() == dev) {
    st = call();
  } else {
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    st = call();
  }
  if (st != MYOS_OK) refuse(st, fn);
}

template <class F>
PyObject* guarded(F&& body) {
  try {
    return body();
  } catch (const PyFailed&) {
    return nullptr;
  } catch (const Refusal& r) {
    if (PyObject* e = PyObject_CallFunction(g_error, "is", r.code, r.why.c_str())) {
      PyErr_SetObject(g_error, e);
      Py_DECREF(e);
    }
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

// ------------------------------------------------------------------- PagedKV
// The two tensors; what they hold is looked up at each call (0.05 us), so a
// tensor that was given other memory, strides or sizes goes by those.
struct PagedKv {
  PyObject_HEAD PyObject* k;
  PyObject* v;
};

struct KvView {
  int dev, heads, dim;
  myos_paged_kv c;
};

KvView kv_view(PyObject* ko, PyObject* vo) {
  Call call(ko, "k");
  const Tensor& k = call.get(ko, "k", {kF32, kBF16});
  const Tensor& v = call.get(vo, "v", {kF32, kBF16});
  if (k.dim() != 4)
    refuse(MYOS_ERR_SHAPE, "k: [pages, heads, slots, dim] wanted, got " + shape_text(k.sizes()));
  if (v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != k.scalar_type())
    refuse(MYOS_ERR_ARG, "k and v differ in shape, strides or dtype");
  int64_t size[4], st[4];
  for (int i = 0; i < 4; ++i) {
    size[i] = k.size(i);
    st[i] = k.stride(i);
    if (size[i] > 0x7fffffff) refuse(MYOS_ERR_SHAPE, "k: " + shape_text(k.sizes()));
  }
  if (size[3] > 1 && st[3] != 1) refuse(MYOS_ERR_ARG, "the last dimension is not contiguous");
  // a dimension of one element has no stride of its own
  int64_t least = size[3];
  for (int i = 1; i < 3; ++i)
    if (size[i] > 1 && st[i] > least) least = st[i];
  for (int i = 0; i < 3; ++i)
    if (size[i] <= 1) st[i] = least;
  return {call.dev,
          (int)size[1],
          (int)size[3],
          {k.data_ptr(),       v.data_ptr(),      (uint64_t)st[0],   (uint64_t)st[1],
           (uint64_t)st[2],    (uint32_t)size[0], (uint32_t)size[2], (uint32_t)size[1],
           (uint32_t)size[3],  k.scalar_type() == kF32 ? MYOS_KV_F32 : MYOS_KV_BF16, 0}};
}

void kv_free(PagedKv* self) {
  Py_XDECREF(self->k);
  Py_XDECREF(self->v);
  Py_TYPE(self)->tp_free((PyObject*)self);
}

int kv_init(PagedKv* self, PyObject* args, PyObject* kw) {
  static const char* names[] = {"k", "v", nullptr};
  PyObject *ko, *vo;
  if (!PyArg_ParseTupleAndKeywords(args, kw, "OO", const_cast<char**>(names), &ko, &vo)) return -1;
  PyObject* ok = guarded([&]() -> PyObject* {
    kv_view(ko, vo);
    Py_XSETREF(self->k, Py_NewRef(ko));
    Py_XSETREF(self->v, Py_NewRef(vo));
    return Py_None;
  });
  return ok ? 0 : -1;
}

PyObject* kv_get_k(PagedKv* s, void*) { return Py_NewRef(s->k ? s->k : Py_None); }
PyObject* kv_get_v(PagedKv* s, void*) { return Py_NewRef(s->v ? s->v : Py_None); }
PyObject* kv_get_int(PagedKv* s, void* which) {
  return guarded([&]() -> PyObject* {
    const KvView kv = kv_view(s->k, s->v);
    const int fields[] = {kv.dev, kv.heads, kv.dim};
    return PyLong_FromLong(fields[(intptr_t)which]);
  });
}

PyGetSetDef kv_fields[] = {
    {"k", (getter)kv_get_k, nullptr, "the K tensor", nullptr},
    {"v", (getter)kv_get_v, nullptr, "the V tensor", nullptr},
    {"dev", (getter)kv_get_int, nullptr, "the device's ordinal", nullptr},
    {"num_kv_heads", (getter)kv_get_int, nullptr, nullptr, (void*)1},
    {"head_dim", (getter)kv_get_int, nullptr, nullptr, (void*)2},
    {nullptr, nullptr, nullptr, nullptr, nullptr}};

PyTypeObject kv_type = {PyVarObject_HEAD_INIT(nullptr, 0) "myos.dev.PagedKV"};

KvView kv_of(PyObject* o, int dev) {
  if (!o || !PyObject_TypeCheck(o, &kv_type) || !((PagedKv*)o)->k)
    refuse(MYOS_ERR_ARG, "kv: not a PagedKV");
  const KvView kv = kv_view(((PagedKv*)o)->k, ((PagedKv*)o)->v);
  if (kv.dev != dev)
    refuse(MYOS_ERR_ARG, "kv: on cuda:" + std::to_string(kv.dev) + ", not cuda:" + std::to_string(dev));
  return kv;
}

// ----------------------------------------------------------------- operators
PyObject* paged_tables(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { TABLE, CTX, NEW, FREE, NUM, PAGE, PAGES, SLOTS, POS, SEQ, LENS, STARTS, RESULT, STREAM, N };
    static const char* const names[N] = {
        "block_table", "ctx_lens",  "new_lens", "free_pages", "num_free",   "page_size", "num_pages",
        "slots",       "positions", "row_seq",  "kv_lens",    "seq_starts", "result",    "stream"};
    PyObject* o[N];
    parse("paged_tables", args, nargs, kwnames, names, N, STREAM, o);
    Call c(o[TABLE], "block_table");
    const Tensor& t = c.get(o[TABLE], "block_table", {kI32});
    if (t.dim() != 2) refuse(MYOS_ERR_SHAPE, "block_table: [nseq, max_blocks] wanted");
    const int64_t nseq = t.size(0);
    size_t stride;
    void* table = c.rows(o[TABLE], "block_table", {kI32}, t.sizes(), &stride);
    const int64_t rows = c.get(o[SLOTS], "slots", {kI64}).numel();
    const int64_t cap = c.get(o[FREE], "free_pages", {kI32}).numel();
    auto i32 = [&](int i, int64_t n) { return (int32_t*)c.vec(o[i], names[i], {kI32}, n); };
    int32_t *ctx = i32(CTX, nseq), *add = i32(NEW, nseq), *free_ = i32(FREE, cap), *num = i32(NUM, 1),
            *pos = i32(POS, rows), *seq = i32(SEQ, rows), *lens = i32(LENS, nseq),
            *starts = i32(STARTS, nseq + 1), *result = i32(RESULT, 2);
    int64_t* slots = (int64_t*)c.vec(o[SLOTS], "slots", {kI64}, rows);
    const uint32_t page = u32(o[PAGE], "page_size"), pages = u32(o[PAGES], "num_pages");
    void* st = stream_of(o[STREAM], c.dev);
    run("paged_tables", c.dev, [&] {
      return myos_dev_paged_tables((int32_t*)table, stride, (size_t)t.size(1), ctx, add, (size_t)nseq,
                                   free_, (size_t)cap, num, page, pages, slots, pos, seq,
                                   (size_t)rows, lens, starts, result, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* qk_norm_rope_store(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { Q, QKV, KV, POS, SLOTS, COS, SIN, QG, KG, EPS, STREAM, N };
    static const char* const names[N] = {"q_out", "qkv",     "kv",      "positions", "slots", "cos",
                                         "sin",   "q_gamma", "k_gamma", "eps",       "stream"};
    PyObject* o[N];
    parse("qk_norm_rope_store", args, nargs, kwnames, names, N, COS, o);
    Call c(o[QKV], "qkv");
    const KvView kv = kv_of(o[KV], c.dev);
    const Tensor& q = c.get(o[Q], "q_out", {kF32});
    if (q.dim() != 3) refuse(MYOS_ERR_SHAPE, "q_out: [rows, num_q_heads, head_dim] wanted");
    const int64_t rows = q.size(0), hq = q.size(1), d = kv.dim;
    size_t q_stride, in_stride, cos_stride = 0, sin_stride = 0;
    void* qp = c.rows(o[Q], "q_out", {kF32}, {rows, hq, d}, &q_stride);
    void* in = c.rows(o[QKV], "qkv", {kF32}, {rows, (hq + 2 * kv.heads) * d}, &in_stride);
    void *cs = nullptr, *sn = nullptr;
    int64_t npos = 0, half = 0;
    if (o[COS] || o[SIN]) {
      const Tensor& t = c.get(o[COS], "cos", {kF32});
      if (t.dim() != 2) refuse(MYOS_ERR_SHAPE, "cos: [num_pos, rot_dim / 2] wanted");
      npos = t.size(0);
      half = t.size(1);
      cs = c.rows(o[COS], "cos", {kF32}, {npos, half}, &cos_stride);
      sn = c.rows(o[SIN], "sin", {kF32}, {npos, half}, &sin_stride);
      if ((int64_t)cos_stride != half || (int64_t)sin_stride != half)
        refuse(MYOS_ERR_ARG, "cos and sin are contiguous");
    }
    void *qg = c.vec(o[QG], "q_gamma", {kBF16}, d), *kg = c.vec(o[KG], "k_gamma", {kBF16}, d);
    int32_t* pos = (int32_t*)c.vec(o[POS], "positions", {kI32}, rows);
    int64_t* slots = (int64_t*)c.vec(o[SLOTS], "slots", {kI64}, rows);
    const float eps = o[EPS] ? f32(o[EPS]) : 1e-6f;
    void* st = stream_of(o[STREAM], c.dev);
    run("qk_norm_rope_store", c.dev, [&] {
      return myos_dev_qk_norm_rope_store((float*)qp, q_stride, (float*)in, in_stride, (size_t)rows,
                                         (size_t)hq, &kv.c, qg, kg, eps, (float*)cs, (float*)sn,
                                         (size_t)npos, (size_t)(2 * half), pos, slots, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { OUT, Q, KV, TABLE, LENS, WORK, SCALE, WINDOW, LSE, STREAM, N };
    static const char* const names[N] = {"out",  "q",     "kv",     "block_table", "kv_lens",
                                         "work", "scale", "window", "lse",         "stream"};
    PyObject* o[N];
    parse("paged_attention", args, nargs, kwnames, names, N, SCALE, o);
    Call c(o[Q], "q");
    const KvView kv = kv_of(o[KV], c.dev);
    const Tensor& q = c.get(o[Q], "q", {kF32});
    if (q.dim() != 3) refuse(MYOS_ERR_SHAPE, "q: [nseq, num_q_heads, head_dim] wanted");
    const int64_t nseq = q.size(0), hq = q.size(1);
    size_t q_stride, out_stride, table_stride, lse_stride = 0;
    void* qp = c.rows(o[Q], "q", {kF32}, {nseq, hq, kv.dim}, &q_stride);
    void* out = c.rows(o[OUT], "out", {kF32}, {nseq, hq, kv.dim}, &out_stride);
    void* lse = o[LSE] ? c.rows(o[LSE], "lse", {kF32}, {nseq, hq}, &lse_stride) : nullptr;
    if (lse && (int64_t)lse_stride != hq) refuse(MYOS_ERR_ARG, "lse is contiguous");
    const Tensor& t = c.get(o[TABLE], "block_table", {kI32});
    const int64_t blocks = t.dim() == 2 ? t.size(1) : 0;
    void* table = c.rows(o[TABLE], "block_table", {kI32}, {nseq, blocks}, &table_stride);
    int32_t* lens = (int32_t*)c.vec(o[LENS], "kv_lens", {kI32}, nseq);
    const int64_t bytes = c.get(o[WORK], "work", {kU8}).numel();
    void* work = c.vec(o[WORK], "work", {kU8}, bytes);
    const float scale = o[SCALE] ? f32(o[SCALE]) : (float)(1.0 / std::sqrt((double)kv.dim));
    const uint32_t window = u32(o[WINDOW], "window");
    void* st = stream_of(o[STREAM], c.dev);
    run("paged_attention", c.dev, [&] {
      return myos_dev_paged_attn((float*)out, out_stride, (float*)lse, (float*)qp, q_stride,
                                 (size_t)nseq, (size_t)hq, &kv.c, (int32_t*)table, table_stride,
                                 (size_t)blocks, lens, scale, window, work, (size_t)bytes, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* logit_controls(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { OUT, LOGITS, HIST, PLENS, HLENS, REP, FREQ, PRES, BSTARTS, BIDS, BVALS, MASK, MROWS, IDS,
           STREAM, N };
    static const char* const names[N] = {
        "out",         "logits",   "history",   "prompt_lens", "hist_lens", "repetition", "frequency", "presence",
        "bias_starts", "bias_ids", "bias_vals", "mask",        "mask_rows", "ids",        "stream"};
    PyObject* o[N];
    parse("logit_controls", args, nargs, kwnames, names, N, HIST, o);
    Call c(o[LOGITS], "logits");
    const Tensor& x = c.get(o[LOGITS], "logits", {kF32});
    if (x.dim() != 2) refuse(MYOS_ERR_SHAPE, "logits: [rows, vocab] wanted");
    const int64_t rows = x.size(0), vocab = x.size(1);
    size_t stride, out_stride = 0;
    void* in = c.rows(o[LOGITS], "logits", {kF32}, {rows, vocab}, &stride);
    void* out = o[OUT] ? c.rows(o[OUT], "out", {kF32}, {rows, vocab}, &out_stride) : nullptr;
    auto i32 = [&](int i, int64_t n) { return (int32_t*)c.vec(o[i], names[i], {kI32}, n); };
    auto fl = [&](int i, int64_t n) { return (float*)c.vec(o[i], names[i], {kF32}, n); };
    myos_logit_controls_args a = {};
    size_t st2;
    if (o[HIST]) {
      const Tensor& h = c.get(o[HIST], "history", {kI32});
      const int64_t width = h.dim() == 2 ? h.size(1) : 0;
      a.history = (int32_t*)c.rows(o[HIST], "history", {kI32}, {rows, width}, &st2);
      a.history_stride = st2;
      a.history_width = (uint64_t)width;
    }
    a.prompt_lens = i32(PLENS, rows);
    a.history_lens = i32(HLENS, rows);
    a.repetition = fl(REP, rows);
    a.frequency = fl(FREQ, rows);
    a.presence = fl(PRES, rows);
    // no tokens: an empty tensor has no address, and the penalties nothing to do
    if (o[HIST] && a.history_width == 0) {
      a.history = nullptr;
      a.repetition = a.frequency = a.presence = nullptr;
    }
    if (o[BSTARTS]) {
      if (!o[BIDS] || !o[BVALS])
        refuse(MYOS_ERR_ARG, "bias_starts, bias_ids and bias_vals come together");
      const int64_t nb = c.get(o[BIDS], "bias_ids", {kI32}).numel();
      a.bias_starts = i32(BSTARTS, rows + 1);
      a.bias_ids = i32(BIDS, nb);
      a.bias_vals = fl(BVALS, nb);
      a.num_bias = (uint64_t)nb;
      if (nb == 0) a.bias_starts = nullptr;
    }
    if (o[MASK]) {
      const Tensor& m = c.get(o[MASK], "mask", {kI32, kU32});
      if (m.dim() != 2 || m.size(1) * 32 < vocab)
        refuse(MYOS_ERR_SHAPE, "mask: fewer bits than the vocabulary");
      // asked here too: a mask of no rows has no address, which to the C call is no mask
      if (!o[MROWS] && m.size(0) < rows) refuse(MYOS_ERR_SHAPE, "mask: fewer rows than logits");
      a.mask = (uint32_t*)c.rows(o[MASK], "mask", {kI32, kU32}, m.sizes(), &st2);
      a.mask_stride = st2;
      a.num_masks = (uint64_t)m.size(0);
      a.mask_rows = i32(MROWS, rows);
    }
    uint32_t* ids = (uint32_t*)c.vec(o[IDS], "ids", {kI32, kU32}, rows);
    void* st = stream_of(o[STREAM], c.dev);
    run("logit_controls", c.dev, [&] {
      return myos_dev_logit_controls((float*)out, out_stride, (float*)in, stride, (size_t)rows,
                                     (size_t)vocab, &a, ids, st);
    });
    Py_RETURN_NONE;
  });
}

// rows [rows, width] of x in 8 bits: q [rows, width], scales [rows]. width: of q.
struct Rows {
  int8_t* q;
  float* scales;
  const void* x;
  size_t q_stride, x_stride;
  int64_t rows, width;
  int32_t x_dtype;
};

Rows rows_of(const Call& c, PyObject* q, PyObject* scales, PyObject* x, const char* what, int64_t times) {
  const Tensor& t = c.get(q, "q", {kI8});
  if (t.dim() != 2) refuse(MYOS_ERR_SHAPE, "q: [rows, width] wanted, got " + shape_text(t.sizes()));
  Rows r;
  r.rows = t.size(0);
  r.width = t.size(1);
  r.q = (int8_t*)c.rows(q, "q", {kI8}, {r.rows, r.width}, &r.q_stride);
  r.x = c.rows(x, what, {kF32, kBF16}, {r.rows, times * r.width}, &r.x_stride);
  r.x_dtype = dtype_of(c.get(x, what, {kF32, kBF16}));
  r.scales = (float*)c.vec(scales, "scales", {kF32}, r.rows);
  return r;
}

PyObject* add_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { Q, SCALES, X, GAMMA, RESIDUAL, TOTAL, EPS, STREAM, N };
    static const char* const names[N] = {"q",        "scales", "x",   "gamma",
                                         "residual", "total",  "eps", "stream"};
    PyObject* o[N];
    parse("add_norm_quant", args, nargs, kwnames, names, N, RESIDUAL, o);
    Call c(o[Q], "q");
    const Rows r = rows_of(c, o[Q], o[SCALES], o[X], "x", 1);
    void* gamma = c.vec(o[GAMMA], "gamma", {kBF16}, r.width);
    size_t res_stride = 0, total_stride = 0;
    void* res = o[RESIDUAL]
                    ? c.rows(o[RESIDUAL], "residual", {kF32}, {r.rows, r.width}, &res_stride)
                    : nullptr;
    void* total = o[TOTAL] ? c.rows(o[TOTAL], "total", {kF32}, {r.rows, r.width}, &total_stride)
                           : nullptr;
    const float eps = o[EPS] ? f32(o[EPS]) : 1e-6f;
    void* st = stream_of(o[STREAM], c.dev);
    run("add_norm_quant", c.dev, [&] {
      return myos_dev_add_norm_quant(r.q, r.q_stride, r.scales, (float*)total, total_stride, r.x,
                                     r.x_dtype, r.x_stride, (float*)res, res_stride, gamma, eps,
                                     (size_t)r.rows, (size_t)r.width, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* quant_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { Q, SCALES, X, STREAM, N };
    static const char* const names[N] = {"q", "scales", "x", "stream"};
    PyObject* o[N];
    parse("quant_rows", args, nargs, kwnames, names, N, STREAM, o);
    Call c(o[Q], "q");
    const Rows r = rows_of(c, o[Q], o[SCALES], o[X], "x", 1);
    void* st = stream_of(o[STREAM], c.dev);
    run("quant_rows", c.dev, [&] {
      return myos_dev_quant_rows(r.q, r.q_stride, r.scales, r.x, r.x_dtype, r.x_stride,
                                 (size_t)r.rows, (size_t)r.width, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* swiglu_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { Q, SCALES, X, STREAM, N };
    static const char* const names[N] = {"q", "scales", "gate_up", "stream"};
    PyObject* o[N];
    parse("swiglu_quant", args, nargs, kwnames, names, N, STREAM, o);
    Call c(o[Q], "q");
    const Rows r = rows_of(c, o[Q], o[SCALES], o[X], "gate_up", 2);
    void* st = stream_of(o[STREAM], c.dev);
    run("swiglu_quant", c.dev, [&] {
      return myos_dev_swiglu_quant(r.q, r.q_stride, r.scales, r.x, r.x_dtype, r.x_stride,
                                   (size_t)r.rows, (size_t)r.width, st);
    });
    Py_RETURN_NONE;
  });
}

PyObject* matmul_i8(PyObject*, PyObject* const* args, Py_ssize_t nargs, PyObject* kwnames) {
  return guarded([&]() -> PyObject* {
    enum { OUT, A, AS, W, WS, BIAS, STREAM, N };
    static const char* const names[N] = {"out", "a", "a_scales", "w", "w_scales", "bias", "stream"};
    PyObject* o[N];
    parse("matmul_i8", args, nargs, kwnames, names, N, BIAS, o);
    Call c(o[OUT], "out");
    const Tensor& a = c.get(o[A], "a", {kI8});
    const Tensor& w = c.get(o[W], "w", {kI8});
    if (a.dim() != 2) refuse(MYOS_ERR_SHAPE, "a: [rows, k] wanted, got " + shape_text(a.sizes()));
    if (w.dim() != 2 || w.size(1) != a.size(1))
      refuse(MYOS_ERR_SHAPE, "w: [channels, " + std::to_string(a.size(1)) + "] wanted, got " +
                                 shape_text(w.sizes()));
    const int64_t rows = a.size(0), k = a.size(1), channels = w.size(0);
    size_t out_stride, a_stride, w_stride;
    void* out = c.rows(o[OUT], "out", {kF32, kBF16}, {rows, channels}, &out_stride);
    void* ap = c.rows(o[A], "a", {kI8}, {rows, k}, &a_stride);
    void* wp = c.rows(o[W], "w", {kI8}, {channels, k}, &w_stride);
    // a single row has no stride of its own, and need not be a multiple of 16 long
    if (rows == 1) a_stride = (size_t)((k + 15) / 16 * 16);
    if (channels == 1) w_stride = (size_t)((k + 15) / 16 * 16);
    void* as = c.vec(o[AS], "a_scales", {kF32}, rows);
    void* ws = c.vec(o[WS], "w_scales", {kF32}, channels);
    void* bias = c.vec(o[BIAS], "bias", {kF32}, channels);
    const int32_t type = dtype_of(c.get(o[OUT], "out", {kF32, kBF16}));
    void* st = stream_of(o[STREAM], c.dev);
    run("matmul_i8", c.dev, [&] {
      return myos_dev_matmul_i8(out, type, out_stride, (int8_t*)ap, a_stride, (float*)as,
                                (int8_t*)wp, w_stride, (float*)ws, (float*)bias, (size_t)rows,
                                (size_t)k, (size_t)channels, st);
    });
    Py_RETURN_NONE;
  });
}

constexpr char k_doc_paged_tables[] =
    "paged_tables(block_table, ctx_lens, new_lens, free_pages, num_free, page_size, num_pages, slots, positions, row_seq, kv_lens, seq_starts, result, stream=None)\n"
    "--\n"
    "\n"
    "Gives each request the pages for its new tokens (from the end of\n"
    "free_pages[:num_free]) and maps the step's packed rows to cache slots:\n"
    "myos_dev_paged_tables. block_table [nseq, max_blocks] is updated in place;\n"
    "slots (int64), positions, row_seq [max_rows], kv_lens [nseq], seq_starts\n"
    "[nseq + 1] and result [2] (pages left, requests refused) are written. All\n"
    "integers but slots are int32.\n";

constexpr char k_doc_qk_norm_rope_store[] =
    "qk_norm_rope_store(q_out, qkv, kv, positions, slots, cos=None, sin=None, q_gamma=None, k_gamma=None, eps = 1e-6, stream=None)\n"
    "--\n"
    "\n"
    "q_out [rows, num_q_heads, d] = the q heads of qkv [rows, (num_q_heads +\n"
    "2 num_kv_heads) d], per-head RMSNorm (bf16 q_gamma; None: none) and rotated\n"
    "by cos/sin [num_pos, rot_dim / 2] at positions [rows]; k likewise with\n"
    "k_gamma, then k and v into the cache at slots [rows] (int64, negative: not\n"
    "stored): myos_dev_qk_norm_rope_store. q_out may be a view of qkv's own q\n"
    "part.\n";

constexpr char k_doc_paged_attention[] =
    "paged_attention(out, q, kv, block_table, kv_lens, work, scale=None, window = 0, lse=None, stream=None)\n"
    "--\n"
    "\n"
    "out [nseq, num_q_heads, d] = attention of q (same shape) over the last\n"
    "window (0: all) of each sequence's kv_lens keys; lse [nseq, num_q_heads]\n"
    "(optional) their log-sum-exp. scale defaults to 1 / sqrt(d). work: at least\n"
    "WORK_BYTES of uint8, zeroed once before its first use, not shared by calls\n"
    "that may run at the same time: myos_dev_paged_attn.\n";

constexpr char k_doc_logit_controls[] =
    "logit_controls(out, logits, history=None, prompt_lens=None, hist_lens=None, repetition=None, frequency=None, presence=None, bias_starts=None, bias_ids=None, bias_vals=None, mask=None, mask_rows=None, ids=None, stream=None)\n"
    "--\n"
    "\n"
    "out [rows, vocab] = logits under each row's penalties (history [rows,\n"
    "width] int32, the first prompt_lens of its hist_lens tokens the prompt),\n"
    "biases (entries bias_starts[r] .. bias_starts[r + 1] of bias_ids /\n"
    "bias_vals) and grammar mask (32 tokens a word, set: allowed; row r uses mask\n"
    "mask_rows[r], negative: none); ids [rows] (int32 or uint32) the greedy ids\n"
    "of the result: myos_dev_logit_controls. out may be logits (in place) or\n"
    "None (only ids).\n";

constexpr char k_doc_add_norm_quant[] =
    "add_norm_quant(q, scales, x, gamma, residual=None, total=None, eps = 1e-6, stream=None)\n"
    "--\n"
    "\n"
    "total = x + residual (f32; None: x), and the rows of its RMSNorm with gamma\n"
    "(bf16 [width]) in 8 bits: q [rows, width] int8 and scales [rows], q * scale\n"
    "standing for the value: myos_dev_add_norm_quant. x is f32 or bf16; total\n"
    "(optional) receives the sum and may be residual, or an f32 x: in place.\n";

constexpr char k_doc_quant_rows[] =
    "quant_rows(q, scales, x, stream=None)\n"
    "--\n"
    "\n"
    "The rows of x [rows, width] (f32 or bf16) in 8 bits: q [rows, width] int8\n"
    "and scales [rows], the row's largest magnitude / 127: myos_dev_quant_rows.\n"
    "For a weight [channels, k] that is a scale for each channel.\n";

constexpr char k_doc_swiglu_quant[] =
    "swiglu_quant(q, scales, gate_up, stream=None)\n"
    "--\n"
    "\n"
    "silu(gate) * up in 8 bits: gate_up [rows, 2 width] (f32 or bf16) holds the\n"
    "gate values of a row, then its up values; q [rows, width] int8 and scales\n"
    "[rows]: myos_dev_swiglu_quant.\n";

constexpr char k_doc_matmul_i8[] =
    "matmul_i8(out, a, a_scales, w, w_scales, bias=None, stream=None)\n"
    "--\n"
    "\n"
    "out [rows, channels] (f32 or bf16) = a w^T of int8 a [rows, k] and\n"
    "w [channels, k], summed exactly, times a_scales [rows] and w_scales\n"
    "[channels], plus bias [channels] (f32): myos_dev_matmul_i8. The rows of a\n"
    "and w begin at multiples of 16 bytes (k itself need not be one).\n";

constexpr char k_doc_PagedKV[] =
    "PagedKV(k, v)\n"
    "--\n"
    "\n"
    "One layer's paged cache: k and v as [num_pages, num_kv_heads, page_size,\n"
    "head_dim] views, f32 or bf16, with the same strides (a cache kept as\n"
    "[num_pages, page_size, num_kv_heads, head_dim] is passed as\n"
    "t.permute(0, 2, 1, 3)). Holds the tensors, copies nothing; each call takes\n"
    "their memory, strides and sizes as they are then.\n";

#define METHOD(f) \
  {#f, (PyCFunction)(void (*)(void))f, METH_FASTCALL | METH_KEYWORDS, k_doc_##f}
PyMethodDef methods[] = {METHOD(paged_tables), METHOD(qk_norm_rope_store), METHOD(paged_attention),
                         METHOD(logit_controls), METHOD(add_norm_quant), METHOD(quant_rows),
                         METHOD(swiglu_quant), METHOD(matmul_i8), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_myos_dev", nullptr, -1, methods,
                      nullptr,               nullptr,     nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__myos_dev(void) {
  PyObject* lib = PyImport_ImportModule("myos._lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "MyosError");
  Py_DECREF(lib);
  if (!g_error) return nullptr;
  kv_type.tp_basicsize = sizeof(PagedKv);
  kv_type.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_BASETYPE;
  kv_type.tp_new = PyType_GenericNew;
  kv_type.tp_init = (initproc)kv_init;
  kv_type.tp_dealloc = (destructor)kv_free;
  kv_type.tp_getset = kv_fields;
  kv_type.tp_doc = k_doc_PagedKV;
  if (PyType_Ready(&kv_type) < 0) return nullptr;
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddObjectRef(m, "PagedKV", (PyObject*)&kv_type) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
