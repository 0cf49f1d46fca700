// The short way from torch tensors to the C ABI for the serving ops.
//
// A decode step's kernels run for a few microseconds, and reading a dozen
// tensors' types, shapes and strides from Python takes longer than that.  Each
// function here makes the checks of the Python wrapper of the same name for
// the plain case (valid arguments on the current device and stream), launches
// through the C ABI and returns the result; anything else it leaves alone and
// returns None, and the wrapper goes its own way, which names what is wrong.
// A non-zero status of the C ABI comes back as an int.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "sonata_b200.h"

namespace {

struct Abi {  // of the loaded libsonata_b200.so, set by bind()
  decltype(&sn_paged_decode_attention) attend;
  decltype(&sn_paged_decode_workspace_size) attend_size;
  decltype(&sn_rotary_paged_append) append;
  decltype(&sn_rotary_paged_append_at) append_at;
  decltype(&sn_copy_pages) copy;
  decltype(&sn_mamba2_prompt) prompt;
  decltype(&sn_mamba2_prompt_workspace_size) prompt_size;
  decltype(&sn_paged_decode_attention_mass) mass;
  decltype(&sn_paged_mass_workspace_size) mass_size;
  decltype(&sn_evict_positions) evict;
  decltype(&sn_evict_workspace_size) evict_size;
  decltype(&sn_update_page_bounds) bounds;
  decltype(&sn_select_blocks) select;
  decltype(&sn_select_blocks_workspace_size) select_size;
  decltype(&sn_paged_sparse_attention) sparse;
} abi;

using at::Tensor;

const Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool is(const Tensor* t, at::ScalarType type, int64_t dim, int dev) {
  return t && t->scalar_type() == type && t->dim() == dim && t->is_cuda() && t->get_device() == dev &&
         t->layout() == at::kStrided;
}
bool dense(const Tensor* t, at::ScalarType type, at::IntArrayRef shape, int dev) {
  return is(t, type, static_cast<int64_t>(shape.size()), dev) && t->sizes() == shape && t->is_contiguous();
}
// An optional tensor: None, or as dense().
bool dense_or_none(PyObject* o, const Tensor** t, at::ScalarType type, at::IntArrayRef shape, int dev) {
  *t = nullptr;
  if (o == Py_None) return true;
  *t = tensor(o);
  return dense(*t, type, shape, dev);
}
void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
bool number(PyObject* o, int* v) {
  if (!PyLong_CheckExact(o)) return false;
  const long n = PyLong_AsLong(o);
  if ((n == -1 && PyErr_Occurred()) || n < INT32_MIN || n > INT32_MAX) {
    PyErr_Clear();
    return false;
  }
  *v = static_cast<int>(n);
  return true;
}
int current_device() { return c10::cuda::current_device(); }
void* current_stream(int dev) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream(); }

struct Pages {
  const Tensor *k, *v, *table, *lens;
  int64_t n, heads, page, hd, streams, width;
  bool read(PyObject* const* a, int dev) {
    k = tensor(a[0]);
    v = tensor(a[1]);
    table = tensor(a[2]);
    lens = tensor(a[3]);
    if (!is(k, at::kBFloat16, 4, dev) || !is(v, at::kBFloat16, 4, dev) || !is(table, at::kInt, 2, dev) ||
        !is(lens, at::kInt, 1, dev) || k->sizes() != v->sizes())
      return false;
    n = k->size(0), heads = k->size(1), page = k->size(2), hd = k->size(3);
    streams = table->size(0), width = table->size(1);
    return n > 0 && heads > 0 && page > 0 && hd > 0 && k->stride(3) == 1 && v->stride(3) == 1 && streams > 0 && width > 0 &&
           (table->stride(1) == 1 || width == 1) && lens->size(0) == streams && lens->is_contiguous() && n <= INT32_MAX &&
           page <= INT32_MAX && width <= INT32_MAX;
  }
  // an axis of extent 1 is never stepped along: its stride may be anything
  int64_t stride(const Tensor* t, int axis) const {
    return t->size(axis) > 1 ? t->stride(axis) : std::max(t->stride(axis), hd);
  }
  int64_t table_stride() const { return streams > 1 ? table->stride(0) : width; }
};

PyObject* status(int rc) { return PyLong_FromLong(rc); }

// One token a stream: q, pages, scale and workspace as all forms of the attention take them.
struct Attend {
  const Tensor *q, *ws;
  Pages p;
  int64_t batch, heads;
  size_t need;  // workspace bytes
  float scale;
  bool read(PyObject* const* a, PyObject* scale_arg, PyObject* ws_arg, int dev) {
    q = tensor(a[0]);
    ws = tensor(ws_arg);
    if (!is(q, at::kBFloat16, 3, dev) || !p.read(a + 1, dev) || !is(ws, at::kByte, 1, dev) || !ws->is_contiguous() ||
        !(scale_arg == Py_None || PyFloat_CheckExact(scale_arg)))
      return false;
    batch = q->size(0), heads = q->size(1);
    if (batch != p.streams || q->size(2) != p.hd || (q->stride(2) != 1 && p.hd > 1) || heads < 1 || heads % p.heads || batch > INT32_MAX)
      return false;
    scale = scale_arg == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(p.hd)))
                                 : static_cast<float>(PyFloat_AS_DOUBLE(scale_arg));
    return true;
  }
  bool room(size_t n) {
    need = n;
    return n > 0 && static_cast<size_t>(ws->numel()) >= n && reinterpret_cast<uintptr_t>(ws->data_ptr()) % 16 == 0;
  }
  // f with the form's own arguments after the lengths, the output's, and the common end.
  template <typename F, typename... Own>
  PyObject* launch(F f, int dev, Own... own) {
    Tensor out = at::empty({batch, heads, p.hd}, q->options());
    const int rc = f(q->data_ptr(), q->stride(0), q->stride(1), p.k->data_ptr(), p.stride(p.k, 0), p.stride(p.k, 1),
                     p.stride(p.k, 2), p.v->data_ptr(), p.stride(p.v, 0), p.stride(p.v, 1), p.stride(p.v, 2),
                     static_cast<int>(p.n), static_cast<int>(p.page), p.table->data_ptr<int>(), p.table_stride(),
                     static_cast<int>(p.width), p.lens->data_ptr<int>(), own..., out.data_ptr(), nullptr, scale,
                     static_cast<int>(batch), static_cast<int>(heads), static_cast<int>(p.heads), static_cast<int>(p.hd),
                     ws->data_ptr(), need, current_stream(dev));
    return rc ? status(rc) : THPVariable_Wrap(std::move(out));
  }
};

PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || a[7] != Py_False) Py_RETURN_NONE;
  const int dev = current_device();
  Attend t;
  if (!t.read(a, a[5], a[6], dev) ||
      !t.room(abi.attend_size(static_cast<int>(t.batch), static_cast<int>(t.heads), static_cast<int>(t.p.hd))))
    Py_RETURN_NONE;
  return t.launch(abi.attend, dev);
  END_HANDLE_TH_ERRORS
}

// Accumulated weights [.., >= room] with a dense last axis and no overlaps.
bool mass_ok(const Tensor* m, int64_t dim, int64_t room, int dev) {
  if (!is(m, at::kFloat, dim, dev) || m->size(dim - 1) < room || m->stride(dim - 1) != 1) return false;
  for (int64_t i = 0; i + 1 < dim; ++i)
    if (m->stride(i) < (m->size(i) > 1 ? room : 0)) return false;
  return true;
}

PyObject* mass(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || a[8] != Py_False) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor* m = tensor(a[5]);
  Attend t;
  if (!t.read(a, a[6], a[7], dev) || !mass_ok(m, 3, t.p.width * t.p.page, dev) || m->size(0) != t.batch || m->size(1) != t.p.heads ||
      !t.room(abi.mass_size(static_cast<int>(t.batch), static_cast<int>(t.heads), static_cast<int>(t.p.heads),
                            static_cast<int>(t.p.hd), t.p.width * t.p.page)))
    Py_RETURN_NONE;
  return t.launch(abi.mass, dev, m->data_ptr<float>(), m->stride(0), m->stride(1));
  END_HANDLE_TH_ERRORS
}

PyObject* sparse(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || a[8] != Py_False) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor* blocks = tensor(a[5]);
  Attend t;
  if (!is(blocks, at::kInt, 3, dev) || !blocks->is_contiguous() || !t.read(a, a[6], a[7], dev) || blocks->size(0) != t.batch ||
      blocks->size(1) != t.p.heads || blocks->size(2) < 1 || blocks->size(2) > INT32_MAX ||
      !t.room(abi.attend_size(static_cast<int>(t.batch), static_cast<int>(t.heads), static_cast<int>(t.p.hd))))
    Py_RETURN_NONE;
  return t.launch(abi.sparse, dev, blocks->data_ptr<int>(), static_cast<int>(blocks->size(2)));
  END_HANDLE_TH_ERRORS
}

// A page table and its streams' lengths.
struct Table {
  const Tensor *table, *lens;
  int64_t streams, width;
  bool read(PyObject* const* a, int dev) {
    table = tensor(a[0]);
    lens = tensor(a[1]);
    if (!is(table, at::kInt, 2, dev) || !is(lens, at::kInt, 1, dev)) return false;
    streams = table->size(0), width = table->size(1);
    return streams > 0 && width > 0 && streams <= INT32_MAX && width <= INT32_MAX && (table->stride(1) == 1 || width == 1) &&
           lens->size(0) == streams && lens->is_contiguous();
  }
  int64_t stride() const { return streams > 1 ? table->stride(0) : width; }
};

PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !PyBool_Check(a[7])) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *pool = tensor(a[0]), *m = tensor(a[3]);
  Table t;
  int keep, recent, sinks;
  if (!is(pool, at::kBFloat16, 6, dev) || !pool->is_contiguous() || pool->numel() == 0 || pool->size(1) != 2 || !t.read(a + 1, dev) ||
      !number(a[4], &keep) || !number(a[5], &recent) || !number(a[6], &sinks) || keep < 1 || recent < 0 || sinks < 0 ||
      recent > keep || sinks > keep - recent)
    Py_RETURN_NONE;
  const int64_t layers = pool->size(0), pages = pool->size(2), heads = pool->size(3), page = pool->size(4), hd = pool->size(5);
  if (layers > INT32_MAX || pages > INT32_MAX || heads > INT32_MAX || page > INT32_MAX || hd > INT32_MAX ||
      !mass_ok(m, 4, t.width * page, dev) || m->size(0) != layers || m->size(1) != t.streams || m->size(2) != heads)
    Py_RETURN_NONE;
  const size_t need = abi.evict_size(static_cast<int>(layers), static_cast<int>(t.streams), static_cast<int>(heads), t.width * page, keep);
  Tensor ws = at::empty({static_cast<int64_t>(need)}, pool->options().dtype(at::kByte)), source;
  if (a[7] == Py_True) source = at::empty({layers, t.streams, heads, keep}, pool->options().dtype(at::kInt));
  const int rc = abi.evict(pool->data_ptr(), static_cast<int>(layers), static_cast<int>(pages), static_cast<int>(page),
                           static_cast<int>(heads), static_cast<int>(hd), t.table->data_ptr<int>(), t.stride(),
                           static_cast<int>(t.width), t.lens->data_ptr<int>(), m->data_ptr<float>(), m->stride(0), m->stride(1),
                           m->stride(2), static_cast<int>(t.streams), keep, recent, sinks,
                           source.defined() ? source.data_ptr<int>() : nullptr, ws.data_ptr(), need, current_stream(dev));
  if (rc) return status(rc);
  if (source.defined()) return THPVariable_Wrap(std::move(source));
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

bool bounds_ok(const Tensor* b, int dev) {
  return is(b, at::kBFloat16, 4, dev) && b->is_contiguous() && b->numel() > 0 && b->size(2) == 2 && b->size(0) <= INT32_MAX;
}

PyObject* bounds(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *k = tensor(a[0]), *b = tensor(a[1]), *cu;
  Table t;
  if (!is(k, at::kBFloat16, 4, dev) || k->numel() == 0 || k->stride(3) != 1 || !bounds_ok(b, dev) || !t.read(a + 2, dev) ||
      !dense_or_none(a[4], &cu, at::kInt, {t.streams + 1}, dev))
    Py_RETURN_NONE;
  const int64_t pages = k->size(0), heads = k->size(1), page = k->size(2), hd = k->size(3);
  if (b->size(0) != pages || b->size(1) != heads || b->size(3) != hd || heads > INT32_MAX || page > INT32_MAX || hd > INT32_MAX)
    Py_RETURN_NONE;
  auto stride = [&](int axis) { return k->size(axis) > 1 ? k->stride(axis) : std::max(k->stride(axis), hd); };
  const int rc = abi.bounds(k->data_ptr(), stride(0), stride(1), stride(2), static_cast<int>(pages), static_cast<int>(page),
                            t.table->data_ptr<int>(), t.stride(), static_cast<int>(t.width), t.lens->data_ptr<int>(),
                            cu ? cu->data_ptr<int>() : nullptr, static_cast<int>(t.streams), static_cast<int>(heads),
                            static_cast<int>(hd), b->data_ptr(), current_stream(dev));
  if (rc) return status(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *q = tensor(a[0]), *b = tensor(a[1]);
  Table t;
  int page, count, first, last;
  if (!is(q, at::kBFloat16, 3, dev) || !bounds_ok(b, dev) || !t.read(a + 2, dev) || !number(a[4], &page) || !number(a[5], &count) ||
      !number(a[6], &first) || !number(a[7], &last) || page < 1 || count < 1 || first < 0 || last < 0 || first > count ||
      last > count - first)
    Py_RETURN_NONE;
  const int64_t batch = q->size(0), heads = q->size(1), hd = q->size(2), hkv = b->size(1);
  if (batch != t.streams || hd != b->size(3) || heads < 1 || heads % hkv || heads > INT32_MAX || hd > INT32_MAX ||
      (q->stride(2) != 1 && hd > 1))
    Py_RETURN_NONE;
  Tensor blocks = at::empty({batch, hkv, count}, t.table->options());
  const size_t need = abi.select_size(static_cast<int>(batch), static_cast<int>(hkv), static_cast<int>(t.width));
  Tensor ws = at::empty({static_cast<int64_t>(need)}, t.table->options().dtype(at::kByte));
  const int rc = abi.select(q->data_ptr(), q->stride(0), q->stride(1), b->data_ptr(), static_cast<int>(b->size(0)), page,
                            t.table->data_ptr<int>(), t.stride(), static_cast<int>(t.width), t.lens->data_ptr<int>(),
                            static_cast<int>(batch), static_cast<int>(heads), static_cast<int>(hkv), static_cast<int>(hd), count,
                            first, last, blocks.data_ptr<int>(), ws.data_ptr(), need, current_stream(dev));
  return rc ? status(rc) : THPVariable_Wrap(std::move(blocks));
  END_HANDLE_TH_ERRORS
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 10 && n != 11) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *qkv = tensor(a[0]), *cos = tensor(a[5]), *sin = tensor(a[6]), *cu, *angle = nullptr;
  Pages p;
  int heads;
  if (!is(qkv, at::kBFloat16, 2, dev) || !p.read(a + 1, dev) || !is(cos, at::kFloat, 2, dev) ||
      !dense(sin, at::kFloat, cos->sizes(), dev) || !cos->is_contiguous() || !number(a[7], &heads) || heads < 1 ||
      !dense_or_none(a[8], &cu, at::kInt, {p.streams + 1}, dev) || !PyBool_Check(a[9]))
    Py_RETURN_NONE;
  const int64_t tokens = qkv->size(0), width = (heads + 2 * p.heads) * p.hd;
  if (tokens < 1 || tokens > INT32_MAX || qkv->size(1) != width || qkv->stride(1) != 1 || cos->size(0) < 1 ||
      cos->size(0) > INT32_MAX || 2 * cos->size(1) > p.hd || (!cu && tokens != p.streams) || p.streams > INT32_MAX ||
      (n == 11 && !dense_or_none(a[10], &angle, at::kInt, {tokens}, dev)))
    Py_RETURN_NONE;
  Tensor q = at::empty({tokens, heads, p.hd}, qkv->options());
  auto launch = [&](auto f, auto... positions) {
    return f(qkv->data_ptr(), tokens > 1 ? qkv->stride(0) : width, q.data_ptr(), p.k->data_ptr(), p.stride(p.k, 0),
             p.stride(p.k, 1), p.stride(p.k, 2), p.v->data_ptr(), p.stride(p.v, 0), p.stride(p.v, 1), p.stride(p.v, 2),
             static_cast<int>(p.n), static_cast<int>(p.page), p.table->data_ptr<int>(), p.table_stride(),
             static_cast<int>(p.width), p.lens->data_ptr<int>(), cu ? cu->data_ptr<int>() : nullptr, positions...,
             cos->data_ptr<float>(), sin->data_ptr<float>(), static_cast<int>(cos->size(0)), static_cast<int>(tokens),
             static_cast<int>(p.streams), heads, static_cast<int>(p.heads), static_cast<int>(p.hd),
             static_cast<int>(2 * cos->size(1)), static_cast<int>(a[9] == Py_True), current_stream(dev));
  };
  const int rc = angle ? launch(abi.append_at, static_cast<const int*>(angle->data_ptr<int>())) : launch(abi.append);
  return rc ? status(rc) : THPVariable_Wrap(std::move(q));
  END_HANDLE_TH_ERRORS
}

PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *pool = tensor(a[0]), *src = tensor(a[1]), *dst = tensor(a[2]);
  if (!pool || !pool->is_cuda() || pool->get_device() != dev || pool->dim() < 4 || !pool->is_contiguous() ||
      pool->numel() == 0 || !is(src, at::kInt, 1, dev) || !src->is_contiguous() || !dense(dst, at::kInt, src->sizes(), dev))
    Py_RETURN_NONE;
  const int64_t pages = pool->size(-4), bytes = pool->size(-1) * pool->size(-2) * pool->size(-3) * pool->element_size();
  const int64_t outer = pool->numel() * pool->element_size() / (pages * bytes);
  if (pages > INT32_MAX || outer > INT32_MAX || src->size(0) > INT32_MAX) Py_RETURN_NONE;
  const int rc = abi.copy(pool->data_ptr(), pages * bytes, bytes, bytes, static_cast<int>(outer), static_cast<int>(pages),
                          src->data_ptr<int>(), dst->data_ptr<int>(), static_cast<int>(src->size(0)), current_stream(dev));
  if (rc) return status(rc);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 14) Py_RETURN_NONE;
  const int dev = current_device();
  const Tensor *zx = tensor(a[0]), *conv = tensor(a[1]), *w = tensor(a[2]), *ssm = tensor(a[4]), *A = tensor(a[5]), *bias, *D,
               *dtb, *cu = nullptr;
  int di, ng, ds, nh;
  if (!is(zx, at::kBFloat16, 2, dev) || !is(conv, at::kBFloat16, 3, dev) || !number(a[8], &di) || !number(a[9], &ng) ||
      !number(a[10], &ds) || !number(a[11], &nh) || di < 1 || ng < 1 || ds < 1 || nh < 1 || di % nh || nh % ng ||
      !PyBool_Check(a[13]))
    Py_RETURN_NONE;
  int64_t batch = 1;
  if (a[12] != Py_None) {
    cu = tensor(a[12]);
    if (!is(cu, at::kInt, 1, dev) || !cu->is_contiguous()) Py_RETURN_NONE;
    batch = cu->size(0) - 1;
  }
  const int64_t tokens = zx->size(0), cd = di + 2 * static_cast<int64_t>(ng) * ds, W = conv->size(2);
  if (tokens < 1 || tokens > INT32_MAX || batch < 1 || batch > INT32_MAX || zx->size(1) < di + cd + nh || zx->stride(1) != 1 ||
      W > INT32_MAX || !dense(conv, at::kBFloat16, {batch, cd, W}, dev) || !dense(w, at::kBFloat16, {cd, W}, dev) ||
      !dense(ssm, at::kBFloat16, {batch, nh, di / nh, ds}, dev) || !dense(A, at::kFloat, {nh}, dev) ||
      !dense_or_none(a[3], &bias, at::kBFloat16, {cd}, dev) || !dense_or_none(a[6], &D, at::kBFloat16, {nh}, dev) ||
      !dense_or_none(a[7], &dtb, at::kBFloat16, {nh}, dev))
    Py_RETURN_NONE;
  const size_t need = abi.prompt_size(static_cast<int>(tokens), static_cast<int>(batch), di, ng, ds, nh);
  Tensor y = at::empty({tokens, nh, di / nh}, zx->options());
  Tensor ws = at::empty({static_cast<int64_t>(need)}, zx->options().dtype(at::kByte));
  const int rc = abi.prompt(zx->data_ptr(), tokens > 1 ? zx->stride(0) : zx->size(1), conv->data_ptr(), w->data_ptr(),
                            ptr(bias), ssm->data_ptr(), A->data_ptr<float>(), ptr(D), ptr(dtb), y.data_ptr(),
                            cu ? cu->data_ptr<int>() : nullptr, static_cast<int>(batch), static_cast<int>(tokens), di, ng, ds,
                            nh, di / nh, static_cast<int>(W), a[13] == Py_True, ws.data_ptr(), need, current_stream(dev));
  return rc ? status(rc) : THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

// bind({name: address}) of the C ABI's functions.
PyObject* bind(PyObject*, PyObject* table) {
  auto get = [&](const char* name, auto& f) {
    PyObject* o = PyDict_Check(table) ? PyDict_GetItemString(table, name) : nullptr;
    void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
    if (!p) {
      if (!PyErr_Occurred()) PyErr_Format(PyExc_KeyError, "%s", name);
      return false;
    }
    f = reinterpret_cast<std::decay_t<decltype(f)>>(p);
    return true;
  };
  if (!get("sn_paged_decode_attention", abi.attend) || !get("sn_paged_decode_workspace_size", abi.attend_size) ||
      !get("sn_rotary_paged_append", abi.append) || !get("sn_rotary_paged_append_at", abi.append_at) || !get("sn_copy_pages", abi.copy) ||
      !get("sn_mamba2_prompt", abi.prompt) || !get("sn_mamba2_prompt_workspace_size", abi.prompt_size) ||
      !get("sn_paged_decode_attention_mass", abi.mass) || !get("sn_paged_mass_workspace_size", abi.mass_size) ||
      !get("sn_evict_positions", abi.evict) || !get("sn_evict_workspace_size", abi.evict_size) ||
       !get("sn_update_page_bounds", abi.bounds) ||
      !get("sn_select_blocks", abi.select) ||
      !get("sn_select_blocks_workspace_size", abi.select_size) || !get("sn_paged_sparse_attention", abi.sparse))
    return nullptr;
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef methods[] = {{"attend", FAST(attend)}, {"append", FAST(append)}, {"copy", FAST(copy)}, {"prompt", FAST(prompt)},
                         {"mass", FAST(mass)}, {"evict", FAST(evict)}, {"bounds", FAST(bounds)}, {"select", FAST(select)}, {"sparse", FAST(sparse)},
                         {"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall() { return PyModule_Create(&module); }
