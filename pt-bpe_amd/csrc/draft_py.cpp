// draft_py.cpp -- geobpe._draft: the checks and the C calls of geobpe/draft.py (which documents them).  In C++
// because a decoding step makes these calls hundreds of times: checked in Python each took 20 to 25 us on the host, more
// than the kernels of small calls.  The entries of libgeobpe.so are bound by address (geobpe._native has loaded it), so
// this module needs the process's PyTorch and nothing else.
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <cstdlib>
#include <functional>
#include <initializer_list>
#include <string>
#include <utility>

#include "../../include/geobpe.h"

namespace {

struct {
  decltype(&geobpe_tree_attention) attend;
  decltype(&geobpe_tree_attention_work) attend_work;
  decltype(&geobpe_verify_draft) verify;
  decltype(&geobpe_commit_draft) commit;
  decltype(&geobpe_draft_error) error;
} lib;
PyObject* geobpe_error;  // geobpe._native.GeoBPEError

constexpr int64_t MAX_NODES = 128, MAX_VOCAB = 1 << 22, MAX_POSITIONS = 0x7ffff000;
constexpr double MAX_SCALE = 2e38;  // times log2 e it is one of float32's finite numbers

struct Refused {};  // thrown with the Python error set

template <typename... A>
[[noreturn]] void refuse(PyObject* kind, const char* fmt, A... a) {
  PyErr_Format(kind, fmt, a...);
  throw Refused();
}
#define VALUE(...) refuse(PyExc_ValueError, __VA_ARGS__)

std::string shape_of(const at::Tensor& x) {
  std::string s = "(";
  for (int64_t i = 0; i < x.dim(); i++) s += (i ? ", " : "") + std::to_string(x.size(i));
  return s + ")";
}

const at::Tensor& tensor(const char* name, PyObject* o) {
  if (!THPVariable_Check(o))
    refuse(PyExc_TypeError, "%s: a torch tensor is expected, not %s", name, Py_TYPE(o)->tp_name);
  const at::Tensor& x = THPVariable_Unpack(o);
  if (x.is_conj() || x.is_neg())
    VALUE("%s is a view that negates or conjugates: pass %s.resolve_conj().resolve_neg()", name, name);
  return x;
}

// x as an operand: its type, its device, its shape (-1: any size)
const at::Tensor& operand(const char* name, PyObject* o, std::initializer_list<at::ScalarType> types, at::Device device,
                          std::initializer_list<int64_t> shape) {
  const at::Tensor& x = tensor(name, o);
  bool ok = false;
  for (at::ScalarType t : types) ok |= x.scalar_type() == t;
  if (!ok) {
    std::string want;
    for (at::ScalarType t : types) want += std::string(want.empty() ? "" : " or ") + at::toString(t);
    refuse(PyExc_TypeError, "%s is of type %s, expected %s", name, at::toString(x.scalar_type()), want.c_str());
  }
  if (x.device() != device) VALUE("%s is on %s, not on %s", name, x.device().str().c_str(), device.str().c_str());
  ok = x.dim() == (int64_t)shape.size();
  int64_t i = 0;
  for (int64_t n : shape) {
    ok = ok && (n < 0 || x.size(i) == n);
    i++;
  }
  if (!ok) {
    std::string want;
    for (int64_t n : shape) want += (want.empty() ? "" : ", ") + (n < 0 ? std::string("any") : std::to_string(n));
    VALUE("%s: shape %s, expected (%s)", name, shape_of(x).c_str(), want.c_str());
  }
  return x;
}

// strides in units of `scale` bytes of a tensor read in 16-byte pieces of its last dimension
void rows(const char* name, const at::Tensor& x, int64_t* out, int64_t scale) {
  const int64_t e = x.element_size(), dims = x.dim();
  bool ok = (x.stride(dims - 1) == 1 || x.size(dims - 1) <= 1) && (uintptr_t)x.data_ptr() % 16 == 0;
  for (int64_t i = 0; i + 1 < dims; i++) {
    const int64_t s = x.size(i) > 1 ? x.stride(i) : 0;
    ok = ok && s * e % 16 == 0;
    out[i] = s * e / scale;
  }
  if (!ok) VALUE("%s: rows must be contiguous and 16-byte aligned: pass %s.contiguous()", name, name);
}

// whether two tensors' spans of memory meet
bool meet(const at::Tensor& x, const at::Tensor& y) {
  const at::Tensor* t[2] = {&x, &y};
  uintptr_t from[2], to[2];
  for (int i = 0; i < 2; i++) {
    int64_t last = 0;
    for (int64_t d = 0; d < t[i]->dim(); d++) last += (t[i]->size(d) - 1) * t[i]->stride(d);
    from[i] = (uintptr_t)t[i]->data_ptr();
    to[i] = t[i]->numel() ? from[i] + (last + 1) * t[i]->element_size() : from[i];
  }
  return from[0] < to[1] && from[1] < to[0];
}

// Whether elements of two tensors of x's sizes and strides, the second `apart` elements further on, share memory (of one tensor,
// apart = 0: two different elements): index differences d with sum d stride = apart.  Largest strides first: of an ordinary
// layout's only a d or two a dimension leave what the smaller ones can make up for.
struct Shared {
  static constexpr int MOST = 5;             // dimensions of a cache
  std::pair<int64_t, int64_t> dims[MOST];    // stride, size
  int64_t rest[MOST + 1] = {}, steps = 0;    // what the dimensions from i on span at most
  int n_dims = 0;
  bool nested = true;  // every stride passes over what the smaller ones span: no two elements of the tensor meet
  explicit Shared(const at::Tensor& x) {
    for (int64_t i = 0; i < x.dim(); i++)
      if (x.size(i) > 1) dims[n_dims++] = {x.stride(i), x.size(i)};
    std::sort(dims, dims + n_dims, std::greater<>());
    for (int i = n_dims; i-- > 0;) {
      rest[i] = rest[i + 1] + dims[i].first * (dims[i].second - 1);
      nested = nested && dims[i].first > rest[i + 1];
    }
  }
  bool any(int64_t apart, int i, bool differ) {
    if (i == n_dims) return apart == 0 && differ;
    if (std::abs(apart) > rest[i] || ++steps > 10000) return false;  // (strides of no ordinary layout: not looked through)
    const int64_t s = dims[i].first, n = dims[i].second;
    if (s == 0) return any(apart, i + 1, true);  // (the smallest: all others were chosen)
    int64_t from = (apart - rest[i + 1]) / s - 1, to = (apart + rest[i + 1]) / s + 1;
    from = std::max(from, 1 - n), to = std::min(to, n - 1);
    for (int64_t d = from; d <= to; d++)
      if (any(apart - d * s, i + 1, differ || d)) return true;
    return false;
  }
};

bool unit(const at::Tensor& x) { return x.size(-1) <= 1 || x.stride(-1) == 1; }

// a contiguous tensor over a part of another's memory: three outputs of one allocation (three at::empty took 2 us longer)
at::Tensor part_of(const at::Tensor& all, int64_t at, at::IntArrayRef shape) {
  at::Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  x.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
  x.unsafeGetTensorImpl()->set_storage_offset(all.storage_offset() + at);
  return x;
}

hipStream_t stream_of(at::Device device) {
  if (!device.is_cuda()) VALUE("tensors on %s: the decoding operators run on a HIP device only", device.str().c_str());
  return c10::hip::getCurrentHIPStream(device.index()).stream();
}

// no derivatives: neither backward nor forward ones, which no_grad() leaves on
void no_grad(std::initializer_list<const at::Tensor*> xs) {
  const c10::AutogradState& now = c10::AutogradState::get_tls_state();
  for (const at::Tensor* x : xs) {
    if (!x) continue;
    if (now.get_grad_mode() && x->requires_grad())
      VALUE("the decoding operators have no backward: call them under torch.no_grad()");
    if (now.get_fw_grad_mode() && x->_fw_grad(0).defined())
      VALUE("the decoding operators have no backward and take no tangents: call them on the primal tensors");
  }
}

void nodes(int64_t N) {
  if (N < 1 || N > MAX_NODES) VALUE("a tree has 1 to %lld nodes, not %lld", (long long)MAX_NODES, (long long)N);
}

struct Tree {
  const at::Tensor* t;
  int64_t stride;
};
Tree parents_of(PyObject* o, int64_t B, int64_t N, at::Device device) {
  const bool one = tensor("parents", o).dim() == 1;
  const at::Tensor& x = one ? operand("parents", o, {at::kInt}, device, {N}) : operand("parents", o, {at::kInt}, device, {B, N});
  if (!unit(x)) VALUE("parents: the nodes must be contiguous");
  return {&x, one || B <= 1 ? 0 : x.stride(0)};
}

struct Cache {
  const at::Tensor *k, *v, *table, *lens;
  int64_t B, P, S, M, Hkv, D, table_stride;
};
void called(int rc) {
  if (rc == GEOBPE_OK) return;
  refuse(rc == GEOBPE_EARG ? PyExc_ValueError : geobpe_error, "%s (code %d)", lib.error(), rc);
}

int half_of(at::ScalarType t) { return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : 2; }

#define GUARDED(n)                                                                             \
  HANDLE_TH_ERRORS                                                                             \
  if (nargs != n) {                                                                            \
    PyErr_Format(PyExc_TypeError, "%d arguments are expected, not %zd", n, nargs);             \
    return nullptr;                                                                            \
  }                                                                                            \
  if (!lib.error) {                                                                            \
    PyErr_SetString(PyExc_RuntimeError, "geobpe._draft is not bound: use geobpe.draft");       \
    return nullptr;                                                                            \
  }                                                                                            \
  try {
#define END_GUARDED          \
  }                          \
  catch (const Refused&) {   \
    return nullptr;          \
  }                          \
  END_HANDLE_TH_ERRORS

// the paged cache's checks
Cache cache_checks(PyObject* const* o, bool layers, std::initializer_list<at::ScalarType> types, at::Device device) {
  Cache c;
  c.k = &tensor("k_cache", o[0]);
  if (layers)
    operand("k_cache", o[0], types, device, {-1, -1, -1, -1, -1});
  else
    operand("k_cache", o[0], types, device, {-1, -1, -1, -1});
  c.v = &tensor("v_cache", o[1]);
  if (c.v->scalar_type() != c.k->scalar_type())
    refuse(PyExc_TypeError, "v_cache is of type %s, k_cache of %s", at::toString(c.v->scalar_type()),
           at::toString(c.k->scalar_type()));
  if (c.v->device() != device) VALUE("v_cache is on %s, not on %s", c.v->device().str().c_str(), device.str().c_str());
  if (c.v->sizes() != c.k->sizes())
    VALUE("v_cache: shape %s, expected %s", shape_of(*c.v).c_str(), shape_of(*c.k).c_str());
  c.lens = &operand("lens", o[3], {at::kInt}, device, {-1});
  c.B = c.lens->size(0);
  c.table = &operand("block_table", o[2], {at::kInt}, device, {c.B, -1});
  c.P = c.k->size(-4), c.S = c.k->size(-3), c.Hkv = c.k->size(-2), c.D = c.k->size(-1);
  c.M = c.table->size(1);
  if (c.P < 1 || c.S < 1) VALUE("k_cache: a cache has at least one page of one position");
  if (c.M > MAX_POSITIONS / c.S)
    VALUE("block_table: %lld pages of %lld positions are more than %lld", (long long)c.M, (long long)c.S,
          (long long)MAX_POSITIONS);
  if (!unit(*c.table)) VALUE("block_table: a sequence's pages must be contiguous");
  if (!unit(*c.lens)) VALUE("lens must be contiguous");
  c.table_stride = c.B > 1 ? c.table->stride(0) : 0;
  return c;
}

// q, k_cache, v_cache, block_table, lens, k, v, parents, scale
PyObject* tree_attention(PyObject*, PyObject* const* o, Py_ssize_t nargs) {
  GUARDED(9)
  const at::Device dev = tensor("q", o[0]).device();
  const at::Tensor& q = operand("q", o[0], {at::kBFloat16, at::kHalf}, dev, {-1, -1, -1, -1});
  const at::ScalarType type = q.scalar_type();
  const int64_t B = q.size(0), N = q.size(1), Hq = q.size(2), D = q.size(3);
  nodes(N);
  if (D % 8 || D < 8 || D > 256) VALUE("head dimension %lld: a multiple of 8 up to 256 is expected", (long long)D);
  const Cache c = cache_checks(o + 1, false, {type}, dev);
  if (c.B != B || c.D != D)
    VALUE("q %s does not fit %lld sequences and heads of %lld", shape_of(q).c_str(), (long long)c.B, (long long)c.D);
  if (c.Hkv < 1 || Hq < 1 || Hq % c.Hkv) VALUE("%lld query heads over %lld key heads", (long long)Hq, (long long)c.Hkv);
  const at::Tensor& k = operand("k", o[5], {type}, dev, {B, N, c.Hkv, D});
  const at::Tensor& v = operand("v", o[6], {type}, dev, {B, N, c.Hkv, D});
  const Tree tree = parents_of(o[7], B, N, dev);
  double scale = 1.0 / std::sqrt((double)D);
  if (o[8] != Py_None) {
    scale = PyFloat_AsDouble(o[8]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused();
    if (!(std::fabs(scale) <= MAX_SCALE)) VALUE("scale %R: a finite number up to 2e38 in size is expected", o[8]);
  }
  no_grad({&q, c.k, c.v, &k, &v});
  geobpe_attend_args a;
  rows("q", q, a.q_stride, 2);
  rows("k", k, a.k_stride, 2);
  rows("v", v, a.v_stride, 2);
  rows("k_cache", *c.k, a.kc_stride, 2);
  rows("v_cache", *c.v, a.vc_stride, 2);
  const hipStream_t stream = stream_of(dev);
  at::Tensor out = at::empty({B, N, Hq, D}, q.options());
  a.d_q = q.data_ptr(), a.d_k_cache = c.k->data_ptr(), a.d_v_cache = c.v->data_ptr();
  a.d_k = k.data_ptr(), a.d_v = v.data_ptr(), a.d_out = out.data_ptr();
  a.d_table = c.table->data_ptr(), a.d_lens = c.lens->data_ptr(), a.d_parents = tree.t->data_ptr();
  a.table_stride = c.table_stride, a.parents_stride = tree.stride;
  a.seqs = B, a.nodes = N, a.heads = Hq, a.kv_heads = c.Hkv, a.head_dim = D;
  a.page_size = c.S, a.pages = c.P, a.max_pages = c.M, a.dtype = half_of(type), a.scale = scale;
  const int64_t need = lib.attend_work(&a);
  at::Tensor work;
  if (need > 0) work = at::empty({need}, q.options().dtype(at::kByte));
  called(lib.attend(dev.index(), stream, &a, need > 0 ? work.data_ptr() : nullptr, need));
  return THPVariable_Wrap(std::move(out));
  END_GUARDED
}

// parents, ids, target, draft, u, ranges, start
PyObject* verify(PyObject*, PyObject* const* o, Py_ssize_t nargs) {
  GUARDED(7)
  const at::Device dev = tensor("target", o[2]).device();
  const at::Tensor& target = operand("target", o[2], {at::kFloat, at::kBFloat16, at::kHalf}, dev, {-1, -1, -1});
  const int64_t B = target.size(0), N = target.size(1), V = target.size(2);
  nodes(N);
  if (V < 1 || V > MAX_VOCAB) VALUE("a vocabulary of %lld: 1 to %lld are expected", (long long)V, (long long)MAX_VOCAB);
  const at::Tensor& ids = operand("ids", o[1], {at::kLong, at::kInt}, dev, {B, N});
  const at::Tensor& u = operand("u", o[4], {at::kFloat}, dev, {B, N});
  const at::Tensor* draft = o[3] == Py_None ? nullptr : &operand("draft", o[3], {target.scalar_type()}, dev, {B, N, V});
  const Tree tree = parents_of(o[0], B, N, dev);
  if ((o[5] == Py_None) != (o[6] == Py_None)) VALUE("ranges and start belong together");
  const at::Tensor *ranges = nullptr, *start = nullptr;
  if (o[5] != Py_None) {
    ranges = &operand("ranges", o[5], {at::kInt}, dev, {-1, 2});
    start = &operand("start", o[6], {at::kInt}, dev, {B});
    if (ranges->size(0) < 1 || !ranges->is_contiguous() || !start->is_contiguous())
      VALUE("ranges and start must be contiguous and not empty");
  }
  if (!unit(ids)) VALUE("ids: the last dimension must be contiguous");
  if (!unit(u)) VALUE("u: the last dimension must be contiguous");
  if (!unit(target)) VALUE("target: the last dimension must be contiguous");
  if (draft && !unit(*draft)) VALUE("draft: the last dimension must be contiguous");
  no_grad({&target, draft});
  const hipStream_t stream = stream_of(dev);
  const at::TensorOptions ints = target.options().dtype(at::kInt);
  const at::Tensor all = at::empty({B + 2 * B * N}, ints);
  at::Tensor n = part_of(all, 0, {B}), path = part_of(all, B, {B, N}), tokens = part_of(all, B + B * N, {B, N});
  geobpe_verify_args a;
  a.d_parents = tree.t->data_ptr(), a.d_ids = ids.data_ptr(), a.d_target = target.data_ptr();
  a.d_draft = draft ? draft->data_ptr() : nullptr, a.d_u = u.data_ptr();
  a.d_ranges = ranges ? ranges->data_ptr() : nullptr, a.d_start = start ? start->data_ptr() : nullptr;
  a.d_n = n.data_ptr(), a.d_path = path.data_ptr(), a.d_tokens = tokens.data_ptr();
  for (int i = 0; i < 2; i++) a.target_stride[i] = target.stride(i), a.draft_stride[i] = draft ? draft->stride(i) : 0;
  a.parents_stride = tree.stride, a.ids_stride = ids.stride(0), a.u_stride = u.stride(0);
  a.seqs = B, a.nodes = N, a.vocab = V, a.classes = ranges ? ranges->size(0) : 0;
  a.ids_int64 = ids.scalar_type() == at::kLong, a.dtype = half_of(target.scalar_type());
  called(lib.verify(dev.index(), stream, &a));
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(n)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(path)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(tokens)));
  return r;
  END_GUARDED
}

// k_cache, v_cache, block_table, lens, k, v, path, n
PyObject* commit(PyObject*, PyObject* const* o, Py_ssize_t nargs) {
  GUARDED(8)
  const at::Tensor& kc = tensor("k_cache", o[0]);
  const at::Device dev = kc.device();
  const bool layers = kc.dim() == 5;
  const Cache c = cache_checks(o, layers, {kc.scalar_type()}, dev);
  const at::Tensor& path = operand("path", o[6], {at::kInt}, dev, {c.B, -1});
  const int64_t N = path.size(1), L = layers ? kc.size(0) : 1, e = kc.element_size();
  nodes(N);
  const at::Tensor *x[2];
  for (int i = 0; i < 2; i++) {
    const char* name = i ? "v" : "k";
    x[i] = layers ? &operand(name, o[4 + i], {kc.scalar_type()}, dev, {L, c.B, N, c.Hkv, c.D})
                  : &operand(name, o[4 + i], {kc.scalar_type()}, dev, {c.B, N, c.Hkv, c.D});
  }
  const at::Tensor& n = operand("n", o[7], {at::kInt}, dev, {c.B});
  if (!unit(path) || !unit(n)) VALUE("path and n must be contiguous");
  if (L < 1) VALUE("k_cache: a cache has at least one layer");
  if (c.Hkv < 1 || c.D < 1 || c.D * e % 16 || c.D * e > 65536)
    VALUE("heads of %lld x %lld bytes: a multiple of 16 bytes is expected", (long long)c.D, (long long)e);
  no_grad({c.k, c.v, x[0], x[1]});
  geobpe_commit_args a;
  int64_t* st[4] = {a.k_stride, a.v_stride, a.kc_stride, a.vc_stride};
  const at::Tensor* all[4] = {x[0], x[1], c.k, c.v};
  const char* names[4] = {"k", "v", "k_cache", "v_cache"};
  for (int i = 0; i < 4; i++) {
    st[i][0] = 0;
    rows(names[i], *all[i], st[i] + !layers, 1);
    if (i < 2) continue;
    Shared own(*all[i]);
    if (!own.nested && own.any(0, 0, false)) VALUE("%s is expanded or its rows overlap: they share memory", names[i]);
  }
  for (int i = 0; i < 2; i++)
    if (meet(*x[i], *c.k) || meet(*x[i], *c.v))
      VALUE("%s lies in the cache's own memory, which the call writes: pass %s.clone()", names[i], names[i]);
  if (c.k->data_ptr() == c.v->data_ptr()) VALUE("v_cache is k_cache: each needs memory of its own");
  if (c.k->strides() == c.v->strides() && meet(*c.k, *c.v) &&
      Shared(*c.k).any(((const char*)c.v->data_ptr() - (const char*)c.k->data_ptr()) / e, 0, true))
    VALUE("v_cache is partly k_cache: each needs memory of its own");
  const hipStream_t stream = stream_of(dev);
  at::Tensor out = at::empty({c.B}, c.lens->options());
  a.d_k = x[0]->data_ptr(), a.d_v = x[1]->data_ptr(), a.d_k_cache = c.k->data_ptr(), a.d_v_cache = c.v->data_ptr();
  a.d_table = c.table->data_ptr(), a.d_lens = c.lens->data_ptr(), a.d_path = path.data_ptr(), a.d_n = n.data_ptr();
  a.d_lens_out = out.data_ptr();
  a.table_stride = c.table_stride, a.path_stride = c.B > 1 ? path.stride(0) : 0;
  a.layers = L, a.seqs = c.B, a.nodes = N, a.kv_heads = c.Hkv, a.head_bytes = c.D * e;
  a.page_size = c.S, a.pages = c.P, a.max_pages = c.M;
  called(lib.commit(dev.index(), stream, &a));
  for (const at::Tensor* x : {c.k, c.v})  // they were written: a backward pass that needs them as they were has to see it
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(std::move(out));
  END_GUARDED
}

// the entries' addresses and the error class
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[5];
  PyObject* error;
  if (!PyArg_ParseTuple(args, "KKKKKO", &p[0], &p[1], &p[2], &p[3], &p[4], &error)) return nullptr;
  Py_INCREF(error);
  geobpe_error = error;
  lib.attend = (decltype(lib.attend))p[0];
  lib.attend_work = (decltype(lib.attend_work))p[1];
  lib.verify = (decltype(lib.verify))p[2];
  lib.commit = (decltype(lib.commit))p[3];
  lib.error = (decltype(lib.error))p[4];
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, nullptr},
                         {"tree_attention", (PyCFunction)(void (*)(void))tree_attention, METH_FASTCALL, nullptr},
                         {"verify", (PyCFunction)(void (*)(void))verify, METH_FASTCALL, nullptr},
                         {"commit", (PyCFunction)(void (*)(void))commit, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_draft", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__draft() { return PyModule_Create(&module); }
