// The calls of the paged caches and of prompt attention from Python: argument checks and argument blocks (include/tqb200.h) without the interpreter.
// A decode step's kernels take 2 to 20 us, so the host's share of a call counts when it is not replayed from a CUDA
// graph: the same checks written in Python took 11 us of the 17 us of a single-token decode call, here about 1.
//
// Module _calls; `paged.py` and `kernels.py` hold the signatures and their documentation.  The entry points come in by address
// (bind), so that whichever libtqb200.so the package has loaded is the one that is called.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <map>
#include <set>
#include <tuple>
#include <vector>

#include "tqb200.h"

namespace {

struct Entry {
  int (*decode)(const tq_paged_params*);
  int (*append)(const tq_paged_params*);
  int (*dequantize)(const tq_paged_params*);
  int64_t (*workspace_bytes)(int);
  int (*copy)(void* const*, const int64_t*, int, int64_t, const int32_t*, const int32_t*, int64_t, void*);
  int (*prefill)(const tq_prefill_params*);
} entry;
PyObject *host_floats, *host_cache, *check_status;      // of the package's _lib (borrowed for good)

// Interned names: dictionary lookups compare pointers.
struct Names {
  PyObject *format, *packed, *norms, *bits, *signs, *centroids, *boundaries, *data;
} names;

struct PyRef {          // owned reference
  PyObject* p;
  explicit PyRef(PyObject* x) : p(x) {}
  PyRef(PyRef&& o) noexcept : p(o.p) { o.p = nullptr; }
  PyRef(const PyRef&) = delete;
  ~PyRef() { Py_XDECREF(p); }
};
[[noreturn]] void raise_python() { throw python_error(); }        // a Python error is set

const at::Tensor& tensor(PyObject* x, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(x), what, " must be a tensor");
  return THPVariable_Unpack(x);
}
void require_cuda(const at::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "libtqb200 operates on CUDA tensors only (no CPU path)");
}
int index_of(const at::Tensor& t) { return t.is_cuda() ? (int)t.get_device() : -1; }
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return TQ_F32;
    case at::kHalf: return TQ_F16;
    case at::kBFloat16: return TQ_BF16;
    default: TORCH_CHECK_VALUE(false, "unsupported dtype ", t, "; use float32, float16 or bfloat16");
  }
}
// A Python integer; beyond 64 bits the nearest 64-bit number.
int64_t integer(PyObject* x) {
  PyRef i(PyNumber_Index(x));
  if (!i.p) raise_python();
  int over = 0;
  const long long v = PyLong_AsLongLongAndOverflow(i.p, &over);
  if (v == -1 && !over && PyErr_Occurred()) raise_python();
  return over > 0 ? INT64_MAX : over < 0 ? INT64_MIN : v;
}
// desc[name]: borrowed for as long as the caller's dict lives (kept in `keep` for other mappings).
PyObject* item(PyObject* desc, PyObject* name, std::vector<PyRef>& keep) {
  if (PyDict_CheckExact(desc)) {
    PyObject* v = PyDict_GetItemWithError(desc, name);
    if (!v) {
      if (!PyErr_Occurred()) PyErr_SetObject(PyExc_KeyError, name);
      raise_python();
    }
    return v;
  }
  PyObject* v = PyObject_GetItem(desc, name);
  if (!v) raise_python();
  keep.emplace_back(v);
  return v;
}

// `count` floats of a codebook-sized parameter on the host: the package's copy (_lib.host_floats), found without a call
// when it is there.
const float* table(PyObject* x, int64_t count, const char* what, const char* name, std::vector<PyRef>& keep) {
  PyObject* arr = nullptr;
  if (THPVariable_Check(x)) {
    PyRef id(PyLong_FromVoidPtr(x));
    if (!id.p) raise_python();
    PyObject* hit = PyDict_GetItemWithError(host_cache, id.p);
    if (hit && PyTuple_CheckExact(hit) && PyTuple_GET_SIZE(hit) == 3 && PyWeakref_GetObject(PyTuple_GET_ITEM(hit, 0)) == x &&
        PyLong_AsLongLong(PyTuple_GET_ITEM(hit, 1)) == (long long)THPVariable_Unpack(x)._version())
      arr = PyTuple_GET_ITEM(hit, 2);
    if (arr) keep.emplace_back(Py_NewRef(arr));
  }
  if (!arr) {
    arr = PyObject_CallOneArg(host_floats, x);
    if (!arr) raise_python();
    keep.emplace_back(arr);
  }
  int64_t n = 0;
  const void* p = nullptr;
  if (arr != Py_None) {
    Py_buffer view;
    if (PyObject_GetBuffer(arr, &view, PyBUF_SIMPLE) != 0) raise_python();
    p = view.buf;                      // the array stays: `keep`
    n = view.len / (int64_t)sizeof(float);
    PyBuffer_Release(&view);
  }
  TORCH_CHECK_VALUE(n == count, what, ": ", name, ": ", n, " entries, ", count, " expected");
  return (const float*)p;
}

struct Geo {
  int64_t pages, heads, page, dim;
  bool operator!=(const Geo& o) const { return pages != o.pages || heads != o.heads || page != o.page || dim != o.dim; }
};

// Words of a packed row, 0 for a width the format does not have.
int64_t row_words(int64_t dim, int64_t bits) {
  const int per = bits == 1 ? 32 : bits == 2 ? 16 : bits == 3 ? 10 : bits == 4 ? 8 : 0;
  return per ? (dim + per - 1) / per : 0;
}

// The fields in front of `rows` from a pool dict; dim < 0: the pool's own.
Geo half(PyObject* desc, const char* what, int64_t dim, int index, bool encode, tq_paged_half* h, std::vector<PyRef>& keep) {
  memset(h, 0, sizeof(*h));
  PyObject* fmt = item(desc, names.format, keep);
  const char* f = PyUnicode_Check(fmt) ? PyUnicode_AsUTF8(fmt) : nullptr;
  if (!f) PyErr_Clear();
  if (f && strcmp(f, "polar") == 0) {
    const at::Tensor& packed = tensor(item(desc, names.packed, keep), "packed");
    const at::Tensor& norms = tensor(item(desc, names.norms, keep), "norms");
    const int64_t bits = integer(item(desc, names.bits, keep));
    TORCH_CHECK_VALUE(bits >= 1 && bits <= 4, "Unsupported bit width: ", bits, ". Use 1-4.");
    PyObject* signs = item(desc, names.signs, keep);
    if (dim < 0) dim = tensor(signs, "signs").numel();
    const int64_t words = row_words(dim, bits);
    TORCH_CHECK_VALUE(packed.scalar_type() == at::kUInt32 && packed.dim() == 4 && packed.size(3) == words &&
                          packed.stride(3) == 1 && packed.stride(2) == words,
                      what, ": packed must be (pages, heads, page, ", words, ") uint32 with contiguous rows");
    TORCH_CHECK_VALUE(norms.scalar_type() == at::kFloat && norms.sizes() == packed.sizes().slice(0, 3) && norms.stride(2) == 1,
                      what, ": norms must be float32 ", packed.sizes().slice(0, 3), ", contiguous along the page");
    TORCH_CHECK_VALUE(index_of(packed) == index && index_of(norms) == index, what, ": all tensors must be on cuda:", index);
    h->format = TQ_KV_POLAR;
    h->bits = (int32_t)bits;
    h->data = packed.data_ptr();
    h->norms = (float*)norms.data_ptr();
    h->page_stride = packed.stride(0);
    h->head_stride = packed.stride(1);
    h->norm_page_stride = norms.stride(0);
    h->norm_head_stride = norms.stride(1);
    h->signs_host = table(signs, dim, what, "signs", keep);
    if (encode)
      h->boundaries_host = table(item(desc, names.boundaries, keep), (1 << bits) - 1, what, "boundaries", keep);
    else
      h->centroids_host = table(item(desc, names.centroids, keep), 1 << bits, what, "centroids", keep);
    return {packed.size(0), packed.size(1), packed.size(2), dim};
  }
  if (f && strcmp(f, "dense") == 0) {
    const at::Tensor& data = tensor(item(desc, names.data, keep), "data");
    TORCH_CHECK_VALUE(data.dim() == 4 && data.stride(3) == 1 && data.stride(2) == data.size(3) && (dim < 0 || data.size(3) == dim),
                      what, ": dense pages must be (pages, heads, page, dim) with contiguous rows");
    TORCH_CHECK_VALUE(index_of(data) == index, what, ": all tensors must be on cuda:", index);
    h->format = TQ_KV_DENSE;
    h->dtype = dtype_code(data.scalar_type());
    h->data = data.data_ptr();
    h->page_stride = data.stride(0);
    h->head_stride = data.stride(1);
    return {data.size(0), data.size(1), data.size(2), data.size(3)};
  }
  PyRef shown(PyObject_Repr(fmt));
  const char* text = shown.p ? PyUnicode_AsUTF8(shown.p) : nullptr;
  TORCH_CHECK_VALUE(false, what, ": unknown page format ", text ? text : "?");
}

const int32_t* lens(const at::Tensor& t, const char* what, int64_t batch, int index) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == batch && (batch <= 1 || t.stride(0) == 1) &&
                        index_of(t) == index,
                    what, " must be a contiguous int32 (", batch, ",) tensor on cuda:", index);
  return (const int32_t*)t.data_ptr();
}
// The table and the lengths.
void pages(const at::Tensor& tab, const at::Tensor& len, const char* what, int index, tq_paged_params* p) {
  require_cuda(tab);
  require_cuda(len);
  TORCH_CHECK_VALUE(tab.scalar_type() == at::kInt && tab.dim() == 2 && index_of(tab) == index,
                    "page_table must be an int32 (batch, width) tensor on cuda:", index);
  const int64_t batch = tab.size(0), width = tab.size(1);
  TORCH_CHECK_VALUE(batch >= 1 && width >= 1 && (tab.stride(1) == 1 || width == 1),
                    "page_table must have at least one sequence and one page, and contiguous rows");
  TORCH_CHECK_VALUE(batch <= INT32_MAX && width <= INT32_MAX, "page_table is too large");
  p->batch = (int32_t)batch;
  p->table_width = (int32_t)width;
  p->page_table = (int32_t*)tab.data_ptr();
  p->table_stride = tab.stride(0);
  p->seq_lens = (int32_t*)lens(len, what, batch, index);
}
void geometry(const Geo& g, tq_paged_params* p) {
  TORCH_CHECK_VALUE(g.heads <= INT32_MAX && g.page <= INT32_MAX && g.dim <= INT32_MAX, "pool is too large");
  p->n_kv_heads = (int32_t)g.heads;
  p->page_size = (int32_t)g.page;
  p->n_pages = g.pages;
  p->dim = (int32_t)g.dim;
}
// Starts a block: a zeroed one of this library's size.
tq_paged_params block(int index) {
  tq_paged_params p;
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(p);
  p.stream = c10::cuda::getCurrentCUDAStream(index).stream();
  return p;
}
void checked(int rc) {
  if (rc == 0) return;
  PyRef r(PyObject_CallFunction(check_status, "i", rc));
  if (!r.p) raise_python();
}
void arguments(Py_ssize_t n, Py_ssize_t want) { TORCH_CHECK_TYPE(n == want, want, " arguments expected, got ", n); }
// The id of the capture the stream is in (never used twice in a process), 0: none.
unsigned long long capture_of(void* stream) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &st, &id) != cudaSuccess) {
    cudaGetLastError();
    return 0;
  }
  return st == cudaStreamCaptureStatusNone ? 0 : id;
}

// (q, k, v, page_table, seq_lens, attn_scale, window, sinks, out, out_dtype, workspace) -> out
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 11);
  at::Tensor q = tensor(args[0], "q");
  require_cuda(q);
  const int index = (int)q.get_device();
  TORCH_CHECK_VALUE(q.dim() == 3, "q must be (batch, heads, dim), got ", q.sizes());
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  if (q.stride(2) != 1) q = q.contiguous();
  const int64_t B = q.size(0), n_q = q.size(1), dim = q.size(2);
  std::vector<PyRef> keep;
  keep.reserve(8);
  tq_paged_params p = block(index);
  pages(tensor(args[3], "page_table"), tensor(args[4], "seq_lens"), "seq_lens", index, &p);
  TORCH_CHECK_VALUE(p.batch == B, "page_table has ", p.batch, " sequences, q has ", B);
  const Geo g = half(args[1], "keys", dim, index, false, &p.k, keep);
  TORCH_CHECK_VALUE(!(half(args[2], "values", dim, index, false, &p.v, keep) != g),
                    "the pools of keys and values must agree in pages, heads, page size and dim");
  geometry(g, &p);
  TORCH_CHECK_VALUE(n_q > 0 && g.heads > 0 && n_q % g.heads == 0 && n_q <= INT32_MAX, "n_q_heads (", n_q, ") must equal n_kv_heads (",
                    g.heads, ") * n_rep");
  p.n_q_heads = (int32_t)n_q;
  const double scale = PyFloat_AsDouble(args[5]);
  if (scale == -1.0 && PyErr_Occurred()) raise_python();
  p.attn_scale = (float)scale;
  const int64_t window = integer(args[6]), sinks = integer(args[7]);
  TORCH_CHECK_VALUE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "window (", window, ") and sinks (", sinks,
                    ") must not be negative, and sinks need a window");
  p.window = (int32_t)std::min<int64_t>(window, INT32_MAX);
  p.sinks = (int32_t)std::min<int64_t>(sinks, INT32_MAX);
  TORCH_CHECK_TYPE(args[9] == Py_None || THPDtype_Check(args[9]), "out_dtype must be a torch.dtype");
  const bool typed = args[9] != Py_None;
  const at::ScalarType want = typed ? reinterpret_cast<THPDtype*>(args[9])->scalar_type : q.scalar_type();
  at::Tensor out;
  if (args[8] == Py_None) {
    dtype_code(want);
    out = at::empty({B, n_q, dim}, q.options().dtype(want));
  } else {
    out = tensor(args[8], "out");
    TORCH_CHECK_VALUE(out.sizes() == q.sizes() && out.stride(2) == 1 && index_of(out) == index && (!typed || out.scalar_type() == want),
                      "out must be ", q.sizes(), " on cuda:", index, ", with a contiguous last dimension and of out_dtype");
  }
  p.q_dtype = dtype_code(q.scalar_type());
  p.out_dtype = dtype_code(out.scalar_type());
  p.q = q.data_ptr();
  p.q_batch_stride = q.stride(0);
  p.q_head_stride = q.stride(1);
  p.out = out.data_ptr();
  p.out_batch_stride = out.stride(0);
  p.out_head_stride = out.stride(1);
  // Scratch of the calls made on a stream outside of captures, and of those captured last on it; never freed (the maps
  // outlive the interpreter).
  using Place = std::tuple<int, void*, int64_t>;
  static auto* kept = new std::map<Place, at::Tensor>;
  static auto* captured = new std::map<Place, std::pair<unsigned long long, at::Tensor>>;
  const Place place(index, p.stream, dim);
  at::Tensor own;
  const at::Tensor* ws = &own;
  if (args[10] != Py_None) {
    own = tensor(args[10], "workspace");
    const int64_t need = entry.workspace_bytes(p.dim);
    TORCH_CHECK_VALUE(own.scalar_type() == at::kByte && own.is_contiguous() && index_of(own) == index && own.numel() >= need,
                      "workspace must be a contiguous uint8 tensor of at least ", need, " bytes on cuda:", index);
  } else if (const unsigned long long id = capture_of(p.stream)) {
    // the graph's own, from its pool, zeroed by every replay: the calls of one capture on one stream follow each other
    auto& mine = (*captured)[place];
    if (mine.first != id) {
      mine.second = at::zeros({entry.workspace_bytes(p.dim)}, q.options().dtype(at::kByte));
      mine.first = id;
    }
    ws = &mine.second;
  } else {
    at::Tensor& mine = (*kept)[place];
    if (!mine.defined()) mine = at::zeros({entry.workspace_bytes(p.dim)}, q.options().dtype(at::kByte));
    ws = &mine;
  }
  p.workspace = ws->data_ptr();
  p.workspace_bytes = ws->numel();
  checked(entry.decode(&p));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// (keys, values, k, v, page_table, starts, counts)
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 7);
  at::Tensor x[2] = {tensor(args[0], "keys"), tensor(args[1], "values")};
  require_cuda(x[0]);
  require_cuda(x[1]);
  const int index = (int)x[0].get_device();
  TORCH_CHECK_VALUE(x[0].dim() == 4 && x[0].sizes() == x[1].sizes(), "keys and values must be (batch, heads, tokens, dim) alike, got ",
                    x[0].sizes(), " and ", x[1].sizes());
  TORCH_CHECK_VALUE(index_of(x[1]) == index, "values must be on cuda:", index);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  const int64_t B = x[0].size(0), H = x[0].size(1), T = x[0].size(2), dim = x[0].size(3);
  std::vector<PyRef> keep;
  keep.reserve(8);
  tq_paged_params p = block(index);
  pages(tensor(args[4], "page_table"), tensor(args[5], "starts"), "starts", index, &p);
  TORCH_CHECK_VALUE(p.batch == B, "page_table has ", p.batch, " sequences, keys have ", B);
  const Geo g = half(args[2], "keys", dim, index, true, &p.k, keep);
  TORCH_CHECK_VALUE(!(half(args[3], "values", dim, index, true, &p.v, keep) != g),
                    "the pools of keys and values must agree in pages, heads, page size and dim");
  TORCH_CHECK_VALUE(g.heads == H, "the pool has ", g.heads, " heads, the new rows ", H);
  geometry(g, &p);
  tq_paged_half* to[2] = {&p.k, &p.v};
  for (int i = 0; i < 2; ++i) {
    if (x[i].stride(3) != 1) x[i] = x[i].contiguous();
    to[i]->rows_dtype = dtype_code(x[i].scalar_type());
    TORCH_CHECK_VALUE(to[i]->format != TQ_KV_DENSE || to[i]->dtype == to[i]->rows_dtype,
                      "rows stored in dense pages must have the pages' dtype");
    to[i]->rows = x[i].data_ptr();
    to[i]->rows_batch_stride = x[i].stride(0);
    to[i]->rows_head_stride = x[i].stride(1);
    to[i]->rows_token_stride = x[i].stride(2);
  }
  if (args[6] != Py_None) {
    const at::Tensor& counts = tensor(args[6], "counts");
    require_cuda(counts);
    p.counts = (int32_t*)lens(counts, "counts", B, index);
  }
  p.tokens = T;
  checked(entry.append(&p));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (pool, page_table, seq_lens, length, dtype, out) -> out
PyObject* dequantize(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 6);
  const at::Tensor& tab = tensor(args[1], "page_table");
  require_cuda(tab);
  const int index = (int)tab.get_device();
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  std::vector<PyRef> keep;
  keep.reserve(8);
  tq_paged_params p = block(index);
  pages(tab, tensor(args[2], "seq_lens"), "seq_lens", index, &p);
  const Geo g = half(args[0], "pages", -1, index, false, &p.v, keep);
  geometry(g, &p);
  const int64_t length = integer(args[3]);
  TORCH_CHECK_VALUE(length >= 0, "length must not be negative, got ", length);
  at::Tensor out;
  if (args[5] == Py_None) {
    TORCH_CHECK_TYPE(THPDtype_Check(args[4]), "dtype must be a torch.dtype");
    const at::ScalarType want = reinterpret_cast<THPDtype*>(args[4])->scalar_type;
    dtype_code(want);
    out = at::empty({p.batch, g.heads, length, g.dim}, tab.options().dtype(want));
  } else {
    out = tensor(args[5], "out");
    TORCH_CHECK_VALUE(out.dim() == 4 && out.size(0) == p.batch && out.size(1) == g.heads && out.size(2) == length &&
                          out.size(3) == g.dim && out.is_contiguous() && index_of(out) == index,
                      "out must be a contiguous (", p.batch, ", ", g.heads, ", ", length, ", ", g.dim, ") tensor on cuda:", index);
  }
  p.out = out.data_ptr();
  p.out_dtype = dtype_code(out.scalar_type());
  p.tokens = length;
  checked(entry.dequantize(&p));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// Page ids: a CUDA tensor as it is (the kernel checks it), anything else as numbers checked here.
struct Ids {
  at::Tensor t;
  std::vector<int32_t> host;
  bool listed = false;
  int64_t count() const { return listed ? (int64_t)host.size() : t.numel(); }
};
Ids ids(PyObject* x, int64_t n_pages, const char* what, int index, bool in_capture) {
  Ids r;
  if (THPVariable_Check(x) && THPVariable_Unpack(x).is_cuda()) {
    r.t = THPVariable_Unpack(x);
    TORCH_CHECK_VALUE(r.t.scalar_type() == at::kInt && r.t.dim() == 1 && r.t.is_contiguous() && index_of(r.t) == index, what,
                      " must be a contiguous one-dimensional int32 tensor on cuda:", index);
    return r;
  }
  TORCH_CHECK(!in_capture, "copy_pages in a captured graph needs ", what, " as a CUDA tensor");
  r.listed = true;
  PyRef seq(PySequence_Fast(x, "page ids must be a list or a tensor"));
  if (!seq.p) raise_python();
  for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(seq.p); ++i) {
    const int64_t id = integer(PySequence_Fast_GET_ITEM(seq.p, i));
    TORCH_CHECK_VALUE(id >= 0 && id < n_pages, what, ": page ", id, " is outside the pool of ", n_pages);
    r.host.push_back((int32_t)id);
  }
  return r;
}

// (pools, src, dst)
PyObject* copy_pages(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 3);
  PyRef seq(PySequence_Fast(args[0], "pools must be a sequence of tensors"));
  if (!seq.p) raise_python();
  const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq.p);
  if (n == 0) Py_RETURN_NONE;
  std::vector<void*> ptrs(n);
  std::vector<int64_t> sizes(n);
  int index = -1;
  int64_t n_pages = 0;
  at::TensorOptions like;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& t = tensor(PySequence_Fast_GET_ITEM(seq.p, i), "pools");
    if (i == 0) {
      require_cuda(t);
      index = (int)t.get_device();
      n_pages = t.dim() ? t.size(0) : 0;
      like = t.options();
    }
    TORCH_CHECK_VALUE(index_of(t) == index && t.dim() > 0 && t.size(0) == n_pages && t.is_contiguous() && ((uintptr_t)t.data_ptr() & 15) == 0,
                      "pools must be contiguous CUDA tensors, 16-byte aligned, of one device and one number of pages");
    ptrs[i] = t.data_ptr();
    sizes[i] = (int64_t)t.nbytes();
  }
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
  const bool in_capture = capture_of(stream) != 0;
  Ids src = ids(args[1], n_pages, "src", index, in_capture), dst = ids(args[2], n_pages, "dst", index, in_capture);
  const int64_t pairs = src.count();
  TORCH_CHECK_VALUE(pairs == dst.count(), pairs, " source and ", dst.count(), " target pages");
  if (dst.listed) {
    const std::set<int32_t> to(dst.host.begin(), dst.host.end());
    TORCH_CHECK_VALUE(to.size() == dst.host.size(), "a target page is named twice");
    for (int32_t s : src.host) TORCH_CHECK_VALUE(!to.count(s), "a page is both read and written");
  }
  if (n_pages == 0 || pairs == 0) Py_RETURN_NONE;
  for (int64_t& s : sizes) {
    TORCH_CHECK_VALUE(s > 0 && s % (16 * n_pages) == 0, "pages must be multiples of 16 bytes");
    s /= n_pages;
  }
  // what came as numbers goes over in one upload
  at::Tensor up;
  const int32_t *from = nullptr, *to = nullptr;
  if (src.listed || dst.listed) {
    std::vector<int32_t> flat(src.host);
    flat.insert(flat.end(), dst.host.begin(), dst.host.end());
    up = at::from_blob(flat.data(), {(int64_t)flat.size()}, at::TensorOptions().dtype(at::kInt))
             .to(like.dtype(at::kInt).device(), at::kInt, /*non_blocking=*/false, /*copy=*/true);
    from = (const int32_t*)up.data_ptr();
    to = from + src.host.size();
  }
  if (!src.listed) from = (const int32_t*)src.t.data_ptr();
  if (!dst.listed) to = (const int32_t*)dst.t.data_ptr();
  checked(entry.copy(ptrs.data(), sizes.data(), (int)n, n_pages, from, to, pairs, stream));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// (queries, keys, values, scale, causal, out, window, sinks, status) -> out
PyObject* prefill(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 9);
  at::Tensor x[3] = {tensor(args[0], "queries"), tensor(args[1], "keys"), tensor(args[2], "values")};
  for (const at::Tensor& t : x) require_cuda(t);
  const int index = (int)x[0].get_device();
  TORCH_CHECK_VALUE(x[0].scalar_type() == at::kHalf || x[0].scalar_type() == at::kBFloat16,
                    "prefill_attention takes float16 or bfloat16 tensors");
  TORCH_CHECK_VALUE(x[1].scalar_type() == x[0].scalar_type() && x[2].scalar_type() == x[0].scalar_type(),
                    "queries, keys and values must share one dtype");
  TORCH_CHECK_VALUE(x[0].dim() == 4 && x[1].dim() == 4 && x[2].dim() == 4, "queries, keys and values must be (batch, heads, length, 128)");
  const int64_t B = x[0].size(0), n_q = x[0].size(1), L = x[0].size(2), D = x[0].size(3), n_kv = x[1].size(1), S = x[1].size(2);
  TORCH_CHECK_VALUE(D == 128 && x[1].size(3) == 128 && x[2].size(3) == 128, "prefill_attention supports head_dim 128, got ", D);
  TORCH_CHECK_VALUE(n_kv > 0 && n_q % n_kv == 0, "n_q_heads (", n_q, ") must equal n_kv_heads (", n_kv, ") * n_rep (",
                    n_q / std::max<int64_t>(n_kv, 1), ")");
  TORCH_CHECK_VALUE(x[1].size(0) == B && x[2].sizes() == x[1].sizes(), "keys and values must have the same (batch, heads, length)");
  TORCH_CHECK_VALUE(index_of(x[1]) == index && index_of(x[2]) == index, "queries, keys and values must be on one device");
  TORCH_CHECK_VALUE(std::max(B, n_q) <= INT32_MAX, "too many heads");
  const int causal = PyObject_IsTrue(args[4]);
  if (causal < 0) raise_python();
  const double scale = PyFloat_AsDouble(args[3]);
  if (scale == -1.0 && PyErr_Occurred()) raise_python();
  const int64_t window = integer(args[6]), sinks = integer(args[7]);
  TORCH_CHECK_VALUE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0) && (window == 0 || causal), "window (", window,
                    ") and sinks (", sinks, ") must not be negative, sinks need a window, and a window needs causal attention");
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  auto usable = [](const at::Tensor& t) {
    return t.stride(3) == 1 && ((t.stride(0) | t.stride(1) | t.stride(2)) & 7) == 0 && ((uintptr_t)t.data_ptr() & 15) == 0;
  };
  for (at::Tensor& t : x)
    if (!usable(t)) t = t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
  at::Tensor out;
  if (args[5] == Py_None) {
    out = at::empty({B, n_q, L, D}, x[0].options());
  } else {
    out = tensor(args[5], "out");
    TORCH_CHECK_VALUE(out.sizes() == x[0].sizes() && out.scalar_type() == x[0].scalar_type() && index_of(out) == index && usable(out),
                      "out must be ", x[0].sizes(), " of the inputs' dtype on cuda:", index,
                      ", 16-byte aligned, with a contiguous last dimension");
  }
  const at::Tensor& status = tensor(args[8], "status");
  tq_prefill_params p;
  memset(&p, 0, sizeof(p));
  p.struct_bytes = (int32_t)sizeof(p);
  p.dtype = dtype_code(x[0].scalar_type());
  p.batch = (int32_t)B;
  p.n_q_heads = (int32_t)n_q;
  p.n_kv_heads = (int32_t)n_kv;
  p.dim = (int32_t)D;
  p.seq_q = L;
  p.seq_k = S;
  p.q = x[0].data_ptr();
  p.k = x[1].data_ptr();
  p.v = x[2].data_ptr();
  p.out = out.data_ptr();
  for (int i = 0; i < 3; ++i) {
    p.q_strides[i] = x[0].stride(i);
    p.k_strides[i] = x[1].stride(i);
    p.v_strides[i] = x[2].stride(i);
    p.o_strides[i] = out.stride(i);
  }
  p.window = window;
  p.sinks = sinks;
  p.attn_scale = (float)scale;
  p.causal = causal;
  p.status = (int*)status.data_ptr();
  p.stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
  checked(entry.prefill(&p));
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// bind(lib, decode, append, dequantize, workspace_bytes, copy, prefill): the package's _lib module and the entry points' addresses
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  arguments(nargs, 7);
  void* at[6];
  for (int i = 0; i < 6; ++i) {
    at[i] = PyLong_AsVoidPtr(args[1 + i]);
    if (!at[i]) raise_python();
  }
  host_floats = PyObject_GetAttrString(args[0], "host_floats");
  host_cache = PyObject_GetAttrString(args[0], "_host_cache");
  check_status = PyObject_GetAttrString(args[0], "check");
  if (!host_floats || !host_cache || !check_status) raise_python();
  TORCH_CHECK_TYPE(PyDict_CheckExact(host_cache), "_host_cache must be a dict");
  entry.decode = reinterpret_cast<decltype(entry.decode)>(at[0]);
  entry.append = reinterpret_cast<decltype(entry.append)>(at[1]);
  entry.dequantize = reinterpret_cast<decltype(entry.dequantize)>(at[2]);
  entry.workspace_bytes = reinterpret_cast<decltype(entry.workspace_bytes)>(at[3]);
  entry.copy = reinterpret_cast<decltype(entry.copy)>(at[4]);
  entry.prefill = reinterpret_cast<decltype(entry.prefill)>(at[5]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
    {"decode", (PyCFunction)(void*)decode, METH_FASTCALL, nullptr},
    {"append", (PyCFunction)(void*)append, METH_FASTCALL, nullptr},
    {"dequantize", (PyCFunction)(void*)dequantize, METH_FASTCALL, nullptr},
    {"copy_pages", (PyCFunction)(void*)copy_pages, METH_FASTCALL, nullptr},
    {"prefill", (PyCFunction)(void*)prefill, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  names = {PyUnicode_InternFromString("format"), PyUnicode_InternFromString("packed"), PyUnicode_InternFromString("norms"),
           PyUnicode_InternFromString("bits"), PyUnicode_InternFromString("signs"), PyUnicode_InternFromString("centroids"),
           PyUnicode_InternFromString("boundaries"), PyUnicode_InternFromString("data")};
  return PyModule_Create(&module);
}
