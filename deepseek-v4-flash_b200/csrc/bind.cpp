// bind.cpp -- Python binding of the draft-tree and eviction calls
// (include/qcau_b200.h) on torch tensors: checks, outputs, workspace and call.
//
// These are calls of single decode steps, short enough on the GPU (6 to 17 us) that
// a binding through ctypes, whose checks read each tensor attribute from Python,
// took as long as the kernels (a tree attention 17.5 us of host time, an eviction
// 17.2, a commit's move 8).  The functions take their arguments by position; the
// Python modules (qcau_b200/tree.py, evict.py, cache.py) name and document them.
// Every refusal is a ValueError or NotImplementedError before anything is launched.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <string>

#include "qcau_b200.h"

namespace {

using at::Tensor;

// An argument: a tensor, or None where `optional`.
const Tensor* tensor_arg(PyObject* o, const char* name, bool optional = false) {
  if (optional && o == Py_None) return nullptr;
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor", optional ? " or None" : "");
  return &THPVariable_Unpack(o);
}

int64_t int_arg(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be an integer of 64 bits");
  }
  return v;
}

double float_arg(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK_TYPE(false, name, " must be a number");
  }
  return v;
}

template <typename T>
T* data(const Tensor* t) {
  return t ? reinterpret_cast<T*>(t->data_ptr()) : nullptr;
}

// The library's status as the exception it stands for.
void check_status(int rc, const char* what) {
  if (rc == QCAU_OK) return;
  const std::string msg = qcau_last_error();
  TORCH_CHECK_VALUE(rc != QCAU_ERR_INVALID && rc != QCAU_ERR_WORKSPACE, msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != QCAU_ERR_UNSUPPORTED, msg);
  TORCH_CHECK(false, what, ": ", msg, " (status ", rc, ")");
}

struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

// Runs call(stream) with device `index` current and its current stream, without
// the GIL: a launch waits where the queue is full.
template <typename Call>
void run(int index, const char* what, Call call) {
  int rc;
  {
    WithoutGil nogil;
    c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
    rc = call(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream());
  }
  check_status(rc, what);
}

int cuda_index(const Tensor& t) {
  TORCH_CHECK_VALUE(t.is_cuda(), "qcau_b200 runs on CUDA tensors only (no CPU path)");
  return t.get_device();
}

struct Paged {
  int64_t num_pages, page, d, b, max_pages;
};

Paged check_paged(const char* what, int index, const Tensor& cache, const Tensor& table) {
  TORCH_CHECK_VALUE(cuda_index(cache) == index && cuda_index(table) == index, what,
                    ": all tensors must be on one device");
  TORCH_CHECK_VALUE(cache.dim() == 3 && cache.scalar_type() == at::kBFloat16 && cache.is_contiguous(), what,
                    ": the cache must be a contiguous bf16 [pages, page, width] tensor");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.scalar_type() == at::kInt && table.is_contiguous(), what,
                    ": the block table must be a contiguous int32 [batch, pages] tensor");
  return {cache.size(0), cache.size(1), cache.size(2), table.size(0), table.size(1)};
}

// int32 [b] or, with cols >= 0, [b, cols].
void check_ints(const char* what, const char* name, const Tensor* t, int index, int64_t b, int64_t cols = -1) {
  if (!t) return;
  const bool shape = cols < 0 ? t->dim() == 1 && t->size(0) == b
                              : t->dim() == 2 && t->size(0) == b && t->size(1) == cols;
  TORCH_CHECK_VALUE(shape && t->scalar_type() == at::kInt && t->is_contiguous() && t->is_cuda() &&
                        t->get_device() == index,
                    what, ": ", name, " must be a contiguous int32 tensor, ",
                    cols < 0 ? "one value" : "one row", " per sequence, on the device of the others");
}

struct Sums {
  int64_t n, stride;
};

Sums check_sums(const char* what, const Tensor& sums, int index, int64_t b) {
  TORCH_CHECK_VALUE(sums.dim() == 2 && sums.scalar_type() == at::kFloat && sums.is_cuda() && sums.get_device() == index,
                    what, ": sums must be fp32 [batch, positions] on the device of the others");
  const int64_t n = sums.size(1), step = sums.stride(0);
  TORCH_CHECK_VALUE(sums.size(0) == b && (n <= 1 || sums.stride(1) == 1) && (b <= 1 || step >= n), what,
                    ": sums needs one contiguous row per sequence");
  return {n, step > n ? step : n};
}

// ---------------------------------------------------------------- attention and weights

// What both take: args gets the shapes and inputs; returns the device.  `q` may be
// replaced by a contiguous copy, which `held` keeps.
int check_step(const char* what, const Tensor*& q, Tensor& held, const Tensor& cache, const Tensor& table,
               const Tensor* seqlens, const Tensor* mask, const Tensor* tree_lens, PyObject* max_seqlen,
               double scale, qcau_tree_args& args) {
  const int index = cuda_index(*q);
  const Paged c = check_paged(what, index, cache, table);
  TORCH_CHECK_VALUE(q->dim() == 4 && q->scalar_type() == at::kBFloat16, what,
                    ": q must be bf16 [batch, nodes, heads, width]");
  const int64_t b = q->size(0), s = q->size(1), h = q->size(2), d = q->size(3);
  TORCH_CHECK_VALUE(s > 0 && h > 0, what, ": q has no rows");
  TORCH_CHECK_VALUE(c.d == d, what, ": q and the cache must have one width");
  TORCH_CHECK_VALUE(c.b == b, what, ": one block-table row per sequence is needed");
  check_ints(what, "seqlens", seqlens, index, b);
  check_ints(what, "tree_lens", tree_lens, index, b);
  if (mask) {
    const auto type = mask->scalar_type();
    const bool each = mask->dim() == 3 && mask->size(0) == b && mask->size(1) == s && mask->size(2) == s;
    const bool one = mask->dim() == 2 && mask->size(0) == s && mask->size(1) == s;
    TORCH_CHECK_VALUE((each || one) && (type == at::kBool || type == at::kByte) && mask->is_contiguous() &&
                          mask->is_cuda() && mask->get_device() == index,
                      what, ": the mask must be a contiguous bool [batch, nodes, nodes] or [nodes, nodes] tensor "
                            "on q's device");
    args.mask_seq_stride = each ? s * s : 0;
  }
  if (!q->is_contiguous()) {
    held = q->contiguous();
    q = &held;
  }
  args.q = q->data_ptr();
  args.cache = cache.data_ptr();
  args.block_table = data<int32_t>(&table);
  args.seqlens = data<int32_t>(seqlens);
  args.tree_lens = data<int32_t>(tree_lens);
  args.tree_mask = data<void>(mask);
  args.b = b;
  args.s = s;
  args.h = h;
  args.d_qk = d;
  args.d_v = 512;
  args.page_size = c.page;
  args.max_pages = c.max_pages;
  args.num_pages = c.num_pages;
  args.max_seqlen = max_seqlen == Py_None ? c.max_pages * c.page : int_arg(max_seqlen, "max_seqlen");
  // before anything is sized by it
  TORCH_CHECK_VALUE(args.max_seqlen >= 1 && args.max_seqlen <= c.max_pages * c.page, what,
                    ": max_seqlen must be at least 1 and within the block table");
  args.softmax_scale = (float)scale;
  return index;
}

PyObject* tree_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 11, "tree_attn takes 11 arguments");
  const Tensor *q = tensor_arg(a[0], "q"), *cache = tensor_arg(a[1], "cache"), *table = tensor_arg(a[2], "block_table");
  const Tensor *seqlens = tensor_arg(a[3], "seqlens"), *mask = tensor_arg(a[4], "mask", true);
  const Tensor *tree_lens = tensor_arg(a[6], "tree_lens", true), *sink = tensor_arg(a[7], "attn_sink", true);
  const Tensor* given = tensor_arg(a[10], "out", true);
  qcau_tree_args args{};
  Tensor held, held_sink;
  const int index = check_step("tree_attn", q, held, *cache, *table, seqlens, mask, tree_lens, a[8],
                               float_arg(a[5], "softmax_scale"), args);
  if (sink) {
    TORCH_CHECK_VALUE(sink->numel() == args.h && sink->is_cuda() && sink->get_device() == index,
                      "tree_attn: attn_sink needs one value per head, on q's device");
    if (sink->scalar_type() != at::kFloat || !sink->is_contiguous()) {
      held_sink = sink->to(at::kFloat).contiguous();
      sink = &held_sink;
    }
  }
  Tensor out;
  if (given) {
    TORCH_CHECK_VALUE(given->dim() == 4 && given->size(0) == args.b && given->size(1) == args.s &&
                          given->size(2) == args.h && given->size(3) == 512 &&
                          given->scalar_type() == at::kBFloat16 && given->is_contiguous() && given->is_cuda() &&
                          given->get_device() == index,
                      "tree_attn: out must be a contiguous bf16 [batch, nodes, heads, 512] tensor");
  } else {
    out = at::empty({args.b, args.s, args.h, 512}, q->options());
  }
  const int want = PyObject_IsTrue(a[9]);
  if (want < 0) throw python_error();
  const bool return_lse = want == 1;
  Tensor lse;
  if (return_lse) lse = at::empty({args.b, args.s, args.h}, q->options().dtype(at::kFloat));
  args.workspace_bytes = qcau_tree_attn_workspace_size(args.b, args.s, args.h, args.max_seqlen);
  const Tensor ws = at::empty({(int64_t)args.workspace_bytes}, q->options().dtype(at::kByte));
  args.attn_sink = data<float>(sink);
  args.o = given ? given->data_ptr() : out.data_ptr();
  args.lse = return_lse ? data<float>(&lse) : nullptr;
  args.workspace = ws.data_ptr();
  run(index, "tree_attn", [&](cudaStream_t st) { return qcau_tree_attn(&args, st); });
  PyObject* o = given ? Py_NewRef(a[10]) : THPVariable_Wrap(std::move(out));
  if (!return_lse) return o;
  PyObject* l = THPVariable_Wrap(std::move(lse));
  PyObject* both = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return both;
  END_HANDLE_TH_ERRORS
}

PyObject* attn_weight_sums(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "attn_weight_sums takes 10 arguments");
  const Tensor *q = tensor_arg(a[0], "q"), *cache = tensor_arg(a[1], "cache"), *table = tensor_arg(a[2], "block_table");
  const Tensor *seqlens = tensor_arg(a[3], "seqlens"), *lse = tensor_arg(a[4], "lse");
  const Tensor *mask = tensor_arg(a[5], "mask", true), *tree_lens = tensor_arg(a[7], "tree_lens", true);
  const Tensor* given = tensor_arg(a[9], "sums", true);
  qcau_tree_args args{};
  Tensor held;
  const int index = check_step("attn_weight_sums", q, held, *cache, *table, seqlens, mask, tree_lens, a[8],
                               float_arg(a[6], "softmax_scale"), args);
  TORCH_CHECK_VALUE(lse->scalar_type() == at::kFloat && lse->dim() == 3 && lse->size(0) == args.b &&
                        lse->size(1) == args.s && lse->size(2) == args.h && lse->is_contiguous() && lse->is_cuda() &&
                        lse->get_device() == index,
                    "attn_weight_sums: lse must be a contiguous fp32 [batch, nodes, heads] tensor");
  Tensor sums;
  if (given) {
    const Sums g = check_sums("attn_weight_sums", *given, index, args.b);
    TORCH_CHECK_VALUE(g.n >= args.max_seqlen, "attn_weight_sums: a row of sums must hold max_seqlen values");
    args.sums_stride = g.stride;
    args.accumulate = 1;
  } else {
    sums = at::empty({args.b, args.max_seqlen}, lse->options());
    args.sums_stride = args.max_seqlen;
  }
  args.workspace_bytes = qcau_attn_weight_sums_workspace_size(args.b, args.s, args.h, args.max_seqlen);
  Tensor ws;
  if (args.workspace_bytes) ws = at::empty({(int64_t)args.workspace_bytes}, q->options().dtype(at::kByte));
  args.lse = data<float>(lse);
  args.sums = given ? data<float>(given) : data<float>(&sums);
  args.workspace = args.workspace_bytes ? ws.data_ptr() : nullptr;
  run(index, "attn_weight_sums", [&](cudaStream_t st) { return qcau_attn_weight_sums(&args, st); });
  return given ? Py_NewRef(a[9]) : THPVariable_Wrap(std::move(sums));
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- selection and moves

// Selection of sequences `b`; select_outputs allocates the outputs.
qcau_select_args check_select(const char* what, int index, const Tensor& sums, const Tensor& seqlens, int64_t b,
                              const Tensor* sums_out) {
  qcau_select_args s{};
  check_ints(what, "seqlens", &seqlens, index, b);
  const Sums in = check_sums(what, sums, index, b);
  s.sums = data<float>(&sums);
  s.seqlens = data<int32_t>(&seqlens);
  s.sums_stride = in.stride;
  s.b = b;
  s.max_seqlen = in.n;
  if (sums_out) {
    const Sums out = check_sums(what, *sums_out, index, b);
    TORCH_CHECK_VALUE(out.n == in.n, what, ": sums_out must have the shape of sums");
    s.sums_out = data<float>(sums_out);
    s.out_stride = out.stride;
  }
  return s;
}

// The outputs of a selection.
void select_outputs(qcau_select_args& s, const Tensor& seqlens, Tensor& keep, Tensor& counts) {
  TORCH_CHECK_VALUE(s.budget >= 1, "evict_select: the budget must be at least 1");
  keep = at::empty({s.b, s.budget}, seqlens.options());
  counts = at::empty_like(seqlens);
  s.keep = data<int32_t>(&keep);
  s.counts = data<int32_t>(&counts);
}

// Where rows come from and go to.
qcau_keep_args check_move(const char* what, int index, const Tensor& cache, const Tensor& table,
                          const Tensor* dst_cache, const Tensor* dst_table) {
  const Paged c = check_paged(what, index, cache, table);
  TORCH_CHECK_VALUE(c.d % 16 == 0, what, ": the row width must be a multiple of 16");
  const Tensor &dc = dst_cache ? *dst_cache : cache, &dt = dst_table ? *dst_table : table;
  const Paged d = dst_cache || dst_table ? check_paged(what, index, dc, dt) : c;
  TORCH_CHECK_VALUE(d.page == c.page && d.d == c.d && d.b == c.b, what,
                    ": one row per sequence in both block tables, and caches of one page size and width are needed");
  qcau_keep_args k{};
  k.cache = cache.data_ptr();
  k.block_table = data<int32_t>(&table);
  k.dst_cache = dc.data_ptr();
  k.dst_table = data<int32_t>(&dt);
  k.max_pages = c.max_pages;
  k.num_pages = c.num_pages;
  k.dst_max_pages = d.max_pages;
  k.dst_num_pages = d.num_pages;
  k.b = c.b;
  k.d = c.d;
  k.page_size = c.page;
  return k;
}

PyObject* pair(Tensor keep, Tensor counts) {
  PyObject *k = THPVariable_Wrap(std::move(keep)), *c = THPVariable_Wrap(std::move(counts));
  PyObject* both = PyTuple_Pack(2, k, c);
  Py_DECREF(k);
  Py_DECREF(c);
  return both;
}

PyObject* select_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 6, "select_rows takes 6 arguments");
  const Tensor *sums = tensor_arg(a[0], "sums"), *seqlens = tensor_arg(a[1], "seqlens");
  const int index = cuda_index(*seqlens);
  qcau_select_args s = check_select("select_rows", index, *sums, *seqlens, seqlens->numel(),
                                    tensor_arg(a[5], "sums_out", true));
  s.budget = int_arg(a[2], "budget");
  s.n_first = int_arg(a[3], "n_first");
  s.n_recent = int_arg(a[4], "n_recent");
  Tensor keep, counts;
  select_outputs(s, *seqlens, keep, counts);
  run(index, "evict_select", [&](cudaStream_t st) { return qcau_evict_select(&s, st); });
  return pair(std::move(keep), std::move(counts));
  END_HANDLE_TH_ERRORS
}

PyObject* evict(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 10, "evict takes 10 arguments");
  const Tensor *cache = tensor_arg(a[0], "cache"), *table = tensor_arg(a[1], "block_table");
  const Tensor *seqlens = tensor_arg(a[2], "seqlens"), *sums = tensor_arg(a[3], "sums");
  const Tensor* sums_out = tensor_arg(a[9], "sums_out", true);
  const int index = cuda_index(*cache);
  qcau_keep_args k = check_move("evict", index, *cache, *table, tensor_arg(a[7], "dst_cache", true),
                                tensor_arg(a[8], "dst_table", true));
  qcau_select_args s = check_select("evict", index, *sums, *seqlens, k.b, sums_out ? sums_out : sums);
  s.budget = int_arg(a[4], "budget");
  s.n_first = int_arg(a[5], "n_first");
  s.n_recent = int_arg(a[6], "n_recent");
  Tensor keep, counts;
  select_outputs(s, *seqlens, keep, counts);
  // (refuses before the selection is launched, which changes the sums)
  run(index, "evict", [&](cudaStream_t st) { return qcau_evict(&s, &k, st); });
  return pair(std::move(keep), std::move(counts));
  END_HANDLE_TH_ERRORS
}

PyObject* keep_rows(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_TYPE(n == 9, "keep_rows takes 9 arguments");
  const Tensor *cache = tensor_arg(a[0], "cache"), *table = tensor_arg(a[1], "block_table");
  const Tensor *keep = tensor_arg(a[2], "keep"), *counts = tensor_arg(a[3], "counts");
  const Tensor *start = tensor_arg(a[4], "start", true), *lens = tensor_arg(a[7], "seqlens", true);
  const Tensor* sums = tensor_arg(a[8], "sums", true);
  const int index = cuda_index(*cache);
  qcau_keep_args k = check_move("keep_rows", index, *cache, *table, tensor_arg(a[5], "dst_cache", true),
                                tensor_arg(a[6], "dst_table", true));
  TORCH_CHECK_VALUE(keep->dim() == 2 && keep->size(1) > 0, "keep_rows: keep must be [batch, rows], with rows");
  k.k = k.keep_stride = keep->size(1);
  check_ints("keep_rows", "keep", keep, index, k.b, k.k);
  check_ints("keep_rows", "counts", counts, index, k.b);
  check_ints("keep_rows", "start", start, index, k.b);
  check_ints("keep_rows", "seqlens", lens, index, k.b);
  k.keep = data<int32_t>(keep);
  k.counts = data<int32_t>(counts);
  k.start = data<int32_t>(start);
  k.lens_out = data<int32_t>(lens);
  if (sums) {
    const Sums s = check_sums("keep_rows", *sums, index, k.b);
    run(index, "keep_rows", [&](cudaStream_t st) {
      return qcau_keep_rows_sums(&k, data<float>(sums), s.stride, s.n, st);
    });
  } else {
    run(index, "keep_rows", [&](cudaStream_t st) { return qcau_keep_rows(&k, st); });
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define QCAU_METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {QCAU_METHOD(tree_attn),   QCAU_METHOD(attn_weight_sums), QCAU_METHOD(select_rows),
                         QCAU_METHOD(evict),       QCAU_METHOD(keep_rows),        {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__bind(void) { return PyModule_Create(&module); }
