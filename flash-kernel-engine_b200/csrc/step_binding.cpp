// Native binding of the serving-step operators (flash_engine/step.py): checks the tensors
// and calls the C entries of libflash_engine_b200.so on the current stream. A decode step
// makes these calls once a layer, and their kernels take a few microseconds: with the checks
// and the argument conversion in Python a call took 14 to 22 us of host time, several times
// its kernels' time.
//
// The C entries are handed over by address (bind), so that the binding follows whichever
// build of the library the package has loaded. Refusals raise TypeError (not CUDA tensors,
// unsupported types), ValueError (shapes, layout) or RuntimeError (a status of the entry),
// as the operators of flash_engine/ops.py do.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cmath>
#include <optional>
#include <string>

#include "../../include/flash_engine_c.h"

namespace {

struct Refusal {
  PyObject* type;
  std::string what;
};
[[noreturn]] void refuse(PyObject* type, std::string what) { throw Refusal{type, std::move(what)}; }
void require(bool ok, const char* what) {
  if (!ok) refuse(PyExc_ValueError, what);
}

decltype(&fe_plan_paged_step) c_plan = nullptr;
decltype(&fe_paged_qkv_append) c_append = nullptr;
decltype(&fe_update_page_bounds) c_bounds = nullptr;
decltype(&fe_sparse_paged_attention) c_sparse = nullptr;
decltype(&fe_sparse_paged_attention_scratch_ints) c_scratch = nullptr;

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda())
    refuse(PyExc_TypeError,
           "flash_engine operators take CUDA tensors; the CPU reference implementation is test "
           "infrastructure, not a fallback");
  return THPVariable_Unpack(o);
}
const at::Tensor& contiguous(PyObject* o) {
  const at::Tensor& t = tensor(o);
  require(t.is_contiguous(), "tensors must be contiguous");
  return t;
}
long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refusal{nullptr, {}};
  return v;
}
int integer32(PyObject* o) {
  const long long v = integer(o);
  require(v >= INT_MIN && v <= INT_MAX, "an integer argument is out of range");
  return static_cast<int>(v);
}
int dim32(const at::Tensor& t, int d) {
  const int64_t n = t.size(d);
  require(n <= INT_MAX, "a tensor dimension is out of range");
  return static_cast<int>(n);
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, {}};
  return v;
}
void same_device(const at::Tensor& a, const at::Tensor& b) {
  require(a.get_device() == b.get_device(), "all tensors must be on one device");
}
// Whether two ranges of bytes, or two contiguous tensors, share memory.
bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const char* x = static_cast<const char*>(a);
  const char* y = static_cast<const char*>(b);
  return na > 0 && nb > 0 && x < y + nb && y < x + na;
}
bool overlap(const at::Tensor& a, const at::Tensor& b) {
  return overlap(a.data_ptr(), a.nbytes(), b.data_ptr(), b.nbytes());
}
int dtype_code(at::ScalarType t) {
  return t == at::kBFloat16 ? 0 : t == at::kHalf ? 1 : t == at::kFloat ? 2 : -1;
}
void check_status(int st, const char* what) {
  if (st != 0)
    refuse(PyExc_RuntimeError, std::string(what) + " failed: CUDA error " + std::to_string(st) +
                                   (st == 1 ? " (cudaErrorInvalidValue (unsupported arguments))"
                                            : " (see cudaError_t)"));
}
// The caller's buffer if it fits, else a new one. Returns a new reference.
PyObject* buffer(PyObject* given, at::IntArrayRef shape, at::ScalarType type,
                 const at::Tensor& like, const char* name) {
  if (given == Py_None)
    return THPVariable_Wrap(at::empty(shape, like.options().dtype(type)));
  const at::Tensor& t = tensor(given);
  if (t.sizes() != shape || t.scalar_type() != type || !t.is_contiguous() ||
      t.get_device() != like.get_device())
    refuse(PyExc_ValueError, std::string(name) +
                                 " must be a contiguous tensor of the expected shape and type on "
                                 "the inputs' device");
  Py_INCREF(given);
  return given;
}
struct Ref {  // an owned reference
  PyObject* p = nullptr;
  ~Ref() { Py_XDECREF(p); }
  PyObject* release() {
    PyObject* q = p;
    p = nullptr;
    return q;
  }
};
template <typename T>
T* data(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
int layout_code(PyObject* o) {
  if (PyUnicode_Check(o)) {
    if (PyUnicode_CompareWithASCIIString(o, "flat") == 0) return 0;
    if (PyUnicode_CompareWithASCIIString(o, "vllm") == 0) return 1;
  }
  refuse(PyExc_ValueError, "kv_layout must be 'flat' or 'vllm'");
}
struct CacheDims {
  int blocks, heads, dim;
};
CacheDims cache_dims(const at::Tensor& k, int block_size, int layout) {
  if (layout == 0 && k.dim() == 4 && k.size(2) == block_size)
    return {dim32(k, 0), dim32(k, 1), dim32(k, 3)};
  if (layout == 1 && k.dim() == 5 && k.size(3) == block_size && k.size(4) == 8)
    return {dim32(k, 0), dim32(k, 1), dim32(k, 2) * 8};
  refuse(PyExc_ValueError,
         "key_cache must be flat [num_blocks, Hkv, block_size, d] or vllm [num_blocks, Hkv, d/8, "
         "block_size, 8]");
}
void check_value_cache(const at::Tensor& k, const at::Tensor& v, const CacheDims& c,
                       int block_size, int layout) {
  const bool shape =
      layout == 0 ? v.sizes() == k.sizes()
                  : v.sizes() == at::IntArrayRef({c.blocks, c.heads, c.dim, block_size});
  require(shape && v.scalar_type() == k.scalar_type(), "key_cache and value_cache must match");
}
void check_bounds(PyObject* pair, const CacheDims& c, const at::Tensor& like,
                  const at::Tensor** values, const at::Tensor** scales) {
  if (!PyTuple_Check(pair) || PyTuple_GET_SIZE(pair) != 2)
    refuse(PyExc_ValueError, "page_bounds must be a pair (values, scales)");
  const at::Tensor& v = contiguous(PyTuple_GET_ITEM(pair, 0));
  const at::Tensor& s = contiguous(PyTuple_GET_ITEM(pair, 1));
  same_device(like, v);
  same_device(like, s);
  require(v.scalar_type() == at::kChar && s.scalar_type() == at::kFloat &&
              v.sizes() == at::IntArrayRef({c.blocks, c.heads, 2, c.dim}) &&
              s.sizes() == at::IntArrayRef({c.blocks, c.heads}),
          "page_bounds must be int8 [num_blocks, Hkv, 2, d] and float32 [num_blocks, Hkv]");
  *values = &v;
  *scales = &s;
}
void* stream_of(const at::Tensor& t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

// (context_lens, new_lens, block_tables, free_blocks, free_state, block_size, max_tokens,
//  finished, out) -> the five tensors of a PagedStep
PyObject* plan(PyObject* const* a) {
  const at::Tensor& ctx = contiguous(a[0]);
  const at::Tensor& add = contiguous(a[1]);
  const at::Tensor& table = contiguous(a[2]);
  const at::Tensor& ring = contiguous(a[3]);
  const at::Tensor& state = contiguous(a[4]);
  for (const at::Tensor* t : {&ctx, &add, &table, &ring, &state}) {
    same_device(ctx, *t);
    if (t->scalar_type() != at::kInt)
      refuse(PyExc_TypeError,
             "lengths, block_tables, free_blocks and free_state must be int32");
  }
  require(ctx.dim() == 1 && add.sizes() == ctx.sizes() && table.dim() == 2 &&
              table.size(0) == ctx.size(0) && ring.dim() == 1 && state.dim() == 1 &&
              state.size(0) >= 2,
          "context_lens, new_lens [S], block_tables [S, max_blocks], free_blocks [num_blocks] and "
          "free_state [>= 2] expected");
  const int S = dim32(table, 0), width = dim32(table, 1);
  const unsigned char* fin = nullptr;
  if (a[7] != Py_None) {
    const at::Tensor& f = contiguous(a[7]);
    same_device(ctx, f);
    require((f.scalar_type() == at::kBool || f.scalar_type() == at::kByte) &&
                f.sizes() == ctx.sizes(),
            "finished must be a bool or uint8 tensor [S]");
    fin = data<unsigned char>(f);
  }
  PyObject* given[5] = {Py_None, Py_None, Py_None, Py_None, Py_None};
  if (a[8] != Py_None) {
    require(PyTuple_Check(a[8]) && PyTuple_GET_SIZE(a[8]) == 5,
            "out must hold the five tensors of a PagedStep");
    for (int i = 0; i < 5; ++i) given[i] = PyTuple_GET_ITEM(a[8], i);
  }
  int64_t cap;
  if (a[6] != Py_None) {
    cap = integer(a[6]);
  } else {
    require(given[2] != Py_None, "max_tokens or out must be given");
    const at::Tensor& p = tensor(given[2]);
    require(p.dim() == 1, "positions must be [max_tokens]");
    cap = p.size(0);
  }
  require(cap >= 0 && cap < (1 << 30), "max_tokens is out of range");
  Ref r[5];
  r[0].p = buffer(given[0], {S}, at::kInt, ctx, "context_lens");
  r[1].p = buffer(given[1], {S + 1}, at::kInt, ctx, "cu_seqlens");
  r[2].p = buffer(given[2], {cap}, at::kInt, ctx, "positions");
  r[3].p = buffer(given[3], {cap}, at::kLong, ctx, "slots");
  r[4].p = buffer(given[4], {4}, at::kInt, ctx, "free_state");
  // every CTA reads all lengths while others write their share of the outputs
  for (int i = 0; i < 5; ++i) {
    const at::Tensor& o = THPVariable_Unpack(r[i].p);
    for (const at::Tensor* t : {&ctx, &add, &table, &ring, &state})
      require(!overlap(o, *t), "out must not hold inputs of the same call");
    require(a[7] == Py_None || !overlap(o, THPVariable_Unpack(a[7])),
            "out must not hold inputs of the same call");
    for (int j = 0; j < i; ++j)
      require(!overlap(o, THPVariable_Unpack(r[j].p)), "the tensors of out must not overlap");
  }
  {
    const c10::cuda::OptionalCUDAGuard guard(ctx.device());
    check_status(c_plan(data<int>(ctx), data<int>(add), fin, data<int>(table), data<int>(ring),
                        data<int>(state), data<int>(THPVariable_Unpack(r[0].p)),
                        data<int>(THPVariable_Unpack(r[1].p)),
                        data<int>(THPVariable_Unpack(r[2].p)),
                        reinterpret_cast<long long*>(data<int64_t>(THPVariable_Unpack(r[3].p))),
                        data<int>(THPVariable_Unpack(r[4].p)), S, width, dim32(ring, 0),
                        integer32(a[5]), static_cast<int>(cap), stream_of(ctx)),
                 "plan_paged_step");
  }
  Ref t;
  t.p = PyTuple_New(5);
  if (!t.p) throw Refusal{nullptr, {}};
  for (int i = 0; i < 5; ++i) PyTuple_SET_ITEM(t.p, i, r[i].release());
  return t.release();
}

// The arguments of the boxes' entry, checked; tokens = 0 asks the entry itself to check its own
// and launch nothing.
struct BoundsCall {
  const at::Tensor *k, *values, *scales, *slots;
  CacheDims c;
  int block_size, dtype, layout;
  BoundsCall(const at::Tensor& key_cache, PyObject* pair, const at::Tensor& slot_list, int bs,
             int lay)
      : k(&key_cache), slots(&slot_list), block_size(bs), dtype(dtype_code(key_cache.scalar_type())),
        layout(lay) {
    if (dtype < 0) refuse(PyExc_TypeError, "unsupported dtype of key_cache");
    c = cache_dims(key_cache, bs, lay);
    check_bounds(pair, c, key_cache, &values, &scales);
    require(slot_list.scalar_type() == at::kLong && slot_list.dim() == 1,
            "slots int64 [T] expected");
    same_device(key_cache, slot_list);
    run(0);
  }
  void run(int tokens) const {
    const c10::cuda::OptionalCUDAGuard guard(k->device());
    check_status(c_bounds(k->data_ptr(), data<signed char>(*values), data<float>(*scales),
                          reinterpret_cast<const long long*>(data<int64_t>(*slots)), tokens,
                          c.heads, c.dim, block_size, c.blocks, dtype, layout, stream_of(*k)),
                 "update_page_bounds");
  }
};

// (key_cache, page_bounds, slots, block_size, kv_layout)
PyObject* bounds(PyObject* const* a) {
  const at::Tensor& slots = contiguous(a[2]);
  BoundsCall(contiguous(a[0]), a[1], slots, integer32(a[3]), layout_code(a[4]))
      .run(dim32(slots, 0));
  Py_RETURN_NONE;
}

// (qkv, key_cache, value_cache, positions, slots, num_heads, block_size, q_weight, k_weight,
//  eps, rope, interleaved, kv_layout, page_bounds, out) -> queries
PyObject* append(PyObject* const* a) {
  const at::Tensor& qkv = tensor(a[0]);
  const at::Tensor& k = contiguous(a[1]);
  const at::Tensor& v = contiguous(a[2]);
  const at::Tensor& pos = contiguous(a[3]);
  const at::Tensor& slots = contiguous(a[4]);
  const int heads = integer32(a[5]), bs = integer32(a[6]), layout = layout_code(a[12]);
  const int dt = dtype_code(qkv.scalar_type());
  if (dt < 0) refuse(PyExc_TypeError, "unsupported dtype of qkv");
  const CacheDims c = cache_dims(k, bs, layout);
  require(k.scalar_type() == qkv.scalar_type(), "the caches must be of qkv's dtype");
  check_value_cache(k, v, c, bs, layout);
  require(layout == 0 || dt != 2, "the fp32 cache takes the flat layout");
  require(heads >= 1 && qkv.dim() == 2 && qkv.size(1) == (heads + 2LL * c.heads) * c.dim,
          "qkv must be [T, (num_heads + 2 Hkv) * d]");
  const int T = dim32(qkv, 0);
  const int64_t stride = T > 1 ? qkv.stride(0) : qkv.size(1);
  require(qkv.stride(1) == 1 && stride >= qkv.size(1),
          "the elements of a row of qkv must be contiguous, rows apart");
  require(pos.scalar_type() == at::kInt && slots.scalar_type() == at::kLong && pos.dim() == 1 &&
              slots.dim() == 1 && pos.size(0) == T && slots.size(0) == T,
          "positions int32 [T] and slots int64 [T] expected");
  for (const at::Tensor* t : {&k, &v, &pos, &slots}) same_device(qkv, *t);
  const void* w[2] = {nullptr, nullptr};
  int wtype = -1;
  for (int i = 0; i < 2; ++i) {
    if (a[7 + i] == Py_None) continue;
    const at::Tensor& x = contiguous(a[7 + i]);
    same_device(qkv, x);
    const int xt = dtype_code(x.scalar_type());
    require(x.dim() == 1 && x.size(0) == c.dim && (xt == dt || xt == 2),
            "norm weights must be [d] of qkv's dtype or float32");
    require(wtype < 0 || wtype == xt, "norm weights must share a dtype");
    wtype = xt;
    w[i] = x.data_ptr();
  }
  const float *cos = nullptr, *sin = nullptr;
  int rotary = 0, max_pos = 0;
  Ref seq;  // until the launch: the tables of an iterator have no other owner
  if (a[10] != Py_None) {
    seq.p = PySequence_Tuple(a[10]);
    if (!seq.p) throw Refusal{nullptr, {}};
    require(PyTuple_GET_SIZE(seq.p) == 2, "rope must be (cos, sin)");
    const at::Tensor& x = contiguous(PyTuple_GET_ITEM(seq.p, 0));
    const at::Tensor& y = contiguous(PyTuple_GET_ITEM(seq.p, 1));
    same_device(qkv, x);
    same_device(qkv, y);
    require(x.scalar_type() == at::kFloat && y.scalar_type() == at::kFloat && x.dim() == 2 &&
                x.sizes() == y.sizes() && x.size(1) >= 1 && x.size(1) <= c.dim / 2,
            "rope tables must be float32 [max_pos, r/2] with r <= d");
    cos = data<float>(x);
    sin = data<float>(y);
    rotary = 2 * dim32(x, 1);
    max_pos = dim32(x, 0);
  }
  const int interleaved = PyObject_IsTrue(a[11]);
  if (interleaved < 0) throw Refusal{nullptr, {}};
  const double eps = number(a[9]);
  // all that can be refused before the caches are written
  std::optional<BoundsCall> boxes;
  if (a[13] != Py_None) boxes.emplace(k, a[13], slots, bs, layout);
  Ref out;
  out.p = buffer(a[14], {T, heads, c.dim}, qkv.scalar_type(), qkv, "out");
  void* const out_at = THPVariable_Unpack(out.p).data_ptr();
  void *const qkv_at = qkv.data_ptr(), *const k_at = k.data_ptr(), *const v_at = v.data_ptr();
  if (a[14] != Py_None) {
    const int64_t e = dt == 2 ? 4 : 2, n = e * T * heads * c.dim;
    const int64_t cache = e * c.blocks * c.heads * bs * c.dim;
    require(!overlap(out_at, n, qkv_at, e * ((T - 1) * stride + (heads + 2LL * c.heads) * c.dim)) &&
                !overlap(out_at, n, k_at, cache) && !overlap(out_at, n, v_at, cache),
            "out must not overlap qkv or the caches");
  }
  {
    const c10::cuda::OptionalCUDAGuard guard(qkv.device());
    check_status(
        c_append(qkv_at, stride, out_at, k_at, v_at, data<int>(pos),
                 reinterpret_cast<const long long*>(data<int64_t>(slots)), w[0], w[1], wtype == 2,
                 static_cast<float>(eps), cos, sin, rotary, max_pos, interleaved, T, heads, c.heads,
                 c.dim, bs, c.blocks, dt, layout, stream_of(qkv)),
        "paged_qkv_append");
  }
  if (boxes) boxes->run(T);
  return out.release();
}

// (query, key_cache, value_cache, page_bounds, block_tables, context_lens, num_pages,
//  block_size, scale, keep_first, keep_last, kv_layout, workspace, out, selected)
//  -> (out, selected)
PyObject* sparse(PyObject* const* a) {
  const at::Tensor& q = contiguous(a[0]);
  const at::Tensor& k = contiguous(a[1]);
  const at::Tensor& v = contiguous(a[2]);
  const at::Tensor& table = contiguous(a[4]);
  const at::Tensor& lens = contiguous(a[5]);
  const int pages = integer32(a[6]), bs = integer32(a[7]), layout = layout_code(a[11]);
  const int first = integer32(a[9]), last = integer32(a[10]);
  const CacheDims c = cache_dims(k, bs, layout);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    refuse(PyExc_TypeError,
           "query and caches must share a dtype: bfloat16, float16 or float32");
  check_value_cache(k, v, c, bs, layout);
  require(q.dim() == 3 && q.size(2) == c.dim, "query [S, H, d] expected");
  const int S = dim32(q, 0), H = dim32(q, 1);
  require(c.heads > 0 && H % c.heads == 0, "num_heads must be a multiple of num_kv_heads");
  if (table.scalar_type() != at::kInt || lens.scalar_type() != at::kInt)
    refuse(PyExc_TypeError, "block_tables and context_lens must be int32");
  require(table.dim() == 2 && table.size(0) == S && lens.dim() == 1 && lens.size(0) == S,
          "block_tables [S, max_blocks] and context_lens [S] expected");
  for (const at::Tensor* t : {&k, &v, &table, &lens}) same_device(q, *t);
  const at::Tensor *values, *scales;
  check_bounds(a[3], c, q, &values, &scales);
  float scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(c.dim)));
  if (a[8] != Py_None) {
    // as the kernels take it: one that is 0 in fp32 would ask the entry for its default
    scale = static_cast<float>(number(a[8]));
    require(scale > 0, "scale must be positive in float32");
  }
  require(first >= 0 && last >= 1 && pages >= first + static_cast<long long>(last),
          "keep_first >= 0, keep_last >= 1 and num_pages >= their sum expected");
  float* ws = nullptr;
  size_t ws_floats = static_cast<size_t>(-1);  // FE_WORKSPACE_LIBRARY
  if (a[12] != Py_None) {
    const at::Tensor& w = contiguous(a[12]);
    same_device(q, w);
    require(w.scalar_type() == at::kFloat, "workspace must be float32");
    ws = data<float>(w);
    ws_floats = static_cast<size_t>(w.numel());
  }
  const int maxb = dim32(table, 1);
  Ref out, sel;
  out.p = buffer(a[13], q.sizes(), q.scalar_type(), q, "out");
  sel.p = buffer(a[14], {S, c.heads, pages}, at::kInt, q, "selected");
  const at::Tensor scratch =
      at::empty({static_cast<int64_t>(c_scratch(S, c.heads, maxb, pages))},
                q.options().dtype(at::kInt));
  {
    const c10::cuda::OptionalCUDAGuard guard(q.device());
    check_status(
        c_sparse(q.data_ptr(), k.data_ptr(), v.data_ptr(), THPVariable_Unpack(out.p).data_ptr(),
                 data<signed char>(*values), data<float>(*scales), data<int>(table),
                 data<int>(lens), data<int>(THPVariable_Unpack(sel.p)), data<int>(scratch), S, H,
                 c.heads, c.dim, bs, maxb, c.blocks, pages, first, last,
                 scale, dt, layout, ws, ws_floats, stream_of(q)),
        "sparse_paged_attention");
  }
  Ref t;
  t.p = PyTuple_New(2);
  if (!t.p) throw Refusal{nullptr, {}};
  PyTuple_SET_ITEM(t.p, 0, out.release());
  PyTuple_SET_ITEM(t.p, 1, sel.release());
  return t.release();
}

// (plan, append, bounds, sparse, scratch): addresses of the C entries
PyObject* bind(PyObject* const* a) {
  c_plan = reinterpret_cast<decltype(c_plan)>(integer(a[0]));
  c_append = reinterpret_cast<decltype(c_append)>(integer(a[1]));
  c_bounds = reinterpret_cast<decltype(c_bounds)>(integer(a[2]));
  c_sparse = reinterpret_cast<decltype(c_sparse)>(integer(a[3]));
  c_scratch = reinterpret_cast<decltype(c_scratch)>(integer(a[4]));
  Py_RETURN_NONE;
}

// No C++ exception leaves an entry.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refusal& r) {
    if (r.type) PyErr_SetString(r.type, r.what.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}
template <PyObject* (*F)(PyObject* const*), int N>
constexpr PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)),
          METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<plan, 9>("plan"),     method<append, 15>("append"),
                         method<bounds, 5>("bounds"), method<sparse, 15>("sparse"),
                         method<bind, 5>("bind"),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_step_native", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__step_native() {
  return PyModule_Create(&module);
}
