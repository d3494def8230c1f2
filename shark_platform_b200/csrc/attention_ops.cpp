// The cache operators of attention.py for torch tensors: argument checks, outputs and the
// call of the C ABI.  They run once per layer and token, beside kernels of a few
// microseconds; the same work in Python and ctypes took the host 20 / 15 / 17 us a call
// (write, read, attend).  The library's entry points come as addresses from the ctypes
// binding, so that there is one copy of it in the process.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <string>

#include "../../include/b200moe.h"

namespace {

decltype(&b200moe_attn_norm_rope_kv8_write) write8 = nullptr;
decltype(&b200moe_attn_norm_rope_kv_write) write_plain = nullptr;
decltype(&b200moe_kv8_read) read8 = nullptr;
decltype(&b200moe_kv8_attend) attend8 = nullptr;
decltype(&b200moe_kv8_attend_scratch_bytes) attend8_scratch = nullptr;
decltype(&b200moe_last_error) last_error = nullptr;
PyObject* error_class = nullptr;  // B200MoeError

struct Refused : std::exception {
  std::string message;
  explicit Refused(std::string m) : message(std::move(m)) {}
};
inline std::string text(const char* s) { return s; }
inline const std::string& text(const std::string& s) { return s; }
inline std::string text(int64_t n) { return std::to_string(n); }
template <typename... A>
[[noreturn]] void refuse(const A&... parts) {
  throw Refused((std::string() + ... + text(parts)));
}
struct PythonError : std::exception {};  // the interpreter has the error already

#define OPS_BEGIN HANDLE_TH_ERRORS try {
#define OPS_END                                             \
  }                                                         \
  catch (const Refused& e) {                                \
    PyErr_SetString(error_class, e.message.c_str());        \
    return nullptr;                                         \
  }                                                         \
  catch (const PythonError&) {                              \
    return nullptr;                                         \
  }                                                         \
  END_HANDLE_TH_ERRORS

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(what, " must be a tensor");
  return THPVariable_Unpack(o);
}
int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError();
  return v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PythonError();
  return v;
}
int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? B200MOE_DT_F32 : t == at::kHalf ? B200MOE_DT_F16 : t == at::kBFloat16 ? B200MOE_DT_BF16 : -1;
}
std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
at::Tensor as_int32(const at::Tensor& t) {
  return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
}

// (blocks, stride, kv_heads, head_dim, scale_block, code): code -1 is a 16- or 32-bit cache
struct Geometry {
  int64_t blocks, stride, kv_heads, head_dim, scale_block, code;
  explicit Geometry(PyObject* t) {
    if (!PyTuple_Check(t) || PyTuple_GET_SIZE(t) != 6) refuse("a cache geometry is a tuple of six numbers");
    int64_t* to[6] = {&blocks, &stride, &kv_heads, &head_dim, &scale_block, &code};
    for (int i = 0; i < 6; ++i) *to[i] = integer(PyTuple_GET_ITEM(t, i));
    for (int i = 0; i < 4; ++i)
      if (*to[i] < 1 || *to[i] > 0x7fffffff) refuse("bad cache geometry");
    if (code >= 0 && (scale_block < 1 || scale_block > 0x7fffffff)) refuse("bad cache geometry");
  }
  bool quantized() const { return code >= 0; }
  at::ScalarType dtype() const { return code == B200MOE_KV8_INT8 ? at::kChar : at::kFloat8_e4m3fn; }
};

// The cache's tensors and page table, looked over.
struct State {
  const at::Tensor* slab;
  const at::Tensor* scales = nullptr;
  at::Tensor ids;
  State(PyObject* list, const Geometry& g, int64_t block_index, PyObject* seq_block_ids, int64_t bs, const at::Device& dev) {
    if (!PyList_Check(list) && !PyTuple_Check(list)) refuse("cache_state is a list of tensors, as allocate() gives it");
    PyObject** items = PySequence_Fast_ITEMS(list);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    if (block_index < 0 || block_index >= g.blocks)
      refuse("block_index ", block_index, " is not one of the cache's ", g.blocks, " transformer blocks");
    if (n < 1) refuse("cache_state is a list of tensors, as allocate() gives it");
    slab = &tensor(items[0], "the page slab");
    if (slab->dim() != 2 || slab->size(1) != g.blocks * 2 * g.stride * g.kv_heads * g.head_dim || !slab->is_contiguous())
      refuse("the page slab must be contiguous, a row of the cache's page size per page");
    if (g.quantized()) {
      if (n != 2) refuse("a cache of 8-bit codes is [page slab, scales], as allocate() gives it");
      scales = &tensor(items[1], "scales");
      if (slab->scalar_type() != g.dtype())
        refuse("the page slab must be ", at::toString(g.dtype()), ", got ", at::toString(slab->scalar_type()));
      if (scales->scalar_type() != at::kFloat || scales->dim() != 2 || scales->size(0) != slab->size(0) ||
          scales->size(1) != g.blocks * g.kv_heads * (g.stride / g.scale_block) * 2 || !scales->is_contiguous() ||
          scales->device() != dev)
        refuse("scales must be fp32, contiguous, beside the slab, a row per page");
    } else if (dtype_code(slab->scalar_type()) < 0) {
      refuse("the page slab must be a contiguous fp32, fp16 or bf16 tensor");
    }
    if (slab->size(0) > 0x7fffffff) refuse("too many pages");
    const at::Tensor& table = tensor(seq_block_ids, "seq_block_ids");
    if (table.dim() != 2 || table.size(0) != bs || table.size(1) < 1 || table.size(1) > 0x7fffffff)
      refuse("seq_block_ids must be [", bs, ", pages of a sequence], got ", shape_of(table));
    if (slab->device() != dev || table.device() != dev) refuse("cache, page ids and activations must be on one device");
    ids = table;
  }
  b200moe_kv8_cache_t desc8(const Geometry& g) const {
    return {static_cast<int32_t>(g.blocks), static_cast<int32_t>(g.stride), static_cast<int32_t>(g.kv_heads),
            static_cast<int32_t>(g.head_dim), static_cast<int32_t>(slab->size(0)), static_cast<int32_t>(g.scale_block),
            static_cast<int32_t>(g.code)};
  }
};

void need_cuda(const at::Tensor& t, const char* what) {
  if (!t.is_cuda()) refuse(what, " must be a CUDA tensor (there is no CPU path)");
}
void need_vector(const at::Tensor& t, int64_t bs, const at::Device& dev, const char* message) {
  if (t.dim() != 1 || t.size(0) != bs || t.device() != dev || at::isFloatingType(t.scalar_type())) refuse(message);
}

// [bs, sl, heads, hd] as rows of heads * hd elements one stride apart, 16-byte aligned (a
// view of a fused projection is that already; another tensor is copied)
struct Rows {
  at::Tensor t;
  int64_t stride;
  explicit Rows(const at::Tensor& x) : t(x) {
    const auto n = x.sizes(), s = x.strides();
    const int64_t row = n[2] * n[3];
    if (s[3] == 1 && (n[2] == 1 || s[2] == n[3]) && (n[0] == 1 || n[1] == 1 || s[0] == n[1] * s[1])) {
      stride = n[1] > 1 ? s[1] : n[0] > 1 ? s[0] : row;
      if (stride >= row && stride * x.element_size() % 16 == 0 && reinterpret_cast<uintptr_t>(x.const_data_ptr()) % 16 == 0)
        return;
    }
    t = x.clone(at::MemoryFormat::Contiguous);
    stride = row;
  }
};

// fn(stream) with `dev` current
template <typename F>
void launch(const char* what, const at::Device& dev, F fn) {
  const c10::cuda::OptionalCUDAGuard guard(dev);
  const int rc = fn(static_cast<void*>(c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  if (rc != 0) refuse(what, " failed (", static_cast<int64_t>(rc), "): ", last_error());
}
int32_t i32(int64_t v, const char* what) {
  if (v < 0 || v > 0x7fffffff) refuse(what, " ", v, " does not fit 32 bits");
  return static_cast<int32_t>(v);
}
const void* data(const at::Tensor& t) { return t.const_data_ptr(); }

// bind(error class, addresses): the library's entry points
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  OPS_BEGIN
  if (n != 7) refuse("bind takes the error class and six addresses");
  auto address = [&](int i) { return reinterpret_cast<void*>(static_cast<uintptr_t>(integer(a[i]))); };
  Py_INCREF(a[0]);
  error_class = a[0];
  write8 = reinterpret_cast<decltype(write8)>(address(1));
  write_plain = reinterpret_cast<decltype(write_plain)>(address(2));
  read8 = reinterpret_cast<decltype(read8)>(address(3));
  attend8 = reinterpret_cast<decltype(attend8)>(address(4));
  attend8_scratch = reinterpret_cast<decltype(attend8_scratch)>(address(5));
  last_error = reinterpret_cast<decltype(last_error)>(address(6));
  Py_RETURN_NONE;
  OPS_END
}

// write(q, k, v, cache_state, geometry, block_index, seq_block_ids, start_positions, new_lens, freqs, q_norm, k_norm,
//       eps, use_hf) -> (rotated q, rotated k)
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  OPS_BEGIN
  if (n != 14) refuse("write takes 14 arguments");
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  const Geometry g(a[4]);
  const int dt = dtype_code(q.scalar_type());
  if (dt < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type())
    refuse("q, k and v must be fp32, fp16 or bf16 alike, got ", at::toString(q.scalar_type()), ", ",
           at::toString(k.scalar_type()), ", ", at::toString(v.scalar_type()));
  if (q.dim() != 4 || q.size(3) != g.head_dim || q.size(2) % g.kv_heads != 0 || k.dim() != 4 || k.size(0) != q.size(0) ||
      k.size(1) != q.size(1) || k.size(2) != g.kv_heads || k.size(3) != g.head_dim || v.sizes() != k.sizes())
    refuse("q ", shape_of(q), ", k ", shape_of(k), ", v ", shape_of(v), " do not fit a cache of ", g.kv_heads, " heads of ",
           g.head_dim);
  const int64_t bs = q.size(0), sl = q.size(1), heads = q.size(2), hd = q.size(3);
  const at::Device dev = q.device();
  const at::Tensor& start = tensor(a[7], "start_positions");
  need_vector(start, bs, dev, "start_positions is one whole number for each sequence, on q's device");
  std::optional<at::Tensor> lens;
  if (a[8] != Py_None) {
    lens = tensor(a[8], "new_lens");
    need_vector(*lens, bs, dev, "new_lens is one whole number for each sequence, on q's device");
    lens = as_int32(*lens);
  }
  const at::Tensor& freqs = tensor(a[9], "freqs");
  if (freqs.scalar_type() != at::kFloat || freqs.dim() != 1 || freqs.size(0) != hd / 2 || !freqs.is_contiguous() ||
      freqs.device() != dev)
    refuse("freqs must be fp32 [", hd / 2, "], on q's device");
  const float* norm[2] = {nullptr, nullptr};
  for (int i = 0; i < 2; ++i) {
    if (a[10 + i] == Py_None) continue;
    const at::Tensor& w = tensor(a[10 + i], "a norm weight");
    if (w.scalar_type() != at::kFloat || w.dim() != 1 || w.size(0) != hd || !w.is_contiguous() || w.device() != dev)
      refuse("norm weights must be fp32 [", hd, "], on q's device");
    norm[i] = static_cast<const float*>(data(w));
  }
  const float eps = static_cast<float>(number(a[12]));
  const int hf = PyObject_IsTrue(a[13]);
  if (hf < 0) throw PythonError();
  const int64_t block_index = integer(a[5]);
  State s(a[3], g, block_index, a[6], bs, dev);
  if (k.device() != dev || v.device() != dev) refuse("all arguments must be on one device");
  need_cuda(q, "q");
  const Rows qr(q), kr(k), vr(v);
  at::Tensor q_out = at::empty({bs, sl, heads, hd}, q.options().memory_format(std::nullopt));
  at::Tensor k_out = at::empty({bs, sl, g.kv_heads, hd}, q.options().memory_format(std::nullopt));
  if (bs * sl > 0) {
    const at::Tensor ids = as_int32(s.ids), at0 = as_int32(start);
    const int32_t n_bs = i32(bs, "batch"), n_sl = i32(sl, "tokens"), n_heads = i32(heads, "heads");
    const int32_t* lens_p = lens ? static_cast<const int32_t*>(data(*lens)) : nullptr;
    if (g.quantized()) {
      const b200moe_kv8_cache_t desc = s.desc8(g);
      launch("attn_norm_rope_kv8_write", dev, [&](void* stream) {
        return write8(data(qr.t), data(kr.t), data(vr.t), dt, qr.stride, kr.stride, vr.stride, norm[0], norm[1], eps,
                      q_out.mutable_data_ptr(), k_out.mutable_data_ptr(), s.slab->mutable_data_ptr(),
                      static_cast<float*>(s.scales->mutable_data_ptr()), &desc, static_cast<int32_t>(block_index),
                      static_cast<const int32_t*>(data(at0)), lens_p, static_cast<const int32_t*>(data(ids)),
                      static_cast<const float*>(data(freqs)), hf, n_bs, n_sl, static_cast<int32_t>(ids.size(1)), n_heads,
                      stream);
      });
    } else {
      const b200moe_kv_cache_t desc = {static_cast<int32_t>(g.blocks), static_cast<int32_t>(g.stride),
                                       static_cast<int32_t>(g.kv_heads), static_cast<int32_t>(hd),
                                       static_cast<int32_t>(s.slab->size(0))};
      launch("attn_norm_rope_kv_write", dev, [&](void* stream) {
        return write_plain(data(qr.t), data(kr.t), data(vr.t), dt, qr.stride, kr.stride, vr.stride, norm[0], norm[1], eps,
                           q_out.mutable_data_ptr(), k_out.mutable_data_ptr(), s.slab->mutable_data_ptr(),
                           dtype_code(s.slab->scalar_type()), &desc, static_cast<int32_t>(block_index),
                           static_cast<const int32_t*>(data(at0)), lens_p, static_cast<const int32_t*>(data(ids)),
                           static_cast<const float*>(data(freqs)), hf, n_bs, n_sl, static_cast<int32_t>(ids.size(1)),
                           n_heads, stream);
      });
    }
  }
  PyObject* first = THPVariable_Wrap(std::move(q_out));
  PyObject* second = THPVariable_Wrap(std::move(k_out));
  return Py_BuildValue("(NN)", first, second);
  OPS_END
}

at::ScalarType scalar_type(PyObject* o, at::ScalarType otherwise) {
  if (o == Py_None) return otherwise;
  if (!THPDtype_Check(o)) refuse("a dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// read(cache_state, geometry, block_index, seq_block_ids, seq_lens, max_seq_len, dtype) -> (K, V)
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  OPS_BEGIN
  if (n != 7) refuse("read takes 7 arguments");
  const Geometry g(a[1]);
  if (!g.quantized()) refuse("kv_read reads caches of 8-bit codes");
  const at::ScalarType type = scalar_type(a[6], at::kBFloat16);
  if (dtype_code(type) < 0) refuse("K and V are read as fp32, fp16 or bf16, not ", at::toString(type));
  const at::Tensor &lens = tensor(a[4], "seq_lens"), &table = tensor(a[3], "seq_block_ids");
  if (table.dim() != 2) refuse("seq_block_ids must be [sequences, pages of a sequence], got ", shape_of(table));
  const int64_t bs = table.size(0), block_index = integer(a[2]);
  const at::Device dev = table.device();
  need_vector(lens, bs, dev, "seq_lens is one whole number for each sequence, on the cache's device");
  State s(a[0], g, block_index, a[3], bs, dev);
  need_cuda(*s.slab, "the page slab");
  const int64_t held = table.size(1) * g.stride, rows = a[5] == Py_None ? held : integer(a[5]);
  if (rows < 0 || rows > held) refuse("max_seq_len ", rows, ": the listed pages hold ", held, " positions");
  const auto options = s.slab->options().dtype(type);
  at::Tensor k = at::empty({bs, rows, g.kv_heads, g.head_dim}, options), v = at::empty({bs, rows, g.kv_heads, g.head_dim}, options);
  if (bs * rows > 0) {
    const at::Tensor ids = as_int32(s.ids), len = as_int32(lens);
    const b200moe_kv8_cache_t desc = s.desc8(g);
    const int32_t n_bs = i32(bs, "batch"), n_rows = i32(rows, "max_seq_len");
    launch("kv8_read", dev, [&](void* stream) {
      return read8(data(*s.slab), static_cast<const float*>(data(*s.scales)), &desc, static_cast<int32_t>(block_index),
                   static_cast<const int32_t*>(data(ids)), static_cast<const int32_t*>(data(len)), n_bs,
                   static_cast<int32_t>(ids.size(1)), n_rows, k.mutable_data_ptr(), v.mutable_data_ptr(), dtype_code(type),
                   stream);
    });
  }
  PyObject* first = THPVariable_Wrap(std::move(k));
  PyObject* second = THPVariable_Wrap(std::move(v));
  return Py_BuildValue("(NN)", first, second);
  OPS_END
}

// attend(q, cache_state, geometry, block_index, seq_block_ids, seq_lens, scale, softcap, out_dtype) -> out
PyObject* attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  OPS_BEGIN
  if (n != 9) refuse("attend takes 9 arguments");
  const at::Tensor& q = tensor(a[0], "q");
  const Geometry g(a[2]);
  if (!g.quantized()) refuse("kv_attend reads caches of 8-bit codes");
  const at::ScalarType type = scalar_type(a[8], q.scalar_type());
  const int dt = dtype_code(q.scalar_type()), out_dt = dtype_code(type);
  if (dt < 0 || out_dt < 0)
    refuse("activations must be fp32, fp16 or bf16, got ", at::toString(q.scalar_type()), ", ", at::toString(type));
  if (q.dim() != 4 || q.size(3) != g.head_dim || q.size(2) % g.kv_heads != 0 || q.size(2) < 1)
    refuse("q ", shape_of(q), " does not fit a cache of ", g.kv_heads, " heads of ", g.head_dim);
  const int64_t bs = q.size(0), sl = q.size(1), heads = q.size(2), hd = q.size(3), block_index = integer(a[3]);
  if (sl < 1 || sl > 16) refuse(sl, " new tokens: 1 to 16; longer stretches attend kv_read's K and V");
  const double scale = a[6] == Py_None ? 1.0 / std::sqrt(static_cast<double>(hd)) : number(a[6]);
  const double softcap = a[7] == Py_None ? 0.0 : number(a[7]);
  if (a[7] != Py_None && !(softcap > 0.0 && std::isfinite(static_cast<float>(softcap)))) refuse("softcap must be positive and finite");
  const at::Device dev = q.device();
  const at::Tensor& lens = tensor(a[5], "seq_lens");
  need_vector(lens, bs, dev, "seq_lens is one whole number for each sequence, on q's device");
  State s(a[1], g, block_index, a[4], bs, dev);
  need_cuda(q, "q");
  const Rows qr(q);
  at::Tensor out = at::empty({bs, sl, heads, hd}, q.options().dtype(type).memory_format(std::nullopt));
  if (bs > 0) {
    const at::Tensor ids = as_int32(s.ids), len = as_int32(lens);
    const b200moe_kv8_cache_t desc = s.desc8(g);
    const int32_t max_len = i32(ids.size(1) * g.stride, "positions"), n_bs = i32(bs, "batch"), n_heads = i32(heads, "heads");
    launch("kv8_attend", dev, [&](void* stream) {
      // per call: other streams and captured graphs have their own
      const size_t bytes = attend8_scratch(&desc, n_bs, static_cast<int32_t>(sl), n_heads, max_len);
      at::Tensor scratch = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte).memory_format(std::nullopt));
      return attend8(data(qr.t), dt, qr.stride, data(*s.slab), static_cast<const float*>(data(*s.scales)), &desc,
                     static_cast<int32_t>(block_index), static_cast<const int32_t*>(data(ids)),
                     static_cast<const int32_t*>(data(len)), n_bs, static_cast<int32_t>(sl),
                     static_cast<int32_t>(ids.size(1)), n_heads, max_len, static_cast<float>(scale),
                     static_cast<float>(softcap), out.mutable_data_ptr(), out_dt, scratch.mutable_data_ptr(), bytes, stream);
    });
  }
  return THPVariable_Wrap(std::move(out));
  OPS_END
}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(bind)), METH_FASTCALL, "the library's entry points"},
    {"write", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(write)), METH_FASTCALL, "attention.norm_rope_kv_write"},
    {"read", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(read)), METH_FASTCALL, "attention.kv_read"},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attend)), METH_FASTCALL, "attention.kv_attend"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention_ops", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__attention_ops() { return PyModule_Create(&module); }
