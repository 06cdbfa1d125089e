// The host side of the operators between two layers, natively: checks of the tensors, outputs, the C call.
//
// A call of a few tokens is 3 to 9 us on the GPU; in Python it took 8 to 12 of the host (now 3.7 to 5.2), most of it
// reading some thirty attributes of tensors.  Here they are read from the tensors themselves.  The kernels stay behind
// the C ABI (include/megaattn_b200.h): this module gets its entry points from the library that the package has
// loaded (bind) and knows nothing else of it.  Refusals are AssertionErrors, as the package's own are.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/megaattn_b200.h"

namespace {

struct Entry {
  decltype(&ma_rmsnorm_quant) norm;
  decltype(&ma_linear_quant) linear;
  decltype(&ma_dequant) dequant;
  decltype(&ma_rope_append) append;
  decltype(&ma_strerror) error;
} entry;

struct Refused {};
#define REQUIRE(condition, message)                          \
  do {                                                       \
    if (!(condition)) {                                      \
      PyErr_SetString(PyExc_AssertionError, message);        \
      throw Refused{};                                       \
    }                                                        \
  } while (0)

const at::Tensor& tensor(PyObject* o, const char* message) {
  REQUIRE(THPVariable_Check(o), message);
  return THPVariable_Unpack(o);
}

uint64_t at_of(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.data_ptr()); }
bool on(const at::Tensor& t, at::ScalarType type, const c10::Device& dev) {
  return t.scalar_type() == type && t.device() == dev;
}
bool vector_of(const at::Tensor& t, int64_t n, at::ScalarType type, const c10::Device& dev) {
  return t.dim() == 1 && t.size(0) == n && on(t, type, dev) && (n <= 1 || t.stride(0) == 1);
}
// Elements from one row to the next (of a single row: its length, up to a multiple of 16).
int64_t pitch_of(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : (t.size(1) + 15) / 16 * 16; }
bool packed_columns(const at::Tensor& t) { return t.size(1) <= 1 || t.stride(1) == 1; }

// Without the dispatcher, 0.3 us of each (a norm's three outputs 6.3 -> 5.5 us of host time), unless somebody wants
// to see it: a dispatch mode, or the filling of fresh memory under deterministic algorithms.
bool outputs_watched() {
  const at::Context& context = at::globalContext();
  return c10::impl::TorchDispatchModeTLS::any_modes_set() ||
         (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory());
}
at::Tensor empty(at::IntArrayRef size, at::ScalarType type, const c10::Device& dev, bool watched) {
  if (watched) return at::empty(size, at::TensorOptions().dtype(type).device(dev));
  return at::Tensor(at::detail::empty_cuda(size, type, dev, std::nullopt));
}

void report(int rc, const char* what) {
  if (rc == MA_OK) return;
  PyErr_Format(PyExc_RuntimeError, "%s: %s (%d)", what, entry.error(rc), rc);
  throw Refused{};
}
// One C call on `stream` (0: the current one of `dev`), with `dev` current.
template <class F, class A>
void queue(F fn, const A& args, const c10::Device& dev, void* stream, const char* what) {
  const c10::cuda::OptionalCUDAGuard guard(dev);
  report(fn(&args, stream ? stream : static_cast<void*>(c10::cuda::getCurrentCUDAStream(dev.index()).stream())), what);
}

// Memory that a call reads or writes, as rows of bytes; a vector is one row.
struct Rows {
  int64_t at, rows, pitch, bytes;
};
Rows rows_of(const at::Tensor& t) {
  const int64_t item = t.element_size();
  const bool vector = t.dim() == 1;
  return {static_cast<int64_t>(at_of(t)), vector ? 1 : t.size(0), vector ? 0 : t.stride(0) * item, t.size(vector ? 0 : 1) * item};
}
// Whether no byte is both's.  What lies between the other's rows is not, if both have the same step from row to row.
bool apart(const Rows& a, const Rows& b) {
  const int64_t gap = b.at - a.at;
  if (gap >= (a.rows - 1) * a.pitch + a.bytes || -gap >= (b.rows - 1) * b.pitch + b.bytes) return true;
  const int64_t step = a.rows <= 1 ? b.pitch : b.rows <= 1 || a.pitch == b.pitch ? a.pitch : 0;
  if (!step) return false;
  const int64_t at = (gap % step + step) % step;
  return at >= a.bytes && at + b.bytes <= step;
}
// Whether a row of one shares memory with the same row of the other only.
bool row_for_row(const Rows& a, const Rows& b) {
  if (a.rows <= 1) return true;
  const int64_t gap = b.at - a.at;
  return a.pitch == b.pitch && (gap >= 0 ? gap + b.bytes : a.bytes - gap) <= a.pitch;
}
bool same_place(const Rows& a, const Rows& b) { return a.at == b.at && (a.rows <= 1 || a.pitch == b.pitch); }

PyObject* optional(PyObject* o) { return o == Py_None ? nullptr : o; }

// An output of `rows` x `n` in the asked type, or the caller's: its row pitch, and whether it is fp32.
at::Tensor output(PyObject* given, PyObject* type, int64_t rows, int64_t n, const c10::Device& dev, int64_t* pitch,
                  int32_t* f32) {
  at::Tensor out;
  if (PyObject* o = optional(given)) {
    out = tensor(o, "out: [rows, columns] bf16 or fp32");
    REQUIRE(out.dim() == 2 && out.size(0) == rows && out.size(1) == n && out.device() == dev,
            "out: [rows, columns] on the device of the inputs");
    REQUIRE(packed_columns(out) && (rows <= 1 || out.stride(0) >= n),
            "out: columns next to each other, no rows that overlap");
    *pitch = rows > 1 ? out.stride(0) : n;
  } else {
    REQUIRE(THPDtype_Check(type), "out_dtype: a torch.dtype");
    const at::ScalarType t = reinterpret_cast<THPDtype*>(type)->scalar_type;
    REQUIRE(t == at::kBFloat16 || t == at::kFloat, "bf16 or fp32");
    out = empty({rows, n}, t, dev, outputs_watched());
    *pitch = n;
  }
  REQUIRE(out.scalar_type() == at::kBFloat16 || out.scalar_type() == at::kFloat, "bf16 or fp32");
  *f32 = out.scalar_type() == at::kFloat;
  return out;
}

// 8-bit rows that a kernel loads 16 bytes at a time.
void eight_bit_rows(const at::Tensor& t, const char* message) {
  REQUIRE(t.dim() == 2 && t.scalar_type() == at::kChar && t.is_cuda(), message);
  REQUIRE(packed_columns(t) && ((at_of(t) | static_cast<uint64_t>(pitch_of(t))) & 15u) == 0,
          "8-bit rows must start at multiples of 16 bytes, columns next to each other");
}

// (x, x_scale, weight, weight_scale, bias, out, out_dtype)
PyObject* linear_int8(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x: [tokens, in] int8");
  const at::Tensor& w = tensor(a[2], "weight: [out, in] int8");
  const at::Tensor& xs = tensor(a[1], "x_scale: [tokens] fp32");
  const at::Tensor& ws = tensor(a[3], "weight_scale: [out] fp32");
  eight_bit_rows(x, "x: [tokens, in] int8 on a CUDA device");
  eight_bit_rows(w, "weight: [out, in] int8 on a CUDA device");
  const c10::Device dev = x.device();
  const int64_t tokens = x.size(0), inner = x.size(1), width = w.size(0);
  REQUIRE(w.size(1) == inner && inner > 0 && w.device() == dev, "x [tokens, in] and weight [out, in] on one device");
  REQUIRE(vector_of(xs, tokens, at::kFloat, dev), "x_scale: [tokens] fp32 on the device of x");
  REQUIRE(vector_of(ws, width, at::kFloat, dev), "weight_scale: [out] fp32 on the device of x");
  uint64_t bias = 0;
  if (PyObject* o = optional(a[4])) {
    const at::Tensor& b = tensor(o, "bias: [out] bf16");
    REQUIRE(vector_of(b, width, at::kBFloat16, dev), "bias: [out] bf16 on the device of x");
    bias = at_of(b);
  }
  REQUIRE(tokens <= INT32_MAX && inner <= INT32_MAX && width <= INT32_MAX, "sizes: 32 bits");
  ma_linear_quant_args args{};
  const at::Tensor out = output(a[5], a[6], tokens, width, dev, &args.out_pitch, &args.out_f32);
  if (tokens && width) {
    if (optional(a[5])) {
      const Rows o = rows_of(out);
      REQUIRE(apart(o, rows_of(x)) && apart(o, rows_of(w)) && apart(o, rows_of(xs)) && apart(o, rows_of(ws)) &&
                  (!bias || apart(o, {static_cast<int64_t>(bias), 1, 0, 2 * width})),
              "out shares memory with an input");
    }
    args.x = at_of(x); args.weight = at_of(w); args.x_scale = at_of(xs); args.weight_scale = at_of(ws);
    args.bias = bias; args.out = at_of(out);
    args.x_pitch = pitch_of(x); args.weight_pitch = pitch_of(w);
    args.tokens = static_cast<int32_t>(tokens); args.inner = static_cast<int32_t>(inner);
    args.width = static_cast<int32_t>(width);
    queue(entry.linear, args, dev, nullptr, "ma_linear_quant");
  }
  return THPVariable_Wrap(out);
}

// (q, scale, out, out_dtype)
PyObject* dequantize_int8(PyObject* const* a) {
  const at::Tensor& q = tensor(a[0], "q: [rows, n] int8");
  const at::Tensor& scale = tensor(a[1], "scale: [rows] fp32");
  eight_bit_rows(q, "q: [rows, n] int8 on a CUDA device");
  const c10::Device dev = q.device();
  const int64_t rows = q.size(0), n = q.size(1);
  REQUIRE(vector_of(scale, rows, at::kFloat, dev), "scale: [rows] fp32 on the device of q");
  REQUIRE(rows <= INT32_MAX && n <= INT32_MAX, "sizes: 32 bits");
  ma_dequant_args args{};
  const at::Tensor out = output(a[2], a[3], rows, n, dev, &args.out_pitch, &args.out_f32);
  if (rows && n) {
    REQUIRE(!optional(a[2]) || (apart(rows_of(out), rows_of(q)) && apart(rows_of(out), rows_of(scale))),
            "out shares memory with an input");
    args.q = at_of(q); args.scale = at_of(scale); args.out = at_of(out);
    args.q_pitch = pitch_of(q);
    args.rows = static_cast<int32_t>(rows); args.cols = static_cast<int32_t>(n);
    queue(entry.dequant, args, dev, nullptr, "ma_dequant");
  }
  return THPVariable_Wrap(out);
}

bool bf16_rows(const at::Tensor& t, int64_t rows, int64_t n, const c10::Device& dev) {
  return t.dim() == 2 && t.size(0) == rows && t.size(1) == n && on(t, at::kBFloat16, dev) && packed_columns(t) &&
         (at_of(t) & 15u) == 0 && (pitch_of(t) & 7) == 0;
}

// (x, weight, eps, residual, inplace, out, scale, tiles): packed rows with tiles None; otherwise x is the fused
// output and tiles (cu_q, fa_b, fa_mb, row tiles, tokens, hidden, row pitch, stream).
PyObject* rmsnorm_int8(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x: [tokens, hidden] bf16");
  const at::Tensor& w = tensor(a[1], "weight: [hidden] bf16");
  REQUIRE(x.is_cuda() && x.scalar_type() == at::kBFloat16, "x: [tokens, hidden] bf16 on a CUDA device");
  const c10::Device dev = x.device();
  ma_rmsnorm_quant_args args{};
  int64_t tokens, hidden, rows;
  void* stream = nullptr;
  if (a[7] == Py_None) {
    REQUIRE(x.dim() == 2 && bf16_rows(x, x.size(0), x.size(1), dev),
            "x: [tokens, hidden], rows must start at multiples of 16 bytes, columns next to each other");
    rows = tokens = x.size(0);
    hidden = x.size(1);
    args.x_pitch = pitch_of(x);
  } else {
    unsigned long long cu_q, fa_b, fa_mb, s;
    long long r, t, h, pitch;
    if (!PyArg_ParseTuple(a[7], "KKKLLLLK", &cu_q, &fa_b, &fa_mb, &r, &t, &h, &pitch, &s)) throw Refused{};
    args.cu_q = cu_q; args.fa_b = fa_b; args.fa_mb = fa_mb;
    rows = r; tokens = t; hidden = h;
    args.x_pitch = pitch;
    stream = reinterpret_cast<void*>(s);
  }
  REQUIRE(hidden % 8 == 0 && hidden > 0 && hidden <= 16384, "hidden: a multiple of 8, up to 16384");
  REQUIRE(vector_of(w, hidden, at::kBFloat16, dev) && (at_of(w) & 15u) == 0, "weight: [hidden] bf16, 16-byte aligned");
  REQUIRE(rows <= INT32_MAX, "sizes: 32 bits");
  const double eps = PyFloat_AsDouble(a[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw Refused{};
  const int inplace = PyObject_IsTrue(a[4]);
  if (inplace < 0) throw Refused{};
  REQUIRE(a[3] != Py_None || !inplace, "inplace needs a residual");
  at::Tensor q, scale, res_out;
  const bool watched = outputs_watched();
  if (PyObject* o = optional(a[5])) {
    q = tensor(o, "out: [tokens, hidden] int8");
    eight_bit_rows(q, "out: [tokens, hidden] int8 on a CUDA device");
    REQUIRE(q.size(0) == tokens && q.size(1) == hidden && q.device() == dev, "out: [tokens, hidden] on the device of x");
    args.q_pitch = pitch_of(q);
  } else {
    args.q_pitch = (hidden + 15) / 16 * 16;
    q = empty({tokens, args.q_pitch}, at::kChar, dev, watched);
    if (args.q_pitch != hidden) q = q.narrow(1, 0, hidden);
  }
  if (PyObject* o = optional(a[6])) {
    scale = tensor(o, "scale: [tokens] fp32");
    REQUIRE(vector_of(scale, tokens, at::kFloat, dev), "scale: [tokens] fp32 on the device of x");
  } else {
    scale = empty({tokens}, at::kFloat, dev, watched);
  }
  if (PyObject* o = optional(a[3])) {
    const at::Tensor& residual = tensor(o, "residual: [tokens, hidden] bf16");
    REQUIRE(bf16_rows(residual, tokens, hidden, dev),
            "residual: [tokens, hidden] bf16 on the device of x, rows must start at multiples of 16 bytes");
    res_out = inplace ? residual : empty({tokens, hidden}, at::kBFloat16, dev, watched);
    args.residual_in = at_of(residual); args.residual_out = at_of(res_out);
    args.residual_in_pitch = pitch_of(residual);
    args.residual_out_pitch = inplace ? args.residual_in_pitch : hidden;
  }
  if (tokens) {
    if (optional(a[5]) || optional(a[6]) || inplace) {
      // A row is read whole before its integers are written, and the residual by the thread that writes it.
      const bool packed = a[7] == Py_None;
      const Rows xr = packed ? rows_of(x) : Rows{static_cast<int64_t>(at_of(x)), 1, 0, x.numel() * 2}, wr = rows_of(w),
                 qr = rows_of(q), sr = rows_of(scale), rr = args.residual_in ? rows_of(tensor(a[3], "")) : wr;
      REQUIRE(apart(qr, wr) && apart(sr, wr) && apart(sr, xr) && apart(sr, rr) && apart(sr, qr) &&
                  (apart(qr, xr) || (packed && row_for_row(qr, xr))) && (apart(qr, rr) || (!inplace && row_for_row(qr, rr))) &&
                  (!inplace || (apart(rr, wr) && (apart(rr, xr) || (packed && same_place(rr, xr))))),
              "out, scale or the updated residual shares memory with an input or another of them");
    }
    args.x = at_of(x); args.weight = at_of(w); args.q_out = at_of(q); args.scale_out = at_of(scale);
    args.rows = static_cast<int32_t>(rows); args.hidden = static_cast<int32_t>(hidden);
    args.eps = static_cast<float>(eps);
    queue(entry.norm, args, dev, stream, "ma_rmsnorm_quant");
  }
  PyObject* result = PyTuple_New(res_out.defined() ? 3 : 2);
  if (!result) throw Refused{};
  const auto put = [&](int i, PyObject* given, const at::Tensor& t) {     // (what was given comes back as it is)
    PyObject* o = given ? (Py_INCREF(given), given) : THPVariable_Wrap(t);
    PyTuple_SET_ITEM(result, i, o);
    return o != nullptr;
  };
  if (!put(0, optional(a[5]), q) || !put(1, optional(a[6]), scale) ||
      (res_out.defined() && !put(2, inplace ? a[3] : nullptr, res_out))) {
    Py_DECREF(result);
    throw Refused{};
  }
  return result;
}

bool heads(const at::Tensor& t, int64_t tokens, int64_t n, const c10::Device& dev) {
  return t.dim() == 3 && t.size(0) == tokens && t.size(1) == n && t.size(2) == 128 && on(t, at::kBFloat16, dev) &&
         t.stride(2) == 1 && (at_of(t) & 15u) == 0 && (t.stride(0) & 7) == 0 && (t.stride(1) & 7) == 0;
}

// Whether two tensors of heads may share memory.  What lies between the other's tokens does not if both have the same
// step from token to token, or else from head to head.
bool mixed(const at::Tensor& a, const at::Tensor& b) {
  const auto reach = [](const at::Tensor& t, int first) {
    int64_t n = 128;
    for (int d = first; d < 2; ++d) n += (t.size(d) - 1) * t.stride(d);
    return n;
  };
  const auto step_of_both = [&](int d) { return a.size(d) <= 1 ? b.stride(d) : b.size(d) <= 1 || a.stride(d) == b.stride(d) ? a.stride(d) : 0; };
  const auto apart = [](int64_t from_a_to_b, int64_t step, int64_t na, int64_t nb) {
    const int64_t at = (from_a_to_b % step + step) % step;
    return at >= na && at + nb <= step;
  };
  const int64_t gap = (static_cast<int64_t>(at_of(b)) - static_cast<int64_t>(at_of(a))) / 2;      // elements
  if (gap >= reach(a, 0) || -gap >= reach(b, 0)) return false;
  const int64_t token = step_of_both(0), head = step_of_both(1);
  if (token && apart(gap, token, reach(a, 1), reach(b, 1))) return false;
  return !(head && (a.size(0) <= 1 || (token && token % head == 0)) && apart(gap, head, 128, 128));
}

// (q, k, v, k_cache, v_cache, page_table, cache_seqlens, cu_seqlens_q, inv_freq, out, dropped)
PyObject* rope_append(PyObject* const* a) {
  const at::Tensor& q = tensor(a[0], "q: [tokens, heads, 128] bf16");
  const at::Tensor& k = tensor(a[1], "k: [tokens, kv heads, 128] bf16");
  const at::Tensor& v = tensor(a[2], "v: [tokens, kv heads, 128] bf16");
  REQUIRE(q.dim() == 3 && k.dim() == 3 && q.is_cuda(), "q [tokens, H, 128]; k, v [tokens, H_kv, 128] on a CUDA device");
  const c10::Device dev = q.device();
  const int64_t tokens = q.size(0), H = q.size(1), Hkv = k.size(1);
  REQUIRE(H > 0 && Hkv > 0 && heads(q, tokens, H, dev) && heads(k, tokens, Hkv, dev) && heads(v, tokens, Hkv, dev),
          "q [tokens, H, 128]; k, v [tokens, H_kv, 128]: bf16 on one CUDA device, heads at multiples of 16 bytes");
  const at::Tensor& kc = tensor(a[3], "k_cache: bf16");
  const at::Tensor& vc = tensor(a[4], "v_cache: bf16");
  for (const at::Tensor* c : {&kc, &vc}) {
    const int64_t d = c->dim();
    REQUIRE((d == 4 ? c->size(1) == 128 : d == 3 && c->size(0) % 128 == 0) && c->size(0) > 0 && c->size(d - 1) == 128 &&
                c->size(d - 2) == Hkv && on(*c, at::kBFloat16, dev) && c->is_contiguous() && (at_of(*c) & 15u) == 0,
            "caches: bf16, contiguous, [num_pages, 128, H_kv, 128] or [num_pages * 128, H_kv, 128]");
  }
  REQUIRE(kc.sizes() == vc.sizes(), "caches of one shape");
  const int64_t pages = kc.dim() == 4 ? kc.size(0) : kc.size(0) / 128;
  const at::Tensor& table = tensor(a[5], "page_table: [batch, pages] int32");
  const at::Tensor& lens = tensor(a[6], "cache_seqlens: [batch] int32");
  const at::Tensor& cu = tensor(a[7], "cu_seqlens_q: [batch + 1] int32, a tensor on the device of q");
  REQUIRE(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0 && on(table, at::kInt, dev) && packed_columns(table),
          "page_table: [batch, pages] int32 on the device of q, columns next to each other");
  const int64_t batch = table.size(0), width = table.size(1);
  REQUIRE(vector_of(lens, batch, at::kInt, dev), "cache_seqlens: [batch] int32 on the device of q");
  REQUIRE(vector_of(cu, batch + 1, at::kInt, dev), "cu_seqlens_q: [batch + 1] int32 on the device of q");
  const at::Tensor& freq = tensor(a[8], "inv_freq: [64] fp32");
  REQUIRE(vector_of(freq, 64, at::kFloat, dev), "inv_freq: [64] fp32 on the device of q");
  at::Tensor out;
  if (PyObject* o = optional(a[9])) {
    out = tensor(o, "out: as q");
    REQUIRE(heads(out, tokens, H, dev), "out: as q");
    const auto apart = [&](int inner, int outer) {        // one dimension's heads lie within a step of the other
      const int64_t ni = out.size(inner), no = out.size(outer), si = out.stride(inner), so = out.stride(outer);
      return (ni <= 1 || si >= 128) && (no <= 1 || so >= (ni <= 1 ? 0 : (ni - 1) * si) + 128);
    };
    REQUIRE(tokens == 0 || apart(1, 0) || apart(0, 1), "heads of out overlap");
    // A warp reads its heads before it writes any of them, and another's at any time.
    const bool in_place = at_of(out) == at_of(q) && (tokens <= 1 || out.stride(0) == q.stride(0)) &&
                          (H <= 1 || out.stride(1) == q.stride(1));
    REQUIRE(tokens == 0 || ((in_place || !mixed(out, q)) && !mixed(out, k) && !mixed(out, v)),
            "out: q itself, or memory that q, k and v have no part in (between their tokens: with their step)");
  } else {
    out = empty({tokens, H, 128}, at::kBFloat16, dev, outputs_watched());
  }
  ma_rope_append_args args{};
  if (PyObject* o = optional(a[10])) {
    const at::Tensor& dropped = tensor(o, "dropped: [1] int32");
    REQUIRE(vector_of(dropped, 1, at::kInt, dev), "dropped: [1] int32 on the device of q");
    args.dropped = at_of(dropped);
  }
  REQUIRE(tokens <= INT32_MAX && H <= INT32_MAX && Hkv <= INT32_MAX && batch < INT32_MAX && width <= INT32_MAX &&
              pages <= INT32_MAX, "sizes: 32 bits");
  if (tokens) {
    args.q = at_of(q); args.k = at_of(k); args.v = at_of(v); args.out = at_of(out);
    args.k_cache = at_of(kc); args.v_cache = at_of(vc);
    args.cu_q = at_of(cu); args.cache_seqlens = at_of(lens); args.page_table = at_of(table); args.inv_freq = at_of(freq);
    args.q_tok = q.stride(0); args.q_head = q.stride(1); args.k_tok = k.stride(0); args.k_head = k.stride(1);
    args.v_tok = v.stride(0); args.v_head = v.stride(1); args.out_tok = out.stride(0); args.out_head = out.stride(1);
    args.table_pitch = batch > 1 ? table.stride(0) : width;
    args.rows = static_cast<int32_t>(tokens); args.num_batch = static_cast<int32_t>(batch);
    args.H_local = static_cast<int32_t>(H); args.H_kv = static_cast<int32_t>(Hkv);
    args.num_pages = static_cast<int32_t>(pages); args.table_width = static_cast<int32_t>(width);
    queue(entry.append, args, dev, nullptr, "ma_rope_append");
  }
  return THPVariable_Wrap(out);
}

// The number of arguments, and C++ exceptions as Python's.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Refused&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// Addresses of the C entry points, in the order of Entry.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[5];
  if (!PyArg_ParseTuple(args, "KKKKK", p, p + 1, p + 2, p + 3, p + 4)) return nullptr;
  entry.norm = reinterpret_cast<decltype(entry.norm)>(p[0]);
  entry.linear = reinterpret_cast<decltype(entry.linear)>(p[1]);
  entry.dequant = reinterpret_cast<decltype(entry.dequant)>(p[2]);
  entry.append = reinterpret_cast<decltype(entry.append)>(p[3]);
  entry.error = reinterpret_cast<decltype(entry.error)>(p[4]);
  Py_RETURN_NONE;
}

#define METHOD(name, n) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<name, n>)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {METHOD(rmsnorm_int8, 8), METHOD(linear_int8, 7), METHOD(dequantize_int8, 4),
                         METHOD(rope_append, 11), {"bind", bind, METH_VARARGS, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", MA_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
