// Host path of the operators around a layer's attention (plan_step, rms_norm_mx8, silu_mul_mx8, fp4_linear): checks, output
// allocation and the call of the C ABI, as a CPython module over torch's C++ tensors.
//
// A decode step calls these several times per layer for 2.5 to 6 us of GPU work each; from Python a call cost the host 11 to 15 us
// (an allocation 1.4 to 2.4 us, twenty attribute reads and comparisons 3 to 5, the launch through ctypes 3).  The entry points
// come from the library that uq_cuda.lib() has loaded (`bind`), as the types that uq_b200.h gives them; a library built from another text of that
// header is refused.
#include <ATen/ATen.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstdint>

#include "uq_b200.h"

namespace {

using at::Tensor;
using std::optional;
typedef long long ll;

decltype(&uqb_plan_step_launch) plan_fn = nullptr;
decltype(&uqb_rms_norm_mx8_launch) norm_fn = nullptr;
decltype(&uqb_silu_mul_mx8_launch) silu_fn = nullptr;
decltype(&uqb_fp4_linear_scratch_bytes) scratch_fn = nullptr;
decltype(&uqb_fp4_linear_launch) linear_fn = nullptr;

#define REFUSE(cond, ...) TORCH_CHECK(!(cond), __VA_ARGS__)

const Tensor& tensor(PyObject* o, const char* what) {
  REFUSE(!THPVariable_Check(o), "uq_cuda: ", what, " must be a tensor");
  return THPVariable_Unpack(o);
}
optional<Tensor> maybe(PyObject* o, const char* what) {
  if (o == Py_None) return std::nullopt;
  return tensor(o, what);
}

// The device of a call: that of its first tensor; every other one has to live there.
struct Place {
  explicit Place(const Tensor& first) : device(first.device()) { need(first); }
  void need(const Tensor& t) const {
    REFUSE(!t.is_cuda(), "uq_cuda: tensors must live on a CUDA device (no CPU path in this library)");
    REFUSE(t.device() != device, "uq_cuda: tensors must live on one device");
  }
  void need(const optional<Tensor>& t) const {
    if (t) need(*t);
  }
  c10::Device device;
};

// Contiguous and 16-byte aligned, as the kernels read it (a copy where it is not).
Tensor rows(const Tensor& t) {
  Tensor c = t.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) ? c.clone() : c;
}
// Do two contiguous tensors share memory?
bool overlap(const Tensor& a, const Tensor& b) {
  const char *p = static_cast<const char*>(a.data_ptr()), *q = static_cast<const char*>(b.data_ptr());
  return p < q + b.nbytes() && q < p + a.nbytes();
}
// An input that shares memory with an output is copied, unless they are the same elements (`in_place`: every thread reads its own before it writes them).
void apart(Tensor& in, const optional<Tensor>& out, bool in_place = false) {
  if (out && overlap(in, *out) && !(in_place && in.data_ptr() == out->data_ptr())) in = in.clone();
}
int dtype_code(at::ScalarType t) { return t == at::kFloat ? 0 : (t == at::kBFloat16 ? 1 : (t == at::kHalf ? 2 : -1)); }
void done(int err, const char* what) {
  REFUSE(err == 1, what, " failed: cudaErrorInvalidValue (shape not served / bad argument)");
  REFUSE(err != 0, what, " failed: cudaError ", err);
}
void* ptr(const optional<Tensor>& t) { return t ? t->data_ptr() : nullptr; }
void* stream_of(const Place& at) { return c10::cuda::getCurrentCUDAStream(at.device.index()).stream(); }
PyObject* wrap(const optional<Tensor>& t) {
  if (t) return THPVariable_Wrap(*t);
  Py_RETURN_NONE;
}
void count(Py_ssize_t n, Py_ssize_t want) { REFUSE(n != want, "uq_host: ", want, " arguments"); }

// A new tensor on x's device (torch's own allocator, without the way through its dispatcher).
Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const Place& place) { return at::detail::empty_cuda(shape, type, place.device, std::nullopt); }

// Outputs of 8-bit rows of n channels: allocated, or checked.
void mx8_out(const Tensor& x, int64_t n, const Place& place, optional<Tensor>& codes, optional<Tensor>& scales) {
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  if (!codes) codes = fresh(shape, at::kFloat8_e4m3fn, place);
  else REFUSE(codes->scalar_type() != at::kFloat8_e4m3fn || codes->sizes() != at::IntArrayRef(shape) || !codes->is_contiguous() || (reinterpret_cast<uintptr_t>(codes->data_ptr()) & 7),
              "codes must be contiguous float8_e4m3fn of the rows' shape (8-byte aligned)");
  shape.back() = n / 32;
  if (!scales) scales = fresh(shape, at::kByte, place);
  else REFUSE(scales->scalar_type() != at::kByte || scales->sizes() != at::IntArrayRef(shape) || !scales->is_contiguous(), "scales must be contiguous uint8 [..., channels / 32]");
}

// plan_step(seq_lens, new_tokens, block_table, page_size, num_tokens, free_pages, slots) -> (slots, taken)
PyObject* plan_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor lens = tensor(a[0], "seq_lens");
  optional<Tensor> starts;
  ll K = 0;
  if (THPVariable_Check(a[1])) {
    starts = THPVariable_Unpack(a[1]);
  } else if (a[1] != Py_None) {
    K = PyLong_AsLongLong(a[1]);
    if (PyErr_Occurred()) return nullptr;
    REFUSE(K < 1 || K > INT32_MAX, "new_tokens: at least one per request (None: whole prompts)");
  }
  const Tensor& table = tensor(a[2], "block_table");
  const ll page = PyLong_AsLongLong(a[3]), T = PyLong_AsLongLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  optional<Tensor> free = maybe(a[5], "free_pages"), slots = maybe(a[6], "slots"), taken;
  const Place place(lens);
  place.need(starts);
  place.need(table);
  place.need(free);
  place.need(slots);
  REFUSE(lens.dim() != 1 || table.dim() != 2 || table.scalar_type() != at::kInt, "seq_lens [B], block_table int32 [>= B, max_pages]");
  const int64_t B = lens.size(0), nrows = table.size(0), pages = table.size(1);
  REFUSE(nrows < B || (table.stride(1) != 1 && pages > 1) || (table.stride(0) < pages && nrows > 1), "block_table: int32 [>= B, max_pages], its rows contiguous and apart");
  REFUSE(starts && (starts->dim() != 1 || starts->size(0) != B + 1), "new_tokens: an int, the B+1 starts, or None");
  REFUSE(B > 16384 || page < 1 || page > INT32_MAX || T < 0 || pages > INT32_MAX, "plan_step: at most 16384 requests, page_size >= 1, num_tokens >= 0");
  if (lens.scalar_type() != at::kInt || !lens.is_contiguous()) lens = lens.to(at::kInt).contiguous();
  if (starts && (starts->scalar_type() != at::kInt || !starts->is_contiguous())) starts = starts->to(at::kInt).contiguous();
  if (!slots) slots = fresh({T}, at::kLong, place);
  else REFUSE(slots->scalar_type() != at::kLong || slots->dim() != 1 || slots->size(0) != T || !slots->is_contiguous(), "slots must be contiguous int64 [num_tokens]");
  if (free) {
    REFUSE(free->scalar_type() != at::kInt || free->dim() != 1 || !free->is_contiguous(), "free_pages must be contiguous int32 [F]");
    taken = fresh({1}, at::kInt, place);
  }
  const c10::cuda::CUDAGuard on(place.device);
  done(plan_fn(static_cast<int32_t*>(lens.data_ptr()), static_cast<int32_t*>(ptr(starts)), (int)K, static_cast<int32_t*>(table.data_ptr()), std::max<ll>(table.stride(0), pages),
               free && free->numel() ? static_cast<int32_t*>(free->data_ptr()) : nullptr, free ? free->numel() : 0, static_cast<int64_t*>(slots->data_ptr()),
               static_cast<int32_t*>(ptr(taken)), (int)B, T, (int)page, (int)pages, stream_of(place)),
       "uq_plan_step_launch");
  return Py_BuildValue("(NN)", wrap(slots), wrap(taken));
  END_HANDLE_TH_ERRORS
}

// rms_norm_mx8(x, weight, residual, eps, codes, scales, sum_out) -> (codes, scales, sum)
PyObject* rms_norm_mx8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 7);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor x = tensor(a[0], "x");
  optional<Tensor> w = maybe(a[1], "weight"), r = maybe(a[2], "residual"), codes = maybe(a[4], "codes"), scales = maybe(a[5], "scales"), sum = maybe(a[6], "sum_out");
  const double eps = PyFloat_AsDouble(a[3]);
  if (PyErr_Occurred()) return nullptr;
  const Place place(x);
  for (const auto* t : {&w, &r, &codes, &scales, &sum}) place.need(*t);
  const at::ScalarType dt = x.scalar_type();
  const int64_t H = x.dim() ? x.size(-1) : 0;
  REFUSE(dtype_code(dt) < 0 || (r && r->scalar_type() != dt) || (w && w->scalar_type() != dt), "x must be fp32, bf16 or fp16; residual and weight of the same type");
  REFUSE(H < 32 || H % 32 || H > 32768, "rms_norm_mx8: a multiple of 32 channels, 32 to 32768");
  REFUSE(!(eps >= 1.1754943508222875e-38), "eps must be positive (and no subnormal)");
  REFUSE(w && (w->dim() != 1 || w->size(0) != H), "weight has x's channels, [H]");
  REFUSE(r && r->sizes() != x.sizes(), "residual has x's shape");
  REFUSE(sum && !r, "sum_out goes with a residual");
  REFUSE(sum && (sum->scalar_type() != dt || sum->sizes() != x.sizes() || !sum->is_contiguous() || (reinterpret_cast<uintptr_t>(sum->data_ptr()) & 15)),
         "sum_out must be contiguous, 16-byte aligned, of x's shape and type");
  const bool given_sum = sum.has_value();
  x = rows(x);
  if (w) w = rows(*w);
  if (r) {
    r = rows(*r);
    if (!sum) sum = fresh(x.sizes(), dt, place);
  }
  if (codes || scales || given_sum)   // (new memory is nobody else's)
    for (const auto* t : {&codes, &scales, &sum}) {
      apart(x, *t, t == &sum);
      if (r) apart(*r, *t, t == &sum);
      if (w) apart(*w, *t);
    }
  mx8_out(x, H, place, codes, scales);
  const c10::cuda::CUDAGuard on(place.device);
  done(norm_fn(x.data_ptr(), ptr(r), ptr(w), ptr(sum), static_cast<uint8_t*>(codes->data_ptr()), static_cast<uint8_t*>(scales->data_ptr()), x.numel() / H, (int)H, dtype_code(dt),
               (float)eps, stream_of(place)),
       "uq_rms_norm_mx8_launch");
  return Py_BuildValue("(NNN)", wrap(codes), wrap(scales), wrap(sum));
  END_HANDLE_TH_ERRORS
}

// silu_mul_mx8(x, codes, scales) -> (codes, scales)
PyObject* silu_mul_mx8(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 3);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor x = tensor(a[0], "x");
  optional<Tensor> codes = maybe(a[1], "codes"), scales = maybe(a[2], "scales");
  const Place place(x);
  place.need(codes);
  place.need(scales);
  REFUSE(dtype_code(x.scalar_type()) < 0, "x must be fp32, bf16 or fp16");
  const int64_t F2 = x.dim() ? x.size(-1) : 0;
  REFUSE(F2 < 64 || F2 % 64 || F2 > (1 << 21), "silu_mul_mx8: twice a multiple of 32 channels, up to 2^21 of them");
  x = rows(x);
  apart(x, codes);
  apart(x, scales);
  mx8_out(x, F2 / 2, place, codes, scales);
  const c10::cuda::CUDAGuard on(place.device);
  done(silu_fn(x.data_ptr(), static_cast<uint8_t*>(codes->data_ptr()), static_cast<uint8_t*>(scales->data_ptr()), x.numel() / F2, (int)(F2 / 2), dtype_code(x.scalar_type()),
               stream_of(place)),
       "uq_silu_mul_mx8_launch");
  return Py_BuildValue("(NN)", wrap(codes), wrap(scales));
  END_HANDLE_TH_ERRORS
}

// fp4_linear(x, wc, ws, n, scales, out, out_dtype, workspace) -> out
PyObject* fp4_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  count(nargs, 8);
  at::AutoDispatchBelowADInplaceOrView below;
  Tensor x = tensor(a[0], "x");
  const Tensor &wc = tensor(a[1], "wc"), &ws = tensor(a[2], "ws");
  optional<Tensor> scales = maybe(a[4], "scales"), out = maybe(a[5], "out"), work = maybe(a[7], "workspace");
  const Place place(x);
  place.need(wc);
  place.need(ws);
  for (const auto* t : {&scales, &out, &work}) place.need(*t);
  REFUSE(wc.dim() != 4 || wc.scalar_type() != at::kByte || ws.scalar_type() != at::kByte || !wc.is_contiguous() || !ws.is_contiguous() || wc.size(2) != 128 || wc.size(3) != 64 ||
             ws.sizes() != at::IntArrayRef({wc.size(0), wc.size(1), 128, 4}),
         "wc, ws must be contiguous uint8 [ceil(n/128), ceil(K/128), 128, 64] and [.., 4]");
  const int64_t tiles = wc.size(0), ksteps = wc.size(1), K = x.dim() ? x.size(-1) : 0;
  int64_t n = tiles * 128;
  if (a[3] != Py_None) n = PyLong_AsLongLong(a[3]);
  if (PyErr_Occurred()) return nullptr;
  REFUSE(K < 32 || K % 32 || K > (1 << 24) || (K + 127) / 128 != ksteps || n < 1 || n > (1 << 24) || (n + 127) / 128 != tiles, "x has ", K, " channels and y ", n, ": not those of a weight of ", tiles,
         " x ", ksteps, " tiles (K a multiple of 32)");
  at::ScalarType od = at::kBFloat16;
  if (a[6] != Py_None) {
    REFUSE(!THPDtype_Check(a[6]), "out_dtype must be a torch.dtype");
    od = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
  } else if (out) {
    od = out->scalar_type();
  }
  REFUSE(dtype_code(od) < 0, "y is bf16, fp16 or fp32");
  c10::SmallVector<int64_t, 6> shape(x.sizes().begin(), x.sizes().end());
  if (scales) {
    shape.back() = K / 32;
    REFUSE(x.scalar_type() != at::kFloat8_e4m3fn || scales->scalar_type() != at::kByte || scales->sizes() != at::IntArrayRef(shape),
           "with scales (uint8 [..., K/32]) x must be float8_e4m3fn [..., K]");
    scales = rows(*scales);
  } else {
    REFUSE(x.scalar_type() != at::kBFloat16, "x must be bf16, or float8_e4m3fn with scales");
  }
  x = rows(x);
  const ll M = x.numel() / K;
  if (!scales) {
    const int64_t need = (int64_t)scratch_fn(M, (int)K);
    if (!work && need) work = fresh({need}, at::kByte, place);
    REFUSE(work && (work->scalar_type() != at::kByte || work->numel() < need || !work->is_contiguous()), "scratch too small");
  }
  shape.back() = n;
  const bool given = out.has_value();
  if (!given) out = fresh(shape, od, place);
  else REFUSE(out->scalar_type() != od || out->sizes() != at::IntArrayRef(shape) || !out->is_contiguous(), "out must be contiguous bf16, fp16 or fp32 [..., n]");
  // (the kernels' CTAs read x until the last one is done, while others write their channels of out)
  if (given) {
    apart(x, out);
    if (scales) apart(*scales, out);
  }
  const c10::cuda::CUDAGuard on(place.device);
  done(linear_fn(x.data_ptr(), static_cast<uint8_t*>(ptr(scales)), static_cast<uint8_t*>(wc.data_ptr()), static_cast<uint8_t*>(ws.data_ptr()), out->data_ptr(),
                 scales ? nullptr : ptr(work), M, (int)n, (int)K, dtype_code(od), stream_of(place)),
       "uq_fp4_linear_launch");
  return wrap(out);
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the five entry points, and of uqb_header_id)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  count(n, 6);
  void* p[6];
  for (int i = 0; i < 6; i++) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    REFUSE(!p[i], "uq_host: an entry point is missing");
  }
  REFUSE(reinterpret_cast<decltype(&uqb_header_id)>(p[5])() != UQB_HEADER_ID, "uq_host: the library and this module are of different builds: python -m all_quant_b200.build");
  plan_fn = reinterpret_cast<decltype(plan_fn)>(p[0]);
  norm_fn = reinterpret_cast<decltype(norm_fn)>(p[1]);
  silu_fn = reinterpret_cast<decltype(silu_fn)>(p[2]);
  scratch_fn = reinterpret_cast<decltype(scratch_fn)>(p[3]);
  linear_fn = reinterpret_cast<decltype(linear_fn)>(p[4]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(plan_step), METHOD(rms_norm_mx8), METHOD(silu_mul_mx8), METHOD(fp4_linear), METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_uq_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

#ifndef UQ_TORCH_VERSION
#define UQ_TORCH_VERSION TORCH_VERSION
#endif
PyMODINIT_FUNC PyInit__uq_host() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", UQ_TORCH_VERSION) < 0) { Py_DECREF(m); return nullptr; }
  return m;
}
