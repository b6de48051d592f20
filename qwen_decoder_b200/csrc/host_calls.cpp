// The host's side of the operators in 8 bits and of the log probabilities: their arguments' checks, room for their results and the call of
// their launchers, as a Python module.  Decode steps replay as graphs and prompts' are launched by prompt_exec.cu, but any other call has its checks,
// two torch.empty and some twenty arguments through ctypes: from Python 13 to 17 us where the device needs 2 to 10, so 5 to 7.
//
// The launchers are those of the kernel libraries, whose addresses ``resolve`` gives (a library is built and loaded when the first call needs
// it); refusals are raised as the package's KernelError before anything is launched.
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Device.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "entry_points.h"

#include <map>
#include <sstream>
#include <string>
#include <tuple>

namespace {

constexpr int F32 = QD_F32, BF16 = QD_BF16, BLOCK = QD_FP8_BLOCK, STORE = QD_FP8_STORE, GATED = QD_FP8_GATED, ACT_SILU = QD_ACT_SILU;
constexpr int ACT_GELU = QD_ACT_GELU_TANH, FEW_TOKENS = QD_FP8_FEW_TOKENS, MOST_TOP = QD_LOGPROBS_MAX_TOP;
constexpr int64_t MOST_VOCABULARY = QD_LOGPROBS_MAX_VOCABULARY;

PyObject *g_error, *g_resolve, *g_rows_type;        // KernelError; (library, function) -> address, ("sms", device) -> multiprocessors; Fp8Rows

struct Refused { std::string what; };
template <typename... A>
[[noreturn]] void refuse(A&&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused{s.str()};
}
struct PythonError {};

// a launcher by its library and name, or a number by "sms" and the device
uintptr_t resolve(const char* library, const char* function) {
  PyObject* got = PyObject_CallFunction(g_resolve, "ss", library, function);
  if (!got) throw PythonError{};
  const uintptr_t v = (uintptr_t)PyLong_AsUnsignedLongLong(got);
  Py_DECREF(got);
  if (PyErr_Occurred()) throw PythonError{};
  return v;
}
template <typename F>
F* entry(F*& kept, const char* library, const char* function) {
  if (!kept) kept = reinterpret_cast<F*>(resolve(library, function));
  return kept;
}
int multiprocessors(int device) {
  static int kept[64];
  if (device < 0 || device >= 64) refuse("device ", device);
  if (!kept[device]) kept[device] = (int)resolve("sms", std::to_string(device).c_str());
  return kept[device];
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(what, " must be a tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor* tensor_or_none(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }
// of whatever a launcher takes there
struct Address {
  void* at;
  template <typename T>
  operator T*() const { return static_cast<T*>(at); }
};
Address address(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("kernel argument is not on a CUDA device (there is no CPU path)");
  return {t.data_ptr()};
}
Address address(const at::Tensor* t) { return t ? address(*t) : Address{nullptr}; }
std::string sizes(const at::Tensor& t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}
void done(int code, const char* what) {
  if (code == 0) return;
  if (code == QD_ERR_UNSUPPORTED) refuse(what, ": the kernel refuses these sizes or types");
  refuse(what, ": CUDA error ", code);
}

// ---- rows in 8 bits
struct Rows {
  const at::Tensor *q, *s;
  int64_t R, K, ldq, lds;
  void *q_at, *s_at;
};
Rows rows_of(PyObject* o, const char* name, int64_t R = -1, int64_t K = -1) {
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) refuse(name, ": rows in 8 bits are a pair of q and s");
  Rows r;
  const at::Tensor &q = tensor(PyTuple_GET_ITEM(o, 0), name), &s = tensor(PyTuple_GET_ITEM(o, 1), name);
  if (q.scalar_type() != at::kFloat8_e4m3fn || s.scalar_type() != at::kFloat8_e8m0fnu || q.dim() != 2 || s.dim() != 2)
    refuse(name, ": rows in 8 bits are q float8_e4m3fn [R, K] and s float8_e8m0fnu [R, ceil(K / 128)]");
  r.q = &q; r.s = &s; r.R = q.size(0); r.K = q.size(1); r.ldq = q.stride(0); r.lds = s.stride(0);
  const int64_t kb = (r.K + BLOCK - 1) / BLOCK;
  if ((R >= 0 && r.R != R) || (K >= 0 && r.K != K) || s.size(0) != r.R || s.size(1) != kb)
    refuse(name, ": q ", sizes(q), " and s ", sizes(s), " do not fit ", R < 0 ? "any" : std::to_string(R), " rows of ", K < 0 ? "any" : std::to_string(K),
           " features");
  r.q_at = q.data_ptr(); r.s_at = s.data_ptr();
  if (r.R == 1) {                                    // (one row is nowhere from the next)
    r.ldq = (r.K + 15) / 16 * 16;
    r.lds = (kb + 3) / 4 * 4;
  }
  if (r.R && r.K) {
    if ((q.stride(1) != 1 && r.K > 1) || r.ldq % 16 || r.ldq < r.K || (uintptr_t)r.q_at % 16)
      refuse(name, ": rows of q must be contiguous, on 16 bytes and a multiple of 16 bytes apart");
    if ((s.stride(1) != 1 && kb > 1) || r.lds % 4 || r.lds < kb || (uintptr_t)r.s_at % 4)
      refuse(name, ": rows of s must be contiguous, on 4 bytes and a multiple of 4 bytes apart");
  }
  if (r.R > INT32_MAX || r.K > INT32_MAX) refuse(name, ": more than 2^31 rows or features");
  return r;
}
void on_device(const Rows& r) {
  address(*r.q);
  address(*r.s);
}
// bfloat16 or float32 [T, K], or float32 parts [n, T, K]
struct Source { int code, parts; int64_t ld, step; };
Source source_of(const at::Tensor& x, const char* name, int64_t T, int64_t K) {
  const auto dt = x.scalar_type();
  const int64_t d = x.dim();
  if ((dt != at::kFloat && dt != at::kBFloat16) || (d != 2 && d != 3) || (d == 3 && (dt != at::kFloat || !x.size(0) || x.size(0) > INT32_MAX)) ||
      x.size(d - 2) != T || x.size(d - 1) != K)
    refuse(name, ": bfloat16 or float32 [", T, ", ", K, "], or float32 parts [n, ", T, ", ", K, "] expected, got ", toString(dt), " ", sizes(x));
  if (x.stride(d - 1) != 1 && K > 1) refuse(name, ": rows must be contiguous");
  return {dt == at::kFloat ? F32 : BF16, d == 3 ? (int)x.size(0) : 1, x.stride(d - 2), d == 3 ? x.stride(0) : 0};
}
void vector_of(const at::Tensor* v, int64_t n, const char* what, const char* name) {
  if (v && (v->scalar_type() != at::kFloat || v->numel() != n || !v->is_contiguous())) refuse(what, ": ", name, " must be contiguous float32 [", n, "]");
}
int act_of(PyObject* o, const char* what) {
  const long act = PyLong_AsLong(o);
  if (PyErr_Occurred()) throw PythonError{};
  if (act != ACT_SILU && act != ACT_GELU) refuse(what, ": act must be ACT_SILU or ACT_GATED_GELU, got ", act);
  return (int)act;
}
cudaStream_t stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// ---- the launchers
decltype(qd_rows_fp8)* g_rows;
decltype(qd_add_rmsnorm_fp8)* g_norm;
decltype(qd_gemm_fp8_plan)* g_plan;
decltype(qd_gemm_fp8)* g_product;
decltype(qd_gemm_fp8_few)* g_few;
decltype(qd_gemm_fp8_few_wanted)* g_few_wanted;
decltype(qd_token_logprobs)* g_logprobs;

struct Plan { int cg, bn, splits; };
// (kept by sizes and device: a few microseconds of estimates)
Plan plan_of(int T, int N, int K, int epi, int code, int device) {
  static std::map<std::tuple<int, int, int, int, int, int>, Plan> kept;
  const auto key = std::make_tuple(T, N, K, epi & 255, code, device);
  const auto at = kept.find(key);
  if (at != kept.end()) return at->second;
  Plan p;
  if (!entry(g_plan, "gemm_fp8", "qd_gemm_fp8_plan")(T, N, K, epi, code, multiprocessors(device), &p.cg, &p.bn, &p.splits))
    refuse("gemm_fp8: no product of ", T, " x ", K, " by ", N, " x ", K);
  if (kept.size() >= 4096) kept.clear();
  return kept[key] = p;
}
// (no kernel is asked for sizes that it does not take)
bool few_wanted(int64_t T, int64_t N, int64_t K, int sms) {
  return T <= FEW_TOKENS && entry(g_few_wanted, "gemm_fp8_few", "qd_gemm_fp8_few_wanted")((int)T, (int)N, (int)K, sms);
}

void product(const Rows& x, const Rows& w, const at::Tensor* bias, void* out, int code, int64_t ldo, void* s_out, int64_t lds_out, int epi, PyObject* plan,
             PyObject* resident_o, const char* what) {
  const int resident = PyObject_IsTrue(resident_o);
  if (resident < 0) throw PythonError{};
  const int T = (int)x.R, N = (int)w.R, K = (int)x.K;
  on_device(x);
  on_device(w);
  if (T == 0 || N == 0) return;
  const cudaStream_t stream = stream_of(*x.q);
  const int sms = multiprocessors(x.q->get_device());
  Plan p = {0, 0, 0};
  bool few = false;
  if (plan == Py_None) {
    few = (epi & 255) == STORE && few_wanted(T, N, K, sms);
    if (!few) p = plan_of(T, N, K, epi, code, x.q->get_device());
  } else {
    if (!PyTuple_Check(plan) || !PyArg_ParseTuple(plan, "iii", &p.cg, &p.bn, &p.splits)) {
      PyErr_Clear();
      refuse(what, ": plan must be a tuple of three whole numbers or None");
    }
    few = p.cg == 0 && (epi & 255) == STORE;
  }
  if (few)
    done(entry(g_few, "gemm_fp8_few", "qd_gemm_fp8_few")(w.q_at, w.ldq, w.s_at, w.lds, x.q_at, x.ldq, x.s_at, x.lds, address(bias), out, code, ldo, T, N, K,
                                                        resident, sms, stream), what);
  else
    done(entry(g_product, "gemm_fp8", "qd_gemm_fp8")(w.q_at, w.ldq, w.s_at, w.lds, x.q_at, x.ldq, x.s_at, x.lds, address(bias), out, code, ldo, s_out, lds_out,
                                                    T, N, K, p.cg, p.bn, p.splits, epi, resident, sms, stream), what);
}

// ---- the module's functions
template <typename F>
PyObject* guarded(F&& f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(g_error, r.what.c_str());
    return nullptr;
  } catch (const PythonError&) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}
#define CALL(name, n) PyObject* name(PyObject*, PyObject* const* a, Py_ssize_t given) {                                     \
    if (given != n) { PyErr_SetString(PyExc_TypeError, #name ": " #n " arguments"); return nullptr; }                        \
    return guarded([&]() -> PyObject* {
#define END }); }

// (rows, features, device) -> Fp8Rows
CALL(fp8_rows, 3)
  const int64_t R = PyLong_AsLongLong(a[0]), K = PyLong_AsLongLong(a[1]), kb = (K + BLOCK - 1) / BLOCK;
  if (PyErr_Occurred()) throw PythonError{};
  if (R < 0 || K < 0 || !THPDevice_Check(a[2])) refuse("fp8_rows: ", R, " rows of ", K, " features");
  const auto options = at::TensorOptions().device(reinterpret_cast<THPDevice*>(a[2])->device);
  PyObject* q = THPVariable_Wrap(at::empty_strided({R, K}, {(K + 15) / 16 * 16, 1}, options.dtype(at::kFloat8_e4m3fn)));
  PyObject* s = THPVariable_Wrap(at::empty_strided({R, kb}, {(kb + 3) / 4 * 4, 1}, options.dtype(at::kFloat8_e8m0fnu)));
  PyObject* both[2] = {q, s};
  PyObject* rows = PyObject_Vectorcall(g_rows_type, both, 2, nullptr);
  Py_DECREF(q);
  Py_DECREF(s);
  return rows;
END

// (rows) -> (R, K)
CALL(check_rows, 2)
  const Rows r = rows_of(a[0], PyUnicode_AsUTF8(a[1]));
  return Py_BuildValue("LL", (long long)r.R, (long long)r.K);
END

// (x, out)
CALL(quantize_fp8, 2)
  const Rows r = rows_of(a[1], "quantize_fp8: out");
  const at::Tensor& x = tensor(a[0], "quantize_fp8: x");
  const Source f = source_of(x, "quantize_fp8: x", r.R, r.K);
  on_device(r);
  done(entry(g_rows, "rows_fp8", "qd_rows_fp8")(address(x), f.code, f.ld, f.parts, f.step, 0, 0, nullptr, r.q_at, r.ldq, r.s_at, r.lds, (int)r.R, (int)r.K,
                                               stream_of(x)), "quantize_fp8");
  Py_RETURN_NONE;
END

// (gate_up, out, bias, act)
CALL(gate_fp8, 4)
  const Rows r = rows_of(a[1], "gate_fp8: out");
  const at::Tensor& x = tensor(a[0], "gate_fp8: gate_up");
  const Source f = source_of(x, "gate_fp8: gate_up", r.R, 2 * r.K);
  const at::Tensor* bias = tensor_or_none(a[2], "gate_fp8: bias");
  vector_of(bias, 2 * r.K, "gate_fp8", "bias");
  const int act = act_of(a[3], "gate_fp8");
  on_device(r);
  done(entry(g_rows, "rows_fp8", "qd_rows_fp8")(address(x), f.code, f.ld, f.parts, f.step, 1, act, address(bias), r.q_at, r.ldq, r.s_at, r.lds, (int)r.R,
                                               (int)r.K, stream_of(x)), "gate_fp8");
  Py_RETURN_NONE;
END

// (x, delta, weight, out, eps, rows, write_back, delta_scale)
CALL(add_rmsnorm_fp8, 8)
  const Rows r = rows_of(a[3], "add_rmsnorm_fp8: out");
  const at::Tensor &x = tensor(a[0], "add_rmsnorm_fp8: x"), &weight = tensor(a[2], "add_rmsnorm_fp8: weight");
  const at::Tensor *delta = tensor_or_none(a[1], "add_rmsnorm_fp8: delta"), *rows = tensor_or_none(a[5], "add_rmsnorm_fp8: rows");
  const at::Tensor* scale = tensor_or_none(a[7], "add_rmsnorm_fp8: delta_scale");
  const double eps = PyFloat_AsDouble(a[4]);
  const int write_back = PyObject_IsTrue(a[6]);
  if (PyErr_Occurred()) throw PythonError{};
  if (x.scalar_type() != at::kFloat || x.dim() != 2 || x.size(1) != r.K || !x.is_contiguous())
    refuse("add_rmsnorm_fp8: x must be contiguous float32 [T, ", r.K, "]");
  const int64_t T = x.size(0);
  vector_of(&weight, r.K, "add_rmsnorm_fp8", "weight");
  vector_of(scale, r.K, "add_rmsnorm_fp8", "delta_scale");
  if (rows ? rows->scalar_type() != at::kInt || rows->numel() != r.R || !rows->is_contiguous() : r.R != T)
    refuse("add_rmsnorm_fp8: out has a row for every row of x, or for every one of rows (contiguous int32)");
  Source f = {F32, 1, 0, 0};
  if (delta) {
    f = source_of(*delta, "add_rmsnorm_fp8: delta", T, r.K);
    if (!delta->is_contiguous()) refuse("add_rmsnorm_fp8: delta must be contiguous");
  }
  on_device(r);
  done(entry(g_norm, "rows_fp8", "qd_add_rmsnorm_fp8")(address(x), address(delta), f.code, address(scale), address(weight), r.q_at, r.ldq, r.s_at, r.lds,
                                                      address(rows), (int)r.R, (int)r.K, (float)eps, write_back, f.parts, T * r.K, stream_of(x)),
       "add_rmsnorm_fp8");
  Py_RETURN_NONE;
END

// (x, w, bias, out, plan, resident)
CALL(gemm_fp8, 6)
  const Rows x = rows_of(a[0], "gemm_fp8: x"), w = rows_of(a[1], "gemm_fp8: w", -1, x.K);
  const at::Tensor& out = tensor(a[3], "gemm_fp8: out");
  const at::Tensor* bias = tensor_or_none(a[2], "gemm_fp8: bias");
  const auto dt = out.scalar_type();
  if ((dt != at::kFloat && dt != at::kBFloat16) || out.dim() != 2 || out.size(0) != x.R || out.size(1) != w.R || (out.stride(1) != 1 && w.R > 1))
    refuse("gemm_fp8: out must be bfloat16 or float32 [", x.R, ", ", w.R, "] with contiguous rows");
  vector_of(bias, w.R, "gemm_fp8", "bias");
  on_device(x);
  product(x, w, bias, address(out), dt == at::kFloat ? F32 : BF16, out.stride(0), nullptr, 0, STORE, a[4], a[5], "gemm_fp8");
  Py_RETURN_NONE;
END

// (x, w, bias, out, act, plan, resident)
CALL(gemm_fp8_gated, 7)
  const Rows x = rows_of(a[0], "gemm_fp8_gated: x"), w = rows_of(a[1], "gemm_fp8_gated: w", -1, x.K);
  if (w.R % 2) refuse("gemm_fp8_gated: w holds as many rows of up as of the gate");
  const Rows out = rows_of(a[3], "gemm_fp8_gated: out", x.R, w.R / 2);
  const at::Tensor* bias = tensor_or_none(a[2], "gemm_fp8_gated: bias");
  vector_of(bias, w.R, "gemm_fp8_gated", "bias");
  const int act = act_of(a[4], "gemm_fp8_gated");
  on_device(out);
  product(x, w, bias, out.q_at, BF16, out.ldq, out.s_at, out.lds, GATED + 256 * act, a[5], a[6], "gemm_fp8_gated");
  Py_RETURN_NONE;
END

// (T, N, K, gated, float32, device) -> (CTAs to a tile of tokens, rows of w to a tile, shares of K), three zeros: the few-token kernel
CALL(gemm_fp8_plan, 6)
  const long T = PyLong_AsLong(a[0]), N = PyLong_AsLong(a[1]), K = PyLong_AsLong(a[2]);
  const int gated = PyObject_IsTrue(a[3]), f32 = PyObject_IsTrue(a[4]), device = (int)PyLong_AsLong(a[5]);
  if (PyErr_Occurred()) throw PythonError{};
  if (T < 1 || N < 1 || K < 1 || T > INT32_MAX || N > INT32_MAX || K > INT32_MAX) refuse("gemm_fp8_plan: no product of ", T, " x ", K, " by ", N, " x ", K);
  Plan p = {0, 0, 0};
  const int sms = multiprocessors(device);
  if (gated || !few_wanted(T, N, K, sms)) p = plan_of((int)T, (int)N, (int)K, gated ? GATED : STORE, f32 ? F32 : BF16, device);
  return Py_BuildValue("iii", p.cg, p.bn, p.splits);
END

// (logits, tokens, top) -> (logprob, entropy, ids, logprobs of the ids)
CALL(token_logprobs, 3)
  const at::Tensor &z = tensor(a[0], "token_logprobs: logits"), &tokens = tensor(a[1], "token_logprobs: tokens");
  const int64_t top = PyLong_AsLongLong(a[2]);
  if (PyErr_Occurred()) throw PythonError{};
  const auto dt = z.scalar_type();
  if ((dt != at::kFloat && dt != at::kBFloat16) || z.dim() != 2 || (z.stride(1) != 1 && z.size(1) > 1))
    refuse("token_logprobs: logits must be float32 or bfloat16 [R, V] with contiguous rows");
  const int64_t R = z.size(0), V = z.size(1);
  if (tokens.scalar_type() != at::kInt || tokens.dim() != 1 || tokens.size(0) != R || !tokens.is_contiguous())
    refuse("token_logprobs: tokens must be contiguous int32 [", R, "]");
  if (V > MOST_VOCABULARY) refuse("token_logprobs: rows of at most ", MOST_VOCABULARY, " logits, got ", V);
  const int64_t most = std::min<int64_t>(MOST_TOP, V);
  if (V < 1 || top < 0 || top > most) refuse("token_logprobs: top must be between 0 and ", most, ", got ", top);
  if (R > INT32_MAX / 16) refuse("token_logprobs: ", R, " rows");
  const Address z_at = address(z), t_at = address(tokens);
  const auto options = z.options();
  const auto f32 = options.dtype(at::kFloat), i32 = options.dtype(at::kInt);
  at::Tensor lp = at::empty_strided({R}, {1}, f32), entropy = at::empty_strided({R}, {1}, f32);
  at::Tensor ids = at::empty_strided({R, top}, {top, 1}, i32), lps = at::empty_strided({R, top}, {top, 1}, f32);
  done(entry(g_logprobs, "logprobs", "qd_token_logprobs")(z_at, dt == at::kFloat ? F32 : BF16, z.stride(0), t_at, address(lp), address(entropy),
                                                         address(ids), address(lps), (int)R, (int)V, (int)top, multiprocessors(z.get_device()),
                                                         stream_of(z)), "token_logprobs");
  PyObject* out = PyTuple_New(4);
  if (!out) throw PythonError{};
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(lp));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(entropy));
  PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(ids));
  PyTuple_SET_ITEM(out, 3, THPVariable_Wrap(lps));
  return out;
END

// (KernelError, resolve, Fp8Rows)
CALL(start, 3)
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  Py_INCREF(a[2]);
  g_error = a[0];
  g_resolve = a[1];
  g_rows_type = a[2];
  Py_RETURN_NONE;
END

#define ENTRY(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(start), ENTRY(fp8_rows), ENTRY(check_rows), ENTRY(quantize_fp8), ENTRY(gate_fp8), ENTRY(add_rmsnorm_fp8), ENTRY(gemm_fp8),
                         ENTRY(gemm_fp8_gated), ENTRY(gemm_fp8_plan), ENTRY(token_logprobs), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "qd_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_qd_host_calls() { return PyModule_Create(&module); }
