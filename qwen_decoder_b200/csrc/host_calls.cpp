// The host's side of the operators in 8 bits, of the log probabilities and of tokens from the nucleus: their arguments' checks, room for their results and the call of
// their launchers, as a Python module.  Decode steps replay as graphs and prompts' are launched by prompt_exec.cu, but any other call has its checks,
// two torch.empty and some twenty arguments through ctypes: from Python 13 to 17 us where the device needs 2 to 10, so 5 to 7.
//
// The launchers are those of the kernel libraries, whose addresses ``resolve`` gives (a library is built and loaded when the first call needs
// it); refusals are raised as the package's KernelError before anything is launched.
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty_strided.h>
#include <c10/cuda/CUDAGuard.h>
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
  if (code == QD_ERR_BUILD) refuse(what, ": the kernel was built with other registers to a thread than its warps share out");
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
decltype(qd_sample_nucleus)* g_nucleus;
decltype(qd_rope_kv_write_fp8)* g_write;
decltype(qd_decode_attention_fp8)* g_decode;
decltype(qd_decode_attention_fp8_scratch)* g_decode_scratch;
decltype(qd_decode_attention_fp8_launches)* g_decode_launches;
decltype(qd_prefill_attention_fp8)* g_prefill;
decltype(qd_prefill_attention_fp8_scratch)* g_prefill_scratch;
decltype(qd_prefill_attention_fp8_launches)* g_prefill_launches;

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

// ---- a cache in 8 bits
constexpr int64_t MOST_OF_PAGE = 1 << 14;            // (heads or tokens of a page: a page's rows are counted in 32 bits)
int whole(PyObject* o, const char* what) {
  const long v = PyLong_AsLong(o);
  if (PyErr_Occurred()) throw PythonError{};
  if (v < INT32_MIN || v > INT32_MAX) refuse(what, " must fit 32 bits, got ", v);
  return (int)v;
}
// ``t`` on the device of the call, of ``dt`` and contiguous; n: numbers, or -1
void* plain(const at::Tensor& t, at::ScalarType dt, int64_t n, int device, const char* what) {
  if (t.scalar_type() != dt || !t.is_contiguous() || (n >= 0 && t.numel() != n))
    refuse(what, " must be contiguous ", toString(dt), n >= 0 ? " [" + std::to_string(n) + "]" : std::string(), ", got ", toString(t.scalar_type()), " ", sizes(t));
  void* at = address(t).at;
  if (t.get_device() != device) refuse(what, " is on another device");
  return at;
}
struct Heads { int H, G, d, ps; };
Heads heads_of(PyObject* const* a, int at_ps, const char* what) {
  const Heads h = {whole(a[0], what), whole(a[1], what), whole(a[2], what), whole(a[at_ps], what)};
  if (h.G < 1 || h.G > MOST_OF_PAGE || h.ps > MOST_OF_PAGE || h.H < 1 || h.H % h.G || h.H / h.G > 16 || (h.d != 64 && h.d != 128) || h.ps < 16 || h.ps % 16)
    refuse(what, ": up to 16 query heads to each of ", h.G, " kv heads of 64 or 128 features and pages of a multiple of 16 tokens, got ", h.H, " heads of ",
           h.d, ", pages of ", h.ps);
  return h;
}
// uint8 [pages, G ps (2 d + 2)]; how many
int64_t pages_of(const at::Tensor& p, const Heads& h, const char* what) {
  const int64_t bytes = (int64_t)h.G * h.ps * (2 * h.d + 2);
  if (p.scalar_type() != at::kByte || p.dim() != 2 || p.size(1) != bytes || p.size(0) < 1 || !p.is_contiguous())
    refuse(what, ": pages must be contiguous uint8 [n, ", bytes, "], got ", toString(p.scalar_type()), " ", sizes(p));
  if (p.size(0) > INT32_MAX / h.ps) refuse(what, ": more than 2^31 tokens of cache");
  return p.size(0);
}
// bfloat16 [T, n], rows 16 bytes apart
int64_t heads_rows(const at::Tensor& t, int64_t n, const char* what) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.size(1) != n || t.stride(1) != 1 || t.stride(0) % 8 || (t.size(0) > 1 && t.stride(0) < n) ||
      (uintptr_t)t.data_ptr() % 16 || t.size(0) > INT32_MAX)
    refuse(what, " must be bfloat16 [T, ", n, "], rows contiguous, on 16 bytes and a multiple of 16 bytes apart, got ", toString(t.scalar_type()), " ", sizes(t));
  return t.size(0);
}

// (pages, G, page_size, d): numbers [n, 2, G, page_size, d] and scales [n, G, page_size, 2]
CALL(fp8_page_views, 4)
  const char* what = "fp8_page_views";
  const at::Tensor& pages = tensor(a[0], "fp8_page_views: pages");
  const int64_t G = whole(a[1], what), ps = whole(a[2], what), d = whole(a[3], what);
  const int64_t bytes = G * ps * (2 * d + 2), n = 2 * G * ps * d;
  if (G < 1 || ps < 1 || d < 1 || G > MOST_OF_PAGE || ps > MOST_OF_PAGE || d > MOST_OF_PAGE || pages.scalar_type() != at::kByte || pages.dim() != 2 || pages.size(1) != bytes || pages.stride(1) != 1)
    refuse(what, ": pages must be uint8 [n, ", bytes, "], rows contiguous, got ", toString(pages.scalar_type()), " ", sizes(pages));
  const int64_t at = pages.storage_offset(), row = pages.stride(0);
  const at::Tensor numbers = pages.view(at::kFloat8_e4m3fn).as_strided({pages.size(0), 2, G, ps, d}, {row, n / 2, ps * d, d, 1}, at);
  const at::Tensor scales = pages.view(at::kFloat8_e8m0fnu).as_strided({pages.size(0), G, ps, 2}, {row, 2 * ps, 2, 1}, at + n);
  PyObject* out = PyTuple_New(2);
  if (!out) throw PythonError{};
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(numbers));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(scales));
  return out;
END

// (qkv, bias, q_out, H, G, d, rotary_dim, pairing, cos, sin, positions, pages, slot_map, page_size, write_kv)
CALL(rope_kv_write_fp8, 15)
  const char* what = "rope_kv_write_fp8";
  const at::Tensor &x = tensor(a[0], "rope_kv_write_fp8: qkv"), &q = tensor(a[2], "rope_kv_write_fp8: q_out"), &pos = tensor(a[10], "rope_kv_write_fp8: positions");
  const at::Tensor *bias = tensor_or_none(a[1], "rope_kv_write_fp8: bias"), *cos = tensor_or_none(a[8], "rope_kv_write_fp8: cos");
  const at::Tensor *sin = tensor_or_none(a[9], "rope_kv_write_fp8: sin"), *pages = tensor_or_none(a[11], "rope_kv_write_fp8: pages");
  const at::Tensor* slots = tensor_or_none(a[12], "rope_kv_write_fp8: slot_map");
  const Heads h = heads_of(a + 3, 10, what);
  const int rot = whole(a[6], what), half = whole(a[7], what), write = PyObject_IsTrue(a[14]);
  if (PyErr_Occurred()) throw PythonError{};
  const int64_t W = (int64_t)(h.H + 2 * h.G) * h.d, T = heads_rows(q, (int64_t)h.H * h.d, "rope_kv_write_fp8: q_out");
  if (!q.is_contiguous()) refuse(what, ": q_out must be contiguous");
  const Source f = source_of(x, "rope_kv_write_fp8: qkv", T, W);
  if (!x.is_contiguous()) refuse(what, ": qkv must be contiguous");
  vector_of(bias, W, what, "bias");
  if (half != 0 && half != 1) refuse(what, ": pairing must be 0 (neighbours) or 1 (halves), got ", half);
  if (rot < 0 || rot > h.d || rot % (half ? 16 : 8)) refuse(what, ": rotary_dim must be a multiple of ", half ? 16 : 8, " up to ", h.d, ", got ", rot);
  const at::Tensor* same[] = {bias, cos, sin, pages, slots};
  const int device = x.is_cuda() ? x.get_device() : -1;
  int64_t n_pos = 0, n_pages = 0;
  if (rot) {
    if (!cos || !sin || cos->dim() != 2 || cos->size(1) != rot / 2 || cos->size(0) < 1 || cos->sizes() != sin->sizes() || cos->size(0) > INT32_MAX)
      refuse(what, ": cos and sin must be float32 [positions, ", rot / 2, "]");
    n_pos = cos->size(0);
    for (const at::Tensor* t : {cos, sin})
      if (t->scalar_type() != at::kFloat || !t->is_contiguous()) refuse(what, ": cos and sin must be contiguous float32");
  }
  if (write) {
    if (!pages || !slots) refuse(what, ": pages and slot_map are needed to write");
    n_pages = pages_of(*pages, h, what);
  }
  void* x_at = address(x).at;
  for (const at::Tensor* t : same)
    if (t && (!t->is_cuda() || t->get_device() != device)) refuse(what, ": a tensor is on another device");
  if (T == 0) Py_RETURN_NONE;
  void *q_at = plain(q, at::kBFloat16, -1, device, "rope_kv_write_fp8: q_out"), *pos_at = plain(pos, at::kInt, T, device, "rope_kv_write_fp8: positions");
  void* slots_at = write ? plain(*slots, at::kInt, T, device, "rope_kv_write_fp8: slot_map") : nullptr;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  done(entry(g_write, "cache_fp8", "qd_rope_kv_write_fp8")(x_at, f.code, f.ld, f.parts, f.step, address(bias), q_at, (int)T, h.H, h.G, h.d, rot, half,
                                                          rot ? address(cos) : Address{nullptr}, rot ? address(sin) : Address{nullptr}, (int)n_pos,
                                                          (const int*)pos_at, write ? address(pages) : Address{nullptr}, n_pages, (const int*)slots_at, h.ps, write,
                                                          multiprocessors(device), stream_of(x)), what);
  Py_RETURN_NONE;
END

// (q, out, pages, block_table, token_req, positions, H, G, d, page_size, scale, window, max_keys) -> kernels launched
CALL(decode_attention_fp8, 13)
  const char* what = "decode_attention_fp8";
  const at::Tensor &q = tensor(a[0], "decode_attention_fp8: q"), &out = tensor(a[1], "decode_attention_fp8: out"), &pages = tensor(a[2], "decode_attention_fp8: pages");
  const at::Tensor &table = tensor(a[3], "decode_attention_fp8: block_table"), &req = tensor(a[4], "decode_attention_fp8: token_req");
  const at::Tensor& pos = tensor(a[5], "decode_attention_fp8: positions");
  const Heads h = heads_of(a + 6, 3, what);
  const double scale = PyFloat_AsDouble(a[10]);
  const int window = whole(a[11], what);
  int64_t max_keys = a[12] == Py_None ? -1 : PyLong_AsLongLong(a[12]);
  if (PyErr_Occurred()) throw PythonError{};
  const int64_t T = heads_rows(q, (int64_t)h.H * h.d, "decode_attention_fp8: q"), n_pages = pages_of(pages, h, what);
  if (heads_rows(out, (int64_t)h.H * h.d, "decode_attention_fp8: out") != T) refuse(what, ": q and out have ", T, " and ", out.size(0), " rows");
  if (table.dim() != 2 || table.size(0) < 1 || table.size(1) < 1) refuse(what, ": block_table must be int32 [requests, pages], got ", sizes(table));
  if (window < 0) refuse(what, ": window must not be negative");
  const int64_t held = table.size(1) * h.ps;
  if (max_keys < 0 || max_keys > held) max_keys = held;
  if (max_keys > INT32_MAX) refuse(what, ": more than 2^31 keys");
  address(q);
  const int device = q.get_device();
  if (!out.is_cuda() || out.get_device() != device) refuse(what, ": out is on another device");
  void *pages_at = plain(pages, at::kByte, -1, device, "decode_attention_fp8: pages"), *table_at = plain(table, at::kInt, -1, device, "decode_attention_fp8: block_table");
  void *req_at = plain(req, at::kInt, T, device, "decode_attention_fp8: token_req"), *pos_at = plain(pos, at::kInt, T, device, "decode_attention_fp8: positions");
  if (T == 0) return PyLong_FromLong(0);
  if (max_keys == 0) max_keys = 1;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const int sms = multiprocessors(device);
  const int64_t floats = entry(g_decode_scratch, "attention_fp8_decode", "qd_decode_attention_fp8_scratch")((int)T, h.H, h.G, h.d, window, (int)max_keys, sms);
  const at::Tensor scratch = at::empty_strided({floats}, {1}, q.options().dtype(at::kFloat));
  done(entry(g_decode, "attention_fp8_decode", "qd_decode_attention_fp8")(address(q), q.stride(0), address(out), out.stride(0), pages_at, n_pages,
                                                                         (const int*)table_at, (int)table.size(1), (int)table.size(0), (const int*)req_at,
                                                                         (const int*)pos_at, (int)T, h.H, h.G, h.d, h.ps, (float)scale, window, (int)max_keys,
                                                                         address(scratch), sms, stream_of(q)), what);
  return PyLong_FromLong(entry(g_decode_launches, "attention_fp8_decode", "qd_decode_attention_fp8_launches")((int)T, h.H, h.G, window, (int)max_keys, sms));
END

// (q, out, pages, block_table, cu_tokens, start_pos, H, G, d, page_size, scale, window, max_keys, n_tokens) -> kernels launched
CALL(prefill_attention_fp8, 14)
  const char* what = "prefill_attention_fp8";
  const at::Tensor &q = tensor(a[0], "prefill_attention_fp8: q"), &out = tensor(a[1], "prefill_attention_fp8: out"), &pages = tensor(a[2], "prefill_attention_fp8: pages");
  const at::Tensor &table = tensor(a[3], "prefill_attention_fp8: block_table"), &cu = tensor(a[4], "prefill_attention_fp8: cu_tokens");
  const at::Tensor& start = tensor(a[5], "prefill_attention_fp8: start_pos");
  const Heads h = heads_of(a + 6, 3, what);
  const double scale = PyFloat_AsDouble(a[10]);
  const int window = whole(a[11], what);
  int64_t max_keys = a[12] == Py_None ? -1 : PyLong_AsLongLong(a[12]), T = a[13] == Py_None ? -1 : PyLong_AsLongLong(a[13]);
  if (PyErr_Occurred()) throw PythonError{};
  const int64_t rows = heads_rows(q, (int64_t)h.H * h.d, "prefill_attention_fp8: q"), n_pages = pages_of(pages, h, what);
  if (heads_rows(out, (int64_t)h.H * h.d, "prefill_attention_fp8: out") != rows) refuse(what, ": q and out have ", rows, " and ", out.size(0), " rows");
  if (table.dim() != 2 || table.size(1) < 1) refuse(what, ": block_table must be int32 [requests, pages], got ", sizes(table));
  const int64_t R = table.size(0);
  if (T > rows) refuse(what, ": ", T, " tokens in ", rows, " rows");
  if (T < 0) T = rows;
  if (window < 0) refuse(what, ": window must not be negative");
  const int64_t held = table.size(1) * h.ps;
  if (max_keys < 0 || max_keys > held) max_keys = held;
  if (max_keys > INT32_MAX || R > INT32_MAX - rows) refuse(what, ": more than 2^31 keys or requests");
  address(q);
  const int device = q.get_device();
  if (!out.is_cuda() || out.get_device() != device) refuse(what, ": out is on another device");
  void *pages_at = plain(pages, at::kByte, -1, device, "prefill_attention_fp8: pages"), *table_at = plain(table, at::kInt, -1, device, "prefill_attention_fp8: block_table");
  void *cu_at = plain(cu, at::kInt, R + 1, device, "prefill_attention_fp8: cu_tokens"), *start_at = plain(start, at::kInt, R, device, "prefill_attention_fp8: start_pos");
  if (T == 0 || R == 0) return PyLong_FromLong(0);
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  const int sms = multiprocessors(device);
  const int64_t floats = entry(g_prefill_scratch, "attention_fp8_chunk", "qd_prefill_attention_fp8_scratch")((int)T, (int)R, h.H, h.G, h.d, window,
                                                                                                         (int)max_keys, sms);
  const at::Tensor scratch = at::empty_strided({floats}, {1}, q.options().dtype(at::kFloat));
  done(entry(g_prefill, "attention_fp8_chunk", "qd_prefill_attention_fp8")(address(q), q.stride(0), address(out), out.stride(0), pages_at, n_pages,
                                                                          (const int*)table_at, (int)table.size(1), (const int*)cu_at, (const int*)start_at,
                                                                          (int)R, (int)T, (int)rows, h.H, h.G, h.d, h.ps, (float)scale, window, (int)max_keys,
                                                                          address(scratch), sms, stream_of(q)), what);
  return PyLong_FromLong(entry(g_prefill_launches, "attention_fp8_chunk", "qd_prefill_attention_fp8_launches")((int)T, (int)R, h.H, h.G, window, (int)max_keys, sms));
END

// (logits, temperature, top_k, top_p, min_p, draws, out, only)
CALL(sample_nucleus, 8)
  const char* what = "sample_nucleus";
  const at::Tensor &z = tensor(a[0], "sample_nucleus: logits"), &temperature = tensor(a[1], "sample_nucleus: temperature"), &k = tensor(a[2], "sample_nucleus: top_k");
  const at::Tensor &p = tensor(a[3], "sample_nucleus: top_p"), &m = tensor(a[4], "sample_nucleus: min_p"), &u = tensor(a[5], "sample_nucleus: draws");
  const at::Tensor& out = tensor(a[6], "sample_nucleus: out");
  const int only = PyObject_IsTrue(a[7]);
  if (PyErr_Occurred()) throw PythonError{};
  if (z.scalar_type() != at::kFloat || z.dim() != 2 || (z.stride(1) != 1 && z.size(1) > 1)) refuse("sample_nucleus: logits must be float32 [R, V] with contiguous rows");
  const int64_t R = z.size(0), V = z.size(1);
  if (V < 1 || V > QD_NUCLEUS_MAX_VOCABULARY) refuse(what, ": rows of 1 to ", QD_NUCLEUS_MAX_VOCABULARY, " logits, got ", V);
  if (R > INT32_MAX / 16) refuse(what, ": ", R, " rows");
  for (const auto& [t, name, dt] : {std::make_tuple(&temperature, "temperature", at::kFloat), std::make_tuple(&k, "top_k", at::kInt), std::make_tuple(&p, "top_p", at::kFloat),
                                    std::make_tuple(&m, "min_p", at::kFloat), std::make_tuple(&u, "draws", at::kFloat), std::make_tuple(&out, "out", at::kInt)})
    if (t->scalar_type() != dt || t->dim() != 1 || t->size(0) != R || !t->is_contiguous()) refuse(what, ": ", name, " must be contiguous ", toString(dt), " [", R, "]");
  address(z);
  const int device = z.get_device();
  for (const at::Tensor* t : {&temperature, &k, &p, &m, &u, &out})
    if (!t->is_cuda() || t->get_device() != device) refuse(what, ": a tensor is on another device");
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  done(entry(g_nucleus, "sampling_nucleus", "qd_sample_nucleus")(address(z), z.stride(0), (int)R, (int)V, address(temperature), address(k), address(p), address(m),
                                                                 address(u), address(out), only, multiprocessors(device), stream_of(z)), what);
  Py_RETURN_NONE;
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
                         ENTRY(gemm_fp8_gated), ENTRY(gemm_fp8_plan), ENTRY(token_logprobs), ENTRY(fp8_page_views), ENTRY(rope_kv_write_fp8),
                         ENTRY(decode_attention_fp8), ENTRY(prefill_attention_fp8), ENTRY(sample_nucleus), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "qd_host_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_qd_host_calls() { return PyModule_Create(&module); }
