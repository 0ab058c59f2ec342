// Host side of the block operators' calls: checks, output tensors and the launch in one native call.
//
// A call of these operators on small inputs (one token, one decode batch) costs the host several times what it costs the GPU;
// checks and ctypes in Python are most of it (measured on the B200 host, us a call: step 16 -> 8, block norm 17 -> 8, an activation
// to eight bits and back 21 -> 11; a block norm with its backward pass 200 -> 170, the rest of it autograd's own).
// Each function here serves a call on dense operands and returns None for every other one (a CPU tensor, mixed dtypes, a gradient to
// record, operands that would have to be copied, and views: the LinearAttention layer's column ranges of one projection among them);
// the Python operator then takes its own way, which serves the call or refuses it by name.  The kernels and the C-ABI entry points are the same on both ways; this file holds no arithmetic.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>
#include <initializer_list>

#include "../../include/orbit_b200.h"

namespace {

// entry points of liborbit_b200.so, handed over as addresses (the library is loaded once, by ctypes)
struct Entry {
  decltype(&orbit_la_step) la_step;
  decltype(&orbit_la_fwd) la_fwd;
  decltype(&orbit_la_bwd) la_bwd;
  decltype(&orbit_la_workspace_bytes) la_workspace;
  decltype(&orbit_block_norm_fwd) block_norm;
  decltype(&orbit_block_norm_bwd) block_norm_bwd;
  decltype(&orbit_block_norm_bwd_workspace_bytes) block_workspace;
  decltype(&orbit_act_pack) pack;
  decltype(&orbit_act_unpack) unpack;
} entry = {};

// a plain torch.Tensor (no subclass) on the current CUDA device for which no gradient is to be recorded and that carries no
// forward-mode tangent
bool plain(PyObject* o, at::Tensor& t, int device) {
  if (!THPVariable_CheckExact(o)) return false;
  t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == device && !(t.requires_grad() && c10::GradMode::is_enabled()) && t.layout() == at::kStrided &&
         !t._fw_grad(0).defined();
}
bool plain_or_none(PyObject* o, at::Tensor& t, int device) { return o == Py_None || plain(o, t, device); }

int io_code(const at::Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? ORBIT_BF16 : t.scalar_type() == at::kFloat ? ORBIT_F32 : -1;
}
// the current device, or -1 for a call whose first operand does not live on a CUDA device (there may be none at all) and for one that
// torch.jit.trace records
int device_for(PyObject* first) {
  if (c10::impl::dispatch_mode_enabled() || at::tracer::impl::is_dispatch_enabled() || !THPVariable_CheckExact(first) || !THPVariable_Unpack(first).is_cuda()) return -1;
  return c10::cuda::current_device();
}
void* stream(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }
template <typename T> T* ptr(const at::Tensor& t) { return t.defined() ? static_cast<T*>(t.data_ptr()) : nullptr; }
bool f32_vector(const at::Tensor& t, int64_t n) {
  return !t.defined() || (t.dim() == 1 && t.size(0) == n && t.scalar_type() == at::kFloat && t.is_contiguous());
}

// the word of each device that a kernel sets when a bounded wait gives up (owned by the Python side)
constexpr int MAX_DEVICES = 64;
int* status_word[MAX_DEVICES] = {};

// (outputs..., status, launches), None for an output that is not there: the caller raises for a nonzero status
PyObject* result(int status, std::initializer_list<at::Tensor> outs, int launches = 1) {
  PyObject* t = PyTuple_New((Py_ssize_t)outs.size() + 2);
  if (t == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& x : outs) PyTuple_SET_ITEM(t, i++, x.defined() ? THPVariable_Wrap(x) : Py_NewRef(Py_None));
  PyTuple_SET_ITEM(t, i++, PyLong_FromLong(status));
  PyTuple_SET_ITEM(t, i, PyLong_FromLong(launches));
  if (PyErr_Occurred()) {
    Py_DECREF(t);
    return nullptr;
  }
  return t;
}

// C++ exceptions become the Python ones that torch raises for them (an out-of-memory error stays one)
#define GUARDED(...)   \
  HANDLE_TH_ERRORS     \
  __VA_ARGS__          \
  END_HANDLE_TH_ERRORS

// the state and the decays of a call: [B, H, Dv, Dk] and [H] float32, dense
bool state_ok(const at::Tensor& s, int64_t B, int64_t H, int64_t Dv, int64_t Dk) {
  return s.dim() == 4 && s.size(0) == B && s.size(1) == H && s.size(2) == Dv && s.size(3) == Dk && s.scalar_type() == at::kFloat && s.is_contiguous();
}

// the scale of a call: None is 1 / sqrt(Dk); false where the other way has to refuse it
bool scale_of(PyObject* o, int64_t Dk, double& scale) {
  if (o == Py_None) {
    scale = 1. / std::sqrt((double)Dk);
    return true;
  }
  scale = PyFloat_AsDouble(o);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  return std::isfinite(scale) && scale != 0.;
}

// step(q, k, v, log_decay, state, scale | None)
PyObject* la_step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) Py_RETURN_NONE;
  GUARDED({
    const int dev = device_for(a[0]);
    if (dev < 0) Py_RETURN_NONE;
    at::Tensor q, k, v, ld, s;
    if (!plain(a[0], q, dev) || !plain(a[1], k, dev) || !plain(a[2], v, dev) || !plain(a[3], ld, dev) || !plain(a[4], s, dev)) Py_RETURN_NONE;
    const int code = io_code(q);
    if (code < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || q.dim() != 3 || v.dim() != 3 ||
        k.sizes() != q.sizes() || v.size(0) != q.size(0) || v.size(1) != q.size(1))
      Py_RETURN_NONE;
    const int64_t B = q.size(0), H = q.size(1), Dk = q.size(2), Dv = v.size(2);
    double scale;
    if (B < 1 || H < 1 || Dk < 1 || Dv < 1 || Dk > 256 || Dv > 256 || !f32_vector(ld, H) || !state_ok(s, B, H, Dv, Dk) || !v.is_contiguous() ||
        q.stride(2) != 1 || k.stride(2) != 1 || B * H > (1 << 24) || !scale_of(a[5], Dk, scale))
      Py_RETURN_NONE;
    at::Tensor y = at::empty_like(v), s1 = at::empty_like(s);
    const int rc = entry.la_step(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
                                 v.stride(1), ptr<float>(ld), ptr<float>(s), ptr<float>(s1), y.data_ptr(), (int)B, (int)H, (int)Dk, (int)Dv,
                                 (float)scale, code, stream(dev));
    return result(rc, {y, s1});
  })
}

// attention(q, k, v, log_decay, state | None, scale | None, return_state) of dense operands
PyObject* la_fwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 7) Py_RETURN_NONE;
  GUARDED({
    const int dev = device_for(a[0]);
    if (dev < 0) Py_RETURN_NONE;
    if (dev >= MAX_DEVICES || status_word[dev] == nullptr) Py_RETURN_NONE;
    at::Tensor q, k, v, ld, s;
    if (!plain(a[0], q, dev) || !plain(a[1], k, dev) || !plain(a[2], v, dev) || !plain(a[3], ld, dev) || !plain_or_none(a[4], s, dev)) Py_RETURN_NONE;
    const int code = io_code(q);
    if (code < 0 || k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() || q.dim() != 4 || v.dim() != 4 ||
        k.sizes() != q.sizes() || v.size(0) != q.size(0) || v.size(1) != q.size(1) || v.size(2) != q.size(2))
      Py_RETURN_NONE;
    const int64_t B = q.size(0), L = q.size(1), H = q.size(2), Dk = q.size(3), Dv = v.size(3);
    double scale;
    const bool want = PyObject_IsTrue(a[6]) == 1;
    if (B < 1 || L < 1 || L > (1 << 30) || H < 1 || Dk < 1 || Dv < 1 || Dk > 256 || Dv > 256 || B * H > (1 << 24) || !f32_vector(ld, H) ||
        (s.defined() && !state_ok(s, B, H, Dv, Dk)) || !q.is_contiguous() || !k.is_contiguous() || !v.is_contiguous() ||
        !scale_of(a[5], Dk, scale))
      Py_RETURN_NONE;
    auto address = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
    if (code == ORBIT_BF16 && (address(q) % 16 || address(k) % 16 || address(v) % 16)) Py_RETURN_NONE;   // copied on the other way
    at::Tensor y = at::empty_like(v), s1;
    if (want) s1 = s.defined() ? at::empty_like(s) : at::empty({B, H, Dv, Dk}, q.options().dtype(at::kFloat));
    orbit_la_args p = {};
    p.B = (int)B; p.L = (int)L; p.H = (int)H; p.Dk = (int)Dk; p.Dv = (int)Dv; p.scale = (float)scale;
    p.q = q.data_ptr(); p.q_bs = L * H * Dk; p.q_ls = H * Dk; p.q_hs = Dk;
    p.k = k.data_ptr(); p.k_bs = L * H * Dk; p.k_ls = H * Dk; p.k_hs = Dk;
    p.v = v.data_ptr(); p.v_bs = L * H * Dv; p.v_ls = H * Dv; p.v_hs = Dv;
    p.y = y.data_ptr(); p.y_bs = L * H * Dv; p.y_ls = H * Dv; p.y_hs = Dv;
    p.log_decay = ptr<float>(ld);
    p.state0 = ptr<float>(s);
    p.state1 = ptr<float>(s1);
    p.status = status_word[dev];
    at::Tensor ws;
    p.workspace_bytes = entry.la_workspace(&p, 0, code);
    if (p.workspace_bytes) {
      ws = at::empty({p.workspace_bytes}, q.options().dtype(at::kByte));
      p.workspace = ws.data_ptr();
    }
    const int rc = entry.la_fwd(&p, code, stream(dev));
    return result(rc, {y, s1}, p.workspace_bytes ? 3 : 1);
  })
}

// attention_bwd(q, k, v, log_decay, state | None, scale, dy, dstate | None, want dstate0) -> (dq, dk, dv, dstate0 | None, status, launches)
PyObject* la_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) Py_RETURN_NONE;
  GUARDED({
    const int dev = device_for(a[0]);
    if (dev < 0 || dev >= MAX_DEVICES || status_word[dev] == nullptr) Py_RETURN_NONE;
    at::Tensor q, k, v, ld, s, dy, ds;
    if (!plain(a[0], q, dev) || !plain(a[1], k, dev) || !plain(a[2], v, dev) || !plain(a[3], ld, dev) || !plain_or_none(a[4], s, dev) ||
        !plain(a[6], dy, dev) || !plain_or_none(a[7], ds, dev))
      Py_RETURN_NONE;
    const int code = io_code(q);
    double scale;
    const bool want = PyObject_IsTrue(a[8]) == 1;
    // q, k, v, log_decay and state are what the forward pass checked and kept
    const int64_t B = q.size(0), L = q.size(1), H = q.size(2), Dk = q.size(3), Dv = v.size(3);
    if (code < 0 || B < 1 || L < 1 || !scale_of(a[5], Dk, scale) || !q.is_contiguous() || !k.is_contiguous() || !v.is_contiguous() ||
        dy.sizes() != v.sizes() || dy.scalar_type() != v.scalar_type() || !dy.is_contiguous() || (ds.defined() && !state_ok(ds, B, H, Dv, Dk)))
      Py_RETURN_NONE;
    auto address = [](const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()); };
    if (code == ORBIT_BF16 && (address(q) % 16 || address(k) % 16 || address(v) % 16 || address(dy) % 16)) Py_RETURN_NONE;
    at::Tensor dq = at::empty_like(q), dk = at::empty_like(k), dv = at::empty_like(v), ds0;
    if (want) ds0 = at::empty({B, H, Dv, Dk}, q.options().dtype(at::kFloat));
    orbit_la_args p = {};
    p.B = (int)B; p.L = (int)L; p.H = (int)H; p.Dk = (int)Dk; p.Dv = (int)Dv; p.scale = (float)scale;
    p.q = q.data_ptr(); p.dq = dq.data_ptr(); p.k = k.data_ptr(); p.dk = dk.data_ptr();
    p.v = v.data_ptr(); p.dv = dv.data_ptr(); p.dy = dy.data_ptr();
    p.q_bs = p.dq_bs = p.k_bs = p.dk_bs = L * H * Dk;
    p.q_ls = p.dq_ls = p.k_ls = p.dk_ls = H * Dk;
    p.q_hs = p.dq_hs = p.k_hs = p.dk_hs = Dk;
    p.v_bs = p.dv_bs = p.dy_bs = L * H * Dv;
    p.v_ls = p.dv_ls = p.dy_ls = H * Dv;
    p.v_hs = p.dv_hs = p.dy_hs = Dv;
    p.log_decay = ptr<float>(ld);
    p.state0 = ptr<float>(s);
    p.dstate1 = ptr<float>(ds);
    p.dstate0 = ptr<float>(ds0);
    p.status = status_word[dev];
    at::Tensor ws;
    p.workspace_bytes = entry.la_workspace(&p, 1, code);
    if (p.workspace_bytes) {
      ws = at::empty({p.workspace_bytes}, q.options().dtype(at::kByte));
      p.workspace = ws.data_ptr();
    }
    const int rc = entry.la_bwd(&p, code, stream(dev));
    return result(rc, {dq, dk, dv, ds0}, p.workspace_bytes ? 3 : 1);
  })
}

// The operands of a block norm: activations of one dense shape, float32 weights of its width; false for the other way.
struct BlockOperands {
  at::Tensor x, h, g, sc, post, pre;
  int dev, code;
  int64_t M, D;
  bool take(PyObject* const* a) {
    dev = device_for(a[0]);
    if (dev < 0 || !plain(a[0], x, dev) || !plain(a[1], h, dev) || !plain_or_none(a[2], g, dev) || !plain_or_none(a[3], sc, dev) ||
        !plain_or_none(a[4], post, dev) || !plain_or_none(a[5], pre, dev))
      return false;
    code = io_code(x);
    if (code < 0 || x.dim() < 1 || x.numel() == 0 || x.size(-1) > (1 << 30) || !x.is_contiguous() || !like_x(h) || (g.defined() && !like_x(g))) return false;
    D = x.size(-1);
    M = x.numel() / D;
    return f32_vector(sc, D) && f32_vector(post, D) && f32_vector(pre, D);
  }
  bool like_x(const at::Tensor& t) const { return t.sizes() == x.sizes() && t.scalar_type() == x.scalar_type() && t.is_contiguous(); }
  at::Tensor floats(int64_t n) const { return at::empty({n}, x.options().dtype(at::kFloat)); }
};

// block_norm(x, h, gate | None, scale | None, post | None, pre | None, eps, keep) -> (r, n | None[, rstd_h | None, rstd_r | None])
PyObject* block_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 8) Py_RETURN_NONE;
  GUARDED({
    BlockOperands o;
    if (!o.take(a)) Py_RETURN_NONE;
    const double eps = PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    if (!(eps >= 0.)) Py_RETURN_NONE;
    const bool keep = PyObject_IsTrue(a[7]) == 1;
    at::Tensor r = at::empty_like(o.x), y, rh, rr;
    if (o.pre.defined()) y = at::empty_like(o.x);
    if (keep && o.post.defined()) rh = o.floats(o.M);
    if (keep && o.pre.defined()) rr = o.floats(o.M);
    const int rc = entry.block_norm(o.x.data_ptr(), o.D, o.h.data_ptr(), o.D, ptr<void>(o.g), o.D, ptr<float>(o.sc), ptr<float>(o.post),
                                    ptr<float>(o.pre), r.data_ptr(), ptr<void>(y), ptr<float>(rh), ptr<float>(rr), o.M, (int)o.D, (float)eps,
                                    o.code, stream(o.dev));
    return keep ? result(rc, {r, y, rh, rr}) : result(rc, {r, y});
  })
}

// block_norm_bwd(x, h, gate | None, scale | None, post | None, pre | None, rstd_h | None, rstd_r | None, dr | None, dn | None, want sums)
// -> (dx, dh, dgate | None, dscale | None, dpost | None, dpre | None); the first eight are what the forward pass kept
PyObject* block_norm_bwd(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 11) Py_RETURN_NONE;
  GUARDED({
    BlockOperands o;
    at::Tensor rh, rr, dr, dn;
    if (!o.take(a) || !plain_or_none(a[6], rh, o.dev) || !plain_or_none(a[7], rr, o.dev) || !plain_or_none(a[8], dr, o.dev) ||
        !plain_or_none(a[9], dn, o.dev))
      Py_RETURN_NONE;
    if ((dr.defined() && !o.like_x(dr)) || (dn.defined() && !o.like_x(dn)) || o.post.defined() != rh.defined() || o.pre.defined() != rr.defined() ||
        !f32_vector(rh, o.M) || !f32_vector(rr, o.M))
      Py_RETURN_NONE;
    const bool sums = PyObject_IsTrue(a[10]) == 1;
    at::Tensor dx = at::empty_like(o.x), dh = at::empty_like(o.x), dg, ds, dpost, dpre, ws;
    if (o.g.defined()) dg = at::empty_like(o.x);
    if (sums && o.sc.defined()) ds = o.floats(o.D);
    if (sums && o.post.defined()) dpost = o.floats(o.D);
    if (sums && o.pre.defined()) dpre = o.floats(o.D);
    const int64_t bytes = ds.defined() || dpost.defined() || dpre.defined() ? entry.block_workspace(o.M, (int)o.D) : 0;
    if (bytes) ws = at::empty({bytes}, o.x.options().dtype(at::kByte));
    const int rc = entry.block_norm_bwd(o.x.data_ptr(), o.D, o.h.data_ptr(), o.D, ptr<void>(o.g), o.D, ptr<float>(o.sc), ptr<float>(o.post),
                                        ptr<float>(o.pre), ptr<float>(rh), ptr<float>(rr), ptr<void>(dr), ptr<void>(dn), dx.data_ptr(),
                                        dh.data_ptr(), ptr<void>(dg), ptr<float>(ds), ptr<float>(dpost), ptr<float>(dpre), ptr<void>(ws), bytes,
                                        o.M, (int)o.D, o.code, stream(o.dev));
    return result(rc, {dx, dh, dg, ds, dpost, dpre}, bytes ? 2 : 1);
  })
}

// pack(x) of a dense activation -> (q, exponent, status)
PyObject* pack(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 1) Py_RETURN_NONE;
  GUARDED({
    const int dev = device_for(a[0]);
    if (dev < 0) Py_RETURN_NONE;
    at::Tensor x = THPVariable_Unpack(a[0]);
    if (x.get_device() != dev || x.layout() != at::kStrided) Py_RETURN_NONE;
    const int code = io_code(x);
    if (code < 0 || x.dim() < 1 || x.numel() == 0 || x.size(-1) > (1 << 30) || !x.is_contiguous()) Py_RETURN_NONE;
    const int64_t D = x.size(-1), M = x.numel() / D;
    auto shape = x.sizes().vec();
    at::Tensor q = at::empty(shape, x.options().dtype(at::kChar));
    shape.back() = (D + 31) / 32;
    at::Tensor e = at::empty(shape, x.options().dtype(at::kByte));
    const int rc = entry.pack(x.data_ptr(), D, q.data_ptr(), e.data_ptr(), M, (int)D, code, stream(dev));
    return result(rc, {q, e});
  })
}

// unpack(q, exponent, bfloat16?) of dense tensors -> (x, None, status)
PyObject* unpack(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3) Py_RETURN_NONE;
  GUARDED({
    const int dev = device_for(a[0]);
    if (dev < 0) Py_RETURN_NONE;
    at::Tensor q, e;
    if (!plain(a[0], q, dev) || !plain(a[1], e, dev)) Py_RETURN_NONE;
    if (q.scalar_type() != at::kChar || e.scalar_type() != at::kByte || q.dim() < 1 || q.numel() == 0 || q.size(-1) > (1 << 30) || !q.is_contiguous() ||
        !e.is_contiguous() || e.dim() != q.dim() || e.size(-1) != (q.size(-1) + 31) / 32 ||
        e.sizes().slice(0, e.dim() - 1) != q.sizes().slice(0, q.dim() - 1))
      Py_RETURN_NONE;
    const bool half = PyObject_IsTrue(a[2]) == 1;
    const int64_t D = q.size(-1);
    at::Tensor x = at::empty(q.sizes(), q.options().dtype(half ? at::kBFloat16 : at::kFloat));
    const int rc = entry.unpack(q.data_ptr(), e.data_ptr(), x.data_ptr(), q.numel() / D, (int)D, half ? ORBIT_BF16 : ORBIT_F32, stream(dev));
    return result(rc, {x});
  })
}

// bind(addresses of the entry points, in the order of `Entry`)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int N = 9;
  static_assert(sizeof(Entry) == N * sizeof(void*), "one address an entry");
  void* p[N];
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", N);
    return nullptr;
  }
  for (int i = 0; i < N; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  std::memcpy(&entry, p, sizeof(entry));
  Py_RETURN_NONE;
}

// bind_status(device, address of its status word)
PyObject* bind_status(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "bind_status takes a device number and an address");
    return nullptr;
  }
  const long dev = PyLong_AsLong(a[0]);
  void* p = PyLong_AsVoidPtr(a[1]);
  if (PyErr_Occurred()) return nullptr;
  if (dev >= 0 && dev < MAX_DEVICES) status_word[dev] = static_cast<int*>(p);
  Py_RETURN_NONE;
}

#define METHOD(name, fn) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fn)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD("bind", bind),
                         METHOD("bind_status", bind_status),
                         METHOD("la_step", la_step),
                         METHOD("la_fwd", la_fwd),
                         METHOD("la_bwd", la_bwd),
                         METHOD("block_norm", block_norm),
                         METHOD("block_norm_bwd", block_norm_bwd),
                         METHOD("pack", pack),
                         METHOD("unpack", unpack),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_orbit_host", "Native host calls of the block operators. " ORBIT_HOST_TAG,
                      -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__orbit_host(void) { return PyModule_Create(&module); }
