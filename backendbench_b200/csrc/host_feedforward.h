// The operators of feedforward.py as kernels of the dispatcher (included by host.cpp, whose helpers they use).
//
// They have no aten overload, so a user calls them as torch.ops.b200.<name>; what bounds a small call there is the way
// from the dispatcher into Python and back, twice where a gradient may have to be recorded (dropout of 16 x 256, forward and backward:
// 30 us through Python kernels, 12 so). As in the callables above, nothing new is decided here: a call of plain
// tensors that need no conversion goes to the entry point that the wrapper of feedforward.py would call with the same
// arguments; any other, and any that fails, goes to the wrapper, and one with a gradient to record to its autograd function.

using TensorOpt = std::optional<Tensor>;

struct Gil {  // the dispatcher lets go of the interpreter lock before it enters a native kernel
  PyGILState_STATE state = PyGILState_Ensure();
  ~Gil() { PyGILState_Release(state); }
};
PyObject* ff_dict = nullptr;  // feedforward.py's names

struct FfOp {
  const char* name;
  const char* autograd_name;
  PyObject *attr = nullptr, *original = nullptr, *autograd = nullptr;
  bool direct() const {  // nobody has replaced the wrapper or its allocator
    return PyDict_GetItemWithError(ops_dict, allocator_key) == Py_None && PyDict_GetItemWithError(ff_dict, attr) == original;
  }
};
enum { kFfGated, kFfGatedTrain, kFfGatedBackward, kFfDropout, kFfDropoutBackward, kFfQuantize, kFfInt8, kFfOps };
FfOp ff_ops[kFfOps] = {{"gated_linear", "gated_linear_autograd"}, {"gated_linear_train", "gated_linear_train_autograd"}, {"gated_linear_backward", nullptr}, {"dropout", "dropout_autograd"},
                       {"dropout_backward", nullptr}, {"quantize_rows", nullptr}, {"mm_int8", nullptr}};

[[noreturn]] void raise_python() {
  python_error e;
  e.persist();
  throw e;
}
PyObject* py(const Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }
PyObject* py(const TensorOpt& t) { return t ? py(*t) : Py_NewRef(Py_None); }
PyObject* py(double v) { return PyFloat_FromDouble(v); }
PyObject* py(int64_t v) { return PyLong_FromLongLong(v); }
PyObject* py(c10::string_view v) { return PyUnicode_FromStringAndSize(v.data(), static_cast<Py_ssize_t>(v.size())); }
PyObject* py(std::array<bool, 2> v) { return Py_BuildValue("[OO]", v[0] ? Py_True : Py_False, v[1] ? Py_True : Py_False); }
PyObject* py(std::optional<at::ScalarType> v) { return v ? Py_NewRef(reinterpret_cast<PyObject*>(torch::getTHPDtype(*v))) : Py_NewRef(Py_None); }
template <typename T> struct Named {
  const char* name;
  T value;
};
template <typename T> void put(PyObject* args, PyObject*, Py_ssize_t& i, const T& v) { PyTuple_SET_ITEM(args, i++, py(v)); }
template <typename T> void put(PyObject*, PyObject* kwargs, Py_ssize_t&, const Named<T>& v) {
  PyObject* o = py(v.value);
  if (o) PyDict_SetItemString(kwargs, v.name, o);
  Py_XDECREF(o);
}
template <typename T> constexpr int positional(const T&) { return 1; }
template <typename T> constexpr int positional(const Named<T>&) { return 0; }
// (with the lock held) `fn` of these arguments, as the interpreter would call it
template <typename... A> PyObject* in_python(PyObject* fn, const A&... a) {
  PyObject *args = PyTuple_New((positional(a) + ... + 0)), *kwargs = PyDict_New();
  Py_ssize_t i = 0;
  (put(args, kwargs, i, a), ...);
  PyObject* r = PyErr_Occurred() ? nullptr : PyObject_Call(fn, args, kwargs);
  Py_DECREF(args);
  Py_DECREF(kwargs);
  if (!r) raise_python();
  return r;
}
Tensor taken(PyObject* r) {  // the tensor of a result, which is given up
  Tensor t = THPVariable_Unpack(r);
  Py_DECREF(r);
  return t;
}
TensorOpt taken_or_none(PyObject* o) { return o == Py_None ? TensorOpt() : TensorOpt(THPVariable_Unpack(o)); }
std::tuple<Tensor, Tensor> taken_pair(PyObject* r) {
  std::tuple<Tensor, Tensor> t{THPVariable_Unpack(PyTuple_GET_ITEM(r, 0)), THPVariable_Unpack(PyTuple_GET_ITEM(r, 1))};
  Py_DECREF(r);
  return t;
}
template <typename... A> PyObject* wrapper(int op, const A&... a) {
  PyObject* fn = PyDict_GetItemWithError(ff_dict, ff_ops[op].attr);
  if (!fn) {
    PyErr_Format(PyExc_RuntimeError, "feedforward.%s is gone", ff_ops[op].name);
    raise_python();
  }
  return in_python(fn, a...);
}
void ff_launched(bool ok) {
  if (!ok) raise_python();
}
// The lock is needed to look whether a call is direct and nowhere else on its way: where the entry point launches and returns, it
// is held for that look alone.
bool ff_direct(int op) {
  Gil gil;
  return ff_ops[op].direct();
}
void ff_check(int rc, const char* what) {
  if (rc == 0) return;
  Gil gil;
  PyObject* r = PyObject_CallFunction(check_fn, "is", rc, what);  // raises
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed with code %d", what, rc);
  raise_python();
}
uint32_t* ff_status(const Tensor& t) {
  static std::atomic<uint32_t*> words[64];
  const size_t d = static_cast<size_t>(t.get_device());
  uint32_t* w = d < 64 ? words[d].load(std::memory_order_acquire) : nullptr;
  if (w) return w;
  Gil gil;
  w = status_word(t);
  if (!w) raise_python();
  if (d < 64) words[d].store(w, std::memory_order_release);
  return w;
}
Tensor ff_scratch(const Tensor& like, int64_t bytes) { return bytes > 0 ? new_tensor({bytes}, at::kByte, like) : Tensor(); }

int activation_code(c10::string_view name) {
  constexpr const char* kNames[B200_ACT_COUNT] = {"silu", "gelu", "gelu_tanh", "relu", "sigmoid"};
  for (int i = 0; i < B200_ACT_COUNT; ++i)
    if (name == kNames[i]) return i;
  return -1;
}
// [..., K] as rows: a matrix as it is, anything else where it is contiguous
struct Rows {
  int64_t M = 0, K = 0, s_m = 0, s_k = 0;
  bool of(const Tensor& t) {
    if (t.dim() < 1) return false;
    K = t.size(t.dim() - 1);
    M = product(t.sizes(), 0, t.dim() - 1);
    if (t.dim() == 2) {
      s_m = t.stride(0);
      s_k = t.stride(1);
      return true;
    }
    s_m = K;
    s_k = 1;
    return t.is_contiguous();
  }
};
at::DimVector with_last(const Tensor& t, int64_t last) {
  at::DimVector s(t.sizes().begin(), t.sizes().end());
  s.back() = last;
  return s;
}

// (with the lock held) a @ b as feedforward._product forms it
Tensor ff_product(const Operand& a, const Operand& b, int64_t M, int64_t N, int64_t K, at::IntArrayRef shape) {
  const int64_t need = dt(a.t) == B200_F32 ? api.b200_linear_f32_scratch_bytes(M, N, K) : 0;
  if (need > 0) {
    Tensor out = new_tensor(shape, a.t.scalar_type(), a.t);
    const Tensor s = ff_scratch(a.t, need);
    ff_check(api.b200_linear_f32(static_cast<const float*>(ptr(a.t)), static_cast<const float*>(ptr(b.t)), static_cast<float*>(ptr(out)), M, N, K, a.row, a.col, b.row, b.col, ptr(s), need,
                                 ff_status(a.t), stream()),
             "b200_linear_f32");
    return out;
  }
  PyObject* r = gemm(a, b, Tensor(), 1, M, N, K, 1.0, 0.0, shape);
  if (!r) raise_python();
  return taken(r);
}

// a @ b as feedforward._scaled_product forms it
Tensor ff_scaled_product(const Operand& a, const Tensor& most, int64_t first, const Operand& b, int64_t M, int64_t N, int64_t K, at::IntArrayRef shape) {
  Tensor out = new_tensor(shape, a.t.scalar_type(), a.t);
  const int64_t need = api.b200_linear_scaled_scratch_bytes(ptr(a.t), ptr(b.t), M, N, K, a.row, a.col, b.row, b.col);
  const Tensor s = ff_scratch(a.t, need);
  ff_check(api.b200_linear_scaled(ptr(a.t), static_cast<const uint32_t*>(ptr(most)) + first, ptr(b.t), ptr(out), M, N, K, a.row, a.col, b.row, b.col, ptr(s), need, ff_status(a.t), stream()),
           "b200_linear_scaled");
  return out;
}

// The pitch of dP's rows: on lines of 128 bytes for the copy engine (fp32 ones are split into planes from anywhere)
int64_t gradient_pitch(int64_t cols, const Tensor& like) { return dt(like) == B200_F32 || cols % 64 == 0 ? cols : cols > 64 ? (cols + 63) / 64 * 64 : (cols + 7) / 8 * 8; }

// (output, projections); an undefined output: the wrapper has to take the call
std::tuple<Tensor, Tensor> gated_direct(const Tensor& x, const Tensor& w, c10::string_view activation, bool keep) {
  Rows r;
  const int act = activation_code(activation);
  if (act < 0 || !floating(x) || x.scalar_type() != w.scalar_type() || w.dim() != 2 || w.size(0) % 2 || !r.of(x) || w.size(1) != r.K || !plain(x, w)) return {};
  const int64_t F = w.size(0) / 2;
  if (r.M == 0 || F == 0 || r.K == 0) return {};
  Tensor projections;
  const int64_t planes = dt(x) == B200_F32 ? api.b200_linear_f32_scratch_bytes(r.M, 2 * F, r.K) : 0;
  if (dt(x) == B200_F32 && planes == 0) {
    Gil gil;
    PyObject* p = gemm(Operand{x, 0, r.s_m, r.s_k}, Operand{w, 0, w.stride(1), w.stride(0)}, Tensor(), 1, r.M, 2 * F, r.K, 1.0, 0.0, with_last(x, 2 * F));
    if (!p) raise_python();
    projections = taken(p);
    Tensor out = new_tensor(with_last(x, F), x.scalar_type(), x);
    ff_launched(launched("b200_gate", [&, st = stream()] { return api.b200_gate(static_cast<const float*>(ptr(projections)), static_cast<float*>(ptr(out)), r.M, F, act, st); }));
    return {out, projections};
  }
  Tensor out = new_tensor(with_last(x, F), x.scalar_type(), x);
  if (keep) projections = new_tensor(with_last(x, 2 * F), at::kFloat, x);
  if (planes > 0) {
    const Tensor s = ff_scratch(x, planes);
    ff_check(api.b200_gated_linear_f32(static_cast<const float*>(ptr(x)), static_cast<const float*>(ptr(w)), static_cast<float*>(ptr(out)), static_cast<float*>(ptr(projections)), r.M, F, r.K, r.s_m,
                                       r.s_k, w.stride(0), w.stride(1), act, ptr(s), planes, ff_status(x), stream()),
             "b200_gated_linear_f32");
    return {out, projections};
  }
  const int64_t ws0 = w.stride(0), ws1 = w.stride(1), need = api.b200_gated_linear_scratch_bytes(ptr(x), ptr(w), r.M, F, r.K, r.s_m, r.s_k, ws0, ws1);
  const Tensor s = ff_scratch(x, need);
  ff_check(api.b200_gated_linear(ptr(x), ptr(w), ptr(out), static_cast<float*>(ptr(projections)), r.M, F, r.K, r.s_m, r.s_k, ws0, ws1, act, dt(x), ptr(s), need, ff_status(x), stream()),
           "b200_gated_linear");
  return {out, projections};
}

Tensor ff_gated_linear(const Tensor& x, const Tensor& w, c10::string_view activation) {
  if (ff_direct(kFfGated)) {
    Tensor out = std::get<0>(gated_direct(x, w, activation, false));
    if (out.defined()) return out;
  }
  Gil gil;
  return taken(wrapper(kFfGated, x, w, activation));
}
std::tuple<Tensor, Tensor> ff_gated_linear_train(const Tensor& x, const Tensor& w, c10::string_view activation) {
  if (ff_direct(kFfGatedTrain)) {
    auto out = gated_direct(x, w, activation, true);
    if (std::get<0>(out).defined()) return out;
  }
  Gil gil;
  return taken_pair(wrapper(kFfGatedTrain, x, w, activation));
}
std::tuple<TensorOpt, TensorOpt> ff_gated_linear_backward(const Tensor& g, const Tensor& x, const Tensor& w, const Tensor& p, c10::string_view activation, std::array<bool, 2> mask) {
  Gil gil;
  Rows r;
  const int act = activation_code(activation);
  if (ff_ops[kFfGatedBackward].direct() && act >= 0 && floating(x) && w.dim() == 2 && w.size(0) % 2 == 0 && r.of(x) && w.size(1) == r.K && (mask[0] || mask[1]) && plain(g, x, w, p)) {
    const int64_t F = w.size(0) / 2;
    if (r.M && F && r.K && w.scalar_type() == x.scalar_type() && g.scalar_type() == x.scalar_type() && p.scalar_type() == at::kFloat && g.is_contiguous() && p.is_contiguous() &&
        g.sizes() == at::IntArrayRef(with_last(x, F)) && p.sizes() == at::IntArrayRef(with_last(x, 2 * F))) {
      const int64_t pitch = gradient_pitch(2 * F, x);
      const bool scaled = dt(x) == B200_F16;
      Tensor dp = new_tensor({r.M, pitch}, x.scalar_type(), x), dp_columns = dp, most;
      if (scaled) {
        if (mask[0] && mask[1]) dp_columns = new_tensor({r.M, pitch}, x.scalar_type(), x);
        most = new_tensor({r.M + 2 * F}, at::kInt, x);
        ff_launched(launched("b200_gate_backward_scaled", [&, st = stream()] {
          return api.b200_gate_backward_scaled(ptr(g), static_cast<const float*>(ptr(p)), mask[0] ? ptr(dp) : nullptr, mask[1] ? ptr(dp_columns) : nullptr, static_cast<uint32_t*>(ptr(most)), pitch, r.M, F,
                                               act, st);
        }));
      } else ff_launched(launched("b200_gate_backward_rows", [&, st = stream()] { return api.b200_gate_backward_rows(ptr(g), static_cast<const float*>(ptr(p)), ptr(dp), pitch, r.M, F, act, dt(x), st); }));
      std::tuple<TensorOpt, TensorOpt> out;
      const int64_t ws0 = w.stride(0), ws1 = w.stride(1);
      const bool fp32 = dt(x) == B200_F32;
      const int64_t need = fp32 ? api.b200_linear_f32_grads_scratch_bytes(r.M, 2 * F, r.K) : (scaled ? api.b200_linear_grads_scaled_scratch_bytes : api.b200_linear_grads_scratch_bytes)(ptr(dp), ptr(x), ptr(w), r.M, 2 * F, r.K, pitch, r.s_m, r.s_k, ws0, ws1);
      if (need >= 0) {
        Tensor dx, dw;
        if (mask[0]) dx = new_tensor(x.sizes(), x.scalar_type(), x);
        if (mask[1]) dw = new_tensor({2 * F, r.K}, x.scalar_type(), x);
        const Tensor s = ff_scratch(x, need);
        auto f = [](const Tensor& t) { return static_cast<float*>(ptr(t)); };
        const int rc = fp32 ? api.b200_linear_f32_grads(f(dp), f(x), f(w), f(dx), f(dw), r.M, 2 * F, r.K, pitch, 1, r.s_m, r.s_k, ws0, ws1, ptr(s), need, ff_status(x), stream())
                       : scaled ? api.b200_linear_grads_scaled(ptr(dp), ptr(dp_columns), static_cast<const uint32_t*>(ptr(most)), ptr(x), ptr(w), ptr(dx), ptr(dw), r.M, 2 * F, r.K, pitch, r.s_m, ws0, ptr(s),
                                                               need, ff_status(x), stream())
                                : api.b200_linear_grads(ptr(dp), ptr(x), ptr(w), ptr(dx), ptr(dw), r.M, 2 * F, r.K, pitch, r.s_m, ws0, dt(x), ptr(s), need, ff_status(x), stream());
        if (rc != B200_ELAUNCH) {  // (a refused cluster launch: one product after the other)
          ff_check(rc, "b200_linear_grads");
          if (mask[0]) std::get<0>(out) = dx;
          if (mask[1]) std::get<1>(out) = dw;
          return out;
        }
      }
      if (scaled) {
        if (mask[0]) std::get<0>(out) = ff_scaled_product(Operand{dp, 0, pitch, 1}, most, 0, Operand{w, 0, ws0, ws1}, r.M, r.K, 2 * F, x.sizes());
        if (mask[1]) std::get<1>(out) = ff_scaled_product(Operand{dp_columns, 0, 1, pitch}, most, r.M, Operand{x, 0, r.s_m, r.s_k}, 2 * F, r.K, r.M, w.sizes());
        return out;
      }
      if (mask[0]) std::get<0>(out) = ff_product(Operand{dp, 0, pitch, 1}, Operand{w, 0, w.stride(0), w.stride(1)}, r.M, r.K, 2 * F, x.sizes());
      if (mask[1]) std::get<1>(out) = ff_product(Operand{dp, 0, 1, pitch}, Operand{x, 0, r.s_m, r.s_k}, 2 * F, r.K, r.M, w.sizes());
      return out;
    }
  }
  PyObject* o = wrapper(kFfGatedBackward, g, x, w, p, activation, mask);
  std::tuple<TensorOpt, TensorOpt> out{taken_or_none(PyTuple_GET_ITEM(o, 0)), taken_or_none(PyTuple_GET_ITEM(o, 1))};
  Py_DECREF(o);
  return out;
}

Tensor dropout_direct(const Tensor& x, double p, const Tensor& state, const Tensor& residual, int64_t subsequence) {
  if (!floating(x) || !(p >= 0. && p <= 1.) || !x.is_contiguous() || x.numel() == 0 || state.scalar_type() != at::kLong || state.dim() != 1 || state.size(0) != 2 || !state.is_contiguous() ||
      (residual.defined() && (residual.scalar_type() != x.scalar_type() || residual.sizes() != x.sizes() || !residual.is_contiguous())) || !plain(x, state, residual))
    return {};
  Tensor out = new_like(x);
  ff_check(api.b200_dropout(ptr(x), ptr(residual), ptr(out), x.numel(), p, static_cast<const int64_t*>(ptr(state)), subsequence, dt(x), stream()), "b200_dropout");
  return out;
}
Tensor ff_dropout(const Tensor& x, double p, const Tensor& state, const TensorOpt& residual, int64_t subsequence) {
  if (ff_direct(kFfDropout)) {
    Tensor out = dropout_direct(x, p, state, residual ? *residual : Tensor(), subsequence);
    if (out.defined()) return out;
  }
  Gil gil;
  return taken(wrapper(kFfDropout, x, p, state, residual, Named<int64_t>{"subsequence", subsequence}));
}
Tensor ff_dropout_backward(const Tensor& g, double p, const Tensor& state, int64_t subsequence) {
  if (ff_direct(kFfDropoutBackward)) {
    Tensor out = dropout_direct(g, p, state, Tensor(), subsequence);
    if (out.defined()) return out;
  }
  Gil gil;
  return taken(wrapper(kFfDropoutBackward, g, p, state, Named<int64_t>{"subsequence", subsequence}));
}

std::tuple<Tensor, Tensor> ff_quantize_rows(const Tensor& x) {
  Rows r;
  if (ff_direct(kFfQuantize) && floating(x) && r.of(x) && r.s_k == 1 && x.numel() && plain(x)) {
    Tensor q = new_tensor(x.sizes(), at::kChar, x), scale = new_tensor(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
    ff_check(api.b200_quantize_rows(ptr(x), ptr(q), static_cast<float*>(ptr(scale)), r.M, r.K, r.s_m, dt(x), stream()), "b200_quantize_rows");
    return {q, scale};
  }
  Gil gil;
  return taken_pair(wrapper(kFfQuantize, x));
}

bool scale_of(const Tensor& t, int64_t n, bool column) {
  return t.scalar_type() == at::kFloat && t.is_contiguous() && ((t.dim() == 1 && t.size(0) == n) || (t.dim() == 2 && t.size(column ? 0 : 1) == n && t.size(column ? 1 : 0) == 1));
}
Tensor ff_mm_int8(const Tensor& a, const Tensor& b, const Tensor& sa, const Tensor& sb, const TensorOpt& bias, std::optional<at::ScalarType> out_dtype) {
  const Tensor none, &c = bias ? *bias : none;
  const at::ScalarType type = out_dtype ? *out_dtype : c.defined() ? c.scalar_type() : at::kBFloat16;
  if (ff_direct(kFfInt8) && a.dim() == 2 && b.dim() == 2 && a.size(1) == b.size(0) && a.numel() && b.numel() && a.size(1) <= B200_INT8_MAX_K && a.scalar_type() == at::kChar &&
      b.scalar_type() == at::kChar && scale_of(sa, a.size(0), true) && scale_of(sb, b.size(1), false) && (type == at::kFloat || type == at::kHalf || type == at::kBFloat16) &&
      (!c.defined() || (c.scalar_type() == type && c.dim() == 1 && c.size(0) == b.size(1) && c.is_contiguous())) && plain(a, b, sa, sb, c)) {
    const int64_t M = a.size(0), K = a.size(1), N = b.size(1), s[4] = {a.stride(0), a.stride(1), b.stride(0), b.stride(1)};
    Tensor out = new_tensor({M, N}, type, a);
    const int64_t need = api.b200_mm_int8_scratch_bytes(ptr(a), ptr(b), M, N, K, s[0], s[1], s[2], s[3]);
    const Tensor scratch = ff_scratch(a, need);
    ff_check(api.b200_mm_int8(ptr(a), ptr(b), static_cast<const float*>(ptr(sa)), static_cast<const float*>(ptr(sb)), ptr(c), ptr(out), M, N, K, s[0], s[1], s[2], s[3], dt(out), ptr(scratch), need,
                              ff_status(a), stream()),
             "b200_mm_int8");
    return out;
  }
  Gil gil;
  return taken(wrapper(kFfInt8, a, b, sa, sb, bias, Named<std::optional<at::ScalarType>>{"out_dtype", out_dtype}));
}

// Where a gradient may have to be recorded: the autograd function of feedforward.py if so, the kernel below if not
// (which refuses a forward-mode one)
bool wants_gradient(const Tensor& a, const Tensor& b) {
  auto of = [](const Tensor& t) { return t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(0).defined()); };
  return of(a) || of(b);
}
// Plain tensors would come to the CUDA kernel by the dispatcher, too
bool straight(const Tensor& a, const Tensor& b) {
  const auto tls = c10::impl::tls_local_dispatch_key_set();
  if (((a.key_set() | b.key_set() | tls.included_) - tls.excluded_).has_any(c10::python_ks)) return false;  // (fake tensors, where there may be no device to ask)
  return !a.requires_grad() && !b.requires_grad() && plain(a, b);
}
template <typename F> auto below(const char* name) { return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>(); }

Tensor ff_gated_linear_autograd(const Tensor& x, const Tensor& w, c10::string_view activation) {
  if (wants_gradient(x, w)) {
    Gil gil;
    return taken(in_python(ff_ops[kFfGated].autograd, x, w, activation));
  }
  if (straight(x, w)) return ff_gated_linear(x, w, activation);
  static const auto op = below<Tensor(const Tensor&, const Tensor&, c10::string_view)>("b200::gated_linear");
  at::AutoDispatchBelowAutograd guard;
  return op.call(x, w, activation);
}
std::tuple<Tensor, Tensor> ff_gated_linear_train_autograd(const Tensor& x, const Tensor& w, c10::string_view activation) {
  if (wants_gradient(x, w)) {
    Gil gil;
    return taken_pair(in_python(ff_ops[kFfGatedTrain].autograd, x, w, activation));
  }
  if (straight(x, w)) return ff_gated_linear_train(x, w, activation);
  static const auto op = below<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, c10::string_view)>("b200::gated_linear_train");
  at::AutoDispatchBelowAutograd guard;
  return op.call(x, w, activation);
}
Tensor ff_dropout_autograd(const Tensor& x, double p, const Tensor& state, const TensorOpt& residual, int64_t subsequence) {
  if (wants_gradient(x, residual ? *residual : Tensor())) {
    Gil gil;
    return taken(in_python(ff_ops[kFfDropout].autograd, x, p, state, residual, Named<int64_t>{"subsequence", subsequence}));
  }
  if (straight(x, state) && (!residual || straight(*residual, state))) return ff_dropout(x, p, state, residual, subsequence);
  static const auto op = below<Tensor(const Tensor&, double, const Tensor&, const TensorOpt&, int64_t)>("b200::dropout");
  at::AutoDispatchBelowAutograd guard;
  return op.call(x, p, state, residual, subsequence);
}

// feedforward(module): the kernels above take the CUDA and Autograd keys of the operators that custom_ops.py has defined
PyObject* feedforward(PyObject*, PyObject* module) {
  HANDLE_TH_ERRORS
  if (!ops_dict || ff_dict) return PyErr_Format(PyExc_RuntimeError, "setup() comes first, and this once");
  PyObject* dict = PyModule_GetDict(module);
  for (FfOp& op : ff_ops) {
    op.attr = PyUnicode_InternFromString(op.name);
    op.original = op.attr ? Py_XNewRef(PyDict_GetItemWithError(dict, op.attr)) : nullptr;
    op.autograd = op.autograd_name ? PyObject_GetAttrString(module, op.autograd_name) : nullptr;
    if (!op.original || (op.autograd_name && !op.autograd)) return PyErr_Format(PyExc_RuntimeError, "feedforward.%s is missing", op.name);
  }
  ff_dict = Py_NewRef(dict);
  static auto* library = new torch::Library(torch::Library::FRAGMENT, "b200", std::nullopt, __FILE__, __LINE__);
  auto cuda = [&](const char* name, auto* f) { library->impl(name, torch::dispatch(c10::DispatchKey::CUDA, f)); };
  auto grad = [&](const char* name, auto* f) { library->impl(name, torch::dispatch(c10::DispatchKey::Autograd, f)); };
  cuda("gated_linear", ff_gated_linear);
  cuda("gated_linear_train", ff_gated_linear_train);
  cuda("gated_linear_backward", ff_gated_linear_backward);
  cuda("dropout", ff_dropout);
  cuda("dropout_backward", ff_dropout_backward);
  cuda("quantize_rows", ff_quantize_rows);
  cuda("mm_int8", ff_mm_int8);
  grad("gated_linear", ff_gated_linear_autograd);
  grad("gated_linear_train", ff_gated_linear_train_autograd);
  grad("dropout", ff_dropout_autograd);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
