// Bindings of the operators that stand beside the factored layers: the AdamW step.
// Part of torch_binding.cpp's namespace, whose helpers it uses.

// ---- types ------------------------------------------------------------------------------------------------------------
int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return B200CP_FLOAT32;
    case at::kBFloat16: return B200CP_BFLOAT16;
    case at::kHalf: return B200CP_FLOAT16;
    default: TORCH_CHECK_TYPE(false, name, " must be a float32, bfloat16 or float16 CUDA tensor, it is ", t.scalar_type());
  }
}
const Tensor& any_tensor(PyObject* o, const char* name) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a CUDA tensor");
  const Tensor& t = THPVariable_Unpack(o);
  TORCH_CHECK_TYPE(t.is_cuda(), name, " must be a CUDA tensor, it is on ", t.device());
  return t;
}
double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
// an operand that is written in place, as autograd has to know it
void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ---- AdamW step -----------------------------------------------------------------------------------------------------------
// A list of tensors by address: what bounds a step over many small tensors is the host, and a copy of a tensor counts its references
struct TensorList {
  pybind11::object hold;
  std::vector<const Tensor*> t;
  TensorList() = default;
  TensorList(PyObject* o, const char* name) {
    PyObject* seq = PySequence_Fast(o, name);
    if (!seq) {
      PyErr_Format(PyExc_TypeError, "%s must be a list of CUDA tensors", name);
      throw python_error();
    }
    hold = pybind11::reinterpret_steal<pybind11::object>(seq);
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
    t.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) t.push_back(&any_tensor(PySequence_Fast_GET_ITEM(seq, i), name));
  }
  size_t size() const { return t.size(); }
  const Tensor& operator[](size_t i) const { return *t[i]; }
};

// (params, grads, exp_avg, exp_avg_sq, scales or None twice, master or None, step, lr, beta1, beta2, eps, weight_decay)
PYFN(py_adamw_step) {
  HANDLE_TH_ERRORS
  count_args(n, 13);
  const TensorList p(a[0], "params"), g(a[1], "grads"), m(a[2], "exp_avg"), v(a[3], "exp_avg_sq");
  const bool small = a[4] != Py_None, copies = a[6] != Py_None;
  TensorList ms, vs, w;
  if (small) {
    ms = TensorList(a[4], "scales");
    vs = TensorList(a[5], "scales");
  }
  if (copies) w = TensorList(a[6], "master");
  const size_t count = p.size();
  TORCH_CHECK_VALUE(g.size() == count && m.size() == count && v.size() == count && (!small || (ms.size() == count && vs.size() == count)) &&
                        (!copies || w.size() == count),
                    "adamw_step: ", count, " params need as many grads, moments, scales and master copies");
  b200cp_adamw h{};
  const Tensor *step = nullptr, *lr = nullptr;
  if (THPVariable_Check(a[7])) {
    step = &any_tensor(a[7], "step");
    TORCH_CHECK_TYPE(step->scalar_type() == at::kLong && step->numel() == 1, "step must be an int or one int64 in a CUDA tensor");
  } else {
    h.step = int_arg(a[7]);
  }
  if (THPVariable_Check(a[8])) {
    lr = &any_tensor(a[8], "lr");
    TORCH_CHECK_TYPE(lr->scalar_type() == at::kFloat && lr->numel() == 1, "lr must be a number or one float32 in a CUDA tensor");
  } else {
    h.lr = float_arg(a[8]);
  }
  h.beta1 = float_arg(a[9]);
  h.beta2 = float_arg(a[10]);
  h.eps = float_arg(a[11]);
  h.weight_decay = float_arg(a[12]);
  if (!count) Py_RETURN_NONE;
  const int type = type_of(p[0], "params"), gtype = type_of(g[0], "grads");
  TORCH_CHECK_TYPE(gtype == type || gtype == B200CP_FLOAT32, "grads must have the params' type or float32");
  TORCH_CHECK_VALUE(!copies || type != B200CP_FLOAT32, "master copies are of 16-bit parameters");
  const at::ScalarType pt = p[0].scalar_type(), gt = g[0].scalar_type(), mt = small ? at::kChar : at::kFloat, vt = small ? at::kByte : at::kFloat;
  const c10::Device device = p[0].device();
  const auto fits = [&](const Tensor& t, const char* name, at::ScalarType want, int64_t numel, bool in_place) {
    TORCH_CHECK_TYPE(t.scalar_type() == want, name, " must be ", want, ", it is ", t.scalar_type());
    TORCH_CHECK_VALUE(t.device() == device, name, " is on ", t.device(), ", the first parameter on ", device);
    TORCH_CHECK_VALUE(t.numel() == numel, name, " has ", t.numel(), " values where ", numel, " are needed");
    TORCH_CHECK_VALUE(!in_place || t.is_contiguous(), name, " is updated in place and has to be contiguous");
  };
  for (const Tensor* t : {step, lr}) TORCH_CHECK_VALUE(!t || t->device() == device, "step and lr have to be on the parameters' device");
  for (size_t i = 0; i < count; ++i) {
    const int64_t numel = p[i].numel(), blocks = (numel + 255) / 256;
    fits(p[i], "params", pt, numel, true);
    fits(g[i], "grads", gt, numel, false);
    fits(m[i], "exp_avg", mt, numel, true);
    fits(v[i], "exp_avg_sq", vt, numel, true);
    TORCH_CHECK_VALUE(g[i].is_contiguous() || g[i].sizes() == p[i].sizes(), "grads have to have the parameters' shapes");
    if (small) {
      fits(ms[i], "scales", at::kFloat, blocks, true);
      fits(vs[i], "scales", at::kFloat, blocks, true);
    }
    if (copies) fits(w[i], "master", at::kFloat, numel, true);
  }
  std::vector<b200cp_adamw_tensor> ts(count);
  std::vector<Tensor> held;   // contiguous copies of gradients
  std::vector<uintptr_t> seen;
  seen.reserve(2 * count);
  const c10::cuda::OptionalCUDAGuard guard(device);
  const auto at_of = [](const Tensor& t) { return t.mutable_data_ptr(); };
  for (size_t i = 0; i < count; ++i) {
    const int64_t numel = p[i].numel();
    if (!numel) continue;
    const void* grad;
    if (g[i].is_contiguous()) {
      grad = g[i].const_data_ptr();
    } else {
      held.push_back(g[i].contiguous());
      grad = held.back().const_data_ptr();
    }
    ts[i] = {at_of(p[i]), grad, at_of(m[i]), at_of(v[i]), small ? mp(ms[i]) : nullptr, small ? mp(vs[i]) : nullptr, copies ? mp(w[i]) : nullptr,
             (unsigned long long)numel};
    seen.push_back((uintptr_t)ts[i].param);
    seen.push_back((uintptr_t)ts[i].exp_avg);
    seen.push_back((uintptr_t)ts[i].exp_avg_sq);
  }
  if (!std::is_sorted(seen.begin(), seen.end())) std::sort(seen.begin(), seen.end());
  TORCH_CHECK_VALUE(std::adjacent_find(seen.begin(), seen.end()) == seen.end(), "adamw_step: a tensor occurs twice in what is updated");
  if (step) h.device_step = reinterpret_cast<const long long*>(step->const_data_ptr());
  if (lr) h.device_lr = static_cast<const float*>(lr->const_data_ptr());
  void* st = stream(p[0]);
  unlocked([&] { ok(b200cp_adamw_step(ts.data(), (int)count, type, gtype, small ? 8 : 32, &h, st)); });
  for (size_t i = 0; i < count; ++i) {
    for (const Tensor* t : {&p[i], &m[i], &v[i]}) written(*t);
    if (small) {
      written(ms[i]);
      written(vs[i]);
    }
    if (copies) written(w[i]);
  }
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
// (exp_avg, exp_avg_sq, scale_avg, scale_sq, out of the type and device wanted)
PYFN(py_adamw_moments) {
  HANDLE_TH_ERRORS
  count_args(n, 6);
  const Tensor &m = any_tensor(a[0], "exp_avg"), &v = any_tensor(a[1], "exp_avg_sq"), &ms = any_tensor(a[2], "scales"),
               &vs = any_tensor(a[3], "scales"), &om = any_tensor(a[4], "out"), &ov = any_tensor(a[5], "out");
  const int64_t count = m.numel();
  TORCH_CHECK_TYPE(m.scalar_type() == at::kChar && v.scalar_type() == at::kByte && ms.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat,
                   "adamw_moments: int8 and uint8 codes with float32 scales");
  TORCH_CHECK_VALUE(v.numel() == count && ms.numel() == (count + 255) / 256 && vs.numel() == ms.numel(),
                    "adamw_moments: codes of one size, a scale per 256 of them");
  for (const Tensor* t : {&m, &v, &ms, &vs, &om, &ov}) {
    TORCH_CHECK_VALUE(t->is_contiguous(), "adamw_moments: contiguous tensors");
    TORCH_CHECK_VALUE(t->device() == m.device(), "adamw_moments: tensors on one device");
  }
  const int type = type_of(om, "out");
  const c10::cuda::OptionalCUDAGuard guard(m.device());
  void* st = stream(m);
  unlocked([&] {
    ok(b200cp_adamw_moments((unsigned long long)count, m.const_data_ptr(), v.const_data_ptr(), cp(ms), cp(vs), type, om.data_ptr(), ov.data_ptr(), st));
  });
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}
