// Bindings of the operators that stand beside the factored layers: low-rank adapters, the gated feed-forward block and the AdamW step.
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

inline Tensor empty_as(at::IntArrayRef size, const Tensor& like) {
  return at::detail::empty_cuda(size, like.scalar_type(), like.device(), std::nullopt);
}
Tensor contiguous(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }
Tensor bytes_on(size_t n, const Tensor& like) {
  return at::detail::empty_cuda({(int64_t)std::max<size_t>(n, 16)}, at::kByte, like.device(), std::nullopt);
}
int size_arg(int64_t n, const char* name) {
  TORCH_CHECK_VALUE(n <= 0x7fffffff, name, " is ", n, ", at most 2**31 - 1 is possible");
  return (int)n;
}

// ---- low-rank adapters ------------------------------------------------------------------------------------------------
// The adapters' numbers as the library takes them
Tensor adapter_numbers(const Tensor& which, int64_t count) {
  TORCH_CHECK_TYPE(which.scalar_type() == at::kInt || which.scalar_type() == at::kLong, "adapters must be an int32 or int64 CUDA tensor");
  return contiguous(which.scalar_type() == at::kInt ? which : which.clamp(-1, count).to(at::kInt));
}
// The plan of a batch: bytes on the device that depend on the rows' adapters and on the number of adapters
Tensor adapter_plan(const Tensor& which_, int64_t count) {
  const int rows = size_arg(which_.numel(), "the number of rows"), n = size_arg(count, "the number of adapters");
  const size_t need = b200cp_adapter_plan_bytes(rows, n);
  TORCH_CHECK_VALUE(need, "adapter_plan: ", rows, " rows and ", n, " adapters (1 to 16384 of them)");
  const c10::cuda::OptionalCUDAGuard guard(which_.device());
  const Tensor which = adapter_numbers(which_, count);
  Tensor plan = bytes_on(need, which);
  ok(b200cp_adapter_plan(rows, n, static_cast<const int*>(which.const_data_ptr()), plan.data_ptr(), need, stream(which)));
  return plan;
}
struct Adapters {   // operands, checked and contiguous
  Tensor x, A, B, scale;
  int rows, I, O, R, count, type;
  Adapters(const Tensor& x_, const Tensor& A_, const Tensor& B_, const Tensor& scale_) {
    type = type_of(x_, "X");
    TORCH_CHECK_VALUE(x_.dim() >= 1 && A_.dim() == 3 && B_.dim() == 3, "expected X [..., I], A [count, I, R] and B [count, R, O]");
    TORCH_CHECK_VALUE(A_.size(1) == x_.size(-1) && B_.size(0) == A_.size(0) && B_.size(1) == A_.size(2), "A ", A_.sizes(), " and B ", B_.sizes(),
                      " do not go with X ", x_.sizes());
    for (const Tensor* t : {&A_, &B_}) same(*t, x_, t == &A_ ? "A" : "B");
    I = size_arg(A_.size(1), "I");
    R = size_arg(A_.size(2), "the rank");
    O = size_arg(B_.size(2), "O");
    count = size_arg(A_.size(0), "the number of adapters");
    TORCH_CHECK_VALUE(I > 0 && O > 0 && R > 0 && count > 0, "A and B may not be empty");
    rows = size_arg(x_.numel() / I, "the number of rows");
    if (scale_.defined()) {
      TORCH_CHECK_TYPE(scale_.is_cuda() && scale_.scalar_type() == at::kFloat, "scale must be a float32 CUDA tensor");
      TORCH_CHECK_VALUE(scale_.device() == x_.device() && scale_.numel() == count, "scale has to have a value per adapter, on X's device");
      scale = contiguous(scale_);
    }
    x = contiguous(x_);
    A = contiguous(A_);
    B = contiguous(B_);
  }
  static void same(const Tensor& t, const Tensor& like, const char* name) {
    TORCH_CHECK_TYPE(t.is_cuda() && t.scalar_type() == like.scalar_type(), name, " must be a CUDA tensor of X's type, ", like.scalar_type());
    TORCH_CHECK_VALUE(t.device() == like.device(), name, " is on ", t.device(), ", X on ", like.device());
  }
  void fits(const Tensor& y, const char* name) const {
    same(y, x, name);
    TORCH_CHECK_VALUE(y.dim() == x.dim() && y.size(-1) == O && y.sizes().slice(0, y.dim() - 1) == x.sizes().slice(0, x.dim() - 1), name, " is ",
                      y.sizes(), " where X is ", x.sizes(), " and B has ", O, " columns");
  }
  // `which`: the adapter of every row, or the bytes of a plan for `planned` adapters (0: no plan)
  Tensor plan(const Tensor& which, int64_t planned) const {
    check_numbers(which, planned);
    return planned ? which : adapter_plan(which, count);
  }
  // the numbers themselves where a batch is small enough to go without a plan, or else a plan (*planned)
  Tensor numbers(const Tensor& which, int64_t* planned) const {
    check_numbers(which, *planned);
    if (*planned) return which;
    if (rows > B200CP_ADAPTERS_WITHOUT_PLAN) *planned = count;
    return *planned ? adapter_plan(which, count) : adapter_numbers(which, count);
  }
  void check_numbers(const Tensor& which, int64_t planned) const {
    TORCH_CHECK_VALUE(which.device() == x.device(), "the adapters' numbers are on ", which.device(), ", X on ", x.device());
    if (!planned) {
      TORCH_CHECK_TYPE(which.scalar_type() == at::kInt || which.scalar_type() == at::kLong, "adapters must be an int32 or int64 CUDA tensor");
      TORCH_CHECK_VALUE(which.sizes() == x.sizes().slice(0, x.dim() - 1), "there are numbers of adapters for ", which.sizes(), ", X is ", x.sizes());
      TORCH_CHECK_VALUE(b200cp_adapter_plan_bytes(rows, count), rows, " rows and ", count, " adapters (1 to 16384 of them)");
      return;
    }
    // (the sizes of two plans may be the same where their counts are not)
    TORCH_CHECK_VALUE(planned == count, "the plan is one of ", planned, " adapters, A and B are of ", count);
    TORCH_CHECK_VALUE(which.scalar_type() == at::kByte && which.is_contiguous() &&
                          (size_t)which.numel() == std::max<size_t>(16, b200cp_adapter_plan_bytes(rows, count)),
                      "the plan is not one of ", rows, " rows and ", count, " adapters");
  }
  void takes(const Tensor& out, const Tensor& y, const Tensor& which) const {   // as the place of the result
    fits(out, "out");
    TORCH_CHECK_VALUE(out.is_contiguous(), "out has to be contiguous");
    const auto meets = [&](const Tensor& t) {   // (from the first to behind the last value that a tensor holds)
      if (!t.numel() || !out.numel()) return false;
      int64_t last = 0;
      for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
      const auto a = reinterpret_cast<uintptr_t>(t.const_data_ptr()), b = reinterpret_cast<uintptr_t>(out.const_data_ptr());
      return a < b + out.nbytes() && b < a + (size_t)(last + 1) * t.element_size();
    };
    for (const Tensor* t : {&x, &A, &B, &which}) TORCH_CHECK_VALUE(!meets(*t), "out may share memory with Y alone");
    TORCH_CHECK_VALUE(!scale.defined() || !meets(scale), "out may share memory with Y alone");
    TORCH_CHECK_VALUE(!meets(y) || (y.is_contiguous() && y.const_data_ptr() == out.const_data_ptr()),
                      "out may be Y, but not another part or order of its memory");
  }
  const float* scales() const { return scale.defined() ? cp(scale) : nullptr; }
};
Tensor dense_adapters(const Adapters& a, const Tensor& y_, const Tensor& which, bool planned, Tensor out, Tensor* V) {
  a.fits(y_, "Y");
  const Tensor y = contiguous(y_);
  if (!out.defined()) out = empty_as(y.sizes(), y);
  const c10::cuda::OptionalCUDAGuard guard(a.x.device());
  if (V) *V = empty_as({a.rows, a.R}, a.x);
  const void* by = which.const_data_ptr();
  ok(b200cp_dense_adapters(a.rows, a.I, a.O, a.R, a.count, a.type, y.const_data_ptr(), a.x.const_data_ptr(), a.A.const_data_ptr(), a.B.const_data_ptr(),
                           a.scales(), planned ? nullptr : static_cast<const int*>(by), planned ? by : nullptr, out.data_ptr(),
                           V ? V->data_ptr() : nullptr, stream(a.x)));
  return out;
}
std::array<Tensor, 3> dense_adapters_backward(const Adapters& a, const Tensor& dy_, const Tensor& V, const Tensor& plan, bool need_x, bool need_a,
                                              bool need_b) {
  std::array<Tensor, 3> g;
  a.fits(dy_, "dY");
  const Tensor dy = contiguous(dy_);
  const c10::cuda::OptionalCUDAGuard guard(a.x.device());
  if (need_x) g[0] = empty_as(a.x.sizes(), a.x);
  if (need_a) g[1] = empty_as(a.A.sizes(), a.x);
  if (need_b) g[2] = empty_as(a.B.sizes(), a.x);
  const Tensor ws = bytes_on(b200cp_dense_adapters_bwd_workspace_bytes(a.rows, a.I, a.O, a.R, a.count, a.type), a.x);
  const auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  ok(b200cp_dense_adapters_bwd(a.rows, a.I, a.O, a.R, a.count, a.type, dy.const_data_ptr(), a.x.const_data_ptr(), V.const_data_ptr(),
                               a.A.const_data_ptr(), a.B.const_data_ptr(), a.scales(), plan.const_data_ptr(), at(g[0]), at(g[1]), at(g[2]),
                               ws.data_ptr(), (size_t)ws.numel(), stream(a.x)));
  return g;
}
struct AdaptersNode : torch::autograd::Function<AdaptersNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& y, const Tensor& x, const Tensor& A, const Tensor& B, const Tensor& plan,
                        const std::optional<Tensor>& scale_) {
    const Tensor scale = scale_.value_or(Tensor());
    const Adapters a(x, A, B, scale);
    Tensor V;
    Tensor out = dense_adapters(a, y, plan, true, Tensor(), &V);
    ctx->save_for_backward({x, A, B, plan, scale, V});
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list v = ctx->get_saved_variables();
    variable_list out(6);
    if (ctx->needs_input_grad(0)) out[0] = grads[0];
    const bool need_x = ctx->needs_input_grad(1), need_a = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
    if (need_x || need_a || need_b) {
      const Adapters a(v[0], v[1], v[2], v[4]);
      const std::array<Tensor, 3> g = dense_adapters_backward(a, grads[0], v[5], v[3], need_x, need_a, need_b);
      for (int i = 0; i < 3; ++i) out[1 + i] = g[i];
    }
    return out;
  }
};

// ---- gated feed-forward block ------------------------------------------------------------------------------------------
struct Gated {   // operands, checked, contiguous and on 16-byte boundaries
  Tensor x, Wg, Wu;
  int rows, I, F, type, act;
  Gated(const Tensor& x_, const Tensor& Wg_, const Tensor& Wu_, int64_t act_) : act((int)act_) {
    type = type_of(x_, "X");
    TORCH_CHECK_TYPE(type != B200CP_FLOAT32, "X must be a bfloat16 or float16 CUDA tensor (float32: dense_matmul)");
    TORCH_CHECK_VALUE(x_.dim() >= 1 && Wg_.dim() == 2 && Wg_.sizes() == Wu_.sizes(), "expected X [..., I], Wg and Wu [I, F]");
    TORCH_CHECK_VALUE(x_.size(-1) == Wg_.size(0), "X ", x_.sizes(), " does not go with weights ", Wg_.sizes());
    Adapters::same(Wg_, x_, "Wg");
    Adapters::same(Wu_, x_, "Wu");
    I = size_arg(Wg_.size(0), "I");
    F = size_arg(Wg_.size(1), "F");
    TORCH_CHECK_VALUE(I > 0 && F > 0, "the weights may not be empty");
    rows = size_arg(x_.numel() / I, "the number of rows");
    x = whole(x_);
    Wg = whole(Wg_);
    Wu = whole(Wu_);
  }
  int64_t kept() const { return ((int64_t)F + 7) / 8 * 8; }   // floats of a row of G and U
  static Tensor whole(const Tensor& t) {
    const Tensor c = contiguous(t);
    return (reinterpret_cast<uintptr_t>(c.const_data_ptr()) & 15) == 0 ? c : c.clone();
  }
  std::vector<int64_t> size(int64_t last) const {
    std::vector<int64_t> s = x.sizes().vec();
    s.back() = last;
    return s;
  }
};
Tensor dense_gated(const Gated& g, Tensor* G, Tensor* U) {
  const c10::cuda::OptionalCUDAGuard guard(g.x.device());
  Tensor H = empty_as(g.size(g.F), g.x);
  if (G) {
    *G = empty({g.rows, g.kept()}, g.x);
    *U = empty({g.rows, g.kept()}, g.x);
  }
  const Scratch ws(b200cp_dense_gated_workspace_bytes(g.rows, g.I, g.F, g.type), g.x);
  ok(b200cp_dense_gated(g.rows, g.I, g.F, g.type, g.act, g.x.const_data_ptr(), g.Wg.const_data_ptr(), g.Wu.const_data_ptr(), H.data_ptr(),
                        G ? mp(*G) : nullptr, U ? mp(*U) : nullptr, ws.ptr, ws.bytes, stream(g.x)));
  return H;
}
std::array<Tensor, 3> dense_gated_backward(const Gated& g, const Tensor& G_, const Tensor& U_, const Tensor& dH_, bool need_x, bool need_w) {
  Adapters::same(dH_, g.x, "dH");
  TORCH_CHECK_VALUE(dH_.sizes() == at::IntArrayRef(g.size(g.F)), "dH is ", dH_.sizes(), ", ", at::IntArrayRef(g.size(g.F)), " is needed");
  // G and U as the forward left them (padded rows, or the columns of those), or any others of the right size
  const auto check = [&](const Tensor& t, const char* name) {
    TORCH_CHECK_TYPE(t.is_cuda() && t.scalar_type() == at::kFloat, name, " must be a float32 CUDA tensor");
    TORCH_CHECK_VALUE(t.device() == g.x.device(), name, " is on ", t.device(), ", X on ", g.x.device());
    TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == g.rows && (t.size(1) == g.F || t.size(1) == g.kept()), name, " is ", t.sizes(), " where [", g.rows,
                      ", ", g.F, "] is needed");
  };
  check(G_, "G");
  check(U_, "U");
  const auto kept = [&](const Tensor& t) {
    const bool as_left = t.stride(1) == 1 && (t.stride(0) == g.kept() || g.rows <= 1) &&
                         (int64_t)(t.storage().nbytes() / sizeof(float)) - t.storage_offset() >= g.rows * g.kept();
    if (as_left && (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0) return t;
    Tensor c = empty({g.rows, g.kept()}, g.x);
    c.narrow(1, 0, t.size(1)).copy_(t);
    return c;
  };
  const c10::cuda::OptionalCUDAGuard guard(g.x.device());
  const Tensor G = kept(G_), U = kept(U_), dH = contiguous(dH_);
  std::array<Tensor, 3> d;
  if (need_x) d[0] = empty_as(g.x.sizes(), g.x);
  if (need_w) {
    d[1] = empty_as(g.Wg.sizes(), g.x);
    d[2] = empty_as(g.Wg.sizes(), g.x);
  }
  if (!need_x && !need_w) return d;
  const auto at = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
  const Scratch ws(b200cp_dense_gated_bwd_workspace_bytes(g.rows, g.I, g.F, g.type), g.x);
  ok(b200cp_dense_gated_bwd(g.rows, g.I, g.F, g.type, g.act, g.x.const_data_ptr(), g.Wg.const_data_ptr(), g.Wu.const_data_ptr(), cp(G), cp(U),
                            dH.const_data_ptr(), at(d[0]), at(d[1]), at(d[2]), ws.ptr, ws.bytes, stream(g.x)));
  return d;
}
struct GatedNode : torch::autograd::Function<GatedNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& Wg, const Tensor& Wu, int64_t act, bool grad) {
    const Gated g(x, Wg, Wu, act);
    ctx->saved_data["act"] = act;
    if (!grad) return dense_gated(g, nullptr, nullptr);
    Tensor G, U;
    Tensor H = dense_gated(g, &G, &U);
    ctx->save_for_backward({x, Wg, Wu, G, U});
    return H;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list v = ctx->get_saved_variables();
    const Gated g(v[0], v[1], v[2], ctx->saved_data["act"].toInt());
    const std::array<Tensor, 3> d =
        dense_gated_backward(g, v[3], v[4], grads[0], ctx->needs_input_grad(0), ctx->needs_input_grad(1) || ctx->needs_input_grad(2));
    return {d[0], d[1], d[2], Tensor(), Tensor()};
  }
};

Tensor optional_tensor(PyObject* o, const char* name) { return o == Py_None ? Tensor() : any_tensor(o, name); }
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
PYFN(py_adapter_plan) {
  HANDLE_TH_ERRORS
  count_args(n, 2);
  const Tensor& which = any_tensor(a[0], "adapters");
  const int64_t count = int_arg(a[1]);
  return wrap(unlocked([&] { return adapter_plan(which, count); }));
  END_HANDLE_TH_ERRORS
}
// (Y, X, A, B, which, the count of the plan or 0, scale or None, out or None)
PYFN(py_dense_adapters) {
  HANDLE_TH_ERRORS
  count_args(n, 8);
  const Tensor &y = any_tensor(a[0], "Y"), &x = any_tensor(a[1], "X"), &A = any_tensor(a[2], "A"), &B = any_tensor(a[3], "B"),
               &which = any_tensor(a[4], "adapters");
  int64_t planned = int_arg(a[5]);
  const Tensor scale = optional_tensor(a[6], "scale"), to = optional_tensor(a[7], "out");
  Tensor out = unlocked([&] {
    const Adapters op(x, A, B, scale);
    op.fits(y, "Y");
    if (to.defined()) op.takes(to, y, which);
    const Tensor by = op.numbers(which, &planned);
    return dense_adapters(op, y, by, planned, to, nullptr);
  });
  if (to.defined()) written(to);
  return wrap(out);
  END_HANDLE_TH_ERRORS
}
// (dY, X, V, A, B, plan, its count, scale or None, need_dx, need_da, need_db)
PYFN(py_dense_adapters_backward) {
  HANDLE_TH_ERRORS
  count_args(n, 11);
  const Tensor &dy = any_tensor(a[0], "dY"), &x = any_tensor(a[1], "X"), &V_ = any_tensor(a[2], "V"), &A = any_tensor(a[3], "A"),
               &B = any_tensor(a[4], "B"), &plan = any_tensor(a[5], "plan");
  const int64_t planned = int_arg(a[6]);
  const Tensor scale = optional_tensor(a[7], "scale");
  const bool nx = truth(a[8]), na = truth(a[9]), nb = truth(a[10]);
  return wrap_tuple(unlocked([&] {
    const Adapters op(x, A, B, scale);
    Adapters::same(V_, x, "V");
    TORCH_CHECK_VALUE(V_.numel() == (int64_t)op.rows * op.R, "V has ", V_.numel(), " values, ", op.rows, " rows of rank ", op.R, " are needed");
    return dense_adapters_backward(op, dy, contiguous(V_), op.plan(plan, planned), nx, na, nb);
  }));
  END_HANDLE_TH_ERRORS
}
// (y, x, A, B, which, the count of the plan or 0, scale or None)
PYFN(py_adapters_apply) {
  HANDLE_TH_ERRORS
  count_args(n, 7);
  const Tensor &y = any_tensor(a[0], "Y"), &x = any_tensor(a[1], "X"), &A = any_tensor(a[2], "A"), &B = any_tensor(a[3], "B"),
               &which = any_tensor(a[4], "adapters");
  int64_t planned = int_arg(a[5]);
  const Tensor scale = optional_tensor(a[6], "scale");
  const bool grad = at::GradMode::is_enabled() && (y.requires_grad() || x.requires_grad() || A.requires_grad() || B.requires_grad());
  return wrap(unlocked([&] {
    if (!grad) {   // nothing is kept, and a small batch needs no plan
      const Adapters op(x, A, B, scale);
      op.fits(y, "Y");
      const Tensor by = op.numbers(which, &planned);
      return dense_adapters(op, y, by, planned, Tensor(), nullptr);
    }
    Tensor plan;
    {
      at::NoGradGuard none;
      const Adapters op(x, A, B, scale);
      op.fits(y, "Y");
      plan = op.plan(which, planned);
    }
    return AdaptersNode::apply(y, x, A, B, plan, scale.defined() ? std::optional<Tensor>(scale) : std::nullopt);
  }));
  END_HANDLE_TH_ERRORS
}

// (X, Wg, Wu, activation)
PYFN(py_dense_gated) {
  HANDLE_TH_ERRORS
  count_args(n, 4);
  const Tensor &x = any_tensor(a[0], "X"), &g = any_tensor(a[1], "Wg"), &u = any_tensor(a[2], "Wu");
  const int64_t act = int_arg(a[3]);
  return wrap(unlocked([&] { return dense_gated(Gated(x, g, u, act), nullptr, nullptr); }));
  END_HANDLE_TH_ERRORS
}
PYFN(py_dense_gated_save) {
  HANDLE_TH_ERRORS
  count_args(n, 4);
  const Tensor &x = any_tensor(a[0], "X"), &g = any_tensor(a[1], "Wg"), &u = any_tensor(a[2], "Wu");
  const int64_t act = int_arg(a[3]);
  std::array<Tensor, 3> r;
  unlocked([&] {
    const Gated op(x, g, u, act);
    r[0] = dense_gated(op, &r[1], &r[2]);
    for (int i = 1; i < 3; ++i) r[i] = r[i].narrow(1, 0, op.F);
  });
  return wrap_tuple(r);
  END_HANDLE_TH_ERRORS
}
// (dH, X, Wg, Wu, G, U, activation, need_dx, need_dw)
PYFN(py_dense_gated_backward) {
  HANDLE_TH_ERRORS
  count_args(n, 9);
  const Tensor &dh = any_tensor(a[0], "dH"), &x = any_tensor(a[1], "X"), &wg = any_tensor(a[2], "Wg"), &wu = any_tensor(a[3], "Wu"),
               &g = any_tensor(a[4], "G"), &u = any_tensor(a[5], "U");
  const int64_t act = int_arg(a[6]);
  const bool nx = truth(a[7]), nw = truth(a[8]);
  return wrap_tuple(unlocked([&] { return dense_gated_backward(Gated(x, wg, wu, act), g, u, dh, nx, nw); }));
  END_HANDLE_TH_ERRORS
}
PYFN(py_gated_apply) {
  HANDLE_TH_ERRORS
  count_args(n, 4);
  const Tensor &x = any_tensor(a[0], "X"), &g = any_tensor(a[1], "Wg"), &u = any_tensor(a[2], "Wu");
  const int64_t act = int_arg(a[3]);
  const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || g.requires_grad() || u.requires_grad());
  return wrap(unlocked([&] { return GatedNode::apply(x, g, u, act, grad); }));
  END_HANDLE_TH_ERRORS
}

// ---- AdamW step -----------------------------------------------------------------------------------------------------------
// The tensors of a list by address: what bounds a step over many small tensors is the host, and a copy of a tensor counts its references.  (`hold` is a tuple of
// its own: the list may be changed by others while the interpreter is given up.)
struct TensorList {
  pybind11::object hold;
  std::vector<const Tensor*> t;
  TensorList() = default;
  TensorList(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(PySequence_Check(o) && !THPVariable_Check(o), name, " must be a list of CUDA tensors");
    PyObject* seq = PySequence_Tuple(o);
    if (!seq) throw python_error();
    hold = pybind11::reinterpret_steal<pybind11::object>(seq);
    const Py_ssize_t n = PyTuple_GET_SIZE(seq);
    t.reserve((size_t)n);
    for (Py_ssize_t i = 0; i < n; ++i) t.push_back(&any_tensor(PyTuple_GET_ITEM(seq, i), name));
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
  // what the launch reads and writes: a list for each kind of tensor
  enum { kParam, kGrad, kAvg, kSq, kScaleAvg, kScaleSq, kMaster, kKinds };
  std::vector<b200cp::Span> spans(kKinds * count);
  const auto span = [&](int kind, size_t i, const void* p, size_t bytes) {
    spans[kind * count + i] = {reinterpret_cast<uintptr_t>(p), reinterpret_cast<uintptr_t>(p) + bytes};
  };
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
    const b200cp_adamw_tensor& e = ts[i];
    span(kParam, i, e.param, p[i].nbytes());
    span(kGrad, i, e.grad, g[i].nbytes());
    span(kAvg, i, e.exp_avg, m[i].nbytes());
    span(kSq, i, e.exp_avg_sq, v[i].nbytes());
    if (small) {
      span(kScaleAvg, i, e.scale_avg, ms[i].nbytes());
      span(kScaleSq, i, e.scale_sq, vs[i].nbytes());
    }
    if (copies) span(kMaster, i, e.master, w[i].nbytes());
  }
  b200cp::SpanList kinds[kKinds];
  size_t used = 0;
  for (int k = 0; k < kKinds; ++k)
    if ((small || (k != kScaleAvg && k != kScaleSq)) && (copies || k != kMaster)) kinds[used++] = {&spans[k * count], count, k != kGrad};
  TORCH_CHECK_VALUE(!b200cp::spans_meet(kinds, used), "adamw_step: a tensor occurs twice in what is updated, or shares memory with another one");
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
