// decoder_ops.h -- the host path of rotary.py, routing.py and adapters.py, a part of
// fast_ops.cpp: the same rule (a function returns None for everything that is not the
// plain case), with the nodes of torch's graph where gradients are to be recorded.
#pragma once

// A float (or an int) that is finite in 32 bits
bool number_of(PyObject* o, double* to) {
  if (PyFloat_CheckExact(o)) {
    *to = PyFloat_AS_DOUBLE(o);
  } else if (PyLong_CheckExact(o)) {
    *to = PyLong_AsDouble(o);
    if (*to == -1.0 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  } else {
    return false;
  }
  return std::isfinite(static_cast<float>(*to));
}

// An int of 1 .. 2^20; None: `fallback`
bool count_of(PyObject* o, int fallback, int* to) {
  if (o == Py_None) {
    *to = fallback;
    return true;
  }
  if (!PyLong_CheckExact(o)) {
    return false;
  }
  int overflow = 0;
  const long v = PyLong_AsLongAndOverflow(o, &overflow);
  *to = static_cast<int>(v);
  return overflow == 0 && v >= 1 && v <= 1 << 20;
}

// A tensor on `device` with something in it, no tangent and, unless `recorded`, no gradient to
// be recorded; of one of the three types
const at::Tensor* operand_of(PyObject* o, c10::DeviceIndex device, bool recorded) {
  if (!THPVariable_CheckExact(o)) {
    return nullptr;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.is_cuda() && t.device().index() == device && t.numel() != 0 &&
          !t.is_conj() && !t.is_neg() && (recorded || !records_grad(t)) &&
          !t._fw_grad(0).defined() && dtype_code(t.scalar_type()) >= 0
      ? &t
      : nullptr;
}

// The elements between rows of the last dimension, which are dense and evenly spaced; -1 if not
int64_t rows_apart(const at::Tensor& t) {
  const int64_t dims = t.dim();
  if (dims < 1 || (t.stride(dims - 1) != 1 && t.size(dims - 1) != 1)) {
    return -1;
  }
  int64_t apart = -1;
  int64_t next = 0; // of the dimension in front
  for (int64_t i = dims - 2; i >= 0; --i) {
    if (t.size(i) == 1) {
      continue;
    }
    if (apart < 0) {
      apart = t.stride(i);
    } else if (t.stride(i) != next) {
      return -1;
    }
    next = t.stride(i) * t.size(i);
  }
  return apart < 0 ? t.size(dims - 1) : apart;
}

// A gradient as rows of the given type
at::Tensor rows_of(const at::Tensor& t, int64_t* apart) {
  *apart = rows_apart(t);
  if (*apart >= 0) {
    return t;
  }
  at::Tensor copy = new_tensor(t.sizes(), t.scalar_type(), t.device().index());
  const int code = dtype_code(t.scalar_type());
  TORCH_CHECK(
      abi.copy_strided(
          t.data_ptr(), code, t.strides().data(), copy.data_ptr(), code, nullptr,
          static_cast<int>(t.dim()), t.sizes().data(), stream_of(t.device().index())) == MLXROCM_OK,
      abi.last_error());
  *apart = t.size(-1);
  return copy;
}

void check_gradient(const char* tag, const at::Tensor& grad, const at::Tensor& of) {
  TORCH_CHECK(grad.scalar_type() == of.scalar_type(), "[", tag, "] gradient of type ",
              grad.scalar_type(), " for a result of type ", of.scalar_type());
}

torch::autograd::variable_list once(torch::autograd::variable_list to) {
  if (!at::GradMode::is_enabled()) {
    return to;
  }
  for (at::Tensor& t : to) {
    if (t.defined()) {
      t.set_requires_grad(true);
    }
  }
  torch::autograd::DelayedError error(
      "trying to differentiate twice a function that was marked with @once_differentiable",
      static_cast<int64_t>(to.size()));
  return error.apply(std::move(to));
}

struct NotPlainCall : std::runtime_error { // (in a backward pass an error like any other)
  NotPlainCall() : std::runtime_error(abi.last_error()) {}
};

// ---- rotary positions -----------------------------------------------------------------------
struct Rotation {
  const at::Tensor* positions = nullptr; // may be null in the cache update
  const at::Tensor* freqs = nullptr;     // may be null
  int dims = 0, traditional = 0, axes = 1;
  double base = 10000.0, scale = 1.0;
  int sections[4] = {0, 0, 0, 0};

  // of positions and of dims, traditional, base, scale, freqs, sections
  bool parse(
      PyObject* at, PyObject* const* args, c10::DeviceIndex device, int64_t D, int64_t B, int64_t L,
      bool needs_positions) {
    if (!count_of(args[0], static_cast<int>(D), &dims) || dims > D || dims % 2 != 0 ||
        !PyBool_Check(args[1]) || !number_of(args[3], &scale)) {
      return false;
    }
    traditional = args[1] == Py_True;
    if (args[2] != Py_None && (!number_of(args[2], &base) || !(base > 0.0))) {
      return false;
    }
    if (args[4] != Py_None) {
      freqs = operand_of(args[4], device, false);
      if (args[2] != Py_None || freqs == nullptr || freqs->scalar_type() != at::kFloat ||
          freqs->dim() != 1 || freqs->size(0) != dims / 2 || !freqs->is_contiguous()) {
        return false;
      }
    }
    if (args[5] != Py_None) {
      if (!PyTuple_CheckExact(args[5]) || at == Py_None) {
        return false;
      }
      const Py_ssize_t n = PyTuple_GET_SIZE(args[5]);
      if (n < 1 || n > 4) {
        return false;
      }
      for (Py_ssize_t i = 0; i < n; ++i) {
        PyObject* v = PyTuple_GET_ITEM(args[5], i);
        if (!PyLong_CheckExact(v)) {
          return false;
        }
        int overflow = 0;
        const long pairs = PyLong_AsLongAndOverflow(v, &overflow);
        if (overflow != 0 || pairs < 0 || pairs > dims) {
          return false;
        }
        sections[i] = static_cast<int>(pairs);
      }
      axes = static_cast<int>(n);
      if (sections[0] + sections[1] + sections[2] + sections[3] != dims / 2) {
        return false;
      }
    }
    if (at == Py_None) {
      return !needs_positions;
    }
    if (!THPVariable_CheckExact(at)) {
      return false;
    }
    const at::Tensor& p = THPVariable_Unpack(at);
    if (!p.defined() || !p.is_cuda() || p.device().index() != device ||
        (p.scalar_type() != at::kInt && p.scalar_type() != at::kLong)) {
      return false;
    }
    const int more = args[5] != Py_None ? 1 : 0;
    positions = &p;
    return p.dim() == 2 + more && p.size(more) == B && p.size(more + 1) == L &&
        (!more || p.size(0) == axes);
  }
  int pointers(const void** at, int64_t (&strides)[3]) const {
    *at = nullptr;
    if (positions == nullptr) {
      return 0;
    }
    *at = positions->data_ptr();
    const int more = positions->dim() == 3;
    strides[0] = more ? positions->stride(0) : 0;
    strides[1] = positions->stride(more);
    strides[2] = positions->stride(more + 1);
    return positions->scalar_type() == at::kLong;
  }
  const float* divisors() const {
    return freqs == nullptr ? nullptr : static_cast<const float*>(freqs->data_ptr());
  }
};

// x [B, H, L, D] with dense columns and sizes that fit
const at::Tensor* columns_of(PyObject* o, c10::DeviceIndex device, bool recorded) {
  const at::Tensor* t = operand_of(o, device, recorded);
  if (t == nullptr || t->dim() != 4 || (t->stride(3) != 1 && t->size(3) != 1)) {
    return nullptr;
  }
  for (int i = 0; i < 4; ++i) {
    if (!fits_int(t->size(i))) {
      return nullptr;
    }
  }
  return t;
}

// A new tensor in x's memory order (dense), with rows that other operators take as they are
at::Tensor in_order_of(const at::Tensor& x) {
  at::Tensor out;
  const c10::DeviceIndex device = x.device().index();
  if (!like(x, device, &out)) {
    const at::AutoGradMode off(false);
    out = at::empty_like(x);
  }
  return dense_rows(out) ? out : new_tensor(x.sizes(), x.scalar_type(), device);
}

int rotate(const at::Tensor& x, const Rotation& r, int inverse, at::Tensor* out) {
  *out = in_order_of(x);
  int64_t strides[6];
  strides_of(x, strides);
  strides_of(*out, strides + 3);
  const void* at = nullptr;
  int64_t along[3] = {0, 0, 0};
  const int wide = r.pointers(&at, along);
  return abi.rope(
      x.data_ptr(), out->data_ptr(), x.size(0), x.size(1), x.size(2), x.size(3), strides, at, along,
      wide, r.axes, r.sections, r.dims, r.traditional, r.base, r.scale, r.divisors(), inverse,
      dtype_code(x.scalar_type()), stream_of(x.device().index()));
}

// A rotation is linear, and its transpose turns back: so any number of derivatives
struct RopeVjp : torch::autograd::Function<RopeVjp> {
  static at::Tensor forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& x, const Rotation* r,
      int64_t inverse) {
    at::Tensor out;
    if (rotate(x, *r, static_cast<int>(inverse), &out) != MLXROCM_OK) {
      throw NotPlainCall();
    }
    ctx->save_for_backward(
        {*r->positions, r->freqs == nullptr ? at::Tensor() : *r->freqs});
    ctx->saved_data["options"] = std::vector<int64_t>{
        r->dims, r->traditional, r->axes, r->sections[0], r->sections[1], r->sections[2],
        r->sections[3], inverse};
    ctx->saved_data["base"] = r->base;
    ctx->saved_data["scale"] = r->scale;
    return out;
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
    Rotation r;
    r.positions = &saved[0];
    r.freqs = saved[1].defined() ? &saved[1] : nullptr;
    r.dims = static_cast<int>(o[0]);
    r.traditional = static_cast<int>(o[1]);
    r.axes = static_cast<int>(o[2]);
    for (int i = 0; i < 4; ++i) {
      r.sections[i] = static_cast<int>(o[3 + i]);
    }
    r.base = ctx->saved_data["base"].toDouble();
    r.scale = ctx->saved_data["scale"].toDouble();
    at::Tensor grad = grads[0];
    if (grad.stride(3) != 1 && grad.size(3) != 1) {
      grad = grad.contiguous();
    }
    return {apply(grad, &r, 1 - o[7]), at::Tensor(), at::Tensor()};
  }
};

// rope(x, positions, dims, traditional, base, scale, freqs, sections)
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const c10::DeviceIndex device = bound && n == 8 ? device_of(args[0]) : -1;
  const at::Tensor* x = device < 0 ? nullptr : columns_of(args[0], device, true);
  Rotation r;
  if (x == nullptr ||
      !r.parse(args[1], args + 2, device, x->size(3), x->size(0), x->size(2), true)) {
    NOT_PLAIN;
  }
  if (records_grad(*x)) {
    return wrap(RopeVjp::apply(*x, &r, static_cast<int64_t>(0)));
  }
  at::Tensor out;
  int rc = 0;
  {
    const WithoutGil free;
    rc = rotate(*x, r, 0, &out);
  }
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  } catch (const NotPlainCall&) {
    Py_RETURN_NONE;
  FAST_CATCH
}

// rope_cache_update(q, k, v, k_pages, v_pages, block_table, lengths, positions, dims, traditional,
// base, scale, freqs, sections): the rotated queries
PyObject* rope_cache_update(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const c10::DeviceIndex device = bound && n == 14 ? device_of(args[0]) : -1;
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* q = columns_of(args[0], device, false);
  const at::Tensor* k = columns_of(args[1], device, false);
  const at::Tensor* v = columns_of(args[2], device, false);
  Cache c;
  Rotation r;
  if (q == nullptr || k == nullptr || v == nullptr || k->sizes() != v->sizes() ||
      k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() ||
      k->size(0) != q->size(0) || k->size(2) != q->size(2) || k->size(3) != q->size(3) ||
      !cache_of(args + 3, device, k->size(0), k->scalar_type(), &c) ||
      k->size(1) != c.k->size(1) || k->size(3) != c.k->size(3) ||
      !r.parse(args[7], args + 8, device, q->size(3), q->size(0), q->size(2), false)) {
    NOT_PLAIN;
  }
  for (int i = 0; i < 3; ++i) { // (what shares memory is refused there)
    if (c.k->size(i) > 1 && (c.k->stride(i) == 0 || c.v->stride(i) == 0)) {
      NOT_PLAIN;
    }
  }
  int rc = 0;
  at::Tensor out;
  {
    const WithoutGil free;
    out = in_order_of(*q);
    int64_t strides[19];
    const at::Tensor* operands[] = {q, k, v, &out, c.k, c.v};
    for (int i = 0; i < 6; ++i) {
      strides_of(*operands[i], strides + 3 * i);
    }
    strides[18] = c.table->stride(0);
    const void* at = nullptr;
    int64_t along[3] = {0, 0, 0};
    const int wide = r.pointers(&at, along);
    rc = abi.rope_cache_update(
        q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), c.k->data_ptr(),
        c.v->data_ptr(), static_cast<const int32_t*>(c.table->data_ptr()),
        static_cast<const int32_t*>(c.lengths->data_ptr()), q->size(0), q->size(1), k->size(1),
        q->size(2), q->size(3), c.k->size(0), c.k->size(2), c.table->size(1), strides, at, along,
        wide, r.axes, r.sections, r.dims, r.traditional, r.base, r.scale, r.divisors(),
        dtype_code(q->scalar_type()), stream_of(device));
  }
  if (rc != MLXROCM_OK) {
    NOT_PLAIN;
  }
  for (const at::Tensor* pages : {c.k, c.v}) { // written to: a graph that saved them is to know
    if (!pages->is_inference()) {
      pages->unsafeGetTensorImpl()->bump_version();
    }
  }
  return wrap(std::move(out));
  FAST_CATCH
}

// ---- the experts of tokens --------------------------------------------------------------------
struct Routing {
  int k = 0, sigmoid = 0, groups = 1, top_groups = 1, group_best = 1, normalize = 1;
  double scale = 1.0;
  const at::Tensor* bias = nullptr;
};

bool route(const at::Tensor& logits, const Routing& r, at::Tensor* indices, at::Tensor* weights) {
  const c10::DeviceIndex device = logits.device().index();
  const auto shape = with_last(logits, r.k);
  *indices = new_tensor(shape, at::kInt, device);
  *weights = new_tensor(shape, logits.scalar_type(), device);
  const int64_t E = logits.size(-1);
  return abi.route_experts(
             logits.data_ptr(),
             r.bias == nullptr ? nullptr : static_cast<const float*>(r.bias->data_ptr()),
             static_cast<int32_t*>(indices->data_ptr()), weights->data_ptr(), logits.numel() / E,
             rows_apart(logits), static_cast<int>(E), r.k, r.sigmoid, r.groups, r.top_groups,
             r.group_best, r.normalize, static_cast<float>(r.scale),
             dtype_code(logits.scalar_type()), stream_of(device)) == MLXROCM_OK;
}

struct RouteVjp : torch::autograd::Function<RouteVjp> {
  static torch::autograd::variable_list forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const Routing* r) {
    at::Tensor indices, weights;
    if (!route(logits, *r, &indices, &weights)) {
      throw NotPlainCall();
    }
    ctx->mark_non_differentiable({indices});
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, indices});
    ctx->saved_data["options"] = std::vector<int64_t>{r->k, r->sigmoid, r->normalize};
    ctx->saved_data["scale"] = r->scale;
    return {indices, weights};
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    if (!grads[1].defined()) {
      return {at::Tensor(), at::Tensor()};
    }
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &logits = saved[0], &indices = saved[1];
    const std::vector<int64_t> o = ctx->saved_data["options"].toIntVector();
    check_gradient("route_experts", grads[1], logits);
    int64_t apart = 0;
    const at::Tensor grad = rows_of(grads[1], &apart);
    const c10::DeviceIndex device = logits.device().index();
    const int64_t E = logits.size(-1);
    at::Tensor out = new_tensor(logits.sizes(), logits.scalar_type(), device);
    TORCH_CHECK(
        abi.route_experts_vjp(
            logits.data_ptr(), static_cast<const int32_t*>(indices.data_ptr()), grad.data_ptr(),
            out.data_ptr(), logits.numel() / E, rows_apart(logits), apart, static_cast<int>(E),
            static_cast<int>(o[0]), static_cast<int>(o[1]), static_cast<int>(o[2]),
            static_cast<float>(ctx->saved_data["scale"].toDouble()),
            dtype_code(logits.scalar_type()), stream_of(device)) == MLXROCM_OK,
        abi.last_error());
    auto to = once({out});
    to.resize(2);
    return to;
  }
};

PyObject* pair_of(at::Tensor&& one, at::Tensor&& two) {
  PyObject* out = PyTuple_New(2);
  if (out != nullptr) {
    PyTuple_SET_ITEM(out, 0, wrap(std::move(one)));
    PyTuple_SET_ITEM(out, 1, wrap(std::move(two)));
  }
  return out;
}

// route_experts(logits, k, scoring, bias, groups, top_groups, group_best, normalize, scale)
PyObject* route_experts(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const c10::DeviceIndex device = bound && n == 9 ? device_of(args[0]) : -1;
  const at::Tensor* logits = device < 0 ? nullptr : operand_of(args[0], device, true);
  Routing r;
  if (logits == nullptr || logits->dim() < 1 || rows_apart(*logits) < 0 ||
      !fits_int(logits->size(-1)) || !PyUnicode_CheckExact(args[2]) ||
      !count_of(args[1], 0, &r.k) || !count_of(args[4], 0, &r.groups) ||
      !count_of(args[5], r.groups, &r.top_groups) || !count_of(args[6], 0, &r.group_best) ||
      !PyBool_Check(args[7]) || !number_of(args[8], &r.scale)) {
    NOT_PLAIN;
  }
  r.sigmoid = PyUnicode_CompareWithASCIIString(args[2], "sigmoid") == 0;
  if (!r.sigmoid && PyUnicode_CompareWithASCIIString(args[2], "softmax") != 0) {
    NOT_PLAIN;
  }
  r.normalize = args[7] == Py_True;
  if (args[3] != Py_None) {
    r.bias = tensor_of(args[3], device);
    if (r.bias == nullptr || r.bias->dim() != 1 || r.bias->size(0) != logits->size(-1) ||
        r.bias->scalar_type() != at::kFloat) {
      NOT_PLAIN;
    }
  }
  at::Tensor indices, weights;
  if (records_grad(*logits)) {
    auto out = RouteVjp::apply(*logits, &r);
    return pair_of(std::move(out[0]), std::move(out[1]));
  }
  bool done = false;
  {
    const WithoutGil free;
    done = route(*logits, r, &indices, &weights);
  }
  if (!done) {
    NOT_PLAIN;
  }
  return pair_of(std::move(indices), std::move(weights));
  } catch (const NotPlainCall&) {
    Py_RETURN_NONE;
  FAST_CATCH
}

// ---- low-rank adapters -----------------------------------------------------------------------
struct Adaption {
  const at::Tensor* indices = nullptr; // may be null
  double scale = 1.0;
  int64_t rows = 0;
  int n = 1, adapters = 0, rank = 0, K = 0, N = 0, code = 0;
  void sizes_of(const at::Tensor& x, const at::Tensor& a, const at::Tensor& b) {
    adapters = static_cast<int>(a.size(0));
    rank = static_cast<int>(a.size(1));
    K = static_cast<int>(a.size(2));
    N = static_cast<int>(b.size(1));
    rows = x.numel() / K;
    n = indices == nullptr ? 1 : static_cast<int>(indices->numel());
    code = dtype_code(x.scalar_type());
  }
  const int32_t* index() const {
    return indices == nullptr ? nullptr : static_cast<const int32_t*>(indices->data_ptr());
  }
  // y may be undefined; h is where scale x a^T stays
  bool run(
      const at::Tensor& x, const at::Tensor& a, const at::Tensor& b, const at::Tensor& y,
      at::Tensor* out, at::Tensor* h) const {
    const c10::DeviceIndex device = x.device().index();
    *out = new_tensor(with_last(x, N), x.scalar_type(), device);
    if (h != nullptr) {
      *h = new_tensor(
          {static_cast<int64_t>(abi.adapter_h_size(rows, n, adapters, rank, K, N, code))},
          at::kByte, device);
    }
    const Workspace ws(abi.adapter_workspace_size(rows, n, adapters, rank, K, N, code), device);
    return abi.adapter_matmul(
               x.data_ptr(), a.data_ptr(), b.data_ptr(), index(), nullptr,
               y.defined() ? y.data_ptr() : nullptr, out->data_ptr(),
               h == nullptr ? nullptr : static_cast<float*>(h->data_ptr()), rows, n, adapters, rank,
               K, N, rows_apart(x), y.defined() ? rows_apart(y) : 0, static_cast<float>(scale),
               code, ws.ptr(), ws.bytes, stream_of(device)) == MLXROCM_OK;
  }
};

struct AdapterVjp : torch::autograd::Function<AdapterVjp> {
  static at::Tensor forward(
      torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& a,
      const at::Tensor& b, const std::optional<at::Tensor>& y, const Adaption* of) {
    at::Tensor out, h;
    if (!of->run(x, a, b, y.value_or(at::Tensor()), &out, &h)) {
      throw NotPlainCall();
    }
    ctx->saved_data["beside"] = y.has_value();
    ctx->save_for_backward(
        {x, a, b, h, of->indices == nullptr ? at::Tensor() : *of->indices});
    ctx->saved_data["scale"] = of->scale;
    return out;
  }
  static torch::autograd::variable_list backward(
      torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &a = saved[1], &b = saved[2], &h = saved[3];
    Adaption of;
    of.indices = saved[4].defined() ? &saved[4] : nullptr;
    of.scale = ctx->saved_data["scale"].toDouble();
    of.sizes_of(x, a, b);
    check_gradient("adapter_matmul", grads[0], x);
    int64_t apart = 0;
    const at::Tensor dout = rows_of(grads[0], &apart);
    const c10::DeviceIndex device = x.device().index();
    torch::autograd::variable_list to(4);
    const at::Tensor* operands[] = {&x, &a, &b};
    void* at[3];
    for (int i = 0; i < 3; ++i) {
      if (ctx->needs_input_grad(i)) {
        to[i] = new_tensor(operands[i]->sizes(), x.scalar_type(), device);
      }
      at[i] = to[i].defined() ? to[i].data_ptr() : nullptr;
    }
    if (at[0] != nullptr || at[1] != nullptr || at[2] != nullptr) {
      const Workspace ws(
          abi.adapter_vjp_workspace_size(
              of.rows, of.n, of.adapters, of.rank, of.K, of.N, of.code),
          device);
      TORCH_CHECK(
          abi.adapter_vjp(
              x.data_ptr(), a.data_ptr(), b.data_ptr(), of.index(), nullptr,
              static_cast<const float*>(h.data_ptr()), dout.data_ptr(), at[0], at[1], at[2],
              of.rows, of.n, of.adapters, of.rank, of.K, of.N, rows_apart(x), apart,
              static_cast<float>(of.scale), of.code, ws.ptr(), ws.bytes,
              stream_of(device)) == MLXROCM_OK,
          abi.last_error());
    }
    if (ctx->saved_data["beside"].toBool() && ctx->needs_input_grad(3)) {
      to[3] = grads[0];
      if (at::GradMode::is_enabled()) {
        to[3] = to[3].detach();
      }
    }
    to = once(std::move(to));
    to.resize(5);
    return to;
  }
};

// adapter_matmul(x, a, b, indices, scale, y)
PyObject* adapter_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) {
  FAST_TRY
  const c10::DeviceIndex device = bound && n == 6 ? device_of(args[0]) : -1;
  if (device < 0) {
    NOT_PLAIN;
  }
  const at::Tensor* x = operand_of(args[0], device, true);
  const at::Tensor* a = operand_of(args[1], device, true);
  const at::Tensor* b = operand_of(args[2], device, true);
  Adaption of;
  if (x == nullptr || a == nullptr || b == nullptr || x->dim() < 1 || a->dim() != 3 ||
      b->dim() != 3 || a->scalar_type() != x->scalar_type() ||
      b->scalar_type() != x->scalar_type() || !a->is_contiguous() || !b->is_contiguous() ||
      a->size(0) != b->size(0) || a->size(1) != b->size(2) || x->size(-1) != a->size(2) ||
      !fits_int(a->size(0)) || !fits_int(a->size(1)) || !fits_int(a->size(2)) ||
      !fits_int(b->size(1)) || rows_apart(*x) < 0 || !number_of(args[4], &of.scale)) {
    NOT_PLAIN;
  }
  if (args[3] == Py_None) {
    if (a->size(0) != 1) {
      NOT_PLAIN;
    }
  } else {
    if (!THPVariable_CheckExact(args[3])) {
      NOT_PLAIN;
    }
    const at::Tensor& i = THPVariable_Unpack(args[3]);
    if (!i.defined() || !i.is_cuda() || i.device().index() != device ||
        i.scalar_type() != at::kInt || !i.is_contiguous() || i.dim() >= x->dim() ||
        i.sizes() != x->sizes().slice(0, i.dim()) || !fits_int(i.numel())) {
      NOT_PLAIN;
    }
    of.indices = &i;
  }
  at::Tensor y;
  if (args[5] != Py_None) {
    const at::Tensor* t = operand_of(args[5], device, true);
    if (t == nullptr || t->scalar_type() != x->scalar_type() || t->dim() != x->dim() ||
        t->sizes() != at::IntArrayRef(with_last(*x, b->size(1))) || rows_apart(*t) < 0) {
      NOT_PLAIN;
    }
    y = *t;
  }
  of.sizes_of(*x, *a, *b);
  if (records_grad(*x) || records_grad(*a) || records_grad(*b) ||
      (y.defined() && records_grad(y))) {
    // (the graph has no place for a tensor that is none)
    const std::optional<at::Tensor> beside = y.defined() ? std::optional(y) : std::nullopt;
    return wrap(AdapterVjp::apply(*x, *a, *b, beside, &of));
  }
  at::Tensor out;
  bool done = false;
  {
    const WithoutGil free;
    done = of.run(*x, *a, *b, y, &out, nullptr);
  }
  if (!done) {
    NOT_PLAIN;
  }
  return wrap(std::move(out));
  } catch (const NotPlainCall&) {
    Py_RETURN_NONE;
  FAST_CATCH
}
