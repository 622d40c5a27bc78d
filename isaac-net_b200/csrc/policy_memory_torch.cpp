// The policy's memory (causal_conv, selective_scan and their steps) and distill_loss on torch tensors: argument checks,
// outputs, autograd, and the calls of the C ABI, as policy_torch.cpp has them for the other operators.
#include "policy_torch.h"

void register_memory(py::module_& m);

namespace {

using Maybe = std::optional<Tensor>;

struct Api {
  int (*conv_fwd)(const InbConvArgs*, void*);
  int (*conv_bwd)(const InbConvArgs*, void*);
  int (*conv_work)(const InbConvArgs*, int64_t*);
  int (*scan_fwd)(const InbScanArgs*, void*);
  int (*scan_bwd)(const InbScanArgs*, void*);
  int (*scan_kept)(const InbScanArgs*, int64_t*);
  int (*scan_work)(const InbScanArgs*, int32_t, int64_t*);
  int (*distill_fwd)(const InbDistillArgs*, void*);
  int (*distill_bwd)(const InbDistillArgs*, void*);
} api;

void bind_memory(const std::map<std::string, uintptr_t>& f, py::object error) {
  api.conv_fwd = reinterpret_cast<decltype(api.conv_fwd)>(f.at("inb_causal_conv_fwd"));
  api.conv_bwd = reinterpret_cast<decltype(api.conv_bwd)>(f.at("inb_causal_conv_bwd"));
  api.conv_work = reinterpret_cast<decltype(api.conv_work)>(f.at("inb_causal_conv_work"));
  api.scan_fwd = reinterpret_cast<decltype(api.scan_fwd)>(f.at("inb_selective_scan_fwd"));
  api.scan_bwd = reinterpret_cast<decltype(api.scan_bwd)>(f.at("inb_selective_scan_bwd"));
  api.scan_kept = reinterpret_cast<decltype(api.scan_kept)>(f.at("inb_selective_scan_kept"));
  api.scan_work = reinterpret_cast<decltype(api.scan_work)>(f.at("inb_selective_scan_work"));
  api.distill_fwd = reinterpret_cast<decltype(api.distill_fwd)>(f.at("inb_distill_fwd"));
  api.distill_bwd = reinterpret_cast<decltype(api.distill_bwd)>(f.at("inb_distill_bwd"));
  unsupported = error.release().ptr();
}

// ------------------------------------------------------------------------------------------------- sequences
// The one stride of axes [0, last) of t, 0 where they hold one element or none, -1 where there is none
int64_t one_stride(const Tensor& t, int64_t last) {
  int64_t ld = -1, next = 0;
  for (int64_t i = last - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (ld < 0)
      ld = t.stride(i);
    else if (t.stride(i) != next)
      return -1;
    next = t.stride(i) * t.size(i);
  }
  return ld < 0 ? 0 : ld;
}
// [..., T, C] as sequences (a step: [..., C]): any stride between sequences and between steps, elements contiguous
bool is_seq(const Tensor& t, bool step) {
  return t.numel() == 0 || ((t.stride(-1) == 1 || t.size(-1) == 1) && one_stride(t, t.dim() - (step ? 1 : 2)) >= 0);
}
InbSeq seq_of(const Tensor& t, void* p, bool step) {
  return {p, one_stride(t, t.dim() - (step ? 1 : 2)), step ? 0 : t.stride(-2)};
}
struct Seq {
  Tensor t;
  InbSeq q = {};
  Seq() = default;
  explicit Seq(const Tensor& in, bool step = false) {
    if (!in.defined()) return;
    t = is_seq(in, step) ? in : in.contiguous();
    q = seq_of(t, const_cast<void*>(t.const_data_ptr()), step);
  }
};
// A new tensor of t's shape in t's order of axes, so that a rollout that lies step by step gives one that does
Tensor like_seq(const Tensor& t, bool step = false) {
  if (!t.defined()) return {};
  Tensor o = at::empty_like(t);
  return is_seq(o, step) ? o : at::empty(t.sizes(), t.options());
}
InbSeq write_seq(const Tensor& t, bool step = false) {
  if (!t.defined()) return {};
  return seq_of(t, t.mutable_data_ptr(), step);
}
// States [..., A, B]: the inner two axes contiguous, one stride between sequences; a copy where that is not so
struct States {
  Tensor t;
  int64_t seq = 0;
  explicit States(const Tensor& in) {
    if (!in.defined()) return;
    t = fits(in) ? in : in.contiguous();
    seq = one_stride(t, t.dim() - 2);
  }
  static bool fits(const Tensor& t) {
    return t.numel() == 0 || ((t.stride(-1) == 1 || t.size(-1) == 1) && (t.stride(-2) == t.size(-1) || t.size(-2) == 1) &&
                              one_stride(t, t.dim() - 2) >= 0);
  }
};
// reset [..., T] (a step: [...]): leading sizes those of x up to some axis, 1 from there on (missing ones count as 1); `lead`: x's
// axes before the steps
int64_t shared_axes(const Tensor& in, int64_t lead, bool step, int64_t& miss) {
  miss = lead + (step ? 0 : 1) - in.dim();
  int64_t axis = lead - 1;
  while (axis >= 0 && (axis < miss || in.size(axis - miss) == 1)) --axis;
  return axis;
}
struct Resets {
  Tensor t;
  InbReset q = {};
  Resets() = default;
  Resets(const Tensor& in, const Tensor& x, int64_t lead, bool step) {
    if (!in.defined()) return;
    int64_t miss = 0, rows = 1;
    const int64_t axis = shared_axes(in, lead, step, miss);
    for (int64_t i = axis + 1; i < lead; ++i) rows *= x.size(i);
    t = in.numel() == 0 || one_stride(in, axis + 1) >= 0 ? in : in.contiguous();
    q = {(const uint8_t*)t.const_data_ptr(), rows > 0 ? rows : 1, axis < 0 ? 0 : one_stride(t, axis + 1), step ? 0 : t.stride(-1)};
  }
};
void check_reset(const Tensor& reset, const Tensor& x, int64_t lead, int64_t steps, bool step) {
  same(reset, "reset", x, at::kBool);
  int64_t miss = 0, axis = shared_axes(reset, lead, step, miss);
  bool fits = miss >= 0 && (step || (reset.dim() >= 1 && reset.size(-1) == steps));
  for (; fits && axis >= 0; --axis) fits = axis >= miss && reset.size(axis - miss) == x.size(axis);
  VALUE_CHECK(fits, "reset of shape ", reset.sizes(), " does not fit x of shape ", x.sizes(), ": its leading sizes, then ones",
              step ? "" : ", then the steps");
}
void check_shape(const Tensor& t, const char* name, const Tensor& x, int64_t lead, std::initializer_list<int64_t> inner) {
  std::vector<int64_t> want(x.sizes().begin(), x.sizes().begin() + lead);
  want.insert(want.end(), inner.begin(), inner.end());
  VALUE_CHECK(t.sizes() == at::IntArrayRef(want), name, " must have shape ", at::IntArrayRef(want), ", got ", t.sizes());
}
Maybe maybe(const Tensor& t) { return t.defined() ? Maybe(t) : std::nullopt; }
Tensor floats(int64_t n, const Tensor& x) { return at::empty({n}, x.options().dtype(at::kFloat)); }
int64_t sequences(const Tensor& x, int64_t lead) {
  int64_t n = 1;
  for (int64_t i = 0; i < lead; ++i) n *= x.size(i);
  return n;
}
// A state that a step updates in place
void check_in_place(const Tensor& t, const char* op) {
  VALUE_CHECK(States::fits(t), "state must hold each sequence's values contiguously and its sequences one stride apart: ", op,
              " updates it in place");
  const int64_t inner = t.size(-1) * t.size(-2), n = t.numel() / std::max<int64_t>(1, inner);
  VALUE_CHECK(n <= 1 || one_stride(t, t.dim() - 2) >= inner, "state's sequences share memory: ", op, " updates it in place");
}
void no_grad_step(std::initializer_list<Tensor> ts, const char* op) {
  if (any_grad(ts)) refuse(op, " is not differentiable: call it under torch.no_grad()");
}
// What autograd saved of the state is not what it holds now
void touched(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// ------------------------------------------------------------------------------------------------- causal_conv
struct ConvIn {
  Tensor x, w, bias, state, reset;      // x [..., T, C], reset's last axis the steps; a step: without them
  int64_t act;
  bool step = false;
  int64_t lead() const { return x.dim() - (step ? 1 : 2); }
};
InbConvArgs conv_args(const ConvIn& i, const Seq& x, const States& st, const Resets& r) {
  InbConvArgs a = {};
  a.dtype = type_code(i.x.scalar_type());
  a.act = (int32_t)i.act;
  a.C = (int32_t)i.x.size(-1), a.K = (int32_t)i.w.size(1);
  a.S = sequences(i.x, i.lead()), a.T = i.step ? 1 : i.x.size(-2);
  a.x = x.q;
  a.w = ptr(i.w), a.bias = ptr(i.bias), a.state = ptr(st.t), a.state_seq = st.seq;
  a.reset = r.q;
  return a;
}
std::vector<int64_t> conv_state_shape(const ConvIn& i) {
  std::vector<int64_t> s(i.x.sizes().begin(), i.x.sizes().end());
  s[s.size() - 2] = i.w.size(1) - 1;
  return s;
}
std::pair<Tensor, Tensor> conv_forward(const ConvIn& i) {
  Tensor y = like_seq(i.x), out = at::empty(conv_state_shape(i), i.x.options());
  if (i.x.numel() == 0) {
    if (i.state.defined())
      out.copy_(i.state);
    else
      out.zero_();
    return {y, out};
  }
  const On on(i.x);
  const Seq x(i.x);
  const States st(i.state);
  const Resets r(i.reset, i.x, i.lead(), false);
  InbConvArgs a = conv_args(i, x, st, r);
  a.y = write_seq(y);
  a.state_out = ::out(out), a.state_out_seq = (int64_t)(a.K - 1) * a.C;
  check(api.conv_fwd(&a, on.stream), "inb_causal_conv_fwd");
  return {y, out};
}
struct CausalConv : torch::autograd::Function<CausalConv> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor w, Maybe bias, Maybe state, Maybe reset, int64_t act) {
    const ConvIn i = {x, w, bias.value_or(Tensor()), state.value_or(Tensor()), reset.value_or(Tensor()), act};
    auto [y, out] = conv_forward(i);
    ctx->save_for_backward({i.x, i.w, i.bias, i.state, i.reset});
    ctx->saved_data["a"] = act;
    ctx->set_materialize_grads(false);
    return {y, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const ConvIn i = {v[0], v[1], v[2], v[3], v[4], ctx->saved_data["a"].toInt()};
    variable_list o = {like_seq(i.x), like(i.w), like(i.bias), i.state.defined() ? at::empty(i.state.sizes(), i.state.options()) : Tensor(),
                       {}, {}};
    if ((!grads[0].defined() && !grads[1].defined()) || i.x.numel() == 0) {
      for (Tensor& t : o)
        if (t.defined()) t.zero_();
      if (i.x.numel() == 0 && o[3].defined() && grads[1].defined()) o[3].copy_(grads[1]);
      return once(o);
    }
    const On on(i.x);
    const Seq x(i.x), gy(grads[0].defined() ? grads[0] : at::zeros_like(i.x));
    const States st(i.state);
    const Resets r(i.reset, i.x, i.lead(), false);
    InbConvArgs a = conv_args(i, x, st, r);
    const Tensor gout = grads[1].defined() ? grads[1].contiguous() : Tensor();
    a.gy = gy.q, a.gx = write_seq(o[0]);
    a.gstate_out = ptr(gout);
    a.gw = out(o[1]), a.gbias = out(o[2]), a.gstate = out(o[3]);
    check(api.conv_work(&a, &a.work_elems), "inb_causal_conv_work");
    const Tensor work = floats(a.work_elems, i.x);
    a.work = (float*)out(work);
    check(api.conv_bwd(&a, on.stream), "inb_causal_conv_bwd");
    return once(o);
  }
};
// Shapes, types and limits; x [..., T, C], a step's [..., C]
void conv_check(const Tensor& x, const Tensor& w, const Maybe& bias, const Maybe& state, const Maybe& reset, bool step) {
  first(x, "x");
  VALUE_CHECK(x.dim() >= (step ? 1 : 2) && x.size(-1) >= 1, "x must be ", step ? "[..., C]" : "[..., T, C]", " with C >= 1, got shape ",
              x.sizes());
  const int64_t lead = x.dim() - (step ? 1 : 2), c = x.size(-1), t = step ? 1 : x.size(-2);
  same(w, "weight", x, x.scalar_type());
  VALUE_CHECK(w.dim() == 2 && w.size(0) == c, "weight must have shape [", c, ", K], got ", w.sizes());
  if (w.size(1) < 2 || w.size(1) > 4) refuse("causal_conv: K = ", w.size(1), ": 2 to 4 taps");
  if (c > INB_MAX_MEMORY_C || t > INB_MAX_MEMORY_S || sequences(x, lead) > INB_MAX_MEMORY_S)
    refuse("causal_conv: sizes of x ", x.sizes(), " are above its limits");
  if (bias) {
    same(*bias, "bias", x, x.scalar_type());
    vector(*bias, "bias", c);
  }
  if (state) {
    same(*state, "state", x, x.scalar_type());
    check_shape(*state, "state", x, lead, {w.size(1) - 1, c});
  }
  if (reset) check_reset(*reset, x, lead, t, step);
  no_tangents({{&x, "x"}, {&w, "weight"}, {given(bias), "bias"}, {given(state), "state"}});
}
py::tuple causal_conv(const Tensor& x, const Tensor& w, const Maybe& bias, const Maybe& state, const Maybe& reset, int64_t act) {
  conv_check(x, w, bias, state, reset, false);
  const ConvIn i = {x, w.contiguous(), bias ? bias->contiguous() : Tensor(), state.value_or(Tensor()), reset.value_or(Tensor()), act};
  if (any_grad({i.x, i.w, i.bias, i.state})) {
    const variable_list o = CausalConv::apply(i.x, i.w, maybe(i.bias), maybe(i.state), maybe(i.reset), act);
    return py::make_tuple(o[0], o[1]);
  }
  auto [y, out] = conv_forward(i);
  return py::make_tuple(y, out);
}
Tensor causal_conv_step(const Tensor& x, const Tensor& w, const Tensor& state, const Maybe& bias, const Maybe& reset, int64_t act) {
  conv_check(x, w, bias, state, reset, true);
  check_in_place(state, "causal_conv_step");
  no_grad_step({x, w, state, bias.value_or(Tensor())}, "causal_conv_step");
  const at::NoGradGuard no_grad;
  const ConvIn i = {x, w.contiguous(), bias ? bias->contiguous() : Tensor(), state, reset.value_or(Tensor()), act, true};
  const Tensor y = like_seq(x, true);
  if (x.numel() > 0) {
    const On on(x);
    const Seq xs(x, true);
    const States st(state);
    const Resets r(i.reset, x, i.lead(), true);
    InbConvArgs a = conv_args(i, xs, st, r);
    a.y = write_seq(y, true);
    a.state_out = out(state), a.state_out_seq = st.seq;
    check(api.conv_fwd(&a, on.stream), "inb_causal_conv_fwd");
    touched(state);
  }
  return y;
}

// ------------------------------------------------------------------------------------------------- selective_scan
struct ScanIn {
  Tensor x, dt, a, b, c, d, z, bias, state, reset;      // x, dt, z [..., T, C], b, c [..., T, N]; a step: without T
  bool step = false;
  int64_t lead() const { return x.dim() - (step ? 1 : 2); }
};
struct ScanRows {
  Seq x, dt, z, b, c;
  States st;
  Resets r;
  explicit ScanRows(const ScanIn& i)
      : x(i.x, i.step), dt(i.dt, i.step), z(i.z, i.step), b(i.b, i.step), c(i.c, i.step), st(i.state),
        r(i.reset, i.x, i.lead(), i.step) {}
};
InbScanArgs scan_args(const ScanIn& i, const ScanRows& r) {
  InbScanArgs a = {};
  a.dtype = type_code(i.x.scalar_type());
  a.C = (int32_t)i.x.size(-1), a.N = (int32_t)i.a.size(1);
  a.S = sequences(i.x, i.lead()), a.T = i.step ? 1 : i.x.size(-2);
  a.x = r.x.q, a.dt = r.dt.q, a.z = r.z.q, a.b = r.b.q, a.c = r.c.q;
  a.a = (const float*)ptr(i.a), a.d = (const float*)ptr(i.d), a.dt_bias = (const float*)ptr(i.bias);
  a.state = (const float*)ptr(r.st.t), a.state_seq = r.st.seq;
  a.reset = r.r.q;
  return a;
}
std::tuple<Tensor, Tensor, Tensor> scan_forward(const ScanIn& i, bool keep) {
  std::vector<int64_t> shape(i.x.sizes().begin(), i.x.sizes().end() - 2);
  shape.insert(shape.end(), {i.x.size(-1), i.a.size(1)});
  Tensor y = like_seq(i.x), out = at::empty(shape, i.a.options()), kept;
  if (i.x.numel() == 0) {
    if (i.state.defined())
      out.copy_(i.state);
    else
      out.zero_();
    return {y, out, kept};
  }
  const On on(i.x);
  const ScanRows r(i);
  InbScanArgs a = scan_args(i, r);
  a.y = write_seq(y);
  a.state_out = (float*)::out(out), a.state_out_seq = (int64_t)a.C * a.N;
  if (keep) {
    int64_t n = 0;
    check(api.scan_kept(&a, &n), "inb_selective_scan_kept");
    kept = floats(n, i.x);
    if (n > 0) a.kept = (float*)::out(kept);
  }
  check(api.scan_work(&a, 0, &a.work_elems), "inb_selective_scan_work");
  Tensor work;
  if (a.work_elems > 0) {
    work = floats(a.work_elems, i.x);
    a.work = (float*)::out(work);
  }
  check(api.scan_fwd(&a, on.stream), "inb_selective_scan_fwd");
  return {y, out, kept};
}
struct SelectiveScan : torch::autograd::Function<SelectiveScan> {
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor dt, Tensor a, Tensor b, Tensor c, Maybe d, Maybe z, Maybe bias,
                               Maybe state, Maybe reset) {
    const ScanIn i = {x, dt, a, b, c, d.value_or(Tensor()), z.value_or(Tensor()), bias.value_or(Tensor()), state.value_or(Tensor()),
                      reset.value_or(Tensor())};
    auto [y, out, kept] = scan_forward(i, true);
    ctx->save_for_backward({i.x, i.dt, i.a, i.b, i.c, i.d, i.z, i.bias, i.state, i.reset, kept});
    ctx->set_materialize_grads(false);
    return {y, out};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const ScanIn i = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8], v[9]};
    auto flat = [](const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); };
    variable_list o = {like_seq(i.x), like_seq(i.dt), flat(i.a), flat(i.b), flat(i.c), flat(i.d), like_seq(i.z), flat(i.bias),
                       flat(i.state), {}};
    if ((!grads[0].defined() && !grads[1].defined()) || i.x.numel() == 0) {
      for (Tensor& t : o)
        if (t.defined()) t.zero_();
      if (i.x.numel() == 0 && o[8].defined() && grads[1].defined()) o[8].copy_(grads[1]);
      return once(o);
    }
    const On on(i.x);
    const ScanRows r(i);
    InbScanArgs a = scan_args(i, r);
    const Seq gy(grads[0].defined() ? grads[0] : at::zeros_like(i.x));
    const Tensor gout = grads[1].defined() ? grads[1].contiguous() : Tensor();
    if (v[10].defined() && v[10].numel() > 0) a.kept = (float*)out(v[10]);
    a.gy = gy.q, a.gstate_out = (const float*)ptr(gout);
    a.gx = write_seq(o[0]), a.gdt = write_seq(o[1]), a.ga = (float*)out(o[2]), a.gb = write_seq(o[3]), a.gc = write_seq(o[4]);
    a.gd = (float*)out(o[5]), a.gz = write_seq(o[6]), a.gdt_bias = (float*)out(o[7]), a.gstate = (float*)out(o[8]);
    check(api.scan_work(&a, 1, &a.work_elems), "inb_selective_scan_work");
    const Tensor work = floats(a.work_elems, i.x);
    a.work = (float*)out(work);
    check(api.scan_bwd(&a, on.stream), "inb_selective_scan_bwd");
    return once(o);
  }
};
void scan_check(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& d, const Maybe& z,
                const Maybe& bias, const Maybe& state, const Maybe& reset, bool step) {
  first(x, "x");
  VALUE_CHECK(x.dim() >= (step ? 1 : 2) && x.size(-1) >= 1, "x must be ", step ? "[..., C]" : "[..., T, C]", " with C >= 1, got shape ",
              x.sizes());
  const int64_t lead = x.dim() - (step ? 1 : 2), ch = x.size(-1), t = step ? 1 : x.size(-2);
  const at::ScalarType type = x.scalar_type();
  same(dt, "dt", x, type);
  VALUE_CHECK(dt.sizes() == x.sizes(), "dt of shape ", dt.sizes(), " does not match x of shape ", x.sizes());
  same(a, "a", x, at::kFloat);
  VALUE_CHECK(a.dim() == 2 && a.size(0) == ch && a.size(1) >= 1, "a must have shape [", ch, ", N], got ", a.sizes());
  const int64_t n = a.size(1);
  if (n > INB_MAX_SCAN_N) refuse("selective_scan: N = ", n, " is above ", (int64_t)INB_MAX_SCAN_N);
  if (ch > INB_MAX_MEMORY_C || t > INB_MAX_MEMORY_S || sequences(x, lead) > INB_MAX_MEMORY_S ||
      sequences(x, lead) * ch > (1ll << 34))
    refuse("selective_scan: sizes of x ", x.sizes(), " are above its limits");
  const std::pair<const Tensor*, const char*> bc[] = {{&b, "b"}, {&c, "c"}};
  for (const auto& [p, name] : bc) {
    same(*p, name, x, type);
    if (step)
      check_shape(*p, name, x, lead, {n});
    else
      check_shape(*p, name, x, lead, {t, n});
  }
  const std::pair<const Tensor*, const char*> per[] = {{given(d), "d"}, {given(bias), "dt_bias"}};
  for (const auto& [p, name] : per)
    if (p != nullptr) {
      same(*p, name, x, at::kFloat);
      vector(*p, name, ch);
    }
  if (z) {
    same(*z, "z", x, type);
    VALUE_CHECK(z->sizes() == x.sizes(), "z of shape ", z->sizes(), " does not match x of shape ", x.sizes());
  }
  if (state) {
    same(*state, "state", x, at::kFloat);
    check_shape(*state, "state", x, lead, {ch, n});
  }
  if (reset) check_reset(*reset, x, lead, t, step);
  no_tangents({{&x, "x"}, {&dt, "dt"}, {&a, "a"}, {&b, "b"}, {&c, "c"}, {given(d), "d"}, {given(z), "z"}, {given(bias), "dt_bias"},
               {given(state), "state"}});
}
ScanIn scan_in(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& d, const Maybe& z,
               const Maybe& bias, const Maybe& state, const Maybe& reset) {
  auto flat = [](const Maybe& t) { return t ? t->contiguous() : Tensor(); };
  return {x, dt, a.contiguous(), b, c, flat(d), z.value_or(Tensor()), flat(bias), state.value_or(Tensor()), reset.value_or(Tensor())};
}
py::tuple selective_scan(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Maybe& d,
                         const Maybe& z, const Maybe& bias, const Maybe& state, const Maybe& reset) {
  scan_check(x, dt, a, b, c, d, z, bias, state, reset, false);
  const ScanIn i = scan_in(x, dt, a, b, c, d, z, bias, state, reset);
  if (any_grad({i.x, i.dt, i.a, i.b, i.c, i.d, i.z, i.bias, i.state})) {
    const variable_list o = SelectiveScan::apply(i.x, i.dt, i.a, i.b, i.c, maybe(i.d), maybe(i.z), maybe(i.bias), maybe(i.state),
                                                 maybe(i.reset));
    return py::make_tuple(o[0], o[1]);
  }
  auto [y, out, kept] = scan_forward(i, false);
  return py::make_tuple(y, out);
}
Tensor selective_scan_step(const Tensor& x, const Tensor& dt, const Tensor& a, const Tensor& b, const Tensor& c, const Tensor& state,
                           const Maybe& d, const Maybe& z, const Maybe& bias, const Maybe& reset) {
  scan_check(x, dt, a, b, c, d, z, bias, state, reset, true);
  check_in_place(state, "selective_scan_step");
  no_grad_step({x, dt, a, b, c, state, d.value_or(Tensor()), z.value_or(Tensor()), bias.value_or(Tensor())}, "selective_scan_step");
  const at::NoGradGuard no_grad;
  ScanIn i = scan_in(x, dt, a, b, c, d, z, bias, state, reset);
  i.step = true;
  const Tensor y = like_seq(x, true);
  if (x.numel() > 0) {
    const On on(x);
    const ScanRows r(i);
    InbScanArgs args = scan_args(i, r);
    args.y = write_seq(y, true);
    args.state_out = (float*)out(state), args.state_out_seq = r.st.seq;
    check(api.scan_fwd(&args, on.stream), "inb_selective_scan_fwd");
    touched(state);
  }
  return y;
}

// ------------------------------------------------------------------------------------------------- distill_loss
struct DistillIn {
  Tensor logits, teacher, index, mask;
  double tau;
};
struct DistillRows {
  Rows logits, mask;
  explicit DistillRows(const DistillIn& i) : logits(rows_of(i.logits, i.logits.size(-1))) {
    if (!i.mask.defined()) return;
    if (i.mask.dim() == 1 && i.logits.dim() > 1)
      mask = {i.mask.contiguous(), 0};
    else
      mask = rows_of(i.mask, i.mask.size(-1));
  }
};
InbDistillArgs distill_args(const DistillIn& i, const DistillRows& r, const Tensor& stats) {
  InbDistillArgs a = {};
  a.dtype = type_code(i.logits.scalar_type()), a.teacher_dtype = type_code(i.teacher.scalar_type());
  a.V = (int32_t)i.logits.size(-1), a.K = (int32_t)i.teacher.size(-1);
  a.N = i.logits.numel() / a.V;
  a.ld = r.logits.ld, a.ld_mask = r.mask.ld;
  a.logits = r.logits.p(), a.mask = (const uint8_t*)r.mask.p();
  a.teacher = ptr(i.teacher), a.index = (const int64_t*)ptr(i.index);
  a.tau = (float)i.tau;
  a.stats = (float*)out(stats);
  return a;
}
std::pair<Tensor, Tensor> distill_forward(const DistillIn& i, bool keep) {
  const Tensor loss = at::empty(i.logits.sizes().slice(0, i.logits.dim() - 1), i.logits.options().dtype(at::kFloat));
  Tensor stats;
  if (keep) stats = at::empty({loss.numel(), 4}, loss.options());
  if (loss.numel() > 0) {
    const On on(i.logits);
    const DistillRows r(i);
    InbDistillArgs a = distill_args(i, r, stats);
    a.loss = (float*)out(loss);
    check(api.distill_fwd(&a, on.stream), "inb_distill_fwd");
  }
  return {loss, stats};
}
struct DistillLoss : torch::autograd::Function<DistillLoss> {
  static Tensor forward(AutogradContext* ctx, Tensor logits, Tensor teacher, Tensor index, Maybe mask, double tau) {
    const DistillIn i = {logits, teacher, index, mask.value_or(Tensor()), tau};
    auto [loss, stats] = distill_forward(i, true);
    ctx->save_for_backward({logits, teacher, index, i.mask, stats});
    ctx->saved_data["t"] = tau;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const DistillIn i = {v[0], v[1], v[2], v[3], ctx->saved_data["t"].toDouble()};
    const Tensor g = at::empty(i.logits.sizes(), i.logits.options());
    if (g.numel() > 0) {
      const On on(i.logits);
      const DistillRows r(i);
      InbDistillArgs a = distill_args(i, r, v[4]);
      const Tensor gl = grads[0].contiguous();
      a.gloss = (const float*)ptr(gl), a.glogits = out(g);
      check(api.distill_bwd(&a, on.stream), "inb_distill_bwd");
    }
    return once({g, {}, {}, {}, {}});
  }
};
Tensor distill_loss(const Tensor& logits, const Tensor& teacher, const Tensor& index, double tau, const Maybe& mask) {
  first(logits, "logits");
  const int64_t v = width(logits, "logits"), n = logits.numel() / v;
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  if (v > INB_MAX_SAMPLE_V || n > INB_MAX_SAMPLE_N)
    refuse("distill_loss: ", n, " rows of ", v, ": at most ", (int64_t)INB_MAX_SAMPLE_N, " rows of ", (int64_t)INB_MAX_SAMPLE_V);
  first(teacher, "teacher");
  VALUE_CHECK(teacher.device() == logits.device(), "teacher is on ", teacher.device().str(), ", the first tensor on ",
              logits.device().str());
  VALUE_CHECK(teacher.dim() == logits.dim() && teacher.sizes().slice(0, lead.size()) == lead && teacher.size(-1) >= 1,
              "teacher must be [..., K] with the leading sizes of logits ", logits.sizes(), ", got ", teacher.sizes());
  if (teacher.size(-1) > INB_MAX_DISTILL_K) refuse("distill_loss: K = ", teacher.size(-1), " is above ", (int64_t)INB_MAX_DISTILL_K);
  same(index, "index", logits, at::kLong);
  VALUE_CHECK(index.sizes() == teacher.sizes(), "index of shape ", index.sizes(), " does not match teacher of shape ", teacher.sizes());
  VALUE_CHECK(tau >= 1e-6 && tau <= 1e6, "temperature = ", tau, " is out of range (1e-6 to 1e6)");
  if (mask) {
    same(*mask, "mask", logits, at::kBool);
    VALUE_CHECK((mask->dim() == 1 && mask->size(0) == v) || mask->sizes() == logits.sizes(), "mask must have shape ", logits.sizes(),
                " or [", v, "], got ", mask->sizes());
  }
  no_tangents({{&logits, "logits"}, {&teacher, "teacher"}});
  if (any_grad({teacher})) refuse("teacher requires a gradient: distill_loss differentiates the logits only (detach it)");
  const DistillIn i = {logits, teacher.contiguous(), index.contiguous(), mask.value_or(Tensor()), tau};
  if (any_grad({logits})) return DistillLoss::apply(i.logits, i.teacher, i.index, maybe(i.mask), tau);
  return distill_forward(i, false).first;
}

}  // namespace

void register_memory(py::module_& m) {
  m.def("bind_memory", &bind_memory);
  m.def("causal_conv", &causal_conv);
  m.def("causal_conv_step", &causal_conv_step);
  m.def("selective_scan", &selective_scan);
  m.def("selective_scan_step", &selective_scan_step);
  m.def("distill_loss", &distill_loss);
}
