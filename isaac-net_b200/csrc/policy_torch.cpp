// The policy operators on torch tensors (isaac-net_b200/policy_ops.py): argument checks, outputs, autograd, and the calls of
// the C ABI (include/isaac_net_b200.h).
//
// A serving call is a few microseconds of device time and a training step on a small batch some tens, less than Python
// needs to check the arguments and to run an autograd function; here a call costs the host two or three launches' time.
// The library's entry points are handed over as addresses by bind(), so the one that Python loaded is the one that runs.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <mutex>

#include "isaac_net_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

struct Api {
  int (*norm_fwd)(const InbNormArgs*, void*);
  int (*norm_bwd)(const InbNormArgs*, void*);
  int (*norm_work)(const InbNormArgs*, int64_t*);
  int (*ffn_fwd)(const InbFfnArgs*, void*);
  int (*ffn_bwd)(const InbFfnArgs*, void*);
  int (*ffn_work)(const InbFfnArgs*, int32_t, int64_t*);
  int (*dropout)(const InbDropoutArgs*, void*);
  int (*sample)(const InbSampleArgs*, void*);
} api;
PyObject* unsupported = nullptr;      // engine.B200Unsupported

void bind(const std::map<std::string, uintptr_t>& f, py::object error) {
  api.norm_fwd = reinterpret_cast<decltype(api.norm_fwd)>(f.at("inb_block_norm_fwd"));
  api.norm_bwd = reinterpret_cast<decltype(api.norm_bwd)>(f.at("inb_block_norm_bwd"));
  api.norm_work = reinterpret_cast<decltype(api.norm_work)>(f.at("inb_block_norm_work"));
  api.ffn_fwd = reinterpret_cast<decltype(api.ffn_fwd)>(f.at("inb_gated_ffn_fwd"));
  api.ffn_bwd = reinterpret_cast<decltype(api.ffn_bwd)>(f.at("inb_gated_ffn_bwd"));
  api.ffn_work = reinterpret_cast<decltype(api.ffn_work)>(f.at("inb_gated_ffn_work"));
  api.dropout = reinterpret_cast<decltype(api.dropout)>(f.at("inb_dropout"));
  api.sample = reinterpret_cast<decltype(api.sample)>(f.at("inb_sample"));
  unsupported = error.release().ptr();
}

// ------------------------------------------------------------------------------------------------- checks
// Messages are put together by hand: formatting a shape through torch's own operator<< crashed in libraries built here
// against the installed torch (a three-line extension shows it).
std::string text(const char* v) { return v; }
std::string text(const std::string& v) { return v; }
std::string text(int64_t v) { return std::to_string(v); }
std::string text(double v) { return std::to_string(v); }
std::string text(at::ScalarType v) { return c10::toString(v); }
std::string text(at::IntArrayRef v) {
  std::string s = "[";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + std::to_string(v[i]);
  return s + "]";
}
template <typename... A>
std::string join(const A&... a) {
  std::string s;
  ((s += text(a)), ...);
  return s;
}
// What the checks raise; called from Python only
template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  PyErr_SetString(unsupported, join(a...).c_str());
  throw py::error_already_set();
}
#define VALUE_CHECK(ok, ...) \
  if (!(ok)) throw py::value_error(join(__VA_ARGS__))

int type_code(at::ScalarType t) {
  return t == at::kBFloat16 ? INB_BF16 : t == at::kHalf ? INB_F16 : t == at::kFloat ? INB_F32 : -1;
}
void on_cuda(const Tensor& t, const char* name) {
  if (!t.is_cuda()) refuse(name, " is on ", t.device().str(), ": the policy operators run on CUDA tensors only");
}
// An operator's first tensor: on a CUDA device, of one of the operators' types
int first(const Tensor& x, const char* name, bool fp32 = true) {
  const int code = type_code(x.scalar_type());
  on_cuda(x, name);
  if (code < 0 || (code == INB_F32 && !fp32))
    refuse(name, " is ", x.scalar_type(), ": this operator takes bfloat16", fp32 ? ", float16 and float32" : " and float16");
  return code;
}
void same(const Tensor& t, const char* name, const Tensor& like, at::ScalarType want) {
  if (t.is_cuda() && t.get_device() == like.get_device() && t.scalar_type() == want) return;
  on_cuda(t, name);
  VALUE_CHECK(t.device() == like.device(), name, " is on ", t.device().str(), ", the first tensor on ", like.device().str());
  throw py::type_error(join(name, " is ", t.scalar_type(), ", expected ", want));
}
void vector(const Tensor& t, const char* name, int64_t n) {
  VALUE_CHECK(t.dim() == 1 && t.size(0) == n, name, " must have shape [", n, "], got ", t.sizes());
}
int64_t width(const Tensor& x, const char* name) {
  VALUE_CHECK(x.dim() >= 1 && x.size(-1) >= 1, name, " must be [..., D] with D >= 1, got shape ", x.sizes());
  return x.size(-1);
}

// [..., D] as rows of one stride; a copy where there is none, or where elements are not contiguous
struct Rows {
  Tensor t;
  int64_t ld = 0;
  const void* p() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
Rows rows_of(const Tensor& t, int64_t d, int64_t most = INT64_MAX) {
  if (!t.defined()) return {};
  if (t.is_contiguous()) return {t, d};
  bool one = t.stride(-1) == 1 || d == 1;
  int64_t ld = -1, next = 0;      // the rows' stride, and the stride that the next axis out has to have
  for (int64_t i = t.dim() - 2; one && i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (ld < 0)
      ld = t.stride(i);
    else
      one = t.stride(i) == next;
    next = t.stride(i) * t.size(i);
  }
  if (one && ld <= most) return {t, ld < 0 ? d : ld};
  return {t.contiguous(), d};
}
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
Tensor like(const Tensor& t) { return t.defined() ? at::empty(t.sizes(), t.options()) : Tensor(); }

// The current stream of a tensor's device, which is the current device while this lives
struct On {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.get_device()).stream()) {}
};
void check(int rc, const char* name) {
  if (rc != 0) throw std::runtime_error(join(name, " failed with status ", (int64_t)rc));
}

bool any_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}
// Forward-mode derivatives are not there: a tangent that came in would be lost, which reads as a zero derivative
void no_tangents(std::initializer_list<std::pair<const Tensor*, const char*>> ts) {
  for (const auto& [t, name] : ts)
    if (t != nullptr && t->_fw_grad(/*level=*/0).defined())
      refuse(name, " carries a tangent: the policy operators have no forward-mode derivatives");
}
const Tensor* given(const std::optional<Tensor>& t) { return t ? &*t : nullptr; }
// A backward pass's results, which cannot be differentiated again: an attempt raises
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (Tensor& g : grads)
    if (g.defined()) g = g.detach().requires_grad_(true);
  auto stop = std::make_shared<torch::autograd::DelayedError>("the policy operators can be differentiated once only",
                                                              (int64_t)grads.size());
  return (*stop)(std::move(grads));
}

// ------------------------------------------------------------------------------------------------- block_norm
struct NormIn {
  Tensor x, w, h, post, gate;
  int64_t rows;
  double scale, eps;
};
InbNormArgs norm_args(const NormIn& i, const Rows& x, const Rows& h) {
  InbNormArgs a = {};
  a.dtype = type_code(i.x.scalar_type());
  a.D = (int32_t)i.x.size(-1);
  a.N = i.x.numel() / a.D;
  a.ldx = x.ld, a.ldh = h.ld;
  a.gate_rows = i.rows;
  a.scale = (float)i.scale, a.eps = (float)i.eps;
  a.x = x.p(), a.h = h.p();
  a.w = ptr(i.w), a.post = ptr(i.post), a.gate = ptr(i.gate);
  return a;
}
std::pair<Tensor, Tensor> norm_forward(const NormIn& i, const Tensor& stats) {
  Tensor y = i.h.defined() ? like(i.x) : Tensor(), n = like(i.x);
  if (i.x.numel() > 0) {
    const On on(i.x);
    const Rows x = rows_of(i.x, i.x.size(-1), INB_MAX_NORM_LD), h = rows_of(i.h, i.x.size(-1), INB_MAX_NORM_LD);
    InbNormArgs a = norm_args(i, x, h);
    a.y = out(y), a.n = out(n), a.stats = (float*)out(stats);
    check(api.norm_fwd(&a, on.stream), "inb_block_norm_fwd");
  }
  return {y, n};
}
struct BlockNorm : torch::autograd::Function<BlockNorm> {
  using Maybe = std::optional<Tensor>;
  static variable_list forward(AutogradContext* ctx, Tensor x, Tensor w, Maybe h_in, Maybe post_in, Maybe gate_in,
                               int64_t rows, double scale, double eps) {
    const Tensor h = h_in.value_or(Tensor()), post = post_in.value_or(Tensor()), gate = gate_in.value_or(Tensor());
    const NormIn i = {x, w, h, post, gate, rows, scale, eps};
    Tensor stats = at::empty({x.numel() / x.size(-1), 2}, x.options().dtype(at::kFloat));
    auto [y, n] = norm_forward(i, stats);
    ctx->save_for_backward({x, w, h, post, gate, stats});
    ctx->saved_data["s"] = c10::List<double>({(double)rows, scale, eps});
    ctx->set_materialize_grads(false);
    return y.defined() ? variable_list{y, n} : variable_list{n};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const auto s = ctx->saved_data["s"].toDoubleList();
    const NormIn i = {v[0], v[1], v[2], v[3], v[4], (int64_t)s.get(0), s.get(1), s.get(2)};
    const Tensor gy = grads.size() == 2 ? grads[0] : Tensor(), gn = grads.back();
    variable_list o = {like(i.x), like(i.w), like(i.h), like(i.post), like(i.gate), {}, {}, {}};
    if ((!gy.defined() && !gn.defined()) || i.x.numel() == 0) {
      for (Tensor& t : o)
        if (t.defined()) t.zero_();
      return once(o);
    }
    const On on(i.x);
    const int64_t d = i.x.size(-1);
    const Rows x = rows_of(i.x, d, INB_MAX_NORM_LD), h = rows_of(i.h, d, INB_MAX_NORM_LD),
               y = rows_of(gy, d, INB_MAX_NORM_LD), n = rows_of(gn, d, INB_MAX_NORM_LD);
    InbNormArgs a = norm_args(i, x, h);
    a.ldgy = y.ld, a.ldgn = n.ld;
    a.gy = y.p(), a.gn = n.p();
    a.stats = (float*)out(v[5]);
    a.gx = out(o[0]), a.gw = out(o[1]), a.gh = out(o[2]), a.gpost = out(o[3]), a.ggate = out(o[4]);
    check(api.norm_work(&a, &a.work_elems), "inb_block_norm_work");
    const Tensor work = at::empty({a.work_elems}, i.x.options().dtype(at::kFloat));
    a.work = (float*)out(work);
    check(api.norm_bwd(&a, on.stream), "inb_block_norm_bwd");
    return once(o);
  }
};

// How many consecutive rows of x [..., D] one gate scales: gate's leading sizes equal x's up to some axis and are 1 from
// there on (missing ones count as 1)
int64_t gate_rows(const Tensor& gate, const Tensor& x) {
  const int64_t dims = x.dim(), miss = dims - gate.dim();
  auto size = [&](int64_t i) { return i < miss ? 1 : gate.size(i - miss); };
  int64_t rows = 1, axis = dims - 2;
  bool fits = miss >= 0 && size(dims - 1) == x.size(-1);
  if (fits)
    for (; axis >= 0 && size(axis) == 1; --axis) rows *= x.size(axis);
  for (; fits && axis >= 0; --axis) fits = size(axis) == x.size(axis);
  VALUE_CHECK(fits, "gate of shape ", gate.sizes(), " does not fit x of shape ", x.sizes(),
                    ": [..., D] with x's leading sizes, then ones");
  return rows;
}

py::object block_norm(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& h,
                      const std::optional<Tensor>& post, const std::optional<Tensor>& gate, double scale, double eps) {
  first(x, "x");
  const int64_t d = width(x, "x");
  no_tangents({{&x, "x"}, {&weight, "weight"}, {given(h), "h"}, {given(post), "post_weight"}, {given(gate), "gate"}});
  if (d > INB_MAX_NORM_D) refuse("block_norm: D = ", d, " is above ", (int64_t)INB_MAX_NORM_D);
  if (x.numel() / d > INT32_MAX) refuse("block_norm: more than 2^31 - 1 rows");
  const at::ScalarType t = x.scalar_type();
  same(weight, "weight", x, t);
  vector(weight, "weight", d);
  NormIn i = {x, weight.contiguous(), {}, {}, {}, 0, scale, eps};
  if (!h) {
    VALUE_CHECK(!post && !gate, "post_weight and gate need h");
  } else {
    same(*h, "h", x, t);
    VALUE_CHECK(h->sizes() == x.sizes(), "h of shape ", h->sizes(), " does not match x of shape ", x.sizes());
    i.h = *h;
    if (post) {
      same(*post, "post_weight", x, t);
      vector(*post, "post_weight", d);
      i.post = post->contiguous();
    }
    if (gate) {
      same(*gate, "gate", x, t);
      i.rows = gate_rows(*gate, x);
      i.gate = gate->contiguous();
    }
  }
  Tensor y, n;
  if (any_grad({i.x, i.w, i.h, i.post, i.gate})) {
    auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
    const variable_list o = BlockNorm::apply(i.x, i.w, maybe(i.h), maybe(i.post), maybe(i.gate), i.rows, scale, eps);
    n = o.back();
    if (h) y = o[0];
  } else {
    std::tie(y, n) = norm_forward(i, Tensor());
  }
  return h ? py::cast(std::make_tuple(y, n)) : py::cast(n);
}

// ------------------------------------------------------------------------------------------------- gated_ffn
std::mutex status_lock;
Tensor status_words[64];
// The device's status word.  The first call makes it on a stream of its own and waits for that: so it is zero before any
// stream's kernels see it, and where that call is captured in a graph neither its memory nor its zeroing is part of the graph.
int32_t* status_word(const Tensor& like) {
  const std::lock_guard<std::mutex> hold(status_lock);
  Tensor& w = status_words[like.get_device() & 63];
  if (!w.defined()) {
    const c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
    auto side = [&] { return c10::cuda::getStreamFromPool(false, like.get_device()); };
    c10::cuda::CUDAStreamGuard on(side());
    // torch hands out 32 streams in turn: this one may be the one that is captured
    for (int i = 0; i < 32 && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None; ++i)
      on.reset_stream(side());
    w = at::zeros({1}, like.options().dtype(at::kInt));
    on.current_stream().synchronize();
  }
  return (int32_t*)out(w);
}
int64_t status(int64_t device) {
  Tensor w;
  {
    const std::lock_guard<std::mutex> hold(status_lock);
    w = status_words[device & 63];
  }
  if (!w.defined()) return 0;
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
  c10::cuda::device_synchronize();         // the operators may run on any stream
  return w.item<int32_t>();
}

struct FfnIn {
  Tensor x, wg, wu, wd;
  int64_t act;
};
struct FfnRows {
  Rows x, wg, wu, wd;
  explicit FfnRows(const FfnIn& i)
      : x(rows_of(i.x, i.x.size(-1))), wg(rows_of(i.wg, i.wg.size(1))), wu(rows_of(i.wu, i.wu.size(1))),
        wd(rows_of(i.wd, i.wd.size(1))) {}
};
InbFfnArgs ffn_args(const FfnIn& i, const FfnRows& r, int64_t ldh) {
  InbFfnArgs a = {};
  a.dtype = type_code(i.x.scalar_type());
  a.act = (int32_t)i.act;
  a.D = (int32_t)i.x.size(-1);
  a.F = (int32_t)i.wg.size(0);
  a.N = i.x.numel() / a.D;
  a.ldx = r.x.ld, a.ldwg = r.wg.ld, a.ldwu = r.wu.ld, a.ldwd = r.wd.ld, a.ldh = ldh;
  a.x = r.x.p(), a.wg = r.wg.p(), a.wu = r.wu.p(), a.wd = r.wd.p();
  a.status = status_word(i.x);
  return a;
}
Tensor ffn_work(InbFfnArgs& a, bool backward, const Tensor& like) {
  check(api.ffn_work(&a, backward, &a.work_bytes), "inb_gated_ffn_work");
  if (a.work_bytes == 0) return {};
  Tensor w = at::empty({a.work_bytes}, like.options().dtype(at::kByte));
  a.work = out(w);
  return w;
}
// y, and what a backward pass needs: h [n, ldh], and g and u as [2, bytes of one]
std::tuple<Tensor, Tensor, Tensor> ffn_forward(const FfnIn& i, bool keep) {
  const int64_t n = i.x.numel() / i.x.size(-1), ldh = (i.wg.size(0) + 7) / 8 * 8;
  Tensor y = like(i.x), h = at::empty({!keep && n <= INB_FFN_ROWS ? 2 * n : n, ldh}, i.x.options()), gu;
  if (keep) gu = at::empty({2, (n + 127) / 128 * 128 * ((ldh + 15) / 16 * 48)}, i.x.options().dtype(at::kByte));
  if (n > 0) {
    const On on(i.x);
    const FfnRows r(i);
    InbFfnArgs a = ffn_args(i, r, ldh);
    a.y = out(y), a.h = out(h);
    if (keep) a.g = out(gu), a.u = (char*)a.g + gu.size(1);
    const Tensor work = ffn_work(a, false, i.x);
    check(api.ffn_fwd(&a, on.stream), "inb_gated_ffn_fwd");
  }
  return {y, h, gu};
}
struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor wg, Tensor wu, Tensor wd, int64_t act) {
    auto [y, h, gu] = ffn_forward({x, wg, wu, wd, act}, true);
    ctx->save_for_backward({x, wg, wu, wd, h, gu});
    ctx->saved_data["a"] = act;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list v = ctx->get_saved_variables();
    const FfnIn i = {v[0], v[1], v[2], v[3], ctx->saved_data["a"].toInt()};
    const Tensor &h = v[4], &gu = v[5];
    bool need[4];
    for (int k = 0; k < 4; ++k) need[k] = ctx->needs_input_grad(k);
    const bool gate = need[1] || need[2];
    variable_list o = {need[0] ? like(i.x) : Tensor(), gate ? like(i.wg) : Tensor(), gate ? like(i.wu) : Tensor(),
                       need[3] ? like(i.wd) : Tensor(), {}};
    if (i.x.numel() == 0) {
      for (Tensor& t : o)
        if (t.defined()) t.zero_();
      return once(o);
    }
    const On on(i.x);
    const FfnRows r(i);
    InbFfnArgs a = ffn_args(i, r, h.size(1));
    const Rows dy = rows_of(grads[0], i.x.size(-1));
    a.dy = dy.p(), a.lddy = dy.ld;
    a.h = out(h), a.g = out(gu), a.u = (char*)a.g + gu.size(1);
    a.dx = out(o[0]), a.dwg = out(o[1]), a.dwu = out(o[2]), a.dwd = out(o[3]);
    Tensor dh;
    if (need[0] || gate) {
      dh = at::empty({2, h.size(0), h.size(1)}, h.options());
      a.dg = out(dh), a.du = (char*)a.dg + h.numel() * h.element_size();
    }
    const Tensor work = ffn_work(a, true, i.x);
    check(api.ffn_bwd(&a, on.stream), "inb_gated_ffn_bwd");
    if (!need[1]) o[1] = Tensor();
    if (!need[2]) o[2] = Tensor();
    return once(o);
  }
};
Tensor gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
  first(x, "x", false);
  const int64_t d = width(x, "x");
  const at::ScalarType t = x.scalar_type();
  same(wg, "w_gate", x, t);
  same(wu, "w_up", x, t);
  same(wd, "w_down", x, t);
  const int64_t f = wg.dim() == 2 ? wg.size(0) : 0;
  auto shaped = [](const Tensor& m, int64_t r, int64_t c) { return m.dim() == 2 && m.size(0) == r && m.size(1) == c; };
  VALUE_CHECK(f >= 1 && shaped(wg, f, d) && shaped(wu, f, d) && shaped(wd, d, f), "w_gate and w_up must be [F, ", d,
                    "] and w_down [", d, ", F], got ", wg.sizes(), ", ", wu.sizes(), ", ", wd.sizes());
  if (d > INB_MAX_FFN || f > INB_MAX_FFN || x.numel() / d > INB_MAX_FFN) refuse("gated_ffn: sizes above ", (int64_t)INB_MAX_FFN);
  no_tangents({{&x, "x"}, {&wg, "w_gate"}, {&wu, "w_up"}, {&wd, "w_down"}});
  if (any_grad({x, wg, wu, wd})) return GatedFfn::apply(x, wg, wu, wd, act);
  return std::get<0>(ffn_forward({x, wg, wu, wd, act}, false));
}

// ------------------------------------------------------------------------------------------------- counter_dropout
// keys [E] is written (made from env_id, episode, ctr) or, without env_id, read
Tensor dropout_run(const Tensor& x_in, int64_t threshold, int64_t s0, int64_t stream, const Tensor& env_id,
                   const Tensor& episode, const Tensor& ctr, const Tensor& keys) {
  const Tensor x = x_in.contiguous(), y = like(x);
  if (x.numel() == 0) return y;
  const On on(x);
  InbDropoutArgs a = {};
  a.dtype = type_code(x.scalar_type());
  a.threshold = (uint32_t)threshold;
  a.E = x.size(0), a.n = x.numel() / a.E;
  a.s0 = (uint32_t)s0, a.stream = (uint32_t)stream;
  a.env_id = (const int64_t*)ptr(env_id), a.episode = (const int64_t*)ptr(episode), a.ctr = (const int64_t*)ptr(ctr);
  if (env_id.defined())
    a.keys_out = (uint32_t*)out(keys);
  else
    a.keys_in = (const uint32_t*)ptr(keys);
  a.x = ptr(x), a.y = out(y);
  check(api.dropout(&a, on.stream), "inb_dropout");
  return y;
}
struct Dropout : torch::autograd::Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, Tensor x, int64_t threshold, int64_t s0, int64_t stream, Tensor env_id,
                        std::optional<Tensor> episode_in, std::optional<Tensor> ctr_in) {
    const Tensor episode = episode_in.value_or(Tensor()), ctr = ctr_in.value_or(Tensor());
    const Tensor keys = at::empty({x.size(0)}, x.options().dtype(at::kInt));
    ctx->save_for_backward({keys});
    ctx->saved_data["t"] = threshold;
    return dropout_run(x, threshold, s0, stream, env_id, episode, ctr, keys);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor keys = ctx->get_saved_variables()[0];
    variable_list o(7);
    o[0] = dropout_run(grads[0], ctx->saved_data["t"].toInt(), 0, 0, {}, {}, {}, keys);
    return once(o);
  }
};
Tensor counter_dropout(const Tensor& x, double p, int64_t s0, const Tensor& env_id, const std::optional<Tensor>& episode,
                       const std::optional<Tensor>& ctr, int64_t stream) {
  first(x, "x");
  VALUE_CHECK(x.dim() >= 1, "x must be [E, ...]");
  no_tangents({{&x, "x"}});
  VALUE_CHECK(p >= 0.0 && p <= 1.0, "p must be in [0, 1], got ", p);
  VALUE_CHECK(s0 >= 0 && s0 <= UINT32_MAX && stream >= 0 && stream <= UINT32_MAX, "s0 and stream are 32-bit words");
  const int64_t e = x.size(0), n = e > 0 ? x.numel() / e : 0;
  Tensor ids[3];
  const std::optional<Tensor> in[3] = {env_id, episode, ctr};
  const char* names[3] = {"env_id", "episode", "ctr"};
  for (int i = 0; i < 3; ++i)
    if (in[i]) {
      same(*in[i], names[i], x, at::kLong);
      vector(*in[i], names[i], e);
      ids[i] = in[i]->contiguous();
    }
  if (n > 0x1FFFFFFFFll || e * std::max<int64_t>(1, (n + 4095) / 4096) > INT32_MAX)
    refuse("counter_dropout: ", e, " envs of ", n, " elements are more than one call can draw");
  const int64_t threshold = std::llround(p * 65536);
  auto maybe = [](const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  if (any_grad({x})) return Dropout::apply(x, threshold, s0, stream, ids[0], maybe(ids[1]), maybe(ids[2]));
  return dropout_run(x, threshold, s0, stream, ids[0], ids[1], ids[2], Tensor());
}

// ------------------------------------------------------------------------------------------------- sample_logits
// A setting that is a number or a tensor of one per row
template <typename V>
struct Setting {
  V value = 0;
  Tensor rows;
  Setting(const py::handle& v, const char* name, const Tensor& logits, at::IntArrayRef lead, at::ScalarType type) {
    if (THPVariable_Check(v.ptr())) {
      rows = THPVariable_Unpack(v.ptr());
      same(rows, name, logits, type);
      VALUE_CHECK(rows.sizes() == lead, name, " must be a number or have shape ", lead, ", got ", rows.sizes());
      rows = rows.contiguous();
      return;
    }
    const double d = PyFloat_AsDouble(v.ptr());
    if (d == -1.0 && PyErr_Occurred()) throw py::error_already_set();      // a TypeError
    const bool whole = std::is_integral<V>::value;
    VALUE_CHECK(d >= 0 && (!whole || d == std::floor(d)), name, " = ", d, " is out of range");
    value = whole ? (V)std::min(d, 2147483647.0) : (V)d;
  }
  const V* p() const { return rows.defined() ? (const V*)rows.const_data_ptr() : nullptr; }
};
py::tuple sample_logits(const Tensor& logits, const Tensor& u, const py::object& temperature, const py::object& top_k,
                        const py::object& top_p, const py::object& min_p, const std::optional<Tensor>& mask) {
  const int code = first(logits, "logits");
  no_tangents({{&logits, "logits"}});
  const int64_t v = width(logits, "logits"), n = logits.numel() / v;
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  if (v > INB_MAX_SAMPLE_V || n > INB_MAX_SAMPLE_N)
    refuse("sample_logits: ", n, " rows of ", v, ": at most ", (int64_t)INB_MAX_SAMPLE_N, " rows of ",
           (int64_t)INB_MAX_SAMPLE_V);
  same(u, "u", logits, at::kFloat);
  VALUE_CHECK(u.sizes() == lead, "u must have shape ", lead, ", got ", u.sizes());
  const Setting<float> t(temperature, "temperature", logits, lead, at::kFloat), p(top_p, "top_p", logits, lead, at::kFloat),
      m(min_p, "min_p", logits, lead, at::kFloat);
  const Setting<int32_t> k(top_k, "top_k", logits, lead, at::kInt);
  VALUE_CHECK(m.value <= 1.f, "min_p = ", (double)m.value, " is out of range");
  const at::NoGradGuard no_grad;
  Rows allowed;
  if (mask) {
    same(*mask, "mask", logits, at::kBool);
    const bool one = mask->dim() == 1 && mask->size(0) == v;
    VALUE_CHECK(one || mask->sizes() == logits.sizes(), "mask must have shape ", logits.sizes(), " or [", v, "], got ",
                      mask->sizes());
    if (one && logits.dim() > 1)
      allowed = {mask->contiguous(), 0};
    else
      allowed = rows_of(*mask, v);
  }
  const Tensor token = at::empty(lead, u.options().dtype(at::kLong)), logp = at::empty(lead, u.options());
  if (n > 0) {
    const On on(logits);
    const Rows l = rows_of(logits, v);
    const Tensor uc = u.contiguous();
    InbSampleArgs a = {};
    a.dtype = code, a.V = (int32_t)v, a.N = n;
    a.ld = l.ld, a.ld_mask = allowed.ld;
    a.logits = l.p(), a.mask = (const uint8_t*)allowed.p(), a.u = (const float*)ptr(uc);
    a.temperature = t.value, a.top_p = p.value, a.min_p = m.value, a.top_k = k.value;
    a.temperature_row = t.p(), a.top_p_row = p.p(), a.min_p_row = m.p(), a.top_k_row = k.p();
    a.token = (int64_t*)out(token), a.logp = (float*)out(logp);
    check(api.sample(&a, on.stream), "inb_sample");
  }
  return py::make_tuple(token, logp);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("status", &status);
  m.def("block_norm", &block_norm);
  m.def("gated_ffn", &gated_ffn);
  m.def("counter_dropout", &counter_dropout);
  m.def("sample_logits", &sample_logits);
}
