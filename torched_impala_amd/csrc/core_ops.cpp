// Host side of the operators of the linear-attention core and of its
// matrices' updates: argument checks that keep the kernels in bounds, output
// and workspace tensors (torch's allocator, so a captured graph owns its
// own), launches on the current stream of the operands' device.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <memory>
#include <tuple>
#include <vector>

#include "attn_kernels.h"
#include "core_ops.h"
#include "ortho_kernels.h"

extern "C" {
long layer_norm_part_elems(int, long, long, int);
int layer_norm_aligned(int, const void*, const void*, long, const void*,
                       const void*, long);
void launch_layer_norm_fwd(int, int, const void*, long, const void*,
                           const void*, void*, float*, float*, long, long,
                           float, hipStream_t);
void launch_layer_norm_bwd(int, int, int, const void*, const void*, long,
                           const void*, const float*, const float*, void*,
                           float*, void*, void*, long, long, hipStream_t);
void launch_attn_chunks(int, const impala::attn::AttnArgs*, int, int,
                        hipStream_t);
void launch_attn_scan(float*, const float*, const float*, const float*, long,
                      int, long, long, int, int, long, long, hipStream_t);
void launch_attn_step(int, const impala::attn::AttnStepArgs*, int,
                      hipStream_t);
void launch_ns_start(impala::ortho::Args*, hipStream_t);
void launch_ns_product(int, int, const impala::ortho::Args*, hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": ", hipGetErrorString(e));
}

hipStream_t stream_here() {
  return c10::hip::getCurrentHIPStream().stream();
}

int type_code(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case torch::kFloat32: return 0;
    case torch::kBFloat16: return 1;
    case torch::kFloat16: return 2;
    default:
      TORCH_CHECK(false, name, " must be fp32, bf16 or fp16");
  }
}

Tensor or_undefined(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }

const void* ptr(const Tensor& t) {
  return t.defined() ? t.data_ptr() : nullptr;
}

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!torch::GradMode::is_enabled()) return false;
  for (const Tensor& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

// the kernels compute no forward-mode derivatives: a tangent is refused, not
// dropped
void refuse_tangents(const char* op, std::initializer_list<Tensor> ts) {
  for (const Tensor& t : ts)
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(), op,
                " has no forward-mode derivative");
}

// gradients of operators that are differentiable once: a second
// differentiation raises instead of taking them for constants
variable_list once(variable_list grads, const char* what) {
  if (!torch::GradMode::is_enabled()) return grads;
  variable_list in;
  for (const Tensor& t : grads)
    if (t.defined()) in.push_back(t.detach().requires_grad_());
  auto stop = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " is differentiable once", (int64_t)in.size());
  const variable_list out = (*stop)(variable_list(in));
  size_t k = 0;
  for (Tensor& t : grads)
    if (t.defined()) t = out[k++];
  return grads;
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------
void check_norm(const Tensor& x, const Tensor& w, const Tensor& b,
                double eps) {
  TORCH_CHECK_TYPE(x.scalar_type() == torch::kFloat32 ||
                       x.scalar_type() == torch::kBFloat16 ||
                       x.scalar_type() == torch::kFloat16,
                   "layer_norm: x must be fp32, bf16 or fp16, not ",
                   x.scalar_type());
  TORCH_CHECK_VALUE(x.is_cuda() && x.dim() >= 1 && x.size(-1) >= 1,
                    "layer_norm: x needs a last axis of one or more");
  for (const Tensor* t : {&w, &b}) {
    if (!t->defined()) continue;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1) &&
                          t->device() == x.device(),
                      "layer_norm: weight and bias must be (", x.size(-1),
                      ",) on x's device");
    TORCH_CHECK_TYPE(t->scalar_type() == torch::kFloat32 ||
                         t->scalar_type() == x.scalar_type(),
                     "layer_norm: weight and bias must be fp32 or of x's "
                     "type");
  }
  TORCH_CHECK_TYPE(!w.defined() || !b.defined() ||
                       w.scalar_type() == b.scalar_type(),
                   "layer_norm: weight and bias must have one type");
  TORCH_CHECK_VALUE(std::isfinite(eps) && eps >= 0.0,
                    "layer_norm: eps must be finite and >= 0, not ", eps);
}

// (rows, cols) with unit column stride: a view where strides allow
Tensor norm_rows(const Tensor& x) {
  Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
  return r.size(1) > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}

Tensor dense(const Tensor& t) { return t.defined() ? t.contiguous() : t; }

// y and, if `save`, the rows' mean and rstd
Tensor norm_fwd(const Tensor& x, const Tensor& w, const Tensor& b, double eps,
                bool save, Tensor* stats) {
  const c10::DeviceGuard guard(x.device());
  const Tensor xr = norm_rows(x), wc = dense(w), bc = dense(b);
  const int xt = type_code(x, "x");
  const int wt = w.defined() ? type_code(w, "weight")
                 : b.defined() ? type_code(b, "bias") : xt;
  const long rows = xr.size(0), cols = xr.size(1);
  Tensor y = torch::empty(x.sizes(), x.options());
  float* mean = nullptr;
  if (save) {
    *stats = torch::empty({2, rows}, x.options().dtype(torch::kFloat32));
    mean = stats->data_ptr<float>();
  }
  if (rows > 0) {
    launch_layer_norm_fwd(xt, wt, xr.data_ptr(), xr.stride(0), ptr(wc),
                          ptr(bc), y.data_ptr(), mean,
                          save ? mean + rows : nullptr, rows, cols,
                          (float)eps, stream_here());
    check_launch("layer_norm");
  }
  return y;
}

class LayerNorm : public torch::autograd::Function<LayerNorm> {
 public:
  static Tensor forward(AutogradContext* ctx, Tensor x, OptTensor weight,
                        OptTensor bias, double eps) {
    const Tensor w = or_undefined(weight), b = or_undefined(bias);
    Tensor stats;
    Tensor y = norm_fwd(x, w, b, eps, true, &stats);
    // x itself, not its 2-D view, so that a change of it in place is caught
    ctx->save_for_backward({x, w, stats});
    ctx->saved_data["dx"] = x.requires_grad();
    ctx->saved_data["dw"] = w.defined() && w.requires_grad();
    ctx->saved_data["db"] = b.defined() && b.requires_grad();
    ctx->saved_data["type"] =
        (int64_t)(w.defined() ? w : b.defined() ? b : x).scalar_type();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
    const bool need_dx = ctx->saved_data["dx"].toBool();
    const bool need_dw = ctx->saved_data["dw"].toBool();
    const bool need_db = ctx->saved_data["db"].toBool();
    const auto ptype = (torch::ScalarType)ctx->saved_data["type"].toInt();
    const c10::DeviceGuard guard(x.device());
    const Tensor xr = norm_rows(x), wc = dense(w);
    const Tensor dy = g[0].contiguous();
    const long rows = xr.size(0), cols = xr.size(1);
    const int xt = type_code(x, "x");
    const int wt = ptype == torch::kFloat32 ? 0 : xt;
    const auto popts = x.options().dtype(ptype);
    Tensor dx, dw, db;
    if (need_dx) dx = torch::empty(x.sizes(), x.options());
    if (need_dw) dw = rows ? torch::empty({cols}, popts)
                           : torch::zeros({cols}, popts);
    if (need_db) db = rows ? torch::empty({cols}, popts)
                           : torch::zeros({cols}, popts);
    if (rows > 0) {
      const int al = layer_norm_aligned(xt, dy.data_ptr(), xr.data_ptr(),
                                        xr.stride(0), ptr(wc), ptr(dx), cols);
      Tensor part;
      if (need_dw || need_db)
        part = torch::empty({layer_norm_part_elems(xt, rows, cols, al)},
                            x.options().dtype(torch::kFloat32));
      launch_layer_norm_bwd(
          xt, wt, al, dy.data_ptr(), xr.data_ptr(), xr.stride(0), ptr(wc),
          stats.data_ptr<float>(), stats.data_ptr<float>() + rows,
          const_cast<void*>(ptr(dx)),
          part.defined() ? part.data_ptr<float>() : nullptr,
          const_cast<void*>(ptr(dw)), const_cast<void*>(ptr(db)), rows, cols,
          stream_here());
      check_launch("layer_norm backward");
    }
    return once({dx, dw, db, Tensor()}, "layer_norm");
  }
};

Tensor layer_norm(Tensor x, OptTensor weight, OptTensor bias, double eps) {
  const Tensor w = or_undefined(weight), b = or_undefined(bias);
  check_norm(x, w, b, eps);
  refuse_tangents("layer_norm", {x, w, b});
  if (wants_grad({x, w, b}))
    return LayerNorm::apply(x, weight, bias, eps);
  return norm_fwd(x, w, b, eps, false, nullptr);
}

// ---------------------------------------------------------------------------
// linear attention. q, k (T, B, H, dk), v (T, B, H, dv) with unit stride on
// the last axis, one type; states (B, H, dk, dv) fp32, contiguous
// ---------------------------------------------------------------------------
using impala::attn::AttnArgs;
using impala::attn::AttnOperand;
using impala::attn::AttnRole;
using impala::attn::AttnStepArgs;

constexpr long MAX_HEAD = 128;   // the largest tile that the kernels have
// heads of a batch: a launch has at most 2^32 threads, 512 to a head in each
// of three roles (a step's 256 are fewer)
constexpr long MAX_HEADS = ((1L << 32) - 1) / (3 * 512);

struct AttnShape {
  long T, B, H, dk, dv;
};

// a head's features side by side; every other stride is free
Tensor unit(const Tensor& t) {
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

AttnShape check_attn(const char* op, const Tensor& q, const Tensor& k,
                     const Tensor& v, const Tensor& g, const Tensor& done,
                     const Tensor& state, int lead) {
  TORCH_CHECK_TYPE(q.scalar_type() == torch::kFloat32 ||
                       q.scalar_type() == torch::kBFloat16 ||
                       q.scalar_type() == torch::kFloat16,
                   op, ": q must be fp32, bf16 or fp16, not ",
                   q.scalar_type());
  TORCH_CHECK_TYPE(k.scalar_type() == q.scalar_type() &&
                       v.scalar_type() == q.scalar_type(),
                   op, ": q, k and v must have one type");
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device() &&
                        v.device() == q.device(),
                    op, ": q, k and v must be on one device");
  TORCH_CHECK_VALUE(q.dim() == lead + 2, op, ": q must have ", lead + 2,
                    " axes, not ", q.dim());
  TORCH_CHECK_VALUE(k.sizes() == q.sizes(), op, ": k is ", k.sizes(), ", q ",
                    q.sizes());
  TORCH_CHECK_VALUE(
      v.dim() == q.dim() &&
          v.sizes().slice(0, lead + 1) == q.sizes().slice(0, lead + 1),
      op, ": v is ", v.sizes(), ", q ", q.sizes());
  const AttnShape s{lead == 2 ? q.size(0) : 1, q.size(lead - 1),
                    q.size(lead), q.size(-1), v.size(-1)};
  TORCH_CHECK_VALUE(
      s.dk >= 1 && s.dk <= MAX_HEAD && s.dv >= 1 && s.dv <= MAX_HEAD, op,
      ": head sizes must be 1 to ", MAX_HEAD, ", not ", s.dk, " and ", s.dv);
  TORCH_CHECK_VALUE(s.B == 0 || s.H <= MAX_HEADS / s.B, op,
                    ": batch times heads must be at most ", MAX_HEADS);
  TORCH_CHECK_TYPE(g.scalar_type() == torch::kFloat32, op,
                   ": log_decay must be fp32, not ", g.scalar_type());
  TORCH_CHECK_VALUE(g.device() == q.device() && g.dim() == 1 &&
                        g.size(0) == s.H,
                    op, ": log_decay must be (", s.H, ",) on q's device");
  TORCH_CHECK_VALUE(!g.requires_grad(), op,
                    ": log_decay is a head's fixed slope and gets no "
                    "gradient; pass it detached");
  if (done.defined()) {
    TORCH_CHECK_TYPE(done.scalar_type() == torch::kBool, op,
                     ": done must be bool, not ", done.scalar_type());
    TORCH_CHECK_VALUE(done.device() == q.device() &&
                          done.sizes() == q.sizes().slice(0, lead),
                      op, ": done must be ", q.sizes().slice(0, lead),
                      " on q's device");
  }
  if (state.defined()) {
    TORCH_CHECK_TYPE(state.scalar_type() == torch::kFloat32, op,
                     ": the state must be fp32, not ", state.scalar_type());
    TORCH_CHECK_VALUE(state.device() == q.device() && state.dim() == 4 &&
                          state.size(0) == s.B && state.size(1) == s.H &&
                          state.size(2) == s.dk && state.size(3) == s.dv,
                      op, ": the state must be (B, H, dk, dv) on q's device, "
                      "not ", state.sizes());
  }
  return s;
}

double scale_of(const char* op, c10::optional<double> scale,
                const AttnShape& s) {
  if (!scale.has_value()) return 1.0 / std::sqrt((double)s.dk);
  TORCH_CHECK_VALUE(std::isfinite(*scale), op, ": scale must be finite");
  return *scale;
}

AttnOperand operand(const Tensor& t, int lead) {
  // the stride of an axis of one does not matter and may be anything
  auto st = [&](int i) { return t.size(i) == 1 ? 0L : (long)t.stride(i); };
  return AttnOperand{t.data_ptr(), lead == 2 ? st(0) : 0L, st(lead - 1),
                     st(lead)};
}

// 16-byte loads: base, strides and row length are multiples of 16 bytes, and
// 64 steps lie within 32 bits of offsets
bool can_vec(const Tensor& t, const AttnOperand& o) {
  const long es = t.element_size();
  const long dense = t.size(1) * t.size(2) * t.size(-1);   // of a result
  if (64 * es * std::max(std::abs(o.st), dense) >= (1L << 31)) return false;
  return ((uintptr_t)o.p & 15) == 0 && (o.st * es) % 16 == 0 &&
         (o.sb * es) % 16 == 0 && (o.sh * es) % 16 == 0 &&
         (t.size(-1) * es) % 16 == 0;
}

// Segments that a sequence is cut into. Workgroups that run at once: what a
// CU holds of the kernel's tiles (one of those for heads above 64, whose LDS
// or registers fill it, else two, or four of the small ones of bf16 and of fp16
// up to heads of 32; fp16, T=4096, B=4, 8 heads of 64: 45 us with two, 51 with
// four; T=2048, B=12, 4 heads of 32: 30 and 26), times 256. Heads that fill
// those by themselves are not cut. Else n segments take about chunks / n * 9 us
// for their two passes and n states of all heads, moved five times at 4 MB a
// us; the sum is least at the root below.
int attn_segments(const AttnShape& s, int type, long* seg_len) {
  const long chunks = (s.T + 63) / 64, heads = s.B * s.H;
  const long d = std::max(s.dk, s.dv);
  const long slots = d > 64 ? 256
                     : type == 1 || (type == 2 && d <= 32) ? 1024 : 512;
  const double best = std::sqrt(chunks * 9.0 * 4e6 /
                                (20.0 * heads * s.dk * s.dv));
  long n = std::min({slots / heads, chunks, (long)std::min(best, 1e6)});
  if (n < 1) n = 1;
  const long per = (chunks + n - 1) / n;
  *seg_len = per * 64;
  return (int)((s.T + *seg_len - 1) / *seg_len);
}

// flags whose 64 steps lie within 32 bits
Tensor near(const Tensor& done) {
  return done.defined() && done.size(0) > 1 && done.stride(0) >= (1L << 25)
             ? done.contiguous() : done;
}

AttnArgs attn_args(const AttnShape& s, int type, const Tensor& g,
                   const Tensor& done) {
  AttnArgs a{};
  a.log_decay = g.data_ptr<float>();
  a.g_stride = g.size(0) > 1 ? g.stride(0) : 0;
  if (done.defined()) {
    TORCH_CHECK(done.size(0) == 1 || done.stride(0) < (1L << 25),
                "linear_attention: steps of done lie too far apart");
    a.done = (const unsigned char*)done.data_ptr();
    a.done_st = done.size(0) > 1 ? done.stride(0) : 0;
    a.done_sb = done.size(1) > 1 ? done.stride(1) : 0;
  }
  a.T = s.T;
  a.B = (int)s.B;
  a.H = (int)s.H;
  a.nseg = attn_segments(s, type, &a.seg_len);
  return a;
}

// entry states of all segments for one direction: (nseg, B, H, x, y)
Tensor attn_entry_states(AttnArgs a, const AttnRole& role,
                         const float* first, int type, bool vec,
                         const Tensor& like, hipStream_t stream) {
  auto fopts = like.options().dtype(torch::kFloat32);
  const long heads = (long)a.B * a.H, size = (long)role.dk * role.dv;
  auto st = torch::empty({(long)a.nseg * heads * size}, fopts);
  auto keep = torch::empty({(long)a.nseg * heads}, fopts);
  a.nroles = 1;
  a.role[0] = role;
  a.role[0].s_in = nullptr;
  a.role[0].s_out = st.data_ptr<float>();
  a.keep = keep.data_ptr<float>();
  launch_attn_chunks(type, &a, vec, 1, stream);
  launch_attn_scan(st.data_ptr<float>(), a.keep, first, a.log_decay,
                   a.g_stride, a.H, heads, size, a.nseg, role.rev, a.T,
                   a.seg_len, stream);
  return st;
}

AttnShape shape_of(const Tensor& q, const Tensor& v) {
  return AttnShape{q.size(0), q.size(1), q.size(2), q.size(3), v.size(3)};
}

// (out, final state, entry states of segments or none)
std::array<Tensor, 3> attn_fwd(const Tensor& q0, const Tensor& k0,
                               const Tensor& v0, const Tensor& g,
                               const Tensor& done0, const Tensor& state0,
                               double scale) {
  const AttnShape s = shape_of(q0, v0);
  const c10::DeviceGuard guard(q0.device());
  const Tensor q = unit(q0), k = unit(k0), v = unit(v0),
               state = dense(state0), done = near(done0);
  const int type = type_code(q, "q");
  Tensor out = torch::empty({s.T, s.B, s.H, s.dv}, q.options());
  Tensor fin = torch::empty({s.B, s.H, s.dk, s.dv},
                            q.options().dtype(torch::kFloat32));
  Tensor entry;
  if (s.B * s.H == 0) return {out, fin, entry};
  if (s.T == 0) {
    if (state.defined()) fin.copy_(state);
    else fin.zero_();
    return {out, fin, entry};
  }
  AttnArgs a = attn_args(s, type, g, done);
  AttnRole r{};
  r.a = operand(q, 2);
  r.b = operand(k, 2);
  r.c = operand(v, 2);
  r.out = out.data_ptr();
  r.dk = (int)s.dk;
  r.dv = (int)s.dv;
  r.p_scale = r.in_scale = (float)scale;
  r.u_scale = 1.f;
  r.sx = s.dv;
  r.sy = 1;
  r.s_in = (const float*)ptr(state);
  r.s_out = fin.data_ptr<float>();
  const bool vec = can_vec(q, r.a) && can_vec(k, r.b) && can_vec(v, r.c);
  hipStream_t stream = stream_here();
  if (a.nseg > 1) {
    entry = attn_entry_states(a, r, r.s_in, type, vec, q, stream);
    r.s_in = entry.data_ptr<float>();
  }
  a.nroles = 1;
  a.role[0] = r;
  launch_attn_chunks(type, &a, vec, 0, stream);
  check_launch("linear_attention");
  return {out, fin, entry};
}

class LinearAttention : public torch::autograd::Function<LinearAttention> {
 public:
  static variable_list forward(AutogradContext* ctx, Tensor q, Tensor k,
                               Tensor v, Tensor g, OptTensor done_,
                               OptTensor state_, double scale) {
    const Tensor done = or_undefined(done_), state = or_undefined(state_);
    ctx->set_materialize_grads(false);
    auto [out, fin, entry] = attn_fwd(q, k, v, g, done, state, scale);
    ctx->save_for_backward({q, k, v, g, done, state, entry});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["ds"] = state.defined() && state.requires_grad();
    return {out, fin};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const double scale = ctx->saved_data["scale"].toDouble();
    const bool need_ds = ctx->saved_data["ds"].toBool();
    if (!grads[0].defined() && !grads[1].defined())
      return variable_list(7);
    const AttnShape s = shape_of(saved[0], saved[2]);
    const c10::DeviceGuard guard(saved[0].device());
    const Tensor q = unit(saved[0]), k = unit(saved[1]), v = unit(saved[2]);
    const Tensor &g = saved[3], &entry = saved[6];
    const Tensor done = near(saved[4]), state = dense(saved[5]);
    const Tensor d_out = grads[0].defined()
                             ? unit(grads[0])
                             : torch::zeros(v.sizes(), v.options());
    const Tensor d_final = dense(grads[1]);
    const int type = type_code(q, "q");
    Tensor dq = torch::empty(q.sizes(), q.options());
    Tensor dk = torch::empty(q.sizes(), q.options());
    Tensor dv = torch::empty(v.sizes(), q.options());
    Tensor ds;
    if (need_ds)
      ds = torch::empty({s.B, s.H, s.dk, s.dv},
                        q.options().dtype(torch::kFloat32));
    if (s.B * s.H > 0 && s.T > 0) {
      AttnArgs a = attn_args(s, type, g, done);
      const AttnOperand oq = operand(q, 2), ok = operand(k, 2),
                        ov = operand(v, 2), od = operand(d_out, 2);
      const bool vec = can_vec(q, oq) && can_vec(k, ok) && can_vec(v, ov) &&
                       can_vec(d_out, od);
      hipStream_t stream = stream_here();
      AttnRole rv{};   // dv: a = k, b = q, c = d_out, from the last step
      rv.a = ok;
      rv.b = oq;
      rv.c = od;
      rv.out = dv.data_ptr();
      rv.dk = (int)s.dk;
      rv.dv = (int)s.dv;
      rv.rev = 1;
      rv.p_scale = rv.u_scale = (float)scale;
      rv.in_scale = 1.f;
      rv.s_in = (const float*)ptr(d_final);
      rv.sx = s.dv;
      rv.sy = 1;
      rv.s_out = need_ds ? ds.data_ptr<float>() : nullptr;
      Tensor back;
      if (a.nseg > 1) {
        back = attn_entry_states(a, rv, rv.s_in, type, vec, q, stream);
        rv.s_in = back.data_ptr<float>();
      }
      AttnRole rk = rv;   // dk: a = v, b = d_out, c = q, the state turned
      rk.a = ov;
      rk.b = od;
      rk.c = oq;
      rk.out = dk.data_ptr();
      rk.dk = (int)s.dv;
      rk.dv = (int)s.dk;
      rk.sx = 1;
      rk.sy = s.dv;
      rk.s_out = nullptr;
      AttnRole rq{};      // dq: a = d_out, b = v, c = k, from the first step
      rq.a = od;
      rq.b = ov;
      rq.c = ok;
      rq.out = dq.data_ptr();
      rq.dk = (int)s.dv;
      rq.dv = (int)s.dk;
      rq.p_scale = rq.in_scale = (float)scale;
      rq.u_scale = 1.f;
      rq.s_in = (const float*)ptr(a.nseg > 1 ? entry : state);
      rq.sx = 1;
      rq.sy = s.dv;
      a.nroles = 3;
      a.role[0] = rv;
      a.role[1] = rk;
      a.role[2] = rq;
      launch_attn_chunks(type, &a, vec, 0, stream);
      check_launch("linear_attention backward");
    } else if (need_ds && s.B * s.H > 0) {
      if (d_final.defined()) ds.copy_(d_final);
      else ds.zero_();
    }
    return once({dq, dk, dv, Tensor(), Tensor(), ds, Tensor()},
                "linear_attention");
  }
};

std::tuple<Tensor, Tensor> linear_attention(Tensor q, Tensor k, Tensor v,
                                            Tensor g, OptTensor done_,
                                            OptTensor state_,
                                            c10::optional<double> scale_) {
  const Tensor done = or_undefined(done_), state = or_undefined(state_);
  const AttnShape s =
      check_attn("linear_attention", q, k, v, g, done, state, 2);
  const double scale = scale_of("linear_attention", scale_, s);
  refuse_tangents("linear_attention", {q, k, v, g, state});
  if (wants_grad({q, k, v, state})) {
    auto r = LinearAttention::apply(q, k, v, g, done_, state_, scale);
    return {r[0], r[1]};
  }
  auto [out, fin, entry] = attn_fwd(q, k, v, g, done, state, scale);
  return {out, fin};
}

bool heads_contiguous(const Tensor& t) {
  return t.numel() == 0 || t.select(0, 0).is_contiguous();
}

// bytes from the first one to behind the last, of the axes from `axis` on
long span_of(const Tensor& t, int axis) {
  long n = 1;
  for (int i = axis; i < t.dim(); ++i) n += (t.size(i) - 1) * t.stride(i);
  return n * t.element_size();
}

// Two tensors of environments, neither empty, without common memory: one
// behind the other, or an environment's parts of both side by side in records
// of one size.
bool apart(const Tensor& a, const Tensor& b) {
  const uintptr_t p = (uintptr_t)a.data_ptr(), q = (uintptr_t)b.data_ptr();
  if (p + span_of(a, 0) <= q || q + span_of(b, 0) <= p) return true;
  const long record = a.stride(0) * a.element_size();
  if (record <= 0 || b.stride(0) * b.element_size() != record) return false;
  const long at = q >= p ? (long)((q - p) % record)
                         : record - 1 - (long)((p - q - 1) % record);
  return at >= span_of(a, 1) && at + span_of(b, 1) <= record;
}

// q, k (B, H, dk), v (B, H, dv); the states' environments may lie apart
std::tuple<Tensor, Tensor> linear_attention_step(
    Tensor q0, Tensor k0, Tensor v0, Tensor g, Tensor state, OptTensor done_,
    c10::optional<double> scale_, OptTensor out_state_) {
  const char* op = "linear_attention_step";
  const Tensor done = or_undefined(done_);
  const AttnShape s = check_attn(op, q0, k0, v0, g, done, state, 1);
  const double scale = scale_of(op, scale_, s);
  TORCH_CHECK(!wants_grad({q0, k0, v0, state}), op,
              " has no gradient; use linear_attention with T = 1");
  refuse_tangents(op, {q0, k0, v0, g, state, or_undefined(out_state_)});
  const c10::DeviceGuard guard(q0.device());
  Tensor next;
  if (out_state_.has_value()) {
    next = *out_state_;
    TORCH_CHECK_TYPE(next.scalar_type() == torch::kFloat32, op,
                     ": out_state must be fp32, not ", next.scalar_type());
    TORCH_CHECK_VALUE(next.sizes() == state.sizes() &&
                          next.device() == state.device(),
                      op, ": out_state must match the state");
    TORCH_CHECK(!wants_grad({next}), op,
                " writes out_state in place; it must not require grad");
    if (next.numel()) {
      TORCH_CHECK_VALUE(heads_contiguous(next) &&
                            (s.B == 1 ||
                             next.stride(0) >= s.H * s.dk * s.dv),
                        op, ": out_state needs an environment's heads "
                        "contiguous and environments that do not overlap");
      TORCH_CHECK_VALUE((next.data_ptr() == state.data_ptr() &&
                         next.strides() == state.strides()) ||
                            apart(next, state),
                        op, ": out_state overlaps the state without being it");
      // a block reads its inputs while others write their states
      for (const Tensor& t : {q0, k0, v0, g, done})
        TORCH_CHECK_VALUE(!t.defined() || apart(next, t), op,
                          ": out_state overlaps an input");
    }
    // autograd has to see the write: the state may be saved somewhere
    if (!next.is_inference()) next.unsafeGetTensorImpl()->bump_version();
  } else {
    next = torch::empty({s.B, s.H, s.dk, s.dv}, state.options());
  }
  if (!heads_contiguous(state)) state = state.contiguous();
  const Tensor q = unit(q0), k = unit(k0), v = unit(v0);
  Tensor out = torch::empty({s.B, s.H, s.dv}, q.options());
  if (s.B * s.H == 0) return {out, next};
  AttnStepArgs a{};
  a.q = operand(q, 1);
  a.k = operand(k, 1);
  a.v = operand(v, 1);
  a.out = out.data_ptr();
  a.log_decay = g.data_ptr<float>();
  a.g_stride = s.H > 1 ? g.stride(0) : 0;
  if (done.defined()) {
    a.done = (const unsigned char*)done.data_ptr();
    a.done_sb = s.B > 1 ? done.stride(0) : 0;
  }
  a.s = state.data_ptr<float>();
  a.d = next.data_ptr<float>();
  a.s_sb = s.B > 1 ? state.stride(0) : 0;
  a.d_sb = s.B > 1 ? next.stride(0) : 0;
  a.scale = (float)scale;
  a.B = (int)s.B;
  a.H = (int)s.H;
  a.dk = (int)s.dk;
  a.dv = (int)s.dv;
  const bool vec = s.dv % 4 == 0 && ((uintptr_t)a.s & 15) == 0 &&
                   ((uintptr_t)a.d & 15) == 0 && a.s_sb % 4 == 0 &&
                   a.d_sb % 4 == 0;
  launch_attn_step(type_code(q, "q"), &a, vec, stream_here());
  check_launch(op);
  return {out, next};
}

// ---------------------------------------------------------------------------
// Newton-Schulz orthogonalisation of lists of matrices
// ---------------------------------------------------------------------------
namespace ns = impala::ortho;

// exponent that brings entries of 1 / sqrt(n) to about 8
int scale_exp(long n) {
  const int e = 3 + (int)std::lround(0.5 * std::log2((double)n));
  return e < 13 ? e : 13;
}

int k_step(int tile) { return tile == 64 ? 64 : 32; }

long k_steps(const ns::Mat& m, int mode, int tile) {
  return (mode == 0 ? m.np : m.mp) / k_step(tile);
}

int tiles_of(const ns::Mat& m, int mode, int tile) {
  const int tm = m.mp / tile, tn = m.np / tile;
  return mode == 2 ? tm * tn : tm * (tm + 1) / 2;
}

// Steps of k that a block takes; what is longer is split over blocks, whose
// parts a second launch adds. Least of an estimate in us, from measured
// products: a step takes a block alone on a CU 1.3 (tiles of 128) or 0.65, two
// on a CU 1.5 or 0.9, and 1.9 or 1.1 where more than the 512 that run at once
// keep all of the card busy; adding takes 6 and the parts' bytes at 2 MB a
// us. Six products of 1024^3: unsplit 47, split in two
// 35 + 16. 10 tiles of 64 over k = 1568: unsplit 21, in four 9 + 7, in seven
// 7 + 6. 2048 x 2048 and 2048 x 8192: k in steps of 4096 193 + 14, of 1024
// 202 + 31.
long block_steps(const ns::Args& a, int mode, int tile) {
  const double alone = tile == 64 ? 0.65 : 1.3;
  const double both = tile == 64 ? 0.9 : 1.5, full = tile == 64 ? 1.1 : 1.9;
  long longest = 0;
  for (int i = 0; i < a.count; ++i)
    longest = std::max(longest, k_steps(a.mat[i], mode, tile));
  long best = longest;
  double least = 1e30;
  for (long n = 1; n <= 64; ++n) {
    const long per = (longest + n - 1) / n;
    if (n > 1 && per * k_step(tile) < 256) break;
    long blocks = 0, parts = 0;
    for (int i = 0; i < a.count; ++i) {
      const long splits = (k_steps(a.mat[i], mode, tile) + per - 1) / per;
      const long mine = splits * tiles_of(a.mat[i], mode, tile);
      blocks += mine;
      if (splits > 1) parts += mine;
    }
    const double t = per * (blocks <= 256   ? alone
                            : blocks <= 512 ? both
                                            : (blocks + 511) / 512 * full) +
                     (parts ? 6.0 + parts * 4.0 * tile * tile / 2e6 : 0.0);
    if (t < least) {
      least = t;
      best = per;
    }
  }
  return best;
}

// tiles of one product of all matrices, and the blocks that share a tile's k;
// returns the floats that the parts of split tiles need
long plan_product(ns::Args& a, int mode, int tile, long per) {
  long part = 0;
  int blocks = 0, sums = 0;
  for (int i = 0; i < a.count; ++i) {
    ns::Mat& m = a.mat[i];
    m.tiles = tiles_of(m, mode, tile);
    m.splits = (int)((k_steps(m, mode, tile) + per - 1) / per);
    a.first[i] = blocks;
    a.first_sum[i] = sums;
    a.part_off[i] = part;
    blocks += m.tiles * m.splits;
    if (m.splits > 1) {
      sums += m.tiles;
      part += (long)m.tiles * m.splits * tile * tile;
    }
  }
  a.first[a.count] = blocks;
  a.first_sum[a.count] = sums;
  return part;
}

// matrices that share their launches, at most MAX_MATS, in tiles of one size
void orthogonalize_group(const std::vector<Tensor>& src,
                         const std::vector<Tensor>& dst,
                         const std::vector<size_t>& take, int tile, long steps,
                         double eps) {
  const Tensor& like = src[take[0]];
  const c10::DeviceGuard guard(like.device());
  hipStream_t stream = stream_here();
  ns::Args a{};
  a.count = (int)take.size();
  long parts = 0;
  for (int i = 0; i < a.count; ++i) {
    const Tensor &s = src[take[i]], &d = dst[take[i]];
    ns::Mat& m = a.mat[i];
    const bool tall = s.size(0) > s.size(1);
    const int r = tall ? 1 : 0, c = tall ? 0 : 1;
    m.src = s.data_ptr();
    m.src_i = s.stride(r);
    m.src_j = s.stride(c);
    m.dst = d.data_ptr();
    m.dst_i = d.stride(r);
    m.dst_j = d.stride(c);
    m.type = type_code(s, "matrix");
    m.m = (int)s.size(r);
    m.n = (int)s.size(c);
    m.mp = (m.m + tile - 1) / tile * tile;
    m.np = (m.n + tile - 1) / tile * tile;
    m.ex = scale_exp(m.n);
    m.ea = scale_exp(m.m);
    const long wide = 2L * m.mp * m.np, square = 2L * m.mp * m.mp;
    m.x = parts;
    m.xt[0] = m.x + wide;
    m.xt[1] = m.xt[0] + wide;
    m.a = m.xt[1] + wide;
    m.b = m.a + square;
    parts = m.b + square;
  }
  int norm_blocks = 0;
  for (int i = 0; i < a.count; ++i) {
    ns::Mat& m = a.mat[i];
    const long want = ((long)m.m * m.n + 8191) / 8192;
    m.norm_blocks = (int)std::min(want, (long)ns::MAX_NORM_BLOCKS);
    a.first_norm[i] = norm_blocks;
    norm_blocks += m.norm_blocks;
  }
  a.first_norm[a.count] = norm_blocks;
  long partial = 0, per[3];
  for (int mode = 0; mode < 3; ++mode) {
    per[mode] = block_steps(a, mode, tile);
    partial = std::max(partial, plan_product(a, mode, tile, per[mode]));
  }
  auto work = torch::empty({parts}, like.options().dtype(torch::kFloat16));
  auto split = torch::empty({partial},
                            like.options().dtype(torch::kFloat32));
  auto sums = torch::empty({norm_blocks},
                           like.options().dtype(torch::kFloat64));
  auto rho = torch::empty({a.count}, like.options().dtype(torch::kFloat32));
  a.parts = (_Float16*)work.data_ptr();
  a.partial = split.data_ptr<float>();
  a.sums = sums.data_ptr<double>();
  a.rho = rho.data_ptr<float>();
  a.eps = eps;
  launch_ns_start(&a, stream);
  for (long k = 0; k < steps; ++k) {
    a.round = (int)k;
    a.last = k + 1 == steps;
    for (int mode = 0; mode < 3; ++mode) {
      plan_product(a, mode, tile, per[mode]);
      launch_ns_product(mode, tile, &a, stream);
    }
  }
  check_launch("orthogonalize");
}

void orthogonalize(std::vector<Tensor> src, std::vector<Tensor> dst,
                   long steps, double eps) {
  TORCH_CHECK(src.size() == dst.size() && steps >= 1 && eps >= 0.0,
              "orthogonalize: bad arguments");
  for (size_t i = 0; i < src.size(); ++i) {
    const Tensor &s = src[i], &d = dst[i];
    TORCH_CHECK(s.is_cuda() && s.dim() == 2 && d.sizes() == s.sizes() &&
                    s.device() == src[0].device() &&
                    d.device() == s.device() &&
                    d.scalar_type() == s.scalar_type(),
                "orthogonalize: matrices and results must match");
    TORCH_CHECK(s.size(0) < (1 << 20) && s.size(1) < (1 << 20) &&
                    std::min(s.size(0), s.size(1)) <= 32768,
                "orthogonalize: matrix too large");
    type_code(s, "matrix");
  }
  size_t at = 0;
  while (at < src.size()) {
    std::vector<size_t> all, few, more;   // up to 64 rows, and the others
    long tiles128 = 0;
    for (; at < src.size() && all.size() < ns::MAX_MATS; ++at) {
      const Tensor& s = src[at];
      if (s.numel() == 0) continue;
      all.push_back(at);
      if (std::min(s.size(0), s.size(1)) <= 64) {
        few.push_back(at);
      } else {
        more.push_back(at);
        tiles128 += ((s.size(0) + 127) / 128) * ((s.size(1) + 127) / 128);
      }
    }
    if (all.empty()) break;
    // A tile of 128 needs half the reads of 64, if there are enough of them.
    // Few rows stay with tiles of 64, which are the exact ones for them
    // (beside 2048 x 2048 in tiles of 128 and by themselves: 4 x 2000 off by
    // 2.7e-6 and 1.5e-6, where fp32 products are by 1.8e-6; 7 x 599 by 0.90
    // and 0.56, fp32 0.69; 64 x 500 by 2.0 and 1.2, fp32 1.65). A second set
    // of launches costs up to 145 us (2048 x 2048 with 8 of 64 x 2048: 1076
    // against 929); few rows by themselves are faster so too (24 of 64 x 2048:
    // 179 against 364 padded to tiles of 128).
    if (tiles128 < 256) {
      orthogonalize_group(src, dst, all, 64, steps, eps);
      continue;
    }
    orthogonalize_group(src, dst, more, 128, steps, eps);
    if (!few.empty()) orthogonalize_group(src, dst, few, 64, steps, eps);
  }
}

}  // namespace

void register_core_ops(pybind11::module_& m) {
  m.def("orthogonalize", &orthogonalize, py::arg("src"), py::arg("dst"),
        py::arg("steps"), py::arg("eps"));
  m.def("linear_attention", &linear_attention, py::arg("q"), py::arg("k"),
        py::arg("v"), py::arg("log_decay"), py::arg("done") = py::none(),
        py::arg("state") = py::none(), py::arg("scale") = py::none());
  m.def("linear_attention_step", &linear_attention_step, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("state"),
        py::arg("done") = py::none(), py::arg("scale") = py::none(),
        py::arg("out_state") = py::none());
  m.def("layer_norm", &layer_norm, py::arg("x"),
        py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5);
}
