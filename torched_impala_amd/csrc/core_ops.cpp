// Host side of the operators of the linear-attention core and of its
// matrices' updates: argument checks that keep the kernels in bounds, output
// and workspace tensors (torch's allocator, so a captured graph owns its
// own), launches on the current stream of the operands' device.

#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
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
void launch_attn_scan(float*, const float*, const float*, long, long, int,
                      int, hipStream_t);
void launch_attn_step(int, const impala::attn::AttnStepArgs*, int,
                      hipStream_t);
void launch_ns_start(impala::ortho::Args*, hipStream_t);
void launch_ns_product(int, int, const impala::ortho::Args*, hipStream_t);
}

namespace {

using torch::Tensor;
using OptTensor = c10::optional<Tensor>;

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

const void* ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

// ---------------------------------------------------------------------------
// layer norm. x (rows, cols) with unit column stride; the row stride is free
// ---------------------------------------------------------------------------
void check_norm_operands(const Tensor& x, const OptTensor& w,
                         const OptTensor& b) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.size(1) > 0 &&
                  (x.stride(1) == 1 || x.size(1) == 1) && x.stride(0) >= 0,
              "layer_norm: x must be a GPU matrix with unit column stride");
  for (const auto* p : {&w, &b}) {
    if (!p->has_value()) continue;
    const Tensor& t = **p;
    TORCH_CHECK(t.device() == x.device() && t.dim() == 1 &&
                    t.size(0) == x.size(1) && t.is_contiguous(),
                "layer_norm: weight and bias must be (cols,) on x's device");
    TORCH_CHECK(t.scalar_type() == torch::kFloat32 ||
                    t.scalar_type() == x.scalar_type(),
                "layer_norm: weight and bias must be fp32 or of x's type");
  }
  TORCH_CHECK(!w.has_value() || !b.has_value() ||
                  w->scalar_type() == b->scalar_type(),
              "layer_norm: weight and bias must have one type");
}

std::vector<Tensor> layer_norm_fwd(Tensor x, OptTensor w, OptTensor b,
                                   double eps, bool save) {
  check_norm_operands(x, w, b);
  const int xt = type_code(x, "x");
  const int wt = w.has_value() ? type_code(*w, "weight")
                 : b.has_value() ? type_code(*b, "bias") : xt;
  const long rows = x.size(0), cols = x.size(1);
  const c10::DeviceGuard guard(x.device());
  auto y = torch::empty({rows, cols}, x.options());
  auto fopts = x.options().dtype(torch::kFloat32);
  auto stats = torch::empty({2, save ? rows : 0}, fopts);
  if (rows > 0) {
    float* mean = save ? stats.data_ptr<float>() : nullptr;
    launch_layer_norm_fwd(xt, wt, x.data_ptr(), x.stride(0), ptr(w), ptr(b),
                          y.data_ptr(), mean, save ? mean + rows : nullptr,
                          rows, cols, (float)eps, stream_here());
    check_launch("layer_norm");
  }
  return {y, stats};
}

std::vector<OptTensor> layer_norm_bwd(Tensor dy, Tensor x, OptTensor w,
                                      Tensor stats, bool need_dx,
                                      bool need_dw, bool need_db,
                                      bool param_fp32) {
  check_norm_operands(x, w, c10::nullopt);
  const long rows = x.size(0), cols = x.size(1);
  TORCH_CHECK(dy.device() == x.device() && dy.sizes() == x.sizes() &&
                  dy.scalar_type() == x.scalar_type() && dy.is_contiguous(),
              "layer_norm: the output's gradient must match the output");
  TORCH_CHECK(stats.device() == x.device() && stats.is_contiguous() &&
                  stats.scalar_type() == torch::kFloat32 &&
                  stats.numel() == 2 * rows,
              "layer_norm: saved statistics do not match x");
  const int xt = type_code(x, "x");
  const int wt = w.has_value() ? type_code(*w, "weight")
                 : param_fp32 ? 0 : xt;
  const c10::DeviceGuard guard(x.device());
  auto popts = x.options();
  if (wt == 0) popts = popts.dtype(torch::kFloat32);
  OptTensor dx, dw, db;
  if (need_dx) dx = torch::empty({rows, cols}, x.options());
  if (rows == 0) {
    if (need_dw) dw = torch::zeros({cols}, popts);
    if (need_db) db = torch::zeros({cols}, popts);
    return {dx, dw, db};
  }
  if (need_dw) dw = torch::empty({cols}, popts);
  if (need_db) db = torch::empty({cols}, popts);
  const int al = layer_norm_aligned(xt, dy.data_ptr(), x.data_ptr(),
                                    x.stride(0), ptr(w), ptr(dx), cols);
  Tensor part;
  if (need_dw || need_db)
    part = torch::empty({layer_norm_part_elems(xt, rows, cols, al)},
                        x.options().dtype(torch::kFloat32));
  launch_layer_norm_bwd(
      xt, wt, al, dy.data_ptr(), x.data_ptr(), x.stride(0), ptr(w),
      stats.data_ptr<float>(), stats.data_ptr<float>() + rows,
      const_cast<void*>(ptr(dx)),
      part.defined() ? part.data_ptr<float>() : nullptr,
      const_cast<void*>(ptr(dw)), const_cast<void*>(ptr(db)), rows, cols,
      stream_here());
  check_launch("layer_norm backward");
  return {dx, dw, db};
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
constexpr long MAX_GRID = 2147483647;

struct AttnShape {
  long T, B, H, dk, dv;
};

void check_unit(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda(), "linear_attention: ", name, " must be on GPU");
  TORCH_CHECK(t.stride(-1) == 1 || t.size(-1) == 1,
              "linear_attention: the last axis of ", name,
              " must be contiguous");
}

AttnShape check_attn(const Tensor& q, const Tensor& k, const Tensor& v,
                     const Tensor& g, const OptTensor& done, int lead) {
  check_unit(q, "q");
  check_unit(k, "k");
  check_unit(v, "v");
  TORCH_CHECK(q.dim() == lead + 2 && k.sizes() == q.sizes() &&
                  v.dim() == q.dim() &&
                  v.sizes().slice(0, lead + 1) == q.sizes().slice(0, lead + 1),
              "linear_attention: shapes of q, k and v do not fit");
  TORCH_CHECK(k.scalar_type() == q.scalar_type() &&
                  v.scalar_type() == q.scalar_type() &&
                  k.device() == q.device() && v.device() == q.device(),
              "linear_attention: q, k and v must have one type and device");
  AttnShape s{lead == 2 ? q.size(0) : 1, q.size(lead - 1), q.size(lead),
              q.size(-1), v.size(-1)};
  TORCH_CHECK(s.dk >= 1 && s.dk <= MAX_HEAD && s.dv >= 1 && s.dv <= MAX_HEAD,
              "linear_attention: head sizes must be 1 to ", MAX_HEAD);
  TORCH_CHECK(s.B <= MAX_GRID && s.H <= MAX_GRID,
              "linear_attention: batch too large");
  TORCH_CHECK(g.device() == q.device() && g.dim() == 1 &&
                  g.size(0) == s.H && g.scalar_type() == torch::kFloat32,
              "linear_attention: log_decay must be (H,) fp32 on q's device");
  if (done.has_value())
    TORCH_CHECK(done->device() == q.device() &&
                    done->scalar_type() == torch::kBool &&
                    done->sizes() == q.sizes().slice(0, lead),
                "linear_attention: done must be bool, one flag a step and "
                "environment, on q's device");
  return s;
}

const float* check_state(const OptTensor& t, const Tensor& q,
                         const AttnShape& s, const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->device() == q.device() &&
                  t->scalar_type() == torch::kFloat32 &&
                  t->is_contiguous() && t->dim() == 4 &&
                  t->size(0) == s.B && t->size(1) == s.H &&
                  t->size(2) == s.dk && t->size(3) == s.dv,
              "linear_attention: ", name, " must be (B, H, dk, dv) fp32, "
              "contiguous, on q's device");
  return t->data_ptr<float>();
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

// segments that a sequence is cut into: none while the heads alone give the
// card two workgroups a CU, else as many as make that up, four chunks each
// at least (a segment's state costs as much traffic as some chunks do)
int attn_segments(const AttnShape& s, long* seg_len) {
  const long chunks = (s.T + 63) / 64, heads = s.B * s.H;
  long n = heads >= 512 ? 1 : 512 / heads;
  const long most = chunks / 4;
  if (n > most) n = most;
  if (n < 1) n = 1;
  const long per = (chunks + n - 1) / n;
  *seg_len = per * 64;
  return (int)((s.T + *seg_len - 1) / *seg_len);
}

AttnArgs attn_args(const AttnShape& s, const Tensor& g,
                   const OptTensor& done) {
  AttnArgs a{};
  a.log_decay = g.data_ptr<float>();
  a.g_stride = g.size(0) > 1 ? g.stride(0) : 0;
  if (done.has_value()) {
    a.done = (const unsigned char*)done->data_ptr();
    a.done_st = done->size(0) > 1 ? done->stride(0) : 0;
    a.done_sb = done->size(1) > 1 ? done->stride(1) : 0;
  }
  a.T = s.T;
  a.B = (int)s.B;
  a.H = (int)s.H;
  a.nseg = attn_segments(s, &a.seg_len);
  TORCH_CHECK(s.B * s.H * a.nseg <= MAX_GRID / 3 &&
                  s.B * s.H * s.dk * s.dv / 256 < MAX_GRID,
              "linear_attention: batch too large");
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
  launch_attn_scan(st.data_ptr<float>(), a.keep, first, heads, size, a.nseg,
                   role.rev, stream);
  return st;
}

// (out, final state, entry states of segments or none)
std::vector<OptTensor> linear_attention_fwd(Tensor q, Tensor k, Tensor v,
                                            Tensor g, OptTensor done,
                                            OptTensor state, double scale) {
  const AttnShape s = check_attn(q, k, v, g, done, 2);
  const float* s0 = check_state(state, q, s, "state");
  const int type = type_code(q, "q");
  const c10::DeviceGuard guard(q.device());
  auto out = torch::empty({s.T, s.B, s.H, s.dv}, q.options());
  auto fin = torch::empty({s.B, s.H, s.dk, s.dv},
                          q.options().dtype(torch::kFloat32));
  if (s.B * s.H == 0) return {out, fin, c10::nullopt};
  if (s.T == 0) {
    if (s0) fin.copy_(*state);
    else fin.zero_();
    return {out, fin, c10::nullopt};
  }
  AttnArgs a = attn_args(s, g, done);
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
  r.s_in = s0;
  r.s_out = fin.data_ptr<float>();
  const bool vec = can_vec(q, r.a) && can_vec(k, r.b) && can_vec(v, r.c);
  hipStream_t stream = stream_here();
  OptTensor entry;
  if (a.nseg > 1) {
    entry = attn_entry_states(a, r, s0, type, vec, q, stream);
    r.s_in = entry->data_ptr<float>();
  }
  a.nroles = 1;
  a.role[0] = r;
  launch_attn_chunks(type, &a, vec, 0, stream);
  check_launch("linear_attention");
  return {out, fin, entry};
}

// (dq, dk, dv, gradient of the state or none)
std::vector<OptTensor> linear_attention_bwd(
    Tensor q, Tensor k, Tensor v, Tensor g, OptTensor done, OptTensor state,
    OptTensor entry, Tensor d_out, OptTensor d_final, double scale,
    bool need_dstate) {
  const AttnShape s = check_attn(q, k, v, g, done, 2);
  const float* s0 = check_state(state, q, s, "state");
  const float* df = check_state(d_final, q, s, "the final state's gradient");
  check_unit(d_out, "the output's gradient");
  TORCH_CHECK(d_out.sizes() == v.sizes() && d_out.device() == q.device() &&
                  d_out.scalar_type() == q.scalar_type(),
              "linear_attention: the output's gradient must match the output");
  const int type = type_code(q, "q");
  const c10::DeviceGuard guard(q.device());
  auto dq = torch::empty(q.sizes(), q.options());
  auto dk = torch::empty(q.sizes(), q.options());
  auto dv = torch::empty(v.sizes(), q.options());
  for (auto* t : {&dq, &dk, &dv}) TORCH_CHECK(t->is_contiguous());
  OptTensor ds;
  if (need_dstate)
    ds = torch::empty({s.B, s.H, s.dk, s.dv},
                      q.options().dtype(torch::kFloat32));
  if (s.B * s.H == 0) return {dq, dk, dv, ds};
  if (s.T == 0) {
    if (need_dstate) {
      if (df) ds->copy_(*d_final);
      else ds->zero_();
    }
    return {dq, dk, dv, ds};
  }
  AttnArgs a = attn_args(s, g, done);
  const long heads = s.B * s.H, size = s.dk * s.dv;
  if (a.nseg > 1)
    TORCH_CHECK(entry.has_value() && entry->device() == q.device() &&
                    entry->scalar_type() == torch::kFloat32 &&
                    entry->is_contiguous() &&
                    entry->numel() == a.nseg * heads * size,
                "linear_attention: saved entry states do not match");
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
  rv.s_in = df;
  rv.sx = s.dv;
  rv.sy = 1;
  rv.s_out = need_dstate ? ds->data_ptr<float>() : nullptr;
  Tensor back;
  if (a.nseg > 1) {
    back = attn_entry_states(a, rv, df, type, vec, q, stream);
    rv.s_in = back.data_ptr<float>();
  }
  AttnRole rk = rv;   // dk: a = v, b = d_out, c = q; the same state turned
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
  rq.s_in = a.nseg > 1 ? entry->data_ptr<float>() : s0;
  rq.sx = 1;
  rq.sy = s.dv;
  a.nroles = 3;
  a.role[0] = rv;
  a.role[1] = rk;
  a.role[2] = rq;
  launch_attn_chunks(type, &a, vec, 0, stream);
  check_launch("linear_attention backward");
  return {dq, dk, dv, ds};
}

// q, k (B, H, dk), v (B, H, dv); the states' environments may lie apart
Tensor linear_attention_step(Tensor q, Tensor k, Tensor v, Tensor g,
                             Tensor state, Tensor out_state, OptTensor done,
                             double scale) {
  const AttnShape s = check_attn(q, k, v, g, done, 1);
  const int type = type_code(q, "q");
  for (const Tensor* t : {&state, &out_state}) {
    TORCH_CHECK(t->device() == q.device() && t->dim() == 4 &&
                    t->scalar_type() == torch::kFloat32 &&
                    t->size(0) == s.B && t->size(1) == s.H &&
                    t->size(2) == s.dk && t->size(3) == s.dv &&
                    (s.B * s.H == 0 || t->select(0, 0).is_contiguous()),
                "linear_attention_step: states must be (B, H, dk, dv) fp32 "
                "on q's device, an environment's heads contiguous");
  }
  const c10::DeviceGuard guard(q.device());
  auto out = torch::empty({s.B, s.H, s.dv}, q.options());
  if (s.B * s.H == 0) return out;
  TORCH_CHECK(s.B * s.H <= MAX_GRID, "linear_attention_step: batch too large");
  TORCH_CHECK(s.B == 1 || out_state.stride(0) >= s.H * s.dk * s.dv,
              "linear_attention_step: environments of the new state overlap");
  AttnStepArgs a{};
  a.q = operand(q, 1);
  a.k = operand(k, 1);
  a.v = operand(v, 1);
  a.out = out.data_ptr();
  a.log_decay = g.data_ptr<float>();
  a.g_stride = s.H > 1 ? g.stride(0) : 0;
  if (done.has_value()) {
    a.done = (const unsigned char*)done->data_ptr();
    a.done_sb = s.B > 1 ? done->stride(0) : 0;
  }
  a.s = state.data_ptr<float>();
  a.d = out_state.data_ptr<float>();
  a.s_sb = s.B > 1 ? state.stride(0) : 0;
  a.d_sb = s.B > 1 ? out_state.stride(0) : 0;
  a.scale = (float)scale;
  a.B = (int)s.B;
  a.H = (int)s.H;
  a.dk = (int)s.dk;
  a.dv = (int)s.dv;
  const bool vec = s.dv % 4 == 0 && ((uintptr_t)a.s & 15) == 0 &&
                   ((uintptr_t)a.d & 15) == 0 && a.s_sb % 4 == 0 &&
                   a.d_sb % 4 == 0;
  launch_attn_step(type, &a, vec, stream_here());
  check_launch("linear_attention_step");
  return out;
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

// tiles of one product of one matrix, and the blocks that share a tile's k
void plan_product(ns::Args& a, int mode, int tile) {
  const int ks = tile == 64 ? 64 : 32;
  long total = 0;
  for (int i = 0; i < a.count; ++i) {
    ns::Mat& m = a.mat[i];
    const int tm = m.mp / tile, tn = m.np / tile;
    m.tiles = mode == 2 ? tm * tn : tm * (tm + 1) / 2;
    total += m.tiles;
  }
  int blocks = 0;
  for (int i = 0; i < a.count; ++i) {
    ns::Mat& m = a.mat[i];
    // two blocks a CU fit; a block keeps 256 values of k at least, so that
    // adding the parts does not outweigh them
    const long steps = (mode == 0 ? m.np : m.mp) / ks;
    long s = total >= 512 ? 1 : 512 / total;
    const long most = steps * ks / 256;
    if (s > most) s = most;
    m.splits = (int)(s < 1 ? 1 : s);
    a.first[i] = blocks;
    blocks += m.tiles * m.splits;
  }
  a.first[a.count] = blocks;
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
    ns::Args a{};
    std::vector<size_t> take;
    long tiles128 = 0;
    for (; at < src.size() && take.size() < ns::MAX_MATS; ++at) {
      if (src[at].numel() == 0) continue;
      take.push_back(at);
      tiles128 += ((src[at].size(0) + 127) / 128) *
                  ((src[at].size(1) + 127) / 128);
    }
    if (take.empty()) break;
    const Tensor& like = src[take[0]];
    const c10::DeviceGuard guard(like.device());
    hipStream_t stream = stream_here();
    // a tile of 128 needs half the reads of 64, if there are enough of them
    const int tile = tiles128 >= 256 ? 128 : 64;
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
    long partial = 1, arrived = 1;
    for (int mode = 0; mode < 3; ++mode) {
      plan_product(a, mode, tile);
      long p = 0, n = 0;
      for (int i = 0; i < a.count; ++i) {
        n += a.mat[i].tiles;
        if (a.mat[i].splits > 1)
          p += (long)a.mat[i].tiles * a.mat[i].splits * tile * tile;
      }
      partial = p > partial ? p : partial;
      arrived = n > arrived ? n : arrived;
    }
    auto work = torch::empty({parts}, like.options().dtype(torch::kFloat16));
    auto split = torch::empty({partial},
                              like.options().dtype(torch::kFloat32));
    auto count = torch::zeros({arrived}, like.options().dtype(torch::kInt32));
    auto sums = torch::empty({(long)a.count * ns::NORM_BLOCKS},
                             like.options().dtype(torch::kFloat64));
    auto rho = torch::empty({a.count}, like.options().dtype(torch::kFloat32));
    a.parts = (_Float16*)work.data_ptr();
    a.partial = split.data_ptr<float>();
    a.arrived = count.data_ptr<int>();
    a.sums = sums.data_ptr<double>();
    a.rho = rho.data_ptr<float>();
    a.eps = eps;
    launch_ns_start(&a, stream);
    for (long k = 0; k < steps; ++k) {
      a.round = (int)k;
      a.last = k + 1 == steps;
      for (int mode = 0; mode < 3; ++mode) {
        plan_product(a, mode, tile);
        long p = 0;
        int n = 0;
        for (int i = 0; i < a.count; ++i) {
          a.part_off[i] = p;
          a.arrive_off[i] = n;
          n += a.mat[i].tiles;
          if (a.mat[i].splits > 1)
            p += (long)a.mat[i].tiles * a.mat[i].splits * tile * tile;
        }
        launch_ns_product(mode, tile, &a, stream);
      }
    }
    check_launch("orthogonalize");
  }
}

}  // namespace

void register_core_ops(pybind11::module_& m) {
  m.def("orthogonalize", &orthogonalize, py::arg("src"), py::arg("dst"),
        py::arg("steps"), py::arg("eps"));
  m.def("linear_attention_fwd", &linear_attention_fwd, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("done"),
        py::arg("state"), py::arg("scale"));
  m.def("linear_attention_bwd", &linear_attention_bwd, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("done"),
        py::arg("state"), py::arg("entry"), py::arg("d_out"),
        py::arg("d_final"), py::arg("scale"), py::arg("need_dstate"));
  m.def("linear_attention_step", &linear_attention_step, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("log_decay"), py::arg("state"),
        py::arg("out_state"), py::arg("done"), py::arg("scale"));
  m.def("layer_norm_fwd", &layer_norm_fwd, py::arg("x"),
        py::arg("weight") = py::none(), py::arg("bias") = py::none(),
        py::arg("eps") = 1e-5, py::arg("save") = false);
  m.def("layer_norm_bwd", &layer_norm_bwd, py::arg("dy"), py::arg("x"),
        py::arg("weight"), py::arg("stats"), py::arg("need_dx"),
        py::arg("need_dw"), py::arg("need_db"), py::arg("param_fp32"));
}
