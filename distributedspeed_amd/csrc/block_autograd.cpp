// block_autograd.cpp -- the block operators as autograd nodes (host code only).
//
// A backward pass runs on autograd's own thread. As Python functions the nodes
// of gated_residual_norm took 143 us of host time forward and backward for 30
// us of GPU work (2048 x 768, fp32), most of it in that thread: waking it, its
// wait for the interpreter lock, and Python at half speed on a cold core. Here
// both directions are C++: the wrappers in block.py check the arguments, this
// file allocates the results and calls the library's entry points, whose
// addresses block.py binds at load.
#include "autograd_common.h"

namespace {

struct Entry {
  decltype(&dsx_last_error) last_error;
  decltype(&dsx_ffn_saved_bytes) ffn_saved_bytes;
  decltype(&dsx_ffn_workspace_bytes) ffn_workspace_bytes;
  decltype(&dsx_ffn_forward) ffn_forward;
  decltype(&dsx_ffn_backward) ffn_backward;
  decltype(&dsx_norm_workspace_bytes) norm_workspace_bytes;
  decltype(&dsx_norm_forward) norm_forward;
  decltype(&dsx_norm_backward) norm_backward;
} entry{};

void check(const char* name, int rc) { check_status(name, rc, entry.last_error); }
Tensor scratch(int64_t bytes, const Tensor& like) { return scratch_of(bytes, like, entry.last_error); }
// A gradient; zeros where nothing is written because there is no row.
Tensor gradient(const Tensor& like, bool wanted, bool rows) {
  if (!wanted || !like.defined()) return {};
  const auto o = like.options().requires_grad(false);
  return rows ? at::empty(like.sizes(), o) : at::zeros(like.sizes(), o);
}

// ---- the gated feed-forward block ------------------------------------------

DsxFfn describe(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, bool keep) {
  DsxFfn q{};
  q.x = at_of(x);
  q.w_gate = at_of(wg);
  q.w_up = at_of(wu);
  q.w_down = at_of(wd);
  q.ld_x = ld_of(x);
  q.ld_gate = ld_of(wg);
  q.ld_up = ld_of(wu);
  q.ld_down = ld_of(wd);
  q.tokens = x.size(0);
  q.width = wg.size(1);
  q.inner = wg.size(0);
  q.dtype = code_of(x.scalar_type());
  q.activation = static_cast<int32_t>(act);
  q.keep = keep;
  return q;
}

Tensor ffn_run(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, bool keep,
               int64_t stream, Tensor* kept) {
  const c10::DeviceGuard guard(x.device());
  Tensor y = result(x);
  DsxFfn q = describe(x, wg, wu, wd, act, keep);
  Tensor saved = scratch(entry.ffn_saved_bytes(q.tokens, q.inner, keep), x);
  Tensor work = scratch(entry.ffn_workspace_bytes(&q, 0), x);
  q.saved = at_of(saved);
  q.workspace = at_of(work);
  q.workspace_bytes = work.numel();
  check("dsx_ffn_forward", entry.ffn_forward(&q, at_of(y), y.size(1), reinterpret_cast<void*>(stream)));
  if (kept) *kept = saved;
  return y;
}

struct GatedFfn : torch::autograd::Function<GatedFfn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& wg_, const Tensor& wu_,
                        const Tensor& wd_, int64_t act, int64_t stream) {
    const Tensor x = rows_of(x_), wg = rows_of(wg_), wu = rows_of(wu_), wd = rows_of(wd_);
    Tensor saved;
    Tensor y = ffn_run(x, wg, wu, wd, act, true, stream, &saved);
    ctx->save_for_backward({x, wg, wu, wd, saved});
    ctx->saved_data["act"] = act;
    ctx->saved_data["stream"] = stream;
    return y;
  }
  // On the forward's stream, which autograd makes current here.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor dy = rows_of(grads[0]);
    const c10::DeviceGuard guard(s[0].device());
    DsxFfn q = describe(s[0], s[1], s[2], s[3], ctx->saved_data["act"].toInt(), true);
    Tensor out[4];
    for (int k = 0; k < 4; k++) out[k] = gradient(s[k], ctx->needs_input_grad(k), q.tokens != 0);
    if (dy.defined()) {
      Tensor work = scratch(entry.ffn_workspace_bytes(&q, 1), dy);
      q.saved = at_of(s[4]);
      q.workspace = at_of(work);
      q.workspace_bytes = work.numel();
      check("dsx_ffn_backward",
            entry.ffn_backward(&q, at_of(dy), ld_of(dy), at_of(out[0]), s[0].size(1), at_of(out[1]), at_of(out[2]),
                               at_of(out[3]), reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())));
    } else {
      for (auto& o : out) o = Tensor();
    }
    return once({out[0], out[1], out[2], out[3], Tensor(), Tensor()});
  }
};

Tensor gated_ffn(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, int64_t stream) {
  for (const Tensor* t : {&x, &wg, &wu, &wd}) refuse_tangent("gated_ffn", *t);
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || wg.requires_grad() || wu.requires_grad() || wd.requires_grad()))
    return GatedFfn::apply(x, wg, wu, wd, act, stream);
  return ffn_run(rows_of(x), rows_of(wg), rows_of(wu), rows_of(wd), act, false, stream, nullptr);
}

// ---- the norms around a block ------------------------------------------------

using MaybeTensor = std::optional<Tensor>;
Tensor or_undefined(const MaybeTensor& t) { return t ? *t : Tensor(); }

DsxNorm describe(const Tensor* in, double alpha, double beta, double eps, const Tensor& rstd) {
  DsxNorm q{};
  q.residual = at_of(in[0]);
  q.branch = at_of(in[1]);
  q.post_weight = at_of(in[2]);
  q.gate = at_of(in[3]);
  q.next_weight = at_of(in[4]);
  q.ld_residual = ld_of(in[0]);
  q.ld_branch = ld_of(in[1]);
  q.rows = in[0].size(0);
  q.width = in[0].size(1);
  q.gate_rows = in[3].defined() ? in[3].numel() / q.width : 0;
  q.dtype = code_of(in[0].scalar_type());
  q.branch_scale = static_cast<float>(alpha);
  q.residual_scale = static_cast<float>(beta);
  q.eps = static_cast<float>(eps);
  q.rstd = static_cast<float*>(at_of(rstd));
  return q;
}

// in: residual, branch, post_weight, gate, next_weight; made contiguous where needed.
variable_list norm_run(Tensor* in, double alpha, double beta, double eps, int64_t stream, bool keep, Tensor* kept) {
  const c10::DeviceGuard guard(in[0].device());
  for (int k = 0; k < 5; k++)
    if (in[k].defined()) in[k] = k < 2 ? rows_of(in[k]) : in[k].contiguous();
  Tensor hidden = result(in[0]), normed = in[4].defined() ? result(in[0]) : Tensor(), rstd;
  if (keep) rstd = at::empty({2, in[0].size(0)}, in[0].options().dtype(at::kFloat).requires_grad(false));
  const DsxNorm q = describe(in, alpha, beta, eps, rstd);
  check("dsx_norm_forward", entry.norm_forward(&q, at_of(hidden), at_of(normed), reinterpret_cast<void*>(stream)));
  if (kept) *kept = rstd;
  return {hidden, normed};
}

struct GatedResidualNorm : torch::autograd::Function<GatedResidualNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& residual, const MaybeTensor& branch,
                               const MaybeTensor& post, const MaybeTensor& gate, const MaybeTensor& next, double alpha,
                               double beta, double eps, int64_t stream) {
    Tensor in[5] = {residual, or_undefined(branch), or_undefined(post), or_undefined(gate), or_undefined(next)}, rstd;
    variable_list out = norm_run(in, alpha, beta, eps, stream, true, &rstd);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({in[0], in[1], in[2], in[3], in[4], rstd});
    ctx->saved_data["scales"] = std::vector<double>{alpha, beta, eps};
    ctx->saved_data["stream"] = stream;
    if (!out[1].defined()) out.pop_back();
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    const Tensor dh = rows_of(grads[0]), dn = grads.size() > 1 ? rows_of(grads[1]) : Tensor();
    Tensor out[5];
    if (dh.defined() || dn.defined()) {
      const c10::DeviceGuard guard(s[0].device());
      const auto scales = ctx->saved_data["scales"].toDoubleVector();
      const DsxNorm q = describe(s.data(), scales[0], scales[1], scales[2], s[5]);
      size_t edge = 0;  // an input that is not there has none
      for (int k = 0; k < 5; k++)
        if (s[k].defined()) out[k] = gradient(s[k], ctx->needs_input_grad(edge++), q.rows != 0);
      Tensor work = scratch(entry.norm_workspace_bytes(&q), s[0]);
      check("dsx_norm_backward",
            entry.norm_backward(&q, at_of(dh), ld_of(dh), at_of(dn), ld_of(dn), at_of(out[0]), at_of(out[1]),
                                at_of(out[2]), at_of(out[3]), at_of(out[4]), at_of(work), work.numel(),
                                reinterpret_cast<void*>(ctx->saved_data["stream"].toInt())));
    }
    return once({out[0], out[1], out[2], out[3], out[4], Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::pair<Tensor, MaybeTensor> gated_residual_norm(const Tensor& residual, const MaybeTensor& branch,
                                                   const MaybeTensor& post, const MaybeTensor& gate,
                                                   const MaybeTensor& next, double alpha, double beta, double eps,
                                                   int64_t stream) {
  Tensor in[5] = {residual, or_undefined(branch), or_undefined(post), or_undefined(gate), or_undefined(next)};
  for (const auto& t : in) refuse_tangent("gated_residual_norm", t);
  bool wanted = false;
  for (const auto& t : in) wanted = wanted || (t.defined() && t.requires_grad());
  variable_list out = wanted && at::GradMode::is_enabled()
                          ? GatedResidualNorm::apply(residual, branch, post, gate, next, alpha, beta, eps, stream)
                          : norm_run(in, alpha, beta, eps, stream, false, nullptr);
  if (out.size() < 2 || !out[1].defined()) return {out[0], std::nullopt};
  return {out[0], out[1]};
}

}  // namespace

PYBIND11_MODULE(_block_autograd, m) {
  m.def("bind", [](const pybind11::dict& d) {
    bind_one(entry.last_error, d, "dsx_last_error");
    bind_one(entry.ffn_saved_bytes, d, "dsx_ffn_saved_bytes");
    bind_one(entry.ffn_workspace_bytes, d, "dsx_ffn_workspace_bytes");
    bind_one(entry.ffn_forward, d, "dsx_ffn_forward");
    bind_one(entry.ffn_backward, d, "dsx_ffn_backward");
    bind_one(entry.norm_workspace_bytes, d, "dsx_norm_workspace_bytes");
    bind_one(entry.norm_forward, d, "dsx_norm_forward");
    bind_one(entry.norm_backward, d, "dsx_norm_backward");
  });
  m.def("gated_ffn", &gated_ffn);
  m.def("gated_residual_norm", &gated_residual_norm);
}
