// sequence_autograd.cpp -- packed attention, the rotary embedding and the
// linear cross entropy as autograd nodes (host code only; why in C++:
// block_autograd.cpp). sequence.py and loss.py check the arguments and bind the
// library's entry points at load.
#include "autograd_common.h"


namespace {

struct Entry {
  decltype(&dsx_last_error) last_error;
  decltype(&dsx_stream_capturing) stream_capturing;
  decltype(&dsx_attention_forward) attention_forward;
  decltype(&dsx_attention_workspace_bytes) attention_workspace_bytes;
  decltype(&dsx_attention_backward) attention_backward;
  decltype(&dsx_rotary) rotary;
  decltype(&dsx_loss_saved_bytes) loss_saved_bytes;
  decltype(&dsx_loss_workspace_bytes) loss_workspace_bytes;
  decltype(&dsx_loss_forward) loss_forward;
  decltype(&dsx_loss_backward) loss_backward;
} entry{};

void check(const char* name, int rc) { check_status(name, rc, entry.last_error); }
Tensor scratch(int64_t bytes, const Tensor& like) { return scratch_of(bytes, like, entry.last_error); }
void* stream_at(int64_t s) { return reinterpret_cast<void*>(s); }

// The stream of a backward pass. One under capture is refused before autograd
// gets to the leaves: where an eager graph of theirs lives, its accumulation nodes
// belong to another stream, and the captured pass ends the process.
void* backward_stream(const char* name, AutogradContext* ctx) {
  void* s = stream_at(ctx->saved_data["stream"].toInt());
  if (entry.stream_capturing(s))
    throw std::runtime_error(std::string(name) + ": a backward pass cannot be captured into a graph (a forward can)");
  return s;
}

// ---- attention ----------------------------------------------------------------

// t [tokens, heads, d] as the kernels take it: features adjacent, 16-byte
// aligned rows and heads that do not overlap. Else a copy, whose heads are
// filled up with zeros to a multiple of eight features.
Tensor heads_of(const Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2);
  const int64_t sn = n > 1 ? t.stride(0) : 0, sh = h > 1 ? t.stride(1) : 0;
  if (d % 8 == 0 && t.stride(2) == 1 && sn % 8 == 0 && sh % 8 == 0 && (n < 2 || (sn >= d && sn <= DSX_ATTENTION_MAX_STRIDE)) &&
      (h < 2 || sh >= d) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0)
    return t;
  const auto o = t.options().requires_grad(false);
  if (d % 8 == 0) {
    Tensor c = at::empty({n, h, d}, o);
    return c.copy_(t.detach());
  }
  Tensor c = at::zeros({n, h, (d + 7) / 8 * 8}, o);
  c.narrow(2, 0, d).copy_(t.detach());
  return c;
}
// A result of `d` features a head, without the ones that were filled up.
Tensor first_features(const Tensor& t, int64_t d) {
  return !t.defined() || t.size(2) == d ? t : t.narrow(2, 0, d).contiguous();
}
// A result for all rows of `like`; those behind the sequences hold zeros.
Tensor rows_for(const Tensor& like, int64_t tokens) {
  Tensor t = at::empty({like.size(0), like.size(1), like.size(2)}, like.options().requires_grad(false));
  if (t.size(0) > tokens) t.narrow(0, tokens, t.size(0) - tokens).zero_();
  return t;
}

struct Sequences {
  Tensor tiles;  // int32 [2, count, 4] on the device
  int64_t tokens, longest, pairs;
};

DsxAttention describe(const Tensor& q, const Tensor& k, const Tensor& v, const Sequences& s, bool causal,
                      double scale) {
  DsxAttention a{};
  auto row = [](const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1) * t.size(2); };
  auto head = [](const Tensor& t) { return t.size(1) > 1 ? t.stride(1) : t.size(2); };
  a.q = at_of(q);
  a.k = at_of(k);
  a.v = at_of(v);
  a.ld_q = row(q);
  a.ld_k = row(k);
  a.ld_v = row(v);
  a.head_q = head(q);
  a.head_k = head(k);
  a.head_v = head(v);
  a.tokens = s.tokens;
  a.tiles = static_cast<const int32_t*>(at_of(s.tiles));
  a.tile_count = s.tiles.size(1);
  a.heads = static_cast<int32_t>(q.size(1));
  a.kv_heads = static_cast<int32_t>(k.size(1));
  a.head_dim = static_cast<int32_t>(q.size(2));
  a.dtype = code_of(q.scalar_type());
  a.causal = causal;
  a.scale = static_cast<float>(scale);
  a.longest = s.longest;
  a.pairs = s.pairs;
  return a;
}

struct Kept {
  Tensor q, k, v, out, out_lo, lse;
};
Kept attention_run(const Tensor& q, const Tensor& k, const Tensor& v, const Sequences& s, bool causal, double scale,
                   int64_t stream, bool keep) {
  const c10::DeviceGuard guard(q.device());
  Kept r{heads_of(q), heads_of(k), heads_of(v), {}, {}, {}};
  r.out = rows_for(r.q, s.tokens);
  if (keep) {
    r.out_lo = at::empty({s.tokens, r.q.size(1), r.q.size(2)}, r.q.options().requires_grad(false));
    r.lse = at::empty({r.q.size(1), s.tokens}, r.q.options().dtype(at::kFloat).requires_grad(false));
  }
  const DsxAttention a = describe(r.q, r.k, r.v, s, causal, scale);
  check("dsx_attention_forward",
        entry.attention_forward(&a, at_of(r.out), at_of(r.out_lo), static_cast<float*>(at_of(r.lse)), stream_at(stream)));
  return r;
}

struct PackedAttention : torch::autograd::Function<PackedAttention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tiles,
                        int64_t tokens, int64_t longest, int64_t pairs, bool causal, double scale, int64_t stream) {
    const Kept r = attention_run(q, k, v, {tiles, tokens, longest, pairs}, causal, scale, stream, true);
    ctx->save_for_backward({r.q, r.k, r.v, r.out, r.out_lo, r.lse, tiles});
    ctx->saved_data["tokens"] = tokens;
    ctx->saved_data["longest"] = longest;
    ctx->saved_data["pairs"] = pairs;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["d"] = q.size(2);
    ctx->saved_data["stream"] = stream;
    return first_features(r.out, q.size(2));
  }
  // On the forward's stream, which autograd makes current here.
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    void* stream = backward_stream("packed_attention", ctx);
    Tensor dq, dk, dv;
    if (grads[0].defined()) {
      const c10::DeviceGuard guard(s[0].device());
      const Sequences seq{s[6], ctx->saved_data["tokens"].toInt(), ctx->saved_data["longest"].toInt(),
                          ctx->saved_data["pairs"].toInt()};
      const int64_t d = ctx->saved_data["d"].toInt();
      const DsxAttention a = describe(s[0], s[1], s[2], seq, ctx->saved_data["causal"].toBool(),
                                      ctx->saved_data["scale"].toDouble());
      const Tensor dout = heads_of(grads[0]);
      const bool keys = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
      if (ctx->needs_input_grad(0)) dq = rows_for(s[0], seq.tokens);
      if (keys) {
        dk = rows_for(s[1], seq.tokens);
        dv = rows_for(s[2], seq.tokens);
      }
      Tensor work = scratch(entry.attention_workspace_bytes(&a), s[0]);
      check("dsx_attention_backward",
            entry.attention_backward(&a, at_of(s[3]), at_of(s[4]), static_cast<const float*>(at_of(s[5])), at_of(dout),
                                     dout.size(0) > 1 ? dout.stride(0) : dout.size(1) * dout.size(2),
                                     dout.size(1) > 1 ? dout.stride(1) : dout.size(2), at_of(dq), at_of(dk), at_of(dv),
                                     at_of(work), work.numel(), stream));
      dq = first_features(dq, d);
      dk = ctx->needs_input_grad(1) ? first_features(dk, d) : Tensor();
      dv = ctx->needs_input_grad(2) ? first_features(dv, d) : Tensor();
    }
    return once({dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor packed_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tiles, int64_t tokens,
                        int64_t longest, int64_t pairs, bool causal, double scale, int64_t stream) {
  for (const Tensor* t : {&q, &k, &v}) refuse_tangent("packed_attention", *t);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return PackedAttention::apply(q, k, v, tiles, tokens, longest, pairs, causal, scale, stream);
  return first_features(attention_run(q, k, v, {tiles, tokens, longest, pairs}, causal, scale, stream, false).out, q.size(2));
}

// ---- rotary --------------------------------------------------------------------

// t [tokens, heads, d] with adjacent features, or a copy.
Tensor features_of(const Tensor& t) {
  return t.size(2) < 2 || t.stride(2) == 1 ? t : t.contiguous();
}

struct Turn {
  Tensor positions;
  double base;
  int64_t dims;
  bool interleaved;
};
variable_list rotary_run(const Tensor& q_, const Tensor& k_, const Turn& r, bool inverse, int64_t stream) {
  const Tensor q = q_.defined() ? features_of(q_) : q_, k = k_.defined() ? features_of(k_) : k_;
  const Tensor& first = q.defined() ? q : k;
  const Tensor second = q.defined() ? k : Tensor();  // one of the two alone: as q
  const c10::DeviceGuard guard(first.device());
  auto empty = [](const Tensor& t) {
    return t.defined() ? at::empty({t.size(0), t.size(1), t.size(2)}, t.options().requires_grad(false)) : Tensor();
  };
  Tensor a = empty(first), b = empty(second);
  DsxRotary d{};
  d.q = at_of(first);
  d.k = at_of(second);
  d.positions = at_of(r.positions);
  d.ld_q = first.stride(0);
  d.head_q = first.stride(1);
  d.ld_k = second.defined() ? second.stride(0) : 0;
  d.head_k = second.defined() ? second.stride(1) : 0;
  d.tokens = first.size(0);
  d.heads = static_cast<int32_t>(first.size(1));
  d.kv_heads = second.defined() ? static_cast<int32_t>(second.size(1)) : 0;
  d.head_dim = static_cast<int32_t>(first.size(2));
  d.dims = static_cast<int32_t>(r.dims);
  d.dtype = code_of(first.scalar_type());
  d.interleaved = r.interleaved;
  d.position_bytes = r.positions.scalar_type() == at::kLong ? 8 : 4;
  d.base = r.base;
  check("dsx_rotary", entry.rotary(&d, at_of(a), at_of(b), inverse, stream_at(stream)));
  if (q.defined()) return {a, b};
  return {Tensor(), a};
}

struct Rotary : torch::autograd::Function<Rotary> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& positions,
                               double base, int64_t dims, bool interleaved, int64_t stream) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({positions});
    ctx->saved_data["base"] = base;
    ctx->saved_data["dims"] = dims;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["stream"] = stream;
    return rotary_run(q, k, {positions, base, dims, interleaved}, false, stream);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    (void)backward_stream("rotary", ctx);
    const Turn r{ctx->get_saved_variables()[0], ctx->saved_data["base"].toDouble(), ctx->saved_data["dims"].toInt(),
                 ctx->saved_data["interleaved"].toBool()};
    Tensor dq = ctx->needs_input_grad(0) ? grads[0] : Tensor(), dk = ctx->needs_input_grad(1) ? grads[1] : Tensor();
    if (dq.defined() || dk.defined()) {
      variable_list out = rotary_run(dq, dk, r, true, ctx->saved_data["stream"].toInt());
      dq = out[0];
      dk = out[1];
    }
    return once({dq, dk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

std::pair<Tensor, Tensor> rotary(const Tensor& q, const Tensor& k, const Tensor& positions, double base, int64_t dims,
                                 bool interleaved, int64_t stream) {
  for (const Tensor* t : {&q, &k}) refuse_tangent("rotary", *t);
  variable_list out = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad())
                          ? Rotary::apply(q, k, positions, base, dims, interleaved, stream)
                          : rotary_run(q, k, {positions, base, dims, interleaved}, false, stream);
  return {out[0], out[1]};
}

// ---- the loss --------------------------------------------------------------------

struct LossOptions {
  int64_t ignore, reduction;
};
DsxLoss describe(const Tensor& x, const Tensor& w, const Tensor& targets, const LossOptions& o) {
  DsxLoss q{};
  q.x = at_of(x);
  q.weight = at_of(w);
  q.targets = at_of(targets);
  q.ld_x = x.defined() ? ld_of(x) : 0;
  q.ld_weight = ld_of(w);
  q.tokens = targets.size(0);
  q.width = w.size(1);
  q.vocab = w.size(0);
  q.ignore_index = o.ignore;
  q.dtype = code_of(w.scalar_type());
  q.target_bytes = targets.scalar_type() == at::kLong ? 8 : 4;
  q.reduction = static_cast<int32_t>(o.reduction);
  return q;
}

Tensor loss_run(const Tensor& x, const Tensor& w, const Tensor& targets, const LossOptions& o, int64_t stream,
                Tensor* kept) {
  const c10::DeviceGuard guard(w.device());
  const auto fp32 = w.options().dtype(at::kFloat).requires_grad(false);
  Tensor loss = o.reduction == DSX_REDUCE_NONE ? at::empty({targets.size(0)}, fp32) : at::empty({}, fp32);
  DsxLoss q = describe(x, w, targets, o);
  Tensor saved = scratch(entry.loss_saved_bytes(&q), w), work = scratch(entry.loss_workspace_bytes(&q, 0), w);
  if (targets.size(0) || o.reduction != DSX_REDUCE_NONE) {
    q.saved = at_of(saved);
    q.workspace = at_of(work);
    q.workspace_bytes = work.numel();
    check("dsx_loss_forward", entry.loss_forward(&q, static_cast<float*>(at_of(loss)), stream_at(stream)));
  }
  if (kept) *kept = saved;
  return loss;
}

struct LinearCrossEntropy : torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x_, const Tensor& w_, const Tensor& targets, int64_t ignore,
                        int64_t reduction, int64_t stream) {
    const Tensor x = rows_of(x_), w = rows_of(w_);
    Tensor saved;
    Tensor loss = loss_run(x, w, targets, {ignore, reduction}, stream, &saved);
    ctx->save_for_backward({w, targets, saved});
    ctx->saved_data["ignore"] = ignore;
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["stream"] = stream;
    return loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto s = ctx->get_saved_variables();
    void* stream = backward_stream("linear_cross_entropy", ctx);
    Tensor dx, dw;
    if (grads[0].defined()) {
      const c10::DeviceGuard guard(s[0].device());
      const Tensor d_loss = grads[0].contiguous();
      DsxLoss q = describe({}, s[0], s[1], {ctx->saved_data["ignore"].toInt(), ctx->saved_data["reduction"].toInt()});
      const auto o = s[0].options().requires_grad(false);
      if (ctx->needs_input_grad(0)) dx = at::empty({q.tokens, q.width}, o);
      if (ctx->needs_input_grad(1))
        dw = q.tokens ? at::empty({q.vocab, q.width}, o) : at::zeros({q.vocab, q.width}, o);
      if (q.tokens) {
        Tensor work = scratch(entry.loss_workspace_bytes(&q, 1), s[0]);
        q.saved = at_of(s[2]);
        q.workspace = at_of(work);
        q.workspace_bytes = work.numel();
        check("dsx_loss_backward", entry.loss_backward(&q, static_cast<const float*>(at_of(d_loss)), at_of(dx), at_of(dw),
                                                       stream));
      }
    }
    return once({dx, dw, Tensor(), Tensor(), Tensor(), Tensor()});
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& w, const Tensor& targets, int64_t ignore, int64_t reduction,
                            int64_t stream) {
  for (const Tensor* t : {&x, &w}) refuse_tangent("linear_cross_entropy", *t);
  const Tensor y = targets.contiguous();
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad()))
    return LinearCrossEntropy::apply(x, w, y, ignore, reduction, stream);
  return loss_run(rows_of(x), rows_of(w), y, {ignore, reduction}, stream, nullptr);
}

}  // namespace

PYBIND11_MODULE(_sequence_autograd, m) {
  m.def("bind", [](const pybind11::dict& d) {
    bind_one(entry.last_error, d, "dsx_last_error");
    bind_one(entry.stream_capturing, d, "dsx_stream_capturing");
    bind_one(entry.attention_forward, d, "dsx_attention_forward");
    bind_one(entry.attention_workspace_bytes, d, "dsx_attention_workspace_bytes");
    bind_one(entry.attention_backward, d, "dsx_attention_backward");
    bind_one(entry.rotary, d, "dsx_rotary");
    bind_one(entry.loss_saved_bytes, d, "dsx_loss_saved_bytes");
    bind_one(entry.loss_workspace_bytes, d, "dsx_loss_workspace_bytes");
    bind_one(entry.loss_forward, d, "dsx_loss_forward");
    bind_one(entry.loss_backward, d, "dsx_loss_backward");
  });
  m.def("packed_attention", &packed_attention);
  m.def("rotary", &rotary);
  m.def("linear_cross_entropy", &linear_cross_entropy);
}
