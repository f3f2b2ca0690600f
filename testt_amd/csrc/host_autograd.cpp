// Host side of the operators around the decoder layer, with their autograd nodes: token_logprobs,
// qk_norm_rope, dropout, embedding.
//
// Each is one native call forward -- checks, allocations, launch and, when a gradient may be asked
// for, the node -- and a native node backward.  Reason: autograd runs the backward of device tensors
// on a worker thread of its own; a node written in Python takes the interpreter to that thread, which
// cost 40 - 75 us a backward on MI355X boxes beside the 25 us of the hand-over itself (eager forward
// + backward: dropout of 888 rows 90 us, q/k norm 133, log probabilities of 333 rows 133, against 32,
// 61 and 67 with the worker thread off).
//
// As the operators of host_ops.cpp, they take plain arguments of the expected types, contiguous, on
// one device, with matching shapes, and return None for anything else; the Python caller then checks,
// converts or raises.  The device of the tensors is made current around the launches.

#include <algorithm>
#include <cmath>
#include <optional>
#include <utility>
#include <vector>

#include "host_args.hpp"
#include "host_autograd.hpp"

namespace soupk_host {
namespace {

// ---- token_logprobs -----------------------------------------------------------------------------

constexpr int64_t kMaxTop = 32;

struct LogitRows {
  int64_t rows, inner, outer_stride, inner_stride, vocab;
};

LogitRows logit_rows(const Tensor& z) {
  const int64_t d = z.dim();
  if (d == 2) return {z.size(0), std::max<int64_t>(z.size(0), 1), 0, z.stride(0), z.size(1)};
  return {z.size(0) * z.size(1), std::max<int64_t>(z.size(1), 1), z.stride(0), z.stride(1),
          z.size(2)};
}

// (logprob, entropy, top_logprobs, top_ids), and the row statistics of the backward when asked.
variable_list logprobs_forward(const Tensor& z, const Tensor& tok, int64_t k, double temperature,
                               Tensor* stats) {
  const c10::DeviceGuard guard(z.device());
  const LogitRows r = logit_rows(z);
  const at::Device dev = z.device();
  std::vector<int64_t> top(tok.sizes().begin(), tok.sizes().end());
  top.push_back(k);
  Tensor lp = empty(tok.sizes(), at::kFloat, dev), ent = empty(tok.sizes(), at::kFloat, dev);
  Tensor top_lp = empty(top, at::kFloat, dev), top_id = empty(top, at::kLong, dev);
  if (stats) *stats = empty({2, r.rows}, at::kFloat, dev);
  if (r.rows > 0) {
    const int32_t code = code_of(z.scalar_type());
    int64_t need = 0;
    check("soupk_token_logprobs_workspace",
          p_soupk_token_logprobs_workspace(r.rows, r.vocab, static_cast<int32_t>(k), code, &need));
    Tensor ws;
    if (need > 0) ws = empty({need}, at::kByte, dev);
    float* const st = stats ? address<float>(*stats) : nullptr;
    check("soupk_token_logprobs_fwd",
          p_soupk_token_logprobs_fwd(
              address(z), code, address<int64_t>(tok), r.rows, r.inner, r.outer_stride,
              r.inner_stride, r.vocab, static_cast<float>(temperature), static_cast<int32_t>(k),
              address<float>(lp), address<float>(ent), st, st ? st + r.rows : nullptr,
              address<float>(top_lp), address<int64_t>(top_id), address(ws), need, stream_of(z)));
  }
  return {lp, ent, top_lp, top_id};
}

struct Logprobs : Function<Logprobs> {
  static variable_list forward(AutogradContext* ctx, Tensor z, Tensor tok, int64_t k,
                               double temperature) {
    Tensor stats;
    variable_list out = logprobs_forward(z, tok, k, temperature, &stats);
    ctx->save_for_backward({z, tok, stats, out[1], out[3]});
    ctx->saved_data["k"] = k;
    ctx->saved_data["t"] = temperature;
    ctx->mark_non_differentiable({out[3]});
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (!g[0].defined() && !g[1].defined() && !g[2].defined()) return variable_list(4);
    return once([&]() -> variable_list {
      const variable_list s = ctx->get_saved_variables();
      const Tensor &z = s[0], &tok = s[1], &stats = s[2];
      const c10::DeviceGuard guard(z.device());
      const int64_t k = ctx->saved_data["k"].toInt();
      const LogitRows r = logit_rows(z);
      for (int i = 0; i < 3; ++i)
        if (g[i].defined()) g[i] = g[i].to(at::kFloat).contiguous();
      Tensor dz = empty(z.sizes(), z.scalar_type(), z.device());
      const float* const st = address<float>(stats);
      check("soupk_token_logprobs_bwd",
            p_soupk_token_logprobs_bwd(
                address(z), code_of(z.scalar_type()), address<int64_t>(tok), r.rows, r.inner,
                r.outer_stride, r.inner_stride, r.vocab,
                static_cast<float>(ctx->saved_data["t"].toDouble()), static_cast<int32_t>(k), st,
                st + r.rows, address<float>(s[3]), address<int64_t>(s[4]), address<float>(g[0]),
                address<float>(g[1]), k > 0 ? address<float>(g[2]) : nullptr, address(dz),
                stream_of(z)));
      return {dz, Tensor(), Tensor(), Tensor()};
    });
  }
};

// ---- qk_norm_rope -------------------------------------------------------------------------------

struct NormShape {
  int64_t batch, seq, nh, nkv, hd;
  double eps;
};

Tensor qk_norm_forward(const Tensor& qkv, const Tensor& lq, const Tensor& lv, const Tensor& wq,
                       const Tensor& wk, const Tensor& cos, const Tensor& sin, const Tensor& pos,
                       const NormShape& n) {
  const c10::DeviceGuard guard(qkv.device());
  Tensor out = empty(qkv.sizes(), qkv.scalar_type(), qkv.device());
  const Tensor& delta = lq.defined() ? lq : lv;
  const int32_t code = code_of(qkv.scalar_type());
  check("soupk_qk_norm_rope_fwd",
        p_soupk_qk_norm_rope_fwd(
            address(qkv), address(lq), address(lv),
            delta.defined() ? code_of(delta.scalar_type()) : code, address<float>(wq),
            address<float>(wk), address<float>(cos), address<float>(sin), address<int64_t>(pos),
            address(out), code, qkv.size(0), static_cast<int32_t>(n.batch),
            static_cast<int32_t>(n.seq), static_cast<int32_t>(n.nh), static_cast<int32_t>(n.nkv),
            static_cast<int32_t>(n.hd), static_cast<float>(n.eps), stream_of(qkv)));
  return out;
}

struct QkNorm : Function<QkNorm> {
  static Tensor forward(AutogradContext* ctx, Tensor qkv, std::optional<Tensor> lq,
                        std::optional<Tensor> lv, Tensor wq, Tensor wk, Tensor cos, Tensor sin,
                        Tensor pos, NormShape n) {
    const Tensor q = lq.value_or(Tensor()), v = lv.value_or(Tensor());
    ctx->save_for_backward({qkv, q, wq, wk, cos, sin, pos});
    ctx->saved_data["n"] = std::vector<int64_t>{n.batch, n.seq, n.nh, n.nkv, n.hd,
                                                q.defined() && q.requires_grad(),
                                                v.defined() && v.requires_grad(),
                                                wq.requires_grad(), wk.requires_grad()};
    ctx->saved_data["e"] = n.eps;
    return qk_norm_forward(qkv, q, v, wq, wk, cos, sin, pos, n);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once([&]() -> variable_list {
      const variable_list s = ctx->get_saved_variables();
      const Tensor &qkv = s[0], &lq = s[1], &wq = s[2], &wk = s[3];
      const c10::DeviceGuard guard(qkv.device());
      const at::Device dev = qkv.device();
      const std::vector<int64_t> n = ctx->saved_data["n"].toIntVector();
      const int64_t nh = n[2], nkv = n[3], hd = n[4];
      const Tensor dout = g[0].to(qkv.scalar_type()).contiguous();
      Tensor dqkv = empty(qkv.sizes(), qkv.scalar_type(), dev), dwq, dwk, ws;
      if (n[7]) dwq = empty({hd}, at::kFloat, dev);
      if (n[8]) dwk = empty({hd}, at::kFloat, dev);
      const int64_t floats = n[7] || n[8] ? int64_t{SOUPK_QK_NORM_BLOCKS} * hd : 0;
      if (floats > 0) ws = empty({floats}, at::kFloat, dev);
      const int32_t code = code_of(qkv.scalar_type());
      check("soupk_qk_norm_rope_bwd",
            p_soupk_qk_norm_rope_bwd(
                address(dout), address(qkv), address(lq),
                lq.defined() ? code_of(lq.scalar_type()) : code, address<float>(wq),
                address<float>(wk), address<float>(s[4]), address<float>(s[5]),
                address<int64_t>(s[6]), address(dqkv), address<float>(dwq), address<float>(dwk),
                address<float>(ws), floats, code, qkv.size(0), static_cast<int32_t>(n[0]),
                static_cast<int32_t>(n[1]), static_cast<int32_t>(nh), static_cast<int32_t>(nkv),
                static_cast<int32_t>(hd), static_cast<float>(ctx->saved_data["e"].toDouble()),
                stream_of(qkv)));
      // The deltas' gradients are columns of qkv's.  Where they are contiguous (one row, or query heads
      // alone) they are copied: autograd would make such a view a leaf's .grad as it is, and adding to
      // it later would change qkv's.
      auto columns = [&](int64_t from, int64_t n_cols) {
        const Tensor view = dqkv.narrow(1, from, n_cols);
        return view.is_contiguous() ? view.clone() : view;
      };
      Tensor dlq, dlv;
      if (n[5]) dlq = columns(0, nh * hd);
      if (n[6]) dlv = columns((nh + nkv) * hd, nkv * hd);
      return {dqkv, dlq, dlv, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

// ---- dropout ------------------------------------------------------------------------------------

struct Draws {
  double p;
  uint64_t seed, call;
  int64_t limit() const { return static_cast<int64_t>(std::nearbyint(p * 4294967296.0)); }
  float scale() const {
    const int64_t l = limit();
    return l < (int64_t{1} << 32) ? static_cast<float>(4294967296.0 / (4294967296.0 - l)) : 0.f;
  }
};

Tensor dropout_forward(const Tensor& x, const Tensor& residual, at::ScalarType out_type,
                       const Tensor& seed, const Tensor& rows, const Draws& d) {
  const c10::DeviceGuard guard(x.device());
  Tensor out = empty(x.sizes(), out_type, x.device());
  const int64_t cols = x.dim() ? x.size(-1) : 1;
  if (x.numel() > 0)
    check("soupk_dropout",
          p_soupk_dropout(address(x), code_of(x.scalar_type()), address(residual), address(out),
                          code_of(out_type), address<int64_t>(rows), address<int64_t>(seed),
                          static_cast<int64_t>(d.seed), static_cast<int64_t>(d.call), d.limit(),
                          d.scale(), x.numel() / cols, cols, stream_of(x)));
  return out;
}

struct Dropout : Function<Dropout> {
  static Tensor forward(AutogradContext* ctx, Tensor x, std::optional<Tensor> residual,
                        std::optional<Tensor> seed, std::optional<Tensor> rows, Draws d) {
    const Tensor r = residual.value_or(Tensor()), s = seed.value_or(Tensor()),
                 w = rows.value_or(Tensor());
    // (a seed tensor changed before the backward raises there, as any saved tensor does)
    ctx->save_for_backward({s, w});
    ctx->saved_data["d"] = std::vector<int64_t>{
        static_cast<int64_t>(d.seed), static_cast<int64_t>(d.call), x.requires_grad(),
        r.defined() && r.requires_grad(), static_cast<int64_t>(x.scalar_type())};
    ctx->saved_data["p"] = d.p;
    return dropout_forward(x, r, r.defined() ? r.scalar_type() : x.scalar_type(), s, w, d);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once([&]() -> variable_list {
      const variable_list s = ctx->get_saved_variables();
      const std::vector<int64_t> v = ctx->saved_data["d"].toIntVector();
      const Draws d{ctx->saved_data["p"].toDouble(), static_cast<uint64_t>(v[0]),
                    static_cast<uint64_t>(v[1])};
      Tensor dx;
      if (v[2])
        dx = dropout_forward(g[0].contiguous(), Tensor(), static_cast<at::ScalarType>(v[4]), s[0],
                             s[1], d);
      return {dx, v[3] ? g[0] : Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

// ---- embedding ----------------------------------------------------------------------------------

Tensor embedding_forward(const Tensor& ids, const Tensor& table, double scale,
                         at::ScalarType out_type) {
  const c10::DeviceGuard guard(table.device());
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(table.size(1));
  Tensor out = empty(shape, out_type, table.device());
  if (out.numel() > 0)
    check("soupk_embedding_fwd",
          p_soupk_embedding_fwd(address(table), code_of(table.scalar_type()),
                                address<int64_t>(ids), address(out), code_of(out_type),
                                static_cast<float>(scale), ids.numel(), table.size(0),
                                table.size(1), stream_of(table)));
  return out;
}

struct Embedding : Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, Tensor table, Tensor ids, double scale,
                        at::ScalarType out_type, int64_t padding) {
    ctx->save_for_backward({ids});
    ctx->saved_data["v"] = std::vector<int64_t>{table.size(0), table.size(1),
                                                static_cast<int64_t>(table.scalar_type()), padding};
    ctx->saved_data["s"] = scale;
    return embedding_forward(ids, table, scale, out_type);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once([&]() -> variable_list {
      const Tensor ids = ctx->get_saved_variables()[0];
      const std::vector<int64_t> v = ctx->saved_data["v"].toIntVector();
      const int64_t vocab = v[0], width = v[1], tokens = ids.numel();
      const at::ScalarType type = static_cast<at::ScalarType>(v[2]);
      const Tensor dout = g[0].contiguous();
      const c10::DeviceGuard guard(dout.device());
      Tensor dtable = empty({vocab, width}, type, dout.device());
      if (dtable.numel() > 0) {
        int64_t need = 0;
        check("soupk_embedding_bwd_workspace",
              p_soupk_embedding_bwd_workspace(tokens, vocab, width, &need));
        Tensor ws = empty({need}, at::kByte, dout.device());
        check("soupk_embedding_bwd",
              p_soupk_embedding_bwd(address(dout), code_of(dout.scalar_type()),
                                    address<int64_t>(ids), address(dtable), code_of(type),
                                    static_cast<float>(ctx->saved_data["s"].toDouble()), v[3],
                                    address(ws), need, tokens, vocab, width, stream_of(dout)));
      }
      return {dtable, Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

}  // namespace

// token_logprobs(logits, tokens, top_k, temperature) -> (logprob, entropy, top_logprobs, top_ids)
OP(token_logprobs) {
  HANDLE_TH_ERRORS
  ARGS(4);
  const Tensor *z = tensor(a[0]), *tok = tensor(a[1]);
  int64_t k;
  double temperature;
  if (!z || !tok || !integer(a[2], k) || !number(a[3], temperature)) ELSE_PYTHON;
  const int64_t d = z->dim();
  if ((d != 2 && d != 3) || code_of(z->scalar_type()) < 0 || !z->is_cuda()) ELSE_PYTHON;
  const int64_t vocab = z->size(d - 1);
  if (!on(*z, z->device()) || (z->stride(d - 1) != 1 && vocab != 1) || vocab < 1 ||
      !is(*tok, at::kLong, d - 1, z->device()) || tok->sizes() != z->sizes().slice(0, d - 1) ||
      k < 0 || k > std::min(kMaxTop, vocab) || !(temperature >= 1e-30 && temperature <= 1e30))
    ELSE_PYTHON;
  variable_list out;
  {
    const NoGil released;
    out = wants_grad({z}) ? Logprobs::apply(*z, *tok, k, temperature)
                          : logprobs_forward(*z, *tok, k, temperature, nullptr);
  }
  return pack({out[0], out[1], out[2], out[3]});
  END_HANDLE_TH_ERRORS
}

// qk_norm_rope(qkv, lora_q, lora_v, q_weight, k_weight, cos, sin, pos, batch, seq, n_heads, n_kv,
// head_dim, eps) -> rows
OP(qk_norm_rope) {
  HANDLE_TH_ERRORS
  ARGS(14);
  const Tensor *qkv = tensor(a[0]), *wq = tensor(a[3]), *wk = tensor(a[4]), *cos = tensor(a[5]),
               *sin = tensor(a[6]), *pos = tensor(a[7]);
  Tensor lq, lv;
  NormShape s;
  if (!qkv || !wq || !wk || !cos || !sin || !pos || !maybe(a[1], lq) || !maybe(a[2], lv) ||
      !integer(a[8], s.batch) || !integer(a[9], s.seq) || !integer(a[10], s.nh) ||
      !integer(a[11], s.nkv) || !integer(a[12], s.hd) || !number(a[13], s.eps))
    ELSE_PYTHON;
  const at::Device dev = qkv->device();
  const at::ScalarType t = qkv->scalar_type();
  if (s.nh < 1 || s.nh > (1 << 16) || s.nkv < 0 || s.nkv > (1 << 16) || s.hd < 16 || s.hd % 16 ||
      s.hd > 256 || s.batch < 0 || s.seq < 0 || s.batch >= (int64_t{1} << 31) ||
      s.seq >= (int64_t{1} << 31) || s.batch * s.seq >= (int64_t{1} << 31) ||
      !(s.eps >= 0.0 && s.eps <= 3e38) || (t != at::kHalf && t != at::kBFloat16) ||
      !is(*qkv, t, 2, dev) || qkv->size(1) != (s.nh + 2 * s.nkv) * s.hd)
    ELSE_PYTHON;
  const int64_t rows = qkv->size(0);
  const Tensor& delta = lq.defined() ? lq : lv;
  const at::ScalarType dt = delta.defined() ? delta.scalar_type() : t;
  auto table = [&](const Tensor& c) {
    return is(c, at::kFloat, 2, dev) && c.size(0) >= s.seq && c.size(1) == s.hd;
  };
  auto weight = [&](const Tensor& w) { return is(w, at::kFloat, 1, dev) && w.size(0) == s.hd; };
  if ((dt != t && dt != at::kFloat) ||
      (lq.defined() && (!is(lq, dt, 2, dev) || !shape2(lq, rows, s.nh * s.hd))) ||
      (lv.defined() && (!is(lv, dt, 2, dev) || !shape2(lv, rows, s.nkv * s.hd))) ||
      !weight(*wq) || !weight(*wk) || !table(*cos) || !table(*sin) ||
      !is(*pos, at::kLong, 1, dev) || pos->size(0) != rows)
    ELSE_PYTHON;
  Tensor out;
  {
    const NoGil released;
    out = wants_grad({qkv, &lq, &lv, wq, wk})
              ? QkNorm::apply(*qkv, given(lq), given(lv), *wq, *wk, cos->detach(), sin->detach(),
                              *pos, s)
              : qk_norm_forward(*qkv, lq, lv, *wq, *wk, *cos, *sin, *pos, s);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// dropout(x, p, seed, call, rows, residual) -> out
OP(dropout) {
  HANDLE_TH_ERRORS
  ARGS(6);
  const Tensor* x = tensor(a[0]);
  Draws d{0.0, 0, 0};
  Tensor seed, rows, residual;
  if (!x || !number(a[1], d.p) || !word(a[3], d.call) || !maybe(a[4], rows) ||
      !maybe(a[5], residual))
    ELSE_PYTHON;
  if (const Tensor* s = tensor(a[2])) seed = *s;
  else if (!word(a[2], d.seed)) ELSE_PYTHON;
  const at::Device dev = x->device();
  const int64_t cols = x->dim() ? x->size(-1) : 1;
  if (!(d.p >= 0.0 && d.p <= 1.0) || code_of(x->scalar_type()) < 0 || !x->is_cuda() ||
      !on(*x, dev) || !x->is_contiguous() || cols > (int64_t{1} << 32) ||
      (seed.defined() && (!on(seed, dev) || seed.scalar_type() != at::kLong || seed.numel() != 1)))
    ELSE_PYTHON;
  int64_t n_rows = 1;
  for (int64_t i = 0; i + 1 < x->dim(); ++i) n_rows *= x->size(i);
  if ((rows.defined() && (!on(rows, dev) || rows.scalar_type() != at::kLong ||
                          !rows.is_contiguous() || rows.numel() != n_rows)) ||
      (residual.defined() &&
       (!on(residual, dev) || !residual.is_contiguous() || residual.sizes() != x->sizes() ||
        (residual.scalar_type() != x->scalar_type() && residual.scalar_type() != at::kFloat))))
    ELSE_PYTHON;
  Tensor out;
  {
    const NoGil released;
    out = wants_grad({x, &residual})
              ? Dropout::apply(*x, given(residual), given(seed), given(rows), d)
              : dropout_forward(*x, residual,
                                residual.defined() ? residual.scalar_type() : x->scalar_type(),
                                seed, rows, d);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// embedding(ids, table, scale, to_float, padding_idx (-1: none)) -> rows in the table's type or fp32
OP(embedding) {
  HANDLE_TH_ERRORS
  ARGS(5);
  const Tensor *ids = tensor(a[0]), *table = tensor(a[1]);
  double scale;
  int64_t padding;
  if (!ids || !table || !number(a[2], scale) || !integer(a[4], padding)) ELSE_PYTHON;
  const at::Device dev = table->device();
  if (code_of(table->scalar_type()) < 0 || !is(*table, table->scalar_type(), 2, dev) ||
      !on(*ids, dev) || ids->scalar_type() != at::kLong || !ids->is_contiguous() || padding < -1)
    ELSE_PYTHON;
  const at::ScalarType to = a[3] == Py_True ? at::kFloat : table->scalar_type();
  Tensor out;
  {
    const NoGil released;
    out = wants_grad({table}) ? Embedding::apply(*table, *ids, scale, to, padding)
                              : embedding_forward(*ids, *table, scale, to);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

}  // namespace soupk_host
