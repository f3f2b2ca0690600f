// Host side of the operators of a generating program: rotary_tables, rotary (with its autograd node),
// rope_append, paged_attention, verify_drafts.
//
// As the operators of host_autograd.cpp: one native call each -- checks, allocations, launch -- that takes
// plain arguments of the expected types and returns None for anything else; the Python caller then checks,
// converts or raises.  Decoding calls them once a layer and token, so what a call costs the host is what
// bounds the small ones.

#include <vector>

#include <c10/hip/HIPFunctions.h>

#include "host_args.hpp"
#include "host_autograd.hpp"

namespace soupk_host {
namespace {

// ---- rotary -------------------------------------------------------------------------------------

// A table of cosines or sines: fp32 [positions, R / 2], its columns adjacent.
bool is_table(const Tensor& t, const at::Device& dev) {
  return on(t, dev) && t.scalar_type() == at::kFloat && t.dim() == 2 && t.size(1) >= 1 &&
         (t.stride(1) == 1 || t.size(1) == 1) && t.stride(0) >= 0;
}
bool are_tables(const Tensor& c, const Tensor& s, const at::Device& dev) {
  return is_table(c, dev) && is_table(s, dev) && c.sizes() == s.sizes() &&
         (c.stride(0) == s.stride(0) || c.size(0) <= 1);
}

Tensor rotate(const Tensor& x, const Tensor& cos, const Tensor& sin, const Tensor& pos, bool interleaved,
              bool inverse) {
  const c10::DeviceGuard guard(x.device());
  Tensor out = empty(x.sizes(), x.scalar_type(), x.device());
  if (out.numel() > 0)
    check("soupk_rotary",
          p_soupk_rotary(address(x), code_of(x.scalar_type()), x.stride(0), x.stride(1), address<float>(cos),
                         address<float>(sin), cos.size(0), cos.stride(0), address<int64_t>(pos), address(out),
                         x.size(0), static_cast<int32_t>(x.size(1)), static_cast<int32_t>(x.size(2)),
                         static_cast<int32_t>(2 * cos.size(1)), interleaved, inverse, stream_of(x)));
  return out;
}

// (Linear: the backward is the inverse rotation of the gradient, differentiable in its turn.)
struct Rotary : Function<Rotary> {
  static Tensor forward(AutogradContext* ctx, Tensor x, Tensor cos, Tensor sin, Tensor pos, bool interleaved,
                        bool inverse) {
    ctx->save_for_backward({cos, sin, pos});
    ctx->saved_data["i"] = interleaved;
    ctx->saved_data["b"] = inverse;
    return rotate(x, cos, sin, pos, interleaved, inverse);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const variable_list s = ctx->get_saved_variables();
    const bool interleaved = ctx->saved_data["i"].toBool(), inverse = !ctx->saved_data["b"].toBool();
    // (the forward's output has x's type, and so has its gradient)
    const Tensor dout = g[0].stride(2) == 1 ? g[0] : g[0].contiguous();
    return {wants_grad({&dout}) ? Rotary::apply(dout, s[0], s[1], s[2], interleaved, inverse)
                                : rotate(dout, s[0], s[1], s[2], interleaved, inverse),
            Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// ---- the paged cache ----------------------------------------------------------------------------

// Pages of keys and values [pages, n_kv, page_size, D]: a page's elements adjacent, pages a stride apart.
bool are_pages(const Tensor& k, const Tensor& v) {
  const at::Device dev = k.device();
  auto inner = [](const Tensor& t) {
    return t.dim() == 4 && t.size(0) >= 1 && t.size(1) >= 1 && t.size(2) >= 1 && t.stride(3) == 1 &&
           t.stride(2) == t.size(3) && t.stride(1) == t.size(2) * t.size(3);
  };
  return k.is_cuda() && on(k, dev) && on(v, dev) && k.scalar_type() == v.scalar_type() &&
         (k.scalar_type() == at::kHalf || k.scalar_type() == at::kBFloat16) && inner(k) && inner(v) &&
         k.sizes() == v.sizes() &&
         (k.size(0) == 1 || (k.stride(0) == v.stride(0) && k.stride(0) >= k.size(1) * k.stride(1))) &&
         k.size(3) >= 16 && k.size(3) <= 256 && k.size(3) % 16 == 0 && k.size(1) <= (1 << 16) &&
         k.size(2) < (int64_t{1} << 31) && k.size(0) < (int64_t{1} << 31);
}

// The sequences' bounds, lengths and pages: int32 [B + 1] or undefined, [B], [B, pages of one].
bool are_sequences(const Tensor& cu, const Tensor& lengths, const Tensor& table, int64_t rows, int64_t page,
                   const at::Device& dev) {
  if (!is(lengths, at::kInt, 1, dev) || !is(table, at::kInt, 2, dev)) return false;
  const int64_t B = lengths.size(0);
  return table.size(0) == B && B < (int64_t{1} << 31) - 1 && table.size(1) <= (int64_t{1} << 30) / page &&
         (cu.defined() ? is(cu, at::kInt, 1, dev) && cu.size(0) == B + 1 : rows == B);
}

void written(const Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

}  // namespace

// rotary_tables(seq, dim, theta, scaling code, factor, original, beta_fast, beta_slow, gain, frequencies (a
// tuple, or None), device index (-1: the current one)) -> (cos, sin)
OP(rotary_tables) {
  HANDLE_TH_ERRORS
  ARGS(11);
  int64_t seq, dim, scaling, device;
  double v[6];
  if (!integer(a[0], seq) || !integer(a[1], dim) || !integer(a[3], scaling) || !integer(a[10], device))
    ELSE_PYTHON;
  const int at_arg[6] = {2, 4, 5, 6, 7, 8};
  for (int i = 0; i < 6; ++i)
    if (!number(a[at_arg[i]], v[i])) ELSE_PYTHON;
  if (seq < 0 || seq >= (int64_t{1} << 31) || dim < 2 || dim > 256 || dim % 2 || !(v[0] > 1.0 && v[0] <= 1e30))
    ELSE_PYTHON;
  std::vector<double> freq;
  if (a[9] != Py_None) {
    if (!PyTuple_Check(a[9]) || PyTuple_GET_SIZE(a[9]) != dim / 2) ELSE_PYTHON;
    freq.resize(dim / 2);
    for (int64_t i = 0; i < dim / 2; ++i)
      if (!number(PyTuple_GET_ITEM(a[9], i), freq[i])) ELSE_PYTHON;
  }
  Tensor cos, sin;
  {
    const NoGil released;
    const at::Device dev(at::kCUDA, device < 0 ? c10::hip::current_device()
                                               : static_cast<c10::DeviceIndex>(device));
    const c10::DeviceGuard guard(dev);
    cos = empty({seq, dim / 2}, at::kFloat, dev);
    sin = empty({seq, dim / 2}, at::kFloat, dev);
    check("soupk_rotary_tables",
          p_soupk_rotary_tables(address<float>(cos), address<float>(sin), seq, static_cast<int32_t>(dim),
                                freq.empty() ? nullptr : freq.data(), v[0], static_cast<int32_t>(scaling), v[1],
                                v[2], v[3], v[4], v[5], stream_of(cos)));
  }
  return pack({cos, sin});
  END_HANDLE_TH_ERRORS
}

// rotary(x [rows, heads, D], cos, sin, pos, interleaved) -> out
OP(rotary) {
  HANDLE_TH_ERRORS
  ARGS(5);
  const Tensor *x = tensor(a[0]), *cos = tensor(a[1]), *sin = tensor(a[2]), *pos = tensor(a[3]);
  if (!x || !cos || !sin || !pos || !PyBool_Check(a[4]) || x->dim() != 3) ELSE_PYTHON;
  const at::Device dev = x->device();
  const int64_t D = x->size(2);
  if (!x->is_cuda() || !on(*x, dev) || code_of(x->scalar_type()) < 0 || (x->stride(2) != 1 && D > 1) ||
      x->stride(0) < 0 || x->stride(1) < 0 || x->size(1) < 1 || x->size(1) > (1 << 16) || D > (1 << 16) ||
      !are_tables(*cos, *sin, dev) || 2 * cos->size(1) > D || !is(*pos, at::kLong, 1, dev) ||
      pos->size(0) != x->size(0))
    ELSE_PYTHON;
  const bool interleaved = a[4] == Py_True;
  // (a gradient of the tables is not given: the Python caller says so)
  if (wants_grad({cos, sin})) ELSE_PYTHON;
  Tensor out;
  {
    const NoGil released;
    out = wants_grad({x}) ? Rotary::apply(*x, *cos, *sin, *pos, interleaved, false)
                          : rotate(*x, *cos, *sin, *pos, interleaved, false);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// rope_append(qkv, lora_q, lora_v, cos, sin, k_pages, v_pages, table, lengths, cu, interleaved) -> q rows
OP(rope_append) {
  HANDLE_TH_ERRORS
  ARGS(11);
  const Tensor *qkv = tensor(a[0]), *k = tensor(a[5]), *v = tensor(a[6]), *table = tensor(a[7]),
               *lengths = tensor(a[8]);
  Tensor lq, lv, cos, sin, cu;
  if (!qkv || !k || !v || !table || !lengths || !maybe(a[1], lq) || !maybe(a[2], lv) || !maybe(a[3], cos) ||
      !maybe(a[4], sin) || !maybe(a[9], cu) || !PyBool_Check(a[10]))
    ELSE_PYTHON;
  if (!are_pages(*k, *v)) ELSE_PYTHON;
  const at::Device dev = k->device();
  const at::ScalarType t = k->scalar_type();
  const int64_t n_kv = k->size(1), page = k->size(2), D = k->size(3);
  if (!is(*qkv, t, 2, dev)) ELSE_PYTHON;
  const int64_t rows = qkv->size(0), nh = qkv->size(1) / D - 2 * n_kv;
  if (qkv->size(1) % D || nh < 1 || nh > (1 << 16)) ELSE_PYTHON;
  const Tensor& delta = lq.defined() ? lq : lv;
  const at::ScalarType dt = delta.defined() ? delta.scalar_type() : t;
  if ((dt != t && dt != at::kFloat) ||
      (lq.defined() && (!is(lq, dt, 2, dev) || !shape2(lq, rows, nh * D))) ||
      (lv.defined() && (!is(lv, dt, 2, dev) || !shape2(lv, rows, n_kv * D))) || cos.defined() != sin.defined() ||
      (cos.defined() && (!are_tables(cos, sin, dev) || 2 * cos.size(1) > D)) ||
      !are_sequences(cu, *lengths, *table, rows, page, dev))
    ELSE_PYTHON;
  if (wants_grad({qkv, &lq, &lv, &cos, &sin, k, v})) ELSE_PYTHON;
  Tensor q;
  {
    const NoGil released;
    const c10::DeviceGuard guard(dev);
    q = empty({rows, nh * D}, t, dev);
    // (tables of no positions have no address, which would mean no rotation: any other, as none is read)
    auto table_at = [&](const Tensor& c) {
      return c.defined() && c.size(0) == 0 ? reinterpret_cast<const float*>(address(*lengths)) : address<float>(c);
    };
    if (rows > 0) {
      check("soupk_rope_append",
            p_soupk_rope_append(
                address(*qkv), address(lq), address(lv), code_of(dt), table_at(cos), table_at(sin),
                cos.defined() ? cos.size(0) : 0, cos.defined() ? cos.stride(0) : 0,
                cos.defined() ? static_cast<int32_t>(2 * cos.size(1)) : 0, a[10] == Py_True,
                address<int32_t>(cu), address<int32_t>(*lengths), address<int32_t>(*table),
                static_cast<int32_t>(lengths->size(0)), table->size(1), address(q), address(*k), address(*v),
                k->size(0), k->stride(0), static_cast<int32_t>(page), code_of(t), rows,
                static_cast<int32_t>(nh), static_cast<int32_t>(n_kv), static_cast<int32_t>(D), stream_of(*qkv)));
      written(*k);
      written(*v);
    }
  }
  return THPVariable_Wrap(q);
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, table, lengths, cu, scale) -> out
OP(paged_attention) {
  HANDLE_TH_ERRORS
  ARGS(7);
  const Tensor *q = tensor(a[0]), *k = tensor(a[1]), *v = tensor(a[2]), *table = tensor(a[3]),
               *lengths = tensor(a[4]);
  Tensor cu;
  double scale;
  if (!q || !k || !v || !table || !lengths || !maybe(a[5], cu) || !number(a[6], scale) || !are_pages(*k, *v))
    ELSE_PYTHON;
  const at::Device dev = k->device();
  const at::ScalarType t = k->scalar_type();
  const int64_t n_kv = k->size(1), page = k->size(2), D = k->size(3);
  if (!on(*q, dev) || q->scalar_type() != t || q->dim() != 2 || (q->stride(1) != 1 && q->size(1) > 1) ||
      q->stride(0) < 0 || q->size(1) % D)
    ELSE_PYTHON;
  const int64_t rows = q->size(0), nh = q->size(1) / D;
  if (nh < 1 || nh > (1 << 16) || nh % n_kv || rows > (int64_t{1} << 23) / nh || !(scale >= -1e30 && scale <= 1e30) ||
      !are_sequences(cu, *lengths, *table, rows, page, dev))
    ELSE_PYTHON;
  auto aligned = [](const Tensor& c) { return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15) == 0; };
  if (!aligned(*k) || !aligned(*v) || (k->size(0) > 1 && k->stride(0) % 8)) ELSE_PYTHON;
  if (wants_grad({q, k, v})) ELSE_PYTHON;
  Tensor out;
  {
    const NoGil released;
    const c10::DeviceGuard guard(dev);
    const int32_t B = static_cast<int32_t>(lengths->size(0));
    if (B == 0) {
      out = at::zeros({rows, nh * D}, q->options());
    } else {
      out = empty({rows, nh * D}, t, dev);
      if (rows > 0) {
        int64_t need = 0;
        check("soupk_paged_attention_workspace",
              p_soupk_paged_attention_workspace(rows, B, static_cast<int32_t>(nh), static_cast<int32_t>(n_kv),
                                                static_cast<int32_t>(D), table->size(1),
                                                static_cast<int32_t>(page), &need));
        const Tensor ws = empty({need}, at::kByte, dev);
        check("soupk_paged_attention",
              p_soupk_paged_attention(
                  address(*q), q->stride(0), address(*k), address(*v), k->size(0), k->stride(0),
                  static_cast<int32_t>(page), address<int32_t>(*table), table->size(1),
                  address<int32_t>(*lengths), address<int32_t>(cu), B, address(out), code_of(t), rows,
                  static_cast<int32_t>(nh), static_cast<int32_t>(n_kv), static_cast<int32_t>(D),
                  static_cast<float>(scale), address(ws), need, stream_of(*q)));
      }
    }
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// verify_drafts(target, drafts, uniforms, draft_probs, lengths) -> (tokens, accepted)
OP(verify_drafts) {
  HANDLE_TH_ERRORS
  ARGS(5);
  const Tensor *p = tensor(a[0]), *x = tensor(a[1]), *u = tensor(a[2]);
  Tensor q, lengths;
  if (!p || !x || !u || !maybe(a[3], q) || !maybe(a[4], lengths) || p->dim() != 3) ELSE_PYTHON;
  const at::Device dev = p->device();
  const at::ScalarType t = p->scalar_type();
  const int64_t B = p->size(0), K = p->size(1) - 1, V = p->size(2);
  if (code_of(t) < 0 || !is(*p, t, 3, dev) || K < 0 || K > (1 << 20) || V < 1 || V >= (int64_t{1} << 40) ||
      B > (int64_t{1} << 14) || !is(*x, at::kLong, 2, dev) || !shape2(*x, B, K) || !is(*u, at::kFloat, 2, dev) ||
      !shape2(*u, B, K + 1) ||
      (q.defined() && (!is(q, t, 3, dev) || q.size(0) != B || q.size(1) != K || q.size(2) != V)) ||
      (lengths.defined() && (!is(lengths, at::kInt, 1, dev) || lengths.size(0) != B)))
    ELSE_PYTHON;
  if (wants_grad({p, u, &q})) ELSE_PYTHON;
  Tensor tokens, accepted;
  {
    const NoGil released;
    const c10::DeviceGuard guard(dev);
    tokens = empty({B, K + 1}, at::kLong, dev);
    accepted = empty({B}, at::kInt, dev);
    if (B > 0) {
      int64_t need = 0;
      check("soupk_verify_drafts_workspace", p_soupk_verify_drafts_workspace(B, V, &need));
      const Tensor ws = empty({need}, at::kByte, dev);
      // (no drafts at all: their distributions are empty tensors, and none is read)
      check("soupk_verify_drafts",
            p_soupk_verify_drafts(address(*p), K > 0 ? address(q) : nullptr, code_of(t), address<int64_t>(*x),
                                  address<float>(*u), address<int32_t>(lengths), address<int64_t>(tokens),
                                  address<int32_t>(accepted), B, static_cast<int32_t>(K), V, address(ws), need,
                                  stream_of(*p)));
    }
  }
  return pack({tokens, accepted});
  END_HANDLE_TH_ERRORS
}

}  // namespace soupk_host
