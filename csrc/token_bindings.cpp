// Tensor entry points of the token-model operators: checks, workspaces and
// launches on the current stream of the inputs' device.  Shapes arrive
// normalised from blades_amd/ops: contiguous [groups, rows, ...] tensors.
#include <torch/extension.h>

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <limits>
#include <optional>
#include <tuple>
#include <vector>

#include "token_ops.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using namespace token_ops;

DType dtype_of(const Tensor& t) {
  TORCH_CHECK(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16,
              "expected float32 or bfloat16, got ", t.scalar_type());
  return t.scalar_type() == at::kFloat ? kF32 : kBF16;
}

void check(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name,
              " must be on ", like.device());
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

void check_typed(const Tensor& t, const Tensor& like, const char* name) {
  check(t, like, name);
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must be ",
              like.scalar_type());
}

// elements between groups: 0 for a shared parameter of `dims` dimensions
long long group_stride(const Tensor& t, long long groups, int dims,
                       const char* name) {
  if (t.dim() == dims) return 0;
  TORCH_CHECK(t.dim() == dims + 1 && t.size(0) == groups, name,
              " must be shared or have one entry per group");
  return groups ? t.numel() / groups : 0;
}

void check_groups(long long groups) {
  TORCH_CHECK(groups >= 1 && groups <= 65535,
              "a batched call holds 1 to 65535 clients, got ", groups);
}

hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

const void* data(const OptTensor& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

Tensor floats(const Tensor& like, at::IntArrayRef sizes) {
  return at::empty(sizes, like.options().dtype(at::kFloat));
}

// ------------------------------------------------------------- layer norm

NormArgs norm_args(const Tensor& x, const OptTensor& w, const OptTensor& b) {
  NormArgs a = {};
  check(x, x, "x");
  TORCH_CHECK(x.dim() == 3, "x must be [groups, rows, dim]");
  a.groups = x.size(0);
  a.rows = x.size(1);
  a.dim = x.size(2);
  check_groups(a.groups);
  TORCH_CHECK(a.dim >= 1 && a.dim < (1ll << 30), "dim out of range");
  a.x = x.data_ptr();
  if (w.has_value()) {
    check_typed(*w, x, "weight");
    TORCH_CHECK(w->size(-1) == a.dim, "weight does not match dim");
    a.w = w->data_ptr();
    a.w_stride = group_stride(*w, a.groups, 1, "weight");
  }
  if (b.has_value()) {
    check_typed(*b, x, "bias");
    TORCH_CHECK(b->size(-1) == a.dim, "bias does not match dim");
    a.b = b->data_ptr();
    a.b_stride = group_stride(*b, a.groups, 1, "bias");
  }
  return a;
}

std::tuple<Tensor, Tensor, Tensor> norm_forward_t(
    const Tensor& x, const OptTensor& w, const OptTensor& b, double eps) {
  NormArgs a = norm_args(x, w, b);
  const DType t = dtype_of(x);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty_like(x);
  Tensor mean = floats(x, {a.groups, a.rows}), rstd = at::empty_like(mean);
  a.y = y.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  a.eps = (float)eps;
  if (a.rows > 0) norm_forward(a, t, stream_of(x));
  return {y, mean, rstd};
}

// dw, db: [groups, dim], empty where params is false
std::tuple<Tensor, Tensor, Tensor> norm_backward_t(
    const Tensor& dy, const Tensor& x, const Tensor& mean, const Tensor& rstd,
    const OptTensor& w, bool params) {
  NormArgs a = norm_args(x, w, std::nullopt);
  const DType t = dtype_of(x);
  check_typed(dy, x, "dy");
  TORCH_CHECK(dy.sizes() == x.sizes(), "dy must have x's shape");
  for (const Tensor* s : {&mean, &rstd}) {
    check(*s, x, "statistics");
    TORCH_CHECK(s->scalar_type() == at::kFloat
                && s->numel() == a.groups * a.rows, "bad statistics");
  }
  c10::DeviceGuard guard(x.device());
  Tensor dx = at::empty_like(x);
  Tensor dw, db, partial;
  const std::vector<int64_t> shape = {params ? a.groups : 0, a.dim};
  a.dy = dy.data_ptr();
  a.y = dx.data_ptr();
  a.mean = mean.data_ptr<float>();
  a.rstd = rstd.data_ptr<float>();
  if (a.rows == 0)
    return {dx, at::zeros(shape, x.options()), at::zeros(shape, x.options())};
  dw = at::empty(shape, x.options());
  db = at::empty(shape, x.options());
  if (params) {
    const long long blocks =
        norm_partial_blocks(a.groups, a.rows, a.dim, t);
    partial = floats(x, {a.groups * blocks * 2, a.dim});
    a.partial = partial.data_ptr<float>();
    a.dw = dw.data_ptr();
    a.db = db.data_ptr();
  }
  norm_backward(a, t, stream_of(x));
  return {dx, dw, db};
}

// [groups, rows, cols] -> [groups, cols]
Tensor colsum_t(const Tensor& x) {
  check(x, x, "x");
  const DType t = dtype_of(x);
  TORCH_CHECK(x.dim() == 3, "x must be [groups, rows, cols]");
  check_groups(x.size(0));
  c10::DeviceGuard guard(x.device());
  const long long groups = x.size(0), rows = x.size(1), cols = x.size(2);
  if (rows == 0 || cols == 0) return at::zeros({groups, cols}, x.options());
  Tensor out = at::empty({groups, cols}, x.options());
  Tensor partial =
      floats(x, {groups * colsum_blocks(groups, rows, cols), cols});
  colsum(x.data_ptr(), out.data_ptr(), partial.data_ptr<float>(), groups, rows,
         cols, t, stream_of(x));
  return out;
}

// ------------------------------------------------------------------- act8

struct Packed {
  Tensor q, e;
};
Packed packed_like(const Tensor& x) {
  auto sizes = x.sizes().vec();
  Packed p;
  p.q = at::empty(sizes, x.options().dtype(at::kChar));
  sizes.back() = (sizes.back() + 127) / 128;
  p.e = at::empty(sizes, x.options().dtype(at::kByte));
  return p;
}

void check_act(const Tensor& x) {
  check(x, x, "x");
  dtype_of(x);
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1
              && x.size(-1) < (1ll << 30), "last axis out of range");
}

void check_packed(const Tensor& q, const Tensor& e, const Tensor& like) {
  check(q, like, "q");
  check(e, like, "e");
  TORCH_CHECK(q.scalar_type() == at::kChar && e.scalar_type() == at::kByte,
              "8-bit storage is int8 values and uint8 exponents");
  TORCH_CHECK(q.dim() >= 1 && q.size(-1) >= 1
              && e.numel() == q.numel() / q.size(-1)
                                  * ((q.size(-1) + 127) / 128),
              "exponents do not match the values");
}

std::tuple<Tensor, Tensor> act8_pack_t(const Tensor& x) {
  check_act(x);
  c10::DeviceGuard guard(x.device());
  Packed p = packed_like(x);
  if (x.numel() > 0)
    act8_pack(x.data_ptr(), p.q.data_ptr<int8_t>(), p.e.data_ptr<uint8_t>(),
              x.numel() / x.size(-1), x.size(-1), dtype_of(x), stream_of(x));
  return {p.q, p.e};
}

std::tuple<Tensor, Tensor, Tensor> gelu_forward_t(const Tensor& x, bool keep) {
  check_act(x);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty_like(x);
  Packed p;
  if (keep) {
    p = packed_like(x);
  } else {
    p.q = at::empty({0}, x.options().dtype(at::kChar));
    p.e = at::empty({0}, x.options().dtype(at::kByte));
  }
  if (x.numel() > 0)
    gelu_forward(x.data_ptr(), y.data_ptr(),
                 keep ? p.q.data_ptr<int8_t>() : nullptr,
                 keep ? p.e.data_ptr<uint8_t>() : nullptr,
                 x.numel() / x.size(-1), x.size(-1), dtype_of(x),
                 stream_of(x));
  return {y, p.q, p.e};
}

Tensor gelu_backward_t(const Tensor& dy, const Tensor& q, const Tensor& e) {
  check_act(dy);
  check_packed(q, e, dy);
  TORCH_CHECK(q.sizes() == dy.sizes(), "q must have dy's shape");
  c10::DeviceGuard guard(dy.device());
  Tensor dx = at::empty_like(dy);
  if (dy.numel() > 0)
    gelu_backward(dy.data_ptr(), q.data_ptr<int8_t>(), e.data_ptr<uint8_t>(),
                  dx.data_ptr(), dy.numel() / dy.size(-1), dy.size(-1),
                  dtype_of(dy), stream_of(dy));
  return dx;
}

// ---------------------------------------------------------------- products

void check_tiles(long long m, long long n) {
  TORCH_CHECK(ceil_div(m, 128) * ceil_div(n, 128) < (1ll << 24),
              "product of ", m, " x ", n, " is too large for one launch");
}

Mat mat(const Tensor& t, long long group) {
  Mat m = {};
  m.p = t.data_ptr();
  m.ld = t.size(-1);
  m.group = group;
  return m;
}

// out = A B (+ bias) with the contraction cut where the output alone would
// not fill the chip
void run_gemm(Gemm& g, const Tensor& like) {
  const int splits = gemm_splits(g.groups, g.m, g.n, g.k);
  const hipStream_t s = stream_of(like);
  if (splits == 1) {
    gemm(g, s);
    return;
  }
  Tensor partial = floats(like, {splits, g.groups, g.m, g.n});
  g.partial = partial.data_ptr<float>();
  g.splits = splits;
  gemm(g, s);
  join_partials(g.partial, splits, g.groups, g.m, g.n, g.out, g.out_ld,
                g.out_group, g.bias, g.bias_group, g.tout, s);
}

// y[g] = x[g] w' + b
Tensor linear_forward_t(const Tensor& x, const Tensor& w, const OptTensor& b) {
  check(x, x, "x");
  check_typed(w, x, "weight");
  TORCH_CHECK(x.dim() == 3, "x must be [groups, rows, in]");
  const long long groups = x.size(0), rows = x.size(1), in = x.size(2);
  check_groups(groups);
  const long long wg = group_stride(w, groups, 2, "weight");
  const long long out = w.size(-2);
  TORCH_CHECK(w.size(-1) == in, "weight does not match x");
  check_tiles(rows, out);
  c10::DeviceGuard guard(x.device());
  Tensor y = at::empty({groups, rows, out}, x.options());
  if (y.numel() == 0) return y;
  Gemm g = {};
  if (b.has_value()) {
    check_typed(*b, x, "bias");
    TORCH_CHECK(b->size(-1) == out, "bias does not match weight");
    g.bias = b->data_ptr();
    g.bias_group = group_stride(*b, groups, 1, "bias");
  }
  g.a = mat(x, rows * in);
  g.b = mat(w, wg);
  g.ta = g.tb = g.tout = dtype_of(x);
  g.groups = groups;
  g.m = rows;
  g.n = out;
  g.k = in;
  g.out = y.data_ptr();
  g.out_ld = out;
  g.out_group = rows * out;
  run_gemm(g, x);
  return y;
}

// dx[g] = dy[g] w
Tensor linear_grad_input_t(const Tensor& dy, const Tensor& w) {
  check(dy, dy, "dy");
  check_typed(w, dy, "weight");
  TORCH_CHECK(dy.dim() == 3, "dy must be [groups, rows, out]");
  const long long groups = dy.size(0), rows = dy.size(1), out = dy.size(2);
  check_groups(groups);
  const long long wg = group_stride(w, groups, 2, "weight");
  const long long in = w.size(-1);
  TORCH_CHECK(w.size(-2) == out, "weight does not match dy");
  check_tiles(rows, in);
  c10::DeviceGuard guard(dy.device());
  Tensor dx = at::empty({groups, rows, in}, dy.options());
  if (dx.numel() == 0) return dx;
  Gemm g = {};
  g.a = mat(dy, rows * out);
  g.b = mat(w, wg);
  g.b_kmajor = true;
  g.ta = g.tb = g.tout = dtype_of(dy);
  g.groups = groups;
  g.m = rows;
  g.n = in;
  g.k = out;
  g.out = dx.data_ptr();
  g.out_ld = in;
  g.out_group = rows * in;
  run_gemm(g, dy);
  return dx;
}

// dw[g] = dy[g]' x[g], x in 8-bit storage
Tensor linear_grad_weight_t(const Tensor& dy, const Tensor& q,
                            const Tensor& e) {
  check(dy, dy, "dy");
  check_packed(q, e, dy);
  TORCH_CHECK(dy.dim() == 3 && q.dim() == 3 && q.size(0) == dy.size(0)
              && q.size(1) == dy.size(1), "q does not match dy");
  const long long groups = dy.size(0), rows = dy.size(1), out = dy.size(2),
                  in = q.size(2);
  check_groups(groups);
  check_tiles(out, in);
  c10::DeviceGuard guard(dy.device());
  if (rows == 0 || out == 0)
    return at::zeros({groups, out, in}, dy.options());
  Tensor dw = at::empty({groups, out, in}, dy.options());
  Gemm g = {};
  g.a = mat(dy, rows * out);
  g.a_kmajor = g.b_kmajor = true;
  g.b = mat(q, rows * in);
  g.b.e = e.data_ptr<uint8_t>();
  g.b.e_ld = e.size(2);
  g.b.e_group = rows * e.size(2);
  g.ta = g.tb = g.tout = dtype_of(dy);
  g.groups = groups;
  g.m = out;
  g.n = in;
  g.k = rows;
  g.out = dw.data_ptr();
  g.out_ld = in;
  g.out_group = out * in;
  run_gemm(g, dy);
  return dw;
}

// -------------------------------------------------------------------- loss

Loss loss_args(const Tensor& x, const Tensor& w, const Tensor& target,
               const OptTensor& bias, int64_t ignore) {
  check(x, x, "x");
  check_typed(w, x, "weight");
  check(target, x, "target");
  TORCH_CHECK(x.dim() == 3, "x must be [groups, rows, dim]");
  Loss l = {};
  l.groups = x.size(0);
  l.rows = x.size(1);
  l.dim = x.size(2);
  l.t = dtype_of(x);
  check_groups(l.groups);
  l.x = mat(x, l.rows * l.dim);
  l.w = mat(w, group_stride(w, l.groups, 2, "weight"));
  l.vocab = w.size(-2);
  TORCH_CHECK(w.size(-1) == l.dim, "weight does not match x");
  TORCH_CHECK(l.vocab >= 1 && l.dim >= 1, "empty weight");
  TORCH_CHECK(target.scalar_type() == at::kLong
              && target.numel() == l.groups * l.rows,
              "target must be int64 [groups, rows]");
  l.target = reinterpret_cast<const long long*>(target.data_ptr<int64_t>());
  l.ignore = ignore;
  if (bias.has_value()) {
    check_typed(*bias, x, "bias");
    TORCH_CHECK(bias->size(-1) == l.vocab, "bias does not match weight");
    l.bias = bias->data_ptr();
    l.bias_group = group_stride(*bias, l.groups, 1, "bias");
  }
  check_tiles(l.vocab, l.rows);
  return l;
}

// reduction 0: none, 1: sum, 2: mean.
// -> loss ([groups] or [groups, rows]), lse [groups, rows], count [groups]
std::tuple<Tensor, Tensor, Tensor> loss_forward_t(
    const Tensor& x, const Tensor& w, const Tensor& target,
    const OptTensor& bias, int64_t ignore, int64_t reduction) {
  Loss l = loss_args(x, w, target, bias, ignore);
  c10::DeviceGuard guard(x.device());
  Tensor lse = floats(x, {l.groups, l.rows});
  Tensor rows = at::empty_like(lse);
  Tensor count = floats(x, {l.groups});
  if (l.rows == 0) {
    count.zero_();
    if (reduction == 0) return {rows, lse, count};
    const double empty =
        reduction == 2 ? std::numeric_limits<double>::quiet_NaN() : 0.0;
    return {at::full({l.groups}, empty, count.options()), lse, count};
  }
  Tensor part = floats(x, {l.groups, loss_tiles(l.vocab), l.rows, 2});
  Tensor picked = at::empty_like(lse);
  Tensor loss, sums;
  if (reduction != 0) {
    loss = floats(x, {l.groups});
    sums = at::empty({l.groups, loss_sum_blocks(l.rows), 2},
                     x.options().dtype(at::kDouble));
  }
  loss_forward(l, part.data_ptr(), picked.data_ptr<float>(),
               lse.data_ptr<float>(), rows.data_ptr<float>(),
               reduction ? sums.data_ptr() : nullptr,
               reduction ? loss.data_ptr<float>() : nullptr,
               count.data_ptr<float>(), reduction == 2, stream_of(x));
  return {reduction ? loss : rows, lse, count};
}

// grad: [groups], or [groups, rows] for reduction 0.
// -> dx like x, dw [groups, vocab, dim], db [groups, vocab] (empty if unused)
std::tuple<Tensor, Tensor, Tensor> loss_backward_t(
    const Tensor& grad, const Tensor& x, const Tensor& w, const Tensor& target,
    const OptTensor& bias, const Tensor& lse, const Tensor& count,
    int64_t ignore, int64_t reduction, bool want_x, bool want_w,
    bool want_b) {
  Loss l = loss_args(x, w, target, bias, ignore);
  check(grad, x, "grad");
  check(lse, x, "lse");
  check(count, x, "count");
  TORCH_CHECK(grad.scalar_type() == at::kFloat
              && lse.scalar_type() == at::kFloat
              && count.scalar_type() == at::kFloat
              && lse.numel() == l.groups * l.rows
              && count.numel() == l.groups
              && grad.numel() == (reduction ? l.groups : l.groups * l.rows),
              "bad saved tensors");
  c10::DeviceGuard guard(x.device());
  const hipStream_t s = stream_of(x);
  const std::vector<int64_t> wshape = {want_w ? l.groups : 0, l.vocab, l.dim};
  const std::vector<int64_t> bshape = {want_b ? l.groups : 0, l.vocab};
  if (l.rows == 0)
    return {at::zeros_like(x), at::zeros(wshape, x.options()),
            at::zeros(bshape, x.options())};
  Tensor dx = at::empty({want_x ? l.groups : 0, l.rows, l.dim}, x.options());
  Tensor dw = at::empty(wshape, x.options());
  Tensor db = at::empty(bshape, x.options());

  // The logits' gradient exists for one piece of the vocabulary at a time.
  // 256 MiB hold it in the last-level cache between the kernel that writes
  // it and the two products that read it.
  const long long size = x.element_size();
  const long long ld = ceil_div(l.rows, 128) * 128;
  long long piece = (256ll << 20) / (l.groups * ld * size) / 128 * 128;
  piece = std::max<long long>(piece, 512);
  piece = std::min(piece, ceil_div(l.vocab, 128) * 128);
  // pieces of nearly equal size
  const long long pieces = ceil_div(l.vocab, piece);
  piece = ceil_div(ceil_div(l.vocab, pieces), 128) * 128;
  Tensor pt = at::empty({l.groups, piece, ld}, x.options());

  const int splits = gemm_splits(l.groups, l.rows, l.dim,
                                 std::min(piece, l.vocab));
  Tensor xsum;
  const bool parts = splits > 1 || l.vocab > piece;
  if (want_x && parts) xsum = floats(x, {splits, l.groups, l.rows, l.dim});

  for (long long v0 = 0; v0 < l.vocab; v0 += piece) {
    const long long nv = std::min(piece, l.vocab - v0);
    loss_logit_grad(l, v0, nv, lse.data_ptr<float>(), grad.data_ptr<float>(),
                    reduction ? 1 : l.rows, reduction ? 0 : 1,
                    reduction == 2 ? count.data_ptr<float>() : nullptr,
                    pt.data_ptr(), ld, piece * ld, s);
    Mat pm = mat(pt, piece * ld);
    pm.padded = true;
    if (want_x) {
      Gemm g = {};
      g.a = pm;
      g.a_kmajor = true;
      g.b = l.w;
      g.b.p = static_cast<const char*>(l.w.p) + v0 * l.dim * size;
      g.b_kmajor = true;
      g.ta = g.tb = g.tout = l.t;
      g.groups = l.groups;
      g.m = l.rows;
      g.n = l.dim;
      g.k = nv;
      g.out = dx.data_ptr();
      g.out_ld = l.dim;
      g.out_group = l.rows * l.dim;
      if (parts) {
        g.partial = xsum.data_ptr<float>();
        g.splits = splits;
        g.accumulate = v0 > 0;
      }
      gemm(g, s);
    }
    if (want_w) {
      Gemm g = {};
      g.a = pm;
      g.b = l.x;
      g.b_kmajor = true;
      g.ta = g.tb = g.tout = l.t;
      g.groups = l.groups;
      g.m = nv;
      g.n = l.dim;
      g.k = l.rows;
      g.out = static_cast<char*>(dw.data_ptr()) + v0 * l.dim * size;
      g.out_ld = l.dim;
      g.out_group = l.vocab * l.dim;
      run_gemm(g, x);
    }
    if (want_b)
      rowsum(pt.data_ptr(), ld, piece * ld, l.groups, nv, ld,
             static_cast<char*>(db.data_ptr()) + v0 * size, l.vocab, l.t, s);
  }
  if (want_x && parts)
    join_partials(xsum.data_ptr<float>(), splits, l.groups, l.rows, l.dim,
                  dx.data_ptr(), l.dim, l.rows * l.dim, nullptr, 0, l.t, s);
  return {dx, dw, db};
}

}  // namespace

void bind_token_ops(pybind11::module_& m) {
  m.def("norm_forward", &norm_forward_t, "layer norm with its statistics");
  m.def("norm_backward", &norm_backward_t, "layer norm gradients per group");
  m.def("colsum", &colsum_t, "sum over rows per group");
  m.def("act8_pack", &act8_pack_t, "activations to 8-bit storage");
  m.def("gelu_forward", &gelu_forward_t, "GELU, keeping its input in 8 bits");
  m.def("gelu_backward", &gelu_backward_t, "GELU gradient from 8-bit input");
  m.def("linear_forward", &linear_forward_t, "x w' + b per group");
  m.def("linear_grad_input", &linear_grad_input_t, "dy w per group");
  m.def("linear_grad_weight", &linear_grad_weight_t,
        "dy' x per group, x in 8-bit storage");
  m.def("loss_forward", &loss_forward_t,
        "cross entropy of a linear head without its logits");
  m.def("loss_backward", &loss_backward_t,
        "gradients of that loss, in pieces of the vocabulary");
}
