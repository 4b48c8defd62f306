// Tensor entry points of the token-model operators: checks, workspaces and
// launches on the current stream of the inputs' device (contiguous
// [groups, rows, ...] tensors), and above them the dispatcher ops with their
// autograd and vmap rules.
#include <torch/extension.h>

#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/functorch/BatchedTensorImpl.h>
#include <ATen/functorch/DynamicLayer.h>
#include <ATen/functorch/PlumbingHelper.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/library.h>

#include <algorithm>
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

// After launches: one that the runtime refused leaves its output unwritten.
void check_launched() { C10_HIP_CHECK(hipGetLastError()); }

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
  if (a.rows > 0) {
    norm_forward(a, t, stream_of(x));
    check_launched();
  }
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
  check_launched();
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
  check_launched();
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
  if (x.numel() > 0) {
    act8_pack(x.data_ptr(), p.q.data_ptr<int8_t>(), p.e.data_ptr<uint8_t>(),
              x.numel() / x.size(-1), x.size(-1), dtype_of(x), stream_of(x));
    check_launched();
  }
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
  if (x.numel() > 0) {
    gelu_forward(x.data_ptr(), y.data_ptr(),
                 keep ? p.q.data_ptr<int8_t>() : nullptr,
                 keep ? p.e.data_ptr<uint8_t>() : nullptr,
                 x.numel() / x.size(-1), x.size(-1), dtype_of(x),
                 stream_of(x));
    check_launched();
  }
  return {y, p.q, p.e};
}

Tensor gelu_backward_t(const Tensor& dy, const Tensor& q, const Tensor& e) {
  check_act(dy);
  check_packed(q, e, dy);
  TORCH_CHECK(q.sizes() == dy.sizes(), "q must have dy's shape");
  c10::DeviceGuard guard(dy.device());
  Tensor dx = at::empty_like(dy);
  if (dy.numel() > 0) {
    gelu_backward(dy.data_ptr(), q.data_ptr<int8_t>(), e.data_ptr<uint8_t>(),
                  dx.data_ptr(), dy.numel() / dy.size(-1), dy.size(-1),
                  dtype_of(dy), stream_of(dy));
    check_launched();
  }
  return dx;
}

// ---------------------------------------------------------------- products

// ld: the longest row of an operand
void check_tiles(long long m, long long n, long long k, long long ld) {
  // offsets within a tile of 256 rows are 32 bits
  TORCH_CHECK(std::max({m, n, k}) < (1ll << 31) - 4096 && ld < 1ll << 22,
              "product of ", m, " x ", n, " x ", k, " is too large");
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
  const int splits = gemm_splits(g);
  const hipStream_t s = stream_of(like);
  if (splits == 1) {
    gemm(g, s);
    check_launched();
    return;
  }
  Tensor partial = floats(like, {splits, g.groups, g.m, g.n});
  g.partial = partial.data_ptr<float>();
  g.splits = splits;
  gemm(g, s);
  TORCH_CHECK(g.out_ld == g.n, "a joined output's rows have no gaps");
  join_partials(g.partial, splits, g.groups, g.m, g.n, g.out, g.out_group,
                g.bias, g.bias_group, g.tout, s);
  check_launched();
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
  check_tiles(rows, out, in, in);
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
  check_tiles(rows, in, out, std::max(in, out));
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
  check_tiles(out, in, rows, std::max(in, out));
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
  check_tiles(l.vocab, l.rows, l.dim, l.dim);
  return l;
}

// reduction 0: none, 1: sum, 2: mean.
// -> loss ([groups] or [groups, rows]), lse [groups, rows, 2], count [groups]
std::tuple<Tensor, Tensor, Tensor> loss_forward_t(
    const Tensor& x, const Tensor& w, const Tensor& target,
    const OptTensor& bias, int64_t ignore, int64_t reduction) {
  Loss l = loss_args(x, w, target, bias, ignore);
  c10::DeviceGuard guard(x.device());
  Tensor lse = floats(x, {l.groups, l.rows, 2});
  Tensor rows = floats(x, {l.groups, l.rows});
  Tensor count = floats(x, {l.groups});
  if (l.rows == 0) {
    count.zero_();
    if (reduction == 0) return {rows, lse, count};
    const double empty =
        reduction == 2 ? std::numeric_limits<double>::quiet_NaN() : 0.0;
    return {at::full({l.groups}, empty, count.options()), lse, count};
  }
  int tile_m, tile_n;
  loss_tile(l, &tile_m, &tile_n);
  Tensor part =
      floats(x, {l.groups, ceil_div(l.vocab, tile_m), l.rows, 2});
  Tensor picked = at::empty_like(rows);
  Tensor loss, sums;
  if (reduction != 0) {
    loss = floats(x, {l.groups});
    sums = at::empty({l.groups, loss_sum_blocks(l.rows), 2},
                     x.options().dtype(at::kDouble));
  }
  loss_forward(l, part.data_ptr(), picked.data_ptr<float>(),
               lse.data_ptr(), rows.data_ptr<float>(),
               reduction ? sums.data_ptr() : nullptr,
               reduction ? loss.data_ptr<float>() : nullptr,
               count.data_ptr<float>(), reduction == 2, stream_of(x));
  check_launched();
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
              && lse.numel() == 2 * l.groups * l.rows
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
  int tile, tile_n;
  loss_tile(l, &tile, &tile_n);
  const long long ld = ceil_div(l.rows, tile_n) * tile_n;
  check_tiles(l.vocab, l.rows, l.dim, ld);
  long long piece = (256ll << 20) / (l.groups * ld * size) / tile * tile;
  piece = std::max<long long>(piece, 512);
  piece = std::min(piece, ceil_div(l.vocab, tile) * tile);
  // pieces of nearly equal size
  const long long pieces = ceil_div(l.vocab, piece);
  piece = ceil_div(ceil_div(l.vocab, pieces), tile) * tile;
  Tensor pt = at::empty({l.groups, piece, ld}, x.options());

  Gemm gx = {};
  gx.a_kmajor = gx.b_kmajor = true;
  gx.ta = gx.tb = gx.tout = l.t;
  gx.groups = l.groups;
  gx.m = l.rows;
  gx.n = l.dim;
  gx.k = std::min(piece, l.vocab);
  gx.out = dx.data_ptr();
  gx.out_ld = l.dim;
  gx.out_group = l.rows * l.dim;
  const int splits = gemm_splits(gx);
  Tensor xsum;
  const bool parts = splits > 1 || l.vocab > piece;
  if (want_x && parts) xsum = floats(x, {splits, l.groups, l.rows, l.dim});

  Scale scale = {grad.data_ptr<float>(),
                 reduction == 2 ? count.data_ptr<float>() : nullptr};
  Tensor top, ratio;
  if (reduction == 0) {
    top = floats(x, {l.groups});
    ratio = floats(x, {l.groups, l.rows});
    row_scale(grad.data_ptr<float>(), l.groups, l.rows,
              top.data_ptr<float>(), ratio.data_ptr<float>(), s);
    scale.num = top.data_ptr<float>();
  }

  Tensor bsum;
  const long long parts_b = loss_row_parts(l);
  if (want_b) bsum = floats(x, {l.groups, parts_b, std::min(piece, l.vocab)});

  for (long long v0 = 0; v0 < l.vocab; v0 += piece) {
    const long long nv = std::min(piece, l.vocab - v0);
    loss_logit_grad(l, v0, nv, lse.data_ptr(),
                    reduction ? nullptr : ratio.data_ptr<float>(),
                    pt.data_ptr(), ld, piece * ld,
                    want_b ? bsum.data_ptr<float>() : nullptr, s);
    Mat pm = mat(pt, piece * ld);
    pm.padded = true;
    if (want_x) {
      Gemm g = gx;
      g.a = pm;
      g.b = l.w;
      g.b.p = static_cast<const char*>(l.w.p) + v0 * l.dim * size;
      g.k = nv;
      g.scale = scale;
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
      g.scale = scale;
      run_gemm(g, x);
    }
    if (want_b)
      join_rows(bsum.data_ptr<float>(), l.groups, parts_b, nv,
                static_cast<char*>(db.data_ptr()) + v0 * size, l.vocab, scale,
                l.t, s);
  }
  if (want_x && parts)
    join_partials(xsum.data_ptr<float>(), splits, l.groups, l.rows, l.dim,
                  dx.data_ptr(), l.rows * l.dim, nullptr, 0, l.t, s);
  check_launched();
  return {dx, dw, db};
}

// ---------------------------------------------------------------- dispatcher
// The operators as torch dispatcher ops, so that autograd and the
// torch.func transforms run without Python between the launches (a vmapped
// forward and backward in Python costs 0.7 ms of host time, here 0.2).
//
//   CUDA             reshapes to [groups, rows, ...] and launches
//   Autograd         records a node; the gradients are dispatcher ops too
//   FuncTorchBatched moves the client axis first and calls the op on the
//                    whole population: shared parameters stay shared,
//                    per-client ones set `groups`
//
// `groups`: 0, or the number of clients on the leading axis of the inputs.
// With groups each parameter is per client or shared by itself.  A gradient op
// called with groups gives both parameters' gradients per client.
//
// The 8-bit input that GELU and linear layers keep is integers and carries no
// autograd history.  An empty float tensor, `tie`, goes with it: it has a
// history at every level that tracks the input, so that the gradient ops see
// that their result depends on it.

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using Int3 = std::tuple<Tensor, Tensor, Tensor>;
using Int4 = std::tuple<Tensor, Tensor, Tensor, Tensor>;

using NormSig = Int3(const Tensor&, const OptTensor&, const OptTensor&, double,
                     int64_t);
using NormGradSig = Int3(const Tensor&, const Tensor&, const OptTensor&,
                         const Tensor&, const Tensor&, int64_t, bool);
using GeluSig = Int4(const Tensor&, bool);
using GeluGradSig = Tensor(const Tensor&, const Tensor&, const Tensor&,
                           const Tensor&);
using LinearSig = Int4(const Tensor&, const Tensor&, const OptTensor&, bool,
                       int64_t);
using LinearGradSig = Int3(const Tensor&, const Tensor&, const Tensor&,
                           const Tensor&, const Tensor&, int64_t, bool, bool,
                           bool);
using LossSig = Int3(const Tensor&, const Tensor&, const Tensor&,
                     const OptTensor&, int64_t, int64_t, int64_t);
using LossGradSig = Int3(const Tensor&, const Tensor&, const Tensor&,
                         const Tensor&, const OptTensor&, const Tensor&,
                         const Tensor&, int64_t, int64_t, int64_t, bool, bool,
                         bool);

template <typename Sig>
c10::TypedOperatorHandle<Sig> find_op(const char* name) {
  return c10::Dispatcher::singleton()
      .findSchemaOrThrow(name, "")
      .typed<Sig>();
}
#define BLADES_OP(fn, name, Sig)                                      \
  const c10::TypedOperatorHandle<Sig>& fn() {                         \
    static const auto op = find_op<Sig>("blades_amd::" name);         \
    return op;                                                        \
  }
BLADES_OP(norm_op, "layer_norm", NormSig)
BLADES_OP(norm_grad_op, "layer_norm_grad", NormGradSig)
BLADES_OP(gelu_op, "gelu_act8", GeluSig)
BLADES_OP(gelu_grad_op, "gelu_act8_grad", GeluGradSig)
BLADES_OP(linear_op, "linear_act8", LinearSig)
BLADES_OP(linear_grad_op, "linear_act8_grad", LinearGradSig)
BLADES_OP(loss_op, "linear_cross_entropy", LossSig)
BLADES_OP(loss_grad_op, "linear_cross_entropy_grad", LossGradSig)
#undef BLADES_OP

// ------------------------------------------------------------ CUDA kernels

OptTensor contig(const OptTensor& t) {
  return t.has_value() && t->defined() ? OptTensor(t->contiguous())
                                       : OptTensor();
}

// [groups or 1, rows, last] contiguous
Tensor groups3(const Tensor& t, int64_t groups) {
  const int64_t g = groups ? groups : 1, last = t.size(-1);
  return t.reshape({g, last ? t.numel() / (g * last) : 0, last}).contiguous();
}
// [groups or 1, rows] contiguous
Tensor groups2(const Tensor& t, int64_t groups) {
  const int64_t g = groups ? groups : 1;
  return t.reshape({g, t.numel() / g}).contiguous();
}
Tensor ungroup(const Tensor& t, int64_t groups, bool have) {
  return groups || !have ? t : t.select(0, 0);
}

Int3 norm_cuda(const Tensor& x, const OptTensor& w, const OptTensor& b,
               double eps, int64_t groups) {
  auto [y, mean, rstd] =
      norm_forward_t(groups3(x, groups), contig(w), contig(b), eps);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  return {y.view(x.sizes()), mean.view(lead), rstd.view(lead)};
}

Int3 norm_grad_cuda(const Tensor& dy, const Tensor& x, const OptTensor& w,
                    const Tensor& mean, const Tensor& rstd, int64_t groups,
                    bool params) {
  auto [dx, dw, db] = norm_backward_t(
      groups3(dy, groups), groups3(x, groups), groups2(mean, groups),
      groups2(rstd, groups), contig(w), params);
  return {dx.view(x.sizes()), ungroup(dw, groups, params),
          ungroup(db, groups, params)};
}

Int4 gelu_cuda(const Tensor& x, bool keep) {
  return std::tuple_cat(gelu_forward_t(x.contiguous(), keep),
                        std::make_tuple(at::empty({0}, x.options())));
}
Tensor gelu_grad_cuda(const Tensor& dy, const Tensor& q, const Tensor& e,
                      const Tensor&) {
  return gelu_backward_t(dy.contiguous(), q.contiguous(), e.contiguous());
}

Int4 linear_cuda(const Tensor& x, const Tensor& w, const OptTensor& b,
                 bool keep, int64_t groups) {
  c10::DeviceGuard guard(x.device());
  auto shape = x.sizes().vec();
  shape.back() = w.size(-2);
  const Tensor y =
      linear_forward_t(groups3(x, groups), w.contiguous(), contig(b));
  Tensor q, e;
  if (keep) {
    std::tie(q, e) = act8_pack_t(x.contiguous());
  } else {
    q = at::empty({0}, x.options().dtype(at::kChar));
    e = at::empty({0}, x.options().dtype(at::kByte));
  }
  return {y.view(shape), q, e, at::empty({0}, x.options())};
}

Int3 linear_grad_cuda(const Tensor& dy, const Tensor& w, const Tensor& q,
                      const Tensor& e, const Tensor&, int64_t groups,
                      bool want_x, bool want_w, bool want_b) {
  c10::DeviceGuard guard(dy.device());
  const Tensor dy3 = groups3(dy, groups);
  Tensor dx, dw, db;
  dx = dw = db = at::empty({0}, dy.options());
  if (want_x) {
    auto shape = dy.sizes().vec();
    shape.back() = w.size(-1);
    dx = linear_grad_input_t(dy3, w.contiguous()).view(shape);
  }
  if (want_w)
    dw = ungroup(linear_grad_weight_t(dy3, groups3(q, groups),
                                      groups3(e, groups)), groups, true);
  if (want_b) db = ungroup(colsum_t(dy3), groups, true);
  return {dx, dw, db};
}

Int3 loss_cuda(const Tensor& x, const Tensor& w, const Tensor& target,
               const OptTensor& b, int64_t ignore, int64_t reduction,
               int64_t groups) {
  auto [loss, lse, count] =
      loss_forward_t(groups3(x, groups), w.contiguous(),
                     groups2(target, groups), contig(b), ignore, reduction);
  if (reduction == 0)
    loss = loss.view(target.sizes());
  else
    loss = ungroup(loss, groups, true);
  auto pairs = target.sizes().vec();
  pairs.push_back(2);
  return {loss, lse.view(pairs), ungroup(count, groups, true)};
}

Int3 loss_grad_cuda(const Tensor& grad, const Tensor& x, const Tensor& w,
                    const Tensor& target, const OptTensor& b,
                    const Tensor& lse, const Tensor& count, int64_t ignore,
                    int64_t reduction, int64_t groups, bool want_x,
                    bool want_w, bool want_b) {
  auto [dx, dw, db] = loss_backward_t(
      groups2(grad, groups).to(at::kFloat), groups3(x, groups),
      w.contiguous(), groups2(target, groups), contig(b),
      groups2(lse, groups), groups2(count, groups), ignore, reduction, want_x,
      want_w, want_b);
  return {want_x ? dx.view(x.sizes()) : dx, ungroup(dw, groups, want_w),
          ungroup(db, groups, want_b)};
}

// ---------------------------------------------------------------- autograd

Tensor or_undefined(const OptTensor& t) {
  return t.has_value() ? *t : Tensor();
}
OptTensor or_none(const Tensor& t) {
  return t.defined() ? OptTensor(t) : OptTensor();
}

// Base of the nodes: tensors to keep, released together.  A saved tensor may be
// asked for once in a backward pass (checkpoints that recompute hold to it).
struct TokenNode : public Node {
  std::vector<SavedVariable> saved;
  void keep(std::initializer_list<Tensor> ts) {
    for (const Tensor& t : ts) saved.emplace_back(t, false);
  }
  Tensor get(size_t i) { return saved[i].unpack(); }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (auto& s : saved) s.reset_data();
  }
  variable_list none(size_t n) { return variable_list(n); }
};

// Of a call with groups: whether a parameter of `dims` dimensions is shared,
// so that its gradients per client have to be summed.
bool is_shared(const Tensor& p, int64_t groups, int64_t dims) {
  return groups && p.defined() && p.dim() == dims;
}
Tensor summed(const Tensor& grad, bool shared) {
  return shared ? grad.sum(0) : grad;
}

struct NormNode : public TokenNode {            // x, w, mean, rstd
  int64_t groups = 0;
  bool shared_w = false, shared_b = false;
  std::string name() const override { return "LayerNormBackward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return none(3);
    const bool want_w = task_should_compute_output(1);
    const bool want_b = task_should_compute_output(2);
    auto [dx, dw, db] =
        norm_grad_op().call(grads[0], get(0), or_none(get(1)), get(2), get(3),
                            groups, want_w || want_b);
    return {dx, want_w ? summed(dw, shared_w) : Tensor(),
            want_b ? summed(db, shared_b) : Tensor()};
  }
};

struct GeluNode : public TokenNode {            // q, e, tie
  std::string name() const override { return "GeluAct8Backward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return none(1);
    return {gelu_grad_op().call(grads[0], get(0), get(1), get(2))};
  }
};

struct LinearNode : public TokenNode {          // w, q, e, tie
  int64_t groups = 0;
  bool shared_w = false, shared_b = false;
  std::string name() const override { return "LinearAct8Backward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return none(3);
    const bool want[3] = {task_should_compute_output(0),
                          task_should_compute_output(1),
                          task_should_compute_output(2)};
    const Tensor w = get(0), q = get(1), e = get(2), tie = get(3);
    // a shared weight's gradient is one product over all clients' rows
    const bool apart = shared_w && !shared_b && want[2];
    auto [dx, dw, db] =
        linear_grad_op().call(grads[0], w, q, e, tie, shared_w ? 0 : groups,
                              want[0], want[1], want[2] && !apart);
    if (apart)
      db = std::get<2>(linear_grad_op().call(grads[0], w, q, e, tie, groups,
                                             false, false, true));
    return {want[0] ? dx : Tensor(), want[1] ? dw : Tensor(),
            want[2] ? summed(db, shared_b && !shared_w) : Tensor()};
  }
};

struct LossNode : public TokenNode {            // x, w, target, b, lse, count
  int64_t ignore = 0, reduction = 0, groups = 0;
  bool shared_w = false, shared_b = false;
  std::string name() const override { return "LinearCrossEntropyBackward"; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return none(3);
    const bool want[3] = {task_should_compute_output(0),
                          task_should_compute_output(1),
                          task_should_compute_output(2)};
    Tensor grad = grads[0], w = get(1), target = get(2), b = get(3),
           count = get(5);
    int64_t red = reduction, g = groups;
    const bool own_b = g && !shared_b && b.defined();
    if (shared_w && !own_b) {
      // shared parameters: one sum over all clients' rows, each row with its
      // client's share of the upstream gradient
      if (red == 2) grad = grad / count;
      if (red != 0) {
        std::vector<int64_t> ones(target.dim(), 1);
        ones[0] = -1;
        grad = grad.reshape(ones).expand(target.sizes());
      }
      red = 0;
      g = 0;
      count = count.narrow(0, 0, 1);
    }
    auto [dx, dw, db] =
        loss_grad_op().call(grad, get(0), w, target, or_none(b), get(4),
                            count, ignore, red, g, want[0], want[1], want[2]);
    return {want[0] ? dx : Tensor(),
            want[1] ? summed(dw, g && shared_w) : Tensor(),
            want[2] ? summed(db, g && shared_b) : Tensor()};
  }
};

template <typename... T>
void refuse_forward_mode(const char* op, const T&... inputs) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !(torch::autograd::isFwGradDefined(inputs) || ...), op,
      " has no forward-mode derivative");
}

template <typename N>
std::shared_ptr<N> make_node(torch::autograd::edge_list&& edges) {
  std::shared_ptr<N> n(new N(), torch::autograd::deleteNode);
  n->set_next_edges(std::move(edges));
  return n;
}

// The gradients are not differentiable again: asking for it raises.
template <typename... T>
std::shared_ptr<Node> refuse_second(const char* op, const T&... inputs) {
  if (!torch::autograd::compute_requires_grad(inputs...)) return nullptr;
  std::shared_ptr<Node> n(new torch::autograd::NotImplemented(op),
                          torch::autograd::deleteNode);
  n->set_next_edges(torch::autograd::collect_next_edges(inputs...));
  return n;
}

Int3 norm_autograd(c10::DispatchKeySet ks, const Tensor& x, const OptTensor& w,
                   const OptTensor& b, double eps, int64_t groups) {
  std::shared_ptr<NormNode> node;
  const Tensor wt = or_undefined(w), bt = or_undefined(b);
  refuse_forward_mode("layer_norm", x, w, b);
  if (torch::autograd::compute_requires_grad(x, wt, bt))
    node = make_node<NormNode>(torch::autograd::collect_next_edges(x, wt, bt));
  Int3 out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = norm_op().redispatch(ks & c10::after_autograd_keyset, x, w, b, eps,
                               groups);
  }
  if (node) {
    node->groups = groups;
    node->shared_w = is_shared(wt, groups, 1);
    node->shared_b = is_shared(bt, groups, 1);
    node->keep({x, wt, std::get<1>(out), std::get<2>(out)});
    torch::autograd::set_history(std::get<0>(out), node);
  }
  return out;
}

// `keep` is set by the first level that needs the 8-bit input; a level below
// it (the call on a vmap's whole population) must not drop it.
Int4 gelu_autograd(c10::DispatchKeySet ks, const Tensor& x, bool keep) {
  std::shared_ptr<GeluNode> node;
  refuse_forward_mode("gelu_act8", x);
  if (torch::autograd::compute_requires_grad(x))
    node = make_node<GeluNode>(torch::autograd::collect_next_edges(x));
  Int4 out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = gelu_op().redispatch(ks & c10::after_autograd_keyset, x,
                               keep || node != nullptr);
  }
  if (node) {
    torch::autograd::set_history(
        std::get<3>(out), refuse_second("gelu_act8's gradient", x));
    node->keep({std::get<1>(out), std::get<2>(out), std::get<3>(out)});
    torch::autograd::set_history(std::get<0>(out), node);
  }
  return out;
}

Int4 linear_autograd(c10::DispatchKeySet ks, const Tensor& x, const Tensor& w,
                     const OptTensor& b, bool keep, int64_t groups) {
  std::shared_ptr<LinearNode> node;
  const Tensor bt = or_undefined(b);
  refuse_forward_mode("linear_act8", x, w, b);
  if (torch::autograd::compute_requires_grad(x, w, bt))
    node =
        make_node<LinearNode>(torch::autograd::collect_next_edges(x, w, bt));
  Int4 out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = linear_op().redispatch(
        ks & c10::after_autograd_keyset, x, w, b,
        keep || torch::autograd::compute_requires_grad(w), groups);
  }
  if (node) {
    node->groups = groups;
    node->shared_w = is_shared(w, groups, 2);
    node->shared_b = is_shared(bt, groups, 1);
    if (auto n = refuse_second("linear_act8's gradient", x))
      torch::autograd::set_history(std::get<3>(out), n);
    node->keep({w, std::get<1>(out), std::get<2>(out), std::get<3>(out)});
    torch::autograd::set_history(std::get<0>(out), node);
  }
  return out;
}

Int3 loss_autograd(c10::DispatchKeySet ks, const Tensor& x, const Tensor& w,
                   const Tensor& target, const OptTensor& b, int64_t ignore,
                   int64_t reduction, int64_t groups) {
  std::shared_ptr<LossNode> node;
  const Tensor bt = or_undefined(b);
  refuse_forward_mode("linear_cross_entropy", x, w, b);
  if (torch::autograd::compute_requires_grad(x, w, bt))
    node = make_node<LossNode>(torch::autograd::collect_next_edges(x, w, bt));
  Int3 out;
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    out = loss_op().redispatch(ks & c10::after_autograd_keyset, x, w, target,
                               b, ignore, reduction, groups);
  }
  if (node) {
    node->ignore = ignore;
    node->reduction = reduction;
    node->groups = groups;
    node->shared_w = is_shared(w, groups, 2);
    node->shared_b = is_shared(bt, groups, 1);
    node->keep({x, w, target, bt, std::get<1>(out), std::get<2>(out)});
    torch::autograd::set_history(std::get<0>(out), node);
  }
  return out;
}

Int3 with_history(Int3 out, const std::shared_ptr<Node>& n) {
  if (n) {
    torch::autograd::set_history(std::get<0>(out), n);
    torch::autograd::set_history(std::get<1>(out), n);
    torch::autograd::set_history(std::get<2>(out), n);
  }
  return out;
}

Int3 norm_grad_autograd(c10::DispatchKeySet ks, const Tensor& dy,
                        const Tensor& x, const OptTensor& w,
                        const Tensor& mean, const Tensor& rstd, int64_t groups,
                        bool params) {
  auto n = refuse_second("layer_norm's gradient", dy, x, or_undefined(w));
  at::AutoDispatchBelowADInplaceOrView guard;
  return with_history(
      norm_grad_op().redispatch(ks & c10::after_autograd_keyset, dy, x, w,
                                mean, rstd, groups, params), n);
}

Tensor gelu_grad_autograd(c10::DispatchKeySet ks, const Tensor& dy,
                          const Tensor& q, const Tensor& e,
                          const Tensor& tie) {
  auto n = refuse_second("gelu_act8's gradient", dy, tie);
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor out = gelu_grad_op().redispatch(ks & c10::after_autograd_keyset, dy,
                                         q, e, tie);
  if (n) torch::autograd::set_history(out, n);
  return out;
}

Int3 linear_grad_autograd(c10::DispatchKeySet ks, const Tensor& dy,
                          const Tensor& w, const Tensor& q, const Tensor& e,
                          const Tensor& tie, int64_t groups, bool wx, bool ww,
                          bool wb) {
  // only the weight's gradient depends on the layer's input
  auto n = refuse_second("linear_act8's gradient", dy, w,
                         ww ? tie : Tensor());
  at::AutoDispatchBelowADInplaceOrView guard;
  return with_history(
      linear_grad_op().redispatch(ks & c10::after_autograd_keyset, dy, w, q, e,
                                  tie, groups, wx, ww, wb), n);
}

Int3 loss_grad_autograd(c10::DispatchKeySet ks, const Tensor& grad,
                        const Tensor& x, const Tensor& w, const Tensor& target,
                        const OptTensor& b, const Tensor& lse,
                        const Tensor& count, int64_t ignore, int64_t reduction,
                        int64_t groups, bool wx, bool ww, bool wb) {
  auto n = refuse_second("linear_cross_entropy's gradient", grad, x, w,
                         or_undefined(b));
  at::AutoDispatchBelowADInplaceOrView guard;
  return with_history(
      loss_grad_op().redispatch(ks & c10::after_autograd_keyset, grad, x, w,
                                target, b, lse, count, ignore, reduction,
                                groups, wx, ww, wb), n);
}

// -------------------------------------------------------------------- vmap

namespace fn = at::functorch;
using Dim = std::optional<int64_t>;

// The vmap level being processed; its key stays off while it lives.
struct Level {
  c10::impl::ExcludeDispatchKeyGuard guard{
      c10::DispatchKey::FuncTorchBatched};
  int64_t level, size;
  Level() {
    const auto layer = fn::maybeCurrentDynamicLayer();
    TORCH_CHECK(layer.has_value(), "a batched tensor escaped its vmap");
    level = layer->layerId();
    size = layer->batchSize().guard_int(__FILE__, __LINE__);
  }
  Tensor open(const Tensor& t, Dim& d) const {
    if (!t.defined()) return t;
    auto [v, dim] = fn::unwrapTensorAtLevel(t, level);
    d = dim;
    return v;
  }
  // client axis first; a tensor without one is repeated
  Tensor all(const Tensor& t) const {
    Dim d;
    Tensor v = open(t, d);
    if (!v.defined()) return v;
    if (d) return v.movedim(*d, 0);
    auto shape = v.sizes().vec();
    shape.insert(shape.begin(), size);
    return v.unsqueeze(0).expand(shape);
  }
  // client axis first, or left shared
  Tensor param(const Tensor& t) const {
    Dim d;
    Tensor v = open(t, d);
    return v.defined() && d ? v.movedim(*d, 0) : v;
  }
  OptTensor param(const OptTensor& t) const {
    return t.has_value() ? OptTensor(param(*t)) : t;
  }
  bool has(const Tensor& t) const {
    return t.defined() && fn::isBatchedAtLevel(t, level);
  }
  bool has(const OptTensor& t) const { return t.has_value() && has(*t); }
  Tensor close(const Tensor& t, bool batched = true) const {
    return batched ? fn::makeBatched(t, 0, level) : t;
  }
  // a tie has no client axis
  Tensor strip(const Tensor& t) const {
    Dim d;
    return open(t, d);
  }
  Int4 close_tied(const Int4& t, bool kept) const {
    return {close(std::get<0>(t)), close(std::get<1>(t), kept),
            close(std::get<2>(t), kept), std::get<3>(t)};
  }
  Int3 close(const Int3& t, bool a, bool b, bool c) const {
    return {close(std::get<0>(t), a), close(std::get<1>(t), b),
            close(std::get<2>(t), c)};
  }
};

void refuse_nested(int64_t groups, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      groups == 0, op,
      ": a vmap over clients inside another vmap is not supported");
}

Int3 norm_vmap(const Tensor& x, const OptTensor& w, const OptTensor& b,
               double eps, int64_t groups) {
  Level v;
  if (!v.has(x) && !v.has(w) && !v.has(b))
    return norm_op().call(x, w, b, eps, groups);
  refuse_nested(groups, "layer_norm");
  const bool own = v.has(w) || v.has(b);
  return v.close(
      norm_op().call(v.all(x), v.param(w), v.param(b), eps, own ? v.size : 0),
      true, true, true);
}

Int3 norm_grad_vmap(const Tensor& dy, const Tensor& x, const OptTensor& w,
                    const Tensor& mean, const Tensor& rstd, int64_t groups,
                    bool params) {
  Level v;
  if (!v.has(dy) && !v.has(x) && !v.has(w) && !v.has(mean) && !v.has(rstd))
    return norm_grad_op().call(dy, x, w, mean, rstd, groups, params);
  refuse_nested(groups, "layer_norm");
  return v.close(
      norm_grad_op().call(v.all(dy), v.all(x), v.param(w), v.all(mean),
                          v.all(rstd), v.size, params), true, params, params);
}

Int4 gelu_vmap(const Tensor& x, bool keep) {
  Level v;
  if (!v.has(x)) return gelu_op().call(x, keep);
  Int4 out = gelu_op().call(v.all(x), keep);
  const bool kept = std::get<1>(out).numel() == std::get<0>(out).numel();
  return v.close_tied(out, kept);
}

Tensor gelu_grad_vmap(const Tensor& dy, const Tensor& q, const Tensor& e,
                      const Tensor& tie) {
  Level v;
  if (!v.has(dy) && !v.has(q) && !v.has(e))
    return gelu_grad_op().call(dy, q, e, tie);
  return v.close(gelu_grad_op().call(v.all(dy), v.all(q), v.all(e),
                                     v.strip(tie)));
}

Int4 linear_vmap(const Tensor& x, const Tensor& w, const OptTensor& b,
                 bool keep, int64_t groups) {
  Level v;
  if (!v.has(x) && !v.has(w) && !v.has(b))
    return linear_op().call(x, w, b, keep, groups);
  refuse_nested(groups, "linear_act8");
  const bool own = v.has(w) || v.has(b);
  const Tensor xa = v.all(x);
  Int4 out = linear_op().call(xa, v.param(w), v.param(b), keep,
                              own ? v.size : 0);
  const bool kept = std::get<1>(out).dim() == xa.dim();
  return v.close_tied(out, kept);
}

Int3 linear_grad_vmap(const Tensor& dy, const Tensor& w, const Tensor& q,
                      const Tensor& e, const Tensor& tie, int64_t groups,
                      bool wx, bool ww, bool wb) {
  Level v;
  if (!v.has(dy) && !v.has(w) && !v.has(q) && !v.has(e))
    return linear_grad_op().call(dy, w, q, e, tie, groups, wx, ww, wb);
  refuse_nested(groups, "linear_act8");
  return v.close(
      linear_grad_op().call(v.all(dy), v.param(w),
                            ww ? v.all(q) : v.param(q),
                            ww ? v.all(e) : v.param(e), v.strip(tie), v.size,
                            wx, ww, wb),
      wx, ww, wb);
}

Int3 loss_vmap(const Tensor& x, const Tensor& w, const Tensor& target,
               const OptTensor& b, int64_t ignore, int64_t reduction,
               int64_t groups) {
  Level v;
  if (!v.has(x) && !v.has(w) && !v.has(target) && !v.has(b))
    return loss_op().call(x, w, target, b, ignore, reduction, groups);
  const bool own = v.has(w) || v.has(b);
  if (!own && groups == 0 && reduction == 0) {
    // rows of shared parameters: no client is told from another
    const Int3 out =
        loss_op().call(v.all(x), w, v.all(target), b, ignore, reduction, 0);
    return v.close(out, true, true, false);
  }
  if (!own && groups && w.dim() == 2 && (!b.has_value() || b->dim() == 1)) {
    // clients of an inner vmap who share the parameters with these: as many
    // groups as pairs
    const int64_t n = v.size;
    const Int3 out =
        loss_op().call(v.all(x).flatten(0, 1), w, v.all(target).flatten(0, 1),
                       b, ignore, reduction, n * groups);
    auto pairs = [&](const Tensor& t) { return t.unflatten(0, {n, groups}); };
    return v.close({pairs(std::get<0>(out)), pairs(std::get<1>(out)),
                    pairs(std::get<2>(out))}, true, true, true);
  }
  refuse_nested(groups, "linear_cross_entropy");
  return v.close(
      loss_op().call(v.all(x), v.param(w), v.all(target), v.param(b), ignore,
                     reduction, v.size),
      true, true, true);
}

Int3 loss_grad_vmap(const Tensor& grad, const Tensor& x, const Tensor& w,
                    const Tensor& target, const OptTensor& b,
                    const Tensor& lse, const Tensor& count, int64_t ignore,
                    int64_t reduction, int64_t groups, bool wx, bool ww,
                    bool wb) {
  Level v;
  if (!v.has(grad) && !v.has(x) && !v.has(w) && !v.has(target) && !v.has(b)
      && !v.has(lse) && !v.has(count))
    return loss_grad_op().call(grad, x, w, target, b, lse, count, ignore,
                               reduction, groups, wx, ww, wb);
  refuse_nested(groups, "linear_cross_entropy");
  return v.close(
      loss_grad_op().call(v.all(grad), v.all(x), v.param(w), v.all(target),
                          v.param(b), v.all(lse), v.all(count), ignore,
                          reduction, v.size, wx, ww, wb), wx, ww, wb);
}

// ------------------------------------------------------------ entry points

Tensor layer_norm_py(const Tensor& x, const OptTensor& w, const OptTensor& b,
                     double eps) {
  return std::get<0>(norm_op().call(x, w, b, eps, 0));
}
Tensor gelu_act8_py(const Tensor& x) {
  return std::get<0>(gelu_op().call(x, false));
}
Tensor linear_act8_py(const Tensor& x, const Tensor& w, const OptTensor& b) {
  return std::get<0>(linear_op().call(x, w, b, false, 0));
}
Tensor linear_cross_entropy_py(const Tensor& x, const Tensor& w,
                               const Tensor& target, const OptTensor& b,
                               int64_t ignore, int64_t reduction) {
  return std::get<0>(loss_op().call(x, w, target, b, ignore, reduction, 0));
}

std::tuple<int, int> product_tiling_py(int64_t groups, int64_t m, int64_t n,
                                       int64_t k, bool deep, bool fp32,
                                       bool act8) {
  int tile, splits;
  product_tiling(groups, m, n, k, deep, fp32 ? kF32 : kBF16, act8, &tile,
                 &splits);
  return {tile, splits};
}

}  // namespace

TORCH_LIBRARY(blades_amd, m) {
  m.def("layer_norm(Tensor x, Tensor? w, Tensor? b, float eps, int groups) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_grad(Tensor dy, Tensor x, Tensor? w, Tensor mean, "
        "Tensor rstd, int groups, bool params) -> (Tensor, Tensor, Tensor)");
  m.def("gelu_act8(Tensor x, bool keep) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("gelu_act8_grad(Tensor dy, Tensor q, Tensor e, Tensor tie) -> Tensor");
  m.def("linear_act8(Tensor x, Tensor w, Tensor? b, bool keep, int groups) "
        "-> (Tensor, Tensor, Tensor, Tensor)");
  m.def("linear_act8_grad(Tensor dy, Tensor w, Tensor q, Tensor e, "
        "Tensor tie, int groups, bool want_x, bool want_w, bool want_b) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("linear_cross_entropy(Tensor x, Tensor w, Tensor target, Tensor? b, "
        "int ignore, int reduction, int groups) -> (Tensor, Tensor, Tensor)");
  m.def("linear_cross_entropy_grad(Tensor grad, Tensor x, Tensor w, "
        "Tensor target, Tensor? b, Tensor lse, Tensor count, int ignore, "
        "int reduction, int groups, bool want_x, bool want_w, bool want_b) "
        "-> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(blades_amd, CUDA, m) {
  m.impl("layer_norm", TORCH_FN(norm_cuda));
  m.impl("layer_norm_grad", TORCH_FN(norm_grad_cuda));
  m.impl("gelu_act8", TORCH_FN(gelu_cuda));
  m.impl("gelu_act8_grad", TORCH_FN(gelu_grad_cuda));
  m.impl("linear_act8", TORCH_FN(linear_cuda));
  m.impl("linear_act8_grad", TORCH_FN(linear_grad_cuda));
  m.impl("linear_cross_entropy", TORCH_FN(loss_cuda));
  m.impl("linear_cross_entropy_grad", TORCH_FN(loss_grad_cuda));
}

TORCH_LIBRARY_IMPL(blades_amd, Autograd, m) {
  m.impl("layer_norm", TORCH_FN(norm_autograd));
  m.impl("layer_norm_grad", TORCH_FN(norm_grad_autograd));
  m.impl("gelu_act8", TORCH_FN(gelu_autograd));
  m.impl("gelu_act8_grad", TORCH_FN(gelu_grad_autograd));
  m.impl("linear_act8", TORCH_FN(linear_autograd));
  m.impl("linear_act8_grad", TORCH_FN(linear_grad_autograd));
  m.impl("linear_cross_entropy", TORCH_FN(loss_autograd));
  m.impl("linear_cross_entropy_grad", TORCH_FN(loss_grad_autograd));
}

TORCH_LIBRARY_IMPL(blades_amd, FuncTorchBatched, m) {
  m.impl("layer_norm", TORCH_FN(norm_vmap));
  m.impl("layer_norm_grad", TORCH_FN(norm_grad_vmap));
  m.impl("gelu_act8", TORCH_FN(gelu_vmap));
  m.impl("gelu_act8_grad", TORCH_FN(gelu_grad_vmap));
  m.impl("linear_act8", TORCH_FN(linear_vmap));
  m.impl("linear_act8_grad", TORCH_FN(linear_grad_vmap));
  m.impl("linear_cross_entropy", TORCH_FN(loss_vmap));
  m.impl("linear_cross_entropy_grad", TORCH_FN(loss_grad_vmap));
}

void bind_token_ops(pybind11::module_& m) {
  using nogil = py::call_guard<py::gil_scoped_release>;
  m.def("layer_norm", &layer_norm_py, nogil(), "layer norm");
  m.def("gelu_act8", &gelu_act8_py, nogil(), "GELU, its input kept in 8 bits");
  m.def("linear_act8", &linear_act8_py, nogil(),
        "linear layer, its input kept in 8 bits");
  m.def("_product_tiling", &product_tiling_py,
        "(tile rows, parts) of a product, for tests");
  m.def("linear_cross_entropy", &linear_cross_entropy_py, nogil(),
        "cross entropy of a linear head without its logits");
}
