"""Token-model training operators against plain forms in 64 bits.

Tolerances are bounds, not fits.  u is half a step of the outputs' type
(2^-8 bf16, 2^-24 fp32), U = 2^-24 the kernels' arithmetic.  A sum of n
products carries at most (n + 8) U times the sum of the products' magnitudes
(n - 1 additions, the products' and the operands' roundings, and slack for
the order), and the output one rounding more.
"""
import math

import pytest
import torch

from blades_amd import ops

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
DTYPES = [torch.float32, torch.bfloat16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
gpu = pytest.mark.gpu


def rand(*shape, dtype=torch.float32, device="cpu", seed=0, scale=1.0,
         shift=0.0):
    g = torch.Generator().manual_seed(seed + sum(shape))
    t = torch.randn(*shape, generator=g) * scale + shift
    return t.to(dtype).to(device)


def near(got, want, bound, name=""):
    """|got - want| <= bound elementwise; NaN only where wanted."""
    got, want = got.double().cpu(), want.double().cpu()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.equal(got.isnan(), want.isnan()), name
    over = ((got - want).abs() - bound).nan_to_num(nan=0.0, posinf=math.inf)
    same = got == want                                   # infinities
    over = torch.where(same, torch.zeros_like(over), over)
    if over.numel():
        assert over.max() <= 0, (name, float(over.max()),
                                 float((got - want).abs().max()))


# ------------------------------------------------------------- definitions

def norm64(x, w, b, dy, eps):
    """y, dx, dw, db and bounds on their errors in units of U."""
    x, dy = x.double(), dy.double()
    n = x.shape[-1]
    w = torch.ones(n, dtype=x.dtype, device=x.device) if w is None \
        else w.double()
    mean = x.mean(-1, keepdim=True)
    c = x - mean
    var = (c * c).mean(-1, keepdim=True)
    r = 1 / (var + eps).sqrt()
    h = c * r
    y = h * w + (0 if b is None else b.double())
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True)
              - h * (g * h).mean(-1, keepdim=True))
    flat = (-1, n)
    dw = (dy * h).reshape(flat).sum(0)
    db = dy.reshape(flat).sum(0)
    # mean: (n + 8) U mean|x|; rstd: relative (n + 8) U plus what an error of
    # the mean does to h
    k = n + 8
    em = k * x.abs().mean(-1, keepdim=True)
    eh = r * (em + c.abs() + x.abs()) + k * h.abs()
    ey = eh * w.abs() + 4 * y.abs()
    gm = g.abs().mean(-1, keepdim=True)
    ghm = (g * h).abs().mean(-1, keepdim=True)
    ehm = (g.abs() * eh).mean(-1, keepdim=True)
    ex = r * (k * (g.abs() + gm + h.abs() * ghm) + eh * ghm
              + h.abs() * ehm) + k * dx.abs()
    rows = max(1, x.numel() // n)
    ew = ((rows + 8) * (dy * h).abs() + dy.abs() * eh).reshape(flat).sum(0)
    eb = (rows + 8) * dy.abs().reshape(flat).sum(0)
    return (y, dx, dw, db), (ey, ex, ew, eb)


def stored64(x):
    """What 8-bit storage holds of x, by search for the exponent."""
    x = x.double()
    out = torch.empty_like(x)
    n = x.shape[-1]
    for lo in range(0, n, 128):
        part = x[..., lo:lo + 128]
        top = part.abs().amax(-1, keepdim=True)
        e = torch.full_like(top, -126.0)
        for _ in range(300):
            e = torch.where(127.0 * torch.exp2(e) < top, e + 1, e)
            if bool((127.0 * torch.exp2(e) >= top).logical_or(
                    ~torch.isfinite(top)).all()):
                break
        unit = torch.exp2(e)
        # what would round to 2^128, beyond fp32, stays one unit below
        v = torch.round(part / unit) * unit
        v = torch.where(v.abs() == 2.0 ** 128, v.sign() * 63 * 2.0 ** 122, v)
        out[..., lo:lo + 128] = torch.where(torch.isfinite(top), v,
                                            torch.full_like(v, math.nan))
    return out


def gelu64(x):
    x = x.double()
    return x * 0.5 * torch.erfc(-x / math.sqrt(2))


def gelu_slope64(v):
    return (0.5 * torch.erfc(-v / math.sqrt(2))
            + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi))


def loss64(x, w, y, b, ignore):
    """Row losses and lse [rows]."""
    z = x.double() @ w.double().t()
    if b is not None:
        z = z + b.double()
    lse = torch.logsumexp(z, -1)
    keep = y != ignore
    at = y.clamp(0, w.shape[0] - 1)
    rows = lse - z.gather(1, at[:, None])[:, 0]
    return torch.where(keep, rows, torch.zeros_like(rows)), lse, z


def loss_grads64(x, w, y, b, ignore, row_grad):
    rows, lse, z = loss64(x, w, y, b, ignore)
    p = torch.exp(z - lse[:, None])
    at = y.clamp(0, w.shape[0] - 1)
    p[torch.arange(len(y)), at] -= 1
    p = torch.where((y != ignore)[:, None], p * row_grad[:, None],
                    torch.zeros_like(p))
    return p @ w.double(), p.t() @ x.double(), p.sum(0), p


# -------------------------------------------------------------- layer norm

NORM_SHAPES = [(1, 1), (3, 2), (7, 16), (33, 64), (130, 65), (64, 128),
               (50, 300), (5, 512), (9, 1000), (3, 1024), (300, 2048),
               (2, 2050), (17, 4096), (2, 5001), (3, 8192), (2, 16384),
               (1, 20001)]


def check_norm(x, w, b, dy, eps=1e-5):
    dtype = x.dtype
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)
              if t is not None]
    it = iter(leaves)
    xl, wl, bl = (next(it) if t is not None else None for t in (x, w, b))
    y = ops.layer_norm(xl, wl, bl, eps)
    grads = torch.autograd.grad(y, leaves, dy)
    want, err = norm64(x, w, b, dy, eps)
    got = [y, grads[0], grads[1] if w is not None else None,
           grads[-1] if b is not None else None]
    assert y.dtype == dtype
    for name, a, r, e in zip(("y", "dx", "dw", "db"), got, want, err):
        if a is not None:
            near(a, r, HALF[dtype] * r.abs() * (1 + 1e-2) + 1.1 * U * e
                 + 1e-38, f"{name} {tuple(x.shape)} {dtype}")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
def test_norm(device, dtype, rows, dim):
    x = rand(rows, dim, dtype=dtype, device=device, scale=2.0, shift=1.0)
    check_norm(x, rand(dim, dtype=dtype, device=device, seed=1),
               rand(dim, dtype=dtype, device=device, seed=2),
               rand(rows, dim, dtype=dtype, device=device, seed=3))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("weight,bias", [(False, False), (True, False),
                                         (False, True)])
def test_norm_without_parameters(device, weight, bias):
    x = rand(2, 5, 96, device=device)
    check_norm(x, rand(96, device=device, seed=1) if weight else None,
               rand(96, device=device, seed=2) if bias else None,
               rand(2, 5, 96, device=device, seed=3))


@pytest.mark.parametrize("device", DEVICES)
def test_norm_layouts(device):
    """Transposed, sliced, misaligned and expanded inputs and gradients."""
    w, b = rand(64, device=device, seed=1), rand(64, device=device, seed=2)
    base = rand(64, 40, device=device)
    dy = rand(40, 64, device=device, seed=3)
    check_norm(base.t(), w, b, dy)
    check_norm(rand(40, 130, device=device)[:, 1:129:2], w, b, dy)
    check_norm(rand(40 * 64 + 1, device=device)[1:].view(40, 64), w, b, dy)
    check_norm(base.t().contiguous(), w, b,
               rand(1, 64, device=device).expand(40, 64))
    check_norm(rand(40, 64, device=device), rand(65, device=device)[1:], b,
               dy)


@pytest.mark.parametrize("device", DEVICES)
def test_norm_offset(device):
    """A mean a thousand deviations away costs what its own size costs."""
    x = rand(20, 256, device=device, shift=1000.0)
    check_norm(x, rand(256, device=device, seed=1),
               rand(256, device=device, seed=2),
               rand(20, 256, device=device, seed=3))


@pytest.mark.parametrize("device", DEVICES)
def test_norm_constant_rows_and_non_finite(device):
    x = torch.full((4, 128), 3.0, device=device)
    y = ops.layer_norm(x)
    assert torch.equal(y, torch.zeros_like(x))
    x[1, 7] = math.inf
    x[2, 9] = math.nan
    y = ops.layer_norm(x)
    assert y[1].isnan().all() and y[2].isnan().all()
    assert torch.equal(y[0], torch.zeros_like(y[0]))
    assert torch.equal(y[3], torch.zeros_like(y[3]))


@pytest.mark.parametrize("device", DEVICES)
def test_norm_no_rows(device):
    x = torch.empty(0, 32, device=device, requires_grad=True)
    w = torch.ones(32, device=device, requires_grad=True)
    y = ops.layer_norm(x, w)
    assert y.shape == (0, 32)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty_like(y))
    assert dx.shape == (0, 32) and torch.equal(dw, torch.zeros_like(dw))


def test_norm_refusals():
    x = torch.randn(3, 8)
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(TypeError):
        ops.layer_norm([1.0])
    with pytest.raises(ValueError):
        ops.layer_norm(torch.tensor(1.0))
    with pytest.raises(ValueError):
        ops.layer_norm(torch.empty(3, 0))
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(7))
    with pytest.raises(TypeError):
        ops.layer_norm(x, torch.ones(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(8), torch.ones(1, 8))
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=math.nan)


# -------------------------------------------------------------------- loss

LOSS_SHAPES = [(1, 1, 1), (7, 256, 1000), (33, 65, 129), (100, 300, 515),
               (128, 128, 128), (129, 31, 2000), (300, 64, 127),
               (2, 513, 300)]


def check_loss(x, w, y, b, ignore=-100, reduction="mean", scale=1.0,
               want_grads=True):
    dtype = x.dtype
    x2, y1 = x.reshape(-1, x.shape[-1]), y.reshape(-1)
    rows, lse, z = loss64(x2.cpu(), w.cpu(), y1.cpu(),
                          None if b is None else b.cpu(), ignore)
    # a logit's error, and through it the loss's (exp and log add a few U)
    za = x2.cpu().double().abs() @ w.cpu().double().abs().t()
    if b is not None:
        za = za + b.cpu().double().abs().nan_to_num(posinf=0.0)
    ez = (x.shape[-1] + 8) * U * za.max(-1).values
    er = 2 * ez + U * (lse.abs() + w.shape[0] + 16) + U * rows.abs()
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)
              if t is not None]
    bl = leaves[2] if b is not None else None
    out = ops.linear_cross_entropy(leaves[0], leaves[1], y, bl,
                                   ignore_index=ignore, reduction=reduction)
    assert out.dtype == torch.float32
    keep = y1.cpu() != ignore
    count = keep.sum().double()
    er = torch.where(keep, er, torch.zeros_like(er))
    if reduction == "none":
        near(out, rows.view(y.shape), er.view(y.shape), "rows")
        up = rand(*y.shape, device=x.device, seed=9) if y.dim() else \
            torch.ones_like(out)
        row_grad = up.reshape(-1).double().cpu()
    else:
        total = rows.sum() / (count if reduction == "mean" else 1)
        bound = er.sum() / (count if reduction == "mean" else 1)
        near(out, total, bound + 2 * U * total.abs(), reduction)
        up = torch.tensor(scale, device=x.device)
        row_grad = torch.full((len(y1),), float(scale), dtype=torch.float64)
        if reduction == "mean":
            row_grad = row_grad / count
    if not want_grads:
        return out, None
    grads = torch.autograd.grad(out, leaves, up)
    dx, dw, db, p = loss_grads64(x2.cpu(), w.cpu(), y1.cpu(),
                                 None if b is None else b.cpu(), ignore,
                                 row_grad)
    # p: relative error 2 ez (exponent) + its exponent's own rounding, and for
    # bf16 one rounding of p itself
    spread = (z - lse[:, None]).abs().nan_to_num(posinf=0.0)
    soft = torch.exp(z - lse[:, None]) * row_grad.abs()[:, None]
    ep = soft * (2 * ez[:, None] + U * (2 * spread + w.shape[0] + 24))
    ep = ep + p.abs() * 4 * U
    # the exponential instruction gives 0 below the smallest normal, 2^-126,
    # and so do the low parts of a split p: at most 2^-126 lost to each,
    # which x or w of any size multiplies
    ep = ep + 2.0 ** -124
    if dtype == torch.bfloat16:
        ep = ep + p.abs() * HALF[dtype] * 1.01
    ep = torch.where(keep[:, None], ep, torch.zeros_like(ep))
    xa, wa = x2.cpu().double().abs(), w.cpu().double().abs()
    n, v = p.shape
    ex = ep @ wa + (v + 8) * U * (p.abs() @ wa)
    ew = ep.t() @ xa + (n + 8) * U * (p.abs().t() @ xa)
    eb = ep.sum(0) + (n + 8) * U * p.abs().sum(0)
    got = [grads[0].reshape(-1, x.shape[-1]), grads[1]]
    want, err = [dx, dw], [ex, ew]
    if b is not None:
        got.append(grads[2]); want.append(db); err.append(eb)
    for name, a, r, e in zip(("dx", "dw", "db"), got, want, err):
        near(a, r, HALF[dtype] * r.abs() * 1.02 + e + 1e-38,
             f"{name} {tuple(x.shape)} {w.shape[0]} {dtype}")
    return out, grads


def loss_inputs(rows, dim, vocab, dtype, device, bias=True):
    x = rand(rows, dim, dtype=dtype, device=device)
    w = rand(vocab, dim, dtype=dtype, device=device, seed=1,
             scale=2 / math.sqrt(dim))
    b = rand(vocab, dtype=dtype, device=device, seed=2) if bias else None
    g = torch.Generator().manual_seed(rows + vocab)
    y = torch.randint(0, vocab, (rows,), generator=g)
    y[0] = vocab - 1
    if rows > 3:
        y[2] = -100
        y[3] = 0
    return x, w, y.to(device), b


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,vocab", LOSS_SHAPES)
def test_loss(device, dtype, rows, dim, vocab):
    x, w, y, b = loss_inputs(rows, dim, vocab, dtype, device)
    check_loss(x, w, y, b)
    check_loss(x, w, y, None, reduction="sum", scale=-0.5)
    check_loss(x.view(1, rows, dim), w, y.view(1, rows), b, reduction="none")


@pytest.mark.parametrize("device", DEVICES)
def test_loss_single_row_without_leading_axis(device):
    x, w, y, b = loss_inputs(1, 40, 77, torch.float32, device)
    check_loss(x[0], w, y[0], b, reduction="none")


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_in_pieces(dtype):
    """More logits than one piece of the vocabulary holds."""
    rows, vocab = 2100, 33000 if dtype == torch.float32 else 64100
    assert rows * vocab * (4 if dtype == torch.float32 else 2) > 256 << 20
    x, w, y, b = loss_inputs(rows, 24, vocab, dtype, "cuda")
    check_loss(x, w, y, b)


@pytest.mark.parametrize("device", DEVICES)
def test_loss_every_row_ignored(device):
    x, w, y, b = loss_inputs(5, 16, 30, torch.float32, device)
    y = torch.full_like(y, -100)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    mean = ops.linear_cross_entropy(x, w, y, b)
    assert mean.isnan()
    for g in torch.autograd.grad(mean, (x, w, b)):
        assert torch.equal(g, torch.zeros_like(g))
    total = ops.linear_cross_entropy(x, w, y, b, reduction="sum")
    assert total == 0


@pytest.mark.parametrize("device", DEVICES)
def test_loss_no_rows(device):
    x = torch.empty(0, 8, device=device, requires_grad=True)
    w = torch.randn(5, 8, device=device, requires_grad=True)
    y = torch.empty(0, dtype=torch.int64, device=device)
    assert ops.linear_cross_entropy(x, w, y).isnan()
    total = ops.linear_cross_entropy(x, w, y, reduction="sum")
    assert total == 0
    dx, dw = torch.autograd.grad(total, (x, w))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros_like(dw))


@pytest.mark.parametrize("device", DEVICES)
def test_loss_switched_off_words(device):
    x, w, y, b = loss_inputs(20, 32, 300, torch.float32, device)
    b[5:290] = -math.inf
    y = torch.where(y == -100, y, y % 5)
    check_loss(x, w, y, b)
    out = ops.linear_cross_entropy(x, w, torch.full_like(y, 7), b,
                                   reduction="none")
    assert torch.isposinf(out).all()         # a switched-off word as target


@pytest.mark.parametrize("device", DEVICES)
def test_loss_large_logits(device):
    """Logits of hundreds: the running maximum keeps the sums finite."""
    x, w, y, b = loss_inputs(16, 64, 400, torch.float32, device)
    check_loss(x * 100, w, y, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [-1, 50, 1 << 40])
def test_loss_target_outside_the_vocabulary(device, bad):
    x, w, y, b = loss_inputs(6, 16, 50, torch.float32, device)
    y[4] = bad
    x.requires_grad_()
    rows = ops.linear_cross_entropy(x, w, y, b, reduction="none")
    assert rows[4].isnan() and not rows[[0, 1, 2, 3, 5]].isnan().any()
    dx, = torch.autograd.grad(rows.sum(), x)
    assert dx[4].isnan().all()
    assert not dx[[0, 1, 2, 3, 5]].isnan().any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_loss_non_finite_upstream_row(device, bad):
    """Only the row's own input gradient, and the parameters', are lost."""
    x, w, y, b = loss_inputs(6, 16, 50, torch.float32, device)
    x.requires_grad_(), w.requires_grad_()
    rows = ops.linear_cross_entropy(x, w, y, b, reduction="none")
    up = torch.ones_like(rows)
    want, = torch.autograd.grad(rows, x, up, retain_graph=True)
    up[4] = bad
    up[5] = 0
    dx, dw = torch.autograd.grad(rows, (x, w), up)
    assert not dx[4].isfinite().any() and not dw.isfinite().any()
    assert torch.equal(dx[5], torch.zeros_like(dx[5]))
    near(dx[:4], want[:4], 1e-6 * want[:4].abs() + 1e-7)


@pytest.mark.parametrize("device", DEVICES)
def test_loss_ignore_index_in_the_vocabulary(device):
    x, w, y, b = loss_inputs(12, 16, 50, torch.float32, device)
    y[1] = 3
    y[y == -100] = 3
    check_loss(x, w, y, b, ignore=3)


@pytest.mark.parametrize("device", DEVICES)
def test_loss_layouts(device):
    x, w, y, b = loss_inputs(40, 64, 90, torch.float32, device)
    check_loss(x.t().contiguous().t(), w, y, b)
    check_loss(x[:, ::2], w[:, 1::2], y, b)
    wide = torch.zeros(90 * 64 + 1, device=device)
    wide[1:] = w.reshape(-1)
    check_loss(x, wide[1:].view(90, 64), y[::2].repeat_interleave(2), b)


def test_loss_refusals():
    x, w, y, b = loss_inputs(4, 8, 10, torch.float32, "cpu")
    f = ops.linear_cross_entropy
    with pytest.raises(TypeError):
        f(x.half(), w.half(), y)
    with pytest.raises(TypeError):
        f(x, w.bfloat16(), y)
    with pytest.raises(TypeError):
        f(x, w, y.int())
    with pytest.raises(ValueError):
        f(x, w[:, :7], y)
    with pytest.raises(ValueError):
        f(x, w[0], y)
    with pytest.raises(ValueError):
        f(x, w[:0], y)
    with pytest.raises(ValueError):
        f(x, w, y[:3])
    with pytest.raises(ValueError):
        f(x, w, y, b[:9])
    with pytest.raises(ValueError):
        f(x, w, y, reduction="max")


# ----------------------------------------------------- 8-bit activations

ACT_SHAPES = [(1, 1), (3, 7), (5, 127), (9, 128), (4, 129), (16, 300),
              (7, 1000), (33, 1024)]


def check_gelu(x, dy):
    dtype = x.dtype
    leaf = x.detach().clone().requires_grad_()
    y = ops.gelu_act8(leaf)
    dx, = torch.autograd.grad(y, leaf, dy)
    want = gelu64(x)
    # Phi: 1.2e-5 of the tail in bf16 kernels, 5e-7 in fp32, and the
    # exponent's rounding; all against |x| Phi <= |x|
    k = 2e-5 if dtype == torch.bfloat16 else 1e-6
    near(y, want, HALF[dtype] * want.abs() * 1.01
         + k * want.abs() + 4 * U * x.double().abs() + 1e-38, "y")
    v = stored64(x)
    slope = gelu_slope64(v)
    d = dy.double()
    near(dx, d * slope, HALF[dtype] * (d * slope).abs() * 1.01
         + d.abs() * (k + 8 * U) * (1 + v.abs()) + 1e-38, "dx")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim", ACT_SHAPES)
def test_gelu(device, dtype, rows, dim):
    check_gelu(rand(rows, dim, dtype=dtype, device=device, scale=2.0),
               rand(rows, dim, dtype=dtype, device=device, seed=1))


@pytest.mark.parametrize("device", DEVICES)
def test_gelu_scales(device):
    """Exponents at their borders: 127 * 2^e and one step beyond, subnormal,
    tiny, huge and all-zero blocks."""
    tops = [127.0, 127.00001, 126.99999, 254.0, 1.984375, 1.9843751, 1.0,
            2.0 ** -120, 2.0 ** -126, 1e-40, 3.0e38, 0.0, 128.0, 64.0, 63.5]
    x = rand(len(tops), 128, device=device)
    x = x.clamp(-1, 1) * torch.tensor(tops, device=device)[:, None]
    x[:, 3] = torch.tensor(tops, device=device)
    x[:, 5] = -torch.tensor(tops, device=device)
    check_gelu(x, torch.ones_like(x))


@pytest.mark.parametrize("device", DEVICES)
def test_gelu_far_values(device):
    x = torch.linspace(-40, 40, 1000, device=device)[None]
    check_gelu(x, torch.ones_like(x))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_gelu_non_finite_block(device, bad):
    x = rand(2, 300, device=device)
    x[0, 140] = bad
    x.requires_grad_()
    y = ops.gelu_act8(x)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert dx[0, 128:256].isnan().all()
    assert not dx[0, :128].isnan().any() and not dx[0, 256:].isnan().any()
    assert not dx[1].isnan().any()


@pytest.mark.parametrize("device", DEVICES)
def test_act8_layouts_and_empty(device):
    x = rand(256, 40, device=device).t()
    check_gelu(x, rand(40, 256, device=device, seed=1))
    flat = rand(40 * 128 + 1, device=device)[1:].view(40, 128)
    check_gelu(flat, rand(1, 128, device=device).expand(40, 128))
    e = torch.empty(0, 64, device=device, requires_grad=True)
    y = ops.gelu_act8(e)
    assert torch.autograd.grad(y, e, torch.empty_like(y))[0].shape == e.shape


LINEAR_SHAPES = [(1, 1, 1), (7, 33, 5), (64, 128, 128), (130, 300, 129),
                 (300, 257, 64), (1000, 40, 200), (2, 512, 1000)]


def check_linear(x, w, b, dy):
    dtype = x.dtype
    leaves = [t.detach().clone().requires_grad_() for t in (x, w, b)
              if t is not None]
    y = ops.linear_act8(leaves[0], leaves[1],
                        leaves[2] if b is not None else None)
    grads = torch.autograd.grad(y, leaves, dy)
    n, m = w.shape[1], w.shape[0]
    x2, dy2 = x.reshape(-1, n).double(), dy.reshape(-1, m).double()
    wd = w.double()
    bd = 0 if b is None else b.double()
    k = len(x2)
    s = stored64(x.reshape(-1, n))
    want = [(x2 @ wd.t() + bd).view(y.shape), (dy2 @ wd).view(x.shape),
            dy2.t() @ s, dy2.sum(0)]
    mags = [(x2.abs() @ wd.abs().t()
             + (bd.abs() if b is not None else 0)).view(y.shape),
            (dy2.abs() @ wd.abs()).view(x.shape), dy2.abs().t() @ s.abs(),
            dy2.abs().sum(0)]
    for name, a, r, e, c in zip(("y", "dx", "dw", "db"), (y, *grads), want,
                                mags, (n, m, k, k)):
        near(a, r, HALF[dtype] * r.abs() * 1.01 + (c + 8) * U * e + 1e-38,
             f"{name} {tuple(x.shape)} {m} {dtype}")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,m", LINEAR_SHAPES)
def test_linear(device, dtype, rows, n, m):
    check_linear(rand(rows, n, dtype=dtype, device=device),
                 rand(m, n, dtype=dtype, device=device, seed=1),
                 rand(m, dtype=dtype, device=device, seed=2),
                 rand(rows, m, dtype=dtype, device=device, seed=3))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_layouts(device):
    x = rand(3, 11, 64, device=device)
    w, b = rand(30, 64, device=device, seed=1), rand(30, device=device)
    dy = rand(3, 11, 30, device=device, seed=2)
    check_linear(x, w, None, dy)
    check_linear(x.transpose(0, 1).contiguous().transpose(0, 1), w, b, dy)
    check_linear(x, rand(64, 30, device=device).t(), b,
                 rand(1, 1, 30, device=device).expand(3, 11, 30))
    check_linear(rand(11, 130, device=device)[:, 1:129:2], w, b,
                 rand(30, 11, device=device).t())


@pytest.mark.parametrize("device", DEVICES)
def test_linear_wide_range(device):
    """fp32 values of very different size: the product keeps fp32's bits."""
    x = rand(50, 96, device=device) * torch.exp2(
        torch.arange(96, device=device) % 40 - 20.0)
    check_linear(x, rand(20, 96, device=device, seed=1), None,
                 rand(50, 20, device=device, seed=2, scale=1e-6))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,n,m", [(1500, 77, 203), (700, 1025, 131),
                                      (4100, 1030, 2051), (9000, 4, 3),
                                      (5001, 520, 777)])
def test_linear_long_and_odd(dtype, rows, n, m):
    """Every tile size with rows that end inside a 16-byte access, and
    contractions long enough for the unchecked steps."""
    check_linear(rand(rows, n, dtype=dtype, device="cuda"),
                 rand(m, n, dtype=dtype, device="cuda", seed=1),
                 rand(m, dtype=dtype, device="cuda", seed=2),
                 rand(rows, m, dtype=dtype, device="cuda", seed=3))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,dim,vocab", [(1000, 333, 1001),
                                            (2500, 77, 5003),
                                            (64, 1030, 9999)])
def test_loss_long_and_odd(dtype, rows, dim, vocab):
    x, w, y, b = loss_inputs(rows, dim, vocab, dtype, "cuda")
    check_loss(x, w, y, b)


@pytest.mark.parametrize("device", DEVICES)
def test_linear_largest_values(device):
    """8-bit blocks that reach fp32's largest values keep them."""
    x = rand(30, 256, device=device).clamp(-1, 1)
    x[:, :128] *= 3.3e38
    x[4, 3], x[5, 4] = 3.4e38, -3.4e38
    w = torch.zeros(20, 256, device=device)
    check_linear(x, w, None, rand(30, 20, device=device, scale=1e-30))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", ["norm", "loss", "gelu", "linear"])
def test_forward_mode_refused(device, fn):
    x, w, y, b = loss_inputs(4, 16, 16, torch.float32, device)
    call = {"norm": lambda x: ops.layer_norm(x, b, b),
            "loss": lambda x: ops.linear_cross_entropy(x, w, y, b),
            "gelu": ops.gelu_act8,
            "linear": lambda x: ops.linear_act8(x, w, b)}[fn]
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))


@pytest.mark.parametrize("device", DEVICES)
def test_linear_no_rows(device):
    x = torch.empty(0, 8, device=device, requires_grad=True)
    w = torch.randn(4, 8, device=device, requires_grad=True)
    b = torch.randn(4, device=device, requires_grad=True)
    y = ops.linear_act8(x, w, b)
    assert y.shape == (0, 4)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert dx.shape == (0, 8)
    assert torch.equal(dw, torch.zeros_like(dw))
    assert torch.equal(db, torch.zeros_like(db))


def test_act8_refusals():
    x = torch.randn(3, 8)
    with pytest.raises(TypeError):
        ops.gelu_act8(x.double())
    with pytest.raises(ValueError):
        ops.gelu_act8(torch.tensor(1.0))
    with pytest.raises(ValueError):
        ops.linear_act8(x, torch.randn(8))
    with pytest.raises(ValueError):
        ops.linear_act8(x, torch.randn(0, 8))
    with pytest.raises(ValueError):
        ops.linear_act8(x, torch.randn(4, 7))
    with pytest.raises(ValueError):
        ops.linear_act8(x, torch.randn(4, 8), torch.randn(3))
    with pytest.raises(TypeError):
        ops.linear_act8(x, torch.randn(4, 8).bfloat16())


# --------------------------------------------- populations (torch.func)

def loss_fn(w, b, x, y):
    return ops.linear_cross_entropy(x, w, y, b)


def norm_fn(w, b, x, y):
    return ops.layer_norm(x, w, b)


def gelu_linear_fn(w, b, x, y):
    return ops.gelu_act8(ops.linear_act8(x, w, b))


def population(fn, clients, device, dtype=torch.float32, seed=0):
    n, d, v = 9, 40, 23
    x = rand(clients, n, d, device=device, dtype=dtype, seed=seed)
    y = torch.randint(0, v, (clients, n),
                      generator=torch.Generator().manual_seed(1)).to(device)
    y[0, 1] = -100
    m = d if fn is norm_fn else v
    shape = (d,) if fn is norm_fn else (v, d)
    w = rand(clients, *shape, device=device, dtype=dtype, seed=seed + 1)
    b = rand(clients, m, device=device, dtype=dtype, seed=seed + 2)
    up = {loss_fn: rand(clients, device=device, seed=3),
          norm_fn: rand(clients, n, d, device=device, dtype=dtype, seed=3),
          gelu_linear_fn: rand(clients, n, v, device=device, dtype=dtype,
                               seed=3)}[fn]
    return w, b, x, y, up


def one_by_one(fn, w, b, x, y, up):
    """Each client alone through ordinary autograd."""
    outs = []
    for i in range(len(x)):
        leaves = [t.detach().clone().requires_grad_()
                  for t in (w[i], b[i], x[i])]
        out = fn(*leaves, y[i])
        outs.append((out.detach(), *torch.autograd.grad(out, leaves, up[i])))
    return [torch.stack(t) for t in zip(*outs)]


FNS = [loss_fn, norm_fn, gelu_linear_fn]


def close(a, b, dtype=torch.float32):
    """Two runs of the same sums in another order or kernel."""
    tol = 1e-5 if dtype == torch.float32 else 2.0 ** -6
    assert a.shape == b.shape
    scale = b.double().abs().max().item() + 1e-30
    assert (a.double() - b.double()).abs().max().item() <= tol * scale


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fn", FNS)
@pytest.mark.parametrize("shared", [True, False])
def test_vmap_of_vjp(device, dtype, fn, shared):
    w, b, x, y, up = population(fn, 4, device, dtype)
    if shared:
        w, b = w[:1].expand_as(w), b[:1].expand_as(b)
    want = one_by_one(fn, w, b, x, y, up)

    def step(w, b, x, y, up):
        out, pull = torch.func.vjp(lambda *a: fn(*a, y), w, b, x)
        return (out, *pull(up))
    if shared:
        got = torch.func.vmap(step, in_dims=(None, None, 0, 0, 0))(
            w[0], b[0], x, y, up)
    else:
        got = torch.func.vmap(step)(w, b, x, y, up)
    for g, r in zip(got, want):
        close(g, r, dtype)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
@pytest.mark.parametrize("shared", [True, False])
def test_grad_of_vmap(device, fn, shared):
    w, b, x, y, up = population(fn, 4, device)
    if shared:
        w, b = w[:1].expand_as(w), b[:1].expand_as(b)
    want = one_by_one(fn, w, b, x, y, up)
    dims = (None, None, 0, 0) if shared else (0, 0, 0, 0)

    def total(w, b, x):
        return (torch.func.vmap(fn, in_dims=dims)(w, b, x, y) * up).sum()
    args = (w[0], b[0], x) if shared else (w, b, x)
    got = torch.func.grad(total, argnums=(0, 1, 2))(*args)
    for i, (g, r) in enumerate(zip(got, want[1:])):
        close(g, r.sum(0) if shared and i < 2 else r)
    # and by ordinary autograd through the vmap
    leaves = [t.detach().clone().requires_grad_() for t in args]
    for g, r in zip(torch.autograd.grad(total(*leaves), leaves), got):
        close(g, r)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_vmap_other_axes(device, fn):
    """Client axes that are not the first, and inputs without one."""
    w, b, x, y, up = population(fn, 4, device)
    want = torch.stack([fn(w[i], b[i], x[i], y[i]) for i in range(4)])
    got = torch.func.vmap(fn, in_dims=(-1, 1, 1, 1))(
        w.movedim(0, -1), b.movedim(0, 1), x.movedim(0, 1), y.movedim(0, 1))
    close(got, want)
    got = torch.func.vmap(fn, in_dims=(0, None, None, None))(
        w, b[0], x[0], y[0])
    close(got, torch.stack([fn(w[i], b[0], x[0], y[0]) for i in range(4)]))
    # no input of the operator depends on the client
    got = torch.func.vmap(lambda s: fn(w[0], b[0], x[0], y[0]) * s)(
        torch.arange(4.0, device=device))
    close(got[1], fn(w[0], b[0], x[0], y[0]))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_vmap_chunks(device, fn):
    w, b, x, y, up = population(fn, 5, device)
    whole = torch.func.vmap(fn, in_dims=(None, None, 0, 0))(w[0], b[0], x, y)
    parts = torch.func.vmap(fn, in_dims=(None, None, 0, 0), chunk_size=2)(
        w[0], b[0], x, y)
    close(parts, whole)


@pytest.mark.parametrize("device", DEVICES)
def test_vmap_loss_rows(device):
    w, b, x, y, _ = population(loss_fn, 3, device)
    f = lambda x, y: ops.linear_cross_entropy(x, w[0], y, b[0],
                                              reduction="none")
    got = torch.func.vmap(f)(x, y)
    close(got, torch.stack([f(x[i], y[i]) for i in range(3)]))
    g = torch.func.vmap(torch.func.grad(lambda x, y: f(x, y).square().sum()))
    want = []
    for i in range(3):
        leaf = x[i].clone().requires_grad_()
        want.append(torch.autograd.grad(f(leaf, y[i]).square().sum(),
                                        leaf)[0])
    close(g(x, y), torch.stack(want))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_only_the_input_needs_a_gradient_of_tracked_parameters(device, fn):
    """vmap(grad) in the input alone while outer levels track parameters."""
    w, b, x, y, up = population(fn, 3, device)
    f = fn
    w0, b0 = w[0].clone().requires_grad_(), b[0].clone().requires_grad_()

    def in_x(x, y, up):
        out, pull = torch.func.vjp(lambda x: f(w0, b0, x, y), x)
        return pull(up)[0]
    got = torch.func.vmap(in_x)(x, y, up)
    want = one_by_one(f, w[:1].expand_as(w), b[:1].expand_as(b), x, y, up)[3]
    close(got.detach(), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_nested_vmap_refused(device, fn):
    w, b, x, y, _ = population(fn, 4, device)
    inner = torch.func.vmap(fn)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.vmap(inner)(w.unflatten(0, (2, 2)), b.unflatten(0, (2, 2)),
                               x.unflatten(0, (2, 2)), y.unflatten(0, (2, 2)))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_second_gradient_refused(device, fn):
    w, b, x, y, up = population(fn, 1, device)
    leaves = [t[0].clone().requires_grad_() for t in (w, b, x)]
    out = (fn(*leaves, y[0]) ** 2).sum()
    first = torch.autograd.grad(out, leaves, create_graph=True)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.autograd.grad(sum(g.square().sum() for g in first), leaves)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
def test_partial_gradients(device, fn):
    """Any subset of the inputs, and no gradient at all."""
    w, b, x, y, up = population(fn, 1, device)
    want = one_by_one(fn, w, b, x, y, up)
    for i in range(3):
        leaves = [w[0].clone(), b[0].clone(), x[0].clone()]
        leaves[i].requires_grad_()
        out = fn(*leaves, y[0])
        close(torch.autograd.grad(out, leaves[i], up[0])[0], want[1 + i][0])
    with torch.no_grad():
        close(fn(w[0], b[0], x[0], y[0]), want[0][0])


def test_gradients_against_differences():
    """The 64-bit definitions' central differences along a direction."""
    x, w, y, b = loss_inputs(9, 24, 50, torch.float32, "cpu")
    vx, vw = rand(9, 24, seed=5).double(), rand(50, 24, seed=6).double()
    h = 1e-5

    def mean64(t):
        r = loss64(x.double() + t * vx, w.double() + t * vw, y, b, -100)[0]
        return r.sum() / (y != -100).sum()
    slope = (mean64(h) - mean64(-h)) / (2 * h)
    leaves = [x.clone().requires_grad_(), w.clone().requires_grad_()]
    gx, gw = torch.autograd.grad(ops.linear_cross_entropy(*leaves, y, b),
                                 leaves)
    got = (gx.double() * vx).sum() + (gw.double() * vw).sum()
    assert abs(got - slope) <= 1e-5 * (1 + abs(slope))

    dy = rand(9, 24, seed=7)
    g = rand(24, seed=8)

    def norm_at(t):
        z = x.double() + t * vx
        c = z - z.mean(-1, keepdim=True)
        return (dy.double() * c / (c.square().mean(-1, keepdim=True)
                                   + 1e-5).sqrt() * g.double()).sum()
    slope = (norm_at(h) - norm_at(-h)) / (2 * h)
    leaf = x.clone().requires_grad_()
    gx, = torch.autograd.grad(ops.layer_norm(leaf, g), leaf, dy)
    assert abs((gx.double() * vx).sum() - slope) <= 1e-4 * (1 + abs(slope))


# --------------------------------------------------- streams and graphs

@gpu
@pytest.mark.parametrize("fn", FNS)
def test_results_repeat(fn):
    w, b, x, y, up = population(fn, 6, "cuda")
    first = one_by_one(fn, w, b, x, y, up)
    for _ in range(3):
        for a, r in zip(one_by_one(fn, w, b, x, y, up), first):
            assert torch.equal(a, r)


@gpu
@pytest.mark.parametrize("fn", FNS)
def test_side_stream(fn):
    w, b, x, y, up = population(fn, 2, "cuda")
    want = one_by_one(fn, w, b, x, y, up)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = one_by_one(fn, w, b, x, y, up)
    torch.cuda.current_stream().wait_stream(s)
    for a, r in zip(got, want):
        assert torch.equal(a, r)


@gpu
@pytest.mark.parametrize("fn", FNS)
@pytest.mark.parametrize("rows", [9, 600])
def test_captured_population_step(fn, rows):
    """A vmapped step in two captured graphs, replayed in turn on new
    inputs, with eager work between the replays."""
    def step(w, b, x, y, up):
        out, pull = torch.func.vjp(lambda *a: fn(*a, y), w, b, x)
        return (out, *pull(up))
    run = torch.func.vmap(step)
    w, b, x, y, up = population(fn, 3, "cuda")
    reps = -(-rows // 9)
    x, y = x.repeat(1, reps, 1)[:, :rows], y.repeat(1, reps)[:, :rows]
    if fn is not loss_fn:
        up = up.repeat(1, reps, 1)[:, :rows]
    static = [t.contiguous().clone() for t in (w, b, x, y, up)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            run(*static)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(*static))
        graphs.append(g)
    for i in range(4):
        for t in static:
            if t.is_floating_point():
                t.copy_(torch.randn(t.shape, device="cuda"))
        graphs[i % 2].replay()
        want = run(*static)
        torch.cuda.synchronize()
        for a, r in zip(outs[i % 2], want):
            assert torch.equal(a, r)


# ------------------------------------------- what is refused at every level

def _calls(device):
    """name -> (scalar function of (x, w), x, w); the upstream gradient of
    each operator is a constant."""
    x, w, y, b = loss_inputs(5, 16, 16, torch.float32, device)
    return {"norm": lambda x, w: ops.layer_norm(x, w[0]).sum(),
            "loss": lambda x, w: ops.linear_cross_entropy(x, w, y, b),
            "gelu": lambda x, w: ops.gelu_act8(x).sum(),
            "linear": lambda x, w: ops.linear_act8(x, w, b).sum()}, x, w


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", ["norm", "loss", "gelu", "linear"])
def test_second_gradient_refused_with_constant_upstream(device, fn):
    """A gradient penalty: the first gradients come, their own raise."""
    calls, x, w = _calls(device)
    x.requires_grad_(), w.requires_grad_()
    leaves = (x,) if fn == "gelu" else (x, w)
    want = torch.autograd.grad(calls[fn](x, w), leaves)
    out = calls[fn](x, w)
    first = torch.autograd.grad(out, leaves, create_graph=True)
    for a, r in zip(first, want):
        assert torch.equal(a, r)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.autograd.grad(out + sum(g.square().sum() for g in first), x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", ["norm", "loss", "gelu"])
@pytest.mark.parametrize("clients", [0, 3])
def test_nested_func_grad_refused(device, fn, clients):
    calls, x, w = _calls(device)

    def penalty(x):
        return torch.func.grad(lambda z: calls[fn](z, w))(x).square().sum()
    outer = torch.func.grad(penalty)
    with pytest.raises((NotImplementedError, RuntimeError)):
        if clients:
            torch.func.vmap(outer)(x.expand(clients, *x.shape))
        else:
            outer(x)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", ["norm", "loss", "linear"])
@pytest.mark.parametrize("clients", [0, 3])
def test_mixed_second_gradient_refused(device, fn, clients):
    """The weight's gradient, differentiated by the input."""
    calls, x, w = _calls(device)

    def penalty(x, w):
        return torch.func.grad(lambda u: calls[fn](x, u))(w).square().sum()
    outer = torch.func.grad(penalty)
    with pytest.raises((NotImplementedError, RuntimeError)):
        if clients:
            torch.func.vmap(outer, in_dims=(0, None))(
                x.expand(clients, *x.shape), w)
        else:
            outer(x, w)


@pytest.mark.parametrize("device", DEVICES)
def test_input_gradient_of_linear_is_constant_in_the_input(device):
    """dx = dy w does not depend on x: nothing is missing from its second
    gradient, and it is not refused."""
    x, w, _, b = loss_inputs(5, 16, 16, torch.float32, device)
    g = torch.func.grad(lambda x: torch.func.grad(
        lambda z: ops.linear_act8(z, w, b).sum())(x).square().sum())(x)
    assert torch.equal(g, torch.zeros_like(g))


@gpu
def test_norm_widest_rows_parameter_gradients():
    """One row of 2**28 values: the kernel that joins the parameters'
    gradients covers them all.  With one row db is dy, bit for bit, and dw is
    dy * h: a rounding of each factor and of the product, and h's own error,
    (n + 8) U of it in the worst order of its sums."""
    n = 1 << 28
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, n, generator=g, device="cuda")
    dy = torch.randn(1, n, generator=g, device="cuda")
    w = torch.ones(n, device="cuda", requires_grad=True)
    b = torch.zeros(n, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), dy)
    assert torch.equal(db, dy[0])
    # y is h here: dw differs from dy * y by the product's rounding alone
    y = y.detach()
    assert bool(((dw - dy[0] * y[0]).abs()
                 <= 4 * U * (dy[0] * y[0]).abs()).all())
    assert abs(float(y.double().mean())) < 1e-3
    assert abs(float(y.double().square().mean()) - 1) < 1e-3


# ------------------------------------------------------ fp32 products' bits

@pytest.mark.parametrize("device", DEVICES)
def test_linear_single_products_keep_fp32(device):
    """Products of two values whose bits are all set: a product's rounding is
    U, and a kernel that multiplies in parts adds at most five more roundings
    of partial sums and U of products left out: 7 U in all, less where sums of
    parts are exact."""
    k = torch.arange(1, 2049, dtype=torch.int32)
    a = (0x3F810000 - k).view(torch.float32)[:, None].to(device)
    got = ops.linear_act8(a, a).double()
    want = a.double() @ a.double().t()
    assert ((got - want) / want).abs().max() <= 7 * U


@pytest.mark.parametrize("device", DEVICES)
def test_linear_single_products_have_no_bias(device):
    """Errors of independent products, each at most 7 U, average out: over
    n of them beyond 7 U sqrt(2 ln(2e9) / n) = 0.18 U once in 1e9 (a mean of
    bounded variables, Hoeffding)."""
    n = 65535
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(0x3F800000, 0x40000000, (n, 1, 1), generator=g,
                          dtype=torch.int32).view(torch.float32).to(device)
            for _ in range(2))
    got = torch.func.vmap(ops.linear_act8)(a, b).double()
    want = a.double() * b.double()
    assert abs(((got - want) / want).mean()) <= 0.18 * U


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["sum", "mean"])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_loss_non_finite_upstream_leaves_ignored_rows(device, dtype, reduction,
                                                      bad):
    """Rows that do not count have no gradient whatever comes from above."""
    x, w, y, b = loss_inputs(6, 16, 50, dtype, device)       # y[2] is ignored
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    out = ops.linear_cross_entropy(x, w, y, b, reduction=reduction)
    up = torch.tensor(bad, device=device)
    dx, dw, db = torch.autograd.grad(out, (x, w, b), up)
    assert torch.equal(dx[2], torch.zeros_like(dx[2]))
    assert not dx[[0, 1, 3, 4, 5]].isfinite().any()
    assert not dw.isfinite().any() and not db.isfinite().any()
    # nothing counts: a sum has no gradient at all
    if reduction == "sum":
        out = ops.linear_cross_entropy(x, w, torch.full_like(y, -100), b,
                                       reduction="sum")
        for g in torch.autograd.grad(out, (x, w, b), up):
            assert torch.equal(g, torch.zeros_like(g))


# ------------------------------------------------- shared parameters, nested

def loss_sum_fn(w, b, x, y):
    return ops.linear_cross_entropy(x, w, y, b, reduction="sum")


def loss_rows_fn(w, b, x, y):
    return ops.linear_cross_entropy(x, w, y, b, reduction="none")


NESTED = [loss_fn, loss_sum_fn, loss_rows_fn, norm_fn, gelu_linear_fn]


def nested_inputs(fn, device):
    """Shared w, b; x, y with two client axes (2, 3); an upstream gradient."""
    w, b, x, y, _ = population(
        fn if fn in (norm_fn, gelu_linear_fn) else loss_fn, 6, device)
    w, b = w[0].contiguous(), b[0].contiguous()
    out = torch.stack([fn(w, b, x[i], y[i]) for i in range(6)])
    up = rand(*out.shape, device=device, seed=11)
    nest = lambda t: t.unflatten(0, (2, 3))
    return w, b, x, y, up, nest


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", NESTED)
def test_nested_vmap_of_shared_parameters(device, fn):
    w, b, x, y, up, nest = nested_inputs(fn, device)
    dims = (None, None, 0, 0)
    twice = torch.func.vmap(torch.func.vmap(fn, in_dims=dims), in_dims=dims)
    want = torch.stack([fn(w, b, x[i], y[i]) for i in range(6)])
    close(twice(w, b, nest(x), nest(y)), nest(want))
    # another axis order, and the inner axis missing from the targets
    got = torch.func.vmap(torch.func.vmap(fn, in_dims=dims),
                          in_dims=(None, None, 1, 1))(
        w, b, nest(x).movedim(0, 1), nest(y).movedim(0, 1))
    close(got, nest(want))
    # the gradients of everything, summed over both axes for the parameters
    def total(w, b, x):
        return (twice(w, b, nest(x), nest(y)) * nest(up)).sum()
    got = torch.func.grad(total, argnums=(0, 1, 2))(w, b, x)
    leaves = [t.clone().requires_grad_() for t in (w, b, x)]
    out = torch.stack([fn(leaves[0], leaves[1], leaves[2][i], y[i])
                       for i in range(6)])
    for g, r in zip(got, torch.autograd.grad((out * up).sum(), leaves)):
        close(g, r)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", NESTED)
def test_gradient_between_vmaps_of_shared_parameters(device, fn):
    """vmap(grad(vmap(...))): the outer clients' gradients of their inner
    populations."""
    w, b, x, y, up, nest = nested_inputs(fn, device)

    def inner(w, b, x, y, up):
        out = torch.func.vmap(fn, in_dims=(None, None, 0, 0))(w, b, x, y)
        return (out * up).sum()
    step = torch.func.grad(inner, argnums=(0, 1, 2))
    got = torch.func.vmap(step, in_dims=(None, None, 0, 0, 0))(
        w, b, nest(x), nest(y), nest(up))
    for i in range(2):
        leaves = [t.clone().requires_grad_() for t in (w, b, nest(x)[i])]
        out = torch.stack([fn(leaves[0], leaves[1], leaves[2][k],
                              nest(y)[i][k]) for k in range(3)])
        want = torch.autograd.grad((out * nest(up)[i]).sum(), leaves)
        for g, r in zip(got, want):
            close(g[i], r)


# ------------------------------- one of weight and bias shared, one per client

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fn", [loss_fn, loss_rows_fn, norm_fn,
                                gelu_linear_fn])
@pytest.mark.parametrize("own", ["w", "b"])
def test_one_parameter_per_client(device, dtype, fn, own):
    w, b, x, y, up = population(loss_fn if fn is loss_rows_fn else fn, 4,
                                device, dtype)
    if fn is loss_rows_fn:
        up = rand(4, x.shape[1], device=device, seed=3)
    if own == "w":
        b = b[:1].expand_as(b)
    else:
        w = w[:1].expand_as(w)
    want = one_by_one(fn, w, b, x, y, up)
    w_in, b_in = (w, b[0]) if own == "w" else (w[0], b)
    dims = (0, None, 0) if own == "w" else (None, 0, 0)

    def step(w, b, x, y, up):
        out, pull = torch.func.vjp(lambda *a: fn(*a, y), w, b, x)
        return (out, *pull(up))
    got = torch.func.vmap(step, in_dims=dims + (0, 0))(w_in, b_in, x, y, up)
    for g, r in zip(got, want):
        close(g, r, dtype)

    def total(w, b, x):
        out = torch.func.vmap(fn, in_dims=dims + (0,))(w, b, x, y)
        return (out * up).sum()
    leaves = [t.detach().clone().requires_grad_() for t in (w_in, b_in, x)]
    got = torch.autograd.grad(total(*leaves), leaves)
    want[1 if own == "b" else 2] = want[1 if own == "b" else 2].float().sum(0)
    for g, r, t in zip(got, want[1:], leaves):
        assert g.dtype == dtype
        close(g.float(), r.float(), dtype)


def test_shared_parameters_are_not_repeated(monkeypatch):
    """A shared parameter reaches the operators' plain forms as it is, also
    where the other one is per client."""
    from blades_amd.ops import torch_ref
    seen = []
    for name, at in (("norm_forward", (1, 2)), ("loss_forward", (1, 3)),
                     ("linear_forward", (1, 2))):
        def spy(*a, _f=getattr(torch_ref, name), _at=at, **kw):
            seen.append(tuple(a[i].dim() for i in _at))
            return _f(*a, **kw)
        monkeypatch.setattr(torch_ref, name, spy)
    for fn, dims in ((norm_fn, (1, 1)), (loss_fn, (2, 1)),
                     (gelu_linear_fn, (2, 1))):
        w, b, x, y, _ = population(fn, 4, "cpu")
        seen.clear()
        torch.func.vmap(fn)(w, b, x, y)
        torch.func.vmap(fn, in_dims=(0, None, 0, 0))(w, b[0], x, y)
        torch.func.vmap(fn, in_dims=(None, 0, 0, 0))(w[0], b, x, y)
        torch.func.vmap(fn, in_dims=(None, None, 0, 0))(w[0], b[0], x, y)
        i, j = dims
        assert seen == [(i + 1, j + 1), (i + 1, j), (i, j + 1), (i, j)]


@gpu
def test_shared_weight_is_not_copied_per_client():
    """64 clients' biases on one head of 20 MB: a copy per client would take
    1.3 GB."""
    w = rand(20000, 256, device="cuda")
    b = rand(64, 20000, device="cuda")
    x = rand(64, 4, 256, device="cuda")
    y = torch.zeros(64, 4, dtype=torch.int64, device="cuda")
    for f in (lambda x, b, y: ops.linear_cross_entropy(x, w, y, b),
              lambda x, b, y: ops.linear_act8(x, w, b)):
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = torch.func.vmap(f)(x, b, y)
        assert torch.cuda.max_memory_allocated() - before < 100 << 20
        del out


# ------------------------------------------- bf16 on the framework's kernels

@gpu
def test_bf16_products_are_the_operators_own():
    """A product that the operators left to the library would take the type
    that autocast gives the library's products."""
    x, w = (rand(64, 48, dtype=torch.bfloat16, device="cuda", seed=i)
            for i in range(2))
    b = rand(64, dtype=torch.bfloat16, device="cuda")
    f = torch.ops.blades_amd.linear_act8
    g = torch.ops.blades_amd.linear_act8_grad
    y, q, e, tie = f(x, w, b, True, 0)
    dy = torch.ones_like(y)
    want = (y, *g(dy, w, q, e, tie, 0, True, True, True))
    with torch.autocast("cuda", torch.float16):
        got = (f(x, w, b, True, 0)[0],
               *g(dy, w, q, e, tie, 0, True, True, True))
    for a, r in zip(got, want):
        assert a.dtype == torch.bfloat16 and torch.equal(a, r)


@gpu
@pytest.mark.parametrize("fn", FNS)
def test_bf16_results_repeat(fn):
    w, b, x, y, up = population(fn, 6, "cuda", torch.bfloat16)
    x = x.repeat(1, 200, 1)
    y = y.repeat(1, 200)
    if fn is not loss_fn:
        up = up.repeat(1, 200, 1)
    first = one_by_one(fn, w, b, x, y, up)
    for _ in range(3):
        for a, r in zip(one_by_one(fn, w, b, x, y, up), first):
            assert torch.equal(a, r)


@gpu
def test_bf16_step_captured():
    """Linear layer and loss of one client, captured and replayed on new
    inputs with eager work between the replays."""
    x = rand(700, 96, dtype=torch.bfloat16, device="cuda")
    w = rand(96, 96, dtype=torch.bfloat16, device="cuda", seed=1)
    v = rand(1000, 96, dtype=torch.bfloat16, device="cuda", seed=2)
    y = torch.randint(0, 1000, (700,), device="cuda")

    def step(x, w, v):
        def loss(x, w, v):
            return ops.linear_cross_entropy(ops.linear_act8(x, w), v, y)
        grads, value = torch.func.grad_and_value(loss, argnums=(0, 1, 2))(
            x, w, v)
        return (value, *grads)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(x, w, v)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x, w, v)
    for i in range(4):
        x.copy_(rand(700, 96, dtype=torch.bfloat16, device="cuda", seed=9 + i))
        graph.replay()
        want = step(x, w, v)
        torch.cuda.synchronize()
        for a, r in zip(out, want):
            assert torch.equal(a, r)


# ---------------------------------------------------------------- autocast

CASTS = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("cast", CASTS)
def test_autocast_types(device, cast):
    """Under autocast an operator is the one of inputs cast beforehand: norms
    in float32, products in bfloat16, and float32 for float16."""
    x, w, y, b = loss_inputs(9, 24, 24, torch.float32, device)
    low = torch.bfloat16 if cast == torch.bfloat16 else torch.float32
    calls = [(lambda x, w, b: ops.layer_norm(x, w[0], b), torch.float32),
             (lambda x, w, b: ops.linear_act8(x, w, b), low),
             (lambda x, w, b: ops.linear_cross_entropy(x, w, y, b), low)]
    for f, typed in calls:
        def run(*args):
            out = f(*args)
            return (out, *torch.autograd.grad(out.float().sum(), args))
        # what a layer before this one may hand over, and parameters
        for given in (torch.float32, cast):
            leaves = [x.to(given), w.clone(), b.clone()]
            for t in leaves:
                t.requires_grad_()
            with torch.autocast(device, cast):
                got = run(*leaves)
            want = run(*[t.detach().to(given if i == 0 else t.dtype).to(typed)
                         .requires_grad_() for i, t in enumerate(leaves)])
            assert got[0].dtype == want[0].dtype
            assert torch.equal(got[0], want[0])
            for a, r, t in zip(got[1:], want[1:], leaves):
                assert a.dtype == t.dtype and torch.equal(a, r.to(a.dtype))
    with torch.autocast(device, cast):
        assert ops.gelu_act8(x).dtype == torch.float32
        assert ops.gelu_act8(x.to(cast)).dtype == low


@pytest.mark.parametrize("device", DEVICES)
def test_autocast_around_forward_and_backward(device):
    """torch.func's transforms run the backward pass inside autocast, too."""
    w, b, x, y, up = population(gelu_linear_fn, 4, device)
    low = [t.bfloat16() for t in (w, b, x)]

    def step(w, b, x):
        return torch.func.grad(lambda *a: gelu_linear_fn(*a, None).float()
                               .sum(), argnums=(0, 1, 2))(w, b, x)
    run = torch.func.vmap(step)
    want = run(*low)
    with torch.autocast(device, torch.bfloat16):
        got = run(w, b, x)
    for a, r in zip(got, want):
        assert torch.equal(a, r.to(a.dtype))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dim", [256, 1000, 4096, 5001, 20001])
def test_norm_mean_is_the_nearest(device, dim):
    """Rows around 1000: the mean (512 to 1024) is off by its rounding to
    fp32, half of 2^-14, and not by that of the sum of a thousand such values.
    A tenth is left for the mean of the centred values; x - mean is exact and
    the rest is 64 U of h: deviation, product and output."""
    x = rand(64, dim, device=device, shift=1000.0)
    y = ops.layer_norm(x).double()
    xd = x.double()
    c = xd - xd.mean(-1, keepdim=True)
    r = 1 / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt()
    near(y, c * r, 1.1 * 2.0 ** -15 * r + 64 * U * (1 + (c * r).abs()))


# ------------------------------------------------------------------ memory

def _peak(f):
    """f's result, and the most that was allocated on the way beyond what was
    before."""
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = f()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_memory(dtype):
    """4096 x 50000 logits are 820 MB in fp32.  Forward: a maximum and a sum
    per row and 64 words or more.  Backward: the gradients returned, 256 MiB
    of logit gradient, 32-bit sums of dx, which may come in parts (at most
    16 here), the join of db, and 16 MiB for what the rows need."""
    rows, dim, vocab = 4096, 128, 50000
    x = rand(rows, dim, dtype=dtype, device="cuda").requires_grad_()
    w = rand(vocab, dim, dtype=dtype, device="cuda").requires_grad_()
    b = rand(vocab, dtype=dtype, device="cuda").requires_grad_()
    y = torch.randint(0, vocab, (rows,), device="cuda")
    loss, peak = _peak(lambda: ops.linear_cross_entropy(x, w, y, b))
    assert peak <= rows * (vocab // 64 + 1) * 8 + (1 << 20)
    grads, peak = _peak(lambda: torch.autograd.grad(loss, (x, w, b)))
    own = sum(g.numel() * g.element_size() for g in grads)
    parts = 16 * rows * dim * 4
    join = 4 * vocab * (rows // 32)
    assert peak <= own + (256 << 20) + parts + join + (16 << 20)


@gpu
def test_act8_memory():
    """Between forward and backward a chain linear, GELU, linear holds its
    three inputs in 129/128 bytes a value (a block's exponent is one byte)."""
    n, d = 1 << 15, 512
    w = [rand(d, d, device="cuda", seed=i).requires_grad_() for i in range(2)]
    x = rand(n, d, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = ops.linear_act8(ops.gelu_act8(ops.linear_act8(x, w[0])), w[1])
    kept = torch.cuda.memory_allocated() - before
    assert kept <= y.numel() * 4 + 3 * n * d * 129 // 128 + (1 << 20)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lo,hi", [(-1.0, 0.0), (0.0, 1.0)])
def test_gelu_rounding_near_zero(device, lo, hi):
    """fp32 values up to 1, where most activations lie.  Roundings are even
    within half a step, U / sqrt(3) each on average: of Phi, of the product,
    and of the part of Phi beyond (or short of) 1/2, which a negative x
    weighs by up to 2.1 and 0.7 on average: together 1.1 U or less."""
    g = torch.Generator().manual_seed(0)
    x = (torch.rand(300, 1024, generator=g) * (hi - lo) + lo).to(device)
    want = gelu64(x)
    err = ((ops.gelu_act8(x).double() - want) / want)[x != 0]
    assert err.square().mean().sqrt() <= 1.25 * U


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("fn", FNS)
@pytest.mark.parametrize("dims", [(None, None), (0, 0), (None, 0), (0, None)])
def test_checkpointed(device, fn, dims):
    """Recomputed in the backward pass, where each saved tensor may be asked
    for once."""
    from torch.utils.checkpoint import checkpoint
    w, b, x, y, up = population(fn, 3, device)
    if dims[0] is None:
        w = w[0]
    if dims[1] is None:
        b = b[0]
    leaves = [t.detach().clone().requires_grad_() for t in (w, b, x)]

    def run(w, b, x):
        return torch.func.vmap(fn, in_dims=dims + (0, 0))(w, b, x, y)
    want = torch.autograd.grad(run(*leaves), leaves, up)
    out = checkpoint(run, *leaves, use_reentrant=False)
    for g, r in zip(torch.autograd.grad(out, leaves, up), want):
        assert torch.equal(g, r)
    one = [t[0] if d == 0 else t for t, d in zip(leaves, dims + (0,))]

    def single(w, b, x):
        return fn(w, b, x, y[0])
    want = torch.autograd.grad(single(*one), leaves, up[0])
    out = checkpoint(single, *one, use_reentrant=False)
    for g, r in zip(torch.autograd.grad(out, leaves, up[0]), want):
        assert torch.equal(g, r)


# --------------------------------------------- logits far from zero, masks

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_loss_masked_by_the_lowest_value(device, dtype):
    """Words masked by the type's lowest value are switched off; where that
    leaves none, all are alike, their softmax 1 / vocab."""
    x, w, y, b = loss_inputs(20, 32, 300, dtype, device)
    low = torch.finfo(dtype).min
    off = b.clone()
    off[5:] = -math.inf
    masked = b.clone()
    masked[5:] = low
    y = torch.where(y == -100, y, y % 5)
    got, want = (
        (out, *torch.autograd.grad(out, leaves)) for out, leaves in (
            (ops.linear_cross_entropy(*leaves[:2], y, leaves[2]), leaves)
            for leaves in ([t.clone().requires_grad_() for t in (x, w, c)]
                           for c in (masked, off))))
    for a, r in zip(got, want):
        assert torch.equal(a, r)
    every = torch.full_like(b, low)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    rows = ops.linear_cross_entropy(*leaves, y, every, reduction="none")
    keep = y != -100
    # logarithm, sum of 300 ones and the last rounding
    near(rows, torch.where(keep, math.log(300.0), 0.0), 32 * U)
    dx, dw = torch.autograd.grad(rows.sum(), leaves)
    p = torch.full((20, 300), 1 / 300, dtype=torch.float64, device=device)
    p[torch.arange(20), y.clamp(min=0)] -= 1
    p = torch.where(keep[:, None], p, torch.zeros_like(p))
    # a term: its softmax's 32 U and its rounding; sums of 300 and 20 terms
    k = (HALF[dtype] * 1.01 if dtype == torch.bfloat16 else 0) + 350 * U
    for a, r, e in ((dx, p @ w.double(), p.abs() @ w.double().abs()),
                    (dw, p.t() @ x.double(), p.abs().t() @ x.double().abs())):
        near(a, r, HALF[dtype] * 1.01 * r.abs() + k * e)


@pytest.mark.parametrize("device", DEVICES)
def test_loss_common_offset_of_the_logits(device):
    """Whole-number logits around 2^20, exact in fp32: what they share costs
    neither the loss nor the softmax any bits.  A loss has 8 U for its
    exponentials and logarithm, U for each of 300 additions at most, and the
    rounding of at most 40; a softmax those and its exponent's, 40 U more."""
    g = torch.Generator().manual_seed(0)
    x = torch.ones(30, 16)
    w = torch.randint(-1, 2, (300, 16), generator=g).float()
    y = torch.randint(0, 300, (30,), generator=g)
    b = torch.full((300,), 2.0 ** 20)
    x, w, y, b = (t.to(device) for t in (x, w, y, b))
    want, lse, z = loss64(x, w, y, b, -100)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    rows = ops.linear_cross_entropy(*leaves[:2], y, leaves[2],
                                    reduction="none")
    near(rows, want, 350 * U)
    up = rand(30, device=device, seed=4)
    dx, dw, db, p = loss_grads64(x, w, y, b, -100, up.double())
    soft = torch.exp(z - lse[:, None]) * up.double().abs()[:, None]
    ep = 400 * U * soft + 8 * U * p.abs()
    got = torch.autograd.grad(rows, leaves, up)
    for a, r, e in zip(got, (dx, dw, db),
                       (ep @ w.double().abs() + 308 * U * (p.abs()
                                                           @ w.double().abs()),
                        ep.t() @ x.double() + 38 * U * (p.abs().t()
                                                        @ x.double()),
                        ep.sum(0) + 38 * U * p.abs().sum(0))):
        near(a, r, e + 2 * U * r.abs())


# ------------------------------------------------ offsets beyond 32 bits

@gpu
@pytest.mark.parametrize("fn", ["norm", "gelu", "linear", "loss"])
def test_more_than_2_31_values(fn):
    """The last rows of inputs of more than 2**31 values, forward and
    gradient, against the same rows alone."""
    dtype = torch.bfloat16
    dim, last = 1032, 40
    rows = (1 << 31) // dim + 100
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, dim, dtype=dtype, device="cuda")
    for lo in range(0, rows, 1 << 18):
        hi = min(rows, lo + (1 << 18))
        x[lo:hi] = torch.randn(hi - lo, dim, generator=g, device="cuda")
    w = rand(24, dim, dtype=dtype, device="cuda", scale=dim ** -0.5)
    b = rand(24, dtype=dtype, device="cuda")
    y = torch.randint(0, 24, (rows,), generator=g, device="cuda")
    f = {"norm": lambda x, y: ops.layer_norm(x, w[0], w[1]),
         "gelu": lambda x, y: ops.gelu_act8(x),
         "linear": lambda x, y: ops.linear_act8(x, w, b),
         "loss": lambda x, y: ops.linear_cross_entropy(
             x, w, y, b, reduction="none")}[fn]

    def run(x, y):
        x = x.requires_grad_()
        out = f(x, y)
        return out[-last:], torch.autograd.grad(
            out, x, torch.ones((), dtype=out.dtype,
                               device="cuda").expand_as(out))[0][-last:]
    want = run(x[-last:].clone(), y[-last:])
    got = run(x, y)
    for a, r in zip(got, want):
        close(a.float(), r.float(), torch.float32 if fn in ("norm", "gelu")
              else dtype)


@gpu
def test_parameter_gradients_of_more_than_2_31_values():
    """Per-client gradients of 24 heads, 2.4e9 values, in the last client."""
    C, v, d = 24, 50000, 2048
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(C, 40, d, generator=g, device="cuda").bfloat16()
    w = (torch.randn(v, d, generator=g, device="cuda")
         * d ** -0.5).bfloat16()
    y = torch.randint(0, v, (C, 40), generator=g, device="cuda")

    def step(x, y):
        return torch.func.grad(
            lambda x, w: ops.linear_cross_entropy(x, w, y),
            argnums=(0, 1))(x, w)
    got = torch.func.vmap(step)(x, y)
    assert got[1].numel() > 1 << 31
    for c in (0, C - 1):
        for a, r in zip(got, step(x[c], y[c])):
            close(a[c].float(), r.float(), torch.bfloat16)
