"""The matrix kernels of the token operators at every tile size.

Operands are chosen so that every partial sum is exact in 32 bits whatever its
order: few terms along the contraction, each with few bits.  The only rounding
left is the output's, so results have to equal the rounded 64-bit ones, and a
lost bit of an operand or a misplaced value shows.  fp32 operands need all
three of the bf16 parts that the kernels cut them into.
"""
import pytest
import torch

from blades_amd import ops

gpu = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
TERMS = 58               # along a contraction: sums stay below 2^7 or 2^8
BF16, F32 = torch.bfloat16, torch.float32


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


def signs(shape, g):
    return torch.randint(0, 2, shape, generator=g, device="cuda") * 2.0 - 1


def dense(shape, dtype, g):
    """Of size 1 to 2, either sign: 18 bits in fp32, 8 in bf16."""
    bits = 17 if dtype == F32 else 7
    j = torch.randint(0, 1 << bits, shape, generator=g, device="cuda")
    return signs(shape, g) * (1 + j * 2.0 ** -bits)


def middling(shape, dtype, g):
    """Of size 1 to 2 with the two upper parts alone: 9 bits."""
    bits = 8 if dtype == F32 else 7
    j = torch.randint(0, 1 << bits, shape, generator=g, device="cuda")
    return signs(shape, g) * (1 + (j | 1) * 2.0 ** -bits)


def sparse(values, axis, g):
    """``values`` with all but TERMS entries zero along ``axis``, the last one
    among those that stay."""
    n = values.shape[axis]
    if n <= TERMS:
        return values
    v = values.movedim(axis, 0)
    at = torch.randint(0, n, (TERMS, *v.shape[1:]), generator=g,
                       device="cuda")
    at[0] = n - 1
    mask = torch.zeros(v.shape, device="cuda").scatter_(0, at, 1.0)
    return (v * mask).movedim(0, axis)


ROLES = ["dense_by_sign", "sign_by_dense", "parts_by_parts"]


def pair(role, a_shape, a_axis, b_shape, b_axis, dtype, seed=0):
    """Two operands contracted along a_axis and b_axis."""
    g = gen(seed)
    if role == "dense_by_sign":
        a, b = dense(a_shape, dtype, g), sparse(signs(b_shape, g), b_axis, g)
    elif role == "sign_by_dense":
        a, b = sparse(signs(a_shape, g), a_axis, g), dense(b_shape, dtype, g)
    else:
        a = middling(a_shape, dtype, g)
        b = sparse(middling(b_shape, dtype, g), b_axis, g)
    a, b = a.float(), b.float()
    for t in (a, b):
        assert torch.equal(t, t.to(dtype).float())
    return a.to(dtype), b.to(dtype)


def exactly(got, want, dtype):
    """``want`` in 64 bits, exact in fp32, rounded once."""
    assert torch.equal(want, want.float().double())
    assert got.dtype == dtype
    assert torch.equal(got, want.float().to(dtype))


def over_clients(clients, f, *args):
    return torch.func.vmap(f)(*args) if clients else f(*args)


def tiled(want, clients, m, n, k, deep, dtype, act8=False):
    from blades_amd import _hip_ops
    tile, parts = _hip_ops._product_tiling(max(clients, 1), m, n, k, deep,
                                           dtype == F32, act8)
    assert (tile, parts > 1) == want


# clients (0: one alone), rows, in, out -> (tile rows, contraction in parts)
FORWARD = [
    (BF16, (0, 72, 75, 65), (64, False)), (BF16, (0, 65, 1441, 71), (64, True)),
    (BF16, (3, 1875, 66, 513), (128, False)),
    (BF16, (3, 65, 3888, 3225), (128, True)),
    (BF16, (0, 4509, 229, 2727), (256, False)),
    (BF16, (0, 8191, 515, 4093), (256, False)),
    (F32, (0, 65, 67, 69), (64, False)), (F32, (0, 85, 535, 75), (64, True)),
    (F32, (3, 4255, 75, 197), (128, False)),
    (F32, (2, 73, 1039, 4591), (128, True)),
    (F32, (0, 6855, 179, 1853), (256, False)),
    (F32, (0, 8191, 515, 4093), (256, False)),
    (F32, (0, 6291, 1949, 487), (256, True)),
]
GRAD_INPUT = [
    (BF16, (0, 72, 75, 65), (64, False)), (BF16, (0, 67, 89, 1809), (64, True)),
    (BF16, (0, 643, 4545, 65), (128, False)),
    (BF16, (3, 3093, 65, 4143), (128, True)),
    (BF16, (0, 3379, 3837, 213), (256, False)),
    (BF16, (0, 4099, 1029, 8195), (256, True)),
    (F32, (0, 65, 67, 69), (64, False)), (F32, (0, 79, 66, 513), (64, True)),
    (F32, (2, 3623, 385, 67), (128, False)),
    (F32, (2, 65, 1755, 2483), (128, True)),
    (F32, (0, 3966, 3139, 185), (256, False)),
    (F32, (3, 4311, 209, 1829), (256, True)),
]
GRAD_WEIGHT = [
    (BF16, (0, 72, 75, 65), (64, False)), (BF16, (0, 1421, 71, 73), (64, True)),
    (BF16, (3, 77, 199, 4133), (128, False)),
    (BF16, (2, 4967, 4377, 79), (128, True)),
    (BF16, (3, 213, 5485, 693), (256, False)),
    (BF16, (2, 7981, 453, 4114), (256, True)),
    (F32, (0, 65, 67, 69), (64, False)), (F32, (0, 877, 71, 73), (64, True)),
    (F32, (2, 65, 425, 3533), (128, False)),
    (F32, (2, 1587, 69, 4609), (128, True)),
    (F32, (0, 179, 2955, 4341), (256, False)),
    (F32, (0, 7093, 3521, 441), (256, True)),
]


def lead(clients):
    return (clients,) if clients else ()


def named(cases):
    return [pytest.param(*c, id=f"{str(c[0])[6:]}-{c[1]}-{c[2][0]}")
            for c in cases]


@gpu
@pytest.mark.parametrize("role", ROLES)
@pytest.mark.parametrize("dtype,size,tile", named(FORWARD))
def test_forward(dtype, size, tile, role):
    c, rows, n, m = size
    tiled(tile, c, rows, m, n, True, dtype)
    x, w = pair(role, lead(c) + (rows, n), -1, lead(c) + (m, n), -1, dtype)
    b = torch.randint(-256, 257, lead(c) + (m,), generator=gen(1),
                      device="cuda").mul(2.0 ** -7).to(dtype)
    with torch.no_grad():
        y = over_clients(c, ops.linear_act8, x, w, b)
    want = x.double() @ w.double().transpose(-1, -2).contiguous()
    exactly(y, want + b.double().unsqueeze(-2), dtype)


@gpu
@pytest.mark.parametrize("role", ROLES)
@pytest.mark.parametrize("dtype,size,tile", named(GRAD_INPUT))
def test_grad_input(dtype, size, tile, role):
    c, rows, n, m = size
    tiled(tile, c, rows, n, m, True, dtype)
    dy, w = pair(role, lead(c) + (rows, m), -1, lead(c) + (m, n), -2, dtype)

    def f(w, dy):
        x = torch.zeros(rows, n, device="cuda", dtype=dtype)
        return torch.func.vjp(lambda x: ops.linear_act8(x, w), x)[1](dy)[0]
    exactly(over_clients(c, f, w, dy), dy.double() @ w.double(), dtype)


@gpu
@pytest.mark.parametrize("role", ROLES)
@pytest.mark.parametrize("dtype,size,tile", named(GRAD_WEIGHT))
def test_grad_weight_from_8_bits(dtype, size, tile, role):
    c, rows, n, m = size
    tiled(tile, c, m, n, rows, True, dtype, act8=True)
    g = gen()
    x_shape, dy_shape = lead(c) + (rows, n), lead(c) + (rows, m)
    if role == "dense_by_sign":
        # 1 is 64 * 2^-6 in a block of signs and zeros
        dy, x = dense(dy_shape, dtype, g), sparse(signs(x_shape, g), -2, g)
    else:
        # whole numbers, 127 in every block: held as they are
        x = torch.randint(-127, 128, x_shape, generator=g,
                          device="cuda").float()
        x[..., ::128] = 127
        dy = signs(dy_shape, g) if role == "sign_by_dense" \
            else middling(dy_shape, dtype, g)
        dy = sparse(dy, -2, g)
    dy, x = dy.to(dtype), x.to(dtype)

    def f(x, dy):
        w = torch.zeros(m, n, device="cuda", dtype=dtype)
        return torch.func.vjp(lambda w: ops.linear_act8(x, w), w)[1](dy)[0]
    want = dy.double().transpose(-1, -2).contiguous() @ x.double()
    exactly(over_clients(c, f, x, dy), want, dtype)


# clients, rows, dim, vocab -> tiles of (logits, dx, dw), which of them in parts
LOSS = [
    (BF16, (0, 72, 69, 131), ((64, False), (64, False), (64, False))),
    (BF16, (0, 1403, 75, 157), ((64, False), (64, False), (64, True))),
    (BF16, (0, 65, 83, 1425), ((64, False), (64, True), (64, False))),
    (BF16, (3, 71, 65, 8443), ((128, False), None, (128, False))),
    (BF16, (0, 4125, 69, 9307), (None, None, (128, True))),
    (BF16, (0, 221, 785, 14743), (None, None, (256, False))),
    (BF16, (2, 7285, 203, 6319), (None, None, (256, True))),
    (BF16, (3, 2733, 324, 139), (None, (128, False), None)),
    (BF16, (3, 2747, 71, 4681), (None, (128, True), None)),
    (BF16, (3, 6071, 763, 217), (None, (256, False), None)),
    (BF16, (3, 4253, 199, 6893), (None, (256, True), None)),
    (BF16, (3, 1537, 217, 2457), ((256, False), None, None)),
    (BF16, (0, 2043, 517, 8183), ((256, False), None, None)),
    (F32, (0, 73, 70, 147), ((64, False), (64, False), (64, False))),
    (F32, (0, 537, 77, 143), ((64, False), (64, False), (64, True))),
    (F32, (0, 65, 69, 627), ((64, False), (64, True), (64, False))),
    (F32, (3, 67, 69, 8657), ((128, False), None, (128, False))),
    (F32, (2, 881, 67, 4143), (None, None, (128, True))),
    (F32, (3, 175, 219, 17523), (None, None, (256, False))),
    (F32, (0, 1735, 195, 13021), (None, None, (256, True))),
    (F32, (3, 2433, 409, 131), (None, (128, False), None)),
    (F32, (2, 4113, 69, 857), (None, (128, True), None)),
    (F32, (3, 4817, 893, 179), (None, (256, False), None)),
    (F32, (0, 6997, 137, 6029), (None, (256, True), None)),
    (F32, (3, 199, 211, 16437), ((256, False), None, None)),
    (F32, (0, 2043, 517, 8183), ((256, False), None, None)),
]


def loss_cases():
    return [pytest.param(*c, id=f"{str(c[0])[6:]}-{c[1]}") for c in LOSS]


def loss_tiled(size, tiles, dtype):
    c, rows, dim, vocab = size
    for t, (m, n, k, deep) in zip(tiles, ((vocab, rows, dim, False),
                                          (rows, dim, vocab, True),
                                          (vocab, dim, rows, True))):
        if t:
            tiled(t, c, m, n, k, deep, dtype)


def test_every_tile_is_reached():
    """Each product of each type at each tile size; logits are never cut."""
    for dtype in (BF16, F32):
        every = {(t, p) for t in (64, 128, 256) for p in (False, True)}
        for cases in (FORWARD, GRAD_INPUT, GRAD_WEIGHT):
            have = {t for d, _, t in cases if d == dtype}
            # no bf16 forward product takes large tiles in parts
            assert every - have <= ({(256, True)} if cases is FORWARD
                                    and dtype == BF16 else set())
        of = [{t[i] for d, _, t in LOSS if d == dtype} for i in range(3)]
        assert {(64, False), (128, False), (256, False)} <= of[0]
        assert every <= of[1] and every <= of[2]


@gpu
@pytest.mark.parametrize("role", ROLES)
@pytest.mark.parametrize("dtype,size,tiles", loss_cases())
def test_loss_gradients_exactly(dtype, size, tiles, role):
    """All words but one are switched off, so that a row's softmax is 1 there
    and 0 elsewhere: with its upstream gradient u the logits' gradient is u at
    that word and -u at the target, and the products that follow are exact."""
    c, rows, dim, vocab = size
    loss_tiled(size, tiles, dtype)
    g = gen()
    live = vocab - 2
    b = torch.full((vocab,), -torch.inf, device="cuda", dtype=dtype)
    b[live] = 0
    y = torch.randint(0, vocab, lead(c) + (rows,), generator=g, device="cuda")
    y[..., 0] = vocab - 1
    y[..., 1] = -100
    y[..., rows - 1] = live
    xs, ws, us = lead(c) + (rows, dim), (vocab, dim), lead(c) + (rows,)
    if role == "dense_by_sign":
        u = dense(us, dtype, g)
        x, w = sparse(signs(xs, g), -2, g), signs(ws, g)
    elif role == "sign_by_dense":
        u = sparse(signs(us, g), -1, g)
        x, w = dense(xs, dtype, g), dense(ws, dtype, g)
    else:
        u = sparse(middling(us, dtype, g), -1, g)
        x, w = middling(xs, dtype, g), middling(ws, dtype, g)
    # the largest is a power of two: the rows' shares of it are exact
    u = (u / 2).float()
    u[..., rows - 1] = 1
    x, w = x.to(dtype), w.to(dtype)

    def f(x, y, u):
        pull = torch.func.vjp(
            lambda x, w, b: ops.linear_cross_entropy(
                x, w, y, b, reduction="none"), x, w, b)[1]
        return pull(u)
    dx, dw, db = over_clients(c, f, x, y, u)
    p = torch.zeros(lead(c) + (rows, vocab), device="cuda",
                    dtype=torch.float64)
    ud = (u * (y != -100)).double()
    p[..., live] = ud
    p.scatter_add_(-1, y.clamp(min=0).unsqueeze(-1), -ud.unsqueeze(-1))
    exactly(dx, p @ w.double(), dtype)
    pt = p.transpose(-1, -2).contiguous()
    exactly(dw, pt @ x.double(), dtype)
    if role != "dense_by_sign":
        exactly(db, p.sum(-2), dtype)


@gpu
@pytest.mark.parametrize("dtype,size,tiles", loss_cases())
def test_loss_of_exact_logits(dtype, size, tiles):
    """Logits without an error of their own (TERMS values a row), so that a
    row's loss has only its exponentials', their sum's and the logarithm's:
    16 U for a term (its exponent, up to 8, times U, twice, and the
    instruction's), 24 U for the order of some hundred additions whose errors
    have no common sign, 4 |lse| U for the logarithm and the last
    subtraction."""
    c, rows, dim, vocab = size
    loss_tiled(size, tiles, dtype)
    g = gen()
    x = sparse(signs(lead(c) + (rows, dim), g), -1, g).to(dtype)
    w = (dense((vocab, dim), dtype, g) / 32).to(dtype)
    b = (torch.randint(-128, 129, (vocab,), generator=g, device="cuda")
         * 2.0 ** -7).to(dtype)
    y = torch.randint(0, vocab, lead(c) + (rows,), generator=g, device="cuda")
    y[..., 0] = vocab - 1
    y[..., 1] = -100

    def rows_of(x, y):
        return ops.linear_cross_entropy(x, w, y, b, reduction="none")
    got = over_clients(c, rows_of, x, y).double()
    z = x.double() @ w.double().t().contiguous() + b.double()
    lse = torch.logsumexp(z, -1)
    keep = y != -100
    want = lse - z.gather(-1, y.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    want = torch.where(keep, want, torch.zeros_like(want))
    assert ((got - want).abs() <= U * (40 + 4 * lse.abs())).all()

    # mean over the rows that count, and its gradients: relative errors of
    # whole tensors.  fp32: a term's 40 + 4 |lse| U as above, no more than 128;
    # bf16: two roundings (logit gradient, output), each uniform within half a
    # step and so HALF / sqrt(3) of the values' size at most, 0.82 HALF.
    def mean(x, w, b, y):
        return ops.linear_cross_entropy(x, w, y, b)
    got = over_clients(
        c, lambda x, y: torch.func.grad(mean, argnums=(0, 1, 2))(x, w, b, y),
        x, y)
    p = torch.exp(z - lse.unsqueeze(-1))
    p.scatter_add_(-1, y.clamp(min=0).unsqueeze(-1),
                   -torch.ones_like(lse).unsqueeze(-1))
    p *= (keep / keep.sum(-1, keepdim=True)).unsqueeze(-1)
    want = (p @ w.double(), p.transpose(-1, -2).contiguous() @ x.double(),
            p.sum(-2))
    for a, r in zip(got, want):
        assert a.dtype == dtype and a.shape == r.shape
        assert (a.double() - r).norm() <= r.norm() * (
            128 * U if dtype == F32 else 0.95 * HALF[dtype])
