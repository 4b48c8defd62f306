"""Pure-PyTorch reference implementations of every aggregation/attack op.

These are (a) the CPU execution path, and (b) the fp32 numerics reference the
HIP kernels are tested against (SURVEY.md §2.4 K1-K18 inventory).  Each
function documents the reference site whose math it reproduces.

All ops take the stacked update matrix ``U ∈ R^{K×d}`` (fp32, K clients,
d model dims) unless noted.
"""
from __future__ import annotations

import functools
from typing import Optional, Tuple

import torch

Tensor = torch.Tensor


# ---------------------------------------------------------------- column ops

def col_mean(U: Tensor) -> Tensor:
    """K1 — column mean (reference: aggregators/mean.py:72)."""
    return U.mean(dim=0)


def col_median(U: Tensor) -> Tensor:
    """K2 — coordinate-wise median, averaging the two middle elements for
    even K (reference: aggregators/median.py:23-25 computes
    ``(median(U) - median(-U)) / 2`` to the same effect)."""
    values_upper, _ = U.median(dim=0)
    values_lower, _ = (-U).median(dim=0)
    return (values_upper - values_lower) / 2


def trimmed_mean(U: Tensor, b: int) -> Tensor:
    """K3 — per coordinate: drop the b largest and b smallest, mean the rest
    (reference: aggregators/trimmedmean.py:38-41).

    Accumulated in fp64: the reference's fp32 ``sum − topk + neg_topk`` form
    cancels catastrophically when Byzantine rows contain huge values (a 1e8
    outlier swallows every honest value's bits before being subtracted —
    caught by tests/test_properties.py::test_single_outlier_bounded_influence;
    the HIP kernel sums in fp64 for the same reason).
    """
    K = U.shape[0]
    if K - 2 * b <= 0:
        raise ValueError(f"trimmed_mean needs K > 2b (K={K}, b={b})")
    if b == 0:
        return U.mean(dim=0)
    Ud = U.double()
    largest, _ = torch.topk(Ud, b, 0)
    neg_smallest, _ = torch.topk(-Ud, b, 0)
    out = (Ud.sum(0) - largest.sum(0) + neg_smallest.sum(0)) / (K - 2 * b)
    return out.to(U.dtype)


def col_var(U: Tensor, unbiased: bool = False) -> Tensor:
    """K17 — column variance diagnostics (reference: simulator.py:309-313)."""
    return U.var(dim=0, unbiased=unbiased)


def weighted_col_sum(U: Tensor, w: Tensor) -> Tensor:
    """Σ_k w_k · U_k — the GeoMed/FLTrust accumulation primitive."""
    return (w.to(U.dtype).unsqueeze(1) * U).sum(dim=0)


def masked_col_mean(U: Tensor, mask: Tensor) -> Tensor:
    """K11 — column mean over rows where ``mask`` is True (IPM honest mean,
    reference: attackers/ipmclient.py:10-16)."""
    m = mask.to(U.dtype)
    return (U * m.unsqueeze(1)).sum(dim=0) / m.sum().clamp_min(1)


def masked_col_mean_std(U: Tensor, mask: Tensor,
                        unbiased: bool = True) -> Tuple[Tensor, Tensor]:
    """K10 — column mean and std over masked (honest) rows
    (reference: attackers/alieclient.py:32-35 uses torch.mean/torch.std,
    i.e. Bessel-corrected std)."""
    rows = U[mask]
    mu = rows.mean(dim=0)
    std = rows.std(dim=0, unbiased=unbiased)
    return mu, std


# ------------------------------------------------------------------- row ops

def row_sq_norms(U: Tensor) -> Tensor:
    """‖u_i‖² per row."""
    return (U * U).sum(dim=1)


def row_norms(U: Tensor) -> Tensor:
    return row_sq_norms(U).sqrt()


def row_diff_norms(U: Tensor, z: Tensor) -> Tensor:
    """K6 — ‖z − u_i‖ for every row (Weiszfeld distance pass,
    reference: aggregators/geomed.py:71-75)."""
    return (U - z.unsqueeze(0)).norm(dim=1)


def row_dots(U: Tensor, v: Tensor) -> Tensor:
    """u_i · v per row (FLTrust cosine numerator)."""
    return U @ v


def pairwise_sq_dists(U: Tensor) -> Tensor:
    """K4 — K×K squared-distance matrix.

    The reference loops K(K-1)/2 norm calls (aggregators/krum.py:73-90);
    here ‖u_i−u_j‖² = ‖u_i‖² + ‖u_j‖² − 2·u_i·u_j via one Gram matmul (the
    HIP path runs this on MFMA).  Clamped at 0 against cancellation.
    """
    G = U @ U.t()
    sq = G.diagonal()
    D = sq.unsqueeze(0) + sq.unsqueeze(1) - 2 * G
    D.fill_diagonal_(0)
    return D.clamp_min_(0)


def cos_sim_gram(U: Tensor, eps: float = 1e-8) -> Tensor:
    """K8 — K×K cosine-similarity matrix (reference: aggregators/
    clustering.py:28-33 computes it with a scipy double loop)."""
    norms = row_norms(U).clamp_min(eps)
    Un = U / norms.unsqueeze(1)
    G = Un @ Un.t()
    return G.clamp_(-1.0, 1.0)


# ----------------------------------------------------------- fused/iterated

def krum_scores(sqdists: Tensor, f: int) -> Tensor:
    """K5 — per-row sum of the n−f−2 smallest squared distances to OTHER
    rows (reference: aggregators/krum.py:9-25)."""
    n = sqdists.shape[0]
    k = n - f - 2
    if k < 1:
        raise ValueError(f"krum needs n - f - 2 >= 1 (n={n}, f={f})")
    # mask the diagonal out by setting it to +inf, then take k smallest
    D = sqdists.clone()
    D.fill_diagonal_(float("inf"))
    smallest, _ = torch.topk(D, k, dim=1, largest=False)
    return smallest.sum(dim=1)


def clip_to_norm(v: Tensor, tau: float) -> Tensor:
    """Scale v to norm ≤ tau (reference: centeredclipping.py:30-33)."""
    v_norm = v.norm()
    scale = torch.clamp(tau / v_norm.clamp_min(1e-12), max=1.0)
    return v * scale


def centered_clip_iter(U: Tensor, v: Tensor, tau: float) -> Tensor:
    """K7 — one centered-clipping iteration:
    v' = v + mean_k(clip(u_k − v, tau)) (reference: centeredclipping.py:40-44).
    """
    diff = U - v.unsqueeze(0)
    norms = diff.norm(dim=1).clamp_min(1e-12)
    scale = torch.clamp(tau / norms, max=1.0)
    return v + (diff * scale.unsqueeze(1)).mean(dim=0)


def row_clip_to_norm_(U: Tensor, max_norms: Tensor) -> Tensor:
    """Clip each row of U to its per-row threshold in place
    (Clippedclustering's historical-median clip, reference:
    clippedclustering.py:37-46 via torch_utils.clip_tensor_norm_)."""
    norms = U.norm(dim=1).clamp_min(1e-12)
    scale = torch.clamp(max_norms / norms, max=1.0)
    U.mul_(scale.unsqueeze(1))
    return U


# ----------------------------------------------------------------- RNG fill

def philox_normal(shape, mean: float, std: float, seed: int,
                  device=None, dtype=torch.float32) -> Tensor:
    """K12 — deterministic normal fill from a dedicated generator stream.

    Counter-based keying happens in the caller via
    :func:`blades_amd.utils.client_philox_seed`; this draws from a private
    torch.Generator so the global RNG stream is untouched (the reference
    instead relied on driver-side RNG save/restore, simulator.py:153-165).
    """
    dev = torch.device(device) if device is not None else torch.device("cpu")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return torch.empty(shape, device=dev, dtype=dtype).normal_(mean, std, generator=g)


# ----------------------------------------------------------- server-side ops

def flat_sgd_step_(theta: Tensor, delta: Tensor, lr: float) -> Tensor:
    """K16 — fused flat-vector pseudo-gradient SGD: θ ← θ + lr·Δ.

    Matches the reference server semantics: ``p.grad = -update_slice`` then
    ``SGD(lr).step()`` (reference: server.py:54-75), i.e. θ ← θ − lr·(−Δ).
    """
    return theta.add_(delta, alpha=lr)


def sanitize_(U: Tensor) -> Tensor:
    """K18 — nan_to_num on update read (reference: client.py:198)."""
    return torch.nan_to_num_(U)


# ------------------------------------------------- token-model operators
# Plain forms of csrc/layer_norm.hip, act8.hip and token_gemm.hip with the
# same interface: [groups, rows, ...] inputs, parameters shared or with a
# leading group axis, 32-bit arithmetic rounded once to the inputs' type.

_ACT8_BLOCK = 128


def _per_row(p: Optional[Tensor]) -> Optional[Tensor]:
    """A parameter [dim] or [groups, dim] against [groups, rows, dim]."""
    if p is None:
        return None
    return p.float() if p.dim() == 1 else p.float().unsqueeze(1)


def norm_forward(x: Tensor, w: Optional[Tensor], b: Optional[Tensor],
                 eps: float):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    c = xf - mean
    # the centred values' own mean: what the first sum rounded away
    off = c.mean(-1, keepdim=True)
    mean, c = mean + off, c - off
    rstd = 1.0 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    y = c * rstd
    if w is not None:
        y = y * _per_row(w)
    if b is not None:
        y = y + _per_row(b)
    return y.to(x.dtype), mean.squeeze(-1), rstd.squeeze(-1)


def norm_backward(dy: Tensor, x: Tensor, mean: Tensor, rstd: Tensor,
                  w: Optional[Tensor], params: bool):
    h = (x.float() - mean.unsqueeze(-1)) * rstd.unsqueeze(-1)
    dyf = dy.float()
    g = dyf if w is None else dyf * _per_row(w)
    dx = rstd.unsqueeze(-1) * (g - g.mean(-1, keepdim=True)
                               - h * (g * h).mean(-1, keepdim=True))
    if not params:
        empty = x.new_empty(0, x.shape[-1])
        return dx.to(x.dtype), empty, empty.clone()
    return (dx.to(x.dtype), (dyf * h).sum(1).to(x.dtype),
            dyf.sum(1).to(x.dtype))


def colsum(x: Tensor) -> Tensor:
    return x.float().sum(1).to(x.dtype)


def act8_pack(x: Tensor):
    """int8 values and biased exponents (255: a block that is not finite)."""
    n = x.shape[-1]
    pad = (-n) % _ACT8_BLOCK
    xf = torch.nn.functional.pad(x.float(), (0, pad))
    nb = (n + pad) // _ACT8_BLOCK
    blocks = xf.reshape(*x.shape[:-1], nb, _ACT8_BLOCK)
    top = blocks.abs().amax(-1, keepdim=True)
    finite = torch.isfinite(top)
    m, k = torch.frexp(torch.where(finite, top, torch.ones_like(top)))
    e = (k - 7 + (m > 127.0 / 128.0).int()).clamp(min=-126)
    e = torch.where(top == 0, torch.full_like(e, -126), e)
    q = torch.round(torch.ldexp(blocks, -e))
    # 64 units of the largest exponent would be 2^128, beyond float32
    most = torch.where(e == 122, 63.0, 127.0)
    q = torch.minimum(torch.maximum(q, -most), most)
    q = torch.where(finite, q, torch.zeros_like(q)).to(torch.int8)
    code = torch.where(finite, e + 127, torch.full_like(e, 255))
    return (q.reshape(*x.shape[:-1], n + pad)[..., :n].contiguous(),
            code.squeeze(-1).to(torch.uint8))


def act8_unpack(q: Tensor, e: Tensor) -> Tensor:
    """The float32 values that 8-bit storage holds."""
    n = q.shape[-1]
    code = e.int().unsqueeze(-1)
    unit = torch.ldexp(torch.ones_like(code, dtype=torch.float32),
                       code.clamp(max=254) - 127)
    unit = torch.where(code == 255, torch.full_like(unit, float("nan")), unit)
    unit = unit.expand(*unit.shape[:-1], _ACT8_BLOCK)
    unit = unit.reshape(*e.shape[:-1], e.shape[-1] * _ACT8_BLOCK)
    return q.float() * unit[..., :n]


def gelu_forward(x: Tensor, keep: bool):
    xf = x.float()
    y = (0.5 * xf * (1.0 + torch.erf(xf * 0.5 ** 0.5))).to(x.dtype)
    if not keep:
        return (y, x.new_empty(0, dtype=torch.int8),
                x.new_empty(0, dtype=torch.uint8))
    return (y, *act8_pack(x))


def gelu_backward(dy: Tensor, q: Tensor, e: Tensor) -> Tensor:
    v = act8_unpack(q, e)
    slope = (0.5 * (1.0 + torch.erf(v * 0.5 ** 0.5))
             + v * torch.exp(-0.5 * v * v) * 0.3989422804014327)
    return (dy.float() * slope).to(dy.dtype)


def _full_precision(fn):
    """Products in the types given to them, also under autocast."""
    @functools.wraps(fn)
    def run(x: Tensor, *args, **kw):
        with torch.autocast(x.device.type, enabled=False):
            return fn(x, *args, **kw)
    return run


@_full_precision
def linear_forward(x: Tensor, w: Tensor, b: Optional[Tensor]) -> Tensor:
    y = torch.matmul(x.float(), w.float().transpose(-1, -2).contiguous())
    if b is not None:
        y = y + _per_row(b)
    return y.to(x.dtype)


@_full_precision
def linear_grad_input(dy: Tensor, w: Tensor) -> Tensor:
    return torch.matmul(dy.float(), w.float()).to(dy.dtype)


@_full_precision
def linear_grad_weight(dy: Tensor, q: Tensor, e: Tensor) -> Tensor:
    dyt = dy.float().transpose(1, 2).contiguous()
    return torch.matmul(dyt, act8_unpack(q, e)).to(dy.dtype)


def _logits(x: Tensor, w: Tensor, bias: Optional[Tensor]) -> Tensor:
    z = torch.matmul(x.float(), w.float().transpose(-1, -2).contiguous())
    return z if bias is None else z + _per_row(bias)


@_full_precision
def loss_forward(x: Tensor, w: Tensor, target: Tensor,
                 bias: Optional[Tensor], ignore: int, reduction: int):
    """reduction 0: rows, 1: sum, 2: mean.  The second output is [..., 2]: a
    row's largest logit and the logarithm of its sum relative to that, whose
    sum would round the logarithm away where logits are large."""
    vocab = w.shape[-2]
    z = _logits(x, w, bias)
    top = z.amax(-1)
    log = torch.log(torch.exp(z - top.unsqueeze(-1)).sum(-1))
    counted = target != ignore
    bad = counted & ((target < 0) | (target >= vocab))
    top = top.masked_fill(bad, float("nan"))
    lse = torch.stack([top, log], -1)
    at = target.clamp(0, vocab - 1).unsqueeze(-1)
    rows = torch.where(counted, (top - z.gather(-1, at).squeeze(-1)) + log,
                       torch.zeros_like(top))
    count = counted.sum(-1).float()
    if reduction == 0:
        return rows, lse, count
    total = rows.double().sum(-1)
    if reduction == 2:
        total = total / count
    return total.float(), lse, count


@_full_precision
def loss_backward(grad: Tensor, x: Tensor, w: Tensor, target: Tensor,
                  bias: Optional[Tensor], lse: Tensor, count: Tensor,
                  ignore: int, reduction: int, want_x: bool, want_w: bool,
                  want_b: bool):
    z = _logits(x, w, bias)
    p = torch.exp((z - lse[..., :1]) - lse[..., 1:])
    counted = (target != ignore).unsqueeze(-1)
    at = target.clamp(0, w.shape[-2] - 1).unsqueeze(-1)
    p.scatter_add_(-1, at, torch.full_like(at, -1.0, dtype=p.dtype))
    if reduction == 2:
        grad = grad / count.unsqueeze(-1)
    p = torch.where(counted, p * grad.unsqueeze(-1), torch.zeros_like(p))
    none = x.new_empty(0)
    dx = torch.matmul(p, w.float()).to(x.dtype) if want_x else none
    dw = (torch.matmul(p.transpose(1, 2).contiguous(), x.float()).to(x.dtype)
          if want_w else none)
    db = p.sum(1).to(x.dtype) if want_b else none
    return dx, dw, db
