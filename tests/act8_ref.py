"""The definitions of the 8-bit activation path in 64 bits, on the CPU, and the tolerances that follow
from the kernels' roundings."""
import torch

U32 = 2.0 ** -24          # half a step of fp32


def half(dt):
    """Half a step of a 16-bit type, relative to the value."""
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def codes(v):
    """Rows in 64 bits -> (q, scale): q = rint(127 v / max|v|) with ties to even, found with whole numbers
    (254 |v| against the odd multiples of max), so that no rounding takes part."""
    v = v.double()
    m = v.abs().amax(1, keepdim=True) if v.shape[1] else torch.zeros(v.shape[0], 1, dtype=torch.float64)
    a = v.abs()
    k = torch.floor(a * 127.0 / torch.where(m > 0, m, torch.ones_like(m)))
    k = torch.where(k * m > 127.0 * a, k - 1, k)                  # the quotient's own rounding
    k = torch.where((k + 1) * m <= 127.0 * a, k + 1, k)
    up, border = 254.0 * a, (2 * k + 1) * m
    k = k + ((up > border) | ((up == border) & (k % 2 == 1))).double()
    k = torch.where(m > 0, k, torch.zeros_like(k))
    return torch.sign(v) * k, (m / 127.0)[:, 0]


def norm(x, residual, gain, eps):
    dt = x.dtype
    r = x.double() if residual is None else (x.double() + residual.double()).to(dt).double()
    rstd = 1.0 / torch.sqrt(r.square().mean(1, keepdim=True) + eps)
    p = r * gain.double()
    q, s = codes(p)
    return r.to(dt), p * rstd, q, s * rstd[:, 0]


def linear(q, scale, w, w_scale, bias):
    """(y unrounded, bound on |kernel's fp32 value - y|): the sum is exact; its conversion, the two scale
    products and the bias's addition round once each."""
    prod = (q.double() @ w.double().t()) * (scale.double()[:, None] * w_scale.double()[None, :])
    y = prod if bias is None else prod + bias.double()
    slack = 4 * U32 * prod.abs() * (1 + U32) + (0 if bias is None else 2 * U32 * (prod.abs() + bias.double().abs()))
    return y, slack


def assert_close16(got, want, dt, slack, what=""):
    """got (16-bit) is want (64-bit, up to slack) rounded once."""
    got, want = got.double().cpu(), want.cpu()
    tol = slack + half(dt) * (want.abs() + slack) + tiny(dt)
    bad = (got - want).abs() > tol
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float(((got - want).abs() / tol.clamp_min(1e-300)).max()):.3g} x the bound")


# ---- the layer, in the kernels' own fp32 operations (bit for bit) -------------------------------------

def _fma(a, b, c):
    """fp32 fused multiply-add: the product of two fp32 values is exact in fp64."""
    return (a.double() * b.double() + c.double()).float()


def expf(x):
    """The kernels' exp from IEEE operations (Cody-Waite reduction by ln 2, Cephes' degree-5 polynomial)."""
    f = lambda v: torch.tensor(v, dtype=torch.float32)
    x = x.clamp(-87.0, 89.0)
    n = torch.round(x * f(1.44269504088896341))
    r = _fma(n, f(-0.693359375), x)
    r = _fma(n, f(2.12194440e-4), r)
    p = f(1.9875691500e-4).expand_as(r)
    for c in (1.3981999507e-3, 8.3334519073e-3, 4.1665795894e-2, 1.6666665459e-1, 5.0000001201e-1):
        p = _fma(p, r, f(c).expand_as(r))
    y = _fma(r * r, p, r) + 1.0
    return (y.double() * torch.exp2(n.double())).float()


def product(q, scale, w, w_scale):
    """fp32(sum) * (scale * w_scale): the sum is exact, each operation rounds to fp32."""
    acc = (q.double() @ w.double().t()).to(torch.int32).float()
    return acc * (scale.float()[:, None] * w_scale.float()[None, :])


def quantise(x16):
    """A row with an infinity or a NaN has codes of 0 and the scale NaN."""
    finite = x16.float().isfinite().all(1)
    q, _ = codes(torch.where(finite[:, None], x16, torch.zeros_like(x16)))
    return q, torch.where(finite, x16.float().abs().amax(1) / 127.0, torch.full_like(finite, float("nan"), dtype=torch.float32))


def expert(q, scale, ew, dt):
    """8-bit rows through one expert (ek_hip.ExpertWeight) -> 16-bit rows."""
    u = product(q, scale, ew.up_w, ew.up_scale).to(dt).float()
    g = product(q, scale, ew.gate_w, ew.gate_scale).to(dt).float()
    h = (u * (g / (1.0 + expf(-g))).to(dt).float()).to(dt)
    hq, hs = quantise(h)
    return product(hq, hs, ew.down_w, ew.down_scale).to(dt)


def layer(q, scale, ids, w, experts, dt, shared=None):
    T, K = ids.shape
    out = torch.zeros(T, K, q.shape[1], dtype=dt)
    for e in torch.unique(ids).tolist():
        t, k = (ids == e).nonzero(as_tuple=True)
        out[t, k] = expert(q[t], scale[t], experts[e], dt)
    acc = torch.zeros(T, q.shape[1])
    for k in range(K):
        p = w[:, k].float()[:, None] * out[:, k].float()
        acc = acc + (p if w.dtype == torch.float32 else p.to(dt).float())
    y = acc.to(dt)
    return y if shared is None else (y.float() + expert(q, scale, shared, dt).float()).to(dt)
