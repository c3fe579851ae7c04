"""ek_norm where its fp32 quantities are few bits away from the definition's: the scale is the definition's value rounded
once, and rows of the largest values keep their y."""
import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


def make(n, H, dt, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + H)
    x = (torch.randn(n, H, generator=g).clamp(-3.9, 3.9) * scale).to(dt)
    r = (torch.randn(n, H, generator=g).clamp(-3.9, 3.9) * scale * 2.0 ** -4).to(dt)
    return x, r, (1 + 0.2 * torch.randn(H, generator=g)).to(dt)


def scale_error(out, x, r, gain, eps=EPS):
    """|scale - definition| in half steps of fp32."""
    _, _, _, s = ref.norm(x, r, gain, eps)
    got = out.scale.cpu().double()
    m = torch.frexp(s.abs())[1].clamp_min(-125)                        # half a step of fp32 at s
    return (got - s).abs() / torch.exp2((m - 25).double())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H", [(3000, 64), (700, 1000), (500, 2048), (300, 4096), (200, 7168), (40, 33000)])
def test_scale_is_rounded_once(ek, cuda, dt, n, H):
    x, r, gain = make(n, H, dt, seed=1)
    op = ek.HipNorm(gain)
    for res in (r, None):
        out = op.forward(x.to(cuda), None if res is None else res.to(cuda))
        # the reciprocal root is within 2^-40 and two fp64 products follow: 2^-15 of a half step
        worst = float(scale_error(out, x, res, gain).max())
        assert worst <= 1.0 + 2.0 ** -14, f"{worst} half steps"


@pytest.mark.parametrize("n,H", [(4, 72), (300, 1000), (400, 7168), (30, 16384), (9, 33000)])
@pytest.mark.parametrize("magnitude", [2.0 ** 100, 2.0 ** 112, 2.0 ** 120, 2.0 ** 125])
def test_rows_near_the_types_largest_values(ek, cuda, n, H, magnitude):
    """bf16 rows whose reciprocal root is near fp32's smallest normal number, or below it: y as at any other magnitude."""
    dt = torch.bfloat16
    x, r, gain = make(n, H, dt, seed=2, scale=magnitude)
    gain = (gain.float() * 2.0 ** -9).to(dt)                           # sum * gain within fp32's range
    out = ek.HipNorm(gain).forward(x.to(cuda), r.to(cuda))
    total, v, q, s = ref.norm(x, r, gain, EPS)
    assert bool(total.isfinite().all()) and torch.equal(out.sum.cpu(), total) and torch.equal(out.q.cpu().double(), q)
    assert float(scale_error(out, x, r, gain).max()) <= 1.0 + 2.0 ** -14
    low, high = (v * (1 - 2.0 ** -38)).float().to(dt), (v * (1 + 2.0 ** -38)).float().to(dt)
    clear, y = low == high, out.y.cpu()                                # away from a border of fp32 the answer is one
    assert int((~clear).sum()) <= 8
    wrong = int((y[clear] != low[clear]).sum())
    assert wrong == 0, f"{wrong} of {y.numel()}"


def test_largest_rows_of_all(ek, cuda):
    """Rows that hold bf16's largest values only: the mean of squares is beyond fp32 and the root at its end."""
    dt, H = torch.bfloat16, 640
    big = torch.finfo(dt).max
    g = torch.Generator().manual_seed(3)
    x = torch.where(torch.rand(20, H, generator=g) < 0.5, -big, big).to(dt)
    x[10:] = (x[10:].float() * (0.5 + 0.5 * torch.rand(10, H, generator=g))).to(dt)
    gain = (0.25 + 0.5 * torch.rand(H, generator=g)).to(dt)
    out = ek.HipNorm(gain).forward(x.to(cuda))
    _, v, q, _ = ref.norm(x, None, gain, EPS)
    assert torch.equal(out.q.cpu().double(), q) and float(scale_error(out, x, None, gain).max()) <= 1.0 + 2.0 ** -14
    low, high = (v * (1 - 2.0 ** -38)).float().to(dt), (v * (1 + 2.0 ** -38)).float().to(dt)
    clear = low == high
    assert torch.equal(out.y.cpu()[clear], low[clear])
