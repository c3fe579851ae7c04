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
