"""ek_norm against its definition in 64 bits: sum and q exactly, y and scale within their roundings."""
import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


def make(n, H, dt, residual=True, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + H)
    x = (torch.randn(n, H, generator=g) * scale).to(dt)
    r = (torch.randn(n, H, generator=g) * scale).to(dt) if residual else None
    gain = (1 + 0.2 * torch.randn(H, generator=g)).to(dt)
    return x, r, gain


def check(out, x, r, gain, eps=EPS):
    dt = x.dtype
    total, v, q, s = ref.norm(x, r, gain, eps)
    if r is not None:
        assert torch.equal(out.sum.cpu(), total)
    else:
        assert out.sum is None
    # p is exact; rstd (fp64, rounded once), its product with p: two roundings to fp32
    ref.assert_close16(out.y, v, dt, 3 * ref.U32 * v.abs(), "y")
    assert torch.equal(out.q.cpu().double(), q), f"{int((out.q.cpu().double() != q).sum())} codes differ"
    # rstd, m * rstd, / 127
    assert bool(((out.scale.cpu().double() - s).abs() <= 4 * ref.U32 * s + 2.0 ** -149).all())


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H", [(1, 8), (1, 7168), (3, 64), (5, 512), (2, 520), (17, 2048), (4, 2056), (33, 4096), (3, 8184),
                                 (3, 8192), (2, 8200), (2, 32768), (2, 32776), (700, 128)])
@pytest.mark.parametrize("residual", [True, False])
def test_norm(ek, cuda, dt, n, H, residual):
    x, r, gain = make(n, H, dt, residual)
    op = ek.HipNorm(gain)
    dev = lambda t: None if t is None else t.to(cuda)
    check(op.forward(dev(x), dev(r)), x, r, gain)                          # blocking, device memory
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    out = op.forward(dev(x), dev(r), stream=s)
    torch.cuda.synchronize()
    check(out, x, r, gain)


def test_norm_host_memory(ek, cuda):
    for n, H, dt, residual in [(3, 136, torch.bfloat16, True), (20, 2048, torch.float16, False), (1, 64, torch.float16, True)]:
        x, r, gain = make(n, H, dt, residual, seed=1)
        op = ek.HipNorm(gain.to(cuda))
        check(op.forward(x, r), x, r, gain)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_norm_borders_of_the_codes(ek, cuda, dt):
    """Rows whose values lie exactly on the borders between codes (max 127: the border of k and k + 1 is k + 1/2)."""
    H = 256
    k = torch.arange(0, 127)
    row = torch.cat([k + 0.5, -(k + 0.5), torch.tensor([127.0, 0.0])]).to(dt).float()
    rows = torch.stack([row * f for f in (1.0, 2.0, 0.25, 64.0 if dt == torch.float16 else 2.0 ** 90, 2.0 ** -10)]).to(dt)
    gain = torch.ones(H, dtype=dt)
    op = ek.HipNorm(gain)
    check(op.forward(rows.to(cuda)), rows, None, gain)
    g = torch.Generator().manual_seed(5)                                   # other maxima, gains that move the borders
    rows = (torch.randint(-40, 41, (64, H), generator=g) / 8.0).to(dt)
    gain = (torch.randint(1, 9, (H,), generator=g) / 4.0).to(dt)
    check(ek.HipNorm(gain).forward(rows.to(cuda)), rows, None, gain)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_norm_extreme_rows(ek, cuda, dt):
    """Zero rows, one value alone, the type's smallest and largest values: finite everywhere."""
    H = 72
    fi = torch.finfo(dt)
    x = torch.zeros(7, H)
    x[1, 5] = 3.0
    x[2] = fi.smallest_normal * fi.eps * torch.arange(1, H + 1)            # subnormal values
    x[3] = fi.max
    x[4, ::2], x[4, 1::2] = fi.max, -fi.max
    x[5, 0], x[5, 1:] = fi.max, fi.smallest_normal
    x[6] = torch.linspace(-1, 1, H) * 1e-4
    x = x.to(dt)
    gain = torch.full((H,), 0.5, dtype=dt)
    out = ek.HipNorm(gain).forward(x.to(cuda))
    check(out, x, None, gain)
    assert float(out.scale[0]) == 0 and not bool(out.y[0].any()) and not bool(out.q[0].any())


def test_norm_not_finite_rows(ek, cuda):
    x, r, gain = make(6, 640, torch.bfloat16, True, seed=3)
    x[1, 17] = float("nan")
    x[3, 600] = float("inf")
    r[4, 0] = -float("inf")
    out = ek.HipNorm(gain).forward(x.to(cuda), r.to(cuda))
    bad = [1, 3, 4]
    good = [0, 2, 5]
    assert bool(out.scale.isnan()[bad].all()) and not bool(out.q[bad].any()) and bool(out.y[bad].isnan().all())
    check(type(out)(*(t[good] for t in out)), x[good], r[good], gain)


def test_norm_in_place_and_outputs_left_out(ek, cuda):
    x, r, gain = make(40, 1000, torch.bfloat16, True, seed=4)
    op = ek.HipNorm(gain)
    want = op.forward(x.to(cuda), r.to(cuda))
    for target in ("residual", "x"):                                       # the stream of residuals updated in place
        dx, dr = x.to(cuda), r.to(cuda)
        keep = dr if target == "residual" else dx
        y = torch.empty_like(dx)
        out = op.forward(dx, dr, out=ek.NormOut(keep, y, torch.empty_like(want.q), torch.empty_like(want.scale)))
        assert out.sum is keep
        for a, b in zip(out, want):
            assert torch.equal(a, b)
    dx, dr = x.to(cuda), r.to(cuda)
    out = op.forward(dx, dr, out=ek.NormOut(dx, dr, None, None))           # both updated in place
    assert torch.equal(out.sum, want.sum) and torch.equal(out.y, want.y)
    only = op.forward(x.to(cuda), r.to(cuda), norm=False)
    assert only.y is None and torch.equal(only.q, want.q) and torch.equal(only.scale, want.scale)
    only = op.forward(x.to(cuda), r.to(cuda), quantize=False)
    assert only.q is None and only.scale is None and torch.equal(only.y, want.y)


def test_norm_does_not_touch_other_rows(ek, cuda):
    x, r, gain = make(5, 264, torch.float16, True, seed=6)
    op = ek.HipNorm(gain)
    big = [torch.full((9, 264), 7, dtype=torch.float16, device=cuda) for _ in range(2)] + [
        torch.full((9, 264), 7, dtype=torch.int8, device=cuda), torch.full((9,), 7.0, device=cuda)]
    part = ek.NormOut(*(t[2:7] for t in big))
    check(op.forward(x.to(cuda), r.to(cuda), out=part), x, r, gain)
    for t in big:
        assert bool((t[:2] == 7).all()) and bool((t[7:] == 7).all())


def test_norm_under_capture(ek, cuda):
    x, r, gain = make(9, 2048, torch.bfloat16, True, seed=7)
    op = ek.HipNorm(gain)
    dx, dr = x.to(cuda), r.to(cuda)
    out = op.forward(dx, dr)
    for t in out:
        t.zero_()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        op.forward(dx, dr, stream=s, out=out)
    for seed in (8, 9, 10):
        x, r, _ = make(9, 2048, torch.bfloat16, True, seed=seed)
        dx.copy_(x)
        dr.copy_(r)
        g.replay()
        torch.cuda.synchronize()
        check(out, x, r, gain)


def test_norm_refusals(ek, cuda):
    from ek_hip import _capi as C
    gain = torch.ones(64, dtype=torch.bfloat16)
    op = ek.HipNorm(gain)
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=cuda)
    lib, h = ek.load(), op._h
    bad = [lambda: op.forward(x.half()), lambda: op.forward(x[:, :56]), lambda: op.forward(x, x[:2]), lambda: op.forward(x, x.cpu()),
           lambda: op.forward(x[0]), lambda: ek.HipNorm(gain, eps=0.0), lambda: ek.HipNorm(gain, eps=float("nan")),
           lambda: ek.HipNorm(gain[:60]), lambda: ek.HipNorm(gain.float()),
           lambda: op.forward(x, out=ek.NormOut(x, None, None, None)),            # a sum without a residual
           lambda: op.forward(x, out=ek.NormOut(None, None, None, None)),
           lambda: op.forward(x, out=ek.NormOut(None, None, torch.empty(4, 64, dtype=torch.int8, device=cuda), None)),
           lambda: op.forward(x, norm=False, quantize=False)]
    for i, f in enumerate(bad):
        with pytest.raises(ek.EKError) as ei:
            f()
        assert ei.value.status == C.EK_INVALID_INPUT, i
    p = x.data_ptr()
    assert lib.ek_norm_forward(h, p + 2, None, 1, None, p, None, None, C.EK_DEVICE, None) == C.EK_INVALID_INPUT      # alignment
    assert lib.ek_norm_forward(h, p, p, 1, p, p, None, None, C.EK_DEVICE, None) == C.EK_INVALID_INPUT                # sum is y
    assert lib.ek_norm_forward(h, p, None, -1, None, p, None, None, C.EK_DEVICE, None) == C.EK_INVALID_INPUT
    assert lib.ek_norm_forward(h, None, None, 1, None, p, None, None, C.EK_DEVICE, None) == C.EK_INVALID_INPUT
    assert lib.ek_norm_forward(h, p, None, 1, None, p, None, None, C.EK_HOST, torch.cuda.Stream().cuda_stream) == C.EK_INVALID_INPUT
    assert lib.ek_norm_forward(h, p, None, 0, None, p, None, None, C.EK_DEVICE, None) == C.EK_OK                     # no rows


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,H,scale", [(400, 2048, 1.0), (60, 7168, 1.0), (9, 33000, 1.0), (500, 512, 2e-7)])
def test_norm_y_is_the_nearest_fp32_value_rounded(ek, cuda, dt, n, H, scale):
    """y by way of fp32: equal wherever the definition's value is further from a border of fp32 than the kernel's arithmetic
    is inexact (2^-40 for rstd, and the product's low part, 2^-48); scale: rows so small that y is subnormal in fp16."""
    x, r, gain = make(n, H, dt, seed=12)
    gain = (gain.float() * scale).to(dt)
    out = ek.HipNorm(gain).forward(x.to(cuda), r.to(cuda))
    _, v, _, _ = ref.norm(x, r, gain, EPS)
    low, high = (v * (1 - 2.0 ** -38)).float().to(dt), (v * (1 + 2.0 ** -38)).float().to(dt)
    y = out.y.cpu()
    clear = low == high
    assert int((~clear).sum()) <= 8
    assert torch.equal(y[clear], low[clear])
