"""The largest sum of an int8 product: every code and every weight -128 over the longest contraction, 128 * 128 * 131072 =
2^31, one more than an int32 holds."""
import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu
K = 131072


def codes(n, cuda):
    """Row r: its first r codes are 127 and the others -128, so row 0 has the largest sum and the others lie just below."""
    q = torch.full((n, K), -128, dtype=torch.int8, device=cuda)
    head = min(n, K)
    q[:, :head] = torch.where(torch.arange(head, device=cuda)[None, :] < torch.arange(n, device=cuda)[:, None], 127, -128).to(torch.int8)
    return q


def sums(n):
    return 2.0 ** 31 - 255.0 * 128.0 * torch.arange(n, dtype=torch.float64)


@pytest.mark.parametrize("n,N", [(3, 16), (16, 40), (20, 32), (33, 130), (2048, 2048)],
                         ids=["one_tile_of_rows", "sixteen_rows", "row_groups", "odd_channels", "tile_kernel"])
@pytest.mark.parametrize("bias", [False, True])
def test_linear(ek, cuda, n, N, bias):
    dt = torch.bfloat16
    w = torch.full((N, K), -128, dtype=torch.int8, device=cuda)
    w[1::2] = 127                                        # sums of -127 * 128 * 131072 beside the largest
    s = torch.full((n,), 2.0 ** -20)
    ws = torch.linspace(0.5, 1.0, N)
    b = torch.linspace(-64, 64, N).to(dt) if bias else None
    op = ek.HipLinear(w, ws.to(cuda), bias=None if b is None else b.to(cuda), act_dtype=dt, max_rows=n)
    y = op.forward(codes(n, cuda), s.to(cuda))
    # a channel of 127: 127 * (127 r - 128 (K - r))
    r = torch.arange(n, dtype=torch.float64)[:, None]
    total = torch.where(torch.arange(N)[None, :] % 2 == 0, sums(n)[:, None], 127.0 * (127.0 * r - 128.0 * (K - r)))
    prod = total * (s.double()[:, None] * ws.double()[None, :])
    want = prod if b is None else prod + b.double()
    slack = 4 * ref.U32 * prod.abs() * (1 + ref.U32) + (0 if b is None else 2 * ref.U32 * (prod.abs() + b.double().abs()))
    ref.assert_close16(y, want, dt, slack, f"{n} x {K} x {N}")


@pytest.mark.parametrize("T", [1, 20, 40, 1040])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_layer(ek, cuda, T, dt):
    """Stage 1 of a layer whose rows are 131072 long, by each of its kernels; bit for bit."""
    I = 128
    i8 = lambda *shape, v: torch.full(shape, v, dtype=torch.int8)
    ew = ek.ExpertWeight(up_w=i8(I, K, v=-128), gate_w=i8(I, K, v=-128), down_w=i8(K, I, v=3), up_scale=torch.linspace(0.5, 1.0, I),
                         gate_scale=torch.linspace(1.0, 0.5, I), down_scale=torch.full((K,), 2.0 ** -10))
    layer = ek.HipLayer(K, I, 1, 1, act_dtype=dt, w_dtype=torch.int8, max_tokens=T, act8=True)
    layer.set_expert(0, ew)
    s = torch.full((T,), 2.0 ** -29)
    y = layer.forward_q8(codes(T, cuda), s.to(cuda), torch.zeros(T, 1, dtype=torch.int32, device=cuda), torch.ones(T, 1, device=cuda))
    total = sums(T).float()[:, None]
    u = (total * (s[:, None] * ew.up_scale[None, :])).to(dt).float()
    g = (total * (s[:, None] * ew.gate_scale[None, :])).to(dt).float()
    h = (u * (g / (1.0 + ref.expf(-g))).to(dt).float()).to(dt)
    hq, hs = ref.quantise(h)
    o = ref.product(hq, hs, ew.down_w[:1], ew.down_scale[:1]).to(dt)              # every channel of down is alike
    assert bool((u > 0).all())
    got = y.cpu()
    assert torch.equal(got, o.expand(T, K)), f"{int((got != o).sum())} elements differ"
