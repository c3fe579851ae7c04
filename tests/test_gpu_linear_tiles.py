"""ek_linear in its tile kernel (products too large for the streaming one): every count of 32-row blocks, contractions of odd
and even numbers of 64-element chunks, channels that end inside a tile, bias, both types; and both kernels bit for bit."""
import pytest
import torch

import act8_ref as ref
import act8_rules

pytestmark = pytest.mark.gpu


def make(cuda, n, K, N, dt, bias, seed):
    g = torch.Generator(device=cuda).manual_seed(seed * 7919 + n * 13 + K * 7 + N)
    q = torch.randint(-128, 128, (n, K), generator=g, device=cuda, dtype=torch.int8)
    s = torch.rand(n, generator=g, device=cuda) * 0.02 + 0.01
    w = torch.randint(-128, 128, (N, K), generator=g, device=cuda, dtype=torch.int8)
    ws = ((torch.rand(N, generator=g, device=cuda) + 0.5) / (73 * K ** 0.5)).to(torch.bfloat16)
    b = torch.randn(N, generator=g, device=cuda).to(dt) if bias else None
    return q, s, w, ws, b


def check(y, q, s, w, ws, b, dt, what):
    q, s, w, ws, b = (None if t is None else t.cpu() for t in (q, s, w, ws, b))
    want, slack = ref.linear(q, s, w, ws, b)
    ref.assert_close16(y, want, dt, slack, what)


# rows of the last item: 1 .. 8 blocks of 32; 3, 3.5 .. 17 steps of 128 elements; channels whole, odd, of 4, ending before, on and
# behind a tile of 16 and a block of 256
SHAPES = [(3841, 384, 4096), (3841 + 32, 448, 4081), (3841 + 70, 576, 4084), (3968, 704, 4088), (3995, 832, 4000), (4032, 1088, 3849),
          (4050, 1216, 4095), (4096, 2176, 3841), (2100, 1088, 4099), (1024, 2048, 7168), (4090, 300, 4093)]


@pytest.mark.parametrize("n,K,N", SHAPES)
def test_tile_kernel_against_the_definition_and_the_streaming_kernel(ek, cuda, n, K, N):
    if act8_rules.available():
        assert not act8_rules.dense_streams(n, K, N) and act8_rules.dense_streams(300, K, N)
    dt = torch.float16 if (n + N) % 2 else torch.bfloat16
    for bias in (True, False):
        q, s, w, ws, b = make(cuda, n, K, N, dt, bias, seed=1)
        op = ek.HipLinear(w, ws, bias=b, act_dtype=dt, max_rows=n)
        big = torch.full((n + 2, N), 7, dtype=dt, device=cuda)
        y = op.forward(q, s, out=big[1:n + 1]) if N % 8 == 0 else op.forward(q, s)
        if N % 8 == 0:
            assert bool((big[0] == 7).all()) and bool((big[n + 1] == 7).all())
        for lo in range(0, n, 300):                                       # slices of 300 rows stream: the same bits
            part = slice(lo, min(lo + 300, n))
            assert torch.equal(y[part], op.forward(q[part].clone(), s[part].clone())), (lo, bias)
        part = slice(max(0, n - 70), n)
        check(y[part], q[part], s[part], w, ws, b, dt, f"{n} x {K} x {N}, bias {bias}")
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        z = op.forward(q, s, stream=st)
        torch.cuda.synchronize()
        assert torch.equal(z, y)


@pytest.mark.parametrize("n,K,N", [(2100, 1088, 4099), (4040, 1003, 4001)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_tile_kernel_on_16_bit_rows(ek, cuda, n, K, N, dt):
    _, _, w, ws, b = make(cuda, 1, K, N, dt, True, seed=2)
    x = torch.randn(n, K, generator=torch.Generator(device=cuda).manual_seed(K), device=cuda).to(dt)
    x[5] = 0
    op = ek.HipLinear(w, ws, bias=b, act_dtype=dt, max_rows=n)
    y = op.forward(x)
    q, s = ref.codes(x.cpu())
    part = slice(n - 70, n)
    check(y[part], q[part], s[part].float(), w, ws, b, dt, "16-bit rows")
    check(y[:40], q[:40], s[:40].float(), w, ws, b, dt, "16-bit rows")
    assert torch.equal(y, op.forward(q.to(torch.int8).to(cuda), s.float().to(cuda)))


def test_tile_kernel_under_capture(ek, cuda):
    n, K, N, dt = 2100, 1088, 4099, torch.bfloat16
    q, s, w, ws, b = make(cuda, n, K, N, dt, True, seed=3)
    op = ek.HipLinear(w, ws, bias=b, act_dtype=dt, max_rows=n)
    y = op.forward(q, s)
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        op.forward(q, s, stream=st, out=y)
    for seed in (4, 5, 6):
        fresh = make(cuda, n, K, N, dt, False, seed=seed)
        q.copy_(fresh[0]), s.copy_(fresh[1]), y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(op.forward(q, s), got)
        check(got[-40:], q[-40:], s[-40:], w, ws, b, dt, "replay")


def test_rows_that_are_not_finite_stay_alone(ek, cuda):
    n, K, N, dt = 2100, 1088, 4099, torch.float16
    q, s, w, ws, b = make(cuda, n, K, N, dt, True, seed=7)
    op = ek.HipLinear(w, ws, bias=b, act_dtype=dt, max_rows=n)
    want = op.forward(q, s)
    bad = [0, 255, 256, 1031, n - 1]
    s[bad] = float("nan")
    q[bad] = 0
    y = op.forward(q, s)
    assert bool(y[bad].isnan().all())
    keep = torch.ones(n, dtype=torch.bool, device=cuda)
    keep[bad] = False
    assert torch.equal(y[keep], want[keep])
