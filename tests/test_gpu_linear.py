"""ek_linear against its definition in 64 bits."""
import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu


def make(n, K, N, dt, bias, seed=0):
    g = torch.Generator().manual_seed(seed * 104729 + n * 13 + K * 7 + N)
    q = torch.randint(-127, 128, (n, K), generator=g, dtype=torch.int8)
    s = torch.rand(n, generator=g) * 0.02 + 0.01
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8)
    ws = ((torch.rand(N, generator=g) + 0.5) / (73 * K ** 0.5)).to(torch.bfloat16)
    b = torch.randn(N, generator=g).to(dt) if bias else None
    return q, s, w, ws, b


def check(y, q, s, w, ws, b, dt):
    want, slack = ref.linear(q, s, w, ws, b)
    ref.assert_close16(y, want, dt, slack, f"{tuple(q.shape)} x {tuple(w.shape)}")


SHAPES = [(1, 128, 16), (1, 7168, 2048), (16, 192, 48), (17, 256, 64), (3, 64, 8), (5, 1, 1), (37, 1003, 131), (64, 2048, 160),
          (65, 320, 272), (128, 128, 512), (129, 448, 528), (300, 1088, 1000), (513, 704, 2047), (1024, 512, 768), (2, 9000, 40),
          (200, 65, 33), (31, 130, 257), (260, 4096, 96)]


@pytest.mark.parametrize("n,K,N", SHAPES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_linear_on_codes(ek, cuda, n, K, N, dt):
    q, s, w, ws, b = make(n, K, N, dt, bias=(n + K) % 2 == 0)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), bias=None if b is None else b.to(cuda), act_dtype=dt, max_rows=n)
    stream = torch.cuda.Stream()
    dq, ds = q.to(cuda), s.to(cuda)
    torch.cuda.synchronize()
    y = op.forward(dq, ds, stream=stream)
    torch.cuda.synchronize()
    check(y, q, s, w, ws, b, dt)
    assert torch.equal(op.forward(dq, ds), y)                              # blocking: the same bits
    assert op.shape() == (K, N)


@pytest.mark.parametrize("n,K,N", [(1, 136, 16), (7, 1003, 131), (70, 2048, 200), (33, 8200, 64), (2, 33000, 32), (129, 77, 515)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_linear_on_16_bit_rows(ek, cuda, n, K, N, dt):
    _, _, w, ws, b = make(n, K, N, dt, True, seed=1)
    x = torch.randn(n, K, generator=torch.Generator().manual_seed(K)).to(dt)
    x[n // 2] = 0
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), bias=b.to(cuda), act_dtype=dt, max_rows=n)
    q, s = ref.codes(x)
    check(op.forward(x.to(cuda)), q, s, w, ws, b, dt)
    check(op.forward(x), q, s, w, ws, b, dt)                               # host memory
    y = op.forward(q.to(torch.int8), s.float())                            # host memory, codes
    check(y, q, s.float(), w, ws, b, dt)


def test_linear_extreme_codes(ek, cuda):
    """All sums at their largest: 127 * 128 * K does not fit fp32's 24 bits, nor does any partial sum."""
    n, K, N = 20, 131072, 16
    q = torch.full((n, K), 127, dtype=torch.int8)
    q[1::2] = -127
    w = torch.full((N, K), -128, dtype=torch.int8)
    w[::2] = 127
    s, ws = torch.full((n,), 1e-6), torch.full((N,), 1e-4)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), act_dtype=torch.bfloat16, max_rows=n)
    check(op.forward(q.to(cuda), s.to(cuda)), q, s, w, ws, None, torch.bfloat16)


def test_linear_row_results_do_not_depend_on_the_batch(ek, cuda):
    q, s, w, ws, _ = make(300, 1024, 528, torch.bfloat16, False, seed=2)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=300)
    y = op.forward(q.to(cuda), s.to(cuda))
    for n in (1, 16, 17, 63, 64, 65, 128, 200):
        assert torch.equal(op.forward(q[:n].to(cuda), s[:n].to(cuda)), y[:n]), n


def test_linear_not_finite_scales_stay_in_their_row(ek, cuda):
    q, s, w, ws, _ = make(20, 256, 64, torch.bfloat16, False, seed=3)
    q[4], s[4] = 0, float("nan")                                           # what ek_norm makes of a row with a NaN
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=20)
    y = op.forward(q.to(cuda), s.to(cuda))
    assert bool(y[4].isnan().all())
    keep = [i for i in range(20) if i != 4]
    check(y[keep], q[keep], s[keep], w, ws, None, torch.bfloat16)
    x = torch.randn(20, 256).to(torch.bfloat16)
    x[7, 3] = float("inf")
    y = op.forward(x.to(cuda))
    assert bool(y[7].isnan().all()) and bool(y[[i for i in range(20) if i != 7]].isfinite().all())


def test_linear_rows_behind_the_last_stay(ek, cuda):
    q, s, w, ws, b = make(19, 320, 50, torch.float16, True, seed=4)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), bias=b.to(cuda), act_dtype=torch.float16, max_rows=64)
    big = torch.full((40, 50), 7, dtype=torch.float16, device=cuda)
    op.forward(q.to(cuda), s.to(cuda), out=big[8:27])
    check(big[8:27], q, s, w, ws, b, torch.float16)
    assert bool((big[:8] == 7).all()) and bool((big[27:] == 7).all())


def test_linear_two_streams_share_the_workspace(ek, cuda):
    """16-bit rows go through the workspace: calls on two streams are ordered on the device."""
    _, _, w, ws, _ = make(1, 1000, 256, torch.bfloat16, False, seed=5)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=512)
    xs = [torch.randn(512, 1000, device=cuda).to(torch.bfloat16) for _ in range(6)]
    want = [op.forward(x) for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [op.forward(x, stream=streams[i % 2]) for i, x in enumerate(xs)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_linear_under_capture(ek, cuda):
    q, s, w, ws, _ = make(33, 1000, 272, torch.bfloat16, False, seed=6)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=64)
    x = torch.randn(33, 1000, device=cuda).to(torch.bfloat16)
    y = op.forward(x)
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        op.forward(x, stream=st, out=y)
    for _ in range(3):
        x.copy_(torch.randn(33, 1000, device=cuda))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = y.clone()
        assert torch.equal(op.forward(x), got)


def test_norm_feeds_linear(ek, cuda):
    """The two together, as a block uses them: norm's codes through a projection."""
    g = torch.Generator().manual_seed(11)
    n, H, N = 50, 1024, 384
    x, r = torch.randn(n, H, generator=g).to(torch.bfloat16), torch.randn(n, H, generator=g).to(torch.bfloat16)
    gain = (1 + 0.1 * torch.randn(H, generator=g)).to(torch.bfloat16)
    _, _, w, ws, b = make(n, H, N, torch.bfloat16, True, seed=7)
    norm, lin = ek.HipNorm(gain), ek.HipLinear(w.to(cuda), ws.to(cuda), bias=b.to(cuda), max_rows=n)
    st = torch.cuda.Stream()
    dx, dr = x.to(cuda), r.to(cuda)
    torch.cuda.synchronize()
    o = norm.forward(dx, dr, stream=st)
    y = lin.forward(o.q, o.scale, stream=st)
    torch.cuda.synchronize()
    _, _, q, _ = ref.norm(x, r, gain, 1e-6)
    check(y, q, o.scale.cpu(), w, ws, b, torch.bfloat16)


def test_linear_refusals(ek, cuda):
    from ek_hip import _capi as C
    q, s, w, ws, _ = make(4, 128, 32, torch.bfloat16, False)
    dq, ds, dw, dws = q.to(cuda), s.to(cuda), w.to(cuda), ws.to(cuda)
    op = ek.HipLinear(dw, dws, max_rows=4)
    bad = [lambda: op.forward(dq), lambda: op.forward(dq[:, :64], ds), lambda: op.forward(dq, ds[:2]), lambda: op.forward(dq, ds.half()),
           lambda: op.forward(dq, s), lambda: op.forward(dq.half(), ds), lambda: op.forward(torch.cat([dq, dq]), torch.cat([ds, ds])),
           lambda: op.forward(dq, ds, out=torch.empty(4, 31, device=cuda, dtype=torch.bfloat16)),
           lambda: ek.HipLinear(dw, dws[:3]), lambda: ek.HipLinear(dw.float(), dws), lambda: ek.HipLinear(dw, dws, act_dtype=torch.float32),
           lambda: ek.HipLinear(dw, dws, max_rows=0), lambda: ek.HipLinear(dw, dws, bias=dws[:5]),
           lambda: ek.HipLinear(dw, dws, max_rows=1 << 23)]
    for i, f in enumerate(bad):
        with pytest.raises(ek.EKError) as ei:
            f()
        assert ei.value.status == C.EK_INVALID_INPUT, i
    lib, h, p = ek.load(), op._h, dq.data_ptr()
    assert lib.ek_linear_forward(h, p + 1, ds.data_ptr(), 1, p, C.EK_DEVICE, None) == C.EK_INVALID_INPUT
    assert lib.ek_linear_forward(h, None, ds.data_ptr(), 1, p, C.EK_DEVICE, None) == C.EK_INVALID_INPUT
    assert lib.ek_linear_forward(h, None, None, 0, None, C.EK_DEVICE, None) == C.EK_OK


@pytest.mark.parametrize("K", [128, 100])
def test_linear_more_rows_than_one_grid_dimension_counts(ek, cuda, K):
    """More 32-row groups than 65535: the same rows as in calls of a few (narrow matrices are where such calls are
    estimated to be faster in 32-row groups)."""
    n, N = 65535 * 32 + 77, 16
    _, _, w, ws, _ = make(1, K, N, torch.bfloat16, False, seed=8)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=n)
    q = torch.randint(-127, 128, (n, K), device=cuda, dtype=torch.int8)
    s = torch.rand(n, device=cuda)
    y = op.forward(q, s)
    for lo in (0, 65535 * 16 + 3, n - 300):
        part = slice(lo, lo + 300)
        check(y[part], q[part].cpu(), s[part].cpu(), w, ws, None, torch.bfloat16)
    small = ek.HipLinear(w.to(cuda), ws.to(cuda), max_rows=1 << 18)
    for lo in range(0, n, 1 << 18):
        part = slice(lo, min(lo + (1 << 18), n))
        assert torch.equal(y[part], small.forward(q[part].contiguous(), s[part].contiguous()))


def test_linear_two_graphs(ek, cuda):
    """Two captured calls that share the workspace, replayed in turn on one stream with an eager call between."""
    _, _, w, ws, _ = make(1, 200, 80, torch.float16, False, seed=9)
    op = ek.HipLinear(w.to(cuda), ws.to(cuda), act_dtype=torch.float16, max_rows=400)
    xs = [torch.randn(n, 200, device=cuda).half() for n in (400, 19)]
    ys = [op.forward(x) for x in xs]
    st, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for x, y in zip(xs, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            op.forward(x, stream=st, out=y)
        graphs.append(g)
    for _ in range(3):
        for x in xs:
            x.normal_()
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            for g in graphs * 2:
                g.replay()
        torch.cuda.synchronize()
        for x, y in zip(xs, ys):
            got = y.clone()
            assert torch.equal(op.forward(x), got)
