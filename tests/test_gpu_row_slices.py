"""Slices of rows whose length is not a multiple of 16 bytes: taken wherever the rows are not read or written 16 bytes at a time."""
import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu


def linear(ek, cuda, K, N, dt, rows, seed=0):
    g = torch.Generator().manual_seed(seed + K * 7 + N)
    w = torch.randint(-128, 128, (N, K), generator=g, dtype=torch.int8).to(cuda)
    ws = ((torch.rand(N, generator=g) + 0.5) / (73 * K ** 0.5)).to(cuda)
    b = torch.randn(N, generator=g).to(dt).to(cuda)
    x = torch.randn(rows, K, generator=g).to(dt)
    return ek.HipLinear(w, ws, bias=b, act_dtype=dt, max_rows=rows), x


@pytest.mark.parametrize("K", [1, 65, 1003, 1004, 1006, 1096])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_linear_row_slices(ek, cuda, K, n, dt):
    op, x = linear(ek, cuda, K, 131, dt, 48)
    q, s = ref.codes(x)
    dx, dq, ds = x.to(cuda), q.to(torch.int8).to(cuda), s.float().to(cuda)
    stream = torch.cuda.Stream()
    for lo in (1, 2, 3, 5):
        part = slice(lo, lo + n)
        assert torch.equal(op.forward(dx[part]), op.forward(dx[part].clone())), f"16-bit rows from {lo} on"
        assert torch.equal(op.forward(dq[part], ds[part]), op.forward(dq[part].clone(), ds[part].clone())), f"8-bit rows from {lo} on"
        torch.cuda.synchronize()
        y = op.forward(dx[part], stream=stream)
        z = op.forward(dq[part], ds[part], stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(y, op.forward(dx[part])) and torch.equal(z, op.forward(dq[part], ds[part])), f"enqueued, from {lo} on"


@pytest.mark.parametrize("K", [64, 128, 1096, 1024])
def test_linear_16_bit_rows_at_any_element(ek, cuda, K):
    """Whole rows that start two bytes off a 16-byte boundary."""
    op, x = linear(ek, cuda, K, 96, torch.bfloat16, 20)
    flat = torch.empty(20 * K + 1, dtype=torch.bfloat16, device=cuda)
    off = flat[1:].view(20, K)
    off.copy_(x)
    torch.cuda.synchronize()
    assert torch.equal(op.forward(off), op.forward(x.to(cuda)))


@pytest.mark.parametrize("n,K,N", [(5, 256, 131), (5, 256, 132), (5, 256, 130), (40, 100, 131), (40, 256, 132), (2100, 1088, 4099), (2100, 1088, 4100)])
def test_linear_output_slices(ek, cuda, n, K, N):
    """Rows of y that start on odd boundaries, and nothing written beside them."""
    op, x = linear(ek, cuda, K, N, torch.float16, n)
    want = op.forward(x.to(cuda))
    for lo in (1, 2, 3):
        big = torch.full((n + 5, N), 7, dtype=torch.float16, device=cuda)
        op.forward(x.to(cuda), out=big[lo:lo + n])
        assert torch.equal(big[lo:lo + n], want), lo
        assert bool((big[:lo] == 7).all()) and bool((big[lo + n:] == 7).all()), lo


def test_linear_alignment_that_is_needed(ek, cuda):
    """Rows read and written where they lie, 16 bytes at a time, are still refused off a boundary."""
    from ek_hip import _capi as C
    op, x = linear(ek, cuda, 256, 128, torch.bfloat16, 4)
    lib, h = ek.load(), op._h
    q = torch.zeros(5, 256, dtype=torch.int8, device=cuda)
    s, y = torch.ones(4, device=cuda), torch.zeros(5, 128, dtype=torch.bfloat16, device=cuda)
    call = lambda xp, sp, yp: lib.ek_linear_forward(h, xp, sp, 4, yp, C.EK_DEVICE, None)
    assert call(q.data_ptr() + 8, s.data_ptr(), y.data_ptr()) == C.EK_INVALID_INPUT
    assert call(q.data_ptr(), s.data_ptr(), y.data_ptr() + 8) == C.EK_INVALID_INPUT
    assert call(q.data_ptr(), s.data_ptr() + 2, y.data_ptr()) == C.EK_INVALID_INPUT
    assert call(q.data_ptr() + 1, None, y.data_ptr()) == C.EK_INVALID_INPUT            # 16-bit rows: half an element off
    assert call(q.data_ptr(), s.data_ptr(), y.data_ptr()) == C.EK_OK
    odd, _ = linear(ek, cuda, 256, 131, torch.bfloat16, 4)
    z = torch.zeros(5, 131, dtype=torch.bfloat16, device=cuda)
    assert lib.ek_linear_forward(odd._h, q.data_ptr(), s.data_ptr(), 4, z.data_ptr() + 1, C.EK_DEVICE, None) == C.EK_INVALID_INPUT


@pytest.mark.parametrize("H,I", [(136, 100), (200, 51), (16, 8), (24, 20)])
@pytest.mark.parametrize("T", [1, 9, 70])
def test_layer_row_slices(ek, cuda, H, I, T):
    """A padded layer copies its 8-bit rows into its own lengths, wherever they start."""
    E, K, dt = 4, 2, torch.bfloat16
    g = torch.Generator().manual_seed(H + I)
    i8 = lambda r, c: torch.randint(-128, 128, (r, c), generator=g, dtype=torch.int8)
    sc = lambda n, k: ((torch.rand(n, generator=g) + 0.5) / (73 * k ** 0.5)).to(torch.bfloat16)
    layer = ek.HipLayer(H, I, E, K, act_dtype=dt, w_dtype=torch.int8, max_tokens=T, act8=True)
    ws = []
    for e in range(E):
        ws.append(ek.ExpertWeight(up_w=i8(I, H), gate_w=i8(I, H), down_w=i8(H, I), up_scale=sc(I, H), gate_scale=sc(I, H), down_scale=sc(H, I)))
        layer.set_expert(e, ws[-1])
    x = torch.randn(T + 3, H, generator=g).to(dt)
    p, ids = torch.topk(torch.softmax(torch.randn(T, E, generator=g), 1), K, dim=1)
    q, s = ref.quantise(x)
    dq, ds, dids, dw = q.to(torch.int8).to(cuda), s.to(cuda), ids.to(torch.int32).to(cuda), p.to(cuda)
    stream = torch.cuda.Stream()
    for lo in (1, 2, 3):
        part = slice(lo, lo + T)
        want = ref.layer(q[part], s[part], ids.to(torch.int32), p, ws, dt)
        assert torch.equal(layer.forward_q8(dq[part], ds[part], dids, dw).cpu(), want), lo
        torch.cuda.synchronize()
        y = layer.forward_q8(dq[part], ds[part], dids, dw, stream=stream)
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), want), f"enqueued, from {lo} on"
