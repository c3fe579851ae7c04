"""Layers on 8-bit activations in each way a call is cut, through every entry point, bit for bit: large layers whose decode calls
stream short segments beside tiles (class 1 of ek::q8_one_class) and whose longer calls are all tiles (class 2), with and
without shared experts; every size of a tile item; per-expert calls and batches that are tiled."""
import pytest
import torch

import act8_ref as ref
import act8_rules
from test_gpu_act8_layer import build, call, same, weight

pytestmark = pytest.mark.gpu

# 40 experts of 1088 x 576: 75 million weights, beyond what small calls stream whole; 17 and 9 chunks of 64 (both odd)
H, I, E = 1088, 576, 40
T_MAX = 330
_built = {}


def layer(ek, K, dt, shared_inter=None, seed=0):
    key = (K, dt, shared_inter, seed)
    if key not in _built:
        _built.clear()                                              # (one large layer at a time)
        _built[key] = build(ek, H, I, E, K, dt, T_MAX, seed=seed, shared_inter=shared_inter)
    return _built[key]


def check_class(T, K, want):
    if act8_rules.available():
        assert act8_rules.layer_class(T * K, E, H, I) == want, (T, K)


def both(layer, x, ids, w, want, cuda, what):
    q, s = ref.quantise(x)
    dx, dids, dw, dq, ds = x.to(cuda), ids.to(cuda), w.to(cuda), q.to(torch.int8).to(cuda), s.to(cuda)
    same(layer.forward(dx, dids, dw), want, what + ", 16-bit rows")
    y, rt = layer.forward_q8(dq, ds, dids, dw, return_route=True)
    same(y, want, what + ", 8-bit rows")
    assert torch.equal(rt.counts.long().cpu(), torch.bincount(ids.reshape(-1).long(), minlength=E))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    y = layer.forward_q8(dq, ds, dids, dw, stream=st)
    z = layer.forward(dx, dids, dw, stream=st)
    torch.cuda.synchronize()
    same(y, want, what + ", enqueued")
    same(z, want, what + ", enqueued 16-bit rows")


@pytest.mark.parametrize("T,K,skew,cls", [(17, 2, 0.0, 1), (64, 2, 1.5, 1), (65, 8, 0.5, 1), (200, 2, 3.0, 1), (300, 2, 4.0, 1), (300, 1, 6.0, 1),
                                          (200, 4, 0.0, 2), (256, 4, 2.0, 2), (330, 2, 0.0, 2), (300, 8, 1.0, 2)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_large_layer(ek, cuda, T, K, skew, cls, dt):
    check_class(T, K, cls)
    lay, ws, _ = layer(ek, K, dt)
    x, ids, w = call(T, H, E, K, dt, seed=T, skew=skew, w32=T % 2 == 1)
    if cls == 1 and skew >= 1.5:                                     # both kernels have work
        counts = torch.bincount(ids.reshape(-1).long(), minlength=E)
        assert int((counts > 16).sum()) and int(((counts > 0) & (counts <= 16)).sum())
    both(lay, x, ids, w, ref.layer(*ref.quantise(x), ids, w, ws, dt), cuda, f"{T} tokens, top-{K}")


@pytest.mark.parametrize("T,K,cls", [(9, 2, 1), (17, 2, 1), (33, 2, 1), (64, 2, 1), (65, 2, 1), (65, 8, 1), (129, 2, 1), (200, 2, 1), (256, 2, 1),
                                     (257, 2, 1), (300, 2, 1), (170, 4, 2), (256, 4, 2), (300, 4, 2)])
@pytest.mark.parametrize("width", [1, 2])
def test_large_layer_with_a_shared_expert(ek, cuda, T, K, cls, width):
    """The shared segment's cuts (16-row items, wide items, tiles; in the routed lists or in its own) beside either class."""
    dt = torch.bfloat16
    check_class(T, K, cls)
    lay, ws, shared = layer(ek, K, dt, shared_inter=width * I, seed=1)
    x, ids, w = call(T, H, E, K, dt, seed=T + 1, skew=2.0, w32=True)
    both(lay, x, ids, w, ref.layer(*ref.quantise(x), ids, w, ws, dt, shared), cuda, f"{T} tokens, top-{K}, shared {width * I}")


@pytest.mark.parametrize("T,K,cls", [(2, 4, 1), (40, 4, 1), (200, 2, 1), (300, 4, 2)])
def test_tokens_that_name_an_expert_twice(ek, cuda, T, K, cls):
    """Routings drawn with replacement, among them tokens whose pairs are all of one expert."""
    dt = torch.float16
    check_class(T, K, cls)
    lay, ws, shared = layer(ek, K, dt, shared_inter=I, seed=9)
    x, _, w = call(T, H, E, K, dt, seed=T + 9, w32=True)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, E, (T, K), generator=g).to(torch.int32)
    ids[:: 3] = ids[:: 3, :1]
    ids[1::4] = 7
    both(lay, x, ids, w, ref.layer(*ref.quantise(x), ids, w, ws, dt, shared), cuda, f"{T} tokens, top-{K}")


@pytest.mark.parametrize("shared_inter", [None, I, 2 * I])
@pytest.mark.parametrize("T,K,cls", [(64, 2, 1), (96, 4, 1), (200, 4, 2)])
def test_static_workspace(ek, cuda, T, K, cls, shared_inter):
    dt = torch.float16
    check_class(T, K, cls)
    lay, ws, shared = layer(ek, K, dt, shared_inter=shared_inter, seed=2)
    x, ids, w = call(T, H, E, K, dt, seed=T + 2, skew=1.0)
    want = ref.layer(*ref.quantise(x), ids, w, ws, dt, shared)
    dx, dids, dw = x.to(cuda), ids.to(cuda), w.to(cuda)
    same(lay.forward_static(dx, dids, dw), want, "static")
    st, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    y = torch.empty_like(dx)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        lay.forward_static(dx, dids, dw, stream=st, out=y)
    for seed in (50, 51, 52):
        x, ids, w = call(T, H, E, K, dt, seed=seed, skew=float(seed - 50))
        dx.copy_(x), dids.copy_(ids), dw.copy_(w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        same(y, ref.layer(*ref.quantise(x), ids, w, ws, dt, shared), f"static, replay {seed}")


@pytest.mark.parametrize("shared_inter", [None, I, 2 * I])
@pytest.mark.parametrize("T,K,cls", [(70, 2, 1), (300, 2, 1), (256, 4, 2)])
def test_capture(ek, cuda, T, K, cls, shared_inter):
    """A captured call replayed on other rows and routings, whose segments fall into other lists, with eager calls between."""
    dt = torch.bfloat16
    check_class(T, K, cls)
    lay, ws, shared = layer(ek, K, dt, shared_inter=shared_inter, seed=3)
    x, ids, w = call(T, H, E, K, dt, seed=0)
    dx, dids, dw = x.to(cuda), ids.to(cuda), w.to(cuda)
    y = lay.forward(dx, dids, dw)
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        lay.forward(dx, dids, dw, stream=st, out=y)
    for seed in (1, 2, 3):
        x, ids, w = call(T, H, E, K, dt, seed=seed, skew=1.5 * seed)
        dx.copy_(x), dids.copy_(ids), dw.copy_(w)
        y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        same(y, ref.layer(*ref.quantise(x), ids, w, ws, dt, shared), f"replay {seed}")
        x2, ids2, w2 = call(23, H, E, K, dt, seed=seed + 50)
        same(lay.forward(x2.to(cuda), ids2.to(cuda), w2.to(cuda)), ref.layer(*ref.quantise(x2), ids2, w2, ws, dt, shared), "eager")


@pytest.mark.parametrize("shared_inter", [None, 2 * I])
def test_two_streams(ek, cuda, shared_inter):
    K, dt = 2, torch.bfloat16
    lay, _, _ = layer(ek, K, dt, shared_inter=shared_inter, seed=4)
    calls = [[t.to(cuda) for t in call(T, H, E, K, dt, seed=T, skew=2.0)] for T in (300, 17, 65, 330, 129, 40)]
    want = [lay.forward(*c) for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [lay.forward(*c, stream=streams[i % 2]) for i, c in enumerate(calls)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("shared_inter", [None, I])
@pytest.mark.parametrize("T,cls", [(70, 1), (200, 2)])
def test_chain(ek, cuda, T, cls, shared_inter):
    K, dt = 4, torch.bfloat16
    check_class(T, K, cls)
    _built.clear()
    layers = [build(ek, H, I, E, K, dt, T_MAX, seed=10 + l, shared_inter=shared_inter) for l in range(2)]
    calls = [call(T, H, E, K, dt, seed=l, skew=1.0 + l) for l in range(2)]
    ids, w = torch.stack([c[1] for c in calls]), torch.stack([c[2] for c in calls])
    want = x = calls[0][0]
    for l in range(2):
        want = ref.layer(*ref.quantise(want), ids[l], w[l], layers[l][1], dt, layers[l][2])
    chain = ek.HipChain([l[0] for l in layers])
    for use_graph in (False, True, True, True):
        same(chain.forward(x.to(cuda), ids.to(cuda), w.to(cuda), use_graph=use_graph), want, f"graph {use_graph}")
    chain.close()


# ---- every item of the tile kernel -------------------------------------------------------------------

COUNTS = [17, 33, 65, 97, 129, 161, 193, 225, 256, 1, 32, 257, 0]      # 1 .. 8 blocks of 32 rows, and their borders


@pytest.mark.parametrize("h,i", [(128, 320), (192, 128), (256, 192), (320, 256), (384, 448), (448, 384), (512, 576), (576, 640), (640, 512), (832, 704)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_every_tile_item(ek, cuda, h, i, dt):
    """Contractions of 1, 1.5, .. 6.5 steps of 128 elements in either stage."""
    n_experts, T = len(COUNTS), sum(COUNTS)
    if act8_rules.available():
        assert act8_rules.layer_class(T, n_experts, h, i) == 2
    lay, ws, _ = build(ek, h, i, n_experts, 1, dt, T, seed=5)
    g = torch.Generator().manual_seed(h + i)
    ids = torch.repeat_interleave(torch.arange(n_experts), torch.tensor(COUNTS))[torch.randperm(T, generator=g)].to(torch.int32)[:, None].contiguous()
    x, w = torch.randn(T, h, generator=g).to(dt), torch.rand(T, 1, generator=g)
    want = ref.layer(*ref.quantise(x), ids, w, ws, dt)
    same(lay.forward(x.to(cuda), ids.to(cuda), w.to(cuda)), want, f"{h} x {i}")


# ---- per-expert calls and batches ----------------------------------------------------------------------

def test_per_expert_calls_as_tiles(ek, cuda):
    h, i, dt = 2048, 1024, torch.bfloat16
    lay, ws, _ = build(ek, h, i, 2, 1, dt, 4700, seed=6)
    g = torch.Generator().manual_seed(7)
    for n in (3601, 4700):
        if act8_rules.available():
            assert not act8_rules.expert_streams(n, h, i) and act8_rules.expert_streams(300, h, i)
        x = torch.randn(n, h, generator=g).to(dt).to(cuda)
        y = lay.expert_forward(1, x)
        part = torch.cat([torch.arange(0, 40), torch.arange(n - 300, n)])
        same(y[part], ref.expert(*ref.quantise(x[part].cpu()), ws[1], dt), f"{n} rows")
        for lo in range(0, n, 300):                                  # streamed, the same bits
            assert torch.equal(lay.expert_forward(1, x[lo:lo + 300].clone()), y[lo:lo + 300]), lo
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        z = lay.expert_forward(1, x, stream=st)
        torch.cuda.synchronize()
        assert torch.equal(z, y)


@pytest.mark.parametrize("rows,streamed", [([100] * 16, False), ([1, 16, 0, 129, 257] + [100] * 16 + [7, 2], False), ([40] * 4 + [1] * 5, True),
                                           ([300, 17, 5, 64, 65], True), ([16, 3, 0, 1], False)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_batches_of_calls(ek, cuda, rows, streamed, dt):
    h, i, n_experts = 2048, 1024, 7
    if act8_rules.available():
        assert act8_rules.batch_streams(rows, h, i) == streamed
    lay, ws, _ = build(ek, h, i, n_experts, 1, dt, 2100, seed=8)
    g = torch.Generator().manual_seed(len(rows))
    xs = [torch.randn(n, h, generator=g).to(dt) for n in rows]
    ids = [(3 * c) % n_experts for c in range(len(rows))]
    want = [ref.expert(*ref.quantise(x), ws[e], dt) if len(x) else None for x, e in zip(xs, ids)]
    for dev in ("cpu", cuda):
        for c, (o, y) in enumerate(zip(lay.experts_forward(ids, [x.to(dev) for x in xs]), want)):
            if y is not None:
                same(o, y, f"call {c} of {rows[c]} rows, {dev}")
    st = torch.cuda.Stream()
    dxs = [x.to(cuda) for x in xs]
    torch.cuda.synchronize()
    outs = lay.experts_forward(ids, dxs, stream=st)
    torch.cuda.synchronize()
    for c, (o, y) in enumerate(zip(outs, want)):
        if y is not None:
            same(o, y, f"call {c}, enqueued")
