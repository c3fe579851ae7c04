"""Layers on 8-bit activations (EK_CFG_ACT8) against the kernels' arithmetic restated on the CPU: the integer
sums are exact and every other operation is an IEEE fp32 one, so the outputs are compared bit for bit."""
import os
import random

import pytest
import torch

import act8_ref as ref

pytestmark = pytest.mark.gpu


def weight(H, I, g):
    import ek_hip
    i8 = lambda r, c: torch.randint(-128, 128, (r, c), generator=g, dtype=torch.int8)
    sc = lambda n, k: ((torch.rand(n, generator=g) + 0.5) / (73 * k ** 0.5)).to(torch.bfloat16)
    return ek_hip.ExpertWeight(up_w=i8(I, H), gate_w=i8(I, H), down_w=i8(H, I), up_scale=sc(I, H), gate_scale=sc(I, H), down_scale=sc(H, I))


def build(ek, H, I, E, K, dt, T, seed=0, shared_inter=None):
    g = torch.Generator().manual_seed(seed * 31 + H + I + E)
    layer = ek.HipLayer(H, I, E, K, act_dtype=dt, w_dtype=torch.int8, max_tokens=T, act8=True)
    ws = [weight(H, I, g) for _ in range(E)]
    for e, w in enumerate(ws):
        layer.set_expert(e, w)
    shared = None
    if shared_inter:
        shared = weight(H, shared_inter, g)
        layer.set_shared_expert(shared)
    return layer, ws, shared


def call(T, H, E, K, dt, seed=0, skew=0.0, w32=False):
    g = torch.Generator().manual_seed(seed * 977 + T)
    x = torch.randn(T, H, generator=g).to(dt)
    logits = torch.randn(T, E, generator=g) - skew * torch.log(torch.arange(E).float() + 1)
    p, ids = torch.topk(torch.softmax(logits, 1), K, dim=1)
    w = p / p.sum(1, keepdim=True)
    return x, ids.to(torch.int32), w if w32 else w.to(dt)


def same(got, want, what=""):
    got = got.cpu()
    eq = (got == want) | (got.isnan() & want.isnan())
    assert bool(eq.all()), f"{what}: {int((~eq).sum())} of {eq.numel()} elements differ, first at {tuple((~eq).nonzero()[0].tolist())}"


CASES = [  # T, H, I, E, K, skew: every class of segment (1-16, 17-32, 33-64, 65-128, longer), every chunk parity
    (1, 128, 128, 4, 2, 0.0), (2, 256, 192, 8, 8, 0.0), (7, 192, 320, 5, 3, 0.0), (64, 1024, 512, 16, 2, 0.0), (100, 320, 256, 6, 2, 1.0),
    (300, 256, 448, 3, 1, 0.5), (513, 512, 128, 12, 4, 2.0), (130, 704, 832, 2, 2, 0.0), (40, 2048, 768, 32, 8, 1.0), (3, 1088, 64, 3, 1, 0.0),
    # padded: sizes the kernels do not take as they are
    (9, 16, 8, 4, 2, 0.0), (70, 136, 100, 5, 3, 0.5), (33, 200, 51, 3, 2, 0.0)]


@pytest.mark.parametrize("T,H,I,E,K,skew", CASES)
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_layer(ek, cuda, T, H, I, E, K, skew, dt):
    layer, ws, _ = build(ek, H, I, E, K, dt, T)
    x, ids, w = call(T, H, E, K, dt, skew=skew, w32=T % 2 == 1)
    q, s = ref.quantise(x)
    want = ref.layer(q, s, ids, w, ws, dt)
    dx, dids, dw, dq, ds = x.to(cuda), ids.to(cuda), w.to(cuda), q.to(torch.int8).to(cuda), s.to(cuda)
    same(layer.forward(dx, dids, dw), want, "16-bit rows")
    same(layer.forward_q8(dq, ds, dids, dw), want, "8-bit rows")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    y = layer.forward_q8(dq, ds, dids, dw, stream=st)
    torch.cuda.synchronize()
    same(y, want, "enqueued")
    same(layer.forward(x, ids, w), want, "host memory")
    y, rt = layer.forward_q8(q.to(torch.int8), s, ids, w, return_route=True)
    same(y, want, "8-bit host memory")
    assert int(rt.counts.sum()) == T * K and torch.equal(rt.counts.long(), torch.bincount(ids.reshape(-1).long(), minlength=E))


@pytest.mark.parametrize("T", [1, 5, 64, 65, 200, 256, 300])
@pytest.mark.parametrize("wide", [1, 2])
def test_shared_expert(ek, cuda, T, wide):
    """The shared expert's segment at each of its cuts, of the routed experts' width and of twice that."""
    H, I, E, K, dt = 256, 192, 6, 3, torch.bfloat16
    layer, ws, shared = build(ek, H, I, E, K, dt, T, seed=1, shared_inter=wide * I)
    x, ids, w = call(T, H, E, K, dt, seed=1, w32=True)
    q, s = ref.quantise(x)
    want = ref.layer(q, s, ids, w, ws, dt, shared)
    same(layer.forward(x.to(cuda), ids.to(cuda), w.to(cuda)), want)
    same(layer.forward_q8(q.to(torch.int8).to(cuda), s.to(cuda), ids.to(cuda), w.to(cuda)), want)
    if T <= 65:
        same(layer.forward_static(x.to(cuda), ids.to(cuda), w.to(cuda)), want, "static")


@pytest.mark.parametrize("H,I", [(256, 192), (1024, 512), (136, 100)])
def test_per_expert_calls(ek, cuda, H, I):
    E, dt = 5, torch.bfloat16
    layer, ws, _ = build(ek, H, I, E, 1, dt, 1300, seed=2)
    g = torch.Generator().manual_seed(3)
    for n in (1, 16, 17, 33, 64, 65, 128, 129, 300, 1300):
        x = torch.randn(n, H, generator=g).to(dt)
        want = ref.expert(*ref.quantise(x), ws[n % E], dt)
        same(layer.expert_forward(n % E, x.to(cuda)), want, f"n = {n}")
        if n < 100:
            same(layer.expert_forward(n % E, x), want, f"n = {n}, host")
    rows = [1, 0, 20, 16, 70, 140, 1, 33]
    xs = [torch.randn(n, H, generator=g).to(dt) for n in rows]
    for dev in ("cpu", cuda):
        outs = layer.experts_forward([i % E for i in range(len(rows))], [x.to(dev) for x in xs])
        for i, (x, o) in enumerate(zip(xs, outs)):
            if rows[i]:
                same(o, ref.expert(*ref.quantise(x), ws[i % E], dt), f"call {i}")


def test_single_expert_object(ek, cuda):
    g = torch.Generator().manual_seed(4)
    w = weight(200, 72, g)
    op = ek.HipFFN.construct(ek.EKInstance(200, 72), w, act8=True, max_rows=64)
    x = torch.randn(40, 200, generator=g).to(torch.bfloat16)
    same(op.forward(x.to(cuda)), ref.expert(*ref.quantise(x), w, torch.bfloat16))
    same(op.forward(x), ref.expert(*ref.quantise(x), w, torch.bfloat16))


def test_wire_and_batcher(ek, cuda):
    from ek_hip import wire
    H, dt = 256, torch.bfloat16
    layer, ws, _ = build(ek, H, 128, 4, 2, dt, 64, seed=5)
    x = torch.randn(12, H, generator=torch.Generator().manual_seed(6)).to(dt)
    import safetensors.torch as st
    req = st.save({"data": x})
    want = ref.expert(*ref.quantise(x), ws[3], dt)
    same(st.load(layer.worker_forward("m/l0-e3", req))["data"], want)
    b = ek.HipBatcher(layer)
    same(st.load(b.forward("m/l0-e3", req))["data"], want)
    b.close()


def test_router_and_chain(ek, cuda):
    H, I, E, K, T, dt = 256, 192, 8, 2, 40, torch.bfloat16
    layers = [build(ek, H, I, E, K, dt, T, seed=10 + l) for l in range(3)]
    g = torch.Generator().manual_seed(8)
    x = torch.randn(T, H, generator=g).to(dt)
    logits = torch.randn(T, E, generator=g)
    y, ids, w = layers[0][0].forward_logits(x.to(cuda), logits.to(cuda), ek.RouterConfig())
    q, s = ref.quantise(x)
    same(y, ref.layer(q, s, ids.cpu(), w.cpu(), layers[0][1], dt))
    calls = [call(T, H, E, K, dt, seed=l)[1:] for l in range(3)]
    ids, w = torch.stack([c[0] for c in calls]), torch.stack([c[1] for c in calls])
    want = x
    for l in range(3):
        q, s = ref.quantise(want)
        want = ref.layer(q, s, ids[l], w[l], layers[l][1], dt)
    chain = ek.HipChain([l[0] for l in layers])
    for use_graph in (False, True, True, True):
        same(chain.forward(x.to(cuda), ids.to(cuda), w.to(cuda), use_graph=use_graph), want, f"graph {use_graph}")
    chain.close()


def test_norm_feeds_the_layer(ek, cuda):
    """The block as it is used: residual and norm -> (router on the 16-bit rows) -> experts on the 8-bit rows."""
    H, I, E, K, T, dt = 512, 256, 8, 2, 70, torch.bfloat16
    layer, ws, _ = build(ek, H, I, E, K, dt, T, seed=20)
    g = torch.Generator().manual_seed(21)
    x, r = torch.randn(T, H, generator=g).to(dt), torch.randn(T, H, generator=g).to(dt)
    gain = (1 + 0.1 * torch.randn(H, generator=g)).to(dt)
    gate = (torch.randn(E, H, generator=g) / H ** 0.5).to(dt)
    norm = ek.HipNorm(gain)
    st = torch.cuda.Stream()
    dx, dr, dgate = x.to(cuda), r.to(cuda), gate.to(cuda)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        o = norm.forward(dx, dr, stream=st)
        ids, w = layer.route((o.y.float() @ dgate.float().t()), ek.RouterConfig(), stream=st)
        y = layer.forward_q8(o.q, o.scale, ids, w, stream=st)
    torch.cuda.synchronize()
    total, _, q, _ = ref.norm(x, r, gain, 1e-6)
    assert torch.equal(o.sum.cpu(), total) and torch.equal(o.q.cpu().double(), q)
    same(y, ref.layer(q, o.scale.cpu(), ids.cpu(), w.cpu(), ws, dt))


def test_under_capture(ek, cuda):
    """A captured call is replayed on other rows and another routing, with eager calls of the same layer between."""
    H, I, E, K, T, dt = 256, 192, 8, 4, 90, torch.float16
    layer, ws, _ = build(ek, H, I, E, K, dt, T, seed=30)
    x, ids, w = call(T, H, E, K, dt, seed=0)
    dx, dids, dw = x.to(cuda), ids.to(cuda), w.to(cuda)
    y = layer.forward(dx, dids, dw)
    g, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    layer.forward(dx, dids, dw, stream=st, out=y)
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=st):
        layer.forward(dx, dids, dw, stream=st, out=y)
    for seed in (1, 2, 3):
        x, ids, w = call(T, H, E, K, dt, seed=seed, skew=float(seed))
        dx.copy_(x), dids.copy_(ids), dw.copy_(w)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        same(y, ref.layer(*ref.quantise(x), ids, w, ws, dt), f"replay {seed}")
        x2, ids2, w2 = call(11, H, E, K, dt, seed=seed + 50)
        same(layer.forward(x2.to(cuda), ids2.to(cuda), w2.to(cuda)), ref.layer(*ref.quantise(x2), ids2, w2, ws, dt), "eager")


def test_two_streams(ek, cuda):
    H, I, E, K, T, dt = 512, 256, 8, 4, 200, torch.bfloat16
    layer, _, _ = build(ek, H, I, E, K, dt, T, seed=40)
    calls = [[t.to(cuda) for t in call(T - 30 * i, H, E, K, dt, seed=i)] for i in range(6)]
    want = [layer.forward(*c) for c in calls]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [layer.forward(*c, stream=streams[i % 2]) for i, c in enumerate(calls)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_rows_that_are_not_finite_stay_alone(ek, cuda):
    H, I, E, K, T, dt = 256, 128, 4, 2, 30, torch.bfloat16
    layer, ws, _ = build(ek, H, I, E, K, dt, T, seed=50)
    x, ids, w = call(T, H, E, K, dt)
    want = ref.layer(*ref.quantise(x), ids, w, ws, dt)
    x[4, 9], x[20, 0] = float("nan"), float("inf")
    y = layer.forward(x.to(cuda), ids.to(cuda), w.to(cuda)).cpu()
    assert bool(y[[4, 20]].isnan().all())
    keep = [t for t in range(T) if t not in (4, 20)]
    same(y[keep], want[keep])
    x[4], x[20] = 0, 0                                             # a row of zeros gives a row of zeros
    y = layer.forward(x.to(cuda), ids.to(cuda), w.to(cuda)).cpu()
    assert not bool(y[[4, 20]].any())
    same(y[keep], want[keep])


def test_errors(ek, cuda):
    from ek_hip import _capi as C
    H, I, E, K, T, dt = 256, 128, 4, 2, 8, torch.bfloat16
    layer, ws, _ = build(ek, H, I, E, K, dt, T, seed=60)
    x, ids, w = (t.to(cuda) for t in call(T, H, E, K, dt))
    q, s = ref.quantise(x.cpu())
    q, s = q.to(torch.int8).to(cuda), s.to(cuda)

    def status(f):
        with pytest.raises(ek.EKError) as ei:
            f()
        return ei.value.status

    plain = ek.HipLayer(H, I, E, K, act_dtype=dt, w_dtype=torch.int8, max_tokens=T)
    assert status(lambda: plain.forward_q8(q, s, ids, w)) == C.EK_INVALID_INPUT
    assert status(lambda: layer.forward_q8(q, s[:3], ids, w)) == C.EK_INVALID_INPUT
    assert status(lambda: layer.forward_q8(q.half(), s, ids, w)) == C.EK_INVALID_INPUT
    assert status(lambda: layer.forward_q8(q[:, :128], s, ids, w)) == C.EK_INVALID_INPUT
    assert status(lambda: layer.forward_q8(q, s.cpu(), ids, w)) == C.EK_INVALID_INPUT
    for kw in (dict(w_dtype=None), dict(w_dtype=torch.float8_e4m3fn), dict(w_dtype=torch.int8, block_scales=True)):
        assert status(lambda: ek.HipLayer(H, I, E, K, act_dtype=dt, max_tokens=T, act8=True, **kw)) == C.EK_INVALID_INPUT
    assert status(lambda: ek.HipLayer(131136, 128, 1, 1, w_dtype=torch.int8, max_tokens=1, act8=True)) == C.EK_INVALID_INPUT
    bad = ids.clone()
    bad[3, 1] = E
    assert status(lambda: layer.forward(x, bad, w)) == C.EK_INVALID_INPUT
    layer.remove_expert(1)
    with_1 = ids.clone()
    with_1[0, 0] = 1
    assert status(lambda: layer.forward(x, with_1, w)) == C.EK_EXPERT_NOT_FOUND
    assert status(lambda: layer.forward_q8(q, s, with_1, w)) == C.EK_EXPERT_NOT_FOUND
    assert layer.forward_q8(q[:0], s[:0], ids[:0], w[:0]).shape == (0, H)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_every_gate_value(ek, cuda, dt):
    """Every finite value of the type as the gate's pre-activation, through the tile kernel (all at once) and the
    streaming one (a few hundred at a time): the row's scale is the value's magnitude, the code of the first column its
    sign, and an expert for each sign and exponent holds up's scale, so that the product is a normal number."""
    v = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dt)
    v = v[v.isfinite()]
    bits = v.view(torch.int16).int() & 0xffff
    frac = 7 if dt == torch.bfloat16 else 10
    eid = (bits >> frac).to(torch.int32)                              # sign and exponent field
    E, H, I = int(eid.max()) + 1, 128, 64
    mag = v.abs().float()
    experts = []
    layer = ek.HipLayer(H, I, E, 1, act_dtype=dt, w_dtype=torch.int8, max_tokens=len(v), act8=True)
    lead = {e: float(mag[eid == e].max()) for e in torch.unique(eid).tolist()}
    unit = lambda rows, cols, at: torch.zeros(rows, cols, dtype=torch.int8).index_put_((torch.tensor(0), torch.tensor(at)), torch.tensor(1, dtype=torch.int8))
    for e in range(E):
        m = lead.get(e, 1.0)
        positive = e < E // 2 and m >= 1.0
        us = 2.0 ** max(-100.0, min(120.0, (0.0 if positive else 8.0) - float(torch.tensor(m).log2().floor())))
        w = ek.ExpertWeight(up_w=unit(I, H, 1), gate_w=unit(I, H, 0), down_w=unit(H, I, 0), up_scale=torch.full((I,), us),
                            gate_scale=torch.ones(I), down_scale=torch.ones(H))
        experts.append(w)
        layer.set_expert(e, w)
    q = torch.zeros(len(v), H, dtype=torch.int8)
    q[:, 0] = torch.where(v < 0, -1, 1).to(torch.int8)
    q[:, 1] = 1
    ids, gw = eid[:, None].contiguous(), torch.ones(len(v), 1)
    want = ref.layer(q, mag, ids, gw, experts, dt)
    assert int((want[:, 0] != 0).sum()) > len(v) // 3
    args = [t.to(cuda) for t in (q, mag, ids, gw)]
    same(layer.forward_q8(*args), want, "all")
    for lo in range(0, len(v), 8192):
        part = slice(lo, lo + 300)
        same(layer.forward_q8(*[t[part].contiguous() for t in args]), want[part], "a few")
    layer.close()


def test_two_graphs(ek, cuda):
    """Two captured calls of one layer, of different sizes and so of different cuts, replayed in turn on one stream."""
    H, I, E, K, dt = 256, 192, 8, 2, torch.bfloat16
    layer, ws, _ = build(ek, H, I, E, K, dt, 700, seed=70)
    sizes = (700, 40, 1)
    data = [[t.to(cuda) for t in call(T, H, E, K, dt, seed=T)] for T in sizes]
    ys = [layer.forward(*d) for d in data]
    st, graphs = torch.cuda.Stream(), []
    torch.cuda.synchronize()
    for d, y in zip(data, ys):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            layer.forward(*d, stream=st, out=y)
        graphs.append(g)
    for rep in range(1, 4):
        fresh = [call(T, H, E, K, dt, seed=T + rep, skew=0.5 * rep) for T in sizes]
        for d, f in zip(data, fresh):
            for t, v in zip(d, f):
                t.copy_(v)
        for y in ys:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        for (x, ids, w), y in zip(fresh, ys):
            same(y, ref.layer(*ref.quantise(x), ids, w, ws, dt), f"replay {rep}, {len(x)} tokens")


def test_tensors_of_another_device_are_refused(ek, cuda):
    from ek_hip import _capi as C
    H, I, E, K, T, dt = 128, 64, 2, 1, 4, torch.bfloat16
    layer, _, _ = build(ek, H, I, E, K, dt, T, seed=80)
    x, ids, w = call(T, H, E, K, dt)
    q, s = ref.quantise(x)
    layer.cfg.device_id = 1                                        # (what the object holds; the handle is untouched)
    with pytest.raises(ek.EKError) as ei:
        layer.forward_q8(q.to(torch.int8).to(cuda), s.to(cuda), ids.to(cuda), w.to(cuda))
    assert ei.value.status == C.EK_INVALID_INPUT


@pytest.mark.parametrize("draw", range(24))
def test_drawn_layers(ek, cuda, draw):
    """Sizes, routings, types and shared experts drawn from a seed (EKSEED=n draws others)."""
    rng = random.Random(int(os.environ.get("EKSEED", "0")) * 1000 + draw)
    H = rng.choice([8 * rng.randint(1, 80), 64 * rng.randint(2, 24)])
    I = rng.choice([rng.randint(1, 300), 64 * rng.randint(2, 16)])
    E = rng.choice([1, 2, 3, 7, 16, 40])
    K, T = rng.randint(1, min(E, 8)), rng.choice([1, rng.randint(2, 70), rng.randint(60, 700), rng.randint(500, 1500)])
    dt, w32 = rng.choice([torch.bfloat16, torch.float16]), rng.random() < 0.5
    whole = H % 64 == 0 and H >= 128 and I % 64 == 0 and I >= 128        # (padded layers take a shared expert of their own width only)
    shared_inter = rng.choice([None, None, I, 64 * rng.randint(2, 6) if whole else I])
    layer, ws, shared = build(ek, H, I, E, K, dt, T, seed=draw, shared_inter=shared_inter)
    x, ids, w = call(T, H, E, K, dt, seed=draw, skew=rng.choice([0.0, 0.7, 2.0]), w32=w32)
    q, s = ref.quantise(x)
    want = ref.layer(q, s, ids, w, ws, dt, shared)
    what = f"H={H} I={I} E={E} K={K} T={T} {dt} shared={shared_inter}"
    dx, dids, dw, dq, ds = [t.to(cuda) for t in (x, ids, w, q.to(torch.int8), s)]
    same(layer.forward(dx, dids, dw), want, what)
    y, _ = layer.forward_q8(dq, ds, dids, dw, return_route=True)
    same(y, want, what + " (8-bit rows, tables)")
    e, n = rng.randrange(E), rng.randint(1, T)
    same(layer.expert_forward(e, dx[:n]), ref.expert(q[:n], s[:n], ws[e], dt), what + f" (expert {e}, {n} rows)")
