"""Cases of the operators on 8-bit activations: the RMS norm that adds the residual and quantises
(HipNorm), the int8 product with a scale per token and channel (HipLinear), and the expert layer whose
activations are 8-bit (HipLayer with act8=True).

Definitions (rnd16: rounding to the 16-bit activation type; rows are quantised to q = rint(127 v / max|v|),
ties to even, which stands for q * scale with scale = max|v| / 127; a row of zeros has scale 0):

  norm    sum = rnd16(x + residual);  v = sum * gain / sqrt(mean(sum^2) + eps);  y = rnd16(v);  q, scale of v
  linear  y = rnd16(sum_k q[n,k] w[c,k] * scale[n] * w_scale[c] + bias[c]);  16-bit rows are quantised first
  layer   per (token, expert) pair: u, g = rnd16 of the two products;  h = rnd16(u * rnd16(g / (1 + exp(-g))));
          h quantised per row;  o = rnd16 of the third product;  y = rnd16(sum_k gate[t,k] * o[t,k]), each
          product rounded to the gate weights' type when that is the 16-bit one
"""
import math
import os
import sys

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # one decoded token of the 7168-wide model, residual stream updated in the same pass
        {"name": "norm decode 1x7168", "op": "norm", "T": 1, "H": 7168, "dtype": "bf16", "residual": True},
        # a ragged batch of the 2048-wide model, first norm of a block (nothing to add yet)
        {"name": "norm ragged 259x2048", "op": "norm", "T": 259, "H": 2048, "dtype": "fp16", "residual": False},
        # a prefill chunk
        {"name": "norm prefill 8192x7168", "op": "norm", "T": 8192, "H": 7168, "dtype": "bf16", "residual": True},
        # one decoded token through a projection: weights read once, latency counts
        {"name": "linear decode 1", "op": "linear", "T": 1, "K": 7168, "N": 2048, "dtype": "bf16", "x16": False, "bias": False},
        # sizes that suit nothing, with a bias, from 16-bit rows
        {"name": "linear odd 37", "op": "linear", "T": 37, "K": 1003, "N": 2531, "dtype": "fp16", "x16": True, "bias": True},
        # a decode batch of 64 sequences through the widest matrix of a 7168 / 2048 expert
        {"name": "linear batch 64", "op": "linear", "T": 64, "K": 2048, "N": 7168, "dtype": "bf16", "x16": False, "bias": False},
        # a prefill chunk through a square-ish projection: the matrix units' case
        {"name": "linear prefill 8192", "op": "linear", "T": 8192, "K": 7168, "N": 4096, "dtype": "bf16", "x16": False, "bias": False},
        # the 64-token layer of 16 small experts
        {"name": "layer tiny 64", "op": "layer", "T": 64, "H": 1024, "I": 512, "E": 16, "top_k": 2, "dtype": "bf16", "zipf": 0.0, "x16": True, "gate32": False},
        # one decoded token: eight experts' weights
        {"name": "layer decode 1", "op": "layer", "T": 1, "H": 7168, "I": 2048, "E": 256, "top_k": 8, "dtype": "bf16", "zipf": 0.0, "x16": False, "gate32": True},
        # a decode batch: nearly every expert's weights, four rows each
        {"name": "layer decode 128", "op": "layer", "T": 128, "H": 7168, "I": 2048, "E": 256, "top_k": 8, "dtype": "bf16", "zipf": 0.0, "x16": False, "gate32": True},
        # a continuous batch (decode tokens beside prefill chunks) with hot experts, fp16
        {"name": "layer ragged 5057", "op": "layer", "T": 5057, "H": 2048, "I": 768, "E": 128, "top_k": 8, "dtype": "fp16", "zipf": 0.8, "x16": True, "gate32": False},
        # a prefill chunk of the large layer
        {"name": "layer prefill 8192", "op": "layer", "T": 8192, "H": 7168, "I": 2048, "E": 256, "top_k": 8, "dtype": "bf16", "zipf": 0.0, "x16": False, "gate32": True},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "linear", "layer"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        H = 8 * log_int(2, 1536)
        return {"op": op, "T": log_int(1, 8192), "H": H, "dtype": dtype, "residual": rng.random() < 0.6}
    if op == "linear":
        return {"op": op, "T": log_int(1, 8192), "K": log_int(48, 7168), "N": log_int(33, 4096), "dtype": dtype,
                "x16": rng.random() < 0.5, "bias": rng.random() < 0.5}
    H, I, E = 8 * log_int(8, 512), log_int(40, 2048), log_int(4, 64)
    top_k = rng.randint(1, min(E, 8))
    T = log_int(1, max(2, min(4096, int(2e11 / (H * I * top_k)))))
    return {"op": op, "T": T, "H": H, "I": I, "E": E, "top_k": top_k, "dtype": dtype, "zipf": rng.choice([0.0, 0.5, 1.0]),
            "x16": rng.random() < 0.5, "gate32": rng.random() < 0.5}


# ---- plain forms -----------------------------------------------------------------------------

def _codes(v):
    """Rows in 64 bits -> (q as numbers, max |v| per row): 127 v / max decides next to a border, so in 64 bits."""
    v = v.double()
    m = v.abs().amax(1, keepdim=True)
    q = torch.round(v * 127.0 / torch.where(m > 0, m, torch.ones_like(m)))
    return q.float(), m


def _rows8(x):
    q, m = _codes(x)
    return q, (m / 127.0).float()[:, 0]


def _norm_plain(s):
    c = s["case"]
    dt = DT[c["dtype"]]
    total = (s["x"].float() + s["residual"].float()).to(dt) if c["residual"] else s["x"]
    r = total.double()
    rstd = torch.rsqrt(r.square().mean(1, keepdim=True) + EPS)
    p = r * s["gain"].double()
    q, m = _codes(p)
    scale = (m * rstd / 127.0).float()
    out = {"y": (p * rstd).float().to(dt), "values": q * scale, "scale": scale[:, 0]}
    if c["residual"]:
        out["sum"] = total
    return out


def _linear_plain(s):
    c = s["case"]
    q, scale = _rows8(s["x"]) if c["x16"] else (s["q"].float(), s["scale"])
    y = (q @ s["w"].float().t()) * (scale[:, None] * s["w_scale"].float()[None, :])
    if c["bias"]:
        y = y + s["bias"].float()
    return y.to(DT[c["dtype"]])


def _layer_plain(s):
    c = s["case"]
    dt, T, K = DT[c["dtype"]], c["T"], c["top_k"]
    q, scale = _rows8(s["x"]) if c["x16"] else (s["q"].float(), s["scale"])
    # the pairs of each active expert as the rows of one padded block, batched products over the experts
    flat = s["ids"].long().reshape(-1)
    counts = torch.bincount(flat, minlength=c["E"])
    active = counts.nonzero()[:, 0]
    order = torch.argsort(flat, stable=True)
    slot = torch.zeros_like(counts).index_put((active,), torch.arange(active.numel(), device=flat.device))[flat[order]]
    pos = torch.arange(T * K, device=flat.device) - (counts.cumsum(0) - counts)[flat[order]]
    cap = int(counts.max())
    n = active.numel()
    X = torch.zeros(n, cap, c["H"], device=flat.device)
    X[slot, pos] = q[order // K]
    XS = torch.zeros(n, 1, cap, device=flat.device)
    XS[slot, 0, pos] = scale[order // K]
    Xt = X.transpose(1, 2).contiguous()
    del X
    u = torch.bmm(s["up"][active].float(), Xt).mul_(XS * s["up_s"][active].float()[:, :, None]).to(dt).float()
    g = torch.bmm(s["gate"][active].float(), Xt).mul_(XS * s["gate_s"][active].float()[:, :, None]).to(dt).float()
    del Xt
    h = (u * (g / (1 + torch.exp(-g))).to(dt).float()).to(dt)                 # [n, I, cap]
    del u, g
    hq, hs = _rows8(h.transpose(1, 2).reshape(n * cap, c["I"]))
    hq = hq.view(n, cap, c["I"]).transpose(1, 2).contiguous()
    o = torch.bmm(s["down"][active].float(), hq).mul_(hs.view(n, 1, cap) * s["down_s"][active].float()[:, :, None]).to(dt)
    pairs = torch.empty(T * K, c["H"], dtype=dt, device=flat.device)
    pairs[order] = o.transpose(1, 2)[slot, pos]
    prod = s["gates"].float()[:, :, None] * pairs.view(T, K, c["H"]).float()
    if not c["gate32"]:
        prod = prod.to(dt).float()
    return prod.sum(1).to(dt)


# ---- inputs -----------------------------------------------------------------------------------

def _weight(shape, g, dev):
    return torch.randint(-127, 128, shape, generator=g, device=dev, dtype=torch.int8)


def _w_scale(shape, k, g, dev):
    # products of unit-variance rows come out with a variance near one
    return ((torch.rand(shape, generator=g, device=dev) + 0.5) / (73.0 * math.sqrt(k))).to(torch.bfloat16)


def _activations(T, H, dt, g, dev):
    """Unit-variance rows with a few channels that stand out, as a residual stream has them."""
    x = torch.randn(T, H, generator=g, device=dev)
    loud = torch.rand(H, generator=g, device=dev) < 0.004
    return (x * torch.where(loud, 8.0, 1.0)).to(dt)


def prepare(case, seed):
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 1000 + 17)
    dt, op, T = DT[case["dtype"]], case["op"], case["T"]
    s = {"case": case}
    if op == "norm":
        s["x"] = _activations(T, case["H"], dt, g, dev)
        if case["residual"]:
            s["residual"] = _activations(T, case["H"], dt, g, dev)
        s["gain"] = (1.0 + 0.1 * torch.randn(case["H"], generator=g, device=dev)).to(dt)
    elif op == "linear":
        K, N = case["K"], case["N"]
        s["x"] = _activations(T, K, dt, g, dev)
        if not case["x16"]:
            q, s["scale"] = _rows8(s.pop("x"))
            s["q"] = q.to(torch.int8)
        s["w"], s["w_scale"] = _weight((N, K), g, dev), _w_scale((N,), K, g, dev)
        if case["bias"]:
            s["bias"] = torch.randn(N, generator=g, device=dev).to(dt)
    else:
        H, I, E, K = case["H"], case["I"], case["E"], case["top_k"]
        s["x"] = _activations(T, H, dt, g, dev)
        if not case["x16"]:
            q, s["scale"] = _rows8(s.pop("x"))
            s["q"] = q.to(torch.int8)
        logits = torch.randn(T, E, generator=g, device=dev)
        if case["zipf"]:
            logits = logits - case["zipf"] * torch.log(torch.randperm(E, generator=g, device=dev).float() + 1)
        p, ids = torch.topk(torch.softmax(logits, 1), K, dim=1)
        s["ids"] = ids.to(torch.int32)
        s["gates"] = (p / p.sum(1, keepdim=True)).to(torch.float32 if case["gate32"] else dt)
        s["up"], s["gate"], s["down"] = _weight((E, I, H), g, dev), _weight((E, I, H), g, dev), _weight((E, H, I), g, dev)
        s["up_s"], s["gate_s"], s["down_s"] = _w_scale((E, I), H, g, dev), _w_scale((E, I), H, g, dev), _w_scale((E, H), I, g, dev)
    if own:
        _hold(s)
    return s


def _hold(s):
    """The handles (weights laid out once), output buffers and stream that a serving program keeps."""
    pkg = os.path.join(os.getcwd(), "expert-kit_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ek_hip

    c = s["case"]
    dt, T = DT[c["dtype"]], c["T"]
    dev = torch.device("cuda:0")
    if "stream" not in _kept:
        _kept["stream"] = torch.cuda.Stream()
    s["stream"] = _kept["stream"]
    if c["op"] == "norm":
        H = c["H"]
        s["norm"] = ek_hip.HipNorm(s["gain"], eps=EPS)
        s["out"] = ek_hip.NormOut(sum=torch.empty(T, H, dtype=dt, device=dev) if c["residual"] else None,
                                  y=torch.empty(T, H, dtype=dt, device=dev), q=torch.empty(T, H, dtype=torch.int8, device=dev),
                                  scale=torch.empty(T, dtype=torch.float32, device=dev))
        s["values"] = torch.empty(T, H, dtype=torch.float32, device=dev)
    elif c["op"] == "linear":
        s["linear"] = ek_hip.HipLinear(s.pop("w"), s.pop("w_scale"), bias=s.pop("bias", None), act_dtype=dt, max_rows=T)
        s["y"] = torch.empty(T, c["N"], dtype=dt, device=dev)
    else:
        layer = ek_hip.HipLayer(c["H"], c["I"], c["E"], c["top_k"], act_dtype=dt, w_dtype=torch.int8, max_tokens=T, act8=True)
        for e in range(c["E"]):
            layer.set_expert(e, ek_hip.ExpertWeight(up_w=s["up"][e], gate_w=s["gate"][e], down_w=s["down"][e], up_scale=s["up_s"][e],
                                                    gate_scale=s["gate_s"][e], down_scale=s["down_s"][e]))
        for k in ("up", "gate", "down", "up_s", "gate_s", "down_s"):
            del s[k]
        s["layer"] = layer
        s["y"] = torch.empty(T, c["H"], dtype=dt, device=dev)


_kept = {}


def run(s):
    c = s["case"]
    if not own:
        return {"norm": _norm_plain, "linear": _linear_plain, "layer": _layer_plain}[c["op"]](s)
    if c["op"] == "norm":
        o = s["norm"].forward(s["x"], s.get("residual"), stream=s["stream"], out=s["out"])
        with torch.cuda.stream(s["stream"]):          # the 8-bit output as the values it stands for
            torch.mul(o.q, o.scale[:, None], out=s["values"])
        out = {"y": o.y, "values": s["values"], "scale": o.scale}
        if c["residual"]:
            out["sum"] = o.sum
        return out
    if c["op"] == "linear":
        if c["x16"]:
            return s["linear"].forward(s["x"], stream=s["stream"], out=s["y"])
        return s["linear"].forward(s["q"], s["scale"], stream=s["stream"], out=s["y"])
    if c["x16"]:
        return s["layer"].forward(s["x"], s["ids"], s["gates"], stream=s["stream"], out=s["y"])
    return s["layer"].forward_q8(s["q"], s["scale"], s["ids"], s["gates"], stream=s["stream"], out=s["y"])


def work(case):
    T = case["T"]
    if case["op"] == "norm":
        n = T * case["H"]
        return {"bytes": n * (2 + 2 + 1 + (4 if case["residual"] else 0)) + 2 * case["H"] + 4 * T, "flops": 10 * n}
    if case["op"] == "linear":
        K, N = case["K"], case["N"]
        return {"bytes": T * K * (2 if case["x16"] else 1) + K * N + 2 * T * N + 2 * N + 4 * T + (2 * N if case["bias"] else 0),
                "flops": 2 * T * K * N}
    H, I, E, K = case["H"], case["I"], case["E"], case["top_k"]
    # experts that T tokens reach when every expert is as likely (with hot experts: somewhat fewer)
    active = E * (1.0 - (1.0 - K / E) ** T)
    return {"bytes": active * (3 * H * I + 2 * (2 * I + H)) + T * H * (4 if case["x16"] else 3) + T * K * (8 if case["gate32"] else 6),
            "flops": 6 * T * K * H * I}


# ---- the definitions in 64 bits, apart from the forms above --------------------------------------

def _near(v, dt):
    """v (64 bits) rounded to the 16-bit type, kept in 64."""
    return v.to(dt).double()


def _quantised(v):
    """(codes, scale) of 64-bit rows by counting half steps: |q| is the number of half-integer multiples of max / 127 below |v|."""
    m = v.abs().max(dim=1).values[:, None]
    t = torch.nan_to_num(254.0 * v.abs() / m)           # twice the code's real value
    k = torch.floor((t + 1.0) / 2.0)
    k = torch.where((t == 2.0 * k - 1.0) & (torch.fmod(k, 2.0) == 1.0), k - 1.0, k)   # a tie goes to the even code
    return torch.sign(v) * k, m / 127.0


def exact(case, seed):
    was = globals()["own"]
    globals()["own"] = False
    try:
        s = prepare(case, seed)
    finally:
        globals()["own"] = was
    dt = DT[case["dtype"]]
    if case["op"] == "norm":
        r = s["x"].double()
        if case["residual"]:
            r = _near(r + s["residual"].double(), dt)
        norm = torch.sqrt(torch.einsum("th,th->t", r, r) / case["H"] + EPS)[:, None]
        gained = r * s["gain"].double()
        k, step = _quantised(gained)
        out = {"y": (gained / norm).to(dt), "values": k * step / norm, "scale": (step / norm)[:, 0]}
        if case["residual"]:
            out["sum"] = r.to(dt)
        return out
    if case["x16"]:
        k, step = _quantised(s["x"].double())
        step = step.float().double()
    else:
        k, step = s["q"].double(), s["scale"].double()[:, None]
    if case["op"] == "linear":
        y = torch.matmul(k * step, (s["w"].double() * s["w_scale"].double()[:, None]).t())
        return (y + s["bias"].double() if case["bias"] else y).to(dt)
    T, K = case["T"], case["top_k"]
    x = k * step
    y = torch.zeros(T, K, case["H"], dtype=dt, device=x.device)
    for e in torch.unique(s["ids"]).tolist():
        t, j = (s["ids"] == e).nonzero(as_tuple=True)
        rows = x[t]
        u = _near(rows @ (s["up"][e].double() * s["up_s"][e].double()[:, None]).t(), dt)
        g = _near(rows @ (s["gate"][e].double() * s["gate_s"][e].double()[:, None]).t(), dt)
        h = _near(u * _near(g * torch.sigmoid(g), dt), dt)
        hk, hstep = _quantised(h)
        o = (hk * hstep) @ (s["down"][e].double() * s["down_s"][e].double()[:, None]).t()
        y[t, j] = o.to(dt)
    total = torch.zeros(T, case["H"], dtype=torch.float64, device=x.device)
    for j in range(K):
        p = s["gates"][:, j].double()[:, None] * y[:, j].double()
        total += p if case["gate32"] else _near(p, dt)
    return total.to(dt)
