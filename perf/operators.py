"""The block operators of a recurrent language model: what is timed, and what their outputs should be.

Three operators of ``cubutterfly_b200.torch_ops``:

``block_norm``       the boundary between two blocks: the block's output is normed, gated and added to the scaled
                     residual stream, and the sum is normed (and Hadamard-rotated) for the next block;
``gated_scan``       the gated linear recurrence h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(i_t) x_t along sequences,
                     dense or packed one after another;
``gated_scan_step``  one token of that recurrence for a batch of requests, their states in a pool of slots.

``run`` computes a case with elementary torch operations in 32 bits, or (``own``) with the framework's operators;
``exact`` computes it in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
EXPONENT = 8.0


def _norm(name, rows, dim, dtype, *, train=False, rotate=False, gate="channel", act="none", groups=1, scale="none",
          residual="same"):
    return {"name": name, "op": "norm", "rows": rows, "dim": dim, "dtype": dtype, "train": train, "rotate": rotate,
            "gate": gate, "act": act, "groups": groups, "scale": scale, "residual": residual}


def _scan(name, batch, length, dim, dtype, *, train=False, sequences=0, state=False, fused=False):
    return {"name": name, "op": "scan", "batch": batch, "length": length, "dim": dim, "dtype": dtype, "train": train,
            "sequences": sequences, "state": state, "fused": fused}


def _step(name, batch, dim, dtype, slots=0):
    return {"name": name, "op": "step", "batch": batch, "dim": dim, "dtype": dtype, "slots": slots}


def listed():
    return [
        # one token of one request between two blocks, the next projection quantised after a rotation: latency
        _norm("norm_decode", 1, 4096, "bf16", rotate=True),
        # a serving step of mixed prefill chunks; the final norm's neighbour: no gate, no rotation, ragged row count
        _norm("norm_chunk", 517, 2048, "fp16", gate="none", scale="float"),
        # prefill of 16384 tokens ahead of a quantised projection, the activation matrix of the rotation benchmark
        _norm("norm_prefill", 16384, 4096, "bf16", rotate=True),
        # a training step's block boundary, residual stream in 32 bits, output gated by a projected silu gate
        _norm("norm_train", 8192, 4096, "bf16", train=True, gate="full", act="silu", residual="fp32"),
        # training with one gate per sequence (conditioning) and a learned residual scale; rows that are not round
        _norm("norm_train_groups", 4101, 1000, "fp16", train=True, gate="group", act="sigmoid", groups=3,
              scale="vector"),
        # training in full precision with the rotation inside (rotation-aware fine-tuning)
        _norm("norm_train_fp32", 2048, 1024, "fp32", train=True, rotate=True),
        # one token of one request
        _step("step_one", 1, 4096, "bf16"),
        # one token of 256 requests whose states are scattered over a pool
        _step("step_batch", 256, 4096, "fp16", slots=300),
        # prefill of one long prompt; the three inputs are slices of one projection
        _scan("scan_prefill", 1, 16384, 4096, "bf16", fused=True),
        # a training step's recurrence
        _scan("scan_train", 8, 2048, 2048, "bf16", train=True),
        # training on documents packed one after another, single tokens and an empty one among them, carried states
        _scan("scan_train_packed", 1, 10007, 1000, "fp16", train=True, sequences=13, state=True),
        # a short full-precision fine-tuning step
        _scan("scan_train_fp32", 2, 257, 384, "fp32", train=True, state=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["norm", "norm", "scan", "scan", "step"])
    if op == "step":
        batch = _log_int(rng, 1, 400)
        return {**_step("", batch, _log_int(rng, 128, 8192), dtype,
                        slots=rng.choice([0, batch + rng.randint(0, 64)]))}
    train = rng.random() < 0.5
    budget = (8192 * 4096 if train else 16384 * 4096) // (2 if dtype == "fp32" else 1)
    if op == "norm":
        rotate = rng.random() < 0.4
        dim = 2 ** rng.randint(6, 13) if rotate else _log_int(rng, 64, 8192)
        groups = rng.randint(2, 8)
        gate = rng.choice(["none", "channel", "group", "full"])
        rows = min(_log_int(rng, 1, 16384), budget // dim)
        if gate == "group":
            rows = max(groups, rows // groups * groups)
        return _norm("", rows, dim, dtype, train=train, rotate=rotate, gate=gate,
                     act=rng.choice(["none", "sigmoid", "silu"]), groups=groups if gate == "group" else 1,
                     scale=rng.choice(["none", "float", "vector"]),
                     residual=rng.choice(["same", "fp32"]))
    budget = 8 * 2048 * 2048 // (2 if dtype == "fp32" else 1) if train else budget
    dim = _log_int(rng, 32, 4096)
    packed = rng.random() < 0.4
    batch = 1 if packed else _log_int(rng, 1, 16)
    length = max(1, min(_log_int(rng, 1, 32768), budget // (dim * batch)))
    return _scan("", batch, length, dim, dtype, train=train, sequences=rng.randint(1, 24) if packed else 0,
                 state=rng.random() < 0.5, fused=rng.random() < 0.3)


# ---- inputs ------------------------------------------------------------------------------------

class _Rand:
    def __init__(self, seed):
        self.generator = torch.Generator("cuda").manual_seed(seed)

    def normal(self, *shape, scale=1.0, mean=0.0, dtype=torch.float32):
        v = torch.randn(*shape, device="cuda", generator=self.generator)
        return v.mul_(scale).add_(mean).to(dtype)

    def uniform(self, *shape, low=0.0, high=1.0):
        return torch.rand(*shape, device="cuda", generator=self.generator).mul_(high - low).add_(low)


def _leaf(state, *names):
    for name in names:
        if torch.is_tensor(state.get(name)):
            state[name] = state[name].detach().requires_grad_()


def _prepare_norm(case, r):
    rows, dim, dtype, groups = case["rows"], case["dim"], DTYPES[case["dtype"]], case["groups"]
    shape = (groups, rows // groups, dim)
    stream = torch.float32 if case["residual"] == "fp32" else dtype
    x = r.normal(*shape)
    # the residual stream has a few channels of large magnitude
    outliers = torch.randperm(dim, device="cuda", generator=r.generator)[:(dim + 999) // 1000]
    x[..., outliers] *= 20.0
    gate_shape = {"none": None, "channel": (dim,), "group": (groups, 1, dim), "full": shape}[case["gate"]]
    s = {"case": case, "x": x.to(stream), "y": r.normal(*shape, scale=0.5, dtype=dtype),
         "pre": r.normal(dim, scale=0.1, mean=1.0), "post": r.normal(dim, scale=0.1, mean=0.5),
         "gate": None if gate_shape is None else r.normal(*gate_shape, dtype=dtype),
         "scale": {"none": 1.0, "float": 0.75, "vector": None}[case["scale"]]}
    if s["scale"] is None:
        s["scale"] = r.normal(dim, scale=0.05, mean=0.9)
    if case["train"]:
        s["dres"] = r.normal(*shape, scale=0.3, dtype=stream)
        s["du"] = r.normal(*shape, scale=0.3, dtype=dtype)
        _leaf(s, "x", "y", "pre", "post", "gate", "scale")
    return s


def _decay(r, dim):
    # decays between 0.9 and 0.999 per step where the recurrence gate is fully open
    return r.uniform(dim, low=0.9, high=0.999).log_().div_(-EXPONENT).expm1_().log_()


def _offsets(case, seed):
    """Document boundaries: one empty, one of a single token, the rest anywhere."""
    n, total = case["sequences"], case["length"]
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, total + 1, (max(n - 3, 0),), generator=g).tolist()
    if n >= 3:
        a = int(torch.randint(0, total, (1,), generator=g))
        cuts += [a, a + 1]
        cuts = sorted(cuts)
        cuts[:0] = cuts[:1]                                # an empty document after the first
        cuts = cuts[:n - 1]
    elif n == 2:
        cuts = [int(torch.randint(0, total + 1, (1,), generator=g))]
    return [0] + sorted(cuts) + [total]


def _prepare_scan(case, r, seed):
    batch, length, dim, dtype = case["batch"], case["length"], case["dim"], DTYPES[case["dtype"]]
    shape = (batch, length, dim)
    if case["fused"]:
        base = r.normal(batch, length, 3 * dim, dtype=dtype)
        x, rg, ig = base[..., :dim], base[..., dim:2 * dim], base[..., 2 * dim:]
    else:
        x, rg, ig = (r.normal(*shape, dtype=dtype) for _ in range(3))
    s = {"case": case, "x": x, "rg": rg, "ig": ig, "decay": _decay(r, dim), "offsets": None, "h0": None}
    states = batch
    if case["sequences"]:
        s["cuts"] = _offsets(case, seed)
        s["offsets"] = torch.tensor(s["cuts"], dtype=torch.int32, device="cuda")
        states = case["sequences"]
        for name in ("x", "rg", "ig"):
            s[name] = s[name][0]
    if case["state"]:
        s["h0"] = r.normal(states, dim)
    if case["train"]:
        s["dh"] = r.normal(*s["x"].shape, scale=0.3, dtype=dtype)
        s["dlast"] = r.normal(states, dim, scale=0.3)
        _leaf(s, "x", "rg", "ig", "decay", "h0")
    return s


def _prepare_step(case, r):
    batch, dim, dtype = case["batch"], case["dim"], DTYPES[case["dtype"]]
    s = {"case": case, "decay": _decay(r, dim), "slots": None,
         **{name: r.normal(batch, dim, dtype=dtype) for name in ("x", "rg", "ig")}}
    pool = case["slots"] or batch
    s["state"] = r.normal(pool, dim)
    s["next"] = torch.zeros(pool, dim, device="cuda")
    if case["slots"]:
        s["slots"] = torch.randperm(pool, device="cuda", generator=r.generator)[:batch].to(torch.int32)
        s["rows"] = s["slots"].long()
    return s


def prepare(case, seed):
    r = _Rand(seed)
    with torch.no_grad():
        if case["op"] == "norm":
            s = _prepare_norm(case, r)
        elif case["op"] == "scan":
            s = _prepare_scan(case, r, seed)
        else:
            s = _prepare_step(case, r)
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _act(g, act):
    if act == "none":
        return g, torch.ones_like(g)
    sig = torch.sigmoid(g)
    if act == "sigmoid":
        return sig, sig * (1 - sig)
    return g * sig, sig * (1 + g * (1 - sig))


def _butterflies(v):
    dim = v.shape[-1]
    half = 1
    while half < dim:
        p = v.reshape(*v.shape[:-1], dim // (2 * half), 2, half)
        a, b = p[..., 0, :], p[..., 1, :]
        v = torch.stack((a + b, a - b), dim=-2).reshape(v.shape)
        half *= 2
    return v * (1.0 / math.sqrt(dim))


def _plain_norm(s):
    case = s["case"]
    dim = case["dim"]
    x, y, pre, post = s["x"].float(), s["y"].float(), s["pre"], s["post"]
    alpha = s["scale"]
    ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    yn = y * ry
    n = yn * post
    if s["gate"] is None:
        act, slope = 1.0, None
    else:
        act, slope = _act(s["gate"].float(), case["act"])
    res = alpha * x + act * n
    rs = torch.rsqrt(res.square().mean(-1, keepdim=True) + EPS)
    sn = res * rs
    u = sn * pre
    if case["rotate"]:
        u = _butterflies(u)
    outs = {"residual": res.to(s["x"].dtype), "normed": u.to(s["y"].dtype)}
    if not case["train"]:
        return outs
    du = s["du"].float()
    if case["rotate"]:
        du = _butterflies(du)
    outs["d_pre"] = (du * sn).sum((0, 1))
    t = du * pre
    ds = s["dres"].float() + rs * (t - sn * (t * sn).mean(-1, keepdim=True))
    outs["d_x"] = (alpha * ds).to(s["x"].dtype)
    if torch.is_tensor(alpha):
        outs["d_scale"] = (ds * x).sum((0, 1))
    dn = ds * act
    outs["d_post"] = (dn * yn).sum((0, 1))
    t = dn * post
    outs["d_y"] = (ry * (t - yn * (t * yn).mean(-1, keepdim=True))).to(s["y"].dtype)
    if slope is not None:
        dg = ds * n * slope
        if case["gate"] == "channel":
            dg = dg.sum((0, 1))
        elif case["gate"] == "group":
            dg = dg.sum(1, keepdim=True)
        outs["d_gate"] = dg.to(s["gate"].dtype)
    return outs


def _coefficients(x, rg, ig, decay):
    rate = EXPONENT * torch.nn.functional.softplus(decay)
    sr, si = torch.sigmoid(rg), torch.sigmoid(ig)
    la = -rate * sr
    return sr, si, la, torch.exp(la), torch.sqrt(-torch.expm1(2 * la))


def _doubling(a, b):
    """Inclusive scan of h -> a h + b along axis 1, in log2(length) sweeps."""
    length, step = a.shape[1], 1
    while step < length:
        b = torch.cat((b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]), 1)
        if 2 * step < length:
            a = torch.cat((a[:, :step], a[:, step:] * a[:, :-step]), 1)
        step *= 2
    return b


def _plain_scan(s):
    case, dtype = s["case"], s["x"].dtype
    packed = s["offsets"] is not None
    x, rg, ig = (s[k].float() for k in ("x", "rg", "ig"))
    if packed:
        x, rg, ig = x[None], rg[None], ig[None]
    sr, si, la, a, m = _coefficients(x, rg, ig, s["decay"])
    u = m * si * x
    batch, length, dim = x.shape
    states = case["sequences"] if packed else batch
    h0 = s["h0"] if s["h0"] is not None else torch.zeros(states, dim, device=x.device)
    if packed:
        cuts = s["cuts"]
        filled = [j for j in range(states) if cuts[j + 1] > cuts[j]]
        first = torch.tensor([cuts[j] for j in filled], device=x.device)
        last = torch.tensor([cuts[j + 1] - 1 for j in filled], device=x.device)
        rows = torch.tensor(filled, device=x.device)
    else:
        first, last = torch.zeros((), dtype=torch.long, device=x.device), length - 1
    # the initial states enter with the first tokens, where the scans are cut
    cut = a.clone()
    if packed:
        cut[0, first] = 0
        u[0, first] += a[0, first] * h0[rows]
    else:
        cut[:, 0] = 0
        u[:, 0] += a[:, 0] * h0
    h = _doubling(cut, u)
    if packed:
        final = h0.clone()
        final[rows] = h[0, last]
    else:
        final = h[:, -1].clone()
    outs = {"h": (h[0] if packed else h).to(dtype), "final": final}
    if not case["train"]:
        return outs
    g = (s["dh"][None] if packed else s["dh"]).float().clone()
    if packed:
        g[0, last] += s["dlast"][rows]
    else:
        g[:, -1] += s["dlast"]
    following = torch.cat((cut[:, 1:], torch.zeros_like(cut[:, :1])), 1)
    g = _doubling(following.flip(1), g.flip(1)).flip(1)
    before = torch.cat((torch.zeros_like(h[:, :1]), h[:, :-1]), 1)
    if packed:
        before[0, first] = h0[rows]
    else:
        before[:, 0] = h0
    ratio = torch.where(la < 0, -la / torch.where(la < 0, m, 1.0), 0.0)
    e = g * (a * before * la + si * x * a * a * ratio)
    view = (lambda v: v[0]) if packed else (lambda v: v)
    outs["d_x"] = view(g * m * si).to(dtype)
    outs["d_rg"] = view(e * (1 - sr)).to(dtype)
    outs["d_ig"] = view(g * m * x * si * (1 - si)).to(dtype)
    outs["d_decay"] = e.sum((0, 1)) * torch.sigmoid(s["decay"]) / torch.nn.functional.softplus(s["decay"])
    if s["h0"] is not None:
        if packed:
            d0 = s["dlast"].clone()
            d0[rows] = a[0, first] * g[0, first]
        else:
            d0 = a[:, 0] * g[:, 0]
        outs["d_h0"] = d0
    return outs


def _plain_step(s):
    x = s["x"].float()
    _, si, _, a, m = _coefficients(x, s["rg"].float(), s["ig"].float(), s["decay"])
    before = s["state"] if s["slots"] is None else s["state"][s["rows"]]
    h = a * before + m * si * x
    if s["slots"] is None:
        s["next"].copy_(h)
    else:
        s["next"][s["rows"]] = h
    return {"h": h.to(s["x"].dtype), "state": s["next"]}


# ---- the framework's operators -----------------------------------------------------------------

def _own_norm(s):
    from cubutterfly_b200 import torch_ops

    case = s["case"]
    res, u = torch_ops.block_norm(s["x"], s["y"], pre_weight=s["pre"], post_weight=s["post"], gate=s["gate"],
                                  gate_activation=case["act"], residual_scale=s["scale"], eps=EPS,
                                  rotate=case["rotate"])
    outs = {"residual": res, "normed": u}
    if case["train"]:
        names = [k for k in ("x", "y", "pre", "post", "gate", "scale") if torch.is_tensor(s[k])]
        grads = dict(zip(names, torch.autograd.grad((res, u), [s[k] for k in names], (s["dres"], s["du"]))))
        for name in ("pre", "x", "scale", "post", "y", "gate"):
            if name in grads:
                outs["d_" + name] = grads[name]
    return outs


def _own_scan(s):
    from cubutterfly_b200 import torch_ops

    h, final = torch_ops.gated_scan(s["x"], s["rg"], s["ig"], s["decay"], exponent=EXPONENT, initial_state=s["h0"],
                                    offsets=s["offsets"])
    outs = {"h": h, "final": final}
    if s["case"]["train"]:
        names = [k for k in ("x", "rg", "ig", "decay", "h0") if s[k] is not None]
        grads = torch.autograd.grad((h, final), [s[k] for k in names], (s["dh"], s["dlast"]))
        outs.update(("d_" + k, g) for k, g in zip(names, grads))
    return outs


def _own_step(s):
    from cubutterfly_b200 import torch_ops

    h = torch_ops.gated_scan_step(s["state"], s["x"], s["rg"], s["ig"], s["decay"], exponent=EXPONENT,
                                  slots=s["slots"], new_state=s["next"])
    return {"h": h, "state": s["next"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "scan": _own_scan, "step": _own_step}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "scan": _plain_scan, "step": _plain_step}[op](state)


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "step":
        n = case["batch"] * case["dim"]
        return {"bytes": n * (4 * size + 8) + 4 * case["dim"], "flops": 20 * n}
    if case["op"] == "norm":
        n, dim = case["rows"] * case["dim"], case["dim"]
        stream = 4 if case["residual"] == "fp32" else size
        gate = {"none": 0, "channel": dim, "group": dim * case["groups"], "full": n}[case["gate"]] * size
        params = 8 * dim + (4 * dim if case["scale"] == "vector" else 0)
        moved = n * (2 * stream + 2 * size) + gate + params
        flops = n * (12 + (case["dim"].bit_length() if case["rotate"] else 0))
        if case["train"]:
            moved += n * (2 * stream + 2 * size) + gate + params
            flops += n * (24 + (case["dim"].bit_length() if case["rotate"] else 0))
        return {"bytes": moved, "flops": flops}
    n, dim = case["batch"] * case["length"] * case["dim"], case["dim"]
    states = (case["sequences"] or case["batch"]) * dim * 4
    moved = 4 * n * size + 4 * dim + states * (2 if case["state"] else 1)
    flops = 20 * n
    if case["train"]:
        moved += 4 * n * size + 4 * dim + states * (2 if case["state"] else 1)
        flops += 35 * n
    return {"bytes": moved, "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _hadamard(dim, device):
    h = torch.ones(1, 1, dtype=torch.float64, device=device)
    while h.shape[0] < dim:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(dim)


def _exact_norm(s):
    """Forward by the definition, gradients by automatic differentiation in 64 bits."""
    case = s["case"]
    t = {k: s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "y", "pre", "post", "gate", "scale")
         if torch.is_tensor(s[k])}
    alpha = t.get("scale", s["scale"])

    def rms(v):
        return v / torch.sqrt((v * v).sum(-1, keepdim=True) / case["dim"] + EPS)

    n = rms(t["y"]) * t["post"]
    if "gate" in t:
        sig = 1 / (1 + torch.exp(-t["gate"]))
        n = n * {"none": t["gate"], "sigmoid": sig, "silu": t["gate"] * sig}[case["act"]]
    res = t["x"] * alpha + n
    u = rms(res) * t["pre"]
    if case["rotate"]:
        u = u @ _hadamard(case["dim"], u.device)
    outs = {"residual": res.detach(), "normed": u.detach()}
    if case["train"]:
        names = [k for k in ("pre", "x", "scale", "post", "y", "gate") if k in t]
        grads = torch.autograd.grad((res, u), [t[k] for k in names], (s["dres"].double(), s["du"].double()))
        outs.update(("d_" + k, g) for k, g in zip(names, grads))
    return outs


def _exact_scan(s):
    """Token by token, each sequence by itself; the gradients backwards through the same recurrence."""
    case, packed = s["case"], s["offsets"] is not None
    x, rg, ig = (s[k].detach().double() for k in ("x", "rg", "ig"))
    lam = s["decay"].detach().double()
    dim, states = case["dim"], case["sequences"] or case["batch"]
    rate = EXPONENT * torch.log1p(torch.exp(lam))
    r, i = 1 / (1 + torch.exp(-rg)), 1 / (1 + torch.exp(-ig))
    a = torch.exp(-rate * r)
    keep = -torch.expm1(-2 * rate * r)
    m = torch.sqrt(keep)
    u = m * i * x
    h0 = torch.zeros(states, dim, dtype=torch.float64, device=x.device) if s["h0"] is None else s["h0"].detach().double()
    spans = [(j, s["cuts"][j], s["cuts"][j + 1]) for j in range(states)] if packed else [(slice(None), 0, case["length"])]
    at = (lambda v, t: v[t]) if packed else (lambda v, t: v[:, t])
    h, before, final = torch.empty_like(x), torch.empty_like(x), torch.empty_like(h0)
    for j, start, stop in spans:
        state = h0[j].clone()
        for t in range(start, stop):
            at(before, t).copy_(state)
            state = torch.addcmul(at(u, t), at(a, t), state)
            at(h, t).copy_(state)
        final[j] = state
    outs = {"h": h, "final": final}
    if not case["train"]:
        return outs
    g, d0 = s["dh"].double().clone(), torch.empty_like(h0)
    for j, start, stop in spans:
        back = s["dlast"].double()[j].clone()
        for t in range(stop - 1, start - 1, -1):
            at(g, t).add_(back)
            back = at(a, t) * at(g, t)
        d0[j] = back
    # d(log a)/d(r) = -rate r (1 - r);  d m/d(log a) = -a^2/m
    d_log = g * (before * a - i * x * a * a / m)
    outs["d_x"] = g * m * i
    outs["d_rg"] = d_log * -rate * r * (1 - r)
    outs["d_ig"] = g * m * x * i * (1 - i)
    d_lam = d_log * -EXPONENT * r / (1 + torch.exp(-lam))
    outs["d_decay"] = d_lam.reshape(-1, dim).sum(0)
    if s["h0"] is not None:
        outs["d_h0"] = d0
    return outs


def _exact_step(s):
    lam, x, r, i = (s[k].double() for k in ("decay", "x", "rg", "ig"))
    a = torch.exp(-EXPONENT * torch.log1p(torch.exp(lam)) / (1 + torch.exp(-r)))
    rows = slice(None) if s["slots"] is None else s["slots"].long()
    h = a * s["state"].double()[rows] + torch.sqrt((1 - a) * (1 + a)) * x / (1 + torch.exp(-i))
    state = torch.zeros_like(s["state"], dtype=torch.float64)
    state[rows] = h
    return {"h": h, "state": state}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        return _exact_norm(s)
    with torch.no_grad():
        return _exact_scan(s) if case["op"] == "scan" else _exact_step(s)
