"""Delta-rule layers of recurrent language models: what is timed, and what the outputs should be.

Three operators of ``cubutterfly_b200.torch_ops``:

``qk_norm``            norms queries and keys head by head (root mean square or length) and rotates them by their
                       positions, of one axis or several, in one pass;
``gated_delta``        the gated delta rule along sequences, dense or packed one after another.  Per head, with a
                       state S of (K, V) values:  S_t = e^{g_t} S_{t-1} + k_t u_t^T  where
                       u_t = beta_t (v_t - e^{g_t} S_{t-1}^T k_t),  and  o_t = scale S_t^T q_t;
``gated_delta_step``   one token of it for a batch of requests, their states in a pool of slots.

``run`` computes a case with elementary torch operations in 32 bits, or (``own``) with the framework's operators;
``exact`` computes it in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
CHUNK = 64


def _norm(name, tokens, q_heads, k_heads, dim, dtype, *, train=False, norm="rms", rotary=0, axes=1, interleaved=False,
          weights="fp32", fused=False):
    return {"name": name, "op": "norm", "tokens": tokens, "q_heads": q_heads, "k_heads": k_heads, "dim": dim,
            "dtype": dtype, "train": train, "norm": norm, "rotary": rotary, "axes": axes, "interleaved": interleaved,
            "weights": weights, "fused": fused}


def _delta(name, batch, length, k_heads, heads, k_dim, v_dim, dtype, *, train=False, sequences=0, state=False,
           gates="same", fused=False):
    return {"name": name, "op": "delta", "batch": batch, "length": length, "k_heads": k_heads, "heads": heads,
            "k_dim": k_dim, "v_dim": v_dim, "dtype": dtype, "train": train, "sequences": sequences, "state": state,
            "gates": gates, "fused": fused}


def _step(name, batch, k_heads, heads, k_dim, v_dim, dtype, slots=0, gates="same"):
    return {"name": name, "op": "step", "batch": batch, "k_heads": k_heads, "heads": heads, "k_dim": k_dim,
            "v_dim": v_dim, "dtype": dtype, "slots": slots, "gates": gates}


def listed():
    return [
        # one token of one request ahead of attention: latency
        _norm("norm_decode", 1, 32, 8, 128, "bf16", rotary=128),
        # prefill of 16384 tokens: queries and keys are slices of one projection
        _norm("norm_prefill", 16384, 32, 8, 128, "bf16", rotary=128, fused=True),
        # a video prompt: time, height and width positions, fp16, a ragged token count, pairs side by side
        _norm("norm_video", 5003, 16, 16, 80, "fp16", rotary=72, axes=3, interleaved=True),
        # a training step ahead of the delta rule: heads brought to length one, no weights, no positions
        _norm("norm_train", 16384, 16, 16, 128, "bf16", train=True, norm="l2", weights="none"),
        # training in full precision, weights learned, part of each head rotated
        _norm("norm_train_fp32", 2048, 12, 4, 96, "fp32", train=True, rotary=48),
        # one token of one request, keys shared by two value heads each
        _step("step_one", 1, 16, 32, 128, 128, "bf16", gates="fp32"),
        # one token of 256 requests whose states are scattered over a pool
        _step("step_batch", 256, 8, 16, 128, 128, "fp16", slots=300),
        # prefill of one long prompt
        _delta("delta_prefill", 1, 16384, 16, 32, 128, 128, "bf16", gates="fp32", fused=True),
        # a training step
        _delta("delta_train", 8, 2048, 16, 16, 128, 128, "bf16", train=True),
        # training on documents packed one after another, single tokens and an empty one among them, carried states,
        # head sizes that are not round
        _delta("delta_train_packed", 1, 10007, 4, 8, 96, 80, "fp16", train=True, sequences=13, state=True),
        # a short full-precision fine-tuning step
        _delta("delta_train_fp32", 2, 257, 3, 3, 64, 64, "fp32", train=True, state=True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _dim(rng, low, high):
    n = _log_int(rng, low, high)
    return n if rng.random() < 0.3 else max(low, n // 16 * 16)


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    op = rng.choice(["norm", "norm", "delta", "delta", "step"])
    if op == "norm":
        train = rng.random() < 0.5
        dim = 2 * _dim(rng, 16, 128)
        axes = rng.choice([0, 1, 1, 3])
        k_heads = _log_int(rng, 1, 16)
        q_heads = k_heads * rng.choice([1, 2, 4])
        rotary = 0 if axes == 0 else rng.choice([dim, dim // 4 * 2])
        budget = 16384 * 40 * 128 // (2 if train else 1) // (2 if dtype == "fp32" else 1)
        tokens = max(1, min(_log_int(rng, 1, 32768), budget // (dim * (q_heads + k_heads))))
        return _norm("", tokens, q_heads, k_heads, dim, dtype, train=train, norm=rng.choice(["rms", "rms", "l2"]),
                     rotary=rotary, axes=max(axes, 1), interleaved=rng.random() < 0.3,
                     weights=rng.choice(["none", "fp32", "same"]), fused=rng.random() < 0.3)
    k_dim, v_dim = _dim(rng, 16, 128), _dim(rng, 16, 128)
    k_heads = _log_int(rng, 1, 16)
    heads = k_heads * rng.choice([1, 1, 2])
    if op == "step":
        batch = max(1, min(_log_int(rng, 1, 400), 256 * 16 // heads))
        return _step("", batch, k_heads, heads, k_dim, v_dim, dtype,
                     slots=rng.choice([0, batch + rng.randint(0, 64)]), gates=rng.choice(["same", "fp32"]))
    train = rng.random() < 0.5
    packed = rng.random() < 0.4
    batch = 1 if packed else _log_int(rng, 1, 16)
    budget = 16384 * (16 if train else 32) // (2 if dtype == "fp32" else 1)
    length = max(1, min(_log_int(rng, 1, 16384), budget // (heads * batch)))
    return _delta("", batch, length, k_heads, heads, k_dim, v_dim, dtype, train=train,
                  sequences=rng.randint(1, 24) if packed else 0, state=rng.random() < 0.5,
                  gates="same" if train else rng.choice(["same", "fp32"]), fused=rng.random() < 0.3)


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


def _prepare_norm(case, r, seed):
    tokens, hq, hk, dim, dtype = (case[k] for k in ("tokens", "q_heads", "k_heads", "dim", "dtype"))
    dtype = DTYPES[dtype]
    spread = r.uniform(dim, low=0.3, high=3.0)               # channels of different size, as a projection's are
    base = (r.normal(tokens, hq + 2 * hk if case["fused"] else hq + hk, dim) * spread).to(dtype)
    s = {"case": case, "q": base[:, :hq], "k": base[:, hq:hq + hk], "q_weight": None, "k_weight": None,
         "positions": None, "frequencies": None, "axes": None}
    if not case["fused"]:
        s["q"], s["k"] = s["q"].contiguous(), s["k"].contiguous()
    if case["weights"] != "none":
        wide = torch.float32 if case["weights"] == "fp32" else dtype
        s["q_weight"], s["k_weight"] = (r.normal(dim, scale=0.2, mean=1.0, dtype=wide) for _ in range(2))
    pairs = case["rotary"] // 2
    if pairs:
        s["frequencies"] = torch.exp(torch.arange(pairs, device="cuda") * (-math.log(1e6) / pairs))
        start = int(torch.randint(0, 100000, (1,), generator=torch.Generator().manual_seed(seed)))
        at = torch.arange(tokens, dtype=torch.int32, device="cuda")
        if case["axes"] == 1:
            s["positions"] = at + start
        else:
            # frames of 24 x 32 patches; the pairs take turns with the axes
            s["positions"] = torch.stack((at // 768 + start, at // 32 % 24 + start, at % 32 + start))
            s["axes"] = torch.arange(pairs, dtype=torch.int32, device="cuda") % 3
    if case["train"]:
        s["dq"] = r.normal(tokens, hq, dim, scale=0.3, dtype=dtype)
        s["dk"] = r.normal(tokens, hk, dim, scale=0.3, dtype=dtype)
        _leaf(s, "q", "k", "q_weight", "k_weight")
    return s


def _gates(r, shape, heads, dtype):
    """Decays between 0.8 and 0.999 a token, head by head, and write strengths over all of (0, 1)."""
    rate = r.uniform(heads, low=math.log(0.001), high=math.log(0.2)).exp()
    log_decay = -rate * torch.nn.functional.softplus(r.normal(*shape)) / math.log(2)
    return log_decay.to(dtype), torch.sigmoid(r.normal(*shape, scale=1.5)).to(dtype)


def _offsets(case, seed):
    """Document boundaries: one empty, one of a single token, the rest anywhere."""
    n, total = case["sequences"], case["length"]
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randint(0, total + 1, (max(n - 3, 0),), generator=g).tolist()
    if n >= 3:
        a = int(torch.randint(0, total, (1,), generator=g))
        cuts = sorted(cuts + [a, a + 1])
        cuts = sorted(cuts[:1] + cuts)[:n - 1]
    elif n == 2:
        cuts = [int(torch.randint(0, total + 1, (1,), generator=g))]
    return [0] + sorted(cuts) + [total]


def _unit(v):
    return v / v.square().sum(-1, keepdim=True).sqrt()


def _prepare_delta(case, r, seed):
    batch, length, hk, heads, kd, vd = (case[k] for k in ("batch", "length", "k_heads", "heads", "k_dim", "v_dim"))
    dtype = DTYPES[case["dtype"]]
    gate_type = torch.float32 if case["gates"] == "fp32" else dtype
    if case["fused"]:
        # one buffer of all three, as a convolution ahead of the layer leaves them
        base = torch.empty(batch, length, 2 * hk * kd + heads * vd, dtype=dtype, device="cuda")
        q = base[..., :hk * kd].view(batch, length, hk, kd)
        k = base[..., hk * kd:2 * hk * kd].view(batch, length, hk, kd)
        v = base[..., 2 * hk * kd:].view(batch, length, heads, vd)
        for t in (q, k):
            t.copy_(_unit(r.normal(batch, length, hk, kd)))
        v.copy_(r.normal(batch, length, heads, vd))
    else:
        q, k = (_unit(r.normal(batch, length, hk, kd)).to(dtype) for _ in range(2))
        v = r.normal(batch, length, heads, vd, dtype=dtype)
    g, beta = _gates(r, (batch, length, heads), heads, gate_type)
    s = {"case": case, "q": q, "k": k, "v": v, "g": g, "beta": beta, "offsets": None, "h0": None}
    states, s["cuts"] = batch, [b * length for b in range(batch + 1)]
    if case["sequences"]:
        s["cuts"] = _offsets(case, seed)
        s["offsets"] = torch.tensor(s["cuts"], dtype=torch.int32, device="cuda")
        states = case["sequences"]
        for name in ("q", "k", "v", "g", "beta"):
            s[name] = s[name][0]
    if case["state"]:
        s["h0"] = r.normal(states, heads, kd, vd, scale=0.3)
    if case["train"]:
        s["do"] = r.normal(*s["v"].shape, scale=0.3, dtype=dtype)
        s["dlast"] = r.normal(states, heads, kd, vd, scale=0.1)
        _leaf(s, "q", "k", "v", "g", "beta", "h0")
    return s


def _prepare_step(case, r):
    batch, hk, heads, kd, vd = (case[k] for k in ("batch", "k_heads", "heads", "k_dim", "v_dim"))
    dtype = DTYPES[case["dtype"]]
    q, k = (_unit(r.normal(batch, hk, kd)).to(dtype) for _ in range(2))
    g, beta = _gates(r, (batch, heads), heads, torch.float32 if case["gates"] == "fp32" else dtype)
    pool = case["slots"] or batch
    s = {"case": case, "q": q, "k": k, "v": r.normal(batch, heads, vd, dtype=dtype), "g": g, "beta": beta,
         "state": r.normal(pool, heads, kd, vd, scale=0.3), "next": torch.zeros(pool, heads, kd, vd, device="cuda"),
         "slots": None}
    if case["slots"]:
        s["slots"] = torch.randperm(pool, device="cuda", generator=r.generator)[:batch].to(torch.int32)
        s["rows"] = s["slots"].long()
    return s


def prepare(case, seed):
    r = _Rand(seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _prepare_norm(case, r, seed)
        return _prepare_delta(case, r, seed) if case["op"] == "delta" else _prepare_step(case, r)


# ---- the plain forms ---------------------------------------------------------------------------

def _angles(s):
    """cos and sin of every token's pairs, (tokens, 1, pairs); far positions times frequencies in 64 bits."""
    at = s["positions"] if s["axes"] is None else s["positions"][s["axes"].long()]
    at = at[:, None].double() if s["axes"] is None else at.t().double()
    angle = (at * s["frequencies"].double())[:, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _turn(v, cos, sin, case):
    """Each rotated pair (a, b) -> (a cos - b sin, b cos + a sin); the rest of a head stays."""
    part = v[..., :case["rotary"]]
    if case["interleaved"]:
        a, b = part[..., 0::2], part[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = part.chunk(2, -1)
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, v[..., case["rotary"]:]), -1)


def _plain_norm(s):
    case = s["case"]
    rms = case["norm"] == "rms"
    if case["rotary"]:
        cos, sin = _angles(s)
    outs = {}
    for name in ("q", "k"):
        x, w = s[name].float(), s[name + "_weight"]
        squares = x.square()
        inv = torch.rsqrt((squares.mean(-1, keepdim=True) if rms else squares.sum(-1, keepdim=True)) + EPS)
        n = x * inv
        y = n if w is None else n * w.float()
        outs[name] = (_turn(y, cos, sin, case) if case["rotary"] else y).to(s[name].dtype)
        if case["train"]:
            d = s["d" + name].float()
            if case["rotary"]:
                d = _turn(d, cos, -sin, case)
            if w is not None:
                outs["d_" + name + "_weight"] = (d * n).sum((0, 1)).to(w.dtype)
                d = d * w.float()
            along = (d * n).mean(-1, keepdim=True) if rms else (d * n).sum(-1, keepdim=True)
            outs["d_" + name] = (inv * (d - n * along)).to(s[name].dtype)
    return outs


def _chunks(cuts):
    """The chunks of all sequences, first chunks first: token indices (N, CHUNK) (the last row of a padded
    tensor where there is none), and for each chunk number the sequences that have it."""
    total, places, owners = cuts[-1], [], []
    longest = max(b - a for a, b in zip(cuts, cuts[1:]))
    for c in range(0, longest, CHUNK):
        owners.append([j for j in range(len(cuts) - 1) if cuts[j] + c < cuts[j + 1]])
        places += [(cuts[j] + c, cuts[j + 1]) for j in owners[-1]]
    first, last = torch.tensor(places, device="cuda").T
    at = first[:, None] + torch.arange(CHUNK, device="cuda")
    return torch.where(at < last[:, None], at, total), owners


def _gather(v, at, group=1):
    """(tokens, heads, ...) -> (N, heads * group, CHUNK, ...) in 32 bits, zeros behind a sequence's end."""
    v = torch.cat((v, torch.zeros_like(v[:1])))[at].transpose(1, 2).float()
    return v.repeat_interleave(group, 1) if group > 1 else v


def _scatter(v, at, total, dtype, group=1):
    """The reverse of _gather, heads of a group summed."""
    if group > 1:
        v = v.unflatten(1, (-1, group)).sum(2)
    out = torch.empty(total + 1, *v.shape[1:2], *v.shape[3:], device=v.device)
    out[at] = v.transpose(1, 2)
    return out[:total].to(dtype)


def _unit_inverse(n):
    """Inverse of I + n for strictly lower triangular n, from blocks of one row to the whole in doublings."""
    inv = torch.eye(CHUNK, device=n.device).expand_as(n).clone()
    size = 1
    while size < CHUNK:
        parts = CHUNK // size
        blocks = n.unflatten(-1, (parts, size)).unflatten(-3, (parts, size)).transpose(-3, -2)
        done = inv.unflatten(-1, (parts, size)).unflatten(-3, (parts, size)).transpose(-3, -2)
        diagonal = done.diagonal(dim1=-4, dim2=-3).movedim(-1, -3)
        even, odd = diagonal[..., 0::2, :, :], diagonal[..., 1::2, :, :]
        below = blocks[..., 1::2, 0::2, :, :].diagonal(dim1=-4, dim2=-3).movedim(-1, -3)
        joint = torch.cat((torch.cat((even, torch.zeros_like(even)), -1), torch.cat((-(odd @ below @ even), odd), -1)), -2)
        inv = torch.zeros_like(n)
        places = inv.unflatten(-1, (parts // 2, 2 * size)).unflatten(-3, (parts // 2, 2 * size)).transpose(-3, -2)
        places.diagonal(dim1=-4, dim2=-3).copy_(joint.movedim(-3, -1))
        size *= 2
    return inv


def _plain_delta(s):
    case = s["case"]
    heads, kd, vd = case["heads"], case["k_dim"], case["v_dim"]
    group, dtype = heads // case["k_heads"], s["q"].dtype
    scale, cuts = case["k_dim"] ** -0.5, s["cuts"]
    total, states = cuts[-1], len(cuts) - 1
    tokens = (lambda t: t) if case["sequences"] else (lambda t: t.flatten(0, 1))
    shaped = lambda t, like: t.view(like.shape)
    at, owners = _chunks(cuts)
    q, k = (_gather(tokens(s[n]), at, group) * (scale if n == "q" else 1.0) for n in ("q", "k"))
    v, g, beta = (_gather(tokens(s[n]), at) for n in ("v", "g", "beta"))
    beta = beta[..., None]
    # sums of log decays in 64 bits: their differences go into exponentials
    run_sum = g.double().cumsum(-1)
    decay = torch.exp((run_sum[..., :, None] - run_sum[..., None, :]).float().tril()).tril()
    from_start = torch.exp(run_sum.float())[..., None]
    to_end = torch.exp((run_sum[..., -1:] - run_sum).float())[..., None]
    whole = from_start[..., -1:, :]
    m = (decay * (k @ k.mT)).tril(-1)
    inverse = _unit_inverse(m * beta.mT)
    attention = decay * (q @ k.mT)
    fresh, used = inverse @ v, inverse @ (from_start * k)
    leaving = (to_end * k).mT
    now = s["h0"].clone() if s["h0"] is not None else torch.zeros(states, heads, kd, vd, device=v.device)
    before = torch.empty(len(at), heads, kd, vd, device=v.device)
    errors = torch.empty_like(v)
    spans, begin = [], 0
    for owner in owners:
        here = slice(begin, begin + len(owner))
        rows = slice(None) if len(owner) == states else torch.tensor(owner, device=v.device)
        spans.append((here, rows))
        old = now[rows]
        before[here] = old
        errors[here] = fresh[here] - used[here] @ old
        now[rows] = whole[here] * old + leaving[here] @ (beta[here] * errors[here])
        begin = here.stop
    u = beta * errors
    out = from_start * (q @ before) + attention @ u
    outs = {"o": shaped(_scatter(out, at, total, dtype), s["v"]), "final": now}
    if not case["train"]:
        return outs
    do = _gather(tokens(s["do"]), at)
    d_now = s["dlast"].clone()
    after = torch.empty_like(before)
    own_part, state_part = attention.mT @ do, (from_start * q).mT @ do
    d_u, d_errors = torch.empty_like(v), torch.empty_like(v)
    for here, rows in reversed(spans):
        old = d_now[rows]
        after[here] = old
        d_u[here] = own_part[here] + leaving[here].mT @ old
        d_errors[here] = inverse[here].mT @ (beta[here] * d_u[here])
        d_now[rows] = whole[here] * old + state_part[here] - (from_start[here] * k[here]).mT @ d_errors[here]
    d_att = do @ u.mT
    d_m = -(d_errors @ u.mT)
    a, b = decay * d_att, (decay * d_m).tril(-1)
    q_state = from_start * (do @ before.mT)
    k_state = -from_start * (d_errors @ before.mT)
    k_after = to_end * (u @ after.mT)
    outs["d_q"] = shaped(_scatter((q_state + a @ k) * scale, at, total, dtype, group), s["q"])
    outs["d_k"] = shaped(_scatter(k_state + k_after + a.mT @ q + b.mT @ k + b @ k, at, total, dtype, group), s["k"])
    outs["d_v"] = shaped(_scatter(d_errors, at, total, dtype), s["v"])
    d_beta = (errors * (d_u - m.mT @ d_errors)).sum(-1)
    outs["d_beta"] = shaped(_scatter(d_beta, at, total, s["beta"].dtype), s["beta"])
    pairs = attention * d_att + m * d_m
    kept = (k * k_after).sum(-1)
    d_sum = (q * q_state).sum(-1) + (k * k_state).sum(-1) - kept + pairs.sum(-1) - pairs.sum(-2)
    d_sum[..., -1] += kept.sum(-1) + whole[..., 0, 0] * (before * after).sum((-1, -2))
    d_g = d_sum.flip(-1).cumsum(-1).flip(-1)
    outs["d_g"] = shaped(_scatter(d_g, at, total, s["g"].dtype), s["g"])
    if s["h0"] is not None:
        outs["d_h0"] = d_now
    return outs


def _plain_step(s):
    case = s["case"]
    group = case["heads"] // case["k_heads"]
    q, k = (s[n].float().repeat_interleave(group, 1) for n in ("q", "k"))
    v, decay, beta = s["v"].float(), torch.exp(s["g"].float()), s["beta"].float()
    before = (s["state"] if s["slots"] is None else s["state"][s["rows"]]) * decay[..., None, None]
    u = beta[..., None] * (v - (before * k[..., None]).sum(-2))
    now = before + k[..., None] * u[..., None, :]
    if s["slots"] is None:
        s["next"].copy_(now)
    else:
        s["next"][s["rows"]] = now
    o = (now * q[..., None]).sum(-2) * case["k_dim"] ** -0.5
    return {"o": o.to(s["v"].dtype), "state": s["next"]}


# ---- the framework's operators -----------------------------------------------------------------

def _own_norm(s):
    from cubutterfly_b200 import torch_ops

    q, k = torch_ops.qk_norm(s["q"], s["k"], q_weight=s["q_weight"], k_weight=s["k_weight"], norm=s["case"]["norm"],
                             eps=EPS, positions=s["positions"], frequencies=s["frequencies"], axes=s["axes"],
                             interleaved=s["case"]["interleaved"])
    outs = {"q": q, "k": k}
    if s["case"]["train"]:
        names = [n for n in ("q", "k", "q_weight", "k_weight") if s[n] is not None]
        grads = torch.autograd.grad((q, k), [s[n] for n in names], (s["dq"], s["dk"]))
        outs.update(("d_" + n, g) for n, g in zip(names, grads))
    return outs


def _own_delta(s):
    from cubutterfly_b200 import torch_ops

    o, final = torch_ops.gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["h0"],
                                     offsets=s["offsets"])
    outs = {"o": o, "final": final}
    if s["case"]["train"]:
        names = [n for n in ("q", "k", "v", "g", "beta", "h0") if s[n] is not None]
        grads = torch.autograd.grad((o, final), [s[n] for n in names], (s["do"], s["dlast"]))
        outs.update(("d_" + n, g) for n, g in zip(names, grads))
    return outs


def _own_step(s):
    from cubutterfly_b200 import torch_ops

    o = torch_ops.gated_delta_step(s["state"], s["q"], s["k"], s["v"], s["g"], s["beta"], slots=s["slots"],
                                   new_state=s["next"])
    return {"o": o, "state": s["next"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "delta": _own_delta, "step": _own_step}[op](state)
    with torch.no_grad():
        return {"norm": _plain_norm, "delta": _plain_delta, "step": _plain_step}[op](state)


# ---- bytes and operations ----------------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        values = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["dim"]
        weights = 0 if case["weights"] == "none" else 2 * case["dim"] * (4 if case["weights"] == "fp32" else size)
        angles = (case["axes"] * case["tokens"] + case["rotary"] // 2) * 4 if case["rotary"] else 0
        passes = 2 + (2 if case["train"] else 0)  # q and k in and out; their gradients in and out
        return {"bytes": passes * values * size + (2 if case["train"] else 1) * weights + angles,
                "flops": (25 if case["train"] else 8) * values}
    hk, heads, kd, vd = (case[k] for k in ("k_heads", "heads", "k_dim", "v_dim"))
    gate = 4 if case["gates"] == "fp32" else size
    state = heads * kd * vd * 4
    if case["op"] == "step":
        row = (2 * hk * kd + 2 * heads * vd) * size + 2 * heads * gate
        return {"bytes": case["batch"] * (row + 2 * state), "flops": case["batch"] * heads * kd * vd * 7}
    tokens = case["batch"] * case["length"]
    states = case["sequences"] or case["batch"]
    # per token and head, state by state: decay and three products of K V values; backward a state and its gradient
    # move (two and three products) and four more give the vectors' gradients
    row = (2 * hk * kd + 2 * heads * vd) * size + 2 * heads * gate
    if not case["train"]:
        return {"bytes": tokens * row + states * state * (2 if case["state"] else 1), "flops": tokens * heads * kd * vd * 7}
    return {"bytes": tokens * 2 * row + states * state * (4 if case["state"] else 2), "flops": tokens * heads * kd * vd * 26}


# ---- 64 bits -----------------------------------------------------------------------------------

def _exact_norm(s):
    case = s["case"]
    tokens, dim, rotary = case["tokens"], case["dim"], case["rotary"]
    # the rotation as a matrix of each token and pair, on complex numbers
    if rotary:
        spots = s["positions"].double().reshape(case["axes"], tokens)
        which = torch.zeros(rotary // 2, dtype=torch.long, device="cuda") if s["axes"] is None else s["axes"].long()
        phase = spots[which].t() * s["frequencies"].double()
        spin = torch.polar(torch.ones_like(phase), phase)[:, None]
        index = torch.arange(rotary, device="cuda")
        first, second = (index[0::2], index[1::2]) if case["interleaved"] else index.chunk(2)

    def rotate(y, spin):
        z = torch.complex(y[..., first], y[..., second]) * spin
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    outs = {}
    for name in ("q", "k"):
        x = s[name].detach().double()
        w = torch.ones(dim, dtype=torch.float64, device="cuda")
        if s[name + "_weight"] is not None:
            w = s[name + "_weight"].detach().double()
        count = dim if case["norm"] == "rms" else 1
        length = torch.sqrt((x * x).sum(-1, keepdim=True) / count + EPS)
        y = x / length * w
        outs[name] = rotate(y, spin) if rotary else y
        if case["train"]:
            d = s["d" + name].double()
            if rotary:
                d = rotate(d, spin.conj())
            if s[name + "_weight"] is not None:
                outs["d_" + name + "_weight"] = (d * x / length).sum((0, 1))
            d = d * w
            outs["d_" + name] = d / length - x * (d * x).sum(-1, keepdim=True) / (count * length ** 3)
    return outs


def _token_step(state, k, v, decay, beta):
    """The state after one token, and the error that it stored; all (sequences, heads, ...)."""
    state = state * decay[..., None, None]
    error = v - torch.einsum("nhkv,nhk->nhv", state, k)
    return state + torch.einsum("nhk,nhv->nhkv", k, beta[..., None] * error), error


def _exact_delta(s):
    """Token by token over all sequences at once; shorter ones are padded with tokens that change nothing."""
    case = s["case"]
    heads, kd, vd, cuts = case["heads"], case["k_dim"], case["v_dim"], s["cuts"]
    group, scale = heads // case["k_heads"], case["k_dim"] ** -0.5
    n, longest, total = len(cuts) - 1, max(b - a for a, b in zip(cuts, cuts[1:])), cuts[-1]
    place = torch.full((longest, n), total, device="cuda")
    for j in range(n):
        place[:cuts[j + 1] - cuts[j], j] = torch.arange(cuts[j], cuts[j + 1], device="cuda")

    def along(name):
        t = s[name].detach()
        t = t if case["sequences"] else t.flatten(0, 1)
        return torch.cat((t, torch.zeros_like(t[:1])))

    def token(t, step):
        return t[place[step]].double()

    q, k, v, g, beta = (along(name) for name in ("q", "k", "v", "g", "beta"))
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    state = torch.zeros(n, heads, kd, vd, dtype=torch.float64, device="cuda")
    if s["h0"] is not None:
        state = s["h0"].detach().double()
    o = torch.zeros(total + 1, heads, vd, dtype=torch.float64, device="cuda")
    block = max(8, int(longest ** 0.5))
    marks = []
    for t in range(longest):
        if case["train"] and t % block == 0:
            marks.append(state)
        state, _ = _token_step(state, token(k, t), token(v, t), token(g, t).exp(), token(beta, t))
        o[place[t]] = torch.einsum("nhkv,nhk->nhv", state, token(q, t)) * scale
    outs = {"o": o[:total].view(s["v"].shape), "final": state}
    if not case["train"]:
        return outs
    do = along("do")
    grads = {name: torch.zeros(total + 1, *like.shape[1:], dtype=torch.float64, device="cuda")
             for name, like in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta))}
    d_state = s["dlast"].double()
    for b in reversed(range(len(marks))):
        steps = range(b * block, min((b + 1) * block, longest))
        states = [marks[b]]
        for t in steps[:-1]:
            states.append(_token_step(states[-1], token(k, t), token(v, t), token(g, t).exp(), token(beta, t))[0])
        for t in reversed(steps):
            old = states.pop()
            at, kt, qt, dot, bt = place[t], token(k, t), token(q, t), token(do, t) * scale, token(beta, t)
            decay = token(g, t).exp()
            new, error = _token_step(old, kt, token(v, t), decay, bt)
            # o = S^T q; S = D + k (beta e)^T; e = v - D^T k; D = decay old
            grads["q"][at] = torch.einsum("nhkv,nhv->nhk", new, dot)
            d_state = d_state + torch.einsum("nhk,nhv->nhkv", qt, dot)
            d_write = torch.einsum("nhkv,nhk->nhv", d_state, kt)
            d_error = bt[..., None] * d_write
            grads["beta"][at] = (d_write * error).sum(-1)
            grads["v"][at] = d_error
            decayed = old * decay[..., None, None]
            grads["k"][at] = (torch.einsum("nhkv,nhv->nhk", d_state, bt[..., None] * error)
                              - torch.einsum("nhkv,nhv->nhk", decayed, d_error))
            d_decayed = d_state - torch.einsum("nhk,nhv->nhkv", kt, d_error)
            grads["g"][at] = (d_decayed * decayed).sum((-1, -2))
            d_state = d_decayed * decay[..., None, None]
    for name, grad in grads.items():
        if name in "qk":
            grad = grad.unflatten(1, (-1, group)).sum(2)
        outs["d_" + name] = grad[:total].view(s[name].shape)
    if s["h0"] is not None:
        outs["d_h0"] = d_state
    return outs


def _exact_step(s):
    case = s["case"]
    group = case["heads"] // case["k_heads"]
    q, k, v, g, beta = (s[name].double() for name in ("q", "k", "v", "g", "beta"))
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    rows = torch.arange(case["batch"], device="cuda") if s["slots"] is None else s["rows"]
    now, _ = _token_step(s["state"][rows].double(), k, v, g.exp(), beta)
    pool = s["next"].double()
    pool[rows] = now
    return {"o": torch.einsum("nhkv,nhk->nhv", now, q) * case["k_dim"] ** -0.5, "state": pool}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "norm":
            return _exact_norm(s)
        return _exact_delta(s) if case["op"] == "delta" else _exact_step(s)
