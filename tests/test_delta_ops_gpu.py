"""The gated delta rule, its single token and the norm of queries and keys on the GPU against their definitions in 64 bits:
types, head layouts, lengths around the chunks of 64, strides, packed and empty sequences, extreme gates, values that are not
finite, gradients against the formulas and against differences.  The bounds stand in delta_reference."""
import threading

import pytest
import torch

import delta_reference as ref
import cubutterfly_b200 as cb
from cubutterfly_b200 import torch_ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, FP16, FP32]


def normal(seed, *shape, dtype=FP32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype)


def unit(t):
    return t / t.float().square().sum(-1, keepdim=True).sqrt()


# ---- gated delta rule --------------------------------------------------------------------------
def delta_case(batch, length, k_heads, heads, k_dim, v_dim, dtype, *, gates=None, cuts=None, state=False, seed=0):
    """Tensors of one call on the CPU, without the batch dimension where `cuts` are given."""
    lead = (length,) if cuts else (batch, length)
    gate_type = gates or dtype
    t = {"q": unit(normal(seed, *lead, k_heads, k_dim)).to(dtype), "k": unit(normal(seed + 1, *lead, k_heads, k_dim)).to(dtype),
         "v": normal(seed + 2, *lead, heads, v_dim, dtype=dtype),
         "g": -(normal(seed + 3, *lead, heads).abs() * 0.1).to(gate_type),
         "beta": torch.sigmoid(normal(seed + 4, *lead, heads, scale=1.5)).to(gate_type), "state": None}
    if state:
        t["state"] = normal(seed + 5, len(cuts) - 1 if cuts else batch, heads, k_dim, v_dim, scale=0.3)
    return t


def run_delta(t, cuts=None, scale=None, views=None):
    offsets = torch.tensor(cuts, dtype=torch.int32, device=t["q"].device) if cuts else None
    v = views or t
    return torch_ops.gated_delta(v["q"], v["k"], v["v"], v["g"], v["beta"], scale=scale, initial_state=v["state"],
                                 offsets=offsets)


def check_delta(t, cuts=None, *, scale=None, grads=("o", "final"), loss=None, view=lambda v: v, cancels=False):
    """Forward and backward of one case against float64 autograd.

    The gradient of a log decay is a sum of what later outputs take from the state, sum over i >= t of d_o_i . o_i and
    d_final . final, less what tokens from t on have put there themselves, the same sums again.  Where keys erase what
    was there before (`cancels`), the two are equal to many places: their own size is then what the error is relative to."""
    names = [n for n, v in t.items() if v is not None]
    dev = {n: None if v is None else view(v.cuda()).detach().requires_grad_() for n, v in t.items()}
    o, final = run_delta(dev, cuts, scale)
    exact = {n: None if v is None else v.double().requires_grad_() for n, v in t.items()}
    eo, efinal = ref.gated_delta(exact["q"], exact["k"], exact["v"], exact["g"], exact["beta"], scale=scale,
                                 initial_state=exact["state"], cuts=cuts)
    loss = ref.DELTA_LOSS[t["q"].dtype] if loss is None else loss
    assert o.dtype == t["v"].dtype and final.dtype == FP32 and o.shape == t["v"].shape
    ref.assert_close(o, eo.detach(), loss, "o")
    ref.assert_close(final, efinal.detach(), loss, "final")
    d = {"o": normal(91, *o.shape, dtype=o.dtype), "final": normal(92, *final.shape, scale=0.3)}
    outs = {"o": (o, eo), "final": (final, efinal)}
    got = torch.autograd.grad([outs[n][0] for n in grads], [dev[n] for n in names], [d[n].cuda() for n in grads])
    want = torch.autograd.grad([outs[n][1] for n in grads], [exact[n] for n in names], [d[n].double() for n in grads],
                               allow_unused=True)
    for n, a, b in zip(names, got, want):
        assert a.dtype == t[n].dtype and a.shape == t[n].shape
        b = torch.zeros_like(exact[n]) if b is None else b
        if cancels and n == "g":
            size = (d["o"].double() * eo.detach()).sum(-1).abs().sum() + (d["final"].double() * efinal.detach()).abs().sum()
            ref.assert_close(a, b, 4 * loss * float(size / b.abs().max()), "d_g")
            continue
        ref.assert_close(a, b, 4 * loss, "d_" + n)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 63, 64, 65, 128, 129, 200])
def test_gated_delta_lengths(cuda, length, dtype):
    check_delta(delta_case(2, length, 2, 2, 32, 48, dtype, state=True, seed=length))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k_dim,v_dim", [(1, 1), (3, 2), (8, 8), (16, 64), (64, 16), (63, 65), (64, 64), (65, 63), (96, 80),
                                         (100, 128), (127, 127), (128, 128), (128, 17)])
def test_gated_delta_head_sizes(cuda, k_dim, v_dim, dtype):
    check_delta(delta_case(1, 90, 1, 2, k_dim, v_dim, dtype, state=True, seed=k_dim))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k_heads,heads", [(1, 1), (1, 5), (3, 3), (2, 6)])
@pytest.mark.parametrize("gates", [None, FP32])
def test_gated_delta_heads_and_gate_types(cuda, k_heads, heads, gates, dtype):
    check_delta(delta_case(2, 70, k_heads, heads, 40, 24, dtype, gates=gates, seed=heads))


def test_gated_delta_many_chains(cuda):
    """More chains than SMs, and more chunks than CTAs fit at once."""
    check_delta(delta_case(10, 66, 16, 16, 16, 16, BF16, seed=3))


PACKINGS = [[0, 5], [0, 0, 5], [0, 1, 2, 3], [0, 64, 128, 130], [0, 63, 63, 190], [0, 130, 130, 130, 131, 200], [0, 0, 0, 1]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cuts", PACKINGS, ids=str)
@pytest.mark.parametrize("state", [False, True])
def test_gated_delta_packed(cuda, cuts, dtype, state):
    check_delta(delta_case(1, cuts[-1], 1, 2, 24, 40, dtype, cuts=cuts, state=state, seed=len(cuts)), cuts)


def test_gated_delta_packed_with_batch_dimension(cuda):
    cuts = [0, 70, 75]
    t = delta_case(1, 75, 2, 2, 16, 16, FP32, cuts=cuts)
    dev = {n: None if v is None else v.cuda() for n, v in t.items()}
    o, final = run_delta(dev, cuts)
    o4, final4 = run_delta({n: None if v is None else v[None] for n, v in dev.items()}, cuts)
    assert torch.equal(o4[0], o) and torch.equal(final4, final)


# Few long chains are cut into segments whose ends are found side by side and joined.
LONG = [(1, 1024, 1, 1, 16, 16, None), (1, 1025, 1, 2, 128, 128, None), (2, 1663, 1, 1, 100, 120, None), (1, 2111, 1, 3, 37, 65, None),
        (1, 2300, 1, 2, 64, 64, [0, 2300]), (1, 2500, 2, 2, 128, 48, [0, 0, 1151, 1152, 1152, 2399, 2500]),
        (1, 2400, 1, 1, 70, 128, [0, 64, 128, 1600, 2400, 2400])]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("batch,length,k_heads,heads,k_dim,v_dim,cuts", LONG, ids=str)
def test_gated_delta_few_long_chains(cuda, batch, length, k_heads, heads, k_dim, v_dim, cuts, state, dtype):
    t = delta_case(batch, length, k_heads, heads, k_dim, v_dim, dtype, cuts=cuts, state=state, seed=40)
    t["g"] = t["g"] * 0.02  # states reach from segment to segment
    check_delta(t, cuts)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first,last", [(1, 200), (70, 190), (700, 2500), (1300, 2431)])
def test_gated_delta_offsets_that_leave_tokens_out(cuda, first, last, dtype):
    """Tokens before the first offset and behind the last one belong to no sequence: what they hold, NaN here, goes nowhere, and
    their outputs and gradients are zero."""
    t = {n: v for n, v in delta_case(1, 2500 if last > 200 else 200, 1, 2, 64, 48, dtype, cuts=[0, 1], seed=48).items()
         if v is not None}
    exact = {n: v[first:last].double().requires_grad_() for n, v in t.items()}
    outside = torch.ones(t["q"].shape[0], dtype=torch.bool)
    outside[first:last] = False
    dev = {}
    for n, v in t.items():
        v[outside] = float("nan")
        dev[n] = v.cuda().requires_grad_()
    names = list(t)
    o, final = run_delta({**dev, "state": None}, [first, last])
    eo, efinal = ref.gated_delta(*(exact[n] for n in names), cuts=[0, last - first])
    loss = ref.DELTA_LOSS[dtype]
    ref.assert_close(o[first:last], eo.detach(), loss, "o")
    ref.assert_close(final, efinal.detach(), loss, "final")
    d_o, d_final = normal(93, *o.shape, dtype=dtype), normal(94, *final.shape, scale=0.3)
    d_o[outside] = float("nan")
    got = torch.autograd.grad([o, final], [dev[n] for n in names], [d_o.cuda(), d_final.cuda()])
    want = torch.autograd.grad([eo, efinal], [exact[n] for n in names], [d_o[first:last].double(), d_final.double()])
    assert not o[outside.cuda()].any()
    for n, x, y in zip(names, got, want):
        ref.assert_close(x[first:last], y, 4 * loss, "d_" + n)
        assert not x[outside.cuda()].any(), n


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_gated_delta_long_chain_is_causal(cuda, dtype):
    t = {n: None if v is None else v.cuda() for n, v in delta_case(1, 2300, 1, 1, 64, 64, dtype, state=True, seed=44).items()}
    o, final = run_delta(t)
    t["v"] = t["v"].clone()
    t["v"][0, 1500] = float("nan")
    bad, _ = run_delta(t)
    assert torch.equal(bad[:, :1472], o[:, :1472])  # the chunk of token 1500 begins there
    assert bad[:, 1500:].isnan().any(-1).all()


@pytest.mark.parametrize("grads", [("o",), ("final",)])
@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_gradient_of_one_output(cuda, grads, dtype):
    check_delta(delta_case(1, 80, 1, 2, 16, 24, dtype, state=True), grads=grads)


@pytest.mark.parametrize("scale", [0.0, -2.0])
def test_gated_delta_scale(cuda, scale):
    check_delta(delta_case(1, 70, 1, 1, 16, 16, BF16, state=True), scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_extreme_gates(cuda, dtype):
    """Decays of one and of nothing (-inf and the type's lowest value), betas of nothing, one and two."""
    t = delta_case(2, 150, 2, 2, 32, 32, dtype, state=True, seed=5)
    t["g"][0, 3:40] = 0
    t["g"][0, 70] = -float("inf")
    t["g"][0, 100] = torch.finfo(dtype).min
    t["g"][1, 0] = -float("inf")
    t["g"][1, 64] = -200.0
    t["beta"][0, 10:30] = 0
    t["beta"][1, 5:20] = 1
    t["beta"][1, 60:70] = 2
    dev = {n: None if v is None else v.cuda().requires_grad_() for n, v in t.items()}
    o, final = run_delta(dev)
    eo, efinal = ref.gated_delta(*(t[n].double() for n in ("q", "k", "v", "g", "beta")), initial_state=t["state"].double())
    loss = 4 * ref.DELTA_LOSS[dtype]     # an undamped state keeps its errors
    ref.assert_close(o, eo, loss, "o")
    ref.assert_close(final, efinal, loss, "final")
    (o.float().sum() + final.sum()).backward()
    # a decay that forgets everything has no gradient, and takes none from others
    finite = {n: v.double().clone().requires_grad_() for n, v in t.items()}
    lowest = finite["g"].clamp(min=-1e4)
    eo, efinal = ref.gated_delta(finite["q"], finite["k"], finite["v"], lowest, finite["beta"], initial_state=finite["state"])
    (eo.sum() + efinal.sum()).backward()
    for n in ("q", "k", "v", "beta", "state", "g"):
        want = finite[n].grad
        if n == "g":
            want = torch.where(t["g"].double() < -100, 0.0, want)
        ref.assert_close(dev[n].grad, want, 4 * loss, "d_" + n)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_repeated_keys(cuda, dtype):
    """Equal keys make the chunk's triangular system as far from the identity as it gets."""
    t = delta_case(1, 140, 1, 1, 32, 32, dtype, seed=8)
    t["k"][:] = t["k"][:, :1]
    t["beta"][:] = 1
    t["g"][:] = 0
    check_delta(t, loss=4 * ref.DELTA_LOSS[dtype], cancels=True)
    t["k"][:, 30:60] = 0
    check_delta(t, loss=4 * ref.DELTA_LOSS[dtype], cancels=True)


@pytest.mark.parametrize("dtype,size", [(BF16, 1e30), (BF16, 1e-30), (FP16, 2000.0), (FP16, 1e-4), (FP32, 1e30), (FP32, 1e-30)])
def test_gated_delta_magnitudes(cuda, dtype, size):
    t = delta_case(1, 100, 1, 1, 16, 16, dtype, seed=9)
    t["v"] = (t["v"].float() * size).to(dtype)
    o, final = run_delta({n: None if v is None else v.cuda() for n, v in t.items()})
    eo, efinal = ref.gated_delta(*(t[n].double() for n in ("q", "k", "v", "g", "beta")))
    ref.assert_close(o, eo, ref.DELTA_LOSS[dtype], "o")
    ref.assert_close(final, efinal, ref.DELTA_LOSS[dtype], "final")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_gated_delta_sequences_do_not_mix(cuda, bad, dtype):
    cuts = [0, 70, 75, 75, 150]
    t = delta_case(1, 150, 1, 2, 24, 24, dtype, cuts=cuts, state=True, seed=4)
    dev = {n: v.cuda() for n, v in t.items()}
    results = []
    for spoil in (False, True):
        leaves = {n: v.clone() for n, v in dev.items()}
        if spoil:
            for n in ("q", "k", "v", "g", "beta"):
                leaves[n][72:74] = bad
            leaves["state"][1:3] = bad
        leaves = {n: v.requires_grad_() for n, v in leaves.items()}
        o, final = run_delta(leaves, cuts)
        grads = torch.autograd.grad((o, final), list(leaves.values()), (torch.ones_like(o), torch.ones_like(final)))
        results.append([o.detach(), final.detach(), *grads])
    keep = torch.ones(150, dtype=torch.bool, device="cuda")
    keep[70:75] = False
    rows = torch.tensor([0, 3], device="cuda")
    for n, (a, b) in enumerate(zip(*results)):
        a, b = (a[rows], b[rows]) if a.shape[0] == 4 else (a[keep], b[keep])
        assert torch.equal(a, b), n
    assert not torch.isfinite(results[1][0][73]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k_dim,v_dim", [(16, 16), (17, 33), (128, 128)])
def test_gated_delta_strided_inputs(cuda, k_dim, v_dim, dtype):
    """Slices of one projection, heads before tokens, one more value a row, and channels that are not adjacent."""
    t = delta_case(2, 70, 2, 4, k_dim, v_dim, dtype, state=True, seed=6)

    def sliced(v):
        return torch.cat((v, torch.full_like(v[..., :3], 7.0)), -1)[..., :v.shape[-1]]

    def odd(v):
        return torch.cat((torch.full_like(v[..., :1], 7.0), v), -1)[..., 1:]

    for view in (sliced, odd, lambda v: v.transpose(1, 2).contiguous().transpose(1, 2),
                 lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2)):
        check_delta(t, view=lambda v: view(v) if v.ndim > 2 else v)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_broadcast_inputs(cuda, dtype):
    """One key for all tokens, one gate for all heads, a gradient of a sum: strides of zero."""
    t = delta_case(2, 70, 2, 2, 16, 16, dtype, seed=7)
    small = {"q": t["q"][:, :1], "k": t["k"][:1, :, :1], "v": t["v"][..., :1], "g": t["g"][:, :, :1], "beta": t["beta"][:, :1]}
    dev = {n: v.cuda().requires_grad_() for n, v in small.items()}
    exact = {n: v.double().requires_grad_() for n, v in small.items()}
    wide = lambda s: {n: v.expand(t[n].shape) for n, v in s.items()}
    o, final = run_delta({**wide(dev), "state": None})
    w = wide(exact)
    eo, efinal = ref.gated_delta(w["q"], w["k"], w["v"], w["g"], w["beta"])
    loss = ref.DELTA_LOSS[dtype]
    ref.assert_close(o, eo.detach(), loss, "o")
    (o.sum(dim=1).float().sum() + final.sum()).backward()
    (eo.sum() + efinal.sum()).backward()
    for n in small:
        # torch adds the copies' gradients in the tensor's own type: a rounding each, relative to the largest sum
        added = 70 * 2 * {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}[dtype]
        ref.assert_close(dev[n].grad, exact[n].grad, 8 * loss + added, "d_" + n)


def test_gated_delta_no_tokens(cuda):
    for dtype in TYPES:
        for batch, length in ((0, 5), (3, 0)):
            t = {n: None if v is None else v.cuda().requires_grad_()
                 for n, v in delta_case(batch, length, 1, 2, 8, 8, dtype, state=True).items()}
            o, final = run_delta(t)
            assert o.shape == t["v"].shape and torch.equal(final, t["state"])
            grads = torch.autograd.grad((o, final), list(t.values()), (torch.ones_like(o), 2 * torch.ones_like(final)))
            assert all(torch.equal(g, torch.zeros_like(g)) for g in grads[:-1]) and (grads[-1] == 2).all()
    empty = {n: v.cuda() for n, v in delta_case(1, 0, 1, 1, 8, 8, BF16, cuts=[0, 0, 0], state=True).items()}
    o, final = run_delta(empty, [0, 0, 0])
    assert o.numel() == 0 and torch.equal(final, empty["state"])


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_carried_over_calls(cuda, dtype):
    """A sequence in two calls is the sequence in one, to what rounding the pieces at other places changes."""
    t = {n: None if v is None else v.cuda() for n, v in delta_case(1, 150, 1, 2, 32, 32, dtype, seed=2).items()}
    o, final = run_delta(t)
    state, parts = None, []
    for a, b in ((0, 37), (37, 101), (101, 150)):
        part, state = run_delta({n: state if n == "state" else v[:, a:b] for n, v in t.items()})
        parts.append(part)
    eo, efinal = ref.gated_delta(*(t[n].double().cpu() for n in ("q", "k", "v", "g", "beta")))
    for a, b in ((o, final), (torch.cat(parts, 1), state)):
        ref.assert_close(a, eo, ref.DELTA_LOSS[dtype], "o")
        ref.assert_close(b, efinal, ref.DELTA_LOSS[dtype], "state")


@pytest.mark.parametrize("packed", [False, True])
def test_gated_delta_gradient_against_differences(cuda, packed):
    cuts = [0, 40, 70] if packed else None
    t = {n: v.cuda() for n, v in delta_case(1, 70, 1, 2, 8, 8, FP32, cuts=cuts, state=True, seed=11).items()}
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}

    def value(s):
        o, final = run_delta(s, cuts)
        return (o.double() * probe_o).sum() + (final.double() * probe_s).sum()

    probe_o, probe_s = normal(1, *t["v"].shape).cuda().double(), normal(2, *t["state"].shape).cuda().double()
    value(leaves).backward()
    for n, leaf in leaves.items():
        way = normal(3, *leaf.shape).cuda()
        step = 2.0 ** -7
        with torch.no_grad():
            up, down = (value({**t, n: t[n] + s * step * way}) for s in (1, -1))
        along = float((leaf.grad.double() * way.double()).sum())
        # the third derivative's step^2 and fp32 values of size about 100 over the step
        size = float(leaf.grad.double().norm() * way.double().norm())
        assert abs(float(up - down) / (2 * step) - along) <= 2e-3 * size + 0.05, n


def test_gated_delta_repeats_bit_for_bit(cuda):
    for dtype in TYPES:
        t = {n: None if v is None else v.cuda().requires_grad_()
             for n, v in delta_case(3, 130, 2, 4, 48, 80, dtype, state=True).items()}
        runs = []
        for _ in range(3):
            o, final = run_delta(t)
            runs.append([o, final, *torch.autograd.grad((o, final), list(t.values()), (torch.ones_like(o), torch.ones_like(final)))])
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_gated_delta_offsets_beyond_32_bits(cuda):
    """Tokens 2^24 + 8 values apart: the last ones lie beyond 2^31 values."""
    step, length = (1 << 24) + 8, 140
    base = torch.empty(step * length, dtype=BF16, device="cuda")
    t = delta_case(1, length, 1, 1, 16, 16, BF16, seed=12)
    dev = {n: None if v is None else v.cuda() for n, v in t.items()}
    want = run_delta(dev)
    far = dict(dev)
    for i, n in enumerate(("q", "k", "v")):
        far[n] = base[16 * i:].as_strided((1, length, 1, 16), (step * length, step, 16, 1))
        far[n].copy_(dev[n])
    for a, b in zip(run_delta(far), want):
        assert torch.equal(a, b)


def test_gated_delta_in_a_graph_and_on_side_streams(cuda):
    """Captured and replayed on new inputs; two streams at once."""
    t = {n: None if v is None else v.cuda() for n, v in delta_case(2, 130, 2, 2, 64, 64, BF16, state=True).items()}
    leaves = {n: v.clone().requires_grad_() for n, v in t.items()}

    def call(s):
        o, final = run_delta(s)
        return [o, final, *torch.autograd.grad((o, final), list(s.values()), (torch.ones_like(o), torch.ones_like(final)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call(leaves)
    with torch.no_grad():
        leaves["v"].mul_(0.5)
    graph.replay()
    other = {n: v.detach().clone().requires_grad_() for n, v in leaves.items()}
    want = call(other)
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
    streams, results = [torch.cuda.Stream() for _ in range(2)], [None, None]
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            results[i] = [call(other) for _ in range(3)][-1]
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_gated_delta_backward_from_several_threads(cuda):
    t = {n: v.cuda().requires_grad_() for n, v in delta_case(1, 100, 1, 1, 16, 16, BF16, state=True).items()}
    o, final = run_delta(t)
    want = torch.autograd.grad(o, list(t.values()), torch.ones_like(o), retain_graph=True)
    results = [None] * 4

    def work(i):
        results[i] = torch.autograd.grad(o, list(t.values()), torch.ones_like(o), retain_graph=True)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [x.start() for x in threads], [x.join() for x in threads]
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, want))


def test_gated_delta_differentiable_once_and_only_asked_gradients(cuda):
    t = {n: None if v is None else v.cuda() for n, v in delta_case(1, 20, 1, 1, 8, 8, FP32).items()}
    v = t["v"].requires_grad_()
    o, _ = run_delta(t)
    (first,) = torch.autograd.grad(o, v, torch.ones_like(o), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice through gated_delta"):
        first.sum().backward()
    o, final = run_delta(t)
    final.sum().backward()
    assert v.grad is not None and t["q"].grad is None


# ---- one token ---------------------------------------------------------------------------------
def step_case(batch, k_heads, heads, k_dim, v_dim, dtype, pool, seed=0, gates=None):
    t = {n: None if v is None else v[:, 0] for n, v in delta_case(batch, 1, k_heads, heads, k_dim, v_dim, dtype, gates=gates,
                                                                  seed=seed).items()}
    t["state"] = normal(seed + 9, pool, heads, k_dim, v_dim, scale=0.5)
    return t


def check_step(t, slots=None, view=lambda v: v):
    batch, pool = t["q"].shape[0], t["state"].shape[0]
    dev = {n: v.cuda() for n, v in t.items()}
    rows = list(range(batch)) if slots is None else slots
    keep = [b for b in range(batch) if 0 <= rows[b] < pool]
    d = {n: v.double() for n, v in t.items()}
    eo = torch.zeros(batch, *t["v"].shape[1:], dtype=torch.float64)
    estate = d["state"].clone()
    if keep:
        at = [rows[b] for b in keep]
        part, new = ref.gated_delta(*(d[n][keep][:, None] for n in ("q", "k", "v", "g", "beta")), initial_state=d["state"][at])
        eo[keep], estate[at] = part[:, 0], new
    index = None if slots is None else torch.tensor(slots, dtype=torch.int32, device="cuda")
    args = [view(dev[n]) for n in ("q", "k", "v", "g", "beta")]
    for inplace in (False, True):
        state = dev["state"].clone()
        new = None if inplace else state.clone()
        o = torch_ops.gated_delta_step(state, *args, slots=index, new_state=new)
        got = state if inplace else new
        ref.assert_close(o, eo, ref.STEP_LOSS, "o")
        ref.assert_close(got, estate, ref.STEP_LOSS, "state")
        idle = [s for s in range(pool) if s not in [rows[b] for b in keep]]
        assert torch.equal(got[idle], dev["state"][idle])
        if not inplace:
            assert torch.equal(state, dev["state"])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k_dim,v_dim", [(1, 1), (3, 5), (16, 16), (64, 32), (65, 33), (100, 36), (128, 128), (127, 126)])
def test_gated_delta_step_sizes(cuda, k_dim, v_dim, dtype):
    check_step(step_case(3, 2, 4, k_dim, v_dim, dtype, 3, seed=k_dim))


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_step_slots_and_padding(cuda, dtype):
    check_step(step_case(6, 1, 3, 32, 24, dtype, 9, gates=FP32), slots=[7, -1, 0, 9, 3, 2 ** 31 - 1])
    check_step(step_case(2, 1, 1, 16, 16, dtype, 4), slots=[-5, 4])


def test_gated_delta_step_strides(cuda):
    t = step_case(4, 2, 2, 24, 20, BF16, 4)
    check_step(t, view=lambda v: torch.cat((v, torch.zeros_like(v)), -1)[..., :v.shape[-1]])
    check_step(t, view=lambda v: v.transpose(0, 1).contiguous().transpose(0, 1))
    # a pool whose rows of states begin 4 bytes off a 16-byte boundary
    dev = {n: v.cuda() for n, v in t.items()}
    odd = torch.empty(dev["state"].numel() + 1, device="cuda")[1:].view_as(dev["state"])
    odd.copy_(dev["state"])
    args = [dev[n] for n in ("q", "k", "v", "g", "beta")]
    a, b = torch_ops.gated_delta_step(odd, *args), torch_ops.gated_delta_step(dev["state"], *args)
    assert torch.equal(a, b) and torch.equal(odd, dev["state"])


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_delta_steps_follow_the_sequence(cuda, dtype):
    t = {n: v.cuda() for n, v in delta_case(2, 70, 1, 2, 32, 32, dtype, state=True).items()}
    o, final = run_delta(t)
    state = t["state"].clone()
    rows = [torch_ops.gated_delta_step(state, *(t[n][:, i] for n in ("q", "k", "v", "g", "beta"))) for i in range(70)]
    loss = ref.DELTA_LOSS[dtype] + 70 * 2.0 ** -24
    ref.assert_close(torch.stack(rows, 1), o.double(), loss + {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 0.0}[dtype], "o")
    ref.assert_close(state, final.double(), loss, "state")


def test_gated_delta_step_beyond_32_bits(cuda):
    """A pool of more than 2^31 values, its last slot used."""
    pool = (1 << 31) // (128 * 128 * 4) + 2
    state = torch.empty(pool, 4, 128, 128, device="cuda")
    t = {n: v.cuda() for n, v in step_case(1, 4, 4, 128, 128, BF16, 1).items()}
    state[-1] = t["state"][0]
    args = [t[n] for n in ("q", "k", "v", "g", "beta")]
    o = torch_ops.gated_delta_step(state, *args, slots=torch.tensor([pool - 1], dtype=torch.int32, device="cuda"))
    want = torch_ops.gated_delta_step(t["state"], *args)
    assert torch.equal(o, want) and torch.equal(state[-1], t["state"][0])


def test_gated_delta_step_marks_its_writes_and_is_inference_only(cuda):
    t = {n: v.cuda() for n, v in step_case(1, 1, 1, 8, 8, BF16, 1).items()}
    args = [t[n] for n in ("q", "k", "v", "g", "beta")]
    version = t["state"]._version
    torch_ops.gated_delta_step(t["state"], *args)
    assert t["state"]._version == version + 1
    for n in range(5):
        with pytest.raises(ValueError, match="inference only"):
            torch_ops.gated_delta_step(t["state"], *(a.clone().requires_grad_() if i == n else a for i, a in enumerate(args)))
    with torch.no_grad():
        torch_ops.gated_delta_step(t["state"], args[0].clone().requires_grad_(), *args[1:])


# ---- norm of queries and keys ------------------------------------------------------------------
def qk_case(lead, q_heads, k_heads, dim, dtype, weights=FP32, seed=0):
    return {"q": normal(seed, *lead, q_heads, dim, dtype=dtype), "k": normal(seed + 1, *lead, k_heads, dim, scale=3.0, dtype=dtype),
            "q_weight": None if weights is None else normal(seed + 2, dim, dtype=weights, scale=0.2, mean=1.0),
            "k_weight": None if weights is None else normal(seed + 3, dim, dtype=weights, scale=0.2, mean=-1.0)}


def check_qk(t, *, norm="rms", eps=1e-6, positions=None, frequencies=None, axes=None, interleaved=False, view=lambda v: v,
             grads=("q", "k")):
    names = [n for n, v in t.items() if v is not None]
    dev = {n: None if v is None else (view(v.cuda()) if v.ndim > 1 else v.cuda()).detach().requires_grad_() for n, v in t.items()}
    turn = {"positions": positions, "frequencies": frequencies, "axes": axes}
    q, k = torch_ops.qk_norm(dev["q"], dev["k"], q_weight=dev["q_weight"], k_weight=dev["k_weight"], norm=norm, eps=eps,
                             interleaved=interleaved, **{n: None if v is None else v.cuda() for n, v in turn.items()})
    exact = {n: None if v is None else v.double().requires_grad_() for n, v in t.items()}
    out = {"q": q, "k": k}
    want = {n: ref.qk_norm(exact[n], exact[n + "_weight"], norm=norm, eps=eps, interleaved=interleaved, **turn) for n in "qk"}
    for n in "qk":
        assert out[n].dtype == t[n].dtype
        ref.assert_close(out[n], want[n].detach(), ref.NORM_LOSS, n)
    d = {n: normal(50 + i, *t[n].shape, dtype=t[n].dtype) for i, n in enumerate("qk")}
    got = torch.autograd.grad([out[n] for n in grads], [dev[n] for n in names], [d[n].cuda() for n in grads], allow_unused=True)
    exp = torch.autograd.grad([want[n] for n in grads], [exact[n] for n in names], [d[n].double() for n in grads],
                              allow_unused=True)
    rows = max(1, t["q"].numel() // t["q"].shape[-1])
    for n, a, b in zip(names, got, exp):
        assert a.dtype == t[n].dtype
        b = torch.zeros_like(exact[n]) if b is None else b
        loss = ref.NORM_LOSS * rows ** 0.5
        if n in ("q", "k"):
            # r t less r n mean(t n), which for few channels are nearly equal: the error is relative to their size, at
            # most r |weight| |d| (turned, so up to sqrt(2) of it)
            x = exact[n].detach()
            r = 1 / torch.sqrt(x.square().mean(-1) + eps if norm == "rms" else x.square().sum(-1) + eps)
            w = 1.0 if t[n + "_weight"] is None else float(t[n + "_weight"].abs().max())
            size = float((r * d[n].double().abs().amax(-1)).max()) * w * 2 ** 0.5 if r.numel() else 0.0
            loss = 4 * ref.NORM_LOSS * max(1.0, size / max(float(b.abs().max()) if b.numel() else 1.0, 1e-300))
        ref.assert_close(a, b, loss, "d_" + n)


def rotary(tokens, pairs, seed=0, far=1 << 20):
    g = torch.Generator().manual_seed(seed)
    return {"positions": torch.randint(0, far, tokens, generator=g, dtype=torch.int32),
            "frequencies": torch.exp(torch.arange(pairs) * (-9.2 / max(1, pairs)))}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 16, 31, 32, 64, 80, 96, 127, 128, 130, 200, 256])
@pytest.mark.parametrize("norm", ["rms", "l2"])
def test_qk_norm_sizes(cuda, dim, norm, dtype):
    check_qk(qk_case((2, 9), 3, 2, dim, dtype, seed=dim), norm=norm)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(2, 2), (16, 16), (24, 8), (64, 64), (72, 50), (80, 72), (96, 48), (128, 128), (129, 64),
                                         (255, 254), (256, 256)])
def test_qk_norm_rotation(cuda, dim, rotated, interleaved, dtype):
    check_qk(qk_case((11,), 2, 1, dim, dtype, seed=dim), interleaved=interleaved, **rotary((11,), rotated // 2, seed=dim))


@pytest.mark.parametrize("weights", [None, "same", FP32])
@pytest.mark.parametrize("dtype", TYPES)
def test_qk_norm_weights(cuda, weights, dtype):
    check_qk(qk_case((700,), 4, 2, 64, dtype, dtype if weights == "same" else weights), **rotary((700,), 32))


def test_qk_norm_one_weight(cuda):
    t = qk_case((5,), 2, 2, 32, BF16)
    for drop in ("q_weight", "k_weight"):
        check_qk({**t, drop: None}, **rotary((5,), 8))


@pytest.mark.parametrize("lead,at", [((3, 5), (5,)), ((3, 5), (3, 5)), ((2, 3, 5), (5,)), ((2, 3, 5), (3, 5)), ((7,), (7,))])
@pytest.mark.parametrize("wide", [False, True])
def test_qk_norm_positions(cuda, lead, at, wide):
    turn = rotary(at, 8)
    if wide:
        turn["positions"] = turn["positions"].long() - 1000     # negative ones too
    check_qk(qk_case(lead, 2, 3, 24, FP32), **turn)


@pytest.mark.parametrize("axes", [1, 3])
@pytest.mark.parametrize("dtype", TYPES)
def test_qk_norm_axes(cuda, axes, dtype):
    turn = rotary((axes, 4, 6), 20)
    turn["axes"] = (torch.arange(20) % axes).int()
    check_qk(qk_case((4, 6), 2, 2, 48, dtype), **turn)


def test_qk_norm_far_positions(cuda):
    """Angles of positions up to 2^31 - 1 keep every bit that the frequencies have."""
    turn = rotary((64,), 16, far=2 ** 31 - 1)
    turn["positions"][:4] = torch.tensor([2 ** 31 - 1, 2 ** 31 - 2, 0, 1])
    check_qk(qk_case((64,), 1, 1, 32, FP32), **turn)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [16, 33, 128])
def test_qk_norm_strided_inputs(cuda, dim, dtype):
    t = qk_case((3, 6), 4, 2, dim, dtype)
    turn = rotary((6,), dim // 4)
    for view in (lambda v: torch.cat((v, v + 1), -2)[..., :v.shape[-2], :], lambda v: torch.cat((v, v), -1)[..., :dim],
                 lambda v: v.transpose(0, 1).contiguous().transpose(0, 1), lambda v: v.transpose(-1, -2).contiguous().transpose(-1, -2)):
        check_qk(t, view=view, **turn)


def test_qk_norm_broadcast_heads(cuda):
    """One head expanded to several, and the gradient of a sum over them."""
    x = normal(1, 5, 1, 32).cuda().requires_grad_()
    q, k = torch_ops.qk_norm(x.expand(5, 4, 32), x.expand(5, 2, 32))
    (q.sum(1).square().sum() + k.sum(0).square().sum()).backward()
    e = x.detach().double().cpu().requires_grad_()
    n = ref.qk_norm(e)
    ((4 * n[:, 0]).square().sum() + n.expand(5, 2, 32).sum(0).square().sum()).backward()
    ref.assert_close(x.grad, e.grad, 64 * ref.NORM_LOSS, "d_x")


@pytest.mark.parametrize("tokens,heads", [(1, 40), (2, 1), (149, 3), (3000, 5)])
def test_qk_norm_shares_of_work(cuda, tokens, heads):
    check_qk(qk_case((tokens,), heads, 1, 64, BF16, None), **rotary((tokens,), 32))


@pytest.mark.parametrize("grads", [("q",), ("k",)])
def test_qk_norm_gradient_of_one_output(cuda, grads):
    check_qk(qk_case((6,), 2, 2, 16, FP32), grads=grads)


def test_qk_norm_zero_and_unusual_rows(cuda):
    """Rows of zeros stay zero with eps, rows do not mix, no tokens are no work."""
    t = qk_case((8,), 2, 2, 32, BF16)
    t["q"][3] = 0
    check_qk(t, norm="l2")
    dev = {n: v.cuda() for n, v in t.items()}
    clean = torch_ops.qk_norm(dev["q"], dev["k"], q_weight=dev["q_weight"])
    dev["q"][5, 1] = float("nan")
    dev["k"][2, 0, 3] = float("inf")
    spoiled = torch_ops.qk_norm(dev["q"], dev["k"], q_weight=dev["q_weight"])
    for a, b, at in zip(clean, spoiled, ((5, 1), (2, 0))):
        same = torch.ones(8, 2, dtype=torch.bool, device="cuda")
        same[at] = False
        assert torch.equal(a[same], b[same]) and torch.isnan(b[at]).any()
    for lead in ((0,), (0, 3), (3, 0)):
        e = {n: v.cuda().requires_grad_() for n, v in qk_case(lead, 2, 1, 16, FP16).items()}
        q, k = torch_ops.qk_norm(e["q"], e["k"], q_weight=e["q_weight"], k_weight=e["k_weight"])
        g = torch.autograd.grad((q, k), list(e.values()), (torch.ones_like(q), torch.ones_like(k)))
        assert q.shape == e["q"].shape and all((x == 0).all() for x in g)


def test_qk_norm_beyond_32_bits(cuda):
    step = (1 << 27) + 8
    base = torch.empty(step * 20, dtype=BF16, device="cuda")
    t = {n: None if v is None else v.cuda() for n, v in qk_case((20,), 1, 1, 64, BF16).items()}
    want = torch_ops.qk_norm(t["q"], t["k"])
    far = []
    for i, n in enumerate("qk"):
        far.append(base[64 * i:].as_strided((20, 1, 64), (step, 64, 1)))
        far[-1].copy_(t[n])
    assert all(torch.equal(a, b) for a, b in zip(torch_ops.qk_norm(*far), want))


def test_qk_norm_repeats_and_in_a_graph(cuda):
    t = {n: v.cuda().requires_grad_() for n, v in qk_case((1000,), 3, 2, 48, BF16).items()}
    turn = {n: v.cuda() for n, v in rotary((1000,), 24).items()}

    def call():
        q, k = torch_ops.qk_norm(t["q"], t["k"], q_weight=t["q_weight"], k_weight=t["k_weight"], **turn)
        return [q, k, *torch.autograd.grad((q, k), list(t.values()), (torch.ones_like(q), torch.ones_like(k)))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(call(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))


def test_qk_norm_differentiable_once(cuda):
    q = normal(1, 4, 2, 16).cuda().requires_grad_()
    out, _ = torch_ops.qk_norm(q, q.detach())
    (first,) = torch.autograd.grad(out, q, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice through qk_norm"):
        first.sum().backward()


# ---- together ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
def test_a_delta_layer(cuda, dtype):
    """Slices of one projection, normed to length one, through the rule, and token by token from a prefilled state."""
    batch, length, k_heads, heads, dim = 2, 100, 2, 4, 32
    proj = normal(1, batch, length, (2 * k_heads + heads) * dim, dtype=dtype).cuda()
    gates = normal(2, batch, length, 2 * heads).cuda()
    g, beta = -torch.nn.functional.softplus(gates[..., :heads]) * 0.1, torch.sigmoid(gates[..., heads:])

    def parts(p):
        q, k, v = p.split([k_heads * dim, k_heads * dim, heads * dim], -1)
        lead = p.shape[:-1]
        return q.view(*lead, k_heads, dim), k.view(*lead, k_heads, dim), v.view(*lead, heads, dim)

    q, k, v = parts(proj)
    qn, kn = torch_ops.qk_norm(q, k, norm="l2")
    o, final = torch_ops.gated_delta(qn, kn, v, g, beta)
    cpu = [t.double().cpu() for t in (qn, kn, v, g, beta)]
    eo, efinal = ref.gated_delta(*cpu)
    ref.assert_close(o, eo, ref.DELTA_LOSS[dtype], "o")
    _, state = torch_ops.gated_delta(qn[:, :90], kn[:, :90], v[:, :90], g[:, :90], beta[:, :90])
    for i in range(90, length):
        qi, ki = torch_ops.qk_norm(q[:, i], k[:, i], norm="l2")
        oi = torch_ops.gated_delta_step(state, qi, ki, v[:, i], g[:, i], beta[:, i])
        ref.assert_close(oi, eo[:, i], ref.DELTA_LOSS[dtype], f"token {i}")
    ref.assert_close(state, efinal, ref.DELTA_LOSS[dtype], "state")


def test_refusals_on_the_device(cuda):
    t = {n: None if v is None else v.cuda() for n, v in delta_case(1, 8, 1, 2, 16, 16, BF16).items()}
    args = [t[n] for n in ("q", "k", "v", "g", "beta")]

    def bad(match, *, at=None, value=None, **kw):
        call = [value if i == at else a for i, a in enumerate(args)]
        with pytest.raises(ValueError, match=match):
            torch_ops.gated_delta(*call, **kw)

    bad("k must have shape", at=1, value=t["k"][:, :7])
    bad("v must have shape", at=2, value=t["v"][:, :7])
    bad("dimensions", at=2, value=t["v"][0])
    bad("dtype", at=2, value=t["v"].half())
    bad("dtype", at=3, value=t["g"].half())
    bad("log_decay must have shape", at=3, value=t["g"][..., :1])
    bad("must be", at=0, value=t["q"][0])
    bad("does not support dtype", at=0, value=t["q"].double())
    bad("CUDA", at=1, value=t["k"].cpu())
    bad("initial_state must have shape", initial_state=torch.zeros(1, 2, 16, 15, device="cuda"))
    bad("initial_state does not support", initial_state=torch.zeros(1, 2, 16, 16, device="cuda", dtype=BF16))
    bad("offsets does not support", offsets=torch.tensor([0, 8], device="cuda"))
    bad("n \\+ 1", offsets=torch.tensor([0], dtype=torch.int32, device="cuda"))
    bad("finite", scale=float("nan"))
    big = torch.zeros(1, 8, 1, 129, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="128 channels"):
        torch_ops.gated_delta(big, big, t["v"], *args[3:])
    three = torch.zeros(1, 8, 3, 16, device="cuda", dtype=BF16)
    with pytest.raises(ValueError, match="multiple"):
        torch_ops.gated_delta(three, three, *args[2:])
    s = {n: v.cuda() for n, v in step_case(2, 1, 2, 16, 16, BF16, 2).items()}
    call = [s[n] for n in ("q", "k", "v", "g", "beta")]
    with pytest.raises(ValueError, match="contiguous"):
        torch_ops.gated_delta_step(s["state"].transpose(2, 3), *call)
    with pytest.raises(ValueError, match="as many states"):
        torch_ops.gated_delta_step(s["state"][:1], *call)
    with pytest.raises(ValueError, match="shape of state"):
        torch_ops.gated_delta_step(s["state"], *call, new_state=s["state"][:1])
    with pytest.raises(ValueError, match="slots must have shape"):
        torch_ops.gated_delta_step(s["state"], *call, slots=torch.zeros(3, dtype=torch.int32, device="cuda"))
    two = torch.zeros(3, *s["state"].shape[1:], device="cuda")
    with pytest.raises(cb.Error, match="overlap"):
        torch_ops.gated_delta_step(two[:2], *call, new_state=two[1:])
    q = torch.zeros(4, 2, 16, device="cuda")
    for match, kw in (("one of rms, l2", {"norm": "max"}), ("eps", {"eps": -1.0}), ("go together", {"positions": torch.zeros(4, device="cuda", dtype=torch.int32)}),
                      ("axes need", {"axes": torch.zeros(8, device="cuda", dtype=torch.int32)}),
                      ("must match the leading", {"positions": torch.zeros(3, device="cuda", dtype=torch.int32), "frequencies": torch.zeros(8, device="cuda")}),
                      ("one value for each rotated pair", {"positions": torch.zeros(4, device="cuda", dtype=torch.int32), "frequencies": torch.zeros(9, device="cuda")}),
                      ("positions does not support", {"positions": torch.zeros(4, device="cuda"), "frequencies": torch.zeros(8, device="cuda")}),
                      ("q_weight must have shape", {"q_weight": torch.zeros(8, device="cuda")}),
                      ("q_weight does not support", {"q_weight": torch.zeros(16, device="cuda", dtype=BF16)})):
        with pytest.raises(ValueError, match=match):
            torch_ops.qk_norm(q, q, **kw)
    with pytest.raises(ValueError, match="256 channels"):
        torch_ops.qk_norm(torch.zeros(4, 2, 257, device="cuda"), torch.zeros(4, 2, 257, device="cuda"))
    with pytest.raises(ValueError, match="heads, D"):
        torch_ops.qk_norm(q[0], q[0])
