"""The block norm and the gated recurrence on the GPU against their definitions in 64 bits: every type, gate and
option, sizes around the kernels' tiles, strides, empty and single-token sequences, values that are not finite, and
gradients against the formulas and against differences.  The bounds stand in block_reference."""
import math

import pytest
import torch

import block_reference as ref
import cubutterfly_b200 as cb
from cubutterfly_b200 import torch_ops

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def normal(seed, *shape, dtype=FP32, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale + mean).to(dtype)


def doubles(*tensors):
    return [t.detach().double().cpu() if torch.is_tensor(t) else t for t in tensors]


# ---- block norm --------------------------------------------------------------------------------
def norm_case(shape, dtype, stream=None, gate=None, scale=None, weights=FP32, seed=0):
    """Tensors of one call on the CPU: x, y, pre, post, gate, residual scale."""
    dim = shape[-1]
    gate_shape = {None: None, "channel": (dim,), "full": shape, "group": (*shape[:1], *(1,) * (len(shape) - 2), dim)}[gate]
    return {"x": normal(seed, *shape, dtype=stream or dtype), "y": normal(seed + 1, *shape, dtype=dtype, scale=0.5),
            "pre": normal(seed + 2, dim, dtype=weights, scale=0.1, mean=1.0),
            "post": normal(seed + 3, dim, dtype=weights, scale=0.1, mean=0.6),
            "gate": None if gate_shape is None else
            normal(seed + 4, *gate_shape, dtype=dtype if gate == "full" else weights),
            "scale": normal(seed + 5, dim, dtype=weights, scale=0.1, mean=0.9) if scale == "vector" else (scale or 1.0)}


def check_norm(t, cuda, *, act="none", rotate=False, loss=None, view=lambda v: v, grads=("residual", "normed")):
    """Forward and backward of one case against float64 autograd."""
    names = [k for k, v in t.items() if torch.is_tensor(v)]
    dev = {k: (view(v.to(cuda)) if k in ("x", "y") or (k == "gate" and v.ndim > 1) else v.to(cuda))
           if torch.is_tensor(v) else v for k, v in t.items()}
    for k in names:
        dev[k] = dev[k].detach().requires_grad_()
    res, u = torch_ops.block_norm(dev["x"], dev["y"], pre_weight=dev["pre"], post_weight=dev["post"], gate=dev["gate"],
                                  gate_activation=act, residual_scale=dev["scale"], rotate=rotate)
    exact = dict(zip(t, doubles(*t.values())))
    for k in names:
        exact[k] = exact[k].requires_grad_()
    eres, eu = ref.block_norm(exact["x"], exact["y"], pre_weight=exact["pre"], post_weight=exact["post"],
                              gate=exact["gate"], gate_activation=act, residual_scale=exact["scale"],
                              rotate_rows=rotate)
    loss = ref.NORM_LOSS if loss is None else loss
    ref.assert_close(res, eres.detach(), loss, "residual")
    ref.assert_close(u, eu.detach(), loss, "normed")
    assert res.dtype == t["x"].dtype and u.dtype == t["y"].dtype
    d = {"residual": normal(91, *res.shape, dtype=res.dtype), "normed": normal(92, *u.shape, dtype=u.dtype)}
    outs = {"residual": (res, eres), "normed": (u, eu)}
    got = torch.autograd.grad([outs[g][0] for g in grads], [dev[k] for k in names],
                              [d[g].to(cuda) for g in grads], allow_unused=True)
    want = torch.autograd.grad([outs[g][1] for g in grads], [exact[k] for k in names],
                               [d[g].double() for g in grads], allow_unused=True)
    rows = res.numel() // res.shape[-1]
    for k, a, b in zip(names, got, want):
        if a is None:
            assert b is None
            continue
        b = torch.zeros_like(exact[k]) if b is None else b
        summed = k in ("pre", "post", "scale") or (k == "gate" and t["gate"].shape != t["x"].shape)
        assert a.dtype == t[k].dtype
        ref.assert_close(a, b, loss * (math.sqrt(rows) if summed else 2), "d_" + k)


@pytest.mark.parametrize("dtype,stream", [(BF16, None), (BF16, FP32), (FP16, None), (FP16, FP32), (FP32, None)])
@pytest.mark.parametrize("dim", [1, 2, 7, 8, 31, 64, 255, 256, 257, 512, 1000, 1024, 1025, 2048, 4095, 4096, 4104,
                                 8192, 10000, 16384])
def test_block_norm_sizes_and_types(cuda, dim, dtype, stream):
    check_norm(norm_case((5, dim), dtype, stream, gate="channel", seed=dim), cuda)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 149, 1201])
@pytest.mark.parametrize("dim", [96, 200, 1000, 4096])
def test_block_norm_rows(cuda, rows, dim):
    check_norm(norm_case((rows, dim), BF16, gate="full", seed=rows), cuda, act="silu")


@pytest.mark.parametrize("act", ["none", "sigmoid", "silu"])
@pytest.mark.parametrize("gate", [None, "channel", "group", "full"])
@pytest.mark.parametrize("scale", [0.5, "vector"])
@pytest.mark.parametrize("dtype,weights", [(BF16, FP32), (FP16, FP16), (FP32, FP32), (BF16, BF16)])
def test_block_norm_gates(cuda, act, gate, scale, dtype, weights):
    check_norm(norm_case((3, 37, 264), dtype, gate=gate, scale=scale, weights=weights, seed=7), cuda, act=act)


@pytest.mark.parametrize("dtype,stream", [(BF16, None), (BF16, FP32), (FP16, None), (FP32, None)])
@pytest.mark.parametrize("dim", [64, 128, 256, 512, 1024, 2048, 4096, 8192, 16384])
def test_block_norm_rotation(cuda, dim, dtype, stream):
    check_norm(norm_case((7, dim), dtype, stream, gate="channel", seed=dim), cuda, rotate=True, act="sigmoid")


@pytest.mark.parametrize("dtype,stream", [(BF16, None), (FP16, FP32), (FP32, None)])
@pytest.mark.parametrize("dim", [256, 1024, 2048, 4096, 8192, 16384])
def test_block_norm_rotation_of_many_rows(cuda, dim, dtype, stream):
    """Beyond two rows per SM the rotated rows take another shape."""
    check_norm(norm_case((301, dim), dtype, stream, gate="channel", scale="vector", seed=dim), cuda, rotate=True)


@pytest.mark.parametrize("dtype,stream", [(BF16, None), (FP16, FP32)])
@pytest.mark.parametrize("dim", [250, 264, 2048])
def test_block_norm_groups_of_many_rows(cuda, dim, dtype, stream):
    """Several CTAs sum each gate group's parameter gradients."""
    check_norm(norm_case((3, 400, dim), dtype, stream, gate="group", scale="vector", seed=dim), cuda, act="sigmoid")


def test_block_norm_many_groups(cuda):
    check_norm(norm_case((300, 2, 40), FP32, gate="group", seed=2), cuda, act="silu")


@pytest.mark.parametrize("rotate", [False, True])
@pytest.mark.parametrize("dim", [256, 1024, 4096])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_block_norm_strided_and_unaligned_rows(cuda, dim, dtype, rotate):
    t = norm_case((6, dim), dtype, gate="full", seed=3)

    def shifted(v):  # rows one element off any vector boundary, of an odd stride
        wide = torch.full((v.shape[0], dim + 3), float("nan"), dtype=v.dtype, device=v.device)
        wide[:, 1:dim + 1] = v
        return wide[:, 1:dim + 1]

    def halves(v):   # every other row of a wider tensor
        wide = torch.full((2 * v.shape[0], 2 * dim), float("nan"), dtype=v.dtype, device=v.device)
        wide[::2, dim:] = v
        return wide[::2, dim:]

    for view in (shifted, halves, lambda v: v.t().contiguous().t()):
        check_norm(t, cuda, rotate=rotate, view=view, act="silu")


@pytest.mark.parametrize("grads", [("residual",), ("normed",)])
@pytest.mark.parametrize("rotate", [False, True])
def test_block_norm_gradient_of_one_output(cuda, grads, rotate):
    check_norm(norm_case((9, 512), BF16, FP32, gate="full", scale="vector"), cuda, grads=grads, rotate=rotate)


def test_block_norm_broadcast_gradients(cuda):
    """Gradients that arrive expanded (stride zero), as from a sum."""
    t = norm_case((4, 5, 128), FP32, gate="group")
    x = t["x"].to(cuda).requires_grad_()
    y = t["y"].to(cuda).requires_grad_()
    gate = t["gate"].to(cuda).requires_grad_()
    res, u = torch_ops.block_norm(x, y, gate=gate)
    (res.sum() + 2 * u.sum()).backward()
    ex, ey, eg = (v.requires_grad_() for v in doubles(t["x"], t["y"], t["gate"]))
    eres, eu = ref.block_norm(ex, ey, gate=eg)
    (eres.sum() + 2 * eu.sum()).backward()
    for got, want in ((x, ex), (y, ey), (gate, eg)):
        ref.assert_close(got.grad, want.grad, 8 * ref.NORM_LOSS)


@pytest.mark.parametrize("pre_norm,post_norm", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("gate", [None, "channel", "full"])
def test_block_norm_parts(cuda, pre_norm, post_norm, gate):
    t = norm_case((11, 320), BF16, FP32, gate=gate)
    leaves = {k: t[k].to(cuda).requires_grad_() for k in ("x", "y")}
    if gate:
        leaves["gate"] = t["gate"].to(cuda).requires_grad_()
    res, u = torch_ops.block_norm(**leaves, pre_norm=pre_norm, post_norm=post_norm)
    exact = {k: v.detach().double().cpu().requires_grad_() for k, v in leaves.items()}
    eres, eu = ref.block_norm(**exact, pre_norm=pre_norm, post_norm=post_norm)
    ref.assert_close(res, eres.detach(), ref.NORM_LOSS)
    assert (u is None) == (not pre_norm)
    outs, eouts = ([res], [eres]) if u is None else ([res, u], [eres, eu])
    if u is not None:
        ref.assert_close(u, eu.detach(), ref.NORM_LOSS)
    ds = [normal(5 + k, *o.shape, dtype=o.dtype) for k, o in enumerate(outs)]
    got = torch.autograd.grad(outs, list(leaves.values()), [d.to(cuda) for d in ds])
    want = torch.autograd.grad(eouts, list(exact.values()), [d.double() for d in ds])
    for k, a, b in zip(leaves, got, want):
        ref.assert_close(a, b, 8 * ref.NORM_LOSS, k)


@pytest.mark.parametrize("dtype", [None, BF16])
def test_block_norm_before_the_first_block(cuda, dtype):
    x, w = normal(1, 3, 7, 200), normal(2, 200, mean=1.0)
    dx, dw = x.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    res, u = torch_ops.block_norm(dx, pre_weight=dw, dtype=dtype)
    assert res is dx and u.dtype == (dtype or FP32)
    ex, ew = (v.requires_grad_() for v in doubles(x, w))
    eu = ref.block_norm(ex, pre_weight=ew)[1]
    ref.assert_close(u, eu.detach(), ref.NORM_LOSS)
    d = normal(3, 3, 7, 200, dtype=u.dtype)
    got = torch.autograd.grad(u, (dx, dw), d.to(cuda))
    want = torch.autograd.grad(eu, (ex, ew), d.double())
    ref.assert_close(got[0], want[0], 2 * ref.NORM_LOSS)
    ref.assert_close(got[1], want[1], 8 * ref.NORM_LOSS)


def test_block_norm_no_rows(cuda):
    x = torch.empty(0, 64, device=cuda, requires_grad=True)
    y = torch.empty(0, 64, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda, requires_grad=True)
    g = torch.ones(64, device=cuda, requires_grad=True)
    res, u = torch_ops.block_norm(x, y, pre_weight=w, gate=g)
    assert res.shape == u.shape == (0, 64)
    (res.sum() + u.sum()).backward()
    assert torch.equal(w.grad, torch.zeros_like(w)) and torch.equal(g.grad, torch.zeros_like(g))
    assert x.grad.shape == (0, 64)


def test_block_norm_rows_do_not_mix(cuda):
    """Zeros, NaN and infinities stay in their rows; a row of zeros is normed by eps alone."""
    x, y = normal(1, 8, 512), normal(2, 8, 512)
    x[1, 3], y[2, 5], y[4, 7], x[5, 9] = float("nan"), float("nan"), float("inf"), -float("inf")
    x[6], y[6] = 0, 0
    for rotate in (False, True):
        res, u = torch_ops.block_norm(x.to(cuda), y.to(cuda), rotate=rotate)
        eres, eu = ref.block_norm(*doubles(x, y), rotate_rows=rotate)
        good = [0, 3, 6, 7]
        ref.assert_close(res[good], eres[good], ref.NORM_LOSS)
        ref.assert_close(u[good], eu[good], ref.NORM_LOSS)
        assert torch.isnan(u[[1, 2, 4, 5]]).any(1).all()
        assert torch.equal(torch.isnan(res.cpu()), torch.isnan(eres))
        assert torch.equal(u[6].cpu(), torch.zeros(512))


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_block_norm_large_values(cuda, dtype):
    """Squares beyond the 16-bit range: the sums are fp32."""
    t = norm_case((4, 1024), dtype, FP32)
    t["x"], t["y"] = t["x"] * 3e4, (t["y"].float() * 2e4).clamp(-6e4, 6e4).to(dtype)
    check_norm(t, cuda)


@pytest.mark.parametrize("rotate,gate", [(False, "full"), (True, "channel"), (False, "group")])
def test_block_norm_gradient_against_differences(cuda, rotate, gate):
    """Directional central differences of the operator itself (fp32, step 1e-2 along a unit-size direction: truncation
    ~1e-4 of the second-order terms, rounding 1e-5 of the loss's terms)."""
    t = norm_case((4, 3, 64), FP32, gate=gate, scale="vector", seed=11)
    names = list(t)
    leaves = {k: v.to(cuda).requires_grad_() for k, v in t.items()}
    c = [normal(70 + k, 4, 3, 64).to(cuda).double() for k in range(2)]

    def loss(p):
        res, u = torch_ops.block_norm(p["x"], p["y"], pre_weight=p["pre"], post_weight=p["post"], gate=p["gate"],
                                      gate_activation="silu", residual_scale=p["scale"], rotate=rotate)
        return (res.double() * c[0]).sum() + (u.double() * c[1]).sum()

    grads = dict(zip(names, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    for k in names:
        v = normal(80, *t[k].shape).to(cuda)
        v /= v.norm()
        with torch.no_grad():
            step = 1e-2
            up = loss({**leaves, k: leaves[k] + step * v})
            down = loss({**leaves, k: leaves[k] - step * v})
        slope = float((up - down) / (2 * step))
        want = float((grads[k].double() * v.double()).sum())
        assert abs(slope - want) <= 5e-3 * float(grads[k].norm()) + 5e-3, (k, slope, want)


# ---- gated scan --------------------------------------------------------------------------------
def decay_of(dim, seed=0, low=0.9, high=0.999):
    g = torch.Generator().manual_seed(seed)
    v = torch.rand(dim, generator=g, dtype=torch.float64) * (high - low) + low
    return torch.log(torch.expm1(-torch.log(v) / 8.0)).float()


def scan_case(batch, length, dim, dtype, states=None, seed=0):
    return {"x": normal(seed, batch, length, dim, dtype=dtype), "r": normal(seed + 1, batch, length, dim, dtype=dtype),
            "i": normal(seed + 2, batch, length, dim, dtype=dtype), "decay": decay_of(dim, seed + 3),
            "initial": None if states is None else normal(seed + 4, states, dim)}


def check_scan(t, cuda, offsets=None, view=lambda v: v, loss=None, d_h=True, d_final=True):
    batch, length, dim = t["x"].shape
    dtype = t["x"].dtype
    loss = ref.SCAN_LOSS if loss is None else loss
    names = [k for k, v in t.items() if v is not None]
    dev = {k: (None if v is None else (view(v.to(cuda)) if k in "xri" else v.to(cuda)).detach().requires_grad_())
           for k, v in t.items()}
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int32, device=cuda)
    h, final = torch_ops.gated_scan(dev["x"], dev["r"], dev["i"], dev["decay"], initial_state=dev["initial"],
                                    offsets=off)
    exact = dict(zip(t, doubles(*t.values())))
    eh, ef = ref.gated_scan(exact["x"], exact["r"], exact["i"], exact["decay"], initial=exact["initial"],
                            offsets=offsets)
    ref.assert_close(h, eh, loss, "h")
    ref.assert_close(final, ef, loss, "final")
    assert h.dtype == dtype and final.dtype == FP32
    dh, df = normal(91, *h.shape, dtype=dtype), normal(92, *final.shape)
    outs, ds = zip(*[p for p, on in (((h, dh), d_h), ((final, df), d_final)) if on])
    got = torch.autograd.grad(outs, [dev[k] for k in names], [d.to(cuda) for d in ds])
    want = ref.gated_scan_gradients(exact["x"], exact["r"], exact["i"], exact["decay"],
                                    dh.double() if d_h else torch.zeros_like(eh), df.double() if d_final else None,
                                    initial=exact["initial"], offsets=offsets)
    want = dict(zip(("x", "r", "i", "decay", "initial"), want))
    for k, a in zip(names, got):
        ref.assert_close(a, want[k], 2 * loss, "d_" + k)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("length", [1, 2, 7, 8, 9, 63, 64, 65, 129, 513, 1025])
def test_gated_scan_lengths(cuda, length, dtype):
    check_scan(scan_case(2, length, 66, dtype, states=2, seed=length), cuda)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("dim", [1, 2, 3, 31, 32, 33, 63, 64, 65, 127, 128, 130, 1000])
def test_gated_scan_channels(cuda, dim, dtype):
    check_scan(scan_case(3, 70, dim, dtype, seed=dim), cuda)


@pytest.mark.parametrize("batch,length,dim", [(1, 4099, 64), (1, 2000, 640), (5, 700, 128), (40, 129, 256)])
def test_gated_scan_splits_of_time(cuda, batch, length, dim):
    """Long sequences of few channels, and short ones of many."""
    check_scan(scan_case(batch, length, dim, BF16, states=batch), cuda)


# (batch, length, dim) whose CTAs take 64, 32, 16 and 8 channels forward, and others backward
SPLITS = [(120, 140, 128), (32, 700, 128), (16, 1100, 128), (3, 1100, 128)]


@pytest.mark.parametrize("dtype", [FP16, FP32])
@pytest.mark.parametrize("extra", [0, 2, 1])
@pytest.mark.parametrize("batch,length,dim", SPLITS)
def test_gated_scan_lane_groups(cuda, batch, length, dim, extra, dtype):
    """Every number of lane groups along time, with rows aligned to 16 and 4 bytes and to single values."""
    check_scan(scan_case(batch, length, dim + extra, dtype, states=batch, seed=extra), cuda)


@pytest.mark.parametrize("dim", [8192, 4096, 2048, 1024, 4098, 4097, 1023])
def test_gated_scan_packed_lane_groups(cuda, dim):
    g = torch.Generator().manual_seed(dim)
    cuts = sorted(torch.randint(0, 701, (25,), generator=g).tolist())
    offsets = [0, 0, 1, 17, 17, *[c for c in cuts if c > 17], 700, 700]
    check_scan(scan_case(1, 700, dim, BF16, states=len(offsets) - 1), cuda, offsets=offsets)


@pytest.mark.parametrize("d_h,d_final", [(True, False), (False, True)])
def test_gated_scan_gradient_of_one_output(cuda, d_h, d_final):
    check_scan(scan_case(2, 100, 64, FP32), cuda, d_h=d_h, d_final=d_final)


PACKINGS = {
    "one": [0, 150],
    "single tokens": list(range(0, 151)),
    "empty around": [0, 0, 0, 40, 40, 41, 41, 41, 104, 105, 150, 150],
    "tile edges": [0, 8, 64, 72, 128, 129, 150],
    "inside a tile": [0, 3, 5, 6, 7, 7, 9, 150],
    "all empty but one": [0, 0, 0, 150, 150, 150],
}


@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("packing", list(PACKINGS))
def test_gated_scan_packed(cuda, packing, dtype, state):
    offsets = PACKINGS[packing]
    for dim in (66, 33):
        check_scan(scan_case(1, 150, dim, dtype, states=len(offsets) - 1 if state else None), cuda, offsets=offsets)


def test_gated_scan_packed_over_many_rounds(cuda):
    g = torch.Generator().manual_seed(1)
    cuts = sorted(torch.randint(0, 3001, (60,), generator=g).tolist())
    offsets = [0, 0, *cuts, 3000, 3000]
    check_scan(scan_case(1, 3000, 96, FP16, states=len(offsets) - 1), cuda, offsets=offsets)


def test_gated_scan_packed_two_dimensional(cuda):
    t = scan_case(1, 60, 40, FP32)
    off = torch.tensor([0, 20, 60], dtype=torch.int32, device=cuda)
    args = [t[k].to(cuda) for k in ("x", "r", "i", "decay")]
    h3, f3 = torch_ops.gated_scan(*args, offsets=off)
    h2, f2 = torch_ops.gated_scan(*(v[0] for v in args[:3]), args[3], offsets=off)
    assert torch.equal(h3[0], h2) and torch.equal(f3, f2) and h2.shape == (60, 40)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_gated_scan_sequences_do_not_mix(cuda, bad):
    """What is not finite in one sequence leaves the others and their gradients alone."""
    offsets = [0, 30, 64, 64, 90, 150]
    t = scan_case(1, 150, 64, FP32, states=5)
    clean = {k: v.clone() for k, v in t.items()}
    t["x"][0, 40:60] = bad
    t["initial"][1] = bad
    t["r"][0, 35] = float("nan")
    off = torch.tensor(offsets, dtype=torch.int32, device=cuda)

    def run(t):
        dev = [t[k].to(cuda).requires_grad_() for k in ("x", "r", "i", "decay", "initial")]
        h, final = torch_ops.gated_scan(*dev[:4], initial_state=dev[4], offsets=off)
        d = normal(5, 1, 150, 64).to(cuda)
        grads = torch.autograd.grad((h, final), [*dev[:3], dev[4]], (d, torch.ones_like(final)))
        return h, final, grads

    (h, f, g), (ch, cf, cg) = run(t), run(clean)
    tokens = [*range(30), *range(64, 150)]
    assert torch.equal(h[0, tokens], ch[0, tokens])
    assert torch.equal(f[[0, 2, 3, 4]], cf[[0, 2, 3, 4]])
    assert not torch.isfinite(f[1]).any()
    for a, b in zip(g[:3], cg[:3]):
        assert torch.equal(a[0, tokens], b[0, tokens])
    assert torch.equal(g[3][[0, 2, 3, 4]], cg[3][[0, 2, 3, 4]])


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_gated_scan_extreme_gates(cuda, dtype):
    """Gates that are shut (the state is kept exactly), wide open, or far out; decays from nearly 0 to nearly 1."""
    t = scan_case(1, 80, 64, dtype, states=1)
    t["r"][0, 10:20], t["r"][0, 20:30] = -float("inf"), float("inf")
    t["r"][0, 30:40], t["r"][0, 40:50] = -90.0, 90.0
    t["i"][0, 5:15], t["i"][0, 50:60] = -float("inf"), float("inf")
    t["decay"] = torch.linspace(-30, 30, 64)
    check_scan(t, cuda)
    h, _ = torch_ops.gated_scan(*(t[k].to(cuda) for k in ("x", "r", "i", "decay")),
                                initial_state=t["initial"].to(cuda))
    # the same bits within a thread's eight tokens; across them the state arrives as a joined map, rounded differently
    assert torch.equal(h[0, 10], h[0, 9]) and torch.equal(h[0, 15], h[0, 9]) and torch.equal(h[0, 19], h[0, 16])


def test_gated_scan_slow_decay(cuda):
    """Decays so slow that 1 - a^2 cancels: the series carries sqrt(1 - a^2)."""
    t = scan_case(1, 64, 64, FP32)
    t["decay"] = decay_of(64, low=1 - 1e-6, high=1 - 1e-7)
    t["r"] -= 6
    check_scan(t, cuda)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_gated_scan_infinite_decay(cuda, dtype):
    """A channel that forgets everything: h is sigmoid(i) x, and so is the final state, whatever the length."""
    for length in (1, 5, 200):
        t = scan_case(2, length, 40, dtype, states=2)
        t["decay"][::2] = math.inf
        x, r, i = (t[k].double() for k in "xri")
        dev = [t[k].to(cuda).requires_grad_() for k in ("x", "r", "i", "decay", "initial")]
        h, final = torch_ops.gated_scan(*dev[:4], initial_state=dev[4])
        want = (torch.sigmoid(i) * x)[..., ::2]
        ref.assert_close(h[..., ::2], want, ref.SCAN_LOSS)
        ref.assert_close(final[:, ::2], want[:, -1], ref.SCAN_LOSS)
        d = normal(6, *h.shape, dtype=dtype)
        grads = torch.autograd.grad((h, final), dev, (d.to(cuda), torch.ones_like(final)))
        g = d.double()
        g[:, -1] += 1
        s = torch.sigmoid(i)
        ref.assert_close(grads[0][..., ::2], (g * s)[..., ::2], ref.SCAN_LOSS)
        ref.assert_close(grads[2][..., ::2], (g * x * s * (1 - s))[..., ::2], ref.SCAN_LOSS)
        for k in (1, 3, 4):
            assert torch.isfinite(grads[k]).all() and not grads[k][..., ::2].any()


@pytest.mark.parametrize("dim", [64, 62, 33])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_gated_scan_strided_inputs(cuda, dim, dtype):
    t = scan_case(2, 90, dim, dtype)

    def slices(v):
        wide = torch.full((*v.shape[:2], 3 * dim), float("nan"), dtype=v.dtype, device=v.device)
        wide[..., dim:2 * dim] = v
        return wide[..., dim:2 * dim]

    def odd(v):
        wide = torch.full((v.shape[0], v.shape[1], dim + 1), float("nan"), dtype=v.dtype, device=v.device)
        wide[..., 1:] = v
        return wide[..., 1:]

    for view in (slices, odd, lambda v: v.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda v: v.transpose(1, 2).contiguous().transpose(1, 2)):
        check_scan(t, cuda, view=view)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("batch,length,dim", [*((b, s, d + 1) for b, s, d in SPLITS),
                                              *((3, 700, d) for d in (1, 3, 5, 7, 9))])
def test_gated_scan_odd_rows_in_wider_ones(cuda, batch, length, dim, dtype):
    """Rows of an odd length whose neighbours in memory, read with them, are NaN; tensors of different shifts."""
    t = scan_case(batch, length, dim, dtype, states=batch, seed=dim)
    for left, right in ((0, 0), (1, 0), (5, 2), (0, 1)):

        def view(v):
            wide = torch.full((*v.shape[:2], left + dim + right), float("nan"), dtype=v.dtype, device=v.device)
            wide[..., left:left + dim] = v
            return wide[..., left:left + dim]

        check_scan(t, cuda, view=view)


def test_gated_scan_no_tokens(cuda):
    decay = decay_of(16).to(cuda).requires_grad_()
    x = torch.empty(2, 0, 16, device=cuda, requires_grad=True)
    s = torch.randn(2, 16, device=cuda, requires_grad=True)
    h, final = torch_ops.gated_scan(x, x, x, decay, initial_state=s)
    assert h.shape == (2, 0, 16) and torch.equal(final, s)
    (3 * final).sum().backward()
    assert torch.equal(s.grad, torch.full_like(s, 3)) and torch.equal(decay.grad, torch.zeros_like(decay))
    h, final = torch_ops.gated_scan(x, x, x, decay)
    assert torch.equal(final, torch.zeros_like(final))
    off = torch.zeros(4, dtype=torch.int32, device=cuda)
    h, final = torch_ops.gated_scan(x[0], x[0], x[0], decay, offsets=off)
    assert h.shape == (0, 16) and torch.equal(final, torch.zeros(3, 16, device=cuda))


def test_gated_scan_carried_over_chunks(cuda):
    """A sequence run in pieces, each from the state before, is the sequence run at once."""
    t = scan_case(2, 300, 70, FP32)
    args = [t[k].to(cuda) for k in ("x", "r", "i")]
    decay = t["decay"].to(cuda)
    h, final = torch_ops.gated_scan(*args, decay)
    state, parts = None, []
    for a, b in ((0, 1), (1, 64), (64, 200), (200, 300)):
        part, state = torch_ops.gated_scan(*(v[:, a:b] for v in args), decay, initial_state=state)
        parts.append(part)
    ref.assert_close(torch.cat(parts, 1), h, ref.SCAN_LOSS)
    ref.assert_close(state, final, ref.SCAN_LOSS)


@pytest.mark.parametrize("packed", [False, True])
def test_gated_scan_gradient_against_differences(cuda, packed):
    t = scan_case(1 if packed else 2, 40, 34, FP32, states=3 if packed else 2, seed=5)
    off = torch.tensor([0, 11, 11, 40], dtype=torch.int32, device=cuda) if packed else None
    leaves = {k: v.to(cuda).requires_grad_() for k, v in t.items()}
    ch, cf = normal(70, *t["x"].shape).to(cuda).double(), normal(71, *t["initial"].shape).to(cuda).double()

    def loss(p):
        h, final = torch_ops.gated_scan(p["x"], p["r"], p["i"], p["decay"], initial_state=p["initial"], offsets=off)
        return (h.double() * ch).sum() + (final.double() * cf).sum()

    grads = dict(zip(leaves, torch.autograd.grad(loss(leaves), list(leaves.values()))))
    for k in leaves:
        v = normal(80, *t[k].shape).to(cuda)
        v /= v.norm()
        with torch.no_grad():
            step = 1e-2
            slope = float((loss({**leaves, k: leaves[k] + step * v}) - loss({**leaves, k: leaves[k] - step * v}))
                          / (2 * step))
        want = float((grads[k].double() * v.double()).sum())
        assert abs(slope - want) <= 5e-3 * float(grads[k].norm()) + 5e-3, (k, slope, want)


def test_gated_scan_offsets_beyond_32_bits(cuda):
    """More than 2^31 values per tensor: the end of a long sequence is that of its last tokens run alone (decays below
    0.999 forget the rest: 0.9995^40000 < 3e-9 for the mildest gate mean used here)."""
    length, dim, tail = (1 << 21) + 5, 1040, 60000
    g = torch.Generator(cuda).manual_seed(1)
    x = torch.randn(1, length, dim, device=cuda, generator=g, dtype=FP16)
    r = torch.randn(1, length, dim, device=cuda, generator=g, dtype=FP16) + 2
    i = torch.randn(1, length, dim, device=cuda, generator=g, dtype=FP16)
    decay = decay_of(dim, high=0.998).to(cuda)
    h, final = torch_ops.gated_scan(x, r, i, decay)
    th, tf = torch_ops.gated_scan(x[:, -tail:], r[:, -tail:], i[:, -tail:], decay)
    ref.assert_close(h[0, -100:], th[0, -100:].double(), ref.SCAN_LOSS + 2 * ref.ROUNDING[FP16])
    ref.assert_close(final, tf, ref.SCAN_LOSS)


# ---- one token ---------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("batch,dim", [(1, 1), (1, 4096), (3, 33), (7, 64), (130, 66), (300, 1000)])
def test_gated_scan_step(cuda, batch, dim, dtype):
    t = scan_case(batch, 1, dim, dtype, states=batch)
    x, r, i = (t[k][:, 0] for k in "xri")
    state = t["initial"].to(cuda)
    h = torch_ops.gated_scan_step(state, x.to(cuda), r.to(cuda), i.to(cuda), t["decay"].to(cuda))
    e = dict(zip(t, doubles(*t.values())))
    eh, ef = ref.gated_scan(e["x"], e["r"], e["i"], e["decay"], initial=e["initial"])
    ref.assert_close(h, eh[:, 0], ref.SCAN_LOSS)
    ref.assert_close(state, ef, ref.SCAN_LOSS)


def test_gated_scan_step_slots_and_padding(cuda):
    pool, batch, dim = 20, 9, 72
    t = scan_case(batch, 1, dim, BF16)
    x, r, i = (t[k][:, 0].clone() for k in "xri")
    slots = torch.tensor([3, -1, 19, 0, 20, 7, -2147483648, 12, 2147483647], dtype=torch.int32)
    padded = [1, 4, 6, 8]
    x[padded], r[padded] = float("nan"), float("nan")
    before = normal(9, pool, dim)
    state = before.to(cuda)
    fresh = torch.full((pool, dim), 7.0, device=cuda)
    args = [v.to(cuda) for v in (x, r, i, t["decay"])]
    h = torch_ops.gated_scan_step(state, *args, slots=slots.to(cuda), new_state=fresh)
    assert torch.equal(state.cpu(), before)
    h2 = torch_ops.gated_scan_step(state, *args, slots=slots.to(cuda))
    assert torch.equal(h, h2) and torch.equal(h[padded].cpu(), torch.zeros(4, dim, dtype=BF16))
    used = [k for k in range(batch) if k not in padded]
    rows = slots[used].long()
    e = doubles(x[used][:, None], r[used][:, None], i[used][:, None], t["decay"], before[rows])
    eh, ef = ref.gated_scan(*e[:4], initial=e[4])
    ref.assert_close(h[used], eh[:, 0], ref.SCAN_LOSS)
    ref.assert_close(state[rows], ef, ref.SCAN_LOSS)
    assert torch.equal(fresh[rows], state[rows])
    others = [k for k in range(pool) if k not in rows.tolist()]
    assert torch.equal(state[others].cpu(), before[others])
    assert torch.equal(fresh[others].cpu(), torch.full((len(others), dim), 7.0))


def test_steps_follow_the_scan(cuda):
    """Prefill, then token by token, is the scan of everything."""
    t = scan_case(3, 90, 130, FP32)
    x, r, i, decay = (t[k].to(cuda) for k in ("x", "r", "i", "decay"))
    h, final = torch_ops.gated_scan(x, r, i, decay)
    _, state = torch_ops.gated_scan(x[:, :70], r[:, :70], i[:, :70], decay)
    for k in range(70, 90):
        step = torch_ops.gated_scan_step(state, x[:, k], r[:, k], i[:, k], decay)
        ref.assert_close(step, h[:, k], ref.SCAN_LOSS)
    ref.assert_close(state, final, ref.SCAN_LOSS)


def test_block_norm_many_gate_groups(cuda):
    """More gate groups than a grid has rows."""
    check_norm(norm_case((66000, 2, 32), BF16, gate="group", seed=3), cuda, act="sigmoid")


# (which leading axes of (3, 5, D) are broadcast)
@pytest.mark.parametrize("axes", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("dtype,dim,rotate", [(BF16, 64, True), (FP16, 33, False), (FP32, 258, False)])
def test_block_norm_broadcast_inputs(cuda, axes, dtype, dim, rotate):
    """x, y and the gate as views whose rows share memory (strides of zero) are their values written out."""
    t = norm_case((3, 5, dim), dtype, gate="full", seed=dim)

    def first(v):
        for a in axes:
            v = v.narrow(a, 0, 1)
        return v

    for k in ("x", "y", "gate"):
        t[k] = first(t[k]).expand(3, 5, dim).contiguous()
    views = []

    def view(v):
        views.append(first(v).clone().expand(3, 5, dim))
        return views[-1]

    check_norm(t, cuda, act="silu", rotate=rotate, view=view)
    assert len(views) == 3 and not any(v.is_contiguous() for v in views)


def test_block_norm_broadcast_gate_per_group(cuda):
    t = norm_case((4, 6, 72), BF16, gate="group")
    t["gate"] = t["gate"][:1].expand(4, 1, 72).contiguous()
    check_norm(t, cuda, act="sigmoid",
               view=lambda v: v[:1].clone().expand(4, 1, 72) if v.shape[1] == 1 else v)


@pytest.mark.parametrize("of", ["residual", "normed"])
@pytest.mark.parametrize("axes", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (FP32, 33)])
def test_block_norm_gradient_of_sums_over_rows(cuda, of, axes, dtype, dim):
    """The gradient of a sum over leading axes arrives with strides of zero there and one along the channels."""
    t = norm_case((3, 5, dim), dtype, gate="channel", seed=dim + 1)
    w = normal(77, dim, dtype=dtype)
    dev = {k: v.to(cuda).requires_grad_() for k, v in t.items() if torch.is_tensor(v)}
    exact = {k: v.double().requires_grad_() for k, v in t.items() if torch.is_tensor(v)}
    call = lambda f, p: f(p["x"], p["y"], pre_weight=p["pre"], post_weight=p["post"], gate=p["gate"])
    pick = 0 if of == "residual" else 1
    seen = []
    out = call(torch_ops.block_norm, dev)[pick]
    out.register_hook(seen.append)
    (out.sum(axes) * w.to(cuda)).sum().backward()
    (call(ref.block_norm, exact)[pick].sum(axes) * w.double()).sum().backward()
    assert seen[0].stride(-1) == 1 and any(seen[0].stride(a) == 0 for a in axes)
    for k in dev:
        if exact[k].grad is not None:
            summed = k in ("pre", "post", "gate")
            ref.assert_close(dev[k].grad, exact[k].grad, ref.NORM_LOSS * (math.sqrt(15) if summed else 2), "d_" + k)


def test_gated_scan_step_broadcast_inputs(cuda):
    """One token's x and gates shared by all requests of the batch."""
    batch, dim = 5, 72
    t = scan_case(1, 1, dim, BF16)
    x, r, i = (t[k][0].to(cuda).expand(batch, dim) for k in "xri")
    before = normal(9, batch, dim)
    state = before.to(cuda)
    h = torch_ops.gated_scan_step(state, x, r, i, t["decay"].to(cuda))
    wide = doubles(*(t[k].expand(batch, 1, dim) for k in "xri"), t["decay"], before)
    eh, ef = ref.gated_scan(*wide[:4], initial=wide[4])
    ref.assert_close(h, eh[:, 0], ref.SCAN_LOSS)
    ref.assert_close(state, ef, ref.SCAN_LOSS)


def test_gated_scan_step_marks_its_writes(cuda):
    """A pool that a backward still needs may not change unnoticed under it."""
    x = normal(1, 2, 5, 64).to(cuda).requires_grad_()
    decay = decay_of(64).to(cuda)
    pool, other = normal(2, 2, 64).to(cuda), torch.zeros(2, 64, device=cuda)
    token = normal(3, 2, 64).to(cuda)
    h, _ = torch_ops.gated_scan(x, x, x, decay, initial_state=pool)
    torch_ops.gated_scan_step(pool, token, token, token, decay, new_state=other)   # the pool stays
    h.sum().backward()
    h, _ = torch_ops.gated_scan(x, x, x, decay, initial_state=pool)
    torch_ops.gated_scan_step(pool, token, token, token, decay)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()
    with torch.inference_mode():   # tensors without a version
        pool = torch.zeros(2, 64, device=cuda)
        torch_ops.gated_scan_step(pool, token, token, token, decay)


# ---- the gates' accuracy -------------------------------------------------------------------------
def relative(got, want):
    want = want.double().cpu()
    return float(((got.detach().double().cpu() - want) / want).abs().max())


@pytest.mark.parametrize("dtype,stream,gate", [(FP32, None, "full"), (FP32, None, "channel"), (BF16, FP32, "full"),
                                               (BF16, FP32, "channel"), (FP16, FP32, "group")])
@pytest.mark.parametrize("act", ["sigmoid", "silu"])
def test_block_norm_gates_to_the_last_bits(cuda, dtype, stream, gate, act):
    """Where the residual is fp32 so are the gate's bits.  exp: one unit of 2^-23; 1 + exp, the quotient and silu's
    product: half a one each."""
    dim, rows = 1024, 4
    wide = dtype if gate == "full" else FP32
    g = torch.linspace(-30, 30, rows * dim).reshape(rows, dim)
    g = {"full": g, "channel": g[1], "group": g[:, None]}[gate].to(wide)
    shape = (rows, 2, dim) if gate == "group" else (rows, dim)
    x, y = torch.zeros(shape, dtype=stream or dtype), torch.ones(shape, dtype=dtype)
    res, _ = torch_ops.block_norm(x.to(cuda), y.to(cuda), gate=g.to(cuda), gate_activation=act, post_norm=False,
                                  pre_norm=False)
    s = torch.sigmoid(g.double())
    want = (s if act == "sigmoid" else g.double() * s).expand(shape)
    assert relative(res, want) <= 3e-7 + (2.0 ** -24 if act == "silu" else 0)


@pytest.mark.parametrize("what", ["step", "scan"])
def test_scan_gates_to_the_last_bits(cuda, what):
    """fp32 gates.  exp and the reciprocal: a unit of 2^-23 each, the reciprocal root two thirds of one, 1 + exp and
    the products half a one each."""
    dim = 4096
    gate = torch.linspace(-30, 30, dim)
    open_, one = torch.full((dim,), math.inf), torch.ones(dim)
    decay = torch.full((dim,), 3.0)

    def run(x, r, i, lam):
        args = [v.to(cuda)[None] for v in (x, r, i)]
        if what == "step":
            return torch_ops.gated_scan_step(torch.zeros(1, dim, device=cuda), *args, lam.to(cuda))[0]
        return torch_ops.gated_scan(*(v[None] for v in args), lam.to(cuda))[0][0, 0]

    # the input gate: a recurrence gate that forgets everything leaves x sigmoid(i)
    s = torch.sigmoid(gate.double())
    assert relative(run(one, open_, gate, torch.full((dim,), 60.0)), s) <= 6e-7
    # the recurrence gate: an open input gate leaves sqrt(1 - a^2)
    la = -8 * torch.nn.functional.softplus(decay.double()) * s
    assert relative(run(one, gate, open_, decay), torch.sqrt(-torch.expm1(2 * la))) <= 6.5e-7
    # far out, with an x to match
    far = torch.linspace(-80, -45, dim)
    x = torch.exp(-far)
    want = x.double() * torch.sigmoid(far.double())
    assert relative(run(x, open_, far, torch.full((dim,), 60.0)), want) <= 6e-7


def test_gated_scan_gradient_gates_to_the_last_bits(cuda):
    dim = 4096
    gate = torch.linspace(-30, 30, dim)
    x = torch.ones(1, 1, dim, device=cuda, requires_grad=True)
    r = torch.full((1, 1, dim), math.inf, device=cuda)
    h, _ = torch_ops.gated_scan(x, r, gate[None, None].to(cuda), torch.full((dim,), 60.0, device=cuda))
    h.backward(torch.ones_like(h))
    assert relative(x.grad[0, 0], torch.sigmoid(gate.double())) <= 6e-7


# ---- streams, graphs, repeatability ------------------------------------------------------------
def all_operators(cuda, seed=0):
    n = norm_case((40, 512), BF16, FP32, gate="channel", scale="vector", seed=seed)
    s = scan_case(2, 200, 128, BF16, states=2, seed=seed)
    n = {k: v.to(cuda).requires_grad_() for k, v in n.items()}
    s = {k: v.to(cuda).requires_grad_() for k, v in s.items()}

    def run():
        res, u = torch_ops.block_norm(n["x"], n["y"], pre_weight=n["pre"], post_weight=n["post"], gate=n["gate"],
                                      gate_activation="silu", residual_scale=n["scale"], rotate=True)
        h, final = torch_ops.gated_scan(s["x"], s["r"], s["i"], s["decay"], initial_state=s["initial"])
        outs = (res, u, h, final)
        return outs + torch.autograd.grad(outs, [*n.values(), *s.values()], [torch.ones_like(o) for o in outs])

    return run


def test_results_repeat_bit_for_bit(cuda):
    run = all_operators(cuda)
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_backward_from_several_threads(cuda):
    """Threads that run one graph's backward: each gets the gradients, or, once one has freed the graph, an error."""
    import threading

    x = normal(1, 3, 50, 64).to(cuda).requires_grad_()
    w, decay = torch.ones(64, device=cuda), decay_of(64).to(cuda)

    def graph():
        u = torch_ops.block_norm(x, x * 2, pre_weight=w)[1]
        return torch_ops.gated_scan(u, u, u, decay)[0].sum()

    want = torch.autograd.grad(graph(), x)[0]
    for _ in range(5):
        loss, got, errors = graph(), [], []

        def run(keep):
            try:
                got.append(torch.autograd.grad(loss, x, retain_graph=keep)[0])
            except RuntimeError as e:
                errors.append(str(e))

        threads = [threading.Thread(target=run, args=(k != 5,)) for k in range(8)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert len(got) + len(errors) == 8 and got and all(torch.equal(g, want) for g in got)
        assert all("second time" in e for e in errors), errors


def test_side_streams(cuda):
    run = all_operators(cuda, 3)
    want = run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run())
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(a, b) for a, b in zip(want, outs))


def test_decode_in_an_inference_graph(cuda):
    """Norm, rotation, recurrence step and norm captured as one graph."""
    dim = 256
    decay = decay_of(dim).to(cuda)
    state = torch.zeros(4, dim, device=cuda)
    w = torch.ones(dim, device=cuda)

    def token(x):
        _, u = torch_ops.block_norm(x, pre_weight=w, rotate=True)
        h = torch_ops.gated_scan_step(state, u, u, u, decay)
        return torch_ops.block_norm(x, h, pre_weight=w, post_weight=w)[1]

    x = normal(1, 4, dim, dtype=BF16).to(cuda)
    graph = torch_ops.InferenceGraph(token, x)
    with torch.cuda.stream(graph.stream):
        state.zero_()
        first = [graph(x * k) for k in range(1, 4)]
        state.zero_()
        want = [token(x * k) for k in range(1, 4)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, want))


# ---- refusals and the frontend's errors --------------------------------------------------------
def test_refusals_on_the_device(cuda):
    x, y = torch.randn(2, 3, 64, device=cuda), torch.randn(2, 3, 64, device=cuda)
    w, state = torch.ones(64, device=cuda), torch.zeros(3, 64, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    bad = [
        (lambda: torch_ops.block_norm(x, y[:1]), "shape"),
        (lambda: torch_ops.block_norm(x, y.double()), "dtype"),
        (lambda: torch_ops.block_norm(x.half(), y.bfloat16()), "residual stream"),
        (lambda: torch_ops.block_norm(x, y, pre_weight=w[:32]), "shape"),
        (lambda: torch_ops.block_norm(x, y, pre_weight=w, pre_norm=False), "turned off"),
        (lambda: torch_ops.block_norm(x, y, rotate=True, pre_norm=False), "rotate"),
        (lambda: torch_ops.block_norm(x, y, gate=w[:3]), "gate"),
        (lambda: torch_ops.block_norm(x, y, gate=w, gate_activation="tanh"), "gate_activation"),
        (lambda: torch_ops.block_norm(x, y, residual_scale=math.inf), "residual_scale"),
        (lambda: torch_ops.block_norm(x, y, eps=-1.0), "eps"),
        (lambda: torch_ops.block_norm(x, gate=w), "block output"),
        (lambda: torch_ops.block_norm(x, residual_scale=0.5), "block output"),
        (lambda: torch_ops.block_norm(x, pre_norm=False), "nothing to compute"),
        (lambda: torch_ops.block_norm(x, y, dtype=BF16), "dtype"),
        (lambda: torch_ops.block_norm(x.half(), y.half(), gate=y), "gate per row"),
        (lambda: torch_ops.gated_scan(x[0], x[0], x[0], w), "must be"),
        (lambda: torch_ops.gated_scan(x, x[:, :2], x, w), "shape"),
        (lambda: torch_ops.gated_scan(x, x.half(), x, w), "dtype"),
        (lambda: torch_ops.gated_scan(x, x, x, w[:8]), "shape"),
        (lambda: torch_ops.gated_scan(x, x, x, w, exponent=0.0), "exponent"),
        (lambda: torch_ops.gated_scan(x, x, x, w, initial_state=state), "shape"),
        (lambda: torch_ops.gated_scan(x, x, x, w, initial_state=state[:2].half()), "dtype"),
        (lambda: torch_ops.gated_scan(x, x, x, w, offsets=torch.zeros(3, **i32)), "packed"),
        (lambda: torch_ops.gated_scan(x[0], x[0], x[0], w, offsets=torch.zeros(1, **i32)), "offsets"),
        (lambda: torch_ops.gated_scan(x[0], x[0], x[0], w, offsets=torch.zeros(3, device=cuda).long()), "dtype"),
        (lambda: torch_ops.gated_scan_step(state, x, x, x, w), "must be"),
        (lambda: torch_ops.gated_scan_step(state[:2], x[0], x[0], x[0], w), "pool"),
        (lambda: torch_ops.gated_scan_step(state.half(), x[0], x[0], x[0], w), "dtype"),
        (lambda: torch_ops.gated_scan_step(state.t(), x[0], x[0], x[0], w), "pool"),
        (lambda: torch_ops.gated_scan_step(state, x[0], x[0], x[0], w, slots=torch.zeros(2, **i32)), "shape"),
        (lambda: torch_ops.gated_scan_step(state, x[0], x[0], x[0], w, new_state=state[:2]), "shape"),
        (lambda: torch_ops.gated_scan_step(state, x[0].clone().requires_grad_(), x[0], x[0], w), "inference only"),
        (lambda: torch_ops.block_norm([1.0]), "CUDA"),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()


def test_forward_mode_tangents_are_refused(cuda):
    import torch.autograd.forward_ad as fwd

    x = torch.randn(3, 64, device=cuda)
    w, state = torch.ones(64, device=cuda), torch.zeros(3, 64, device=cuda)
    with fwd.dual_level():
        dual, dw = fwd.make_dual(x, torch.ones_like(x)), fwd.make_dual(w, torch.ones_like(w))
        ds = fwd.make_dual(state, torch.ones_like(state))
        for call in (lambda: torch_ops.block_norm(dual), lambda: torch_ops.block_norm(x, dual),
                     lambda: torch_ops.block_norm(x, x, gate=dual), lambda: torch_ops.block_norm(x, x, pre_weight=dw),
                     lambda: torch_ops.block_norm(x, x, post_weight=dw),
                     lambda: torch_ops.block_norm(x, x, residual_scale=dw),
                     lambda: torch_ops.gated_scan(x[None], dual[None], x[None], w),
                     lambda: torch_ops.gated_scan(x[None], x[None], dual[None], w),
                     lambda: torch_ops.gated_scan(x[None], x[None], x[None], dw),
                     lambda: torch_ops.gated_scan(x[None], x[None], x[None], w, initial_state=ds[:1]),
                     lambda: torch_ops.gated_scan_step(ds, x, x, x, w), lambda: torch_ops.gated_scan_step(state, x, x, x, dw)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        torch_ops.block_norm(x, x, pre_weight=w)  # a level without a tangent among the arguments


def test_wrapped_weights_are_refused(cuda):
    """A weight without storage of its own is refused wherever it stands, not left out."""
    from test_block_ops import Wrapper

    x = torch.randn(3, 64, device=cuda)
    w = Wrapper(64)
    for call in (lambda: torch_ops.block_norm(x, x, pre_weight=w), lambda: torch_ops.block_norm(x, x, post_weight=w),
                 lambda: torch_ops.block_norm(x, x, gate=w), lambda: torch_ops.block_norm(x, x, residual_scale=w),
                 lambda: torch_ops.gated_scan(x[None], x[None], x[None], x[0], initial_state=Wrapper(1, 64)),
                 lambda: torch_ops.gated_scan_step(x, x, x, x, x[0], slots=Wrapper(3))):
        with pytest.raises(ValueError, match="storage of its own"):
            call()


def test_counting_modes_pass(cuda):
    """Modes that only watch the dispatcher do not stand in the way."""
    from torch.utils.flop_counter import FlopCounterMode

    x = torch.randn(3, 64, device=cuda)
    want = torch_ops.block_norm(x)[1]
    with FlopCounterMode(display=False):
        assert torch.equal(torch_ops.block_norm(x)[1], want)


def test_gated_scan_step_refuses_a_decay_that_requires_grad(cuda):
    state, x = torch.zeros(3, 64, device=cuda), torch.randn(3, 64, device=cuda)
    decay = decay_of(64).to(cuda).requires_grad_()
    leaf = torch.zeros(3, 64, device=cuda, requires_grad=True)
    with pytest.raises(ValueError, match="inference only"):
        torch_ops.gated_scan_step(state, x, x, x, decay)
    with pytest.raises(ValueError, match="inference only"):
        torch_ops.gated_scan_step(state, x, x, x, decay.detach(), new_state=leaf)
    with torch.no_grad():
        torch_ops.gated_scan_step(state, x, x, x, decay)


def test_library_refusals_name_their_status(cuda):
    x = torch.randn(2, 96, device=cuda)
    with pytest.raises(cb.Error, match="power-of-two") as e:
        torch_ops.block_norm(x, x, rotate=True)
    assert e.value.status == cb.Status.NOT_SUPPORTED
    wide = torch.randn(1, 16385, device=cuda)
    with pytest.raises(cb.Error, match="16384"):
        torch_ops.block_norm(wide, wide)


def test_differentiable_once(cuda):
    x = torch.randn(2, 8, 32, device=cuda, requires_grad=True)
    w = torch.ones(32, device=cuda)
    for out in (torch_ops.block_norm(x, x * 2)[1], torch_ops.gated_scan(x, x, x, w)[0]):
        (g,) = torch.autograd.grad(out.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()


def test_only_asked_gradients_are_returned(cuda):
    x, y = torch.randn(4, 64, device=cuda), torch.randn(4, 64, device=cuda, requires_grad=True)
    w = torch.ones(64, device=cuda)
    res, u = torch_ops.block_norm(x, y, pre_weight=w)
    (res.sum() + u.sum()).backward()
    assert y.grad is not None and x.grad is None and w.grad is None
    with torch.no_grad():
        assert not torch_ops.block_norm(x, y)[1].requires_grad


def test_low_precision_decay(cuda):
    """A decay in the block's type is widened, and its gradient comes back in that type."""
    x = normal(1, 2, 20, 64, dtype=BF16).to(cuda)
    decay = decay_of(64).to(BF16).to(cuda).requires_grad_()
    h, _ = torch_ops.gated_scan(x, x, x, decay)
    want, _ = torch_ops.gated_scan(x, x, x, decay.detach().float())
    assert torch.equal(h, want)
    h.float().sum().backward()
    assert decay.grad.dtype == BF16 and torch.isfinite(decay.grad).all()
