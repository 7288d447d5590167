"""Block norm and gated recurrence by their definitions, in 64 bits on the CPU, and the bounds the kernels are held to.

A kernel computes in fp32 and rounds once, so an output may be off by
  * half a unit in the last place of its type, relative to itself (ROUNDING), and
  * what fp32 loses, relative to the largest value of the tensor (the `loss` a test passes).
"""
import math

import torch

ROUNDING = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}  # half a step among the subnormals
# Row sums of up to 16384 squares, two norms in turn and fourteen butterfly
# stages, each a few units of 2^-24 relative to the row's largest values: ~50 in
# all; sums over the rows add at most rows x 2^-24 of the sum of magnitudes.
NORM_LOSS = 64 * 2.0 ** -24
# A decay carries two units of 2^-24 and is applied 1/(1 - a) times before it
# is forgotten, 1000 for a = 0.999; the gates' and sqrt(1 - a^2)'s approximations
# stay below 25 units.
SCAN_LOSS = 2048 * 2.0 ** -24


def assert_close(got, want, loss, what=""):
    want = want.double().cpu()
    assert tuple(got.shape) == tuple(want.shape), (what, got.shape, want.shape)
    if not want.numel():
        return
    g = got.detach().double().cpu()
    same = torch.isnan(g) == torch.isnan(want)
    assert same.all(), f"{what}: NaN in {int((~same).sum())} wrong places"
    infinite = torch.isinf(want)
    assert torch.equal(g[infinite], want[infinite]), f"{what}: infinities differ"
    ok = torch.isfinite(want)
    if not ok.any():
        return
    w, e = want[ok], (g[ok] - want[ok]).abs()
    bound = (ROUNDING[got.dtype] + 2.0 ** -22) * w.abs() + loss * w.abs().max() + TINY[got.dtype]
    worst = (e / bound).max()
    assert worst <= 1.0, f"{what}: error {float(e.max()):.3e}, {float(worst):.2f} of the bound"


def hadamard(dim):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < dim:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    return h / math.sqrt(dim)


def rotate(v):
    """v H_D / sqrt(D): by the matrix, or by butterflies where the matrix is large."""
    dim = v.shape[-1]
    if dim <= 1024:
        return v @ hadamard(dim)
    low = hadamard(64).to(v.dtype)
    w = v.reshape(*v.shape[:-1], dim // 64, 64) @ low
    return (hadamard(dim // 64) @ w).reshape(v.shape)


def block_norm(x, y=None, *, pre_weight=None, post_weight=None, gate=None, gate_activation="none", residual_scale=1.0,
               eps=1e-6, pre_norm=True, post_norm=True, rotate_rows=False):
    def rms(v, w):
        v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)
        return v if w is None else v * w

    residual, normed = x, None
    if y is not None:
        n = rms(y, post_weight) if post_norm else y
        if gate is not None:
            s = torch.sigmoid(gate)
            n = n * {"none": gate, "sigmoid": s, "silu": gate * s}[gate_activation]
        residual = residual_scale * x + n
    if pre_norm:
        normed = rms(residual, pre_weight)
        if rotate_rows:
            normed = rotate(normed)
    return residual, normed


def spans(batch, length, offsets):
    if offsets is None:
        return [(b, b, 0, length) for b in range(batch)]
    return [(0, j, offsets[j], offsets[j + 1]) for j in range(len(offsets) - 1)]


def gated_scan(x, r, i, decay, exponent=8.0, initial=None, offsets=None):
    """(h, final) of (B, S, D) float64 tensors, token by token."""
    la = -exponent * torch.nn.functional.softplus(decay, threshold=1e9) * torch.sigmoid(r)
    a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    u = m * torch.sigmoid(i) * x
    batch, length, dim = x.shape
    runs = spans(batch, length, offsets)
    h, final = torch.zeros_like(x), torch.zeros(len(runs), dim, dtype=x.dtype)
    for b, j, start, stop in runs:
        state = torch.zeros(dim, dtype=x.dtype) if initial is None else initial[j]
        for t in range(start, stop):
            state = a[b, t] * state + u[b, t]
            h[b, t] = state
        final[j] = state
    return h, final


def gated_scan_gradients(x, r, i, decay, d_h, d_final, exponent=8.0, initial=None, offsets=None):
    """(dx, dr, di, ddecay, dinitial) by the backward recurrence."""
    sr, si = torch.sigmoid(r), torch.sigmoid(i)
    rate = exponent * torch.nn.functional.softplus(decay, threshold=1e9)
    la = -rate * sr
    a, m = torch.exp(la), torch.sqrt(-torch.expm1(2 * la))
    u = m * si * x
    batch, length, dim = x.shape
    runs = spans(batch, length, offsets)
    g, before = torch.zeros_like(x), torch.zeros_like(x)
    d_initial = torch.zeros(len(runs), dim, dtype=x.dtype)
    for b, j, start, stop in runs:
        state = torch.zeros(dim, dtype=x.dtype) if initial is None else initial[j]
        for t in range(start, stop):
            before[b, t] = state
            state = a[b, t] * state + u[b, t]
        p = torch.zeros(dim, dtype=x.dtype) if d_final is None else d_final[j]
        for t in range(stop - 1, start - 1, -1):
            g[b, t] = d_h[b, t] + p
            p = a[b, t] * g[b, t]
        d_initial[j] = p
    # d m/d la = -a^2/m; with la -> 0 it is only ever used times la, where it vanishes
    ratio = torch.where(m > 0, -la / torch.where(m > 0, m, torch.ones_like(m)), torch.zeros_like(m))
    e = g * (a * before * la + si * x * a * a * ratio)          # dL/d(la) la
    slope = torch.sigmoid(decay) / torch.nn.functional.softplus(decay, threshold=1e9)
    return g * m * si, e * (1 - sr), g * m * x * si * (1 - si), e.sum((0, 1)) * slope, d_initial
