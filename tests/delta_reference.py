"""The gated delta rule and the norm of queries and keys by their definitions, in 64 bits on the CPU, and the bounds that the
kernels are held to (beside one rounding of an output to its type; see block_reference)."""
import torch

from block_reference import assert_close  # noqa: F401

# Products take fp32 values as two bf16 pieces beside 16-bit tensors, each within 2^-16 of itself, and three (2^-24) beside
# fp32 ones, where the accumulation's truncation, 2^-23 of the largest partial sum a step of 16 terms, is what remains.  From
# an input to an output lie at most 8 such products forward and as many more backward, each with two split operands; the
# errors that tokens leave in the state decay with it.
DELTA_LOSS = {torch.bfloat16: 16 * 2.0 ** -16, torch.float16: 16 * 2.0 ** -16, torch.float32: 16 * 8 * 2.0 ** -23}
# A step is fp32 arithmetic: sums of 128 products, two of them in turn.
STEP_LOSS = 256 * 2.0 ** -24
# Sums of 256 squares in a tree, a square root, a division, the angle's 2e-7 and the sine's two units.
NORM_LOSS = 32 * 2.0 ** -24


def gated_delta(q, k, v, log_decay, beta, *, scale=None, initial_state=None, cuts=None):
    """(B, S, heads, channels) tensors of float64; `cuts` of a packed batch, whose tensors have no batch dimension."""
    if cuts is None:
        outs = [_sequence(q[b], k[b], v[b], log_decay[b], beta[b], scale, None if initial_state is None else initial_state[b])
                for b in range(q.shape[0])]
        return torch.stack([o for o, _ in outs]), torch.stack([s for _, s in outs])
    outs = [_sequence(*(t[a:e] for t in (q, k, v, log_decay, beta)), scale, None if initial_state is None else initial_state[j])
            for j, (a, e) in enumerate(zip(cuts, cuts[1:]))]
    return torch.cat([o for o, _ in outs]), torch.stack([s for _, s in outs])


def _sequence(q, k, v, log_decay, beta, scale, state):
    group = v.shape[1] // k.shape[1]
    scale = k.shape[-1] ** -0.5 if scale is None else scale
    q, k = q.repeat_interleave(group, 1), k.repeat_interleave(group, 1)
    if state is None:
        state = torch.zeros(v.shape[1], k.shape[-1], v.shape[-1], dtype=v.dtype)
    rows = []
    for t in range(q.shape[0]):
        state = state * log_decay[t].exp()[:, None, None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", state, k[t]))
        state = state + k[t][:, :, None] * u[:, None, :]
        rows.append(scale * torch.einsum("hkv,hk->hv", state, q[t]))
    return torch.stack(rows) if rows else v.new_zeros(v.shape), state


def qk_norm(x, weight=None, *, norm="rms", eps=1e-6, positions=None, frequencies=None, axes=None, interleaved=False):
    """One of the two tensors, (..., heads, D)."""
    squares = x.square()
    y = x / torch.sqrt((squares.mean(-1, keepdim=True) if norm == "rms" else squares.sum(-1, keepdim=True)) + eps)
    if weight is not None:
        y = y * weight
    if positions is None:
        return y
    at = positions.double()
    at = at[..., None].expand(*at.shape, frequencies.numel()) if axes is None else at[axes.long()].movedim(0, -1)
    angle = (at * frequencies.double())[..., None, :]
    pairs = frequencies.numel()
    a, b = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if interleaved else (y[..., :pairs], y[..., pairs:2 * pairs])
    c, s = angle.cos(), angle.sin()
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., 2 * pairs:]), -1)
