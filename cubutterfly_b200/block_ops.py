"""Block operators of recurrent language models on torch tensors.

``block_norm``       the boundary between two blocks: norm, gate and residual add of a block's output, and the norm
                     (and Hadamard rotation) that makes the next block's input, in one pass over the rows;
``gated_scan``       the gated linear recurrence along sequences, dense or packed;
``gated_scan_step``  one token of it for a batch of requests with states in a pool.

The calls run on the caller's current CUDA stream, allocate only through torch, never synchronise and can be captured
in CUDA graphs.  ``block_norm`` and ``gated_scan`` are differentiable (once); arithmetic is fp32 whatever the tensors'
type, with one rounding per output.  ``cubutterfly_b200.torch_ops`` exports them beside the transforms.
"""
from __future__ import annotations

import ctypes as ct
import math
import struct

import torch
from torch.autograd.function import once_differentiable

import cubutterfly_b200 as cb

__all__ = ["block_norm", "gated_scan", "gated_scan_step"]

_TYPES = {torch.bfloat16: int(cb.DataType.BF16), torch.float16: int(cb.DataType.FP16),
          torch.float32: int(cb.DataType.FP32)}
_ACTIVATIONS = {"none": 0, "sigmoid": 1, "silu": 2}
_POST_NORM, _PRE_NORM, _ROTATE = 1, 2, 4
_CHUNK = 16  # tokens per state kept for the backward of gated_scan

# the structs of include/cubutterfly/cubutterfly_b200.h, in field order
_NORM = struct.Struct("@4N8i2d6P3N6P2N6PPN")
_SCAN = struct.Struct("@5N2id3P6N7P2N6PPN")
_STEP = struct.Struct("@4N2id3P3N5P")


def _launch(name, device, packed):
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        cb.load().invoke(name, packed, stream)
    else:
        with torch.cuda.device(device):
            cb.load().invoke(name, packed, stream)


def _workspace(name, device, packed):
    size = ct.c_size_t(0)
    cb.load().invoke(name, packed, ct.byref(size))
    return torch.empty(size.value, dtype=torch.uint8, device=device)


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _check(t, what, dtypes, device=None, shape=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} does not support dtype {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _rows(t, dim):
    """`t` as rows of `dim` consecutive values one stride apart: (tensor to keep alive, row stride)."""
    if not t.is_contiguous():
        try:
            v = t.view(-1, dim)
        except RuntimeError:
            v = None
        if v is not None and v.stride(1) == 1 and v.shape[0] > 1 and v.stride(0) >= dim:
            return v, v.stride(0)
        t = t.contiguous()
    return t, dim


# ---- block norm --------------------------------------------------------------------------------
class _NormCall:
    """The checked arguments of one block_norm call."""

    __slots__ = ("dim", "rows", "block", "stream", "gate_rows", "activation", "flags", "scale", "eps")

    def pack(self, x, y, gate, pre, post, scale, residual=None, normed=None, rms=None, d_residual=None, d_normed=None,
             grads=(None,) * 6, workspace=None):
        dim = self.dim
        x, x_row = _rows(x, dim)
        y, y_row = (None, 0) if y is None else _rows(y, dim)
        gate, gate_row = (None, 0) if gate is None else _rows(gate, dim)
        d_residual, dr_row = (None, 0) if d_residual is None else _rows(d_residual, dim)
        d_normed, dn_row = (None, 0) if d_normed is None else _rows(d_normed, dim)
        block = _TYPES[self.block]
        kind = [block if v is None else _TYPES[v.dtype] for v in (pre, post, scale, gate)]
        post_rms = pre_rms = 0
        if rms is not None:
            post_rms = rms.data_ptr()
            pre_rms = post_rms + 4 * self.rows
        packed = _NORM.pack(_NORM.size, self.rows, dim, self.gate_rows, block, _TYPES[self.stream], *kind, self.flags,
                            self.activation, self.scale, self.eps, _ptr(x), _ptr(y), _ptr(gate), _ptr(pre), _ptr(post),
                            _ptr(scale), x_row, y_row, gate_row, _ptr(residual), _ptr(normed), post_rms, pre_rms,
                            _ptr(d_residual), _ptr(d_normed), dr_row, dn_row, *map(_ptr, grads), _ptr(workspace),
                            0 if workspace is None else workspace.numel())
        return packed, (x, y, gate, d_residual, d_normed)  # copies stay alive until the launch is enqueued

    def forward(self, x, y, gate, pre, post, scale, keep):
        residual = None if y is None else torch.empty(x.shape, dtype=self.stream, device=x.device)
        normed = torch.empty(x.shape, dtype=self.block, device=x.device) if self.flags & _PRE_NORM else None
        rms = torch.empty(2 * self.rows, dtype=torch.float32, device=x.device) if keep else None
        if self.rows:
            packed, _alive = self.pack(x, y, gate, pre, post, scale, residual, normed, rms)
            _launch("B200BlockNormForward", x.device, packed)
        return residual, normed, rms

    def backward(self, x, y, gate, pre, post, scale, rms, d_residual, d_normed):
        grads = [torch.empty(t.shape, dtype=t.dtype, device=t.device) if t is not None else None
                 for t in (x, y, gate, pre, post, scale)]
        if not self.rows or (d_residual is None and d_normed is None):
            return [g if g is None else g.zero_() for g in grads]
        args = (x, y, gate, pre, post, scale)
        packed, _alive = self.pack(*args)
        workspace = _workspace("B200BlockNormGetWorkspaceSize", x.device, packed)
        packed, _alive = self.pack(*args, rms=rms, d_residual=d_residual, d_normed=d_normed, grads=grads,
                                   workspace=workspace)
        _launch("B200BlockNormBackward", x.device, packed)
        return grads


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, x, y, gate, pre, post, scale):
        residual, normed, rms = call.forward(x, y, gate, pre, post, scale, True)
        ctx.call = call
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, y, gate, pre, post, scale, rms)
        return residual, normed

    @staticmethod
    @once_differentiable
    def backward(ctx, d_residual, d_normed):
        *args, rms = ctx.saved_tensors
        return (None, *ctx.call.backward(*args, rms, d_residual, d_normed))


def _gate_rows(gate, x, rows):
    """How many gate rows a gate broadcast to x's shape has: 1, one per group of leading indices, or one per row."""
    shape, full = tuple(gate.shape), tuple(x.shape)
    if shape[-1:] != full[-1:] or len(shape) > len(full):
        raise ValueError(f"gate of shape {shape} does not broadcast over {full}")
    if shape == full:
        return max(rows, 1)
    shape = (1,) * (len(full) - len(shape)) + shape
    lead = 0
    while lead < len(full) - 1 and shape[lead] == full[lead]:
        lead += 1
    if any(n != 1 for n in shape[lead:-1]):
        raise ValueError(f"gate of shape {tuple(gate.shape)} must be one per channel, or equal to x's {full} in its "
                         "leading dimensions and 1 in the others")
    return math.prod(shape[:-1])


def block_norm(x, y=None, *, pre_weight=None, post_weight=None, gate=None, gate_activation="none", residual_scale=1.0,
               eps=1e-6, pre_norm=True, post_norm=True, rotate=False, dtype=None):
    """The boundary between two blocks: returns (residual, normed).

    With r(v) = 1/sqrt(mean(v^2) + eps) over the last axis::

        n        = y r(y) post_weight                       (n = y with post_norm=False)
        residual = residual_scale x + act(gate) n
        normed   = residual r(residual) pre_weight          (None with pre_norm=False)
        normed   = normed H_D / sqrt(D)                     (with rotate=True, torch_ops.hadamard_rotate)

    ``x`` is the residual stream (bf16, fp16 or fp32), ``y`` the block's output: the same shape, and x's type or, with
    an fp32 stream, bf16 or fp16.  ``residual`` has x's type, ``normed`` y's.  Without ``y`` (the norm before the first
    block) ``residual`` is x itself and ``normed`` has type ``dtype`` (default x's).  The second norm is taken of the
    sum before it is rounded.  ``gate`` is None, one value per channel (D,), one row per leading index ((B, 1, D) for
    x of (B, S, D)) or of x's shape; ``gate_activation`` is "none", "sigmoid" or "silu".  ``residual_scale`` is a
    number or a tensor (D,).  Vectors may be fp32 or y's type; a gate per row has y's type.  D is at most 16384, with
    ``rotate`` a power of two from 64.  Differentiable in every tensor argument.
    """
    _check(x, "block_norm: x", _TYPES)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("block_norm requires a non-empty last dimension")
    call = _NormCall()
    call.stream, device, dim = x.dtype, x.device, x.shape[-1]
    if y is None:
        if gate is not None or post_weight is not None:
            raise ValueError("block_norm: gate and post_weight need a block output y")
        if isinstance(residual_scale, torch.Tensor) or residual_scale != 1.0:
            raise ValueError("block_norm: residual_scale needs a block output y")
        if not pre_norm:
            raise ValueError("block_norm: without y and pre_norm there is nothing to compute")
        call.block, post_norm = dtype or x.dtype, False
        if call.block not in _TYPES:
            raise ValueError(f"block_norm does not support dtype {call.block}")
    else:
        _check(y, "block_norm: y", _TYPES, device, x.shape)
        call.block = y.dtype
        if dtype not in (None, y.dtype):
            raise ValueError("block_norm: dtype is y's when y is given")
    if call.stream not in (call.block, torch.float32):
        raise ValueError(f"block_norm: the residual stream must have the block's type {call.block} or float32, "
                         f"got {call.stream}")
    if post_weight is not None and not post_norm or pre_weight is not None and not pre_norm:
        raise ValueError("block_norm: a weight of a norm that is turned off")
    if rotate and not pre_norm:
        raise ValueError("block_norm: rotate needs pre_norm")
    if gate_activation not in _ACTIVATIONS:
        raise ValueError(f"block_norm: gate_activation must be one of {sorted(_ACTIVATIONS)}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("block_norm: eps must be finite and not negative")
    call.dim, call.rows = dim, x.numel() // dim
    call.eps, call.activation = float(eps), _ACTIVATIONS[gate_activation]
    call.flags = (_POST_NORM if post_norm else 0) | (_PRE_NORM if pre_norm else 0) | (_ROTATE if rotate else 0)
    call.scale, scale = 1.0, None
    if isinstance(residual_scale, torch.Tensor):
        scale = residual_scale
    else:
        call.scale = float(residual_scale)
        if not math.isfinite(call.scale):
            raise ValueError("block_norm: residual_scale must be finite")
    vectors = (call.block, torch.float32)
    for name, v in (("pre_weight", pre_weight), ("post_weight", post_weight), ("residual_scale", scale)):
        if v is not None:
            _check(v, f"block_norm: {name}", vectors, device, (dim,))
    call.gate_rows = 0
    if gate is not None:
        _check(gate, "block_norm: gate", vectors, device)
        call.gate_rows = _gate_rows(gate, x, call.rows)
        if call.gate_rows == call.rows and call.rows > 1 and gate.dtype != call.block:
            raise ValueError(f"block_norm: a gate per row must have the block's type {call.block}")
    tensors = (x, y, gate, pre_weight, post_weight, scale)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        residual, normed = _BlockNorm.apply(call, x, y, gate, *(_contiguous(v) for v in tensors[3:]))
    else:
        residual, normed, _ = call.forward(x, y, gate, *(_contiguous(v) for v in tensors[3:]), False)
    return x if y is None else residual, normed


def _contiguous(v):
    return v if v is None else v.contiguous()


# ---- gated scan --------------------------------------------------------------------------------
def _tokens(t, dim):
    """(tensor to keep alive, batch stride, token stride) of a (batch, tokens, dim) tensor with adjacent channels."""
    batch, length, _ = t.shape
    token = t.stride(1) if length > 1 else dim
    if (dim > 1 and t.stride(2) != 1) or token < dim:
        t = t.contiguous()
        token = dim
    return t, (t.stride(0) if batch > 1 else 0), token


class _ScanCall:
    __slots__ = ("batch", "length", "dim", "sequences", "dtype", "exponent", "offsets")

    def chunks(self):
        return self.batch * ((self.length + _CHUNK - 1) // _CHUNK)

    def pack(self, x, r, i, decay, initial, h=None, final=None, chunk_states=None, d_h=None, d_final=None,
             grads=(None,) * 5, workspace=None):
        dim = self.dim
        alive, strides = [], []
        for t in (x, r, i):
            t, batch, token = _tokens(t, dim)
            alive.append(t)
            strides += (batch, token)
        dh_strides = (0, 0)
        if d_h is not None:
            d_h, *dh_strides = _tokens(d_h, dim)
            alive.append(d_h)
        packed = _SCAN.pack(_SCAN.size, self.batch, self.length, dim, self.sequences, _TYPES[self.dtype], 0,
                            self.exponent, *map(_ptr, alive[:3]), *strides, _ptr(decay), _ptr(initial),
                            _ptr(self.offsets), _ptr(h), _ptr(final), _ptr(chunk_states), _ptr(d_h), *dh_strides,
                            _ptr(d_final), *map(_ptr, grads), _ptr(workspace),
                            0 if workspace is None else workspace.numel())
        return packed, alive

    def forward(self, x, r, i, decay, initial, keep):
        h = torch.empty((self.batch, self.length, self.dim), dtype=self.dtype, device=x.device)
        states = (self.sequences or self.batch, self.dim)
        if not self.length or not self.batch:  # no tokens: the states stay as they are
            final = torch.zeros(states, dtype=torch.float32, device=x.device)
            return h, final if initial is None else final.copy_(initial), None
        final = torch.empty(states, dtype=torch.float32, device=x.device)
        chunk_states = None
        if keep:
            chunk_states = torch.empty((self.chunks(), self.dim), dtype=torch.float32, device=x.device)
        packed, _alive = self.pack(x, r, i, decay, initial, h, final, chunk_states)
        _launch("B200GatedScanForward", x.device, packed)
        return h, final, chunk_states

    def backward(self, x, r, i, decay, initial, chunk_states, d_h, d_final):
        shape = (self.batch, self.length, self.dim)
        grads = [torch.empty(shape, dtype=self.dtype, device=x.device) for _ in range(3)]
        grads.append(torch.empty_like(decay))
        grads.append(None if initial is None else torch.empty_like(initial))
        if not self.length or not self.batch:
            grads[3].zero_()
            if initial is not None:
                grads[4] = torch.zeros_like(initial) if d_final is None else d_final.clone()
            return grads
        if d_h is None:
            d_h = torch.zeros(shape, dtype=self.dtype, device=x.device)
        if d_final is not None:
            d_final = d_final.contiguous()
        args = (x, r, i, decay, initial)
        packed, _alive = self.pack(*args)
        workspace = _workspace("B200GatedScanGetWorkspaceSize", x.device, packed)
        packed, _alive = self.pack(*args, chunk_states=chunk_states, d_h=d_h, d_final=d_final, grads=grads,
                                   workspace=workspace)
        _launch("B200GatedScanBackward", x.device, packed)
        return grads


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, call, x, r, i, decay, initial):
        h, final, chunk_states = call.forward(x, r, i, decay, initial, True)
        ctx.call = call
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, r, i, decay, initial, chunk_states, call.offsets)
        return h, final

    @staticmethod
    @once_differentiable
    def backward(ctx, d_h, d_final):
        x, r, i, decay, initial, chunk_states, _ = ctx.saved_tensors
        if d_h is None and d_final is None:
            return (None,) * 6
        return (None, *ctx.call.backward(x, r, i, decay, initial, chunk_states, d_h, d_final))


def _check_exponent(exponent, what):
    if not (math.isfinite(exponent) and exponent > 0):
        raise ValueError(f"{what}: exponent must be finite and positive")
    return float(exponent)


def gated_scan(x, recurrence_gate, input_gate, decay, *, exponent=8.0, initial_state=None, offsets=None):
    """The gated linear recurrence along sequences: returns (h, final_state).

    Per channel, with a_t = exp(-exponent softplus(decay) sigmoid(recurrence_gate_t))::

        h_t = a_t h_{t-1} + sqrt(1 - a_t^2) sigmoid(input_gate_t) x_t

    ``x`` and the gates are (B, S, D) of one type (bf16, fp16 or fp32), ``h`` too; rows may be strided (slices of one
    projection).  ``decay`` is (D,); the states are fp32 (B, D), ``initial_state`` zero unless given.  With ``offsets``
    (int32 on the device, n + 1 ascending values from 0 to T) the batch is packed: x is (T, D) or (1, T, D), sequence j
    the tokens offsets[j] .. offsets[j + 1] - 1 (there may be none: its final state is its initial one), the states are
    (n, D), and nothing of one sequence, NaN included, reaches another.  Differentiable in x, both gates, decay and
    initial_state.
    """
    _check(x, "gated_scan: x", _TYPES)
    call = _ScanCall()
    call.offsets, call.sequences, shape = offsets, 0, x.shape
    if offsets is not None:
        _check(offsets, "gated_scan: offsets", (torch.int32,), x.device)
        if offsets.ndim != 1 or offsets.numel() < 2:
            raise ValueError("gated_scan: offsets must hold n + 1 values, n at least 1")
        if not (x.ndim == 2 or (x.ndim == 3 and x.shape[0] == 1)):
            raise ValueError("gated_scan: a packed batch is (T, D) or (1, T, D)")
        call.offsets = offsets.contiguous()
        call.sequences = offsets.numel() - 1
    elif x.ndim != 3:
        raise ValueError("gated_scan: x must be (B, S, D), or packed with offsets")
    if shape[-1] < 1:
        raise ValueError("gated_scan requires a non-empty last dimension")
    for name, t in (("recurrence_gate", recurrence_gate), ("input_gate", input_gate)):
        _check(t, f"gated_scan: {name}", (x.dtype,), x.device, shape)
    inputs = (x, recurrence_gate, input_gate)
    if x.ndim == 2:
        inputs = tuple(t.unsqueeze(0) for t in inputs)
    call.batch, call.length, call.dim = inputs[0].shape
    call.dtype, call.exponent = x.dtype, _check_exponent(exponent, "gated_scan")
    _check(decay, "gated_scan: decay", _TYPES, x.device, (call.dim,))
    decay = decay.float().contiguous()
    if initial_state is not None:
        _check(initial_state, "gated_scan: initial_state", (torch.float32,), x.device,
               (call.sequences or call.batch, call.dim))
        initial_state = initial_state.contiguous()
    tensors = (*inputs, decay, initial_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        h, final = _GatedScan.apply(call, *tensors)
    else:
        h, final, _ = call.forward(*tensors, False)
    return (h.squeeze(0) if x.ndim == 2 else h), final


def gated_scan_step(state, x, recurrence_gate, input_gate, decay, *, exponent=8.0, slots=None, new_state=None):
    """One token of ``gated_scan`` for a batch of requests: returns h (B, D) and updates the states.

    ``x`` and the gates are (B, D); ``state`` is a pool of fp32 states (P, D), contiguous, updated in place unless
    ``new_state`` (another such pool) takes the new rows.  Request b's state is row ``slots[b]`` (int32, on the device;
    row b without ``slots``).  A slot outside the pool, such as -1, marks padding: that request's h is zero and no
    state changes.  Distinct requests need distinct slots.  Inference only.
    """
    _check(x, "gated_scan_step: x", _TYPES)
    if x.ndim != 2 or x.shape[1] < 1:
        raise ValueError("gated_scan_step: x must be (B, D)")
    batch, dim = x.shape
    device, dtype = x.device, x.dtype
    for name, t in (("recurrence_gate", recurrence_gate), ("input_gate", input_gate)):
        _check(t, f"gated_scan_step: {name}", (dtype,), device, (batch, dim))
    _check(decay, "gated_scan_step: decay", _TYPES, device, (dim,))
    decay = decay.detach().float().contiguous()
    new_state = state if new_state is None else new_state
    for name, t in (("state", state), ("new_state", new_state)):
        _check(t, f"gated_scan_step: {name}", (torch.float32,), device)
        if t.ndim != 2 or t.shape[1] != dim or not t.is_contiguous():
            raise ValueError(f"gated_scan_step: {name} must be a contiguous (slots, {dim}) pool")
    if new_state.shape != state.shape:
        raise ValueError("gated_scan_step: new_state must have the shape of state")
    if slots is not None:
        _check(slots, "gated_scan_step: slots", (torch.int32,), device, (batch,))
        slots = slots.contiguous()
    elif state.shape[0] < batch:
        raise ValueError(f"gated_scan_step: {batch} requests without slots need a pool of as many rows")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (state, x, recurrence_gate, input_gate)):
        raise ValueError("gated_scan_step is inference only: an input requires grad")
    exponent = _check_exponent(exponent, "gated_scan_step")
    h = torch.empty((batch, dim), dtype=dtype, device=device)
    if batch:
        alive = [_rows(t, dim) for t in (x, recurrence_gate, input_gate)]
        packed = _STEP.pack(_STEP.size, batch, dim, state.shape[0], _TYPES[dtype], 0, exponent,
                            *(t.data_ptr() for t, _ in alive), *(row for _, row in alive), decay.data_ptr(),
                            state.data_ptr(), new_state.data_ptr(), _ptr(slots), h.data_ptr())
        _launch("B200GatedScanStep", device, packed)
    return h
