"""Block operators of recurrent language models on torch tensors.

``block_norm``       the boundary between two blocks: norm, gate and residual add of a block's output, and the norm
                     (and Hadamard rotation) that makes the next block's input, in one pass over the rows;
``gated_scan``       the gated linear recurrence along sequences, dense or packed;
``gated_scan_step``  one token of it for a batch of requests with states in a pool.

The calls run on the caller's current CUDA stream, allocate only through torch, never synchronise and can be captured
in CUDA graphs.  ``block_norm`` and ``gated_scan`` are differentiable (once); arithmetic is fp32 whatever the tensors'
type, with one rounding per output.  They take plain tensors: one with a forward-mode tangent, without storage of its
own (DTensor, FakeTensor, under ``torch.func`` transforms) or under a trace (``torch.jit.trace``, ``make_fx``) is
refused.  ``cubutterfly_b200.torch_ops`` exports the operators beside the transforms.

Arguments are checked, outputs allocated and gradients recorded by the extension ``_block_ops``
(csrc/block_ops_torch.cpp), which calls the C entry points of the loaded library.
"""
from __future__ import annotations

import ctypes as ct

import torch  # noqa: F401  (the extension links against its libraries)

import cubutterfly_b200 as cb

try:
    from cubutterfly_b200 import _block_ops
except ImportError as e:
    raise ImportError(f"the torch extension of the block operators is not built or does not load ({e}); build it with "
                      "`python -m cubutterfly_b200._build`") from e

__all__ = ["block_norm", "gated_scan", "gated_scan_step"]

_ENTRIES = ("BlockNormForward", "BlockNormBackward", "BlockNormGetWorkspaceSize", "GatedScanForward",
            "GatedScanBackward", "GatedScanGetWorkspaceSize", "GatedScanStep")


def _bind():
    lib = cb.load()

    def fail(status):
        raise cb.Error(lib.describe(status), status)

    _block_ops.bind(*(ct.cast(lib.fn["B200" + name], ct.c_void_p).value for name in _ENTRIES), fail)


_bind()


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
    return _block_ops.block_norm(x, y, pre_weight, post_weight, gate, gate_activation, residual_scale, eps, pre_norm,
                                 post_norm, rotate, dtype)


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
    return _block_ops.gated_scan(x, recurrence_gate, input_gate, decay, exponent, initial_state, offsets)


def gated_scan_step(state, x, recurrence_gate, input_gate, decay, *, exponent=8.0, slots=None, new_state=None):
    """One token of ``gated_scan`` for a batch of requests: returns h (B, D) and updates the states.

    ``x`` and the gates are (B, D); ``state`` is a pool of fp32 states (P, D), contiguous, updated in place unless
    ``new_state`` (another such pool, apart from it) takes the new rows.  Request b's state is row ``slots[b]`` (int32,
    on the device; row b without ``slots``).  A slot outside the pool, such as -1, marks padding: that request's h is
    zero and no state changes.  Distinct requests need distinct slots.  Inference only: under grad mode no argument may
    require grad.
    """
    return _block_ops.gated_scan_step(state, x, recurrence_gate, input_gate, decay, exponent, slots, new_state)
