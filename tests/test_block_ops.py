"""What the block operators refuse, on any host: the torch frontend's argument checks, and the C entry points' (checked
before anything is launched)."""
import ctypes as ct
import math
import struct
from pathlib import Path

import pytest
import torch

import cubutterfly_b200 as cb
from cubutterfly_b200 import block_ops, torch_ops

STATUS = cb.Status

# the structs of include/cubutterfly/cubutterfly_b200.h, in field order
NORM = struct.Struct("@4N8i2d6P3N6P2N6PPN")
SCAN = struct.Struct("@5N2id3P6N7P2N6PPN")
STEP = struct.Struct("@4N2id3P3N5P")


def test_cpu_tensors_are_rejected():
    x = torch.randn(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        torch_ops.block_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        torch_ops.gated_scan(x[None], x[None], x[None], x[0])
    with pytest.raises(ValueError, match="CUDA"):
        torch_ops.gated_scan_step(x, x, x, x, x[0])


def test_forward_mode_tangents_are_refused():
    """A tangent would be dropped, which reads as a derivative of zero."""
    import torch.autograd.forward_ad as fwd

    zeros = torch.zeros(4, 64, device="meta")  # no CUDA tensor either: the tangent is looked at first
    with fwd.dual_level():
        dual = fwd.make_dual(torch.zeros(4, 64), torch.ones(4, 64))
        with pytest.raises(ValueError, match="x carries a forward-mode tangent"):
            torch_ops.block_norm(dual)
        with pytest.raises(ValueError, match="x carries a forward-mode tangent"):
            torch_ops.gated_scan(dual[None], zeros, zeros, zeros)
        with pytest.raises(ValueError, match="x carries a forward-mode tangent"):
            torch_ops.gated_scan_step(zeros, dual, zeros, zeros, zeros)
        with fwd._set_fwd_grad_enabled(False), pytest.raises(ValueError, match="CUDA"):
            torch_ops.block_norm(dual)


class Wrapper(torch.Tensor):
    """A tensor whose values are somewhere else: the data pointer is null."""
    @staticmethod
    def __new__(cls, *shape):
        return torch.Tensor._make_wrapper_subclass(cls, shape, device="cuda", dtype=torch.float32)

    def __init__(self, *shape):
        pass

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError(func)


def test_wrapper_tensors_are_refused():
    """A wrapped weight's data pointer is null, as that of a weight left out."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    x = torch.zeros(4, 64)
    with FakeTensorMode():
        fake = torch.empty(4, 64, device="cuda")
    for v in (Wrapper(4, 64), fake):
        for call in (lambda: torch_ops.block_norm(v), lambda: torch_ops.gated_scan(v, x, x, x),
                     lambda: torch_ops.gated_scan_step(x, v, x, x, x)):
            with pytest.raises(ValueError, match="x must be a CUDA tensor with storage of its own"):
                call()
    for transform in (torch.func.vmap, torch.func.grad):
        with pytest.raises(ValueError, match="storage of its own"):
            transform(lambda v: torch_ops.block_norm(v)[1])(x)


def test_traces_are_refused():
    """A trace would record the outputs as constants, or as the empty tensors they begin as."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.zeros(4, 64)
    for call in (lambda v: torch_ops.block_norm(v)[1], lambda v: torch_ops.gated_scan(v, v, v, v)[0],
                 lambda v: torch_ops.gated_scan_step(v, v, v, v, v)):
        with pytest.raises(ValueError, match="x is being traced"):
            torch.jit.trace(call, (x,))
        with pytest.raises(ValueError, match="x is being traced"):
            make_fx(call)(x)


def test_torch_ops_exports_the_block_operators():
    for name in ("block_norm", "gated_scan", "gated_scan_step"):
        assert name in torch_ops.__all__ and getattr(torch_ops, name) is getattr(block_ops, name)
    with pytest.raises(AttributeError):
        torch_ops.no_such_operator


def test_gate_shapes():
    """A gate is one row per channel vector, leading index or row; what does not broadcast so is refused."""
    x = torch.empty(6, 5, 8)
    rows = lambda *shape: block_ops._block_ops.gate_rows(torch.empty(*shape), x, 30)
    assert rows(8) == rows(1, 8) == rows(1, 1, 8) == 1
    assert rows(6, 1, 8) == 6 and rows(6, 5, 8) == 30
    for shape in ((6, 5, 1), (5, 8), (1, 5, 8), (2, 1, 8), (6, 8), (1, 6, 5, 8), (4,)):
        with pytest.raises(ValueError, match="gate"):
            rows(*shape)


def test_row_strides():
    t = torch.empty(4, 6, 16)
    assert block_ops._block_ops.rows(t, 16)[1] == 16
    assert block_ops._block_ops.rows(t[..., :8], 8)[1] == 16            # collapses to rows 16 apart
    assert block_ops._block_ops.rows(t[:, :3, :8], 8)[0].is_contiguous()  # two strides: copied
    assert block_ops._block_ops.rows(t.transpose(0, 2), 4)[1] == 4
    assert block_ops._block_ops.rows(torch.empty(1, 16).expand(5, 16), 16)[1] == 16
    assert block_ops._block_ops.tokens(t[..., :8], 8)[1:] == (96, 16)
    assert block_ops._block_ops.tokens(t[:1, :, :8], 8)[1:] == (0, 16)
    assert block_ops._block_ops.tokens(torch.empty(4, 1, 16).expand(4, 6, 16), 16)[1:] == (96, 16)


# (shape of the values, shape they are broadcast to)
BROADCASTS = [((1, 16), (5, 16)), ((3, 1, 16), (3, 5, 16)), ((16,), (3, 5, 16)), ((1, 5, 16), (3, 5, 16)),
              ((1, 1, 16), (3, 1, 16)), ((2, 1, 3, 16), (2, 4, 3, 16)), ((2, 3, 1, 16), (2, 3, 4, 16)), ((1, 1), (5, 1))]


@pytest.mark.parametrize("small,wide", BROADCASTS)
def test_broadcast_rows_are_copied(small, wide):
    """Rows that share memory have no stride of their own; so has the gradient of a sum over rows."""
    dim = wide[-1]
    base = torch.randn(*small)
    for t in (base.expand(*wide), base.expand(*wide).unsqueeze(0)):
        rows, stride = block_ops._block_ops.rows(t, dim)
        assert stride == dim and rows.is_contiguous() and torch.equal(rows, t)
        assert rows.untyped_storage().nbytes() >= 4 * t.numel()
    seen = []
    v = torch.zeros(*wide, requires_grad=True)
    w = v * 1
    w.register_hook(seen.append)
    (w.sum_to_size(*small) * base).sum().backward()
    rows, stride = block_ops._block_ops.rows(seen[0], dim)
    assert stride == dim and rows.is_contiguous() and torch.equal(rows, seen[0])
    assert rows.untyped_storage().nbytes() >= 4 * v.numel()


def test_overlapping_rows_are_copied():
    base = torch.randn(200)
    for size, strides in (((5, 16), (4, 1)), ((4, 1, 16), (7, 3, 1)), ((2, 5, 16), (75, 15, 1))):
        t = base.as_strided(size, strides)
        rows, stride = block_ops._block_ops.rows(t, 16)
        assert stride == 16 and rows.is_contiguous() and torch.equal(rows, t)
    one = base.as_strided((1, 3, 16), (0, 20, 1))   # a stride of a single index means nothing
    rows, stride = block_ops._block_ops.rows(one, 16)
    assert stride == 20 and rows.data_ptr() == base.data_ptr()


def test_polynomial_of_the_decay():
    """(2^f - 1)/f over [-1/2, 1/2] with the coefficients that the kernels hold: the bound stated beside them."""
    import re
    import numpy as np

    source = (Path(cb.__file__).parent / "csrc" / "gated_scan.cuh").read_text()
    body = source[source.index("CUBF_DEV void decay("):]
    body = body[:body.index("\n}\n")]
    coefficients = [float(np.float32(c)) for c in re.findall(r"both\((0\.\d+)f\)", body)]
    assert len(coefficients) == 6
    f = np.linspace(-0.5, 0.5, 200001)
    f = f[f != 0]
    p = np.polyval(coefficients, f)
    assert np.abs(p * f / np.expm1(f * math.log(2)) - 1).max() <= 2.15e-8
    assert np.abs((1 + f * p) / 2 ** f - 1).max() <= 6.6e-9


# Fields of a valid call; device pointers are never dereferenced by the checks.
P = 4096


def norm_fields(**change):
    f = dict(size=NORM.size, rows=4, dim=64, gate_rows=0, data=1, residual_type=1, pre_type=2, post_type=2,
             scale_type=2, gate_type=2, flags=3, activation=0, scale=1.0, eps=1e-6, x=P, y=P * 2, gate=0, pre=0, post=0,
             scales=0, x_row=64, y_row=64, gate_row=0, residual=P * 3, normed=P * 4, post_rms=0, pre_rms=0, d_res=0,
             d_normed=0, dr_row=0, dn_row=0, d_x=0, d_y=0, d_gate=0, d_pre=0, d_post=0, d_scale=0, workspace=0, bytes=0)
    unknown = set(change) - set(f)
    assert not unknown
    return NORM.pack(*{**f, **change}.values())


def scan_fields(**change):
    f = dict(size=SCAN.size, batch=2, length=10, dim=64, sequences=0, data=1, reserved=0, exponent=8.0, x=P,
             r=P, i=P, xb=640, xt=64, rb=640, rt=64, ib=640, it=64, decay=P, initial=0, offsets=0, h=2 * P,
             final=3 * P, chunks=0, d_h=0, db=0, dt=0, d_final=0, d_x=0, d_r=0, d_i=0, d_decay=0, d_initial=0,
             workspace=0, bytes=0)
    assert not set(change) - set(f)
    return SCAN.pack(*{**f, **change}.values())


def step_fields(**change):
    f = dict(size=STEP.size, batch=2, dim=64, pool=2, data=1, reserved=0, exponent=8.0, x=P, r=P, i=P,
             x_row=64, r_row=64, i_row=64, decay=P, state=P, new_state=P, slots=0, h=P)
    assert not set(change) - set(f)
    return STEP.pack(*{**f, **change}.values())


def refused(lib, name, packed, status, text):
    assert lib.fn[name](packed, None) == status
    assert text in lib.fn["GetLastErrorString"]().decode()


@pytest.mark.parametrize("change,status,text", [
    (dict(size=8), STATUS.INVALID_VALUE, "struct_size"),
    (dict(dim=0), STATUS.INVALID_VALUE, "dim"),
    (dict(dim=16385, x_row=16385, y_row=16385), STATUS.NOT_SUPPORTED, "16384"),
    (dict(rows=1 << 31), STATUS.NOT_SUPPORTED, "rows"),
    (dict(data=3), STATUS.NOT_SUPPORTED, "data_type"),
    (dict(data=2, residual_type=1), STATUS.NOT_SUPPORTED, "residual_type"),
    (dict(x=0), STATUS.INVALID_VALUE, "null x"),
    (dict(y=0), STATUS.INVALID_VALUE, "block output"),
    (dict(x_row=63), STATUS.INVALID_VALUE, "stride"),
    (dict(y_row=1), STATUS.INVALID_VALUE, "stride"),
    (dict(x=P + 1), STATUS.INVALID_VALUE, "misaligned"),
    (dict(gate=P), STATUS.INVALID_VALUE, "gate_rows"),
    (dict(gate=P, gate_rows=3, gate_row=64), STATUS.INVALID_VALUE, "divisor"),
    (dict(gate=P, gate_rows=2, gate_row=8), STATUS.INVALID_VALUE, "stride"),
    (dict(gate=P, gate_rows=1, gate_type=0), STATUS.NOT_SUPPORTED, "gate_type"),
    (dict(pre=P + 2), STATUS.INVALID_VALUE, "misaligned"),
    (dict(flags=1, normed=0, pre=P), STATUS.INVALID_VALUE, "PRE_NORM"),
    (dict(flags=2, post=P), STATUS.INVALID_VALUE, "POST_NORM"),
    (dict(flags=9), STATUS.INVALID_VALUE, "flags"),
    (dict(flags=5, normed=0), STATUS.INVALID_VALUE, "ROTATE"),
    (dict(flags=7, dim=60, x_row=60, y_row=60), STATUS.NOT_SUPPORTED, "power-of-two"),
    (dict(flags=7, dim=32), STATUS.NOT_SUPPORTED, "power-of-two"),
    (dict(normed=0), STATUS.INVALID_VALUE, "normed"),
    (dict(normed=P), STATUS.INVALID_VALUE, "alias"),
    (dict(residual=2 * P), STATUS.INVALID_VALUE, "alias"),
    (dict(residual=P, x_row=65), STATUS.INVALID_VALUE, "in-place"),
    (dict(post_rms=P), STATUS.INVALID_VALUE, "pre_rms"),
    (dict(activation=3), STATUS.INVALID_VALUE, "activation"),
    (dict(eps=-1.0), STATUS.INVALID_VALUE, "epsilon"),
    (dict(eps=math.nan), STATUS.INVALID_VALUE, "epsilon"),
    (dict(scale=math.inf), STATUS.INVALID_VALUE, "residual_scale"),
])
def test_block_norm_refusals(lib, change, status, text):
    refused(lib, "B200BlockNormForward", norm_fields(**change), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(d_x=0), STATUS.INVALID_VALUE, "d_x"),
    (dict(d_y=0), STATUS.INVALID_VALUE, "d_y"),
    (dict(pre=P), STATUS.INVALID_VALUE, "its gradient"),
    (dict(d_normed=P, dn_row=1), STATUS.INVALID_VALUE, "stride"),
    (dict(post_rms=0), STATUS.INVALID_VALUE, "post_rms"),
    (dict(d_normed=P, dn_row=64, pre_rms=0), STATUS.INVALID_VALUE, "pre_rms"),
    (dict(workspace=0), STATUS.INVALID_VALUE, "workspace"),
    (dict(bytes=16), STATUS.INVALID_VALUE, "workspace"),
    (dict(rows=0), STATUS.NOT_SUPPORTED, "zero rows"),
    (dict(dim=16384, x_row=16384, y_row=16384, dr_row=16384, rows=1 << 23, gate=P, d_gate=P, gate_rows=1 << 22,
          gate_row=16384), STATUS.NOT_SUPPORTED, "gate groups"),
])
def test_block_norm_backward_refusals(lib, change, status, text):
    valid = dict(post_rms=P, pre_rms=P, d_res=P, dr_row=64, d_x=P, d_y=P, workspace=P, bytes=1 << 20)
    refused(lib, "B200BlockNormBackward", norm_fields(**{**valid, **change}), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(size=0), STATUS.INVALID_VALUE, "struct_size"),
    (dict(dim=0), STATUS.INVALID_VALUE, "dim"),
    (dict(length=(1 << 30) + 1), STATUS.NOT_SUPPORTED, "2^30"),
    (dict(data=9), STATUS.NOT_SUPPORTED, "data_type"),
    (dict(exponent=0.0), STATUS.INVALID_VALUE, "exponent"),
    (dict(exponent=math.nan), STATUS.INVALID_VALUE, "exponent"),
    (dict(x=0), STATUS.INVALID_VALUE, "null input"),
    (dict(r=P + 1), STATUS.INVALID_VALUE, "misaligned"),
    (dict(decay=0), STATUS.INVALID_VALUE, "decay"),
    (dict(final=0), STATUS.INVALID_VALUE, "final_state"),
    (dict(h=0), STATUS.INVALID_VALUE, "null or misaligned h"),
    (dict(h=P), STATUS.INVALID_VALUE, "alias"),
    (dict(xt=63), STATUS.INVALID_VALUE, "stride"),
    (dict(initial=3 * P), STATUS.INVALID_VALUE, "alias"),
    (dict(offsets=P, sequences=3), STATUS.INVALID_VALUE, "packed"),
    (dict(offsets=P, batch=1), STATUS.INVALID_VALUE, "packed"),
    (dict(sequences=3), STATUS.INVALID_VALUE, "without offsets"),
    (dict(length=0), STATUS.NOT_SUPPORTED, "zero tokens"),
])
def test_gated_scan_refusals(lib, change, status, text):
    refused(lib, "B200GatedScanForward", scan_fields(**change), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(chunks=0), STATUS.INVALID_VALUE, "chunk_states"),
    (dict(d_h=0), STATUS.INVALID_VALUE, "d_h"),
    (dict(d_i=0), STATUS.INVALID_VALUE, "null gradient"),
    (dict(dt=8), STATUS.INVALID_VALUE, "stride"),
    (dict(d_decay=0), STATUS.INVALID_VALUE, "d_decay"),
    (dict(workspace=P + 4), STATUS.INVALID_VALUE, "workspace"),
    (dict(bytes=0), STATUS.INVALID_VALUE, "workspace"),
    (dict(batch=0), STATUS.NOT_SUPPORTED, "zero tokens"),
])
def test_gated_scan_backward_refusals(lib, change, status, text):
    valid = dict(chunks=P, d_h=P, db=640, dt=64, d_x=P, d_r=P, d_i=P, d_decay=P, workspace=P, bytes=1 << 20)
    refused(lib, "B200GatedScanBackward", scan_fields(**{**valid, **change}), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(size=1), STATUS.INVALID_VALUE, "struct_size"),
    (dict(dim=0), STATUS.INVALID_VALUE, "dim"),
    (dict(data=4), STATUS.NOT_SUPPORTED, "data_type"),
    (dict(exponent=-8.0), STATUS.INVALID_VALUE, "exponent"),
    (dict(h=0), STATUS.INVALID_VALUE, "null tensor"),
    (dict(state=0), STATUS.INVALID_VALUE, "null state"),
    (dict(pool=1), STATUS.INVALID_VALUE, "pool"),
    (dict(x_row=2), STATUS.INVALID_VALUE, "stride"),
    (dict(state=P + 2), STATUS.INVALID_VALUE, "misaligned"),
])
def test_gated_scan_step_refusals(lib, change, status, text):
    refused(lib, "B200GatedScanStep", step_fields(**change), status, text)


@pytest.mark.parametrize("change,text", [
    (dict(post_rms=P + 2), "misaligned post_rms"),
    (dict(pre_rms=P + 1), "misaligned post_rms"),
    (dict(gate=P, gate_rows=1, d_gate=P + 2), "misaligned gradient of a gate"),
    (dict(gate=P, gate_rows=4, gate_row=64, d_gate=P + 1), "misaligned gradient of a gate"),
    (dict(pre=P, d_pre=P + 2), "misaligned gradient of a gate"),
    (dict(post=P, post_type=1, d_post=P + 1), "misaligned gradient of a gate"),
    (dict(scales=P, d_scale=P + 3), "misaligned gradient of a gate"),
])
def test_block_norm_backward_refuses_misaligned_vectors(lib, change, text):
    valid = dict(post_rms=P, pre_rms=P, d_res=P, dr_row=64, d_x=P, d_y=P, workspace=P, bytes=1 << 20)
    refused(lib, "B200BlockNormBackward", norm_fields(**{**valid, **change}), STATUS.INVALID_VALUE, text)


def test_forward_and_scan_refuse_misaligned_vectors(lib):
    refused(lib, "B200BlockNormForward", norm_fields(post_rms=P + 2, pre_rms=P), STATUS.INVALID_VALUE,
            "misaligned post_rms")
    valid = dict(chunks=P, d_h=P, db=640, dt=64, d_x=P, d_r=P, d_i=P, workspace=P, bytes=1 << 20)
    refused(lib, "B200GatedScanBackward", scan_fields(**valid, d_decay=P + 2), STATUS.INVALID_VALUE, "misaligned")


@pytest.mark.parametrize("rows", [-1, 1])
def test_gated_scan_step_refuses_overlapping_pools(lib, rows):
    """A new pool some rows beside the old one: a request's state could be overwritten before it is read."""
    refused(lib, "B200GatedScanStep", step_fields(state=P, new_state=P + rows * 64 * 4), STATUS.INVALID_VALUE, "overlap")


def test_null_arguments(lib):
    for name in ("BlockNormForward", "BlockNormBackward", "GatedScanForward", "GatedScanBackward", "GatedScanStep"):
        refused(lib, "B200" + name, None, STATUS.INVALID_VALUE, "null arguments")
    size = ct.c_size_t()
    assert lib.fn["B200BlockNormGetWorkspaceSize"](None, ct.byref(size)) == STATUS.INVALID_VALUE
    assert lib.fn["B200GatedScanGetWorkspaceSize"](scan_fields(), None) == STATUS.INVALID_VALUE


def test_nothing_to_do(lib):
    assert lib.fn["B200BlockNormForward"](norm_fields(rows=0), None) == STATUS.SUCCESS
    assert lib.fn["B200GatedScanForward"](scan_fields(batch=0), None) == STATUS.SUCCESS
    assert lib.fn["B200GatedScanStep"](step_fields(batch=0), None) == STATUS.SUCCESS


def test_workspace_sizes(lib):
    size = ct.c_size_t(1)

    def norm(**change):
        assert lib.fn["B200BlockNormGetWorkspaceSize"](norm_fields(**change), ct.byref(size)) == STATUS.SUCCESS
        return size.value

    def scan(**change):
        assert lib.fn["B200GatedScanGetWorkspaceSize"](scan_fields(**change), ct.byref(size)) == STATUS.SUCCESS
        return size.value

    assert norm(rows=0) == 0 and scan(length=0) == 0
    assert norm() >= 3 * 64 * 4 and norm(rows=100000) > norm()
    # every gate group has its own sums
    assert norm(rows=1000, gate=P, gate_rows=500, gate_row=64) >= 500 * 3 * 64 * 4
    assert scan() >= 2 * 64 * 4
    assert norm(rows=1) % 16 == 0 and scan(dim=3) % 16 == 0
