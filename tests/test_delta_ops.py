"""What the gated delta rule and the norm of queries and keys refuse, on any host: the torch frontend's argument checks, and
the C entry points' (checked before anything is launched); and the reference that the GPU tests compare with, against
sums written out."""
import math
import struct

import pytest
import torch

import cubutterfly_b200 as cb
import delta_reference as ref
from cubutterfly_b200 import block_ops, torch_ops

STATUS = cb.Status

# the structs of include/cubutterfly/cubutterfly_b200.h, in field order
HEAD = "P3N"
DELTA = struct.Struct("@8N4id" + 5 * HEAD + "4P" + HEAD + "7PPN")
STEP = struct.Struct("@7N4id" + 5 * HEAD + "4P")
QK = struct.Struct("@10N4id" + 2 * HEAD + "7P" + 2 * HEAD + "4PPN")
P = 4096  # device pointers are never dereferenced by the checks


def delta_fields(**change):
    f = dict(size=DELTA.size, batch=2, length=100, k_heads=2, heads=4, k_dim=16, v_dim=32, sequences=0, data=1, g_type=2,
             b_type=2, reserved=0, scale=1.0)
    for n in ("q", "k", "v", "g", "beta"):
        f.update({n: P, n + "b": 3200, n + "t": 32, n + "h": 16})
    f.update(initial=0, offsets=0, o=2 * P, final=3 * P, d_o=0, d_ob=0, d_ot=0, d_oh=0, d_final=0, d_q=0, d_k=0, d_v=0, d_g=0,
             d_beta=0, d_initial=0, workspace=1 << 20, bytes=1 << 40)
    assert not set(change) - set(f)
    return DELTA.pack(*{**f, **change}.values())


def step_fields(**change):
    f = dict(size=STEP.size, batch=2, k_heads=2, heads=4, k_dim=16, v_dim=32, pool=2, data=1, g_type=2, b_type=1, reserved=0,
             scale=1.0)
    for n in ("q", "k", "v", "g", "beta"):
        f.update({n: P, n + "b": 3200, n + "t": 0, n + "h": 16})
    f.update(state=P, new_state=P, slots=0, o=2 * P)
    assert not set(change) - set(f)
    return STEP.pack(*{**f, **change}.values())


def qk_fields(**change):
    f = dict(size=QK.size, batch=1, tokens=10, q_heads=4, k_heads=2, dim=64, rotary=32, axis_count=1, axis=10, period=10, data=1,
             qw_type=2, kw_type=2, flags=0, eps=1e-6, q=P, qb=0, qt=256, qh=64, k=P, kb=0, kt=128, kh=64, q_weight=P, k_weight=P,
             positions=P, frequencies=P, axes=0, q_out=2 * P, k_out=3 * P, d_q_out=0, dqb=0, dqt=0, dqh=0, d_k_out=0, dkb=0,
             dkt=0, dkh=0, d_q=0, d_k=0, d_qw=0, d_kw=0, workspace=0, bytes=0)
    assert not set(change) - set(f)
    return QK.pack(*{**f, **change}.values())


def refused(lib, name, packed, status, text):
    assert lib.fn[name](packed, None) == status
    assert text in lib.fn["GetLastErrorString"]().decode()


INVALID, UNSUPPORTED = STATUS.INVALID_VALUE, STATUS.NOT_SUPPORTED


@pytest.mark.parametrize("change,status,text", [
    (dict(size=8), INVALID, "struct_size"),
    (dict(k_heads=0), INVALID, "at least 1"),
    (dict(v_dim=0), INVALID, "at least 1"),
    (dict(k_heads=3), INVALID, "multiple"),
    (dict(k_heads=8), UNSUPPORTED, "key heads"),
    (dict(k_dim=129), UNSUPPORTED, "128"),
    (dict(v_dim=129), UNSUPPORTED, "128"),
    (dict(length=(1 << 30) + 1), UNSUPPORTED, "2^30"),
    (dict(batch=1 << 20, length=1 << 20), UNSUPPORTED, "chunks"),
    (dict(batch=1 << 24, length=1, heads=16), UNSUPPORTED, "sequences"),
    (dict(data=7), UNSUPPORTED, "data_type"),
    (dict(g_type=0), UNSUPPORTED, "log_decay_type"),
    (dict(b_type=0), UNSUPPORTED, "beta_type"),
    (dict(scale=math.nan), INVALID, "scale"),
    (dict(q=0), INVALID, "q"),
    (dict(k=P + 1), INVALID, "misaligned k"),
    (dict(v=0), INVALID, "misaligned v"),
    (dict(g=P + 2), INVALID, "misaligned"),
    (dict(beta=0), INVALID, "beta"),
    (dict(o=0), INVALID, "null or misaligned o"),
    (dict(o=P), INVALID, "alias"),
    (dict(final=0), INVALID, "final_state"),
    (dict(initial=3 * P), INVALID, "alias"),
    (dict(initial=P + 2), INVALID, "misaligned state"),
    (dict(offsets=P, sequences=3), INVALID, "packed"),
    (dict(offsets=P, batch=1), INVALID, "packed"),
    (dict(sequences=3), INVALID, "without offsets"),
    (dict(length=0), UNSUPPORTED, "zero tokens"),
    (dict(workspace=0), INVALID, "workspace"),
    (dict(workspace=P + 16), INVALID, "workspace"),
    (dict(bytes=100), INVALID, "workspace"),
])
def test_gated_delta_refusals(lib, change, status, text):
    refused(lib, "B200GatedDeltaForward", delta_fields(**change), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(d_o=0), INVALID, "d_o"),
    (dict(d_q=0), INVALID, "null gradient"),
    (dict(d_k=P + 1), INVALID, "misaligned gradient"),
    (dict(d_g=P + 2), INVALID, "gradient of a gate"),
    (dict(d_beta=0), INVALID, "null gradient"),
    (dict(batch=0), UNSUPPORTED, "zero tokens"),
    (dict(bytes=0), INVALID, "workspace"),
])
def test_gated_delta_backward_refusals(lib, change, status, text):
    valid = dict(d_o=P, d_ob=3200, d_ot=32, d_oh=8, d_q=P, d_k=P, d_v=P, d_g=P, d_beta=P)
    refused(lib, "B200GatedDeltaBackward", delta_fields(**{**valid, **change}), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(size=1), INVALID, "struct_size"),
    (dict(heads=0), INVALID, "at least 1"),
    (dict(k_dim=200), UNSUPPORTED, "128"),
    (dict(data=4), UNSUPPORTED, "data_type"),
    (dict(q=0), INVALID, "q"),
    (dict(o=0), INVALID, "null or misaligned o"),
    (dict(state=0), INVALID, "null state"),
    (dict(pool=1), INVALID, "pool"),
    (dict(state=P + 2), INVALID, "misaligned"),
    (dict(new_state=P + 256), INVALID, "overlap"),
    (dict(scale=math.inf), INVALID, "scale"),
])
def test_gated_delta_step_refusals(lib, change, status, text):
    refused(lib, "B200GatedDeltaStep", step_fields(**change), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(size=0), INVALID, "struct_size"),
    (dict(q_heads=0), INVALID, "at least 1"),
    (dict(dim=257), UNSUPPORTED, "256"),
    (dict(rotary=33), INVALID, "even"),
    (dict(rotary=66), INVALID, "even"),
    (dict(rotary=0), INVALID, "go together"),
    (dict(positions=0), INVALID, "go together"),
    (dict(period=0), INVALID, "period"),
    (dict(axis_count=3), INVALID, "axes"),
    (dict(data=8), UNSUPPORTED, "data_type"),
    (dict(qw_type=0), UNSUPPORTED, "q_weight_type"),
    (dict(flags=8), INVALID, "flags"),
    (dict(eps=-1.0), INVALID, "epsilon"),
    (dict(q=0), INVALID, "q"),
    (dict(k=P + 1), INVALID, "misaligned k"),
    (dict(positions=P + 4, flags=4), INVALID, "misaligned positions"),
    (dict(q_out=0), INVALID, "output"),
    (dict(k_out=P), INVALID, "alias"),
    (dict(k_out=2 * P), INVALID, "alias"),
])
def test_qk_norm_refusals(lib, change, status, text):
    refused(lib, "B200QkNormForward", qk_fields(**change), status, text)


@pytest.mark.parametrize("change,status,text", [
    (dict(d_q_out=0), INVALID, "d_q_out"),
    (dict(d_k=0), INVALID, "gradient"),
    (dict(d_kw=0), INVALID, "its gradient"),
    (dict(d_qw=P + 2), INVALID, "misaligned"),
    (dict(workspace=0), INVALID, "workspace"),
    (dict(bytes=16), INVALID, "workspace"),
    (dict(tokens=0), UNSUPPORTED, "zero tokens"),
])
def test_qk_norm_backward_refusals(lib, change, status, text):
    valid = dict(d_q_out=P, dqt=256, dqh=64, d_k_out=P, dkt=128, dkh=64, d_q=P, d_k=P, d_qw=P, d_kw=P, workspace=P, bytes=1 << 20)
    refused(lib, "B200QkNormBackward", qk_fields(**{**valid, **change}), status, text)


def test_workspace_sizes(lib):
    """Enough for every chunk that the sequences can have, and nothing without tokens."""
    import ctypes as ct

    size = ct.c_size_t()

    def query(backward=0, **change):
        assert lib.fn["B200GatedDeltaGetWorkspaceSize"](delta_fields(**change), backward, ct.byref(size)) == STATUS.SUCCESS
        return size.value

    one = query(batch=1, length=64)
    assert one > 0 and query(batch=1, length=65) >= 2 * one - 4096 and query(batch=0) == 0 and query(length=0) == 0
    assert query(1, batch=1, length=64) > one
    packed = [query(batch=1, length=128, offsets=P, sequences=n) for n in (1, 2, 40)]
    assert packed == sorted(packed) and packed[0] >= query(batch=1, length=128)
    assert lib.fn["B200QkNormGetWorkspaceSize"](qk_fields(), ct.byref(size)) == STATUS.SUCCESS and size.value >= 2 * 64 * 4
    assert lib.fn["B200QkNormGetWorkspaceSize"](qk_fields(q_weight=0, k_weight=0), ct.byref(size)) == STATUS.SUCCESS
    assert size.value == 0


def test_cpu_tensors_are_rejected():
    x = torch.randn(1, 4, 2, 8)
    with pytest.raises(ValueError, match="q must be a CUDA"):
        torch_ops.gated_delta(x, x, x, x[..., 0], x[..., 0])
    with pytest.raises(ValueError, match="q must be a CUDA"):
        torch_ops.gated_delta_step(x, x[0], x[0], x[0], x[0, ..., 0], x[0, ..., 0])
    with pytest.raises(ValueError, match="q must be a CUDA"):
        torch_ops.qk_norm(x, x)


def test_traces_tangents_and_wrappers_are_refused():
    import torch.autograd.forward_ad as fwd
    from torch._subclasses.fake_tensor import FakeTensorMode

    x = torch.zeros(1, 4, 2, 8)
    calls = (lambda v: torch_ops.gated_delta(v, v, v, v[..., 0], v[..., 0])[0], lambda v: torch_ops.qk_norm(v, v)[0],
             lambda v: torch_ops.gated_delta_step(v, v[0], v[0], v[0], v[0, ..., 0], v[0, ..., 0]))
    with FakeTensorMode():
        fake = torch.empty(1, 4, 2, 8, device="cuda")
    for call in calls:
        with pytest.raises(ValueError, match="is being traced"):
            torch.jit.trace(call, (x,))
        with pytest.raises(ValueError, match="storage of its own"):
            call(fake)
        with fwd.dual_level(), pytest.raises(ValueError, match="forward-mode tangent"):
            call(fwd.make_dual(x, torch.ones_like(x)))


def test_torch_ops_exports_the_operators():
    for name in ("gated_delta", "gated_delta_step", "qk_norm"):
        assert name in torch_ops.__all__ and getattr(torch_ops, name) is getattr(block_ops, name)


def test_places_of_chunks():
    """The places floor(start / 64) + j + c of sequences' chunks never coincide and never pass floor(T / 64) + n."""
    import random

    rng = random.Random(3)
    for _ in range(300):
        total, n = rng.randint(0, 700), rng.randint(1, 12)
        cuts = [0, *sorted(rng.randint(0, total) for _ in range(n - 1)), total]
        places = [a // 64 + j + c for j, (a, b) in enumerate(zip(cuts, cuts[1:])) for c in range(-(-(b - a) // 64))]
        assert len(set(places)) == len(places) and all(0 <= p < total // 64 + n for p in places)


def test_the_reference_against_sums_written_out():
    """Two tokens of one head by hand, and a rotation by a right angle."""
    q, k, v = (torch.tensor(x, dtype=torch.float64).view(1, 2, 1, 2) for x in ([[1., 2.], [3., -1.]], [[1., 0.], [.6, .8]], [[2., 4.], [1., 1.]]))
    g, beta = torch.log(torch.tensor([[[1.0], [0.5]]], dtype=torch.float64)), torch.tensor([[[0.5], [1.0]]], dtype=torch.float64)
    o, final = ref.gated_delta(q, k, v, g, beta, scale=1.0)
    s1 = torch.tensor([[1., 2.], [0., 0.]], dtype=torch.float64)     # k1 (beta v1)^T
    u2 = torch.tensor([1., 1.], dtype=torch.float64) - 0.5 * 0.6 * torch.tensor([1., 2.], dtype=torch.float64)
    s2 = 0.5 * s1 + torch.tensor([[.6], [.8]], dtype=torch.float64) * u2
    assert torch.allclose(final[0, 0], s2) and torch.allclose(o[0, 0, 0], torch.tensor([1., 2.], dtype=torch.float64))
    assert torch.allclose(o[0, 1, 0], 3 * s2[0] - s2[1])
    x = torch.tensor([[[3.0, 4.0]]], dtype=torch.float64)
    turned = ref.qk_norm(x, norm="l2", eps=0.0, positions=torch.tensor([1]), frequencies=torch.tensor([math.pi / 2], dtype=torch.float64))
    assert torch.allclose(turned, torch.tensor([[[-0.8, 0.6]]], dtype=torch.float64))
