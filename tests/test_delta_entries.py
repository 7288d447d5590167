"""C entry points of the delta rule and the norm of queries and keys, on any host: tensors that share memory are refused."""
import pytest

from test_delta_ops import INVALID, delta_fields, qk_fields, refused, step_fields

G = 1 << 22  # apart from everything that a call below has


def places(*names, start=1):
    return {n: G * (start + i) for i, n in enumerate(names)}


# 2 x 100 tokens, 2 key heads of 16 and 4 heads of 32 in bf16: rows of (heads, channels) beside one another
DELTA = dict(qb=3200, qt=32, qh=16, kb=3200, kt=32, kh=16, vb=12800, vt=128, vh=32, gb=400, gt=4, gh=1, betab=400, betat=4, betah=1,
             **places("q", "k", "v", "g", "beta", "initial", "o", "final"))
BACKWARD = dict(DELTA, d_ob=12800, d_ot=128, d_oh=32,
                **places("d_o", "d_final", "d_q", "d_k", "d_v", "d_g", "d_beta", "d_initial", start=9))
READ = ("q", "k", "v", "g", "beta", "initial")
SIZES = dict(q=6400, k=6400, v=51200, g=3200, beta=1600, initial=2 * 4 * 16 * 32 * 4, d_o=51200)  # bytes


@pytest.mark.parametrize("other", READ)
@pytest.mark.parametrize("out", ["o", "final"])
def test_forward_outputs_apart(lib, out, other):
    """The same address, the other's last value, and an output that ends in it."""
    size = {"o": 51200, "final": SIZES["initial"]}[out]
    for place in (DELTA[other], DELTA[other] + SIZES[other] - 16, DELTA[other] - size + 16):
        refused(lib, "B200GatedDeltaForward", delta_fields(**{**DELTA, out: place}), INVALID, "alias")


@pytest.mark.parametrize("out,size", [("d_q", 6400), ("d_k", 6400), ("d_v", 51200), ("d_g", 3200), ("d_beta", 1600),
                                      ("d_initial", SIZES["initial"])])
def test_gradients_apart(lib, out, size):
    for other in (*READ, "d_o", "d_final"):
        for place in (BACKWARD[other], BACKWARD[other] - size + 16):
            refused(lib, "B200GatedDeltaBackward", delta_fields(**{**BACKWARD, out: place}), INVALID, "a tensor that is read")
    for other in ("d_q", "d_k", "d_v", "d_g", "d_beta", "d_initial"):
        if other != out:
            refused(lib, "B200GatedDeltaBackward", delta_fields(**{**BACKWARD, out: BACKWARD[other]}), INVALID, "one another")
    packed = {**BACKWARD, "batch": 1, "sequences": 3, "offsets": BACKWARD[out]}
    refused(lib, "B200GatedDeltaBackward", delta_fields(**packed), INVALID, "a tensor that is read")


def test_step_output_apart(lib):
    step = dict(qb=32, qh=16, kb=32, kh=16, vb=128, vh=32, gb=4, gh=1, betab=4, betah=1, pool=5,
                **places("q", "k", "v", "g", "beta", "state", "o"))
    step["new_state"] = step["state"]
    for other in ("q", "k", "g", "beta", "state"):
        refused(lib, "B200GatedDeltaStep", step_fields(**{**step, "o": step[other]}), INVALID, "alias")
    refused(lib, "B200GatedDeltaStep", step_fields(**{**step, "new_state": 9 * G, "o": 9 * G + 5 * 4 * 16 * 32 * 4 - 16}), INVALID, "alias")
    refused(lib, "B200GatedDeltaStep", step_fields(**{**step, "o": step["v"] + 16}), INVALID, "alias")
    refused(lib, "B200GatedDeltaStep", step_fields(**{**step, "o": step["v"], "vb": 256}), INVALID, "alias")


def test_norm_outputs_apart(lib):
    qk = dict(positions=0, frequencies=0, rotary=0, axis_count=0, **places("q", "k", "q_weight", "k_weight", "q_out", "k_out"))
    for change in (dict(q_out=qk["q"]), dict(q_out=qk["k"] - 16), dict(k_out=qk["q"] + 16), dict(k_out=qk["k"]),
                   dict(k_out=qk["q_out"] + 10 * 256 * 2 - 16)):
        refused(lib, "B200QkNormForward", qk_fields(**{**qk, **change}), INVALID, "alias")
    back = dict(qk, dqt=256, dqh=64, dkt=128, dkh=64, workspace=G, bytes=1 << 20,
                **places("d_q_out", "d_k_out", "d_q", "d_k", "d_qw", "d_kw", start=9))
    for change in (dict(d_q=qk["q"] + 16), dict(d_q=qk["k"]), dict(d_q=back["d_k_out"]), dict(d_k=qk["q"]), dict(d_k=back["d_q_out"]),
                   dict(d_k=back["d_k_out"] - 16), dict(d_k=back["d_q"] + 16), dict(d_q=qk["q"], qt=512)):
        refused(lib, "B200QkNormBackward", qk_fields(**{**back, **change}), INVALID, "alias")


@pytest.mark.gpu
def test_outputs_in_place(cuda, lib):
    """o of a step where v was, and a head's gradient where its output's gradient or the head itself was."""
    import ctypes as ct

    import torch

    from cubutterfly_b200 import Status, torch_ops

    def normal(seed, *shape):
        return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().to(torch.bfloat16)

    stream = ct.c_void_p(torch.cuda.current_stream().cuda_stream)
    q, k, v, g, beta = normal(1, 2, 2, 16), normal(2, 2, 2, 16), normal(3, 2, 4, 32), -normal(4, 2, 4).abs(), normal(5, 2, 4).abs()
    pool = torch.randn(2, 4, 16, 32, device="cuda")
    state = pool.clone()
    want = torch_ops.gated_delta_step(state, q, k, v, g, beta, scale=1.0)
    step = dict(g_type=1, q=q.data_ptr(), qb=32, qh=16, k=k.data_ptr(), kb=32, kh=16, v=v.data_ptr(), vb=128, vh=32, g=g.data_ptr(),
                gb=4, gh=1, beta=beta.data_ptr(), betab=4, betah=1, state=pool.data_ptr(), new_state=pool.data_ptr(), o=v.data_ptr())
    assert lib.fn["B200GatedDeltaStep"](step_fields(**step), stream) == Status.SUCCESS
    assert torch.equal(v, want) and torch.equal(pool, state)
    q, k, dq, dk = (normal(i, 10, 4 - 2 * (i % 2), 64) for i in (6, 7, 8, 9))
    leaves = [q.clone().requires_grad_(), k.clone().requires_grad_()]
    want = torch.autograd.grad(torch_ops.qk_norm(*leaves), leaves, [dq, dk])
    fields = dict(q_weight=0, k_weight=0, positions=0, frequencies=0, rotary=0, axis_count=0, q=q.data_ptr(), k=k.data_ptr(), q_out=0,
                  k_out=0, d_q_out=dq.data_ptr(), dqt=256, dqh=64, d_k_out=dk.data_ptr(), dkt=128, dkh=64)
    assert lib.fn["B200QkNormBackward"](qk_fields(**fields, d_q=dq.data_ptr(), d_k=k.data_ptr()), stream) == Status.SUCCESS
    assert torch.equal(dq, want[0]) and torch.equal(k, want[1])
