"""Waits of the delta rule's kernels that run out: the call ends, nothing of what depends on them passes for a result, and the
next call is as ever.  The limit is the C struct's `wait_limit`: none at all, or so few tries that some waits last and
others do not."""
import ctypes as ct

import pytest
import torch

from cubutterfly_b200 import Status
from test_delta_ops import delta_fields

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# (batch, length, key heads, heads, K, V, cuts): one chunk, several, segments (two and more), packed with tokens of no sequence
CASES = [(2, 50, 1, 2, 64, 64, None), (2, 300, 2, 2, 128, 96, None), (1, 1100, 1, 1, 40, 128, None), (1, 4000, 1, 2, 128, 128, None),
         (1, 2500, 1, 2, 96, 80, [3, 3, 90, 2400, 2490])]


def inputs(batch, length, k_heads, heads, k_dim, v_dim, cuts, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    states = len(cuts) - 1 if cuts else batch
    k = normal(batch, length, k_heads, k_dim)
    return {"q": normal(batch, length, k_heads, k_dim).to(dtype), "k": (k / k.norm(dim=-1, keepdim=True)).to(dtype),
            "v": normal(batch, length, heads, v_dim).to(dtype), "g": normal(batch, length, heads).abs().mul(-0.02).to(dtype),
            "beta": torch.sigmoid(normal(batch, length, heads)).to(dtype), "initial": normal(states, heads, k_dim, v_dim),
            "d_o": normal(batch, length, heads, v_dim).to(dtype), "d_final": normal(states, heads, k_dim, v_dim)}


def call(lib, t, cuts, wait_limit):
    """Outputs and gradients by the C entry points, out of buffers that hold 7 before."""
    batch, length, k_heads, k_dim = t["q"].shape
    heads, v_dim = t["v"].shape[2:]
    kind = {FP16: 0, BF16: 1, FP32: 2}[t["q"].dtype]
    offsets = torch.tensor(cuts, dtype=torch.int32, device="cuda") if cuts else None
    out = {"o": torch.full_like(t["v"], 7), "final": torch.full_like(t["initial"], 7)}
    out.update({"d_" + n: torch.full_like(t[n], 7) for n in ("q", "k", "v", "g", "beta", "initial")})
    fields = dict(batch=batch, length=length, k_heads=k_heads, heads=heads, k_dim=k_dim, v_dim=v_dim, data=kind, g_type=kind,
                  b_type=kind, sequences=len(cuts) - 1 if cuts else 0, offsets=offsets.data_ptr() if cuts else 0,
                  scale=k_dim ** -0.5, reserved=wait_limit, initial=t["initial"].data_ptr(), o=out["o"].data_ptr(),
                  final=out["final"].data_ptr(), d_final=t["d_final"].data_ptr())
    for n, x in (("q", t["q"]), ("k", t["k"]), ("v", t["v"]), ("g", t["g"]), ("beta", t["beta"]), ("d_o", t["d_o"])):
        b, token, head = x.stride()[:3]
        names = (n, n + "b", n + "t", n + "h")
        fields.update(zip(names, (x.data_ptr(), b, token, head)))
    fields.update({"d_" + n: out["d_" + n].data_ptr() for n in ("q", "k", "v", "g", "beta", "initial")})
    stream = torch.cuda.current_stream().cuda_stream
    for backward, name in enumerate(("B200GatedDeltaForward", "B200GatedDeltaBackward")):
        size = ct.c_size_t()
        assert lib.fn["B200GatedDeltaGetWorkspaceSize"](delta_fields(**fields), backward, ct.byref(size)) == Status.SUCCESS
        workspace = torch.empty(size.value, dtype=torch.uint8, device="cuda").fill_(17)
        packed = delta_fields(**fields, workspace=workspace.data_ptr(), bytes=size.value)
        assert lib.fn[name](packed, ct.c_void_p(stream)) == Status.SUCCESS
    torch.cuda.synchronize()
    return out


def of_sequences(x, name, cuts):
    return x[:, cuts[0]:cuts[-1]] if cuts and name not in ("final", "d_initial") else x


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_waits_that_run_out_at_once(cuda, lib, case, dtype):
    cuts = case[-1]
    t = inputs(*case, dtype)
    want = call(lib, t, cuts, 0)
    assert all(torch.isfinite(x).all() for x in want.values())
    got = call(lib, t, cuts, -1)
    for n, x in got.items():
        if cuts and n in ("final", "d_initial"):     # of a sequence without tokens the state passes through
            assert torch.equal(x[0], want[n][0])
            x = x[1:]
        assert torch.isnan(of_sequences(x, n, cuts)).all(), n
        if cuts and n not in ("final", "d_initial"):
            assert not x[:, :cuts[0]].any() and not x[:, cuts[-1]:].any(), n
    again = call(lib, t, cuts, 0)
    assert all(torch.equal(again[n], want[n]) for n in want)


@pytest.mark.parametrize("tries", [1, 2])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("case", CASES, ids=str)
def test_some_waits_run_out(cuda, lib, case, dtype, tries):
    """Every value is the right one or NaN, and of a chain all or none."""
    cuts = case[-1]
    t = inputs(*case, dtype, seed=1)
    want = call(lib, t, cuts, 0)
    for _ in range(3):
        for n, x in call(lib, t, cuts, tries).items():
            lost = torch.isnan(x)
            assert torch.equal(torch.where(lost, want[n], x), want[n]), n
            if n in ("final", "d_initial"):
                assert torch.equal(lost.all(-1).all(-1), lost.any(-1).any(-1)), n
            elif n in ("o", "d_v", "d_q", "d_k"):
                assert torch.equal(lost.all(-1), lost.any(-1)), n


def test_fp32_tensors_have_no_such_waits(cuda, lib):
    t = inputs(*CASES[1], FP32)
    want, got = call(lib, t, None, 0), call(lib, t, None, -1)
    assert all(torch.equal(got[n], want[n]) for n in want)
