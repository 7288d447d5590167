"""How much of 64 bits the delta rule's fp32 results keep: relative errors in the mean square over a whole tensor, where a
lost piece of an operand or a sum that is cut off shows, as it does not beside the largest value's bound."""
import pytest
import torch

import delta_reference as ref
from test_delta_ops_gpu import delta_case, normal, run_delta

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
# 16-bit calls take fp32 operands as two bf16 pieces.  The second is at most 2^-8 of the value's power of two, so its half step
# at most 2^-17 of that; an error that is even within it has the root mean square 2^-17 / sqrt(3) of the operand, and a sum of
# products the same of the sum.  On the way to a final state, or back to an initial one, lie eight such operands (M beta, the
# blocks' inverses, L's rows before, L beta or beta L, Y or E, U or Z, the state, P), whose errors are independent.
TWO_PIECES = 8 ** 0.5 * 2.0 ** -17 / 3 ** 0.5
# fp32 calls take three pieces.  A product leaves out two products of pieces (2^-8 2^-16 each, 2^-24 in all or less), the tensor
# pipe cuts the sum of 16 terms three times at the size of the result (2^-23 at most, half of it in the mean: 3 2^-24) and the
# sum is added with one rounding (2^-24).  Four products follow one another, and the substitution, which is no worse than
# one: 5 x 5 x 2^-24.  Gradients go through as many again.
THREE_PIECES = 25 * 2.0 ** -24
# 64-token chunks: several, the last one cut; slow decays, which carry a state through all of them; long ones in segments.
SHAPES = [(2, 257, 3, 3, 64, 64, None), (1, 300, 1, 2, 128, 128, None), (1, 200, 2, 2, 40, 100, [0, 1, 90, 200]), (1, 1400, 1, 1, 128, 64, None)]


def error(got, want):
    got, want = got.detach().double().cpu(), want.double()
    return float(((got - want).square().sum() / want.square().sum()).sqrt())


def errors(batch, length, k_heads, heads, k_dim, v_dim, cuts, dtype, slow):
    t = delta_case(batch, length, k_heads, heads, k_dim, v_dim, dtype, cuts=cuts, state=True, seed=length)
    if slow:
        t["g"] = t["g"] * 0.05
    dev = {n: v.cuda().requires_grad_() for n, v in t.items()}
    exact = {n: v.double().requires_grad_() for n, v in t.items()}
    o, final = run_delta(dev, cuts)
    eo, efinal = ref.gated_delta(exact["q"], exact["k"], exact["v"], exact["g"], exact["beta"], initial_state=exact["state"], cuts=cuts)
    d_o, d_final = normal(91, *o.shape, dtype=o.dtype), normal(92, *final.shape, scale=0.3)
    got = torch.autograd.grad([o, final], list(dev.values()), [d_o.cuda(), d_final.cuda()])
    want = torch.autograd.grad([eo, efinal], list(exact.values()), [d_o.double(), d_final.double()])
    names = ["o", "final", *("d_" + n for n in t)]
    return {n: error(a, b.detach()) for n, a, b in zip(names, (o, final, *got), (eo, efinal, *want))}


@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_states_of_16_bit_calls(cuda, shape, dtype, slow):
    e = errors(*shape, dtype, slow)
    assert e["final"] <= TWO_PIECES and e["d_state"] <= TWO_PIECES, e


@pytest.mark.parametrize("slow", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_fp32_calls(cuda, shape, slow):
    e = errors(*shape, FP32, slow)
    for n, x in e.items():
        assert x <= (2 if n.startswith("d_") else 1) * THREE_PIECES, e
