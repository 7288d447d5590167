"""The recurrent language model of examples/recurrent_lm.py with the gated delta rule in its blocks: norm of queries and keys,
delta rule, its single token and the block norm between them run together, and the model's gradients are those of the same
model written out in 64 bits."""
import math
import sys
import types
from pathlib import Path

import pytest
import torch

import delta_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture()
def example():
    examples = str(Path(__file__).resolve().parents[1] / "examples")
    sys.path.insert(0, examples)
    try:
        import recurrent_lm
    finally:
        sys.path.remove(examples)
    return recurrent_lm


def test_example_with_delta_rule_runs(cuda, example):
    out = example.main(["--steps", "3", "--mixer", "delta"])
    assert len(out["losses"]) == 3 and all(math.isfinite(v) for v in out["losses"])
    # bf16 activations (2^-8 a rounding) through two blocks in two different orders of the same sums
    assert out["decode"] < 0.05
    # bf16 weights rounded once more by their rotation (2^-9 rms of each), and the activations likewise
    assert out["rotation"] < 0.05


def plain_ops():
    def rms(t):
        return t / torch.sqrt(t.square().mean(-1, keepdim=True) + 1e-6)

    def block_norm(x, y=None, *, pre_weight, post_weight=None, gate=None, rotate=False, dtype=None):
        assert not rotate
        residual = x.double() if y is None else x + gate * rms(y) * post_weight
        return residual, rms(residual) * pre_weight

    def qk_norm(q, k, *, norm, positions, frequencies):
        assert norm == "l2"
        half = frequencies.numel()
        angle = (positions.double()[:, None] * frequencies)[:, None, :]

        def one(t):
            t = t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6)
            a, b, rest = t[..., :half], t[..., half:2 * half], t[..., 2 * half:]
            return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), rest), -1)

        return one(q), one(k)

    def gated_delta(q, k, v, log_decay, beta, *, initial_state=None, offsets=None):
        cuts = None if offsets is None else offsets.tolist()
        return ref.gated_delta(q, k, v, log_decay, beta, initial_state=initial_state, cuts=cuts)

    return types.SimpleNamespace(block_norm=block_norm, qk_norm=qk_norm, gated_delta=gated_delta)


@pytest.mark.parametrize("packed", [False, True])
def test_example_with_delta_rule_gradients(cuda, example, monkeypatch, packed):
    torch.manual_seed(5)
    vocabulary, dim = 32, 64
    model = example.RecurrentLM(vocabulary, dim, 2, dtype=torch.float32, block=example.DeltaBlock)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.05 * torch.randn_like(p))
    exact = example.RecurrentLM(vocabulary, dim, 2, dtype=torch.float32, block=example.DeltaBlock)
    exact.load_state_dict(model.state_dict())
    exact.double()
    exact.dtype = torch.float64
    for block in exact.blocks:  # the gates stay in 64 bits
        block._project = types.MethodType(_project64, block)
    model.cuda()
    tokens = torch.randint(vocabulary, (150,) if packed else (2, 150))
    offsets = torch.tensor([0, 70, 70, 150], dtype=torch.int32) if packed else None
    weights = torch.randn(*tokens.shape, vocabulary)

    logits, states = model(tokens.cuda(), None if offsets is None else offsets.cuda())
    (logits * weights.cuda()).sum().backward()
    monkeypatch.setattr(example, "torch_ops", plain_ops())
    want, want_states = exact(tokens, offsets)
    (want * weights.double()).sum().backward()
    # fp32 throughout: two blocks of some ten products and norms each way, sums of up to 300 terms whose roundings (2^-24)
    # add up like their root, and the delta rule's own bound; the errors meet at random, the bound takes them all together
    bound = 40 * math.sqrt(300) * 2.0 ** -24 + 2 * ref.DELTA_LOSS[torch.float32]
    pairs = [("logits", logits, want), *(("state", a, b) for a, b in zip(states, want_states)),
             *((n, p.grad, e.grad) for (n, p), e in zip(model.named_parameters(), exact.parameters()))]
    for name, a, b in pairs:
        error = float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())
        assert error < bound, (name, error, bound)


def _project64(self, u, positions):
    from recurrent_lm import torch_ops

    q, k, v, decay, beta = self.inward(u).split(self.widths, dim=-1)
    q, k, v = (t.unflatten(-1, (-1, self.head)) for t in (q, k, v))
    q, k = torch_ops.qk_norm(q, k, norm="l2", positions=positions, frequencies=self.frequencies)
    return q, k, v, -torch.nn.functional.softplus(decay + self.decay), torch.sigmoid(beta)
