"""A small recurrent language model on the block operators: trained, prefilled and decoded.

Every block is  norm -> projection -> gated_scan -> projection , and between two blocks one ``block_norm`` call norms
the block's output, gates it, adds it to the residual stream and makes the next block's normed input.  With
``rotate=True`` that input is Hadamard-rotated in the same pass, as the input of a quantised projection is; the
projections' weights are rotated once to match, so the model's function stays the same.

    python examples/recurrent_lm.py [--steps N] [--dim D] [--layers L]

needs a CUDA device and the built library.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cubutterfly_b200 import torch_ops  # noqa: E402


class RecurrentBlock(torch.nn.Module):
    """u -> y: one projection to x and the two gates, the recurrence, one projection back."""

    def __init__(self, dim, dtype):
        super().__init__()
        self.dim = dim
        self.inward = torch.nn.Linear(dim, 3 * dim, bias=False, dtype=dtype)
        self.outward = torch.nn.Linear(dim, dim, bias=False, dtype=dtype)
        # decays between 0.9 and 0.999 a token where the recurrence gate is open
        a = torch.rand(dim) * 0.099 + 0.9
        self.decay = torch.nn.Parameter(torch.log(torch.expm1(-torch.log(a) / 8.0)))
        self.post_weight = torch.nn.Parameter(torch.ones(dim))
        self.gate = torch.nn.Parameter(torch.full((dim,), 0.5, dtype=dtype))

    def forward(self, u, state=None, offsets=None):
        x, r, i = self.inward(u).split(self.dim, dim=-1)
        h, state = torch_ops.gated_scan(x, r, i, self.decay, initial_state=state, offsets=offsets)
        return self.outward(h), state

    def step(self, u, pool, slots):
        x, r, i = self.inward(u).split(self.dim, dim=-1)
        return self.outward(torch_ops.gated_scan_step(pool, x, r, i, self.decay, slots=slots))


class RecurrentLM(torch.nn.Module):
    def __init__(self, vocabulary, dim, layers, dtype=torch.bfloat16):
        super().__init__()
        self.dtype, self.rotate = dtype, False
        self.embedding = torch.nn.Embedding(vocabulary, dim)
        self.blocks = torch.nn.ModuleList(RecurrentBlock(dim, dtype) for _ in range(layers))
        # the norm before block k, and the last one before the head
        self.norms = torch.nn.ParameterList(torch.nn.Parameter(torch.ones(dim)) for _ in range(layers + 1))
        self.head = torch.nn.Linear(dim, vocabulary, bias=False, dtype=dtype)

    def _run(self, tokens, mixer):
        residual = self.embedding(tokens)  # the residual stream is fp32
        residual, u = torch_ops.block_norm(residual, pre_weight=self.norms[0], rotate=self.rotate, dtype=self.dtype)
        for k, block in enumerate(self.blocks):
            residual, u = torch_ops.block_norm(residual, mixer(k, block, u), post_weight=block.post_weight,
                                               gate=block.gate, pre_weight=self.norms[k + 1], rotate=self.rotate)
        return self.head(u)

    def forward(self, tokens, offsets=None):
        """(logits, final states of every layer) of (B, S) tokens, or of (T,) packed ones with offsets."""
        states = []

        def mixer(k, block, u):
            y, state = block(u, offsets=offsets)
            states.append(state)
            return y

        return self._run(tokens, mixer), states

    @torch.no_grad()
    def step(self, tokens, pools, slots=None):
        """Logits of one token per request; the states in `pools` (one per layer) move on."""
        return self._run(tokens, lambda k, block, u: block.step(u, pools[k], slots))

    @torch.no_grad()
    def rotate_inputs(self):
        """From here on every projection's input is rotated, and its weights with it: (u H)(W H)^T = u W^T."""
        for linear in [*(b.inward for b in self.blocks), self.head]:
            linear.weight.copy_(torch_ops.hadamard_rotate(linear.weight.float()).to(linear.weight.dtype))
        self.rotate = True


def main(argv=None):
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--steps", type=int, default=60)
    p.add_argument("--dim", type=int, default=256)
    p.add_argument("--layers", type=int, default=2)
    args = p.parse_args(argv)
    device, vocabulary = torch.device("cuda"), 64
    torch.manual_seed(0)
    model = RecurrentLM(vocabulary, args.dim, args.layers).to(device)
    optimizer = torch.optim.AdamW(model.parameters(), lr=3e-3)

    # counting with a stride that each sequence keeps: the next token needs the two before it
    def batch(rows, length):
        start = torch.randint(vocabulary, (rows, 1), device=device)
        stride = torch.randint(1, 4, (rows, 1), device=device)
        return (start + stride * torch.arange(length + 1, device=device)) % vocabulary

    losses = []
    for _ in range(args.steps):
        tokens = batch(32, 96)
        logits, _ = model(tokens[:, :-1])
        loss = torch.nn.functional.cross_entropy(logits[:, 2:].flatten(0, 1).float(), tokens[:, 3:].flatten())
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(loss.item())
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f} (log {vocabulary} = {math.log(vocabulary):.3f})")

    # prefill a packed batch of prompts, then decode them together, their states in a pool of slots
    with torch.no_grad():
        lengths = [40, 7, 23]
        tokens = batch(len(lengths), 60)
        packed = torch.cat([tokens[k, :n] for k, n in enumerate(lengths)])
        offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device=device)
        logits, states = model(packed, offsets)
        slots = torch.tensor([4, 1, 2], dtype=torch.int32, device=device)
        pools = [torch.zeros(6, args.dim, device=device) for _ in states]
        for pool, state in zip(pools, states):
            pool[slots.long()] = state
        worst = 0.0
        for t in range(8):
            given = torch.stack([tokens[k, n + t] for k, n in enumerate(lengths)])
            step = model.step(given, pools, slots)
            for k, n in enumerate(lengths):
                whole, _ = model(tokens[k:k + 1, :n + t + 1])
                worst = max(worst, float((whole[0, -1].float() - step[k].float()).abs().max()))
        scale = float(logits.float().abs().max())
        print(f"decoding against the whole sequence: largest difference {worst:.4f} of logits up to {scale:.1f}")

        tokens = batch(4, 64)[:, :-1]
        plain, _ = model(tokens)
        model.rotate_inputs()
        rotated, _ = model(tokens)
        change = float((plain - rotated).float().norm() / plain.float().norm())
        print(f"rotated projections: relative change of the logits {change:.4f}")
    return {"losses": losses, "decode": worst / scale, "rotation": change}


if __name__ == "__main__":
    main()
