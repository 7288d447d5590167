"""Angles of the norm of queries and keys at far positions, against exact rational arithmetic."""
import math
from fractions import Fraction

import pytest
import torch

from cubutterfly_b200 import torch_ops

pytestmark = pytest.mark.gpu

# 1 / 2 pi to 2^-160, from pi = 16 arctan(1/5) - 4 arctan(1/239)
_ARC = [sum(Fraction((-1) ** k, (2 * k + 1) * n ** (2 * k + 1)) for k in range(60)) for n in (5, 239)]
TURNS = 1 / (2 * (16 * _ARC[0] - 4 * _ARC[1]))
# The half turn, between -1 and 1, is rounded to fp32: pi 2^-25 = 0.94e-7; the sine and the cosine are off by two units of
# 2^-24 and each takes two more roundings of 2^-24, of the whole and the half of which the angle sees at most the root.
WORST = math.pi * 2.0 ** -25 + 4 * 2.0 ** -24
# In the mean over positions the roundings cancel: 2^-64 of a turn a position, and 2^-32 of it cut off, are left, 2 pi (2^-33 +
# 2^-33), and of 4000 roundings of 1e-7 the mean's 5 deviations.
MEAN = 2 * math.pi * 2.0 ** -32 + 5 * 1e-7 / 4000 ** 0.5


@pytest.mark.parametrize("width", [torch.int32, torch.int64])
@pytest.mark.parametrize("first", [0, 1 << 24, (1 << 31) - 4000])
def test_angles(cuda, first, width):
    frequencies = torch.cat((10000.0 ** (-torch.arange(96) / 96), torch.tensor([1.0, 0.1, 1 / 3, -1.0, -0.7, 0.5, 1e-9, -1e-30]),
                             torch.rand(24, generator=torch.Generator().manual_seed(1)))).float()
    positions = torch.arange(first, first + 4000, dtype=torch.int64)
    x = torch.zeros(4000, 1, 256)
    x[..., :128] = 1.0                   # pairs (1, 0), which become (cos, sin) times one factor
    y, _ = torch_ops.qk_norm(x.cuda(), x.cuda(), positions=positions.to(width).cuda(), frequencies=frequencies.cuda())
    y = y[:, 0].double().cpu()
    got = torch.atan2(y[:, 128:], y[:, :128])
    step = [Fraction(f) * TURNS for f in frequencies.tolist()]
    base = [s * first % 1 for s in step]
    scale = 1 << 80                      # turns as integers, since fractions of fractions grow
    rows = [[(int(b * scale) + int(s * scale) * i) % scale / scale * 2 * math.pi for i in range(4000)] for s, b in zip(step, base)]
    want = torch.tensor(rows, dtype=torch.float64).T
    off = torch.remainder(got - want + math.pi, 2 * math.pi) - math.pi
    assert off.abs().max() <= WORST, float(off.abs().max())
    assert off.mean(0).abs().max() <= MEAN, float(off.mean(0).abs().max())
