"""The recurrent language model of examples/recurrent_lm.py: it learns, decodes token by token what it computes for
whole sequences (packed prefill, states in a pool), and keeps its function when its projections are rotated."""
import math
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_example_trains_decodes_and_rotates(cuda):
    examples = str(Path(__file__).resolve().parents[1] / "examples")
    sys.path.insert(0, examples)
    try:
        import recurrent_lm
    finally:
        sys.path.remove(examples)
    out = recurrent_lm.main(["--steps", "60"])
    assert all(math.isfinite(v) for v in out["losses"])
    # an untrained model is at log 64 = 4.16; half of that is far below what chance gives
    assert out["losses"][-1] < 0.5 * out["losses"][0]
    # bf16 activations (2^-8 a rounding) through two blocks in two different orders of the same sums
    assert out["decode"] < 0.05
    # bf16 weights rounded once more by their rotation (2^-9 rms of each), and the activations likewise
    assert out["rotation"] < 0.05
