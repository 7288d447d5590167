"""Segments that long sequences of the delta rule are cut into, as the size of the workspace tells them, on any host."""
import ctypes as ct

import pytest

from cubutterfly_b200 import Status
from test_delta_ops import delta_fields

SMS = 148


def segments(lib, batch, length, heads, backward):
    """Of all sequences, K = V = 128 in bf16: what a workspace holds beside what every chunk needs."""
    size = ct.c_size_t()
    fields = delta_fields(batch=batch, length=length, k_heads=heads, heads=heads, k_dim=128, v_dim=128)
    assert lib.fn["B200GatedDeltaGetWorkspaceSize"](fields, backward, ct.byref(size)) == Status.SUCCESS
    chunks = batch * -(-length // 64) * heads
    matrix, state = 2 * 64 * 64 * 2, 2 * 128 * 128 * 2               # two pieces of 64 x 64 values, of a state
    rows = 64 * 128 * 2
    chunk = 8 * 64 * 4 + 2 * matrix + rows + 2 * rows                # factors, L and P, v, q and k
    if backward:
        chunk += matrix + rows + 2 * state + 4 * rows                # beta L, dO, S and dS, two pieces of R and W
    rest, per = size.value - chunks * chunk, heads * 128 * 128 * 4 * (3 if backward else 2)
    assert rest >= 0 and rest % per == 0
    return rest // per


@pytest.mark.parametrize("batch,length,heads,backward", [
    (1, 16384, 10, 0), (2, 8192, 4, 0), (1, 8192, 8, 0), (1, 8192, 14, 0), (1, 16384, 6, 1), (1, 16384, 14, 1), (2, 8192, 3, 1),
    (1, 4096, 14, 1), (1, 8192, 6, 1), (1, 65536, 3, 1), (1, 65536, 14, 1)])
def test_first_runs_fit_the_sms(lib, batch, length, heads, backward):
    """Ends and maps of so few chains run in one round: s - 1 and s - 2 of s segments, and s - 1 more backward."""
    each = segments(lib, batch, length, heads, backward) // batch
    assert each > 1 and (each * (3 if backward else 2) - (4 if backward else 3)) * batch * heads <= SMS


@pytest.mark.parametrize("batch,length,heads,backward", [(2, 8192, 40, 1), (4, 4096, 20, 1), (4, 4096, 24, 1), (1, 960, 1, 0), (64, 4096, 16, 0)])
def test_not_cut(lib, batch, length, heads, backward):
    """Two segments' first runs would be a round of their own; short sequences; chains enough."""
    assert segments(lib, batch, length, heads, backward) == 0
