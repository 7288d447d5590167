"""The workspace queries of the delta rule and the norm of queries and keys, on any host, with no more than their documented
fields."""
import ctypes as ct

import pytest

from cubutterfly_b200 import Status
from test_delta_ops import UNSUPPORTED, P, delta_fields, qk_fields

NOTHING = dict(scale=0.0, **{n: 0 for n in ("q", "k", "v", "g", "beta", "o", "final", "workspace", "bytes")})


def query(lib, name, *args):
    size = ct.c_size_t()
    assert lib.fn[name](*args, ct.byref(size)) == Status.SUCCESS, lib.fn["GetLastErrorString"]().decode()
    return size.value


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("data", [0, 1, 2])
@pytest.mark.parametrize("shape", [dict(), dict(batch=1, length=4096, k_heads=1, heads=1, k_dim=128, v_dim=128),
                                   dict(batch=1, length=5000, sequences=7, offsets=P)], ids=str)
def test_delta_workspace_of_sizes_alone(lib, shape, data, backward):
    bare = query(lib, "B200GatedDeltaGetWorkspaceSize", delta_fields(**{**NOTHING, **shape, "data": data, "g_type": 0, "b_type": 0}), backward)
    assert bare > 0 and bare == query(lib, "B200GatedDeltaGetWorkspaceSize", delta_fields(**shape, data=data, g_type=2, b_type=2), backward)


def test_norm_workspace_of_sizes_alone(lib):
    nothing = {n: 0 for n in ("q_heads", "k_heads", "rotary", "axis_count", "axis", "period", "q", "k", "k_weight", "positions",
                              "frequencies", "q_out", "k_out", "data", "qw_type", "kw_type", "eps")}
    bare = query(lib, "B200QkNormGetWorkspaceSize", qk_fields(**nothing))
    assert bare == query(lib, "B200QkNormGetWorkspaceSize", qk_fields()) > 0


def test_queries_still_refuse_sizes(lib):
    size = ct.c_size_t()
    assert lib.fn["B200GatedDeltaGetWorkspaceSize"](delta_fields(**{**NOTHING, "k_dim": 129}), 0, ct.byref(size)) == UNSUPPORTED
    assert lib.fn["B200QkNormGetWorkspaceSize"](qk_fields(dim=257), ct.byref(size)) == UNSUPPORTED
