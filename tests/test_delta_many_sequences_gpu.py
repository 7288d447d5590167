"""Packed batches of many sequences, whose chains start by length: equal lengths, empty sequences, the longest ones first, last
and in between, at and around the numbers where the order is found by one value a lane, by two, and not at all."""
import pytest
import torch

from test_delta_ops_gpu import check_delta, delta_case

pytestmark = pytest.mark.gpu

COUNTS = [2, 31, 32, 33, 34, 63, 64, 65, 100]


def lengths(count, order):
    some = [(7 * j + 3) % 23 // 3 for j in range(count)]      # 0 to 7, each several times
    some[order % count], some[(order + count // 2) % count] = 150, 70
    return some


def offsets(sizes):
    cuts = [0]
    for n in sizes:
        cuts.append(cuts[-1] + n)
    return cuts


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("order", [0, 31, 32, -1])
@pytest.mark.parametrize("count", COUNTS)
def test_order_of_sequences(cuda, count, order, dtype):
    cuts = offsets(lengths(count, order))
    check_delta(delta_case(1, cuts[-1], 1, 2, 16, 24, dtype, cuts=cuts, state=True, seed=count), cuts)


@pytest.mark.parametrize("sizes", [[3] * 64, [3] * 65, [0] * 40 + [5], [0] * 63 + [1], [1, 0] * 32, list(range(50)), list(range(50, 0, -1))],
                         ids=lambda s: f"{len(s)} of {s[0]} to {s[-1]}")
def test_equal_empty_and_sorted_sequences(cuda, sizes):
    cuts = offsets(sizes)
    check_delta(delta_case(1, cuts[-1], 1, 1, 16, 16, torch.bfloat16, cuts=cuts, state=True, seed=7), cuts)
