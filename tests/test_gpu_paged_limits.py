"""The paged cache at the ends of its ranges on a B200: ids that no pool can have, the most rows of a call, the
end of a step.

Oracles: expected arrays written out by hand, a host loop, fp64 torch.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HD = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BAD_PAGE = 4  # the device status bit of an id that fits no pool


@pytest.fixture(scope="module")
def K(cuda_device):
    from pyrite_b200.kernels import cuda
    cuda.status()
    return cuda


@pytest.fixture(scope="module")
def paged(cuda_device):
    from pyrite_b200.kernels import paged
    return paged


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---- page ids that no pool can have ----------------------------------------------------------
@pytest.mark.parametrize("row_stride", [1, 0])
@pytest.mark.parametrize("ps,bad", [(16, 1 << 27), (16, 1 << 28), (16, (1 << 28) + 1), (16, 2 ** 31 - 1), (16, -1),
                                    (16, -2 ** 31), (256, 1 << 23), (256, 1 << 24)])
def test_tables_give_no_slot_for_a_page_that_no_pool_has(paged, K, ps, bad, row_stride):
    """A page whose slots pass 2^31 - 1, or a negative one: slot -1 and the status bit, not a slot of another page."""
    lens, free = ints([0, 5, ps, 3]), ints([7, bad, 9])
    table = torch.full((4, 2), -1, dtype=torch.int32, device="cuda")
    table[1, 0], table[2, 0], table[3, 0] = 4, 5, bad
    out = paged.TokenSlots.empty(4, capacity=4, row_stride=row_stride)
    paged.page_tables(lens, ints([1, 1, 1, 1]), ps, free, ints([0]), table, out)
    torch.cuda.synchronize()
    assert K.status() == BAD_PAGE
    assert out.slots.tolist() == [7 * ps, 4 * ps + 5, -1, -1]  # request 2's fresh page, request 3's held one
    assert out.positions.tolist() == [0, 5, ps, 3] and out.kv_lens.tolist() == [1, 6, ps + 1, 4]
    assert table.tolist() == [[7, -1], [4, -1], [5, bad], [bad, -1]]


@pytest.mark.parametrize("ps", [16, 64, 256])
def test_tables_take_the_last_page_that_a_pool_can_have(paged, K, ps):
    last = 0x7FFFFFFF // ps
    last -= (last * ps + ps - 1) > 0x7FFFFFFF
    out = paged.TokenSlots.empty(1, capacity=ps)
    table = torch.full((1, 1), -1, dtype=torch.int32, device="cuda")
    paged.page_tables(ints([0]), ints([ps]), ps, ints([last]), ints([0]), table, out)
    torch.cuda.synchronize()
    assert K.status() == 0 and out.slots.tolist() == list(range(last * ps, last * ps + ps))


@pytest.mark.parametrize("slot", [-2, -17, -2 ** 31])
def test_append_and_store_report_slots_below_none(paged, K, slot):
    """-1 stores nothing, quietly; any other slot outside the pool stores nothing and is reported."""
    pool = paged.KVPool.zeros(2, 1, 16, torch.float32)
    rope = torch.zeros(4, 64, 2, dtype=torch.float64, device="cuda")
    x = torch.ones(2, 3 * HD, device="cuda")
    for other in (-1, slot):
        paged.append_kv(x, pool, ints([other, 5]), ints([0, 1]), rope, 1)
        torch.cuda.synchronize()
        assert K.status() == (0 if other == -1 else BAD_PAGE)
        paged.store_kv(x[:, :HD], x[:, HD:2 * HD], pool, ints([6, other]))
        torch.cuda.synchronize()
        assert K.status() == (0 if other == -1 else BAD_PAGE)
    assert pool.v[:, 0].any(-1).flatten().nonzero().flatten().tolist() == [5, 6]
