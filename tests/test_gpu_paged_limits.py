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


# ---- the most rows of a call --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [1, 3, 5, 8, 12])
@pytest.mark.parametrize("rows,prefix", [(4096, 0), (3712, 21), (4096, 150)])
def test_attention_of_the_most_rows(paged, K, dtype, group, rows, prefix):
    """Every tile of query rows (1 to 2, 3 to 4, 5 to 8 and more heads a KV head) at up to 4096 rows."""
    ps, t = 16, DTYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(rows + group + prefix)
    shared = -(-prefix // ps)
    k = torch.randn(shared + 400, 1, ps, HD, generator=g, device="cuda").to(t)
    v = torch.randn(shared + 400, 1, ps, HD, generator=g, device="cuda").to(t)
    pool = paged.KVPool(k, v)
    pre = torch.arange(shared, dtype=torch.int32, device="cuda")
    table = torch.randint(shared, shared + 400, (rows, 2), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.randint(0, 33, (rows,), generator=g, device="cuda", dtype=torch.int32)
    q = torch.randn(rows, group * HD, generator=g, device="cuda")
    got = paged.attention(q, pool, table, lens, prefix_pages=pre if prefix else None, prefix_len=prefix)
    torch.cuda.synchronize()
    assert K.status() == 0
    # fp64, a few hundred rows at a time; a score of 128 products, ~9 in magnitude sum, has roundings of 2^-24 in at most
    # 16 steps, so a weight is off by under 1e-4 of itself
    for at in range(0, rows, 512):
        s = slice(at, min(at + 512, rows))
        n = s.stop - s.start

        def keys(x):
            own = x[table[s].long()].reshape(n, 2 * ps, HD).double()
            shared_part = x[:shared].reshape(1, -1, HD)[:, :prefix].double().expand(n, -1, -1)
            return torch.cat([shared_part, own], 1)

        live = torch.arange(2 * ps, device="cuda")[None] < lens[s][:, None]
        live = torch.cat([torch.ones(n, prefix, dtype=torch.bool, device="cuda"), live], 1)
        score = torch.einsum("bgd,btd->bgt", q[s].double().view(n, group, HD), keys(k)) / math.sqrt(HD)
        p = torch.softmax(score.masked_fill(~live[:, None], -math.inf), -1).nan_to_num(0.0)  # no key: zeros
        want = torch.einsum("bgt,btd->bgd", p, keys(v)).reshape(n, -1)
        mag = torch.einsum("bgt,btd->bgd", p, keys(v).abs()).reshape(n, -1)
        assert bool(((got[s].double() - want).abs() <= 1e-4 * mag).all())


# ---- the end of a step --------------------------------------------------------------------------
def host_commit(ids, tokens, pos, fresh, current, prompt_lens, limits):
    for j in range(len(ids)):
        if fresh[j] != 1:
            continue
        p, lim = pos[j] + 1, min(limits[j], tokens.shape[1])
        pos[j], nxt = p, -1
        if 0 <= p < lim:
            if p >= prompt_lens[j]:
                tokens[j, p] = ids[j]
            nxt = current[j] = tokens[j, p]
        if p + 1 >= lim or nxt < 0:
            fresh[j] = 0


@pytest.mark.parametrize("count,width", [(1, 4), (5, 9), (300, 33)])
def test_commit_tokens_against_a_host_loop(K, count, width):
    """Requests at every place of their rows: in the prompt, at its end, sampling, at the last position, ended, and
    without a token to take (-1), step after step."""
    from pyrite_b200 import _lib
    lib, rng = _lib.require(), np.random.default_rng(count)
    tokens = rng.integers(0, 1000, (count, width)).astype(np.int32)
    prompt_lens = rng.integers(1, width + 1, count).astype(np.int32)
    limits = np.minimum(prompt_lens + rng.integers(0, width, count), width + 2).astype(np.int32)  # some past the row
    pos = rng.integers(0, 2, count).astype(np.int32)
    fresh = (rng.random(count) < 0.9).astype(np.int32)
    current = rng.integers(0, 1000, count).astype(np.int32)
    dev = [torch.from_numpy(x.copy()).cuda() for x in (tokens, pos, fresh, current, prompt_lens, limits)]
    for step in range(width + 1):
        ids = rng.integers(0, 1000, count).astype(np.int32)
        ids[rng.random(count) < 0.05] = -1
        host_commit(ids, tokens, pos, fresh, current, prompt_lens, limits)
        d_ids = torch.from_numpy(ids).cuda()
        p = [x.data_ptr() for x in dev]
        assert lib.pyrite_cuda_commit_tokens(d_ids.data_ptr(), count, p[0], width, p[1], p[2], p[3], p[4], p[5],
                                             torch.cuda.current_stream().cuda_stream) == 0
        for got, want in zip(dev, (tokens, pos, fresh, current)):
            assert np.array_equal(got.cpu().numpy(), want), f"step {step}"
    assert not fresh.any() and K.status() == 0
