"""Operators on drafted tokens at calls that are allowed and rare: expanded and padded tensors, the largest shapes, random numbers next to a border, values next to the types' ends."""
import pytest
import torch

from tests.gpu_util import ctx
from tests.test_gpu_draft import gen_of, ints, make_cache

pytestmark = pytest.mark.gpu


# ---- rows that are one row in memory
EXPANDED = [((1, 1), (5, 3)), ((5, 1), (5, 3)), ((1, 3), (5, 3)), ((1,), (15,))]


def expanded(g, small, shape, heads, dim):
    return torch.randn((*small, heads, dim), generator=g).bfloat16().cuda().expand(*shape, heads, dim)


@pytest.mark.parametrize("small,shape", EXPANDED)
def test_expanded_rows_turn_as_dense_ones_do(small, shape):
    g = gen_of(3)
    q, k = expanded(g, small, shape, 4, 64), expanded(g, small, shape, 2, 64)
    positions, freq = torch.arange(15, dtype=torch.int32).cuda() * 7, (0.5 ** torch.arange(32)).float().cuda()
    got = ctx().rope_rows(q, k, positions, freq)
    want = ctx().rope_rows(q.contiguous(), k.contiguous(), positions, freq)
    ctx().sync()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and got[0].shape == q.shape


@pytest.mark.parametrize("small,shape", EXPANDED)
@pytest.mark.parametrize("which", ["query", "key", "value"])
def test_expanded_rows_are_appended_as_dense_ones_are(small, shape, which):
    g = gen_of(4)
    table, context, positions, freq = torch.randperm(10, generator=g).to(torch.int32).reshape(5, 2).cuda(), ints(0, 1, 4, 5, 2), torch.arange(15, dtype=torch.int32).cuda(), (0.5 ** torch.arange(32)).float().cuda()
    rows = {n: torch.randn((15, h, 64), generator=g).bfloat16().cuda() for n, h in (("query", 4), ("key", 2), ("value", 2))}
    rows[which] = expanded(g, small, shape, rows[which].shape[1], 64)
    done = []
    for dense in (False, True):
        k_pages, v_pages = (torch.zeros((10, 4, 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q, k, v = (rows[n].contiguous() if dense else rows[n] for n in ("query", "key", "value"))
        done.append((ctx().rope_append(q, k, v, k_pages, v_pages, table, context, positions, freq), k_pages, v_pages))
    ctx().sync()
    assert all(torch.equal(x, y) for x, y in zip(*done))


@pytest.mark.parametrize("small,shape", EXPANDED[:3])
@pytest.mark.parametrize("heads", [4, 48])
def test_expanded_queries_attend_as_dense_ones_do(small, shape, heads):
    g = gen_of(5)
    k_pages, v_pages, table = make_cache(g, 5, 2, 64, 16, 4, torch.bfloat16)
    q, context = expanded(g, small, shape, heads, 64), ints(40, 0, 7, 61, 33)
    got = ctx().tree_attention(q, k_pages, v_pages, table, context)
    want = ctx().tree_attention(q.contiguous(), k_pages, v_pages, table, context)
    ctx().sync()
    assert torch.equal(got, want)
