"""Operators on drafted tokens over a paged cache against plain 64-bit forms (tests/draft_ref.py)."""
import math

import pytest
import torch

from tests import draft_ref as R
from tests.gpu_util import ctx

pytestmark = pytest.mark.gpu


def gen_of(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make_cache(gen, batch, kv, dim, page, blocks, dtype, spare=3, scale=1.0):
    """Pages in random order, some that nobody uses."""
    pages = batch * blocks + spare
    table = torch.randperm(pages, generator=gen)[:batch * blocks].to(torch.int32).reshape(batch, blocks).cuda()
    k, v = ((torch.randn((pages, page, kv, dim), generator=gen) * scale).to(dtype).cuda() for _ in range(2))
    return k, v, table


# ---- trees
@pytest.mark.parametrize("batch,rows,chain", [(1, 1, True), (2, 7, False), (5, 64, False), (3, 65, True), (2, 130, False), (1, 1024, True)])
def test_tree_positions_and_mask(batch, rows, chain):
    g = gen_of(rows)
    parents = R.trees(g, batch, rows, chain)
    context = torch.randint(0, 1 << 20, (batch,), generator=g, dtype=torch.int32)
    drafted = torch.randint(0, rows + 1, (batch,), generator=g, dtype=torch.int32)
    drafted[0] = rows
    positions, mask = ctx().draft_tree(parents.cuda(), context.cuda(), drafted.cuda())
    ctx().sync()
    want, sees = R.tree(parents, context, drafted)
    assert torch.equal(positions.cpu(), want)
    assert torch.equal(mask.cpu(), R.words(sees))


def test_one_tree_for_all_sequences_and_no_lengths():
    parents = R.trees(gen_of(3), 1, 21)
    context = ints(4, 0, 100)
    positions, mask = ctx().draft_tree(parents[0].cuda(), context)
    ctx().sync()
    want, sees = R.tree(parents.expand(3, -1), context.cpu(), [21] * 3)
    assert torch.equal(positions.cpu(), want) and torch.equal(mask.cpu(), R.words(sees))


def test_bad_parents_and_lengths_are_left_out_and_reported():
    from zllm_b200 import ffi

    parents = torch.tensor([[-1, 0, 2, 2, 1], [-1, -2, 1, 0, 9]], dtype=torch.int32)  # row 2 of the first tree below itself; rows 1 and 4 of the second
    positions, mask = ctx().draft_tree(parents.cuda(), ints(10, 20))
    with pytest.raises(ffi.ZqFailure) as e:
        ctx().sync()
    assert e.value.code == 5
    want, sees = R.tree(parents, [10, 20], [5, 5])
    assert want.tolist() == [[10, 11, -1, -1, 12], [20, -1, -1, 21, -1]]
    assert torch.equal(positions.cpu(), want) and torch.equal(mask.cpu(), R.words(sees))
    for context, drafted in ((ints(3, -1), ints(5, 5)), (ints(3, 2 ** 31 - 2), ints(5, 5)), (ints(3, 0), ints(5, 6)), (ints(3, 0), ints(5, -1))):
        positions, mask = ctx().draft_tree(R.trees(gen_of(1), 2, 5).cuda(), context, drafted)
        with pytest.raises(ffi.ZqFailure):
            ctx().sync()
        assert (positions[1] == -1).all() and (mask[1] == 0).all() and (positions[0] >= 3).all()


# ---- rotary positions
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved,suffix,inverse", [(False, False, False), (True, False, True), (False, True, True), (True, True, False)])
@pytest.mark.parametrize("rows,heads,kv,dim,rotary", [(1, 24, 8, 64, 64), (5, 3, 1, 10, 6), (9, 4, 4, 80, 32), (2, 1, 1, 128, 8), (33, 5, 1, 72, 72), (3, 40, 8, 256, 250), (7, 6, 2, 16, 16), (4, 3, 3, 2, 2), (2, 64, 64, 128, 128)])
def test_rope_rows(dtype, interleaved, suffix, inverse, rows, heads, kv, dim, rotary):
    g = gen_of(rows * dim)
    q, k = torch.randn((rows, heads, dim), generator=g).to(dtype), torch.randn((rows, kv, dim), generator=g).to(dtype)
    positions = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=torch.int32)
    positions[0] = 0
    positions[rows // 2] = -1
    freq = (10000.0 ** (-torch.arange(rotary // 2) / (rotary // 2))).float()
    got_q, got_k = ctx().rope_rows(q.cuda(), k.cuda(), positions.cuda(), freq.cuda(), interleaved=interleaved, suffix=suffix, factor=1.25, inverse=inverse)
    ctx().sync()
    for got, x in ((got_q, q), (got_k, k)):
        want = R.rotate(x, positions, freq, 1.25, interleaved, suffix, inverse)
        # the result is rounded once; cos and sin are off by 1.5e-7 at most (half a turn in f32: 2^-25 of a turn, twice sincospif's 2^-23), both products and the sum by half a step of f32
        reach = 1.25 * 2 * x.double().abs().amax()
        assert ((got.cpu().double() - want).abs() <= R.half_step(dtype) * want.abs() + reach * 6 * 2.0 ** -23).all()


def test_rope_rows_takes_strided_rows_and_works_in_place_of_nothing():
    g = gen_of(8)
    fused = torch.randn((6, 7, 32), generator=g).cuda()
    before = fused.clone()
    positions, freq = ints(5, 0, 9, 100, -1, 3), (0.5 ** torch.arange(16)).float().cuda()
    q, k = ctx().rope_rows(fused[:, :4], fused[:, 4:6], positions, freq)
    dense_q, dense_k = ctx().rope_rows(fused[:, :4].contiguous(), fused[:, 4:6].contiguous(), positions, freq)
    ctx().sync()
    assert torch.equal(q, dense_q) and torch.equal(k, dense_k) and torch.equal(fused, before)
    turned, none = ctx().rope_rows(fused[:, :4].transpose(1, 2).contiguous().transpose(1, 2), None, positions, freq)
    ctx().sync()
    assert none is None and torch.equal(turned, dense_q)
    back, _ = ctx().rope_rows(turned, None, positions, freq, inverse=True)
    ctx().sync()
    # each turn is off by 6 * 2^-23 of the largest value
    assert (back - fused[:, :4]).abs().max() <= 4 * 6 * 2.0 ** -23 * fused.abs().max() * 2


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,heads,kv,dim,page,rotary", [(1, 1, 8, 8, 64, 16, 64), (3, 13, 8, 2, 128, 8, 64), (2, 5, 3, 1, 24, 1, 10), (2, 70, 4, 1, 96, 64, 96)])
def test_rope_append_writes_the_cache_and_nothing_else(dtype, batch, rows, heads, kv, dim, page, rotary):
    g = gen_of(rows + dim)
    context = torch.randint(0, 40, (batch,), generator=g, dtype=torch.int32)
    drafted = torch.randint(0, rows + 1, (batch,), generator=g, dtype=torch.int32)
    drafted[0] = rows
    k_pages, v_pages, table = make_cache(g, batch, kv, dim, page, -(-(40 + rows) // page), dtype)
    q = torch.randn((batch, rows, heads, dim), generator=g).to(dtype).cuda()
    kv_rows = torch.randn((batch, rows, 2 * kv, dim), generator=g).to(dtype).cuda()  # k and v of one projection, side by side
    positions = torch.randint(0, 5000, (batch * rows,), generator=g, dtype=torch.int32)
    if rows > 4:
        positions[2] = -1
    freq = (1000.0 ** (-torch.arange(rotary // 2) / (rotary // 2))).float().cuda()
    want_k, want_v = k_pages.clone(), v_pages.clone()
    turned_q, turned_k = ctx().rope_rows(q, kv_rows[:, :, :kv], positions.cuda(), freq, factor=0.75)
    for b in range(batch):
        for i in range(int(drafted[b])):
            if positions[b * rows + i] >= 0:
                at = R.cache_row(table[b].cpu(), page, int(context[b]) + i)
                want_k[at], want_v[at] = turned_k[b, i], kv_rows[b, i, kv:]
    got_q = ctx().rope_append(q, kv_rows[:, :, :kv], kv_rows[:, :, kv:], k_pages, v_pages, table, context.cuda(), positions.cuda(), freq, draft_lens=drafted.cuda(), factor=0.75)
    ctx().sync()
    assert torch.equal(got_q, turned_q) and torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved,suffix", [(False, False), (True, True)])
@pytest.mark.parametrize("heads,kv,dim,rotary", [(4, 1, 64, 64), (6, 3, 96, 32), (3, 1, 128, 128), (40, 8, 128, 128), (1, 1, 8, 8)])
def test_many_rows_turn_as_few_do(dtype, interleaved, suffix, heads, kv, dim, rotary):
    """Rows by the thousand get fewer threads each than rows by the hundred; same values, same sines, same order of operations."""
    g = gen_of(heads + dim)
    rows = 5000
    q, k = torch.randn((rows, heads, dim), generator=g).to(dtype).cuda(), torch.randn((rows, kv, dim), generator=g).to(dtype).cuda()
    positions = torch.randint(-1, 1 << 17, (rows,), generator=g, dtype=torch.int32).cuda()
    freq = (10000.0 ** (-torch.arange(rotary // 2) / (rotary // 2))).float().cuda()
    got_q, got_k = ctx().rope_rows(q, k, positions, freq, interleaved=interleaved, suffix=suffix, factor=1.1)
    parts = [ctx().rope_rows(q[i:i + 500], k[i:i + 500], positions[i:i + 500], freq, interleaved=interleaved, suffix=suffix, factor=1.1) for i in range(0, rows, 500)]
    ctx().sync()
    assert torch.equal(got_q, torch.cat([p[0] for p in parts])) and torch.equal(got_k, torch.cat([p[1] for p in parts]))


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (5, 5, 40)])
def test_many_rows_are_appended_as_few_are(heads, kv, dim):
    g = gen_of(dim)
    batch, rows, page = 13, 150, 16
    k_pages, v_pages, table = make_cache(g, batch, kv, dim, page, 14, torch.bfloat16)
    table[3, 2] = 10 ** 6  # a page that is none
    q, k, v = (torch.randn((batch, rows, h, dim), generator=g).bfloat16().cuda() for h in (heads, kv, kv))
    context = torch.randint(0, 70, (batch,), generator=g, dtype=torch.int32).cuda()
    drafted = torch.randint(0, rows + 1, (batch,), generator=g, dtype=torch.int32).cuda()
    positions = torch.randint(-1, 9000, (batch * rows,), generator=g, dtype=torch.int32).cuda()
    freq = (10000.0 ** (-torch.arange(dim // 2) / (dim // 2))).float().cuda()
    want_k, want_v = k_pages.clone(), v_pages.clone()
    got_q = ctx().rope_append(q, k, v, k_pages, v_pages, table, context, positions, freq, draft_lens=drafted)
    want_q = [ctx().rope_append(q[b:b + 1], k[b:b + 1], v[b:b + 1], want_k, want_v, table[b:b + 1], context[b:b + 1], positions[b * rows:(b + 1) * rows], freq, draft_lens=drafted[b:b + 1]) for b in range(batch)]
    from zllm_b200 import ffi

    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    assert torch.equal(got_q, torch.cat(want_q)) and torch.equal(k_pages, want_k) and torch.equal(v_pages, want_v)


def test_rope_append_skips_rows_without_a_page():
    from zllm_b200 import ffi

    k_pages, v_pages = torch.zeros((4, 4, 1, 8), dtype=torch.float16, device="cuda"), torch.zeros((4, 4, 1, 8), dtype=torch.float16, device="cuda")
    table = torch.tensor([[0, 1], [4, 2], [3, -1], [0, 0]], dtype=torch.int32, device="cuda")
    ones = torch.ones((4, 3, 1, 8), dtype=torch.float16, device="cuda")
    ctx().rope_append(ones, ones, ones, k_pages, v_pages, table, ints(6, 2, 3, -5), torch.zeros(12, dtype=torch.int32, device="cuda"), torch.ones(4, device="cuda"))
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    # sequence 0: positions 6, 7, then past its table; sequence 1: 2, 3 in a page that is none, 4 in page 2; sequence 2: 3 in page 3, then none; sequence 3: no length
    want = torch.zeros((4, 4))
    want[1, 2:] = 1
    want[2, 0] = 1
    want[3, 3] = 1
    assert torch.equal(v_pages[:, :, 0, 0].cpu().float(), want) and torch.equal(k_pages[:, :, 0, 0].cpu().float(), want)


# ---- attention
def run_attention(g, batch, rows, heads, kv, dim, page, contexts, dtype, tree, drafted=None, scale=None, stride_pages=False, sharpen=1.0):
    blocks = -(-(max(contexts) + rows) // page)
    k_pages, v_pages, table = make_cache(g, batch, kv, dim, page, blocks, dtype)
    if stride_pages:  # K and V pages side by side
        both = torch.stack([k_pages, v_pages], 1)
        k_pages, v_pages = both[:, 0], both[:, 1]
    q = (torch.randn((batch, rows, heads, dim), generator=g) * sharpen).to(dtype).cuda()
    context = ints(*contexts)
    n = torch.tensor(drafted if drafted is not None else [rows] * batch, dtype=torch.int32)
    parents = R.trees(g, batch, rows)
    _, sees = R.tree(parents, context.cpu(), n)
    mask = R.words(sees).cuda()
    if not tree:
        mask, sees = None, torch.ones((rows, rows), dtype=torch.bool).tril().expand(batch, -1, -1)
    got = ctx().tree_attention(q, k_pages, v_pages, table, context, mask=mask, draft_lens=n.cuda() if drafted is not None else None, scale=scale)
    ctx().sync()
    want, bound = R.attention(q, k_pages, v_pages, table, context, sees, n, scale or 1 / math.sqrt(dim))
    assert ((got.double() - want).abs() <= bound).all(), float(((got.double() - want).abs() - bound).max())
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [8, 64, 80, 96, 128, 192, 256])
@pytest.mark.parametrize("rows,heads,kv", [(1, 4, 4), (3, 16, 2), (7, 8, 2), (17, 5, 1), (9, 32, 1)])
def test_attention_of_head_shapes(dtype, dim, rows, heads, kv):
    run_attention(gen_of(dim + rows), 2, rows, heads, kv, dim, 16, [37, 300], dtype, tree=rows > 1)


@pytest.mark.parametrize("context", [0, 1, 15, 16, 31, 32, 63, 64, 65, 127, 128, 255, 256, 257, 1000])
@pytest.mark.parametrize("rows,page,tree", [(1, 16, False), (2, 1, True), (6, 64, True), (20, 8, False)])
def test_attention_at_borders_of_tiles_and_pages(context, rows, page, tree):
    run_attention(gen_of(context), 1, rows, 4, 2, 64, page, [context], torch.float16, tree)


@pytest.mark.parametrize("rows,group", [(1, 1), (13, 4), (64, 8)])
def test_attention_of_unequal_lengths(rows, group):
    drafted = [rows, max(0, rows - 1), rows, 0, 1, rows]
    run_attention(gen_of(rows), 6, rows, 2 * group, 2, 128, 32, [2000, 3, 0, 77, 511, 1024], torch.bfloat16, True, drafted=drafted)


@pytest.mark.parametrize("rows,group,dim,page", [(5, 5, 64, 4), (9, 7, 128, 2), (3, 8, 96, 4), (40, 2, 80, 1), (17, 1, 40, 32), (9, 4, 48, 8)])
def test_attention_of_pages_and_heads_that_the_fast_kernel_does_not_take(rows, group, dim, page):
    run_attention(gen_of(dim), 2, rows, 2 * group, 2, dim, page, [33, 500], torch.bfloat16, True)
    run_attention(gen_of(dim + 1), 3, rows, 2 * group, 2, dim, page, [0, 1200, 7], torch.float16, False, drafted=[rows, 2, 0])


@pytest.mark.parametrize("rows,group", [(1024, 1), (700, 3), (129, 2)])
def test_attention_of_many_rows(rows, group):
    run_attention(gen_of(rows), 1, rows, group, 1, 64, 16, [70], torch.float16, rows != 700)


def test_attention_of_queries_that_lie_apart():
    g = gen_of(13)
    k_pages, v_pages, table = make_cache(g, 2, 2, 64, 16, 8, torch.float16)
    for extra in (0, 2, 3, 8):  # rows of a fused projection; with 3 more values their distance is odd
        fused = torch.randn((2, 6, 8 * 64 + extra), generator=g).half().cuda()
        q = fused[..., :8 * 64].unflatten(-1, (8, 64))
        got = ctx().tree_attention(q, k_pages, v_pages, table, ints(100, 17))
        want = ctx().tree_attention(q.contiguous(), k_pages, v_pages, table, ints(100, 17))
        ctx().sync()
        assert torch.equal(got, want)
    got = ctx().tree_attention(q.transpose(0, 1).contiguous().transpose(0, 1), k_pages, v_pages, table, ints(100, 17))
    ctx().sync()
    assert torch.equal(got, want)


def test_attention_over_a_long_context():
    run_attention(gen_of(1), 1, 2, 4, 1, 128, 64, [40000], torch.bfloat16, True)


def test_attention_of_sharp_scores_and_strided_pages():
    run_attention(gen_of(2), 2, 4, 8, 2, 64, 16, [90, 700], torch.float16, True, stride_pages=True, sharpen=30.0)
    run_attention(gen_of(3), 2, 4, 8, 2, 64, 16, [90, 700], torch.bfloat16, False, scale=0.9)


def test_attention_of_many_sequences():
    g = gen_of(11)
    contexts = torch.randint(0, 60, (700,), generator=g).tolist()
    run_attention(g, 700, 1, 2, 1, 64, 16, contexts, torch.float16, False)


# more units than CTAs: shares that end and begin inside items, between them, and over many short ones
@pytest.mark.parametrize("rows,group,dim", [(1, 1, 128), (1, 8, 64), (3, 8, 128), (6, 8, 128), (9, 5, 64), (20, 8, 128), (70, 4, 64)])
@pytest.mark.parametrize("longest", [60, 400, 1500])
def test_attention_of_shares_that_cross_items(rows, group, dim, longest):
    g = gen_of(90 + rows + longest)
    contexts = torch.randint(0, longest + 1, (93,), generator=g).tolist()
    drafted = torch.randint(0, rows + 1, (93,), generator=g).tolist()
    run_attention(g, 93, rows, 2 * group, 2, dim, 16, contexts, torch.bfloat16, tree=True, drafted=drafted)


# few long items over all CTAs, many parts each
@pytest.mark.parametrize("rows,group,context", [(1, 4, 30011), (2, 24, 9001), (66, 2, 20000), (1, 1, 148 * 128 - 1)])
@pytest.mark.parametrize("dim", [64, 128, 192])
def test_attention_of_items_in_many_parts(rows, group, context, dim):
    run_attention(gen_of(300 + rows), 1, rows, group, 1, dim, 64, [context], torch.float16, tree=True)


@pytest.mark.parametrize("rows,group", [(6, 1), (6, 5), (12, 8)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, rows, group, poison):
    """Masked drafted rows, unused parts of pages and pages of nobody hold infinities and NaN; one row sees an infinity."""
    g = gen_of(5)
    kv, dim, page, context = 2, 64, 16, 45
    k_pages, v_pages, table = make_cache(g, 1, kv, dim, page, 6, dtype)
    q = torch.randn((1, rows, group * kv, dim), generator=g).to(dtype).cuda()
    parents = torch.tensor([[-1] + [0] * (rows - 1)], dtype=torch.int32)
    n = rows - 1
    _, sees = R.tree(parents, [context], [n])
    mask = R.words(sees).cuda()
    clean = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask, draft_lens=ints(n))
    for pages in (k_pages, v_pages):
        flat = pages.view(-1, kv, dim)
        used = torch.zeros(flat.shape[0], dtype=torch.bool)
        for p in range(context + n):
            b, o = R.cache_row(table[0].cpu(), page, p)
            used[b * page + o] = True
        flat[~used.cuda()] = poison
        b, o = R.cache_row(table[0].cpu(), page, context + 2)  # a drafted row that row 2 alone sees
        pages[b, o] = poison
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask, draft_lens=ints(n))
    ctx().sync()
    others = [i for i in range(rows) if i != 2]
    assert torch.equal(got[:, others], clean[:, others]) and torch.isfinite(got[:, others]).all()
    assert not torch.isfinite(got[:, 2]).any()
    assert (got[:, n:] == 0).all()


def test_a_visible_infinity_of_a_value_keeps_its_sign_and_column():
    g = gen_of(6)
    k_pages, v_pages, table = make_cache(g, 1, 1, 64, 16, 4, torch.float16)
    q = torch.randn((1, 3, 2, 64), generator=g).half().cuda()
    b, o = R.cache_row(table[0].cpu(), 16, 21)
    v_pages[b, o, 0, 7], v_pages[b, o, 0, 30] = math.inf, -math.inf
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(20))  # a chain: rows 1 and 2 see position 21
    ctx().sync()
    assert torch.isfinite(got[:, 0]).all()
    assert (got[:, 1:, :, 7] == math.inf).all() and (got[:, 1:, :, 30] == -math.inf).all()
    rest = [c for c in range(64) if c not in (7, 30)]
    assert torch.isfinite(got[..., rest]).all()


def test_rows_that_see_nothing_are_zero():
    g = gen_of(7)
    k_pages, v_pages, table = make_cache(g, 2, 2, 64, 16, 2, torch.bfloat16)
    q = torch.randn((2, 5, 4, 64), generator=g).bfloat16().cuda()
    mask = torch.zeros((2, 5, 1), dtype=torch.int64, device="cuda")
    mask[0, 1] = 0b10
    mask[0, 4] = 0b10010
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(0, 0), mask=mask)
    ctx().sync()
    assert (got[0, [0, 2, 3]] == 0).all() and (got[1] == 0).all() and (got[0, 1] != 0).any()
    one = R.gathered(v_pages, table[0], 5)[1].repeat_interleave(2, 0)
    assert torch.equal(got[0, 1].double(), one)  # one key: its value as it is


def test_bad_pages_and_lengths_are_reported():
    from zllm_b200 import ffi

    g = gen_of(9)
    k_pages, v_pages, table = make_cache(g, 3, 1, 64, 16, 4, torch.float16)
    q = torch.randn((3, 2, 2, 64), generator=g).half().cuda()
    good = ctx().tree_attention(q, k_pages, v_pages, table, ints(30, 20, 10))
    ctx().sync()
    for change in ("page", "negative page", "context", "negative context", "drafted"):
        t, c, n = table.clone(), ints(30, 20, 10), ints(2, 2, 2)
        if "page" in change:
            t[1, 0] = 15 if change == "page" else -1
        elif change == "drafted":
            n[1] = 3
        else:
            c[1] = 63 if change == "context" else -1
        got = ctx().tree_attention(q, k_pages, v_pages, t, c, draft_lens=n)
        with pytest.raises(ffi.ZqFailure):
            ctx().sync()
        assert torch.equal(got[[0, 2]], good[[0, 2]])
        if "page" not in change:
            assert (got[1] == 0).all()


# ---- verification
def run_verify(g, batch, rows, vocab, dtype, drawn, temperature, drafted=None, spread=2.0, chain=False):
    logits = (torch.randn((batch, rows, vocab), generator=g) * spread).to(dtype)
    near = logits.float() + torch.randn((batch, rows, vocab), generator=g) * 0.7
    parents = R.trees(g, batch, rows, chain)
    heat = torch.tensor(temperature, dtype=torch.float32).expand(batch).contiguous()
    up = parents.clamp(min=0).long().unsqueeze(2).expand(-1, -1, vocab)
    noise = -torch.log(-torch.log(torch.rand((batch, rows, vocab), generator=g).clamp(1e-9, 1 - 1e-6)))
    draft = near.to(dtype)
    tokens = (torch.gather(draft.float(), 1, up) / heat.clamp(min=0.05).reshape(-1, 1, 1) + noise * (1.0 if drawn else 0.4)).argmax(2).to(torch.int32)
    accept_u, sample_u = torch.rand((batch, rows), generator=g), torch.rand(batch, generator=g)
    n = torch.tensor(drafted if drafted is not None else [rows] * batch, dtype=torch.int32)
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), accept_u.cuda(), sample_u.cuda(), heat.cuda(), draft_logits=draft.cuda() if drawn else None, draft_lens=n.cuda() if drafted is not None else None)
    ctx().sync()
    want = R.verify(logits, draft if drawn else None, tokens, parents, accept_u, sample_u, heat, n)
    check_verify(got, want, rows)
    return want


def check_verify(got, want, rows):
    path, accepted, token = (t.cpu().tolist() for t in got)
    for b, (p, a, t) in enumerate(want):
        assert accepted[b] == a and path[b] == p + [-1] * (rows - len(p)), (b, path[b], p)
        assert t is None or token[b] == t, (b, token[b], t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("batch,rows,vocab", [(1, 1, 1), (1, 4, 3), (40, 9, 17), (5, 6, 255), (3, 8, 4099), (2, 5, 70001), (200, 3, 1000)])
def test_verification(dtype, drawn, batch, rows, vocab):
    run_verify(gen_of(vocab + rows), batch, rows, vocab, dtype, drawn, 0.9)


@pytest.mark.parametrize("drawn", [False, True])
def test_verification_of_unequal_sequences_and_temperatures(drawn):
    g = gen_of(4)
    want = run_verify(g, 8, 12, 300, torch.float32, drawn, [0.0, 0.3, 1.0, 2.5, 0.0, 0.01, 1.0, 1e-30], drafted=[12, 12, 5, 1, 7, 12, 0, 12])
    assert want[6] == ([], 0, -1)


@pytest.mark.parametrize("drawn", [False, True])
def test_verification_of_long_chains_and_wide_nodes(drawn):
    run_verify(gen_of(21), 4, 200, 50, torch.float32, drawn, 1.5, chain=True, spread=0.3)
    g = gen_of(22)
    vocab, rows = 40, 120
    logits = torch.randn((6, rows, vocab), generator=g)
    draft = torch.randn((6, rows, vocab), generator=g) * 2
    parents = torch.zeros((6, rows), dtype=torch.int32)
    parents[:, 0] = -1
    tokens = torch.randint(0, vocab, (6, rows), generator=g, dtype=torch.int32)  # every token several times
    accept_u, sample_u = 0.9 + 0.1 * torch.rand((6, rows), generator=g), torch.rand(6, generator=g)
    accept_u[:3] = 1 - 2.0 ** -24
    heat = torch.ones(6)
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents[0].cuda(), accept_u.cuda(), sample_u.cuda(), heat.cuda(), draft_logits=draft.cuda() if drawn else None)
    ctx().sync()
    check_verify(got, R.verify(logits, draft if drawn else None, tokens, parents, accept_u, sample_u, heat, [rows] * 6), rows)


def test_ties_go_to_the_lowest_token_and_masked_tokens_never_come():
    logits = torch.full((3, 2, 9000), -math.inf)
    logits[0, 0, [17, 4000, 8999]] = 2.0
    logits[1, 0, 8999] = -5.0
    logits[2, 0, [0, 8998]] = 1.0
    tokens = torch.tensor([[0, 4000], [0, 8999], [0, 5]], dtype=torch.int32)
    parents = torch.tensor([-1, 0], dtype=torch.int32)
    for heat in (0.0, 1.0):
        for u in (0.0, 0.5, 1 - 2.0 ** -24):
            args = [logits, None, tokens, parents.expand(3, 2), torch.full((3, 2), 0.99), torch.full((3,), u), torch.full((3,), heat), [2, 2, 2]]
            got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), args[4].cuda(), args[5].cuda(), args[6].cuda())
            from zllm_b200 import ffi

            with pytest.raises(ffi.ZqFailure):  # the second sequence keeps its child, whose row has no finite logit
                ctx().sync()
            want = R.verify(*args)
            assert want[1] == ([0, 1], 2, -1)
            if heat == 0:
                assert want[0][2] == 17
            check_verify(got, want, 2)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("drawn", [False, True])
def test_rows_without_a_distribution_end_the_walk(bad, drawn):
    from zllm_b200 import ffi

    g = gen_of(2)
    logits, draft = torch.randn((2, 3, 5000), generator=g), torch.randn((2, 3, 5000), generator=g)
    (draft if drawn else logits)[0, 0, 4321] = bad
    tokens, parents = torch.zeros((2, 3), dtype=torch.int32), torch.tensor([[-1, 0, 0]] * 2, dtype=torch.int32)
    accept_u, sample_u, heat = torch.rand((2, 3), generator=g), torch.rand(2, generator=g), torch.ones(2)
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), accept_u.cuda(), sample_u.cuda(), heat.cuda(), draft_logits=draft.cuda() if drawn else None)
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    want = R.verify(logits, draft if drawn else None, tokens, parents, accept_u, sample_u, heat, [3, 3])
    assert want[0] == ([0], 1, -1)
    check_verify(got, want, 3)
    heat[1] = -1.0
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), accept_u.cuda(), sample_u.cuda(), heat.cuda())
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    assert int(got[2][1]) == -1


def test_a_token_out_of_range_is_not_tried():
    from zllm_b200 import ffi

    g = gen_of(12)
    logits = torch.randn((1, 4, 100), generator=g)
    tokens, parents = torch.tensor([[0, 100, -1, 7]], dtype=torch.int32), torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    logits[0, 0, 7] = 20.0
    one = torch.full((1, 4), 0.5)
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), one.cuda(), one[0, :1].cuda(), one[0, :1].cuda())
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    check_verify(got, R.verify(logits, None, tokens, parents.unsqueeze(0), one, one[0, :1], one[0, :1], [4]), 4)
    assert int(got[1]) == 2


def test_kept_tokens_are_distributed_as_the_target_draws_them():
    """200 000 draws of the first token, of nine: each share within five standard deviations of the target's."""
    g = gen_of(31)
    n, vocab = 200000, 9
    target, draft = torch.randn(vocab, generator=g), torch.randn(vocab, generator=g)
    p, q = torch.softmax(target.double(), 0), torch.softmax(draft.double(), 0)
    per = 50000
    counts = torch.zeros(vocab, dtype=torch.float64)
    for i in range(n // per):
        tokens = torch.multinomial(q, 3 * per, replacement=True, generator=g).reshape(per, 3).to(torch.int32)
        tokens[:, 0] = 0
        logits, near = target.expand(per, 3, vocab).contiguous(), draft.expand(per, 3, vocab).contiguous()
        path, accepted, token = ctx().verify_draft(logits.cuda(), tokens.cuda(), ints(-1, 0, 0), torch.rand((per, 3), generator=g).cuda(), torch.rand(per, generator=g).cuda(), torch.ones(per).cuda(), draft_logits=near.cuda())
        ctx().sync()
        first = torch.where(accepted.cpu() > 1, torch.gather(tokens, 1, path.cpu()[:, 1:2].clamp(min=0).long()).squeeze(1), token.cpu())
        counts += torch.bincount(first.long(), minlength=vocab)
    assert ((counts / n - p).abs() <= 5 * (p * (1 - p) / n).sqrt()).all()


# ---- the cache follows
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,layers,kv,dim,page", [(1, 1, 1, 1, 8, 16), (3, 9, 2, 2, 64, 4), (2, 40, 3, 8, 128, 32), (2, 200, 1, 1, 24, 1)])
def test_cache_rows_of_the_path_move_together(dtype, batch, rows, layers, kv, dim, page):
    g = gen_of(rows)
    blocks = -(-(30 + rows) // page)
    pages = batch * blocks + 2
    table = torch.randperm(pages, generator=g)[:batch * blocks].to(torch.int32).reshape(batch, blocks)
    k, v = (torch.randn((layers, pages, page, kv, dim), generator=g).to(dtype) for _ in range(2))
    context = torch.randint(0, 30, (batch,), generator=g, dtype=torch.int32)
    accepted = torch.randint(0, rows + 1, (batch,), generator=g, dtype=torch.int32)
    path = torch.full((batch, rows), -1, dtype=torch.int32)
    for b in range(batch):
        a = int(accepted[b])
        path[b, :a] = torch.randperm(rows, generator=g)[:a].sort().values
    got_k, got_v = k.cuda(), v.cuda()
    ctx().cache_keep_path(got_k, got_v, table.cuda(), context.cuda(), path.cuda(), accepted.cuda())
    ctx().sync()
    for b in range(batch):
        for i in range(int(accepted[b])):
            src, dst = R.cache_row(table[b], page, int(context[b]) + int(path[b, i])), R.cache_row(table[b], page, int(context[b]) + i)
            for pages_ in (k, v):
                pages_[:, dst[0], dst[1]] = pages_[:, src[0], src[1]].clone()
    assert torch.equal(got_k.cpu(), k) and torch.equal(got_v.cpu(), v)


def test_paths_that_lead_nowhere_are_skipped_and_reported():
    from zllm_b200 import ffi

    k = torch.arange(2 * 4 * 8, dtype=torch.float32).reshape(2, 4, 1, 8).half().cuda()
    v = k.clone()
    want = k.clone()
    table = ints(0, 1).reshape(1, 2)
    ctx().cache_keep_path(k, v, table, ints(3), ints(0, 3, 1, 5, 4).reshape(1, 5), ints(5))  # row 2 <- 1 would go back; 5 is no row; 4 stays
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    want[1, 0] = want[1, 2]
    assert torch.equal(k, want) and torch.equal(v, want)
    ctx().cache_keep_path(k, v, table, ints(3), ints(0, 3, -1, -1, -1).reshape(1, 5), ints(6))
    with pytest.raises(ffi.ZqFailure):
        ctx().sync()
    assert torch.equal(k, want)


# ---- streams, graphs, and all of it together
def step_inputs(g, batch, rows, kv, group, dim, vocab, dtype, contexts):
    blocks = -(-(max(contexts) + rows) // 16)
    k_pages, v_pages, table = make_cache(g, batch, kv, dim, 16, blocks, dtype)
    return dict(k_pages=k_pages, v_pages=v_pages, table=table, context=ints(*contexts), parents=R.trees(g, batch, rows).cuda(), drafted=ints(*[rows - (b % 2) for b in range(batch)]),
                q=torch.randn((batch, rows, kv * group, dim), generator=g).to(dtype).cuda(), k=torch.randn((batch, rows, kv, dim), generator=g).to(dtype).cuda(), v=torch.randn((batch, rows, kv, dim), generator=g).to(dtype).cuda(),
                freq=(10000.0 ** (-torch.arange(dim // 2) / (dim // 2))).float().cuda(), logits=(torch.randn((batch, rows, vocab), generator=g) * 2).to(dtype).cuda(),
                tokens=torch.randint(0, vocab, (batch, rows), generator=g, dtype=torch.int32).cuda(), accept_u=(torch.rand((batch, rows), generator=g) * 0.05).cuda(), sample_u=torch.rand(batch, generator=g).cuda(),
                heat=torch.ones(batch).cuda())


def step(c, s):
    positions, mask = c.draft_tree(s["parents"], s["context"], s["drafted"])
    q = c.rope_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["context"], positions.reshape(-1), s["freq"], draft_lens=s["drafted"])
    y = c.tree_attention(q, s["k_pages"], s["v_pages"], s["table"], s["context"], mask=mask, draft_lens=s["drafted"])
    path, accepted, token = c.verify_draft(s["logits"], s["tokens"], s["parents"], s["accept_u"], s["sample_u"], s["heat"], draft_lens=s["drafted"])
    c.cache_keep_path(s["k_pages"], s["v_pages"], s["table"], s["context"], path, accepted)
    return q, y, path, accepted, token, s["k_pages"], s["v_pages"]


SHAPES = [(1, 5, 2, 1, 64, 900), (3, 12, 2, 4, 128, 5000), (2, 70, 1, 8, 64, 300)]


def check_step(s, batch, rows, kv, group, dim, vocab, dtype):
    """Each operator against its 64-bit form on what the one before it left on the device; the rows that each sequence keeps."""
    before_k, before_v = s["k_pages"].clone(), s["v_pages"].clone()
    q, y, path, accepted, token, k_pages, v_pages = step(ctx(), s)
    ctx().sync()
    context, drafted, table = s["context"].cpu(), s["drafted"].cpu(), s["table"].cpu()
    positions, sees = R.tree(s["parents"].cpu(), context, drafted)
    turned = R.rotate(s["k"].reshape(-1, kv, dim).cpu(), positions.reshape(-1), s["freq"].cpu(), 1.0, False, False).reshape(batch, rows, kv, dim)
    for b in range(batch):
        for i in range(int(drafted[b])):
            at = R.cache_row(table[b], 16, int(context[b]) + i)
            before_k[at], before_v[at] = turned[b, i].to(dtype).cuda(), s["v"][b, i]
    want, bound = R.attention(q, before_k, before_v, s["table"], s["context"], sees, drafted, 1 / math.sqrt(dim))
    # a key of the cache may be rounded the other way than the plain form's: one step of a key's value, in every product
    moved = 2 * R.half_step(dtype) * float(before_k.abs().max()) * float(q.abs().max()) * math.sqrt(dim) * float(before_v.abs().max()) * 2.0 ** -4
    assert ((y.double() - want).abs() <= bound + moved).all()
    result = R.verify(s["logits"].cpu(), None, s["tokens"].cpu(), s["parents"].cpu(), s["accept_u"].cpu(), s["sample_u"].cpu(), s["heat"].cpu(), drafted)
    check_verify((path, accepted, token), result, rows)
    for b, (kept, n, _) in enumerate(result):
        for i in range(n):
            src, dst = R.cache_row(table[b], 16, int(context[b]) + kept[i]), R.cache_row(table[b], 16, int(context[b]) + i)
            before_k[dst], before_v[dst] = before_k[src].clone(), before_v[src].clone()
    assert torch.equal(v_pages, before_v)
    assert ((k_pages.double() - before_k.double()).abs() <= 2 * R.half_step(dtype) * before_k.double().abs() + 1e-6).all()
    return [kept for kept, _, _ in result]


@pytest.mark.parametrize("batch,rows,kv,group,dim,vocab", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_step_of_all_operators(batch, rows, kv, group, dim, vocab, dtype):
    s = step_inputs(gen_of(rows), batch, rows, kv, group, dim, vocab, dtype, [200 + 37 * b for b in range(batch)])
    check_step(s, batch, rows, kv, group, dim, vocab, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_step_that_keeps_rows(dtype):
    """The last child of every row drafts its row's likeliest token, and is kept at temperature 0."""
    batch, rows, kv, group, dim, vocab = 3, 20, 2, 4, 128, 700
    s = step_inputs(gen_of(77), batch, rows, kv, group, dim, vocab, dtype, [90, 31, 0])
    parents = s["parents"].clone()
    for b in range(batch):
        for i in range(rows):
            child = (parents[b] == i).nonzero().flatten().tolist()
            if child:
                s["tokens"][b, child[-1]] = int((s["logits"][b, i] == s["logits"][b, i].max()).nonzero()[0])
    s["heat"].zero_()
    kept = check_step(s, batch, rows, kv, group, dim, vocab, dtype)
    assert max(len(k) for k in kept) > 2 and any(k != list(range(len(k))) for k in kept)


def test_a_captured_step_replays_and_two_graphs_run_at_once():
    """Graphs captured on two streams, replayed at once and in turns with eager calls: each has scratch of its own."""
    from zllm_b200.backend import B200Context

    c = B200Context(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = [[step_inputs(gen_of(40 + i), *shape[:6], torch.float16, [3000 + 700 * b for b in range(shape[0])]) for shape in SHAPES[1:]] for i in range(2)]
    torch.cuda.synchronize()
    keep = ("k_pages", "v_pages")
    first = [[{n: s[n].clone() for n in keep} for s in m] for m in made]

    def restore(i):
        for s, f in zip(made[i], first[i]):
            for n in keep:
                s[n].copy_(f[n])

    want = []
    for i in range(2):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        want.append([[t.clone() for t in step(c, s)] for s in made[i]])
        c.sync()
        restore(i)
    graphs, outs = [], []
    for i in range(2):
        c.set_stream(streams[i].cuda_stream)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[i]):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=streams[i]):
                outs.append([step(c, s) for s in made[i]])
            graphs.append(g)
    for _ in range(20):
        torch.cuda.synchronize()
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                restore(i)
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            for got, w in zip(outs[i], want[i]):
                assert all(torch.equal(x, y) for x, y in zip(got, w))
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    restore(0)
    again = [step(c, s) for s in made[0]]
    c.sync()
    assert all(torch.equal(x, y) for got, w in zip(again, want[0]) for x, y in zip(got, w))
    torch.cuda.synchronize()
    del graphs, outs


def test_calls_on_two_streams_at_once():
    from zllm_b200.backend import B200Context

    c = B200Context(0)
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = [step_inputs(gen_of(60 + i), 4, 20, 2, 4, 64, 2000, torch.bfloat16, [2000, 3000, 10, 0]) for i in range(2)]
    torch.cuda.synchronize()
    want = []
    for s in made:
        q, mask = s["q"], c.draft_tree(s["parents"], s["context"], s["drafted"])[1]
        want.append(c.tree_attention(q, s["k_pages"], s["v_pages"], s["table"], s["context"], mask=mask, draft_lens=s["drafted"]))
        c.sync()
    for _ in range(30):
        got = []
        for i, s in enumerate(made):
            c.set_stream(streams[i].cuda_stream)
            with torch.cuda.stream(streams[i]):
                mask = c.draft_tree(s["parents"], s["context"], s["drafted"])[1]
                got.append(c.tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["context"], mask=mask, draft_lens=s["drafted"]))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    c.sync()


def test_operators_between_projections_of_the_framework():
    """Two tokens of a small layer: q, k and v from packed weights, rotated into the cache, attended to, and through the output projection."""
    import numpy as np

    from tests import helpers as H
    from zllm_b200.backend import rope_frequencies

    hidden, kv, dim, heads = 256, 2, 64, 4
    w = {n: ctx().prepare_weight(H.Q8_0, H.random_weight(H.Q8_0, rows, hidden, seed=i), rows, hidden) for i, (n, rows) in enumerate((("q", heads * dim), ("k", kv * dim), ("v", kv * dim), ("o", hidden)))}
    deq = {n: ctx().dequantize(v).double() for n, v in w.items()}
    x = torch.from_numpy(np.random.default_rng(3).standard_normal((2, hidden)).astype(np.float32)).cuda().half()
    k_pages, v_pages = torch.zeros((4, 16, kv, dim), dtype=torch.float16, device="cuda"), torch.zeros((4, 16, kv, dim), dtype=torch.float16, device="cuda")
    table, freq = ints(2, 0).reshape(1, 2), rope_frequencies(dim, 10000.0, device="cuda")[0]
    for position in range(2):
        q, k, v = ctx().triple_linear(x[position:position + 1], w["q"], w["k"], w["v"])
        q = ctx().rope_append(q.view(1, 1, heads, dim), k.view(1, 1, kv, dim), v.view(1, 1, kv, dim), k_pages, v_pages, table, ints(position), ints(position), freq)
        y = ctx().linear(ctx().tree_attention(q, k_pages, v_pages, table, ints(position)).reshape(1, heads * dim), w["o"])
    ctx().sync()
    rows = x.double()
    q, k, v = (rows @ deq[n].T for n in ("q", "k", "v"))
    angle = torch.arange(2, device="cuda").double().reshape(-1, 1, 1) * freq.double()

    def turn(t):
        a, b = t[..., :dim // 2], t[..., dim // 2:]
        return torch.cat([a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()], -1)

    q, k, v = turn(q.view(2, heads, dim)), turn(k.view(2, kv, dim)), v.view(2, kv, dim)
    p = torch.softmax(torch.einsum("hd,khd->hk", q[1], k.repeat_interleave(heads // kv, 1)) / 8, 1)
    want = torch.einsum("hk,khd->hd", p, v.repeat_interleave(heads // kv, 1)).reshape(1, -1) @ deq["o"].T
    # f16 rows between five steps, each product within 3e-4 of its largest value by its integer activations and 2^-11 by rounding
    assert (y.double() - want).abs().max() <= 5 * (3e-4 + 2.0 ** -11) * 4 * want.abs().max()
