"""Operators on drafted tokens at calls that are allowed and rare: expanded and padded tensors, the largest shapes, random numbers next to a border, values next to the types' ends."""
import math

import pytest
import torch

from tests import draft_ref as R
from tests.gpu_util import ctx
from tests.test_gpu_draft import check_verify, gen_of, ints, make_cache, run_attention

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


# ---- verification
def test_verification_of_the_largest_vocabulary_by_many_sequences():
    """Many sequences have few CTAs each, and these have the sums of a long run of the vocabulary in shared memory."""
    batch, vocab = 300, 1 << 22
    logits = torch.zeros((1, 1, vocab), dtype=torch.float16, device="cuda").repeat(batch, 1, 1)
    g = gen_of(6)
    at = torch.randint(0, vocab, (batch,), generator=g)
    at[:4] = torch.tensor([0, vocab - 1, vocab // 2, vocab // 2 - 1])
    logits[torch.arange(batch), 0, at.cuda()] = 40.0  # e^40 times as likely as each other one, 5.6e10 times as all of them
    u, heat, parents = torch.rand(batch, generator=g), torch.ones(batch), torch.full((1,), -1, dtype=torch.int32)
    u[:] = 0.25 + 0.5 * u
    heat[::3] = 0.0
    for device_heat in (heat, torch.ones(batch) * 1e30):
        path, accepted, token = ctx().verify_draft(logits, torch.zeros((batch, 1), dtype=torch.int32).cuda(), parents.cuda(), torch.zeros((batch, 1)).cuda(), u.cuda(), device_heat.cuda())
        ctx().sync()
        assert (path == 0).all() and (accepted == 1).all()
        if device_heat is heat:
            assert torch.equal(token.cpu().long(), at)
        else:  # all tokens as likely to 1e-28: the first whose number of tokens up to it exceeds u vocab, but where the two are within the sums' 1e-9 of each other
            want = torch.floor(u.double() * vocab)
            clear = (u.double() * vocab - want - 0.5).abs() < 0.49
            assert clear.sum() > batch // 2 and torch.equal(token.cpu().double()[clear], want[clear])


def test_two_threads_verify_vocabularies_of_unlike_sizes():
    """Contexts of two threads, on streams of their own: what one launch asks for must not be taken from the other's."""
    import threading

    from zllm_b200.backend import B200Context

    batch = 300
    done, made = {}, {}
    for name, vocab in (("small", 1000), ("large", 1 << 17)):
        logits = torch.zeros((batch, 1, vocab), dtype=torch.bfloat16, device="cuda")
        logits[:, 0, vocab - 2] = 60.0
        made[name] = (logits, torch.zeros((batch, 1), dtype=torch.int32).cuda(), ints(-1), torch.zeros((batch, 1)).cuda(), torch.full((batch,), 0.5).cuda(), torch.ones(batch).cuda())
    torch.cuda.synchronize()

    def work(name):
        try:
            stream = torch.cuda.Stream()
            c = B200Context(0)
            c.set_stream(stream.cuda_stream)
            with torch.cuda.stream(stream):
                got = [c.verify_draft(*made[name])[2] for _ in range(200)]
            c.sync()
            done[name] = all((t == made[name][0].shape[2] - 2).all().item() for t in got)
            c.close()
        except Exception as e:  # reported by the assertion below
            done[name] = repr(e)

    threads = [threading.Thread(target=work, args=(n,)) for n in made]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert done == {"small": True, "large": True}


def verified(logits, draft, tokens, parents, accept_u, sample_u, heat):
    """Of one sequence for each row of `tokens`, against the definition; the paths and tokens."""
    batch, rows = tokens.shape
    got = ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), accept_u.cuda(), sample_u.cuda(), heat.cuda(), draft_logits=draft.cuda() if draft is not None else None)
    ctx().sync()
    want = R.verify(logits, draft, tokens, parents.expand(batch, -1), accept_u, sample_u, heat, [rows] * batch)
    check_verify(got, want, rows)
    return want


LAST = 1 - 2.0 ** -24  # the largest random number


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.1, 1.0, 4.0, 12.0])
@pytest.mark.parametrize("vocab", [2, 7, 33, 4099])
def test_children_that_hold_all_that_is_likely(dtype, spread, vocab):
    """The children of the root are all tokens of finite logit: with the largest random numbers every child but the last is rejected, and the last one has all of p."""
    g = gen_of(vocab)
    batch, rows = 40, 8
    few = min(rows - 1, vocab)
    logits = torch.full((batch, rows, vocab), -math.inf, dtype=dtype)
    tokens = torch.zeros((batch, rows), dtype=torch.int32)
    for b in range(batch):
        some = torch.randperm(vocab, generator=g)[:few]
        logits[b, :, some] = (torch.randn((rows, few), generator=g) * spread).to(dtype)
        tokens[b, 1:1 + few] = some[torch.randperm(few, generator=g)].to(torch.int32)
        tokens[b, 1 + few:] = some[0]
    parents = torch.tensor([-1] + [0] * (rows - 1), dtype=torch.int32)
    accept_u, sample_u, heat = torch.full((batch, rows), LAST), torch.rand(batch, generator=g), torch.ones(batch)
    sample_u[::2] = LAST
    want = verified(logits, None, tokens, parents, accept_u, sample_u, heat)
    assert all(n == 2 for _, n, _ in want)
    # as many children but one: what is left is the token that is no child's
    if few > 1:
        tokens[:, few:] = tokens[:, 1:2]
        want = verified(logits, None, tokens, parents, accept_u, sample_u, heat)
        assert spread > 4 or any(n == 1 for _, n, _ in want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_random_numbers_next_to_a_childs_border(dtype):
    """The f32 number in front of p(t) / (1 - what is gone), and the one behind it: one child is kept, the other is not."""
    g = gen_of(17)
    batch, vocab = 64, 3001
    logits = (torch.randn((batch, 1, vocab), generator=g) * 2).to(dtype).expand(batch, 4, vocab).contiguous()
    tokens = torch.zeros((batch, 4), dtype=torch.int32)
    accept_u = torch.full((batch, 4), 0.999)
    for b in range(batch):
        p = torch.softmax(logits[b, 0].double(), 0)
        top = p.topk(3).indices
        tokens[b, 1:] = top.to(torch.int32)
        border = float(p[top[1]] / (1 - p[top[0]]))
        at = torch.tensor(border, dtype=torch.float32)
        lower, upper = (at, torch.nextafter(at, torch.tensor(2.0))) if float(at) < border else (torch.nextafter(at, torch.tensor(-1.0)), at)
        accept_u[b, 2] = lower if b % 2 else upper
    parents = torch.tensor([-1, 0, 0, 0], dtype=torch.int32)
    want = verified(logits, None, tokens, parents, accept_u, torch.rand(batch, generator=g), torch.ones(batch))
    assert [w[0][1] if w[1] > 1 else 0 for w in want] == [2 if b % 2 else 0 for b in range(batch)]


@pytest.mark.parametrize("near", [1e-2, 1e-4, 1e-6])
@pytest.mark.parametrize("vocab", [50, 1003, 40000])
def test_drafts_near_the_target(near, vocab):
    """Draft and target differ by so little that a rejection leaves less than f32 sums tell apart; several children are rejected."""
    g = gen_of(vocab + 1)
    batch, rows = 24, 7
    logits = torch.randn((batch, rows, vocab), generator=g) * 2
    draft = logits + torch.randn((batch, rows, vocab), generator=g) * near
    tokens = torch.stack([torch.multinomial(torch.softmax(draft[b, 0], 0), rows, replacement=True, generator=g) for b in range(batch)]).to(torch.int32)
    parents = torch.tensor([-1] + [0] * (rows - 1), dtype=torch.int32)
    accept_u = torch.full((batch, rows), LAST)
    accept_u[::3] = 1 - 2.0 ** -10 * torch.rand((len(accept_u[::3]), rows), generator=g)
    want = verified(logits, draft, tokens, parents, accept_u, torch.rand(batch, generator=g), torch.ones(batch))
    assert any(n == 1 for _, n, _ in want) and any(n > 1 for _, n, _ in want)


def test_drafts_that_are_the_target():
    """Every drawn child is kept; with random numbers that are none (1 and above) all are rejected, nothing is left, and p stays as it was."""
    g = gen_of(23)
    batch, rows, vocab = 6, 5, 5003
    logits = torch.randn((batch, rows, vocab), generator=g).half()
    tokens = torch.randint(0, vocab, (batch, rows), generator=g, dtype=torch.int32)
    parents = torch.tensor([-1, 0, 1, 2, 3], dtype=torch.int32)
    accept_u, sample_u, heat = torch.full((batch, rows), LAST), torch.rand(batch, generator=g), torch.ones(batch)
    want = verified(logits, logits.clone(), tokens, parents, accept_u, sample_u, heat)
    assert all(n == rows for _, n, _ in want)
    want = verified(logits, logits.clone(), tokens, parents, torch.full((batch, rows), 1.5), sample_u, heat)
    assert all(n == 1 and t is not None for _, n, t in want)


@pytest.mark.parametrize("drawn", [False, True])
@pytest.mark.parametrize("row,parent", [(0, 0), (1, -2), (3, 3), (3, 7), (2, 2 ** 31 - 1), (4, -2 ** 31)])
def test_parents_out_of_range_are_reported_by_verification(drawn, row, parent):
    from zllm_b200 import ffi

    g = gen_of(29)
    logits, draft = torch.randn((3, 6, 700), generator=g), torch.randn((3, 6, 700), generator=g)
    parents = R.trees(g, 3, 6)
    tokens, accept_u, sample_u = torch.randint(0, 700, (3, 6), generator=g, dtype=torch.int32), torch.rand((3, 6), generator=g) * 0.01, torch.rand(3, generator=g)

    def run(lens):
        return ctx().verify_draft(logits.cuda(), tokens.cuda(), parents.cuda(), accept_u.cuda(), sample_u.cuda(), torch.ones(3).cuda(), draft_logits=draft.cuda() if drawn else None, draft_lens=ints(*lens))

    parents[1, row] = parent
    got = run([6, 6, 6])
    with pytest.raises(ffi.ZqFailure) as e:
        ctx().sync()
    assert e.value.code == 5
    check_verify(got, R.verify(logits, draft if drawn else None, tokens, parents, accept_u, sample_u, torch.ones(3), [6, 6, 6]), 6)
    got = run([6, row, 6])  # a row of padding is not looked at
    ctx().sync()
    check_verify(got, R.verify(logits, draft if drawn else None, tokens, parents, accept_u, sample_u, torch.ones(3), [6, row, 6]), 6)


# ---- caches
def odd_strides(t, dims):
    """The same values, with another stride in each of `dims`, which are of size 1."""
    return t.as_strided(t.shape, [999 if i in dims else s for i, s in enumerate(t.stride())])


@pytest.mark.parametrize("pages,page,kv,layers", [(1, 8, 2, 1), (3, 1, 2, 1), (3, 8, 1, 1), (1, 1, 1, 1), (1, 8, 1, 3), (4, 8, 2, 1)])
def test_strides_of_dimensions_of_one_mean_nothing(pages, page, kv, layers):
    g = gen_of(31)
    k, v = (torch.randn((layers, pages, page, kv, 16), generator=g).half().cuda() for _ in range(2))
    ones = [i for i in range(5) if k.shape[i] == 1]
    table, context = torch.arange(pages, dtype=torch.int32).reshape(1, pages).cuda(), ints(0)
    q = torch.randn((1, 1, 2 * kv, 16), generator=g).half().cuda()
    odd, inner = odd_strides(v, ones), [i - 1 for i in ones if i > 0]
    got = ctx().tree_attention(q, k[0], odd_strides(v[0], inner), table, context)
    want = ctx().tree_attention(q, k[0], v[0], table, context)
    ctx().sync()
    assert torch.equal(got, want)
    if pages * page > 2:
        want_k, want_v = k.clone(), v.clone()
        want_k.view(layers, -1, kv, 16)[:, 1], want_v.view(layers, -1, kv, 16)[:, 1] = k.view(layers, -1, kv, 16)[:, 2], v.view(layers, -1, kv, 16)[:, 2]
        ctx().cache_keep_path(k, odd, table, context, ints(0, 2, -1).reshape(1, 3), ints(2))
        ctx().sync()
        assert torch.equal(k, want_k) and torch.equal(v, want_v)


def test_caches_of_unlike_strides_are_refused():
    from zllm_b200 import ffi

    k = torch.zeros((4, 8, 2, 16), dtype=torch.float16, device="cuda")
    v = torch.zeros((8, 8, 2, 16), dtype=torch.float16, device="cuda")[::2]
    with pytest.raises(ffi.ZqFailure) as e:
        ctx().tree_attention(torch.zeros((1, 1, 2, 16), dtype=torch.float16, device="cuda"), k, v, ints(0).reshape(1, 1), ints(0))
    assert e.value.code == 1


# ---- attention
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,group,dim", [(12, 4, 64), (20, 2, 128), (40, 4, 64), (70, 4, 128), (66, 4, 72)])
def test_several_visible_infinities_of_a_tile(dtype, rows, group, dim):
    """A chain whose drafted keys hold an infinity each, in a column of their own: a row has those of all rows up to itself, in 16-row, 128-row and 256-row tiles."""
    g = gen_of(37)
    k_pages, v_pages, table = make_cache(g, 1, 2, dim, 16, 8, dtype)
    q = torch.randn((1, rows, 2 * group, dim), generator=g).to(dtype).cuda()
    context, bad = 19, {2: (7, math.inf), 3: (30, -math.inf), 4: (7, math.inf), 5: (31, math.inf), 9: (0, -math.inf), 10: (dim - 1, math.inf)}
    for i, (column, value) in bad.items():
        b, o = R.cache_row(table[0].cpu(), 16, context + i)
        v_pages[b, o, :, column] = value
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(context))
    ctx().sync()
    want = torch.zeros((rows, dim))
    for i, (column, value) in bad.items():
        want[i:, column] = value
    want = want.cuda().reshape(1, rows, 1, dim).expand_as(got)
    assert torch.equal(torch.where(torch.isfinite(got), 0.0, got.float()), want)


@pytest.mark.parametrize("rows,group,dim,page", [(66, 4, 64, 16), (66, 4, 128, 16), (70, 8, 72, 32), (40, 2, 104, 8), (6, 1, 72, 16), (20, 4, 128, 128)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("poison", [math.nan, math.inf, -math.inf])
def test_what_rows_of_large_tiles_do_not_see_does_not_reach_them(dtype, rows, group, dim, page, poison):
    """Masked drafted rows, rows of padding, the ends of pages and pages of nobody hold infinities and NaN; three rows see one each, of which two are neighbours in a tile."""
    g = gen_of(41)
    kv, context = 2, 101
    k_pages, v_pages, table = make_cache(g, 1, kv, dim, page, -(-(context + rows) // page) + 1, dtype)
    q = torch.randn((1, rows, group * kv, dim), generator=g).to(dtype).cuda()
    parents, n = torch.tensor([[-1] + [0] * (rows - 1)], dtype=torch.int32), rows - 1
    _, sees = R.tree(parents, [context], [n])
    mask = R.words(sees).cuda()
    clean = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask, draft_lens=ints(n))
    hit = sorted({2, 3, n - 1})
    for pages in (k_pages, v_pages):
        flat = pages.view(-1, kv, dim)
        used = torch.zeros(flat.shape[0], dtype=torch.bool)
        for p in range(context + n):
            b, o = R.cache_row(table[0].cpu(), page, p)
            used[b * page + o] = True
        flat[~used.cuda()] = poison
        for i in hit:
            b, o = R.cache_row(table[0].cpu(), page, context + i)
            pages[b, o] = poison
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask, draft_lens=ints(n))
    ctx().sync()
    others = [i for i in range(rows) if i not in hit]
    assert torch.equal(got[:, others], clean[:, others]) and torch.isfinite(got[:, others]).all()
    assert not torch.isfinite(got[:, hit]).any()
    assert (got[:, n:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [72, 88, 104, 112, 120])
@pytest.mark.parametrize("rows,group", [(9, 4), (40, 2), (70, 4)])
def test_attention_of_heads_between_the_tiles_sizes(dtype, dim, rows, group):
    run_attention(gen_of(dim + rows), 2, rows, 2 * group, 2, dim, 16, [37, 300], dtype, tree=True, drafted=[rows, rows - 3])


@pytest.mark.parametrize("rows,group,dim", [(3, 2, 64), (12, 4, 128), (40, 2, 64), (70, 4, 128), (9, 8, 192)])
@pytest.mark.parametrize("context", [0, 127, 128, 300])
def test_a_row_whose_only_visible_score_is_none(rows, group, dim, context):
    """The last row sees itself alone among the drafted rows, in a share of the keys of which it sees no other, and that score is a NaN: so is the row."""
    g = gen_of(43)
    k_pages, v_pages, table = make_cache(g, 1, 1, dim, 16, -(-(context + rows) // 16), torch.bfloat16)
    q = torch.randn((1, rows, group, dim), generator=g).bfloat16().cuda()
    mask = torch.zeros((1, rows, -(-rows // 64)), dtype=torch.int64)
    for i in range(rows):
        mask[0, i, i // 64] = (1 << (i % 64)) - ((1 << 64) if i % 64 == 63 else 0)
    clean = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask.cuda())
    b, o = R.cache_row(table[0].cpu(), 16, context + rows - 1)
    k_pages[b, o, 0, 5] = math.nan
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(context), mask=mask.cuda())
    ctx().sync()
    assert torch.isnan(got[0, -1]).all() and torch.equal(got[0, :-1], clean[0, :-1])


# few sequences: a row's keys are cut into parts, each relative to its own largest weight; many: they lie in one
@pytest.mark.parametrize("batch", [1, 300])
@pytest.mark.parametrize("rows,group,dim,n", [(1, 1, 64, 100000), (1, 8, 128, 70001), (9, 4, 64, 20000), (66, 4, 128, 10000), (3, 2, 192, 10000), (1, 4, 64, 900), (40, 1, 64, 3000)])
@pytest.mark.parametrize("first", [True, False])
def test_many_small_weights_in_f16(batch, rows, group, dim, n, first):
    """One key with a weight of 1 and a value of 0, and n that are alike: weights of 2^-26 and values of 1. Their share is sum / (1 + sum), which f16's smallest step must not take away."""
    page = 64
    pages = -(-(n + 1 + rows) // page)
    k_pages, v_pages = torch.zeros((pages, page, 1, dim), dtype=torch.float16, device="cuda"), torch.ones((pages, page, 1, dim), dtype=torch.float16, device="cuda")
    score = -18.03125  # exp: 1.478e-8, 2^-26.01
    k_pages[:, :, 0, 0] = score
    at = 0 if first else n
    k_pages[at // page, at % page, 0, 0], v_pages[at // page, at % page] = 0.0, 0.0
    q = torch.zeros((batch, rows, group, dim), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    mask = torch.zeros((batch, rows, -(-rows // 64)), dtype=torch.int64, device="cuda")  # the context alone: n + 1 keys
    table = torch.arange(pages, dtype=torch.int32).cuda().reshape(1, pages).expand(batch, pages)  # of the same pages for all
    got = ctx().tree_attention(q, k_pages, v_pages, table, ints(*[n + 1] * batch), mask=mask, scale=1.0)
    ctx().sync()
    total = n * math.exp(score)
    want = total / (1 + total)
    # weights come 2^7 times as large at least, so that each is off by half of f16's smallest step, 2^-25, over 2^7; the result is rounded once, below f16's normal range by 2^-25; a
    # score has one product, and two roundings of 2^-24 of its 26 on the way to an exponential of 2^-22, in each weight alike
    bound = n * 2.0 ** -32 + want * (2.0 ** -11 + 2 * 26.02 * 2.0 ** -24 + 2.0 ** -21) + 2.0 ** -25
    assert float((got.double() - want).abs().max()) <= bound < want / 2
