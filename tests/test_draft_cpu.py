"""Operators on drafted tokens without a device: frequencies of the rotary embedding, and what is refused before anything is launched."""
import ctypes as C
import math

import pytest
import torch

from zllm_b200 import ffi
from zllm_b200.backend import rope_frequencies


def yarn(half, base, factor, context, slow, fast):
    out = []
    for i in range(half):
        f = base ** (-i / half)
        keep = min(1.0, max(0.0, (context * f / (2 * math.pi) - slow) / (fast - slow)))
        out.append(f * keep + f / factor * (1 - keep))
    return out


def test_frequencies_plain_linear_and_yarn():
    for rotary in (2, 64, 80, 128):
        half = rotary // 2
        plain, one = rope_frequencies(rotary, 10000.0)
        assert one == 1.0 and torch.equal(plain, torch.tensor([10000.0 ** (-i / half) for i in range(half)]))
        linear, one = rope_frequencies(rotary, 10000.0, ffi.ROPE_SCALE_LINEAR, factor=4.0)
        assert one == 1.0 and torch.equal(linear, torch.tensor([10000.0 ** (-i / half) / 4.0 for i in range(half)]))
        long, by = rope_frequencies(rotary, 500000.0, ffi.ROPE_SCALE_YARN, factor=8.0, original_context=8192)
        assert torch.allclose(long, torch.tensor(yarn(half, 500000.0, 8.0, 8192, 1, 32)), rtol=2.0 ** -23, atol=0)  # both sides round once from f64
        assert by == pytest.approx(0.1 * math.log(8.0) + 1, rel=2.0 ** -23)
    assert rope_frequencies(64, 10000.0, ffi.ROPE_SCALE_YARN, factor=0.5, original_context=100)[1] == 1.0


def test_frequencies_with_pair_factors():
    factors = [1.0, 2.0, 0.5, 8.0]
    got, _ = rope_frequencies(8, 100.0, pair_factors=factors)
    assert torch.equal(got, torch.tensor([100.0 ** (-i / 4) / f for i, f in enumerate(factors)]))
    with pytest.raises(ffi.ZqFailure):
        rope_frequencies(8, 100.0, pair_factors=[1.0, 0.0, 1.0, 1.0])
    with pytest.raises(ffi.ZqFailure):
        rope_frequencies(8, 100.0, pair_factors=[1.0])


@pytest.mark.parametrize("kwargs", [dict(rotary_dim=7), dict(rotary_dim=0), dict(base=0.0), dict(base=math.inf), dict(scaling=9), dict(scaling=ffi.ROPE_SCALE_LINEAR, factor=0.0), dict(scaling=ffi.ROPE_SCALE_LINEAR, factor=math.nan),
                                    dict(scaling=ffi.ROPE_SCALE_YARN, factor=2.0), dict(scaling=ffi.ROPE_SCALE_YARN, factor=2.0, original_context=100, beta_slow=32, beta_fast=32)])
def test_frequencies_that_are_refused(kwargs):
    with pytest.raises(ffi.ZqFailure):
        rope_frequencies(**{"rotary_dim": 64, **kwargs})


# Every refusal comes before the context is looked at, so a block of zeros stands for one.
FAKE = C.create_string_buffer(4096)
ADDRESS = C.addressof(FAKE) & ~15
P = C.c_void_p(ADDRESS + 16)


def cache(**changes):
    fields = dict(dev_k=P.value, dev_v=P.value, dtype=ffi.F16, pages=4, page_size=16, heads=2, head_dim=64, page_stride=16 * 2 * 64, layers=1, layer_stride=0, dev_blocks=P.value, batch=2, max_blocks=2, dev_context_lens=P.value)
    return ffi.ZqKvCache(**{**fields, **changes})


BAD_CACHES = [dict(dev_k=None), dict(dev_v=None), dict(dev_blocks=None), dict(dev_context_lens=None), dict(dtype=ffi.F32), dict(page_size=0), dict(page_size=24), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264, page_stride=1 << 20), dict(heads=0),
              dict(batch=0), dict(batch=65536), dict(pages=0), dict(max_blocks=0), dict(page_stride=16 * 2 * 64 - 8), dict(page_stride=16 * 2 * 64 + 4), dict(dev_k=P.value + 2)]


def attention(c, q_heads=4, q_stride=256, rows=3, mask=None, scale=0.125, q=P, out=P):
    ffi.call("zq_tree_attention", P, q, q_heads, q_stride, rows, C.byref(c), mask, None, scale, out)


def append(c, q_stride=256, k_stride=128, v_stride=128, rows=3, rotary=64, layout=0, placement=0, factor=1.0, k=P):
    ffi.call("zq_rope_append", P, P, 4, q_stride, k, k_stride, P, v_stride, rows, C.byref(c), None, rotary, layout, placement, P, P, factor, P)


def keep(c, rows=3, path=P):
    ffi.call("zq_cache_keep_path", P, C.byref(c), path, rows, P)


@pytest.mark.parametrize("call", [attention, append, keep])
@pytest.mark.parametrize("changes", BAD_CACHES)
def test_caches_that_are_refused(call, changes):
    with pytest.raises(ffi.ZqFailure) as e:
        call(cache(**changes))
    assert e.value.code in (1, 2, 4)


@pytest.mark.parametrize("kwargs", [dict(q_heads=0), dict(q_heads=3), dict(q_stride=255), dict(q_stride=257), dict(rows=0), dict(rows=1025), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
                                    dict(mask=C.c_void_p(P.value + 4)), dict(q=None), dict(out=None), dict(q=C.c_void_p(P.value + 2))])
def test_attention_that_is_refused(kwargs):
    with pytest.raises(ffi.ZqFailure):
        attention(cache(), **kwargs)


def test_attention_over_more_positions_than_an_int_counts_is_refused():
    with pytest.raises(ffi.ZqFailure):
        attention(cache(max_blocks=1 << 28))


@pytest.mark.parametrize("kwargs", [dict(q_stride=255), dict(k_stride=127), dict(v_stride=64), dict(rows=0), dict(rotary=0), dict(rotary=63), dict(rotary=66), dict(layout=2), dict(placement=-1), dict(factor=math.nan), dict(k=None)])
def test_appending_that_is_refused(kwargs):
    with pytest.raises(ffi.ZqFailure):
        append(cache(), **kwargs)


@pytest.mark.parametrize("kwargs", [dict(rows=0), dict(rows=1025), dict(path=None)])
def test_paths_that_are_refused(kwargs):
    with pytest.raises(ffi.ZqFailure):
        keep(cache(), **kwargs)
    with pytest.raises(ffi.ZqFailure):
        keep(cache(layers=0))
    with pytest.raises(ffi.ZqFailure):
        keep(cache(layers=2, layer_stride=4))


def rope(q_heads=4, q_stride=256, k=P, k_heads=2, k_stride=128, dtype=ffi.F32, rows=3, head_dim=64, rotary=64, layout=0, placement=0, factor=1.0, q_out=P, k_out=P, positions=P):
    ffi.call("zq_rope_rows", P, P, q_heads, q_stride, k, k_heads, k_stride, dtype, rows, head_dim, rotary, layout, placement, positions, P, factor, 0, q_out, k_out)


@pytest.mark.parametrize("kwargs", [dict(q_heads=0), dict(q_stride=200), dict(k_stride=100), dict(dtype=3), dict(rows=0), dict(head_dim=0), dict(head_dim=514, q_stride=4096, k_stride=4096), dict(rotary=65), dict(rotary=66), dict(layout=5), dict(placement=2),
                                    dict(factor=math.inf), dict(q_out=None), dict(k_out=None), dict(k_heads=0), dict(positions=None), dict(q_stride=264), dict(q_heads=1 << 16, q_stride=1 << 22)])
def test_rotations_that_are_refused(kwargs):
    with pytest.raises(ffi.ZqFailure):  # q_stride=264: in place, but not dense
        rope(**kwargs)


@pytest.mark.parametrize("batch,rows", [(0, 1), (65536, 1), (1, 0), (1, 1025)])
def test_trees_that_are_refused(batch, rows):
    with pytest.raises(ffi.ZqFailure):
        ffi.call("zq_draft_tree", P, P, 0, batch, rows, P, None, P, P)
    with pytest.raises(ffi.ZqFailure):
        ffi.call("zq_draft_tree", P, None, 0, 1, 1, P, None, P, P)


@pytest.mark.parametrize("kwargs", [dict(dtype=7), dict(batch=0), dict(batch=65536), dict(rows=0), dict(rows=1025), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(logits=C.c_void_p(P.value + 1)), dict(logits=None)])
def test_verification_that_is_refused(kwargs):
    a = {**dict(logits=P, dtype=ffi.BF16, batch=1, rows=1, vocab=10), **kwargs}
    with pytest.raises(ffi.ZqFailure):
        ffi.call("zq_verify_draft", P, a["logits"], None, a["dtype"], a["batch"], a["rows"], a["vocab"], P, P, 0, P, P, P, None, P, P, P)


def test_null_contexts_are_refused():
    none = C.c_void_p()
    for name, args in (("zq_draft_tree", (none, P, 0, 1, 1, P, None, P, P)), ("zq_tree_attention", (none, P, 4, 256, 1, C.byref(cache()), None, None, 0.1, P)), ("zq_cache_keep_path", (none, C.byref(cache()), P, 1, P)),
                       ("zq_rope_rows", (none, P, 1, 64, None, 0, 0, 0, 1, 64, 64, 0, 0, P, P, 1.0, 0, P, None)), ("zq_verify_draft", (none, P, None, 0, 1, 1, 1, P, P, 0, P, P, P, None, P, P, P))):
        with pytest.raises(ffi.ZqFailure) as e:
            ffi.call(name, *args)
        assert e.value.code == 4


def test_tensors_of_another_device_are_refused():
    native, i, f = ffi.native(), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    rows, pages, table = torch.zeros((2, 2, 1, 8), dtype=torch.float16), torch.zeros((2, 4, 1, 8), dtype=torch.float16), torch.zeros((2, 2), dtype=torch.int32)
    for name, args in (("draft_tree", (i, i, None)), ("rope_rows", (rows, None, i, f, False, False, 1.0, False)), ("rope_append", (rows, rows, rows, pages, pages, table, i, i, f, None, False, False, 1.0)),
                       ("tree_attention", (rows, pages, pages, table, i, None, None, None)), ("verify_draft", (rows, i, i, f, f, f, None, None)), ("cache_keep_path", (pages, pages, table, i, table, i))):
        with pytest.raises(ffi.ZqFailure) as e:
            getattr(native, name)(0, 0, *args)
        assert e.value.code == 4 and "device" in e.value.message
        with pytest.raises(TypeError):
            getattr(native, name)(0, 0, *args, None)  # one argument too many
        with pytest.raises(TypeError):
            getattr(native, name)(0, 0, *[None] * len(args))
