"""Attention (q4b_attention) at the ends of what its arguments may be."""
import math

import numpy as np
import pytest

from cache_cases import Batch, attention_reference, narrow, widen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


@pytest.mark.parametrize("scale", [3e38, -3e38, 2.4e38])
def test_scales_that_overflow_are_refused(q4b, ctx, scale):
    """Scores are counted in powers of two: scale x log2(e) has to be a number, or 0 x scale would be none."""
    rng = np.random.default_rng(1)
    for counts in ([1], [40]):
        batch = Batch(rng, counts, [50], 16, 1, 64, "f16")
        cache, described = batch.upload(q4b, ctx)
        d_q, d_out = ctx.to_device(np.zeros((batch.tokens, 2, 64), np.float16)), ctx.alloc(batch.tokens * 256)
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.attention(cache, described, d_q.ptr, 2, d_out.ptr, scale)
        assert refused.value.status == 1 and "scale" in refused.value.message
        # the largest that there is: queries of zeros see all keys alike
        ctx.attention(cache, described, d_q.ptr, 2, d_out.ptr, math.copysign(2.3e38, scale))
        got = widen(d_out.download(np.float16, (batch.tokens, 2, 64)), "f16")
        want, tolerance = attention_reference(batch, np.zeros((batch.tokens, 2, 64), np.float16), 2, 0.0, 0, 0)
        assert (np.abs(got - want) <= tolerance).all()


@pytest.mark.parametrize("head,group,counts,lengths,window,sinks", [(64, 4, [1, 1], [100, 33], 0, 0), (256, 6, [40, 3], [90, 50], 0, 0),
                                                                     (128, 8, [33], [300], 50, 4)])
def test_a_cache_declared_with_more_rows_than_the_copies_count(q4b, ctx, head, group, counts, lengths, window, sinks):
    """`pages` only bounds the table's entries: past 2^31 rows of a pool the kernel without tensor maps takes prompts too."""
    rng = np.random.default_rng(head)
    batch = Batch(rng, counts, lengths, 16, 2, head, "bf16")
    q = narrow(rng.standard_normal((batch.tokens, 2 * group, head)), "bf16")
    want, tolerance = attention_reference(batch, q, 2 * group, 1 / math.sqrt(head), window, sinks)
    cache, described = batch.upload(q4b, ctx)
    d_q, d_out = ctx.to_device(q), ctx.alloc(q.nbytes)
    for pages in ((1 << 31) // 32, 0xffffffff):   # every entry of the table is a page that is there
        cache.pages = pages
        ctx.attention(cache, described, d_q.ptr, 2 * group, d_out.ptr, 1 / math.sqrt(head), window, sinks)
        ctx.sync()
        got = widen(d_out.download(np.uint16, q.shape), "bf16")
        assert (np.abs(got - want) <= tolerance).all(), pages


@pytest.mark.parametrize("head,page", [(256, 16), (64, 128)])
def test_pages_far_behind_the_pools_start(q4b, ctx, head, page):
    """Pools of 9 GB: the last pages begin beyond 2^32 values.  Written and read there, a cache gives the same bits as a small
    one."""
    rng = np.random.default_rng(page)
    kv_heads, group, length = 2, 6, 2 * page + 5
    far = 9 * 2 ** 30 // (2 * page * kv_heads * head)
    assert (far - 3) * page * kv_heads * head > 2 ** 32
    x = {name: narrow(rng.standard_normal((length, heads * head)), "bf16") for name, heads in
         (("q", kv_heads * group), ("k", kv_heads), ("v", kv_heads))}
    d = {name: ctx.to_device(bits) for name, bits in x.items()}
    begin, lengths = ctx.to_device(np.array([0, length], np.uint32)), ctx.to_device(np.array([length], np.uint32))
    one = ctx.to_device(np.array([0, 1], np.uint32))
    answers = []
    for pages in (3, far):
        pools = [ctx.alloc(pages * page * kv_heads * head * 2) for _ in range(2)]
        table = ctx.to_device(np.array([pages - 1, pages - 3, pages - 2], np.uint32))
        cache = q4b.KVCache(keys=pools[0].ptr, values=pools[1].ptr, dtype=q4b.BF16, pages=pages, page_tokens=page, kv_heads=kv_heads,
                            head_size=head)
        batch = q4b.TokenBatch(sequences=1, tokens=length, most_tokens=length, token_begin=begin.ptr, lengths=lengths.ptr,
                               page_table=table.ptr, table_stride=3)
        turned = ctx.alloc(x["q"].nbytes)
        ctx.rope_append(cache, batch, q4b.Rope(rotary_size=head, pairing=q4b.ROPE_HALVES, base=1e4), d["q"].ptr, d["k"].ptr, d["v"].ptr,
                        q4b.BF16, kv_heads * group, turned.ptr)
        prompt, single = ctx.alloc(x["q"].nbytes), ctx.alloc(x["q"].nbytes // length)
        ctx.attention(cache, batch, turned.ptr, kv_heads * group, prompt.ptr, 0.1)
        last = q4b.TokenBatch(sequences=1, tokens=1, most_tokens=1, token_begin=one.ptr, lengths=lengths.ptr, page_table=table.ptr,
                              table_stride=3)
        ctx.attention(cache, last, turned.ptr + (length - 1) * kv_heads * group * head * 2, kv_heads * group, single.ptr, 0.1)
        ctx.sync()
        answers.append((turned.download(np.uint16, x["q"].shape), prompt.download(np.uint16, x["q"].shape),
                        single.download(np.uint16, (kv_heads * group * head,))))
        for pool in pools:
            pool.free()
    for near, away in zip(*answers):
        assert (near == away).all()
    tolerance = 2.0 ** -7 * np.abs(widen(answers[0][1][-1], "bf16")).max()   # two kernels' roundings of one row
    assert (np.abs(widen(answers[0][1][-1], "bf16") - widen(answers[0][2], "bf16")) <= tolerance).all()
