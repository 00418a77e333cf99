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
