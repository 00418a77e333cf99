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
