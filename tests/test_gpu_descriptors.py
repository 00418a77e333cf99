"""What the device arrays of a batch may hold and what is reported: the entries of pages that nobody sees, sequences without
new tokens, and each kind of mistake wherever in the batch it stands."""
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


def seen_pages(batch, window, sinks):
    """[sequences, table columns]: whether any new token of the sequence sees a token of that page."""
    seen = np.zeros(batch.table.shape, dtype=bool)
    for s in range(len(batch.counts)):
        for i in range(int(batch.counts[s])):
            at = batch.place(s, i)
            for j in range(at + 1):
                if window == 0 or j > at - window or j < sinks:
                    seen[s, j // batch.page] = True
    return seen


@pytest.mark.parametrize("most_tokens", [1, 10 ** 6])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("head,dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("counts,lengths,window,sinks", [([1, 4], [700, 333], 40, 4), ([40, 1], [500, 450], 100, 20),
                                                          ([150], [900], 33, 0), ([3, 2], [290, 61], 1, 1)])
def test_entries_of_pages_that_nobody_sees(q4b, ctx, counts, lengths, window, sinks, head, dtype, page, most_tokens):
    """A host gives the pages in front of a window to others and marks their entries: both kernels (the hint picks one)
    answer as before, and nothing is reported."""
    rng = np.random.default_rng(page + window)
    batch = Batch(rng, counts, lengths, page, 1, head, dtype, pad=1)
    q = narrow(rng.standard_normal((batch.tokens, 6, head)), dtype)
    want, tolerance = attention_reference(batch, q, 6, 1 / math.sqrt(head), window, sinks)
    unseen = ~seen_pages(batch, window, sinks)
    assert (unseen & (batch.table < batch.pages)).any()
    batch.table[unseen] = 0xffffffff
    cache, described = batch.upload(q4b, ctx, most_tokens)
    d_q, d_out = ctx.to_device(q), ctx.to_device(np.zeros_like(q))
    ctx.attention(cache, described, d_q.ptr, 6, d_out.ptr, 1 / math.sqrt(head), window, sinks)
    ctx.sync()
    got = widen(d_out.download(q.dtype, q.shape), dtype)[:batch.used]
    assert (np.abs(got - want[:batch.used]) <= tolerance[:batch.used]).all()
    # and the entry of a page that is seen is still reported
    s, column = np.argwhere(~unseen & (batch.table < batch.pages))[-1]
    batch.table[s, column] = batch.pages
    batch.d_table.upload(batch.table)
    ctx.attention(cache, described, d_q.ptr, 6, d_out.ptr, 1 / math.sqrt(head), window, sinks)
    with pytest.raises(q4b.Q4Error) as refused:
        ctx.sync()
    assert refused.value.status == 1 and "page" in refused.value.message
