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


def append(q4b, ctx, batch, kv_heads, head):
    """Keys and values of ones for all rows, without a rotation; returns q_out."""
    cache, described = batch.upload(q4b, ctx)
    ones = np.ones((batch.tokens, kv_heads * head), np.float16)
    d_x, d_out = ctx.to_device(ones), ctx.to_device(np.zeros_like(ones))
    ctx.rope_append(cache, described, q4b.Rope(rotary_size=0, pairing=q4b.ROPE_HALVES), d_x.ptr, d_x.ptr, d_x.ptr, q4b.F16,
                    kv_heads, d_out.ptr)
    return d_out, d_x


# rows 8 and on belong to nobody, or a begin falls in front of the rows that are there
BEGINS = [(8, [0, 8, 12]), (8, [0, 0, 8, 9]), (8, [5, 0, 8]), (8, [8, 7, 8]), (40, [0, 40, 41]),
          (8, [0, 8] + [8] * 300 + [9]), (40, [0, 40] + [40] * 300 + [2]), (40, [3] + [0] * 70 + [40])]


def begins(tokens, begin, head, dtype="f16"):
    """A batch of `tokens` rows whose token_begin is replaced by `begin`."""
    rng = np.random.default_rng(tokens)
    counts = np.zeros(len(begin) - 1, dtype=int)
    counts[0] = tokens
    batch = Batch(rng, counts, [50] * len(counts), 16, 1, head, dtype)
    batch.begin = np.asarray(begin, dtype=np.uint32)
    return batch


@pytest.mark.parametrize("tokens,begin", BEGINS)
def test_the_append_reports_every_begin(q4b, ctx, tokens, begin):
    batch = begins(tokens, begin, 64)
    append(q4b, ctx, batch, 1, 64)
    with pytest.raises(q4b.Q4Error) as refused:
        ctx.sync()
    assert refused.value.status == 1 and "token_begin" in refused.value.message
    ctx.sync()


@pytest.mark.parametrize("most_tokens", [1, 0])
@pytest.mark.parametrize("tokens,begin", BEGINS)
@pytest.mark.parametrize("group", [1, 24])
def test_attention_reports_every_begin(q4b, ctx, tokens, begin, most_tokens, group):
    batch = begins(tokens, begin, 64)
    cache, described = batch.upload(q4b, ctx, most_tokens)
    q = np.zeros((tokens, group, 64), np.float16)
    d_q, d_out = ctx.to_device(q), ctx.to_device(q)
    ctx.attention(cache, described, d_q.ptr, group, d_out.ptr, 0.1)
    with pytest.raises(q4b.Q4Error) as refused:
        ctx.sync()
    assert refused.value.status == 1 and "token_begin" in refused.value.message
    ctx.sync()


@pytest.mark.parametrize("counts,lengths", [([1, 0, 0], [40, 3, 9]), ([0, 60, 0], [3, 60, 5]), ([1] + [0] * 400, [20] + [1] * 400),
                                            ([40] + [0] * 400, [50] + [1] * 400)])
def test_the_length_of_a_sequence_without_new_tokens_may_be_anything(q4b, ctx, counts, lengths):
    """Slots of a batch that are empty in this step keep what they held."""
    rng = np.random.default_rng(len(counts))
    batch = Batch(rng, counts, lengths, 16, 1, 64, "f16")
    q = narrow(rng.standard_normal((batch.tokens, 4, 64)), "f16")
    want, tolerance = attention_reference(batch, q, 4, 0.125, 0, 0)
    batch.lengths = np.where(np.asarray(counts) == 0, 0xfffffff0, batch.lengths)
    for most_tokens in (0, 1):
        cache, described = batch.upload(q4b, ctx, most_tokens)
        d_q, d_out = ctx.to_device(q), ctx.to_device(np.zeros_like(q))
        ctx.attention(cache, described, d_q.ptr, 4, d_out.ptr, 0.125)
        ctx.sync()
        assert (np.abs(widen(d_out.download(np.float16, q.shape), "f16") - want) <= tolerance).all()
    d_out, d_x = append(q4b, ctx, batch, 1, 64)
    ctx.sync()
    assert (d_out.download(np.float16, (batch.tokens, 64)) == 1).all()
