"""Attention over the paged cache (q4b_attention) against its definition in 64 bits, at the sizes, masks and contents
where it can go wrong."""
import math

import numpy as np
import pytest

from cache_cases import Batch, attention_reference, narrow, storage, widen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


def attend(q4b, ctx, batch, q, q_heads, scale, window, sinks, most_tokens=None, pad_columns=0):
    """Through device buffers with `pad_columns` spare columns; returns [tokens, q_heads, head] bits and the spare ones."""
    cache, described = batch.upload(q4b, ctx, most_tokens)
    width = q_heads * batch.head
    ld = width + pad_columns
    rows = np.zeros((batch.tokens, ld), dtype=storage(batch.dtype))
    rows[:, :width] = q.reshape(batch.tokens, width)
    before = narrow(np.arange(batch.tokens * ld).reshape(batch.tokens, ld) % 113 - 56.0, batch.dtype)
    d_q, d_out = ctx.to_device(rows), ctx.to_device(before)
    ctx.attention(cache, described, d_q.ptr, q_heads, d_out.ptr, scale, window, sinks, ldq=ld, ldo=ld)
    got = d_out.download(storage(batch.dtype), (batch.tokens, ld))
    assert (got[:, width:] == before[:, width:]).all()
    assert (got[batch.used:] == before[batch.used:]).all(), "rows behind the last sequence"
    return got[:, :width].reshape(batch.tokens, q_heads, batch.head)


def check(q4b, ctx, batch, q_heads, window=0, sinks=0, seed=0, scale=None, **how):
    rng = np.random.default_rng(seed + 1)
    q = narrow(rng.standard_normal((batch.tokens, q_heads, batch.head)) * 1.5, batch.dtype)
    scale = 1.0 / math.sqrt(batch.head) if scale is None else scale
    got = widen(attend(q4b, ctx, batch, q, q_heads, scale, window, sinks, **how), batch.dtype)
    want, tolerance = attention_reference(batch, q, q_heads, scale, window, sinks)
    used = slice(0, batch.used)
    off = np.abs(got[used] - want[used])
    assert np.isfinite(got[used]).all()
    worst = np.max(off / np.maximum(tolerance[used], 1e-30)) if off.size else 0.0
    assert worst <= 1.0, f"{worst:.2f} times the tolerance"
    return got


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 6), (1, 8), (2, 3), (1, 17)])
def test_single_tokens(q4b, ctx, dtype, head, kv_heads, group):
    rng = np.random.default_rng(head + group)
    lengths = [1, 15, 16, 17, 63, 130]
    batch = Batch(rng, [1] * len(lengths), lengths, 16, kv_heads, head, dtype, pad=2)
    check(q4b, ctx, batch, kv_heads * group, pad_columns=8)


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 2), (7, 4), (16, 1), (40, 33), (500, 4), (20, 10 ** 9)])
@pytest.mark.parametrize("head,page", [(256, 16), (128, 64), (64, 32)])
def test_windows_and_sinks(q4b, ctx, window, sinks, head, page):
    rng = np.random.default_rng(window + sinks % 97)
    batch = Batch(rng, [1, 4, 2, 9, 40], [200, 77, 2, 9, 161], page, 2, head, "bf16")
    check(q4b, ctx, batch, 12, window, sinks)


@pytest.mark.parametrize("counts,lengths", [([4, 4], [4, 100]), ([3, 0, 5], [40, 33, 5]), ([0, 0, 2], [0, 9, 31]),
                                            ([23], [23]), ([70, 1, 33], [70, 50, 333]), ([150], [150]), ([130], [700])])
@pytest.mark.parametrize("dtype,head", [("f16", 256), ("bf16", 128), ("f16", 64)])
def test_several_tokens_and_prompts(q4b, ctx, counts, lengths, dtype, head):
    rng = np.random.default_rng(sum(counts))
    batch = Batch(rng, counts, lengths, 32, 2, head, dtype, pad=1)
    check(q4b, ctx, batch, 12)


@pytest.mark.parametrize("page", [16, 128, 1024])
def test_a_long_context_is_split_and_joined(q4b, ctx, page):
    rng = np.random.default_rng(page)
    batch = Batch(rng, [1, 2], [5003, 2999], page, 1, 128, "f16")
    check(q4b, ctx, batch, 4)


@pytest.mark.parametrize("dtype,head,page,kv_heads,group,counts,lengths,window,sinks", [
    ("f16", 256, 64, 2, 6, [500], [2300], 0, 0), ("bf16", 128, 16, 2, 4, [700, 33], [701, 1400], 0, 0),
    ("f16", 64, 32, 1, 8, [400], [5000], 0, 0), ("bf16", 256, 16, 2, 8, [900], [900], 300, 5),
    ("f16", 128, 128, 1, 5, [7, 300], [4000, 2000], 1000, 200), ("bf16", 64, 1024, 4, 1, [777], [777], 0, 0),
    ("f16", 256, 16, 1, 24, [1, 2], [3000, 1000], 0, 0), ("bf16", 256, 32, 1, 6, [4, 4, 4], [2000, 3, 900], 512, 4)])
def test_prompts_and_pieces_of_prompts(q4b, ctx, dtype, head, page, kv_heads, group, counts, lengths, window, sinks):
    """Many tiles of rows and of keys: rings and barriers go round, keys are split over clusters or are not."""
    rng = np.random.default_rng(head + page)
    batch = Batch(rng, counts, lengths, page, kv_heads, head, dtype, pad=2)
    check(q4b, ctx, batch, kv_heads * group, window, sinks)


def test_growing_scores(q4b, ctx):
    """Keys whose scores grow along the sequence: the running maximum is passed again and again."""
    rng = np.random.default_rng(8)
    for head in (64, 128, 256):
        batch = Batch(rng, [60], [1500], 32, 1, head, "f16")
        ramp = np.zeros(batch.stride * batch.page)
        ramp[:1500] = np.linspace(0, 1, 1500)
        direction = rng.choice([-1.0, 1.0], size=head)
        for j in range(1500):
            page, place = batch.slot(0, j)
            batch.keys[page, 0, place] = narrow(direction * ramp[j] * 2 + rng.standard_normal(head) * 0.1, "f16")
        q = narrow(np.broadcast_to(direction, (batch.tokens, 4, head)) * 2.0 + rng.standard_normal((batch.tokens, 4, head)) * 0.1, "f16")
        for scale in (0.3, -0.3):
            got = widen(attend(q4b, ctx, batch, q, 4, scale, 0, 0), "f16")
            want, tolerance = attention_reference(batch, q, 4, scale, 0, 0)
            assert (np.abs(got - want) <= tolerance).all()


@pytest.mark.parametrize("dtype,head,page,kv_heads,group,new,length,window,sinks", [
    ("f16", 256, 16, 4, 6, 1, 1, 0, 0), ("f16", 256, 16, 4, 6, 1, 130, 0, 0), ("bf16", 256, 64, 4, 6, 1, 9001, 0, 0),
    ("f16", 128, 32, 1, 4, 1, 20011, 0, 0), ("bf16", 64, 16, 2, 8, 2, 5000, 0, 0), ("f16", 128, 16, 3, 3, 5, 3001, 777, 20),
    ("bf16", 256, 16, 1, 1, 16, 40, 0, 0), ("f16", 64, 64, 24, 1, 1, 700, 0, 0), ("f16", 64, 16, 1, 16, 1, 4097, 4000, 3)])
def test_one_sequence(q4b, ctx, dtype, head, page, kv_heads, group, new, length, window, sinks):
    """Its heads are cut into shares that meet in clusters, and those in the workspace -- or not, with many heads."""
    rng = np.random.default_rng(length)
    batch = Batch(rng, [new], [length], page, kv_heads, head, dtype, pad=1)
    check(q4b, ctx, batch, kv_heads * group, window, sinks)
    check(q4b, ctx, batch, kv_heads * group, window, sinks, most_tokens=1)   # a hint that is too small


def test_many_unlike_sequences(q4b, ctx):
    rng = np.random.default_rng(5)
    lengths = rng.integers(1, 90, size=300)
    batch = Batch(rng, np.ones(300, dtype=int), lengths, 16, 2, 64, "bf16")
    check(q4b, ctx, batch, 4)


@pytest.mark.parametrize("most_tokens", [0, 1, 10 ** 6])
def test_the_hint_changes_no_result(q4b, ctx, most_tokens):
    rng = np.random.default_rng(6)
    batch = Batch(rng, [5, 1, 60], [80, 30, 60], 16, 1, 128, "f16")
    check(q4b, ctx, batch, 6, most_tokens=most_tokens)


def test_rows_in_front_of_the_sequence_are_zeros(q4b, ctx):
    rng = np.random.default_rng(7)
    batch = Batch(rng, [5, 3, 40], [3, 0, 22], 16, 2, 128, "bf16")
    got = check(q4b, ctx, batch, 4)
    assert (got[0:2] == 0).all() and (got[5:8] == 0).all() and (got[8:26] == 0).all()
    assert (got[2:5] != 0).any() and (got[26:48] != 0).any()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("counts,lengths", [([1, 6], [37, 50]), ([40], [90]), ([100, 50], [100, 300])])
def test_what_is_not_visible_has_no_influence(q4b, ctx, dtype, head, counts, lengths):
    """NaN and infinities behind a sequence's end, in pages of nobody, in front of a window, and in later tokens."""
    rng = np.random.default_rng(head)
    batch = Batch(rng, counts, lengths, 32, 1, head, dtype)
    window, sinks, group = 20, 3, 6
    rows = rng.standard_normal((batch.tokens, group, head)) * 1.5
    q = narrow(rows, dtype)
    bad = narrow(np.array([np.nan, np.inf, -np.inf, np.nan]), dtype)
    mark = np.zeros((batch.pages, batch.page), dtype=bool)      # slots of visible tokens
    poisoned_from = {}
    for s, length in enumerate(lengths):
        first = max(0, batch.place(s, 0) - window + 1)
        for j in list(range(min(sinks, length))) + list(range(first, length)):
            mark[batch.slot(s, j)] = True
    for pool in (batch.keys, batch.values):
        pool[~mark[:, None, :].repeat(1, axis=1)] = bad[rng.integers(0, 4)]
    # the last token's values hold an infinity, the first one's behind the sinks a NaN: rows that do not see them are clean
    for s, length in enumerate(lengths):
        page, place = batch.slot(s, length - 1)
        batch.values[page, 0, place, ::3] = bad[1]
        poisoned_from[s] = length - 1
    got = widen(attend(q4b, ctx, batch, q, group, 1 / math.sqrt(head), window, sinks), dtype)
    clean = Batch.__new__(Batch)
    clean.__dict__.update(batch.__dict__)
    clean.keys, clean.values = batch.keys.copy(), batch.values.copy()
    for s, length in enumerate(lengths):
        page, place = batch.slot(s, length - 1)
        clean.values[page, 0, place, ::3] = 0
    want, tolerance = attention_reference(clean, q, group, 1 / math.sqrt(head), window, sinks)
    for s in range(len(counts)):
        for i in range(counts[s]):
            row = int(batch.begin[s]) + i
            if batch.place(s, i) < poisoned_from[s]:
                assert np.isfinite(got[row]).all() and (np.abs(got[row] - want[row]) <= tolerance[row]).all(), (s, i)
            else:  # it sees the infinity, and only in those columns
                assert not np.isfinite(got[row][:, ::3]).any()
                others = np.arange(head) % 3 != 0
                assert (np.abs(got[row] - want[row]) <= tolerance[row])[:, others].all()


def test_scores_of_any_size(q4b, ctx):
    """Scores of thousands: the maximum is taken off before the exponential.  One key wins by far."""
    rng = np.random.default_rng(9)
    for head in (64, 256):
        batch = Batch(rng, [1, 33], [100, 150], 16, 1, head, "f16")
        check(q4b, ctx, batch, 2, scale=30.0)
        check(q4b, ctx, batch, 2, scale=-2.0)
        check(q4b, ctx, batch, 2, scale=0.0)


def test_equal_calls_give_equal_bits(q4b, ctx):
    rng = np.random.default_rng(10)
    batch = Batch(rng, [1, 1, 4, 90], [3000, 50, 900, 400], 16, 2, 256, "bf16")
    q = narrow(rng.standard_normal((batch.tokens, 12, 256)), "bf16")
    first = attend(q4b, ctx, batch, q, 12, 0.0625, 0, 0)
    for _ in range(5):
        assert (attend(q4b, ctx, batch, q, 12, 0.0625, 0, 0) == first).all()


def test_a_recorded_call_follows_the_lengths(q4b, ctx):
    """Lengths and pages are read when the recorded call runs: two graphs share the workspace, replayed in turn."""
    rng = np.random.default_rng(11)
    batch = Batch(rng, [1, 1], [700, 90], 16, 2, 128, "f16")
    long = Batch(rng, [1, 2], [4000, 3000], 16, 2, 128, "f16")
    check(q4b, ctx, batch, 8)
    runs = []
    for b in (batch, long):
        cache, described = b.upload(q4b, ctx)
        q = narrow(rng.standard_normal((b.tokens, 8, 128)), "f16")
        d_q, d_out = ctx.to_device(q), ctx.alloc(q.nbytes)
        ctx.graph_begin()
        ctx.attention(cache, described, d_q.ptr, 8, d_out.ptr, 0.1)
        runs.append((b, q, d_q, d_out, ctx.graph_end()))
    for step in range(3):
        for b, q, d_q, d_out, graph in runs:
            b.lengths = b.lengths - 30 * step   # 90, 60, 0 of the shortest
            b.d_lengths.upload(b.lengths.astype(np.uint32))
            graph.launch()
            got = widen(d_out.download(np.float16, q.shape), "f16")
            want, tolerance = attention_reference(b, q, 8, 0.1, 0, 0)
            assert (np.abs(got - want) <= tolerance).all(), step


@pytest.mark.parametrize("counts,lengths", [([1], [4000]), ([1, 1], [4000, 2000]), ([64], [4000])])
def test_many_small_weights_of_fp16_are_not_lost(q4b, ctx, counts, lengths):
    """One key far above 4,000 others whose weights are 2^-25 of its own: together they are a ten-thousandth of the sum, and
    below the last bit that fp16 has next to 1.

    Tolerance: that of attention_reference for what is as large as the answer; a weight's rounding is half an eps of
    itself, or 2^-32 of the largest one's where that is more (fp16's steps end at 2^-24; the largest is set to 2^7 or
    more)."""
    rng = np.random.default_rng(21)
    batch = Batch(rng, counts, lengths, 64, 1, 64, "f16")
    batch.keys[:], batch.values[:] = 0.0, 1.0
    for s in range(len(counts)):
        page, place = batch.slot(s, 5)
        batch.keys[page, 0, place, 0] = 1.0
        batch.values[page, 0, place] = 0.0
    q = np.zeros((batch.tokens, 2, 64), np.float16)
    q[:, :, 0] = 1.0
    scale = 25.0 * math.log(2.0)
    got = widen(attend(q4b, ctx, batch, q, 2, scale, 0, 0), "f16")
    want, tolerance = attention_reference(batch, q, 2, scale, 0, 0)
    tolerance = tolerance + max(lengths) * 2.0 ** -32
    assert (want > 40 * tolerance).all()   # losing them would show
    assert (np.abs(got - want) <= tolerance).all()


def test_sequences_that_share_pages(q4b, ctx):
    """A common beginning is held once; the same page may even stand in a table twice."""
    rng = np.random.default_rng(22)
    for counts in ([1, 2, 1], [40, 33, 1]):
        batch = Batch(rng, counts, [130, 170, 90], 32, 2, 128, "bf16")
        batch.table[1, :2] = batch.table[0, :2]
        batch.table[2, :2] = batch.table[0, 1]
        check(q4b, ctx, batch, 4)


def test_the_output_beside_the_queries(q4b, ctx):
    """q and out may be columns of one matrix."""
    rng = np.random.default_rng(23)
    for counts, lengths in (([1, 3], [40, 20]), ([50], [60])):
        batch = Batch(rng, counts, lengths, 16, 1, 64, "f16")
        cache, described = batch.upload(q4b, ctx)
        q = narrow(rng.standard_normal((batch.tokens, 2, 64)), "f16")
        rows = np.zeros((batch.tokens, 264), np.float16)
        rows[:, :128], rows[:, 256:] = q.reshape(batch.tokens, 128), 3.0
        d = ctx.to_device(rows)
        ctx.attention(cache, described, d.ptr, 2, d.ptr + 256, 0.125, ldq=264, ldo=264)
        after = d.download(np.float16, rows.shape)
        want, tolerance = attention_reference(batch, q, 2, 0.125, 0, 0)
        assert (np.abs(widen(after[:, 128:256], "f16").reshape(want.shape) - want) <= tolerance).all()
        assert (after[:, :128] == rows[:, :128]).all() and (after[:, 256:] == 3.0).all()
        with pytest.raises(q4b.Q4Error):
            ctx.attention(cache, described, d.ptr, 2, d.ptr + 240, 0.125, ldq=264, ldo=264)
        with pytest.raises(q4b.Q4Error):   # its last columns reach into the next row's queries
            ctx.attention(cache, described, d.ptr, 2, d.ptr + 400, 0.125, ldq=264, ldo=264)


def test_two_contexts_at_once(q4b):
    """Each has its own stream and workspace; their calls run next to each other, from a host thread each."""
    import threading
    failures = []

    def work(seed):
        try:
            with q4b.Q4Context(0) as own:
                rng = np.random.default_rng(seed)
                for counts, lengths in (([1], [6000]), ([1, 1, 3], [3000, 70, 900]), ([200], [500]), ([1], [3000])):
                    check(q4b, own, Batch(rng, counts, lengths, 64, 2, 128, "f16"), 4, seed=seed)
        except BaseException as error:  # noqa: BLE001 -- told to the test
            failures.append(error)
    threads = [threading.Thread(target=work, args=(seed,)) for seed in (31, 32)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


@pytest.mark.parametrize("begin", [[0, 3, 2, 5], [0, 40, 10, 60], [0, 2, 900, 5], [7, 7, 90, 91]])
def test_begins_that_fall_or_pass_the_rows_are_reported(q4b, ctx, begin):
    rng = np.random.default_rng(24)
    batch = Batch(rng, [30, 20, 10], [100, 50, 40], 16, 2, 64, "f16")
    for most in (1, 40):
        cache, described = batch.upload(q4b, ctx, most)
        batch.d_begin.upload(np.asarray(begin, dtype=np.uint32))
        d_q, d_out = ctx.to_device(np.zeros((batch.tokens, 4, 64), np.float16)), ctx.alloc(batch.tokens * 4 * 64 * 2)
        ctx.attention(cache, described, d_q.ptr, 4, d_out.ptr, 0.1)
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.sync()
        assert refused.value.status == 1 and "token_begin" in refused.value.message
        check(q4b, ctx, Batch(rng, [30, 20, 10], [100, 50, 40], 16, 2, 64, "f16"), 4)


def test_bad_pages_are_reported_and_not_followed(q4b, ctx):
    rng = np.random.default_rng(12)
    for counts in ([1, 1], [90, 40]):
        batch = Batch(rng, counts, [200, 100], 16, 1, 128, "f16")
        batch.table[1, 2] = batch.pages
        cache, described = batch.upload(q4b, ctx)
        d_q, d_out = ctx.alloc(batch.tokens * 4 * 128 * 2), ctx.alloc(batch.tokens * 4 * 128 * 2)
        ctx.attention(cache, described, d_q.ptr, 4, d_out.ptr, 0.1)
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.sync()
        assert refused.value.status == 1 and "page" in refused.value.message
        ctx.sync()
        described.table_stride = 2   # too short for both
        ctx.attention(cache, described, d_q.ptr, 4, d_out.ptr, 0.1)
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.sync()
        assert refused.value.status == 1
        check(q4b, ctx, Batch(rng, counts, [200, 100], 16, 1, 128, "f16"), 4)


def test_nothing_to_do(q4b, ctx):
    cache = q4b.KVCache(keys=1 << 20, values=1 << 20, dtype=q4b.F16, pages=1, page_tokens=16, kv_heads=1, head_size=64)
    launches = ctx.launches
    ctx.attention(cache, q4b.TokenBatch(), 1 << 20, 1, 1 << 21, 1.0)
    assert ctx.launches == launches
    rng = np.random.default_rng(13)
    batch = Batch(rng, [0, 0], [5, 0], 16, 1, 64, "f16", pad=3)   # rows, but none of a sequence
    check(q4b, ctx, batch, 1, most_tokens=0)


def test_refusals(q4b, ctx):
    rng = np.random.default_rng(14)
    batch = Batch(rng, [1], [10], 16, 2, 64, "f16")
    cache, described = batch.upload(q4b, ctx)
    buffer = ctx.alloc(1 << 16)
    good = dict(q_ptr=buffer.ptr, q_heads=4, out_ptr=buffer.ptr + 4096, scale=0.1, ldq=256, ldo=256)

    def refused(cache_change=None, batch_change=None, **change):
        c, b = q4b.KVCache.from_buffer_copy(cache), q4b.TokenBatch.from_buffer_copy(described)
        for target, fields in ((c, cache_change), (b, batch_change)):
            for name, value in (fields or {}).items():
                setattr(target, name, value)
        with pytest.raises(q4b.Q4Error) as error:
            ctx.attention(c, b, **{**good, **change})
        assert error.value.status == 1 and error.value.message
    for change in ({"dtype": q4b.F32}, {"pages": 0}, {"page_tokens": 8}, {"page_tokens": 24}, {"page_tokens": 2048},
                   {"head_size": 96}, {"kv_heads": 0}, {"kv_heads": 3}, {"keys": None}, {"values": cache.values + 2}):
        refused(cache_change=change)
    for change in ({"token_begin": None}, {"lengths": None}, {"page_table": None}, {"table_stride": 0},
                   {"lengths": described.lengths + 2}):
        refused(batch_change=change)
    for change in ({"q_heads": 0}, {"q_heads": 5}, {"ldq": 248}, {"ldo": 248}, {"ldq": 260}, {"q_ptr": buffer.ptr + 2},
                   {"out_ptr": buffer.ptr}, {"out_ptr": 0}, {"scale": math.nan}, {"scale": math.inf}):
        refused(**change)
    with q4b.Q4Context(0) as fresh:   # a first call while recording would have to allocate
        fresh.graph_begin()
        with pytest.raises(q4b.Q4Error) as error:
            fresh.attention(cache, described, **good)
        assert error.value.status == 1 and "recording" in error.value.message
        fresh.graph_end().free()
        fresh.attention(cache, described, **good)
        fresh.sync()
