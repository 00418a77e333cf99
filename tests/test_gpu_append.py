"""New tokens into the paged cache with their rotation (q4b_rope_append) against the definition in 64 bits."""
import ctypes

import numpy as np
import pytest

from cache_cases import EPS, Batch, narrow, rope_reference, storage, widen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


def reference(batch, q, k, v, q_heads, rotary, pairing, frequencies, positions=None):
    """q_out, keys, values in 64 bits, and which of them are written."""
    head, kv_heads = batch.head, batch.kv_heads
    out = np.zeros((batch.tokens, q_heads, head))
    keys, values = widen(batch.keys, batch.dtype), widen(batch.values, batch.dtype)
    wrote, touched = np.zeros(batch.tokens, dtype=bool), np.zeros((batch.pages, batch.page), dtype=bool)
    for s in range(len(batch.counts)):
        for i in range(int(batch.counts[s])):
            row, at = int(batch.begin[s]) + i, batch.place(s, i)
            if at < 0:
                continue
            position = [at if positions is None else positions[row]]
            wrote[row] = True
            out[row] = rope_reference(q[row][None], position, rotary, pairing, frequencies)[0]
            page, place = batch.slot(s, at)
            touched[page, place] = True
            keys[page, :, place] = rope_reference(k[row][None], position, rotary, pairing, frequencies)[0]
            values[page, :, place] = v[row]
    return out, keys, values, wrote, touched


def near(got, want, size, dtype, turns_error=0.0):
    """The type's rounding, and fp32 of three operations with a cosine that is off by 2^-22 at most: relative to the pair's
    two values, whose sizes `size` bounds."""
    eps = EPS[dtype]
    return np.abs(got - want) <= eps / 2 * np.abs(want) + (1 + eps) * size * (2.0 ** -21 + turns_error) + 2.0 ** -25


def run(q4b, ctx, batch, q, k, v, source, q_heads, rotary, pairing, base=1e4, frequencies=None, positions=None):
    cache, described = batch.upload(q4b, ctx)
    head = batch.head
    d_q, d_k, d_v = (ctx.to_device(narrow(x, source)) for x in (q, k, v))
    before = narrow(np.arange(batch.tokens * q_heads * head).reshape(batch.tokens, -1) % 97 - 48.0, batch.dtype)
    d_out = ctx.to_device(before)
    table = (ctypes.c_double * max(1, len(frequencies)))(*frequencies) if frequencies is not None else None
    d_positions = ctx.to_device(np.asarray(positions, dtype=np.int32)) if positions is not None else None
    rope = q4b.Rope(rotary_size=rotary, pairing=q4b.ROPE_HALVES if pairing == "halves" else q4b.ROPE_NEIGHBOURS, base=base,
                    frequencies=table, positions=d_positions.ptr if d_positions else None)
    ctx.rope_append(cache, described, rope, d_q.ptr, d_k.ptr, d_v.ptr, getattr(q4b, source.upper()), q_heads, d_out.ptr)
    pool = (batch.pages, batch.kv_heads, batch.page, head)
    return (d_out.download(storage(batch.dtype), before.shape), d_batch(batch.d_keys, batch, pool),
            d_batch(batch.d_values, batch, pool), before)


def d_batch(buffer, batch, shape):
    return buffer.download(storage(batch.dtype), shape)


def check(q4b, ctx, batch, source, q_heads, rotary, pairing, base=1e4, frequencies=None, positions=None, seed=0):
    rng = np.random.default_rng(seed)
    head = batch.head
    q, k, v = (widen(narrow(rng.standard_normal((batch.tokens, n, head)), source), source)
               for n in (q_heads, batch.kv_heads, batch.kv_heads))
    used = frequencies if frequencies is not None else [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    out, keys, values, wrote, touched = reference(batch, q, k, v, q_heads, rotary, pairing, used, positions)
    got_q, got_k, got_v, before = run(q4b, ctx, batch, q, k, v, source, q_heads, rotary, pairing, base, frequencies, positions)
    top = max(1.0, np.abs(q).max(), np.abs(k).max()) * 2
    assert near(widen(got_q[wrote], batch.dtype), out[wrote].reshape(-1, q_heads * head), top, batch.dtype).all()
    assert (got_q[~wrote] == before[~wrote]).all(), "rows of no sequence"
    mark = np.broadcast_to(touched[:, None, :, None], got_k.shape)
    assert near(widen(got_k, batch.dtype), keys, top, batch.dtype)[mark].all()
    assert (got_k[~mark] == batch.keys[~mark]).all() and (got_v[~mark] == batch.values[~mark]).all(), "slots of nobody"
    assert (got_v[mark] == narrow(values, batch.dtype)[mark]).all(), "values are copied and rounded once"


@pytest.mark.parametrize("source", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head,rotary,pairing", [(256, 64, "halves"), (128, 128, "neighbours"), (64, 16, "halves"),
                                                 (64, 48, "neighbours"), (256, 256, "halves"), (128, 0, "halves")])
def test_types_and_pairings(q4b, ctx, source, dtype, head, rotary, pairing):
    rng = np.random.default_rng(head + rotary)
    batch = Batch(rng, [1, 5, 0, 18], [1, 21, 9, 40], 16, 2, head, dtype, pad=3)
    check(q4b, ctx, batch, source, 6, rotary, pairing)


@pytest.mark.parametrize("page", [16, 64, 1024])
@pytest.mark.parametrize("counts", [[1], [1] * 70, [130], [3, 65, 2]])
def test_batches_and_pages(q4b, ctx, page, counts):
    rng = np.random.default_rng(page + len(counts))
    batch = Batch(rng, counts, np.asarray(counts) + rng.integers(0, 100, size=len(counts)), page, 1, 64, "bf16", pad=1)
    check(q4b, ctx, batch, "f32", 3, 32, "halves", base=1e6)


def test_far_positions(q4b, ctx):
    """At a million radians and at the end of int32's range, by the positions that the caller gives."""
    rng = np.random.default_rng(1)
    batch = Batch(rng, [6], [20], 16, 1, 128, "f16")
    # 2^31 / 2 pi turns x two roundings of 2^-53 each are 2^-23 turns, 2^-20.4 radians: inside nothing but its own bound
    positions = [999_999, 1_000_000, 123_456_789, 16_777_217, 3, 0]
    check(q4b, ctx, batch, "f32", 2, 128, "halves", base=1e7, positions=positions)
    check(q4b, ctx, batch, "f32", 2, 64, "neighbours", frequencies=list(np.linspace(1.0, 1e-6, 32)), positions=positions)
    check(q4b, ctx, batch, "f32", 2, 64, "neighbours", frequencies=[0.5 ** i for i in range(32)], positions=[-5, -1, 7, 0, 2, -1000])


def test_left_padding_is_skipped(q4b, ctx):
    rng = np.random.default_rng(2)
    batch = Batch(rng, [5, 4, 3], [3, 0, 9], 16, 2, 64, "f16")
    check(q4b, ctx, batch, "f16", 4, 64, "halves")


def test_columns_of_one_matrix_interleaved_heads_and_in_place(q4b, ctx):
    rng = np.random.default_rng(3)
    head, q_heads, kv_heads = 64, 4, 2
    batch = Batch(rng, [3, 2], [30, 2], 16, kv_heads, head, "f16")
    rope = q4b.Rope(rotary_size=32, pairing=q4b.ROPE_HALVES, base=1e4)
    frequencies = [1e4 ** (-i / 16) for i in range(16)]
    # per query head: head values of q, then head of something else (a gate); then k, then v
    width = q_heads * 2 * head + 2 * kv_heads * head
    matrix = narrow(rng.standard_normal((batch.tokens, width)), "f16")
    wide = widen(matrix, "f16")
    q = wide[:, :q_heads * 2 * head].reshape(batch.tokens, q_heads, 2 * head)[..., :head]
    k = wide[:, q_heads * 2 * head:][:, :kv_heads * head].reshape(batch.tokens, kv_heads, head)
    v = wide[:, q_heads * 2 * head + kv_heads * head:].reshape(batch.tokens, kv_heads, head)
    out, keys, values, wrote, touched = reference(batch, q, k, v, q_heads, 32, "halves", frequencies)
    cache, described = batch.upload(q4b, ctx)
    d = ctx.to_device(matrix)
    d_out = ctx.alloc(batch.tokens * q_heads * head * 2)
    ctx.rope_append(cache, described, rope, d.ptr, d.ptr + q_heads * 2 * head * 2, d.ptr + (q_heads * 2 + kv_heads) * head * 2,
                    q4b.F16, q_heads, d_out.ptr, ldq=width, q_head_stride=2 * head, ldk=width, ldv=width)
    got = widen(d_out.download(np.float16, (batch.tokens, q_heads, head)), "f16")
    assert near(got, out, 10.0, "f16").all()
    got_k = d_batch(batch.d_keys, batch, batch.keys.shape)
    mark = np.broadcast_to(touched[:, None, :, None], got_k.shape)
    assert near(widen(got_k, "f16"), keys, 10.0, "f16")[mark].all()
    assert (d_batch(batch.d_values, batch, batch.keys.shape)[mark] == narrow(values, "f16")[mark]).all()
    assert (d.download(np.float16, matrix.shape) == matrix).all()
    # in place: q is turned where it lies, next to k and v in the same rows
    dense = np.concatenate([q.reshape(batch.tokens, -1), k.reshape(batch.tokens, -1), v.reshape(batch.tokens, -1)], 1)
    d = ctx.to_device(narrow(dense, "f16"))
    ld = dense.shape[1]
    ctx.rope_append(cache, described, rope, d.ptr, d.ptr + q_heads * head * 2, d.ptr + (q_heads + kv_heads) * head * 2, q4b.F16,
                    q_heads, d.ptr, ldq=ld, ldk=ld, ldv=ld, ldq_out=ld)
    after = d.download(np.float16, dense.shape)
    assert near(widen(after[:, :q_heads * head], "f16"), out.reshape(batch.tokens, -1), 10.0, "f16").all()
    assert (after[:, q_heads * head:] == narrow(dense, "f16")[:, q_heads * head:]).all()


def test_bad_pages_are_reported_and_not_followed(q4b, ctx):
    rng = np.random.default_rng(4)
    batch = Batch(rng, [2, 2], [20, 40], 16, 1, 64, "f16")
    batch.table[1, 2] = batch.pages + 7
    cache, described = batch.upload(q4b, ctx)
    rope = q4b.Rope(rotary_size=64, pairing=q4b.ROPE_HALVES, base=1e4)
    d = ctx.alloc(4 * 3 * 64 * 2)
    out = ctx.alloc(4 * 64 * 2)
    for change in ({}, {"table_stride": 1}, {"tokens": 3}):
        for name, value in change.items():
            setattr(described, name, value)
        ctx.rope_append(cache, described, rope, d.ptr, d.ptr, d.ptr, q4b.F16, 1, out.ptr)
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.sync()
        assert refused.value.status == 1
        ctx.sync()


def test_a_recorded_call_follows_the_lengths(q4b, ctx):
    rng = np.random.default_rng(5)
    batch = Batch(rng, [1], [33], 16, 1, 64, "f16")
    cache, described = batch.upload(q4b, ctx)
    rope = q4b.Rope(rotary_size=64, pairing=q4b.ROPE_HALVES, base=1e4)
    x = narrow(rng.standard_normal((1, 1, 64)), "f16")
    d_x, d_out = ctx.to_device(x), ctx.alloc(256)
    ctx.graph_begin()
    ctx.rope_append(cache, described, rope, d_x.ptr, d_x.ptr, d_x.ptr, q4b.F16, 1, d_out.ptr)
    graph = ctx.graph_end()
    for length in (33, 17, 1, 32):
        batch.lengths = np.array([length])
        batch.d_lengths.upload(batch.lengths.astype(np.uint32))
        graph.launch()
        got = d_batch(batch.d_keys, batch, batch.keys.shape)
        page, place = batch.slot(0, length - 1)
        want = rope_reference(widen(x, "f16"), [length - 1], 64, "halves", [1e4 ** (-i / 32) for i in range(32)])
        assert near(widen(got[page, :, place], "f16"), want[0], 10.0, "f16").all()


def test_refusals(q4b, ctx):
    rng = np.random.default_rng(6)
    batch = Batch(rng, [1], [10], 16, 2, 64, "f16")
    cache, described = batch.upload(q4b, ctx)
    d = ctx.alloc(1 << 16)
    good = dict(q_ptr=d.ptr, k_ptr=d.ptr + 4096, v_ptr=d.ptr + 8192, dtype=q4b.F16, q_heads=4, q_out_ptr=d.ptr + 16384)

    def refused(rope=None, **change):
        fields = {"rotary_size": 64, "pairing": 0, "base": 1e4, **(rope or {})}
        with pytest.raises(q4b.Q4Error) as error:
            ctx.rope_append(cache, described, q4b.Rope(**fields), **{**good, **change})
        assert error.value.status == 1 and error.value.message
    for rope in ({"rotary_size": 8}, {"rotary_size": 80}, {"pairing": 2}, {"base": 0.0}, {"base": -1.0}, {"base": float("nan")},
                 {"frequencies": (ctypes.c_double * 32)(*[float("inf")] * 32)}, {"positions": d.ptr + 2}):
        refused(rope)
    for change in ({"dtype": 7}, {"q_heads": 3}, {"q_ptr": d.ptr + 2}, {"k_ptr": 0}, {"ldq": 248}, {"ldq": 260},
                   {"q_head_stride": 32}, {"ldk": 120}, {"ldv": 132}, {"ldq_out": 248}, {"q_out_ptr": d.ptr + 16},
                   {"q_out_ptr": d.ptr + 4096}, {"q_out_ptr": d.ptr, "ldq": 512}, {"q_out_ptr": d.ptr, "k_ptr": d.ptr + 256}, {"dtype": q4b.F32, "q_out_ptr": d.ptr}):
        refused(**change)
