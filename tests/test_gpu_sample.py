"""Sampling (q4b_sample) against its definition in 64 bits: equal tokens, shares to fp32's rounding."""
import math

import numpy as np
import pytest

from cache_cases import narrow, widen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


def reference(logit, u, temperature=1.0, k=0, p=1.0, m=0.0):
    """(token, probability, margin): margin is how near the choice came to going to a neighbour, relative to the sums."""
    logit, k = np.where(np.isnan(logit), -np.inf, logit), int(k)
    top = logit.max()
    if top == -np.inf:
        return 0xffffffff, 0.0, 1.0
    if not temperature > 0:
        return int(logit.argmax()), 1.0, 1.0
    with np.errstate(invalid="ignore", divide="ignore"):
        weight = np.where(logit == top, 1.0, np.where(np.isneginf(logit - top), 0.0, np.exp((logit - top) / np.float64(temperature))))
    order = np.argsort(-logit, kind="stable")
    if 0 < k < len(order):
        order = order[:k]
    margin = 1.0
    if p < 1:
        running = np.cumsum(weight[order])
        target = max(p, 0.0) * running[-1]
        count = max(1, int((running - weight[order] < target).sum()))
        if target > 0:
            # a difference within rounding of the border decides nothing where it is exact on both sides
            gaps = np.abs(running - target)
            margin = min(margin, float(gaps.min() / running[-1])) if gaps.min() > 0 else margin
        order = order[:count]
    if m > 0:
        kept = weight[order] >= min(m, 1.0)
        margin = min(margin, float(np.abs(weight[order] - min(m, 1.0)).min())) if m < 1 else margin
        order = order[kept]
    chosen = np.sort(order)
    running = np.cumsum(weight[chosen])
    target = (u if u > 0 else 0.0) * running[-1]
    at = int((running <= target).sum())
    last = int(np.flatnonzero(weight[chosen] > 0)[-1])
    at = min(at, last)
    if target > 0:
        margin = min(margin, float(np.abs(running - target).min() / running[-1]))
    return int(chosen[at]), float(weight[chosen[at]] / running[-1]), margin


def run(q4b, ctx, logits, dtype, u, rules, ld=None, offset=0):
    rows, vocab = logits.shape
    ld = vocab if ld is None else ld
    bits = narrow(logits, dtype)
    flat = np.zeros(offset + rows * ld, dtype=bits.dtype)
    flat[offset:].reshape(rows, ld)[:, :vocab] = bits
    d_logits, d_u = ctx.to_device(flat), ctx.to_device(np.asarray(u, dtype=np.float32))
    d_tokens = ctx.to_device(np.full(rows + 1, 77, dtype=np.uint32))
    d_share = ctx.to_device(np.full(rows + 1, -7.0, dtype=np.float32))
    held = {name: ctx.to_device(np.asarray(values, dtype=np.uint32 if name == "top_k" else np.float32))
            for name, values in rules.items()}
    ctx.sample(d_logits.ptr + offset * bits.itemsize, getattr(q4b, dtype.upper()), rows, vocab, d_u.ptr, d_tokens.ptr,
               probability_ptr=d_share.ptr, ld=ld, **{name: d.ptr for name, d in held.items()})
    tokens, share = d_tokens.download(np.uint32, rows + 1), d_share.download(np.float32, rows + 1)
    assert tokens[rows] == 77 and share[rows] == -7.0
    return tokens[:rows], share[:rows], widen(bits, dtype)


def check(q4b, ctx, logits, dtype="f32", u=None, seed=0, **rules):
    rows, vocab = logits.shape
    ld, offset = rules.pop("ld", None), rules.pop("offset", 0)
    rng = np.random.default_rng(seed + 100)
    u = rng.random(rows).astype(np.float32) if u is None else np.asarray(u, dtype=np.float32)
    tokens, share, held = run(q4b, ctx, logits, dtype, u, rules, ld, offset)
    rule = {name: np.asarray(values, dtype=np.float32 if name != "top_k" else np.uint32) for name, values in rules.items()}
    for r in range(rows):
        want, probability, margin = reference(held[r], float(u[r]), *(
            float(rule[name][r]) if name in rule else default
            for name, default in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0))))
        # A weight on the device is a whole number of units of 2^-42 of the largest one's (half a unit off), made from a
        # table entry rounded to 2^-31 (half of that, of at least one half), a sum with the rest's product rounded to
        # 2^-31, and a cubic in fp32 whose value is below 2^-9 (four roundings): 2^-31 + 2^-31 + 2^-31 < 2^-29 of it in
        # all.  So a running sum of n is off by 2^-29 of itself and n 2^-43 units of the largest weight, and where the
        # definition is nearer to a border than twice that, either neighbour is right.
        if margin <= 2.0 ** -28 + vocab * 2.0 ** -42:
            continue
        assert tokens[r] == want, (r, tokens[r], want, margin)
        # fp32's rounding, and the errors of a weight and of the sum
        assert abs(share[r] - probability) <= (2.0 ** -24 + 2.0 ** -28) * probability + vocab * 2.0 ** -42 + 2.0 ** -149, (r, share[r], probability)


def logits_of(rng, rows, vocab, spread=2.0):
    x = rng.standard_normal((rows, vocab)) * spread
    for r in range(rows):
        likely = rng.integers(0, vocab, size=min(vocab, 12))
        x[r, likely] += rng.random(likely.size) * 8
    return x


VOCABS = [1, 2, 31, 256, 257, 1000, 8191, 8192, 16384, 32769, 70001, 248320]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", VOCABS)
def test_every_rule(q4b, ctx, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 9
    logits = logits_of(rng, rows, vocab)
    temperature = rng.uniform(0.3, 2.0, rows)
    temperature[3] = 0.0
    k = rng.integers(1, 60, rows)
    k[5] = 0
    p, m = rng.uniform(0.2, 0.999, rows), rng.uniform(0, 0.3, rows)
    check(q4b, ctx, logits, dtype, seed=1)
    check(q4b, ctx, logits, dtype, seed=2, temperature=temperature)
    check(q4b, ctx, logits, dtype, seed=3, top_k=k)
    check(q4b, ctx, logits, dtype, seed=4, top_p=p)
    check(q4b, ctx, logits, dtype, seed=5, min_p=m)
    check(q4b, ctx, logits, dtype, seed=6, temperature=temperature, top_k=k, top_p=p, min_p=m, ld=vocab + 3, offset=1)


def test_large_counts_and_shares(q4b, ctx):
    """Cuts deep in the row: more elements at the border than are ranked at once."""
    rng = np.random.default_rng(1)
    vocab = 50_000
    logits = rng.standard_normal((6, vocab))
    check(q4b, ctx, logits, top_k=[1, 5000, 20_000, 49_999, 50_000, 60_000])
    check(q4b, ctx, logits, top_p=[0.5, 0.9, 0.99, 0.999, 0.9999, 1e-6])
    check(q4b, ctx, logits, top_k=[30_000] * 6, top_p=[0.5, 0.9, 0.99, 0.999, 0.0, 0.7])


def test_equal_logits(q4b, ctx):
    """Ties go to the lowest index, at every border."""
    for vocab in (7, 3000, 40_000):
        flat = np.zeros((5, vocab))
        check(q4b, ctx, flat, "f16", top_k=[1, 2, vocab // 2, vocab - 1, vocab])
        check(q4b, ctx, flat, "f32", u=[0.0, 0.25, 0.5, 0.75, 0.999])
        two = np.where(np.arange(vocab) % 3 == 0, 1.0, 0.0)[None].repeat(5, axis=0)
        check(q4b, ctx, two, "bf16", top_k=[1, vocab // 4 + 1, vocab // 3 + 2, vocab // 2, vocab - 1])
        check(q4b, ctx, two, "f32", temperature=[0.0, 0.0, 0.5, 1.0, 4.0])
    # half of the weight of equal logits is exactly half of them
    tokens, share, _ = run(q4b, ctx, np.zeros((4, 4096)), "f32", [0.0, 0.4999, 0.99999, 0.5], {"top_p": [0.5] * 4})
    assert list(tokens) == [0, int(0.4999 * 2048), 2047, 1024] and np.allclose(share, 1 / 2048)


def test_one_outlier_and_wide_ranges(q4b, ctx):
    rng = np.random.default_rng(2)
    vocab = 20_000
    logits = rng.standard_normal((4, vocab)) * 1e-3
    logits[0, 777] = 1e30
    logits[1, 5] = -1e30
    logits[2] *= 1e36
    logits[3, 9] = 12.0
    check(q4b, ctx, logits, top_k=[100] * 4)
    check(q4b, ctx, logits, top_p=[0.9] * 4)
    check(q4b, ctx, logits, temperature=[1e-30, 1e30, 3e38, 1e-3])


def test_infinities_and_nan(q4b, ctx):
    rng = np.random.default_rng(3)
    for vocab in (40, 9000):
        logits = rng.standard_normal((8, vocab))
        logits[0, 3] = np.nan
        logits[1] = np.nan
        logits[2] = -np.inf
        logits[3, 5:] = -np.inf
        logits[4, [7, 9]] = np.inf
        logits[5, ::2] = np.nan
        logits[6] = np.inf
        logits[7, 1:] = -np.inf
        u = [0.3, 0.3, 0.3, 0.9, 0.75, 0.5, 0.5, 0.9]
        check(q4b, ctx, logits, u=u)
        check(q4b, ctx, logits, u=u, temperature=[0.0] * 8)
        check(q4b, ctx, logits, u=u, top_k=[3] * 8, top_p=[0.9] * 8, min_p=[0.01] * 8)
        check(q4b, ctx, logits, u=u, top_k=[vocab - 1] * 8, temperature=[math.inf] * 8)
    tokens, share, _ = run(q4b, ctx, np.array([[0.0, -0.0, 0.0]]), "f32", [0.5], {"temperature": [math.nan]})
    assert tokens[0] == 0 and share[0] == 1.0
    check(q4b, ctx, np.zeros((3, 8)), u=[math.nan, -1.0, 5.0])
    check(q4b, ctx, rng.standard_normal((3, 500)), top_p=[math.nan, 1.0, 2.0], min_p=[math.nan, 0.0, -1.0])
    check(q4b, ctx, rng.standard_normal((3, 500)), top_p=[-1.0, 0.0, 1e-30], min_p=[0.0, 2.0, 1.0])


def test_random_numbers_at_the_ends(q4b, ctx):
    rng = np.random.default_rng(4)
    logits = logits_of(rng, 4, 30_000)
    check(q4b, ctx, logits, u=[0.0, 1.0 - 2.0 ** -24, 2.0 ** -30, 0.5])
    # at 1 and beyond the last token with any weight
    tokens, _, _ = run(q4b, ctx, np.array([[1.0, 2.0, -200.0]] * 2), "f32", [1.0, 3.0], {})
    assert list(tokens) == [1, 1]


def test_many_rows_and_the_largest_vocabulary(q4b, ctx):
    rng = np.random.default_rng(5)
    check(q4b, ctx, logits_of(rng, 700, 300), top_p=rng.uniform(0.3, 1.0, 700), top_k=rng.integers(0, 50, 700))
    big = logits_of(rng, 2, 1 << 20)
    check(q4b, ctx, big, "f32", top_p=[0.9, 0.3])
    check(q4b, ctx, big, "bf16", top_k=[1000, 7])


def test_a_row_does_not_depend_on_its_neighbours(q4b, ctx):
    rng = np.random.default_rng(6)
    logits, u = logits_of(rng, 40, 33_000), rng.random(40).astype(np.float32)
    together, share, _ = run(q4b, ctx, logits, "f32", u, {"top_p": np.full(40, 0.8)})
    for r in (0, 17, 39):
        alone, own, _ = run(q4b, ctx, logits[r:r + 1], "f32", u[r:r + 1], {"top_p": [0.8]})
        assert alone[0] == together[r] and own[0] == share[r]


def test_a_recorded_call(q4b, ctx):
    rng = np.random.default_rng(7)
    logits = logits_of(rng, 3, 9000)
    d_logits, d_u = ctx.to_device(logits.astype(np.float32)), ctx.alloc(12)
    d_tokens = ctx.alloc(12)
    ctx.graph_begin()
    ctx.sample(d_logits.ptr, q4b.F32, 3, 9000, d_u.ptr, d_tokens.ptr)
    graph = ctx.graph_end()
    for step in range(4):
        u = rng.random(3).astype(np.float32)
        d_u.upload(u)
        graph.launch()
        got = d_tokens.download(np.uint32, 3)
        assert [reference(logits.astype(np.float32)[r].astype(np.float64), float(u[r]))[0] for r in range(3)] == list(got)


def test_refusals(q4b, ctx):
    d = ctx.alloc(4096)
    good = dict(logits_ptr=d.ptr, dtype=q4b.F32, rows=1, vocab=100, uniform_ptr=d.ptr + 1024, tokens_ptr=d.ptr + 2048)
    for change in ({"dtype": 9}, {"vocab": 0}, {"vocab": (1 << 20) + 1}, {"ld": 99}, {"logits_ptr": 0}, {"logits_ptr": d.ptr + 2},
                   {"uniform_ptr": 0}, {"tokens_ptr": 0}, {"tokens_ptr": d.ptr + 2}, {"top_k": d.ptr + 1}, {"rows": (1 << 24) + 1}):
        with pytest.raises(q4b.Q4Error) as refused:
            ctx.sample(**{**good, **change})
        assert refused.value.status == 1 and refused.value.message
    launches = ctx.launches
    ctx.sample(**{**good, "rows": 0})
    assert ctx.launches == launches
