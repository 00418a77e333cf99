"""Sampling (q4b_sample) where the weights' last bits show, and next to the borders of its rules."""
import math

import numpy as np
import pytest

from cache_cases import narrow, widen
from test_gpu_sample import reference, run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("high,tiny,temperature", [(8.0, 2.0 ** -22, 1.0), (12.0, 2.0 ** -21, 1.0), (32.0, 2.0 ** -20, 4.0),
                                                   (12.0, -2.0 ** -21, 1.0), (12.0, 3 * 2.0 ** -22, 1.0)])
@pytest.mark.parametrize("rules", [{}, {"top_k": 400}, {"top_p": 0.9999999}])
def test_tiny_logits_beside_a_large_one(q4b, ctx, dtype, high, tiny, temperature, rules):
    """high - tiny has more bits than fp32: what is left of the distance moves a weight by 2^-22 of itself.

    Tolerance of a share = weight / total: a weight is off by half a unit of 2^-42 and by 2^-29 of itself (a table entry, a
    product and a cubic, 2^-31 each), the total by n such halves and 2^-29 of itself, and the share is rounded to fp32."""
    vocab = 700
    logits = np.full((3, vocab), tiny)
    logits[:, 5] = high
    assert (widen(narrow(logits, dtype), dtype) == logits).all()
    u = [0.9, 0.9999, 0.0]
    device = {"temperature": [temperature] * 3, **{name: [value] * 3 for name, value in rules.items()}}
    tokens, share, held = run(q4b, ctx, logits, dtype, u, device)
    asked = {"temperature": float(np.float32(temperature)), "k": rules.get("top_k", 0), "p": float(np.float32(rules.get("top_p", 1.0)))}
    total = 1 + vocab * math.exp((tiny - high) / temperature)
    small = 0
    for r in range(3):
        want, probability, margin = reference(held[r], float(np.float32(u[r])), **asked)
        assert margin > 2.0 ** -28 + vocab * 2.0 ** -42   # nowhere near a border: the token is determined
        small += want != 5
        off = probability * (2.0 ** -24 + 2.0 ** -28 + vocab * 2.0 ** -43) + 2.0 ** -43 / total
        assert tokens[r] == want and abs(float(share[r]) - probability) <= off, (share[r], probability, off)
    assert small


@pytest.mark.parametrize("dtype,largest", [("f32", 3.4028234663852886e38), ("bf16", 3.3895313892515355e38), ("f16", 65504.0)])
@pytest.mark.parametrize("vocab", [40, 9000, 50_000])
def test_the_largest_finite_logit_beside_infinities(q4b, ctx, dtype, largest, vocab):
    """Logits of +infinity share everything: nothing is left for a finite one, however large."""
    rng = np.random.default_rng(vocab)
    logits = rng.standard_normal((4, vocab))
    places = np.sort(rng.choice(np.arange(4, vocab), size=4, replace=False))
    logits[:, places] = np.inf
    logits[:, [0, 2, vocab - 1]] = largest
    logits[:, 3] = -largest
    logits[:, 1] = np.nan
    if vocab - 1 in places:
        logits[:, vocab - 1] = np.inf
    u = [0.0, 0.3, 0.6, 0.99]
    want = places[[0, 1, 2, 3]]
    for rules in ({}, {"temperature": [0.01, 1.0, 100.0, 1e30]}, {"top_k": [6] * 4}, {"top_p": [0.999] * 4},
                  {"min_p": [1e-6] * 4}, {"top_k": [vocab - 1] * 4, "top_p": [0.99] * 4, "min_p": [0.5] * 4}):
        tokens, share, _ = run(q4b, ctx, logits, dtype, u, rules)
        assert list(tokens) == list(want) and (share == 0.25).all(), (rules, tokens, share)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [7, 3000, 40_000, 248_320, 1 << 20])
def test_equal_logits_at_exact_shares(q4b, ctx, dtype, vocab):
    """Equal logits have equal whole weights, so a random number that falls on a border falls on it exactly: the token is
    floor(u n) of the n that stay, and those are the first k, or the first ceil(p n)."""
    u = np.array([0.0, 0.25, 0.5, 0.75, 1.0 - 2.0 ** -24], dtype=np.float32)
    flat = np.full((5, vocab), -1.5)
    third, half = max(1, vocab // 3), vocab // 2
    for rules, stay in (({}, vocab), ({"top_k": third}, third), ({"top_p": 0.5}, math.ceil(0.5 * vocab)),
                        ({"top_k": max(1, half), "top_p": 0.25}, math.ceil(0.25 * max(1, half))),
                        ({"min_p": 1.0, "temperature": 0.25}, vocab)):
        tokens, share, _ = run(q4b, ctx, flat, dtype, u, {name: [value] * 5 for name, value in rules.items()})
        assert list(tokens) == [int(float(x) * stay) for x in u], (rules, tokens)
        assert (share == np.float32(1 / stay)).all(), (rules, share)


def acceptable(logit, u, temperature=1.0, k=0, p=1.0):
    """({token: share}, doubt) of every token that an answer may name when the device's running sums are off by 2^-29 of themselves and
    n halves of 2^-42 of the largest weight, at either border; the definition in 64 bits elsewhere."""
    weight = np.exp((logit - logit.max()) / temperature)
    order = np.argsort(-logit, kind="stable")[:k if 0 < k < len(logit) else len(logit)]
    running = np.cumsum(weight[order])
    off = running[-1] * 2.0 ** -28 + len(logit) * 2.0 ** -42
    fewest = most = len(order)
    if p < 1:
        fewest, most = (min(len(order), int(np.searchsorted(running, p * running[-1] + way * off)) + 1) for way in (-1, 1))
    chosen = np.sort(order[:most])
    running = np.cumsum(weight[chosen])
    doubt = off + weight[order[fewest:most]].sum()
    total, aim = running[-1], u * running[-1]
    low, high = np.searchsorted(running, aim - 2 * doubt, side="right"), np.searchsorted(running, aim + 2 * doubt, side="right")
    return {int(chosen[i]): float(weight[chosen[i]] / total) for i in range(low, min(high, len(chosen) - 1) + 1)}, doubt / total


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [50_000, 248_320, 1 << 20])
@pytest.mark.parametrize("rules", [{"top_p": 0.9}, {"top_p": 0.5}, {"top_p": 0.999}, {"top_k": 30_000, "top_p": 0.95}, {}])
def test_deep_cuts_of_long_rows(q4b, ctx, dtype, vocab, rules):
    """Every row is compared, also where a border is nearer than the sums are sure of: then with what either side gives."""
    rng = np.random.default_rng(vocab + len(rules))
    rows = 4
    logits = rng.standard_normal((rows, vocab)) * 2.0
    for r in range(rows):
        logits[r, rng.integers(0, vocab, size=12)] += rng.random(12) * 8
    u = rng.random(rows).astype(np.float32)
    temperature = np.array([1.0, 0.7, 1.5, 1.0], dtype=np.float32)
    tokens, share, held = run(q4b, ctx, logits, dtype, u, {"temperature": temperature, **{name: [value] * rows for name, value in rules.items()}})
    for r in range(rows):
        may, doubt = acceptable(held[r], float(u[r]), float(temperature[r]), rules.get("top_k", 0), float(np.float32(rules.get("top_p", 1.0))))
        assert len(may) < 64   # of tens of thousands
        assert int(tokens[r]) in may, (r, tokens[r], may)
        want = may[int(tokens[r])]
        assert abs(float(share[r]) - want) <= want * (2.0 ** -24 + 2.0 ** -28 + 2 * doubt) + 2.0 ** -42, (r, share[r], want)
