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
        assert tokens[r] == want and abs(share[r] - probability) <= off, (share[r], probability, off)
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
