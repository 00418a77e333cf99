"""What the rounding of attention's weights to 16 bits does to its outputs: nothing where the values are equal, and no more
than the values' spread lets it elsewhere."""
import math

import numpy as np
import pytest

from cache_cases import EPS, Batch, narrow, widen
from test_gpu_attention import attend

pytestmark = pytest.mark.gpu

# the last two have more units than the chip has pairs of SMs: a prompt's keys are not split, one maximum runs along them
CASES = [(1, 4, [1, 1, 1], [700, 20, 1], 0, 0), (2, 6, [1], [600], 0, 0), (1, 4, [2, 1], [333, 450], 100, 4),
         (1, 16, [70, 3], [70, 400], 0, 0), (2, 4, [130], [640], 0, 0), (3, 16, [280], [660], 0, 0), (3, 16, [280], [660], 300, 3)]


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


def rising(kv_heads, group, counts, lengths, head, dtype):
    """(batch, q): along a sequence a few keys are each 2^5.4 to 2^7.8 above all before them, which is less than a prompt's
    running maximum is moved for, so that their weights are any numbers."""
    rng = np.random.default_rng(head)
    batch = Batch(rng, counts, lengths, 32, kv_heads, head, dtype)
    direction = rng.choice([-1.0, 1.0], size=head)
    for s, length in enumerate(lengths):
        for n, j in enumerate(range(2, length, 150)):
            page, place = batch.slot(s, j)
            batch.keys[page, :, place] = narrow(direction * (1.0 + 0.45 * n), dtype)
    shape = (batch.tokens, kv_heads * group)
    rows = direction * rng.uniform(8.4, 12.0, shape + (1,)) + rng.standard_normal(shape + (head,))
    return batch, narrow(rows / math.sqrt(head), dtype)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,counts,lengths,window,sinks", CASES)
def test_equal_values_come_back_as_they_are(q4b, ctx, dtype, head, kv_heads, group, counts, lengths, window, sinks):
    """sum w v / sum w with the same w in both is v.  The two sums take at most 700 weights and their joins, each addition off
    by 2^-23 at most (the products are exact): 2^-13 in all, the reciprocal and its product 2^-22 more, and half the
    distance from a value to its neighbour is 2^-12 of it in fp16 and 2^-9 in bf16, so the nearest value is the value itself."""
    batch, q = rising(kv_heads, group, counts, lengths, head, dtype)
    rng = np.random.default_rng(head + 1)
    column = narrow(rng.standard_normal((kv_heads, 1, head)) * 3 + 0.01, dtype)
    batch.values[:] = column
    want = np.broadcast_to(np.repeat(column[:, 0], group, axis=0), q.shape)
    assert (attend(q4b, ctx, batch, q, kv_heads * group, 1 / math.sqrt(head), window, sinks) == want).all()
    flat = narrow(rng.standard_normal(q.shape), dtype)   # rows that see many keys alike
    assert (attend(q4b, ctx, batch, flat, kv_heads * group, 1 / math.sqrt(head), window, sinks) == want).all()


def reference(batch, q, q_heads, scale, window, sinks, rows):
    """(mean, spread, size, relative error of a weight by its score) of some rows in 64 bits: sum w v, sum w |v - mean| and
    sum w |v|, each over sum w; an fp32 score has (head + 8) additions and products of half an fp32 eps of scale x sum |q||k|
    each, before and after the subtraction of the maximum."""
    group, shape = q_heads // batch.kv_heads, (len(rows), q_heads, batch.head)
    mean, spread, size, error = np.zeros(shape), np.zeros(shape), np.zeros(shape), np.zeros(shape[:2] + (1,))
    keys, values, q = (widen(x, batch.dtype) for x in (batch.keys, batch.values, q))
    for n, row in enumerate(rows):
        s = int(np.searchsorted(batch.begin, row, side="right")) - 1
        held = batch.table[s, :-(-int(batch.lengths[s]) // batch.page)].astype(np.int64)
        at = batch.place(s, row - int(batch.begin[s]))
        every = np.arange(at + 1)
        seen = every[(every > at - window) | (every < sinks)] if window else every
        for h in range(batch.kv_heads):
            heads = slice(h * group, (h + 1) * group)
            k, v = (x[held, h].reshape(-1, batch.head)[seen] for x in (keys, values))
            x = q[row, heads]
            score = x @ k.T * scale
            weight = np.exp(score - score.max(axis=1, keepdims=True))
            weight /= weight.sum(axis=1, keepdims=True)
            mean[n, heads], size[n, heads] = weight @ v, weight @ np.abs(v)
            spread[n, heads] = np.einsum("gk,gkd->gd", weight, np.abs(v[None] - mean[n, heads][:, None]))
            error[n, heads] = abs(scale) * (np.abs(x) @ np.abs(k).T).max(axis=1)[:, None] * (batch.head + 8) * 2.0 ** -23
    return mean, spread, size, error


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,counts,lengths,window,sinks", CASES)
def test_rows_that_one_key_dominates(q4b, ctx, dtype, head, kv_heads, group, counts, lengths, window, sinks):
    """A row's outputs are its last large key's values, nearly.

    Tolerance: the output's own rounding (half an eps of it); the weights' roundings e, half an eps at most, which move
    sum w v / sum w by sum w e (v - mean) / sum w; and, times the weighted size of the values, the weights' relative errors
    by their scores and 2^-19 for the exponential and the fp32 sums."""
    batch, q = rising(kv_heads, group, counts, lengths, head, dtype)
    scale = 1 / math.sqrt(head)
    rows = np.arange(0, batch.used, max(1, batch.used // 20))
    got = widen(attend(q4b, ctx, batch, q, kv_heads * group, scale, window, sinks), dtype)[rows]
    mean, spread, size, error = reference(batch, q, kv_heads * group, scale, window, sinks, rows)
    half = EPS[dtype] / 2
    tolerance = half * np.abs(mean) + (1 + 2 * half) * (half * spread + (2 * error + 2.0 ** -19) * size) + 2.0 ** -24
    off = np.abs(got - mean)
    assert (off <= tolerance).all(), (off / tolerance).max()
