"""Attention over contexts of 130,000 to 16 million tokens: no chain of additions may get so long that it loses what it adds.
Matrix instructions cut a running sum off instead of rounding it.  The page table names a few pages again and again, so the
cache is small and the definition's sums are over the pages' tokens, each as often as it is seen."""
import numpy as np
import pytest

from cache_cases import EPS, narrow, storage, widen

pytestmark = pytest.mark.gpu

PAGE, PAGES = 1024, 4


@pytest.fixture(scope="module")
def ctx(q4b):
    context = q4b.Q4Context(0)
    yield context
    context.close()


class Long:
    """`sequences` sequences of `new` new tokens behind a context that the same four pages make up."""

    def __init__(self, q4b, ctx, dtype, head, kv_heads, group, sequences, new, length, equal, seed=1):
        rng = np.random.default_rng(seed)
        self.q4b, self.ctx, self.dtype, self.head, self.kv_heads, self.group = q4b, ctx, dtype, head, kv_heads, group
        self.sequences, self.new, self.length = sequences, new, length
        pool = (PAGES, kv_heads, PAGE, head)
        self.keys = narrow(rng.standard_normal(pool), dtype)
        self.values = narrow(rng.standard_normal(pool) + 0.5, dtype)
        if equal:
            self.values[:] = narrow(rng.standard_normal((1, kv_heads, 1, head)) * 3 + 0.01, dtype)
        self.q = narrow(rng.standard_normal((sequences * new, kv_heads * group, head)) * 0.7, dtype)
        self.columns = -(-length // PAGE)
        self.table = np.broadcast_to(np.arange(self.columns, dtype=np.uint32) % PAGES, (sequences, self.columns)).copy()
        self.scale = head ** -0.5

    def run(self, most_tokens):
        q4b, ctx = self.q4b, self.ctx
        held = [ctx.to_device(x) for x in (self.keys, self.values, self.table, self.q, np.full(self.sequences, self.length, np.uint32),
                                           np.arange(self.sequences + 1, dtype=np.uint32) * self.new)]
        out = ctx.alloc(self.q.nbytes)
        cache = q4b.KVCache(keys=held[0].ptr, values=held[1].ptr, dtype=getattr(q4b, self.dtype.upper()), pages=PAGES, page_tokens=PAGE,
                            kv_heads=self.kv_heads, head_size=self.head)
        batch = q4b.TokenBatch(sequences=self.sequences, tokens=len(self.q), most_tokens=most_tokens, token_begin=held[5].ptr,
                               lengths=held[4].ptr, page_table=held[2].ptr, table_stride=self.columns)
        ctx.attention(cache, batch, held[3].ptr, self.kv_heads * self.group, out.ptr, self.scale)
        ctx.sync()
        return out.download(storage(self.dtype), self.q.shape)

    def check_equal(self, got):
        """Every chain loses less than a quarter of the half step between a value and its neighbour, see the kernels."""
        want = np.broadcast_to(np.repeat(self.values[0, :, 0], self.group, axis=0), self.q.shape)
        assert (got == want).all()

    def check_rows(self, got, rows):
        """Tolerance: the output's own rounding; the weights' roundings, half an eps at most, against the values' spread; and,
        times the weighted size of the values, the weights' relative errors by their fp32 scores ((head + 8) additions and
        products, before and after the subtraction of the maximum), 2^-19 for the exponential and the rounded additions, and
        an eighth of an eps for what chains of products lose."""
        keys, values, q = (widen(x, self.dtype) for x in (self.keys, self.values, self.q))
        half = EPS[self.dtype] / 2
        for row in rows:
            places = np.arange(self.length - self.new + row % self.new + 1)
            times = np.bincount(places // PAGE % PAGES * PAGE + places % PAGE, minlength=PAGES * PAGE)
            for h in range(self.kv_heads):
                heads = slice(h * self.group, (h + 1) * self.group)
                k, v = (x[:, h].reshape(-1, self.head) for x in (keys, values))
                score = q[row, heads] @ k.T * self.scale
                weight = np.exp(score - score.max(axis=1, keepdims=True)) * times
                weight /= weight.sum(axis=1, keepdims=True)
                mean, size = weight @ v, weight @ np.abs(v)
                spread = np.stack([w @ np.abs(v - m) for w, m in zip(weight, mean)])
                error = self.scale * (np.abs(q[row, heads]) @ np.abs(k).T).max(axis=1)[:, None] * (self.head + 8) * 2.0 ** -23
                tolerance = half * np.abs(mean) + (1 + 2 * half) * (half * spread + (2 * error + 2.0 ** -19 + half / 4) * size)
                off = np.abs(widen(got[row, heads], self.dtype) - mean)
                assert (off <= tolerance).all(), (row, h, (off / tolerance).max())


# kv_heads, group, sequences, new tokens, length: prompts whose keys are not split over a cluster (more units than pairs of
# SMs) and that are; single tokens of many users, a unit to a thread block; one user, whose heads are cut into shares
SHAPES = [(3, 16, 1, 280, 2 ** 17 + 17), (1, 6, 1, 40, 2 ** 20 + 5), (2, 4, 150, 1, 2 ** 20 + 17), (1, 16, 150, 1, 2 ** 19 + 3),
          (1, 4, 1, 1, 2 ** 24 + 9), (2, 8, 1, 2, 2 ** 24)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 128, 256])
@pytest.mark.parametrize("kv_heads,group,sequences,new,length", SHAPES)
def test_equal_values_over_long_contexts(q4b, ctx, dtype, head, kv_heads, group, sequences, new, length):
    case = Long(q4b, ctx, dtype, head, kv_heads, group, sequences, new, length, equal=True)
    case.check_equal(case.run(new))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("head", [64, 256])
@pytest.mark.parametrize("kv_heads,group,sequences,new,length", SHAPES)
def test_long_contexts(q4b, ctx, dtype, head, kv_heads, group, sequences, new, length):
    case = Long(q4b, ctx, dtype, head, kv_heads, group, sequences, new, length, equal=False)
    rows = sorted({0, len(case.q) // 2, len(case.q) - 1})
    got = case.run(new)
    case.check_rows(got, rows)
    assert (case.run(new) == got).all()


def test_lengths_around_a_fold(q4b, ctx):
    """A prompt of bf16 folds its sums every 65,536 keys, one of fp16 every 8,192: just below, at and behind that."""
    for dtype, fold in (("f16", 8192), ("bf16", 65536)):
        for length in (fold, fold + 1, 2 * fold, 2 * fold + 129):
            case = Long(q4b, ctx, dtype, 64, 3, 16, 1, 280, length, equal=True)
            case.check_equal(case.run(280))
            case = Long(q4b, ctx, dtype, 128, 3, 16, 1, 280, length, equal=False)
            case.check_rows(case.run(280), [0, 279])


@pytest.mark.parametrize("most_tokens", [300, 1])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_an_infinity_at_the_end_of_a_long_context(q4b, ctx, dtype, most_tokens):
    """The last row alone sees it: its tile is gone through key by key, the others' rows are what they were."""
    case = Long(q4b, ctx, dtype, 64, 3, 16, 1, 280 if most_tokens > 1 else 3, 2 ** 17 + 17, equal=True)
    case.table[0, -1] = PAGES - 1                      # the last page is nobody else's
    case.table[0, :-1] = np.arange(case.columns - 1) % (PAGES - 1)
    case.values[PAGES - 1, :, (case.length - 1) % PAGE, ::3] = narrow(np.array(np.inf), dtype)
    got, want = case.run(most_tokens), np.repeat(case.values[0, :, 0], case.group, axis=0)
    assert (got[:-1] == want).all()
    assert not np.isfinite(widen(got[-1][:, ::3], dtype)).any()
    assert (got[-1] == want)[:, np.arange(64) % 3 != 0].all()


def test_a_context_that_takes_longer_than_one_wait(q4b, ctx):
    """268 million tokens: between a unit's first and its masked last tile pass more clocks than a bounded wait lasts, and the
    warp that looks at the last tile's values waits all that time."""
    case = Long(q4b, ctx, "bf16", 64, 3, 16, 1, 280, 2 ** 28 + 17, equal=True)
    case.check_equal(case.run(280))


def test_two_contexts_fold_at_once(q4b):
    """Each lends places of its own; their thread blocks share the chip."""
    import threading
    failures = []

    def work(seed):
        try:
            with q4b.Q4Context(0) as own:
                for shape in ((3, 16, 1, 280, 2 ** 17 + 17), (1, 6, 1, 40, 2 ** 20 + 5), (2, 4, 150, 1, 2 ** 20 + 17)):
                    case = Long(q4b, own, "f16", 64, *shape, equal=True, seed=seed)
                    for _ in range(3):
                        case.check_equal(case.run(shape[3]))
        except BaseException as error:  # noqa: BLE001 -- told to the test
            failures.append(error)
    threads = [threading.Thread(target=work, args=(seed,)) for seed in (31, 32)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failures, failures


def test_recorded_calls_that_fold(q4b, ctx):
    """Two graphs share the workspace and its places; the lengths move between replays, across and back behind a fold."""
    runs = []
    for shape in ((3, 16, 1, 280, 40_000), (1, 16, 150, 1, 2 ** 17)):
        case = Long(q4b, ctx, "f16", 64, *shape, equal=True)
        case.run(shape[3])
        held = [ctx.to_device(x) for x in (case.keys, case.values, case.table, case.q, np.full(case.sequences, case.length, np.uint32),
                                           np.arange(case.sequences + 1, dtype=np.uint32) * case.new)]
        out = ctx.alloc(case.q.nbytes)
        cache = q4b.KVCache(keys=held[0].ptr, values=held[1].ptr, dtype=q4b.F16, pages=PAGES, page_tokens=PAGE,
                            kv_heads=case.kv_heads, head_size=64)
        batch = q4b.TokenBatch(sequences=case.sequences, tokens=len(case.q), most_tokens=case.new, token_begin=held[5].ptr,
                               lengths=held[4].ptr, page_table=held[2].ptr, table_stride=case.columns)
        ctx.graph_begin()
        ctx.attention(cache, batch, held[3].ptr, case.kv_heads * case.group, out.ptr, case.scale)
        runs.append((case, held, out, ctx.graph_end()))
    for length in (40_000, 5_000, 8_193, 300, 39_999):
        for case, held, out, graph in runs:
            held[4].upload(np.full(case.sequences, length * (case.length // 40_000), np.uint32))
            graph.launch()
            graph.launch()
            case.check_equal(out.download(np.float16, case.q.shape))
    ctx.sync()
