"""Plain 64-bit forms of the paged-cache operators and the makings of small cases, shared by their tests."""
import numpy as np

EPS = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7, "f32": 2.0 ** -23}  # finfo.eps: a rounding is off by half of it at most


def narrow(values, dtype):
    """float64 -> the type's bits (round to nearest even), NaN and infinities kept."""
    values = np.asarray(values, dtype=np.float64)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return values.astype(np.float16)
    if dtype == "f32":
        return values.astype(np.float32)
    bits = values.astype(np.float32).view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7fff + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(values), np.uint16(0x7fc0), out).astype(np.uint16)


def widen(bits, dtype):
    if dtype == "bf16":
        return (np.asarray(bits).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(bits).astype(np.float64)


def storage(dtype):
    return {"f16": np.float16, "bf16": np.uint16, "f32": np.float32}[dtype]


class Batch:
    """Sequences with `counts` new tokens and `lengths` tokens in all, their pages dealt out of order."""

    def __init__(self, rng, counts, lengths, page, kv_heads, head, dtype, pad=0, spare=2):
        self.counts, self.lengths = np.asarray(counts), np.asarray(lengths)
        self.page, self.kv_heads, self.head, self.dtype = page, kv_heads, head, dtype
        self.begin = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.uint32)
        self.used = int(self.begin[-1])
        self.tokens = self.used + pad
        held = -(-self.lengths // page)
        self.stride = max(1, int(held.max())) + 1
        self.pages = int(held.sum()) + spare
        order = rng.permutation(self.pages)
        self.table = np.full((len(self.counts), self.stride), 0xfffffff0, dtype=np.uint32)  # never to be followed
        at = 0
        for s, n in enumerate(held):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.keys = narrow(rng.standard_normal((self.pages, kv_heads, page, head)), dtype)
        self.values = narrow(rng.standard_normal((self.pages, kv_heads, page, head)), dtype)

    def place(self, s, i):
        return int(self.lengths[s]) - int(self.counts[s]) + i

    def slot(self, s, j):
        return int(self.table[s, j // self.page]), j % self.page

    def upload(self, q4b, ctx, most_tokens=None):
        self.d_keys, self.d_values = ctx.to_device(self.keys), ctx.to_device(self.values)
        self.d_begin, self.d_lengths = ctx.to_device(self.begin), ctx.to_device(self.lengths.astype(np.uint32))
        self.d_table = ctx.to_device(self.table)
        cache = q4b.KVCache(keys=self.d_keys.ptr, values=self.d_values.ptr, dtype=getattr(q4b, self.dtype.upper()),
                            pages=self.pages, page_tokens=self.page, kv_heads=self.kv_heads, head_size=self.head)
        batch = q4b.TokenBatch(sequences=len(self.counts), tokens=self.tokens,
                               most_tokens=int(self.counts.max()) if most_tokens is None else most_tokens,
                               token_begin=self.d_begin.ptr, lengths=self.d_lengths.ptr, page_table=self.d_table.ptr,
                               table_stride=self.stride)
        return cache, batch


def attention_reference(batch, q, q_heads, scale, window, sinks):
    """(out, tolerance) in 64 bits, [tokens, q_heads, head]; rows of no sequence are NaN in both.

    Tolerance: the output's own rounding (half of eps x |out|); a weight's rounding to 16 bits, half of eps of each, so
    half of eps x sum w|v| / sum w; a weight's relative error from its exponent, which is the fp32 score's error --
    (head + 8) additions and products of half an fp32 eps each of scale x sum |q||k|, before and after the subtraction
    of the maximum -- and 2^-20 for the exponential and the fp32 sums, which are divided by each other (twice)."""
    head, group = batch.head, q_heads // batch.kv_heads
    eps = EPS[batch.dtype]
    out = np.full((batch.tokens, q_heads, head), np.nan)
    tolerance = np.full_like(out, np.nan)
    keys, values, q = widen(batch.keys, batch.dtype), widen(batch.values, batch.dtype), widen(q, batch.dtype)
    for s in range(len(batch.counts)):
        held = batch.table[s, :-(-int(batch.lengths[s]) // batch.page)].astype(np.int64)
        own_keys = keys[held].transpose(1, 0, 2, 3).reshape(batch.kv_heads, -1, head)      # [kv_heads, places, head]
        own_values = values[held].transpose(1, 0, 2, 3).reshape(batch.kv_heads, -1, head)
        for i in range(int(batch.counts[s])):
            row, at = int(batch.begin[s]) + i, batch.place(s, i)
            every = np.arange(at + 1)
            seen = every[(every > at - window) | (every < sinks)] if window else every
            out[row] = tolerance[row] = 0.0
            if len(seen) == 0:
                continue
            for h in range(batch.kv_heads):
                k, v = own_keys[h, seen], own_values[h, seen]
                x = q[row].reshape(batch.kv_heads, group, head)[h]
                score = x @ k.T * scale
                error = abs(scale) * (np.abs(x) @ np.abs(k).T).max(axis=1) * (head + 8) * 2.0 ** -24 * 2
                weight = np.exp(score - score.max(axis=1, keepdims=True))
                weight /= weight.sum(axis=1, keepdims=True)
                mean, spread = weight @ v, weight @ np.abs(v)
                heads = slice(h * group, (h + 1) * group)
                out[row, heads] = mean
                relative = eps / 2 + 2 * error[:, None] + 2.0 ** -19
                tolerance[row, heads] = eps / 2 * np.abs(mean) + (1 + eps) * relative * spread + 2.0 ** -24
    return out, tolerance


def rope_reference(x, positions, rotary, pairing, frequencies):
    """x [tokens, heads, head] turned, in 64 bits."""
    half = rotary // 2
    out = np.array(x, dtype=np.float64)
    if half == 0:
        return out
    angle = np.asarray(positions, dtype=np.float64)[:, None, None] * np.asarray(frequencies, dtype=np.float64)
    lower, upper = (slice(0, half), slice(half, rotary)) if pairing == "halves" else (slice(0, rotary, 2), slice(1, rotary, 2))
    a, b = out[..., lower].copy(), out[..., upper].copy()
    out[..., lower] = a * np.cos(angle) - b * np.sin(angle)
    out[..., upper] = b * np.cos(angle) + a * np.sin(angle)
    return out
