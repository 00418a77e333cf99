"""What is measured of the operators between a layer's projections and behind the lm_head.

Three operators, each in its plain form (elementary torch operations) and as the library's call:

  append  q4b_rope_append: the keys and values of new tokens go into a paged cache, keys and queries turned by their
          positions on the way
  attend  q4b_attention: causal attention of new tokens over the paged cache, grouped heads, with an optional sliding
          window behind which the first few tokens (sinks) stay visible
  sample  q4b_sample: one token per row of logits from given random numbers, by temperature, top-k, top-p and min-p

Sizes: "27b" is the attention of the 27B layer set (24 query and 4 key heads of 256, 64 of them rotary), "small" that of
the hidden-1024 set (16 query and 4 key heads of 128); the vocabulary is the lm_head's, 248,320.
"""
from __future__ import annotations

import importlib
import math

import numpy as np
import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
ITEM = {"f16": 2, "bf16": 2, "f32": 4}
GOLDEN = 0.6180339887498949


# ---- cases ------------------------------------------------------------------------------------------------------

def listed():
    big = {"q_heads": 24, "kv_heads": 4, "head": 256}
    small = {"q_heads": 16, "kv_heads": 4, "head": 128}
    append, attend, sample = {"op": "append"}, {"op": "attend"}, {"op": "sample"}
    return [
        # one chat user's next token, in fp16 as the decode projections write it
        {"name": "append one token", **append, **big, "dtype": "f16", "input": "f16", "page": 16, "sequences": 1, "new": 1,
         "context": 4095, "ragged": False, "pad": 0, "rotary": 64, "pairing": "halves", "base": 1e7},
        # a decode step of 61 users with long histories, fp32 projections, a batch padded to 64 rows
        {"name": "append 61 users", **append, **small, "dtype": "bf16", "input": "f32", "page": 32, "sequences": 61,
         "new": 1, "context": 1000003, "ragged": True, "pad": 3, "rotary": 128, "pairing": "neighbours", "base": 1e6},
        # a prompt's largest block of rows
        {"name": "append prompt 8192", **append, **big, "dtype": "bf16", "input": "bf16", "page": 64, "sequences": 1,
         "new": 8192, "context": 0, "ragged": False, "pad": 0, "rotary": 64, "pairing": "halves", "base": 1e7},
        # one user's next token after a short history: latency
        {"name": "attend one token", **attend, **big, "dtype": "f16", "page": 16, "sequences": 1, "new": 1, "context": 1024,
         "ragged": False, "pad": 0, "window": 0, "sinks": 0},
        # a decode step of 32 users, histories of 4,000 to 16,384 tokens: the cache's bytes
        {"name": "attend 32 users", **attend, **big, "dtype": "bf16", "page": 16, "sequences": 32, "new": 1,
         "context": 16383, "ragged": True, "pad": 0, "window": 0, "sinks": 0},
        # the verify step (three drafted tokens and one) of six users behind a window with sinks
        {"name": "attend verify window", **attend, **big, "dtype": "f16", "page": 64, "sequences": 6, "new": 4,
         "context": 32761, "ragged": True, "pad": 0, "window": 4096, "sinks": 4},
        # the next 511 tokens of a long prompt that is taken in pieces
        {"name": "attend piece of a prompt", **attend, **small, "dtype": "bf16", "page": 32, "sequences": 1, "new": 511,
         "context": 30001, "ragged": False, "pad": 1, "window": 0, "sinks": 0},
        # four prompts of unlike lengths in one call, with a window and sinks
        {"name": "attend prompts window", **attend, **big, "dtype": "bf16", "page": 64, "sequences": 4, "new": 4001,
         "context": 0, "ragged": True, "pad": 5, "window": 1024, "sinks": 4},
        # a prompt's largest block of rows, all of it visible
        {"name": "attend prompt 8192", **attend, **big, "dtype": "f16", "page": 64, "sequences": 1, "new": 8192,
         "context": 0, "ragged": False, "pad": 0, "window": 0, "sinks": 0},
        # one user's next token, every rule on
        {"name": "sample one row", **sample, "dtype": "f32", "rows": 1, "vocab": 248320, "rules": "tkpm", "spread": 2.0},
        # 33 users with fp16 logits, top-p alone, over logits with a fat tail
        {"name": "sample 33 rows top-p", **sample, "dtype": "f16", "rows": 33, "vocab": 248320, "rules": "tp", "spread": 3.0},
        # many rows (drafts, best of n), the whole distribution
        {"name": "sample 256 rows", **sample, "dtype": "f32", "rows": 256, "vocab": 248320, "rules": "t", "spread": 2.5},
    ]


def draw(rng):
    def log_int(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        vocab = log_int(200, 300000)
        rules = rng.choice(["tkpm", "tkpm", "tk", "tp", "tm", "t", "kp", "p"])
        return {"op": op, "dtype": rng.choice(["f32", "f16", "bf16"]), "rows": log_int(1, max(1, min(400, 60000000 // vocab))),
                "vocab": vocab, "rules": rules, "spread": rng.choice([0.5, 1.0, 2.0, 3.0])}
    head = rng.choice([64, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"op": op, "q_heads": kv_heads * rng.choice([1, 2, 4, 6, 8]), "kv_heads": kv_heads, "head": head,
            "dtype": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 32, 64, 128]), "ragged": rng.random() < 0.6,
            "pad": rng.choice([0, 0, 1, 7])}
    if op == "append":
        sequences = log_int(1, 100)
        return {**case, "input": rng.choice(["f16", "bf16", "f32"]), "sequences": sequences,
                "new": log_int(1, max(1, 6000 // sequences)), "context": log_int(1, 1500000), "rotary": rng.choice([head, head // 2, 32]),
                "pairing": rng.choice(["halves", "neighbours"]), "base": rng.choice([1e4, 1e6, 1e7])}
    kind = rng.choice(["decode", "verify", "prompt", "piece"])
    if kind in ("decode", "verify"):
        sequences = log_int(1, 64)
        new = 1 if kind == "decode" else rng.randint(2, 8)
        context = log_int(1, max(2, min(60000, 400000 * 1024 // (kv_heads * head * sequences) // 2)))
    elif kind == "prompt":
        sequences, context = rng.randint(1, 4), 0
        new = log_int(2, 6000 // sequences)
    else:
        sequences, new, context = rng.randint(1, 3), log_int(9, 700), log_int(16, 12000)
    windowed = rng.random() < 0.5
    return {**case, "sequences": sequences, "new": new, "context": context,
            "window": log_int(1, 5000) if windowed else 0, "sinks": rng.choice([0, 1, 4, 17, 64]) if windowed else 0}


def layout(case):
    """(new tokens, tokens in the cache afterwards) of every sequence: whole numbers by the case alone."""
    count = case["sequences"]
    part = (np.arange(1, count + 1) * GOLDEN % 1.0) if case["ragged"] else np.ones(count)
    part = 0.25 + 0.75 * part if case["ragged"] else part
    context = np.floor(case["context"] * part).astype(np.int64)
    # where there is no history the new tokens themselves are ragged
    new = np.maximum(1, np.floor(case["new"] * part)).astype(np.int64) if case["context"] == 0 or case["op"] == "append" \
        else np.full(count, case["new"], dtype=np.int64)
    if case["ragged"]:
        new[0], context[0] = case["new"], case["context"]
    return new, context + new


def visible(case):
    """(pairs of a new token and a token that it sees, cached tokens that any new one sees), over all sequences."""
    new, length = layout(case)
    pairs = keys = 0
    for n, total in zip(new.tolist(), length.tolist()):
        at = np.arange(total - n, total, dtype=np.int64)
        if case["window"]:
            first = np.maximum(0, at - case["window"] + 1)
            pairs += int((at - first + 1 + np.minimum(first, case["sinks"])).sum())
            first0 = int(first[0])
            keys += total - first0 + min(first0, case["sinks"])
        else:
            pairs += int((at + 1).sum())
            keys += total
    return pairs, keys


def work(case):
    if case["op"] == "sample":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * ITEM[case["dtype"]] + case["rows"] * 28, "flops": 4 * cells}
    new, length = layout(case)
    tokens, head = int(new.sum()), case["head"]
    if case["op"] == "append":
        values = tokens * (case["q_heads"] + 2 * case["kv_heads"]) * head
        turned = tokens * (case["q_heads"] + case["kv_heads"]) * case["rotary"]
        return {"bytes": values * (ITEM[case["input"]] + 2) + tokens * 4, "flops": 3 * turned}
    pairs, keys = visible(case)
    return {"bytes": 2 * 2 * tokens * case["q_heads"] * head + 2 * 2 * keys * case["kv_heads"] * head + 4 * keys // case["page"],
            "flops": 4 * pairs * case["q_heads"] * head}


# ---- inputs -----------------------------------------------------------------------------------------------------

def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device)
    g.manual_seed(int(seed))

    def normal(*shape, dtype=torch.float32):
        out = torch.empty(shape, dtype=dtype, device=device)
        return out.normal_(generator=g)

    def uniform(*shape):
        return torch.rand(shape, generator=g, device=device)

    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        logits = normal(rows, vocab) * case["spread"]
        # a model's few likely tokens
        likely = torch.randint(0, vocab, (rows, min(vocab, 24)), generator=g, device=device)
        logits.scatter_add_(1, likely, 9.0 * uniform(rows, likely.shape[1]) + case["spread"])
        state = {"case": case, "logits": logits.to(DTYPES[case["dtype"]]), "uniform": uniform(rows),
                 "tokens": torch.zeros(rows, dtype=torch.int32, device=device),
                 "probability": torch.zeros(rows, dtype=torch.float32, device=device)}
        if "t" in case["rules"]:  # one row in eight is greedy
            state["temperature"] = torch.where(uniform(rows) < 0.125, 0.0, 0.5 + uniform(rows))
        if "k" in case["rules"]:  # one row in four has it off
            state["top_k"] = torch.where(uniform(rows) < 0.25, 0, torch.randint(1, 200, (rows,), generator=g, device=device)).to(torch.int32)
        if "p" in case["rules"]:
            state["top_p"] = torch.where(uniform(rows) < 0.125, 1.0, 0.5 + 0.499 * uniform(rows))
        if "m" in case["rules"]:
            state["min_p"] = torch.where(uniform(rows) < 0.25, 0.0, 0.2 * uniform(rows))
        return state

    new, length = layout(case)
    sequences, page, kv_heads, head = case["sequences"], case["page"], case["kv_heads"], case["head"]
    tokens = int(new.sum())
    rows = tokens + case["pad"]
    dtype = DTYPES[case["dtype"]]
    held = -(-length // page)                      # pages of every sequence
    width = int(held.max())
    cpu = torch.Generator().manual_seed(int(seed))
    if case["op"] == "attend":
        pages = int(held.sum()) + 3
        order = torch.randperm(pages, generator=cpu)
        begin = np.cumsum(held) - held
        table = torch.zeros(sequences, width, dtype=torch.int64)
        at = torch.arange(width)[None, :] + torch.from_numpy(begin)[:, None]
        inside = torch.arange(width)[None, :] < torch.from_numpy(held)[:, None]
        table = torch.where(inside, order[torch.where(inside, at, 0)], 0)
    else:  # only the pages that the new tokens fall into are there; the rest of a long history is not touched
        first = (length - new) // page
        touched = held - first
        pages = int(touched.sum()) + 3
        order = torch.randperm(pages, generator=cpu)
        begin = np.cumsum(touched) - touched
        column = torch.arange(width)[None, :] - torch.from_numpy(first)[:, None]
        inside = (column >= 0) & (column < torch.from_numpy(touched)[:, None])
        table = torch.where(inside, order[torch.where(inside, column + torch.from_numpy(begin)[:, None], 0)], 0)
    state = {"case": case, "tokens": tokens, "rows": rows, "most": int(new.max()), "pages": pages,
             "keys": normal(pages, kv_heads, page, head, dtype=dtype), "values": normal(pages, kv_heads, page, head, dtype=dtype),
             "token_begin": torch.from_numpy(np.concatenate([[0], np.cumsum(new)])).to(torch.int32).to(device),
             "lengths": torch.from_numpy(length).to(torch.int32).to(device), "table": table.to(torch.int32).to(device)}
    if case["op"] == "append":
        source = DTYPES[case["input"]]
        state["q"] = normal(rows, case["q_heads"] * head, dtype=source)
        state["k"] = normal(rows, kv_heads * head, dtype=source)
        state["v"] = normal(rows, kv_heads * head, dtype=source)
    else:
        # queries that pick tokens out: scores of a few units
        state["q"] = (normal(rows, case["q_heads"] * head) * 1.5).to(dtype)
    # padded rows keep what they hold
    state["out"] = normal(rows, case["q_heads"] * head, dtype=dtype)
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------

def places(state):
    """Of every new token: its sequence, and its position in it."""
    begin, rows = state["token_begin"].long(), torch.arange(state["tokens"], device="cuda")
    sequence = torch.searchsorted(begin, rows, right=True) - 1
    new = begin[1:] - begin[:-1]
    return sequence, state["lengths"].long()[sequence] - new[sequence] + rows - begin[sequence], rows - begin[sequence]


def plain_append(state):
    case, tokens = state["case"], state["tokens"]
    head, rotary, page = case["head"], case["rotary"], case["page"]
    sequence, position, _ = places(state)
    # angles in 64 bits: a position of a million radians leaves 32 bits with two digits
    power = torch.arange(rotary // 2, dtype=torch.float64, device="cuda") * (-2.0 / rotary)
    angle = position.double()[:, None] * torch.pow(torch.tensor(case["base"], dtype=torch.float64, device="cuda"), power)
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]

    def turned(x):
        x = x[:tokens].float().view(tokens, -1, head)
        part, rest = x[..., :rotary], x[..., rotary:]
        if case["pairing"] == "halves":
            a, b = part[..., :rotary // 2], part[..., rotary // 2:]
            part = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([part, rest], -1).to(state["keys"].dtype)

    state["out"][:tokens] = turned(state["q"]).view(tokens, -1)
    where = state["table"][sequence, position // page].long()
    state["keys"][where, :, position % page] = turned(state["k"])
    state["values"][where, :, position % page] = state["v"][:tokens].view(tokens, -1, head).to(state["values"].dtype)
    return {"q": state["out"], "keys": state["keys"], "values": state["values"]}


def plain_attend(state):
    case, tokens = state["case"], state["tokens"]
    head, kv_heads, page = case["head"], case["kv_heads"], case["page"]
    group, sequences, most = case["q_heads"] // kv_heads, case["sequences"], state["most"]
    sequence, position, index = places(state)
    width = state["table"].shape[1] * page

    def gathered(pool):  # [sequences][kv_heads][width][head]
        return pool[state["table"].long()].transpose(1, 2).reshape(sequences, kv_heads, width, head).float()

    # the pages hold anything behind a sequence's end
    inside = (torch.arange(width, device="cuda")[None, :] < state["lengths"][:, None])[:, None, :, None]
    keys = torch.where(inside, gathered(state["keys"]), 0.0)
    values = torch.where(inside, gathered(state["values"]), 0.0)
    q = torch.zeros(sequences, most, kv_heads, group, head, device="cuda")
    q[sequence, index] = state["q"][:tokens].float().view(tokens, kv_heads, group, head)
    at = torch.full((sequences, most), -1, dtype=torch.int64, device="cuda")
    at[sequence, index] = position
    q = q.permute(0, 2, 3, 1, 4).reshape(sequences, kv_heads, group * most, head)
    score = torch.matmul(q, keys.transpose(2, 3)) * (1.0 / math.sqrt(head))
    key = torch.arange(width, device="cuda")
    seen = key <= at[..., None]
    if case["window"]:
        seen &= (key > at[..., None] - case["window"]) | (key < case["sinks"])
    score = score.view(sequences, kv_heads, group, most, width).masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top > -math.inf, top, 0.0)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(sequences, kv_heads, group * most, width), values)
    out = out.view(sequences, kv_heads, group, most, head) / torch.where(total > 0, total, 1.0)
    out = out.permute(0, 3, 1, 2, 4)[sequence, index]
    state["out"][:tokens] = out.reshape(tokens, -1).to(state["out"].dtype)
    return state["out"]


def plain_sample(state):
    logits = state["logits"].float()
    logits = torch.where(torch.isnan(logits), -math.inf, logits)
    rows, vocab = logits.shape
    ones = torch.ones(rows, dtype=torch.float64, device="cuda")
    temperature = state["temperature"].double() if "temperature" in state else ones
    best, first = logits.max(1, keepdim=True)
    first = (logits == best).to(torch.uint8).argmax(1)
    greedy = temperature <= 0
    # weights and their sums in 64 bits: a sum's last digits decide between neighbours of a border
    scale = torch.where(greedy, 1.0, 1.0 / torch.where(greedy, 1.0, temperature))[:, None]
    weight = torch.where(logits == best, 1.0, ((logits.double() - best) * scale).exp())
    order = torch.sort(logits, dim=1, descending=True, stable=True).indices
    sorted_weight = weight.gather(1, order)
    running = sorted_weight.cumsum(1)
    rank = torch.arange(vocab, device="cuda")[None, :]
    k = state["top_k"].long() if "top_k" in state else torch.zeros(rows, dtype=torch.int64, device="cuda")
    k = torch.where((k <= 0) | (k > vocab), vocab, k)[:, None]
    keep = rank < k
    if "top_p" in state:
        p = state["top_p"].double()[:, None]
        keep &= (p >= 1) | (running - sorted_weight < p * running.gather(1, k - 1)) | (rank == 0)
    if "min_p" in state:
        keep &= sorted_weight >= state["min_p"].double()[:, None]
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    weight = weight * kept
    running = weight.cumsum(1)
    total = running[:, -1:]
    token = (running <= state["uniform"].double()[:, None] * total).sum(1)
    last = vocab - 1 - kept.flip(1).to(torch.uint8).argmax(1)
    token = torch.where(greedy, first, torch.minimum(token, last))
    chance = torch.where(greedy[:, None], 1.0, weight.gather(1, token[:, None]) / total)[:, 0]
    state["tokens"].copy_(token)
    state["probability"].copy_(chance)
    return {"tokens": state["tokens"], "probability": state["probability"]}


# ---- the library's calls ----------------------------------------------------------------------------------------

_context = None


def context():
    """The program's context on the GPU, opened once."""
    global _context
    if _context is None:
        package = importlib.import_module("cpu-llms-in-c_b200")
        _context = (package, package.Q4Context(torch.cuda.current_device()))
    return _context


def handles(state):
    """The descriptors of a program's cache and batch: built once, like the buffers that they name."""
    if "handles" not in state:
        package, _ = context()
        case = state["case"]
        code = {"f16": package.F16, "bf16": package.BF16}[case["dtype"]]
        cache = package.KVCache(keys=state["keys"].data_ptr(), values=state["values"].data_ptr(), dtype=code, pages=state["pages"],
                                page_tokens=case["page"], kv_heads=case["kv_heads"], head_size=case["head"])
        batch = package.TokenBatch(sequences=case["sequences"], tokens=state["rows"], most_tokens=state["most"],
                                   token_begin=state["token_begin"].data_ptr(), lengths=state["lengths"].data_ptr(),
                                   page_table=state["table"].data_ptr(), table_stride=state["table"].shape[1])
        rope = package.Rope(rotary_size=case["rotary"], base=case["base"],
                            pairing=package.ROPE_HALVES if case["pairing"] == "halves" else package.ROPE_NEIGHBOURS) \
            if case["op"] == "append" else None
        state["handles"] = (cache, batch, rope)
    return state["handles"]


def own_append(state):
    package, ctx = context()
    case = state["case"]
    cache, batch, rope = handles(state)
    code = {"f16": package.F16, "bf16": package.BF16, "f32": package.F32}[case["input"]]
    ctx.rope_append(cache, batch, rope, state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(), code,
                    case["q_heads"], state["out"].data_ptr())
    return {"q": state["out"], "keys": state["keys"], "values": state["values"]}


def own_attend(state):
    _, ctx = context()
    case = state["case"]
    cache, batch, _ = handles(state)
    ctx.attention(cache, batch, state["q"].data_ptr(), case["q_heads"], state["out"].data_ptr(), scale=1.0 / math.sqrt(case["head"]),
                  window=case["window"], sinks=case["sinks"])
    return state["out"]


def own_sample(state):
    package, ctx = context()
    case = state["case"]
    code = {"f16": package.F16, "bf16": package.BF16, "f32": package.F32}[case["dtype"]]
    rules = {name: state[name].data_ptr() for name in ("temperature", "top_k", "top_p", "min_p") if name in state}
    ctx.sample(state["logits"].data_ptr(), code, case["rows"], case["vocab"], state["uniform"].data_ptr(),
               state["tokens"].data_ptr(), probability_ptr=state["probability"].data_ptr(), **rules)
    return {"tokens": state["tokens"], "probability": state["probability"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": own_append, "attend": own_attend, "sample": own_sample}[op](state)
    return {"append": plain_append, "attend": plain_attend, "sample": plain_sample}[op](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        tokens, chances = [], []
        for r in range(rows):
            logit = np.nan_to_num(state["logits"][r].double().cpu().numpy(), nan=-np.inf, posinf=np.inf, neginf=-np.inf)
            setting = {name: float(state[name][r]) for name in ("temperature", "top_k", "top_p", "min_p") if name in state}
            heat = setting.get("temperature", 1.0)
            if heat <= 0:
                tokens.append(int(logit.argmax()))
                chances.append(1.0)
                continue
            weight = np.exp((logit - logit.max()) / heat)
            order = np.argsort(-logit, kind="stable")
            k = int(setting.get("top_k", 0)) or vocab
            order = order[:min(k, vocab)]
            ordered = weight[order]
            running = np.cumsum(ordered)
            count = len(order)
            if setting.get("top_p", 1.0) < 1:
                # the fewest tokens whose sum reaches the share
                count = int(np.searchsorted(running, setting["top_p"] * running[-1], side="left")) + 1
            ordered = ordered[:count]
            count = max(1, int((ordered >= setting.get("min_p", 0.0)).sum()))
            chosen = np.sort(order[:count])
            running = np.cumsum(weight[chosen])
            at = min(int(np.searchsorted(running, float(state["uniform"][r]) * running[-1], side="right")), count - 1)
            tokens.append(int(chosen[at]))
            chances.append(float(weight[chosen[at]] / running[-1]))
        return {"tokens": torch.tensor(tokens, dtype=torch.int32), "probability": torch.tensor(chances, dtype=torch.float64)}
    new, length = layout(case)
    begin = np.cumsum(new) - new
    head, kv_heads, page = case["head"], case["kv_heads"], case["page"]
    table = state["table"].long()
    if case["op"] == "append":
        half = case["rotary"] // 2
        out, keys, values = state["out"].double(), state["keys"].double(), state["values"].double()
        for s in range(case["sequences"]):
            rows = slice(int(begin[s]), int(begin[s] + new[s]))
            at = torch.arange(int(length[s] - new[s]), int(length[s]), device="cuda")
            turn = torch.tensor([case["base"] ** (-i / half) for i in range(half)], dtype=torch.float64, device="cuda")
            unit = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"), at.double()[:, None] * turn)[:, None, :]
            for name, heads in (("q", case["q_heads"]), ("k", kv_heads)):
                x = state[name][rows].double().view(-1, heads, head).clone()
                if case["pairing"] == "halves":
                    real, imaginary = slice(0, half), slice(half, 2 * half)
                else:
                    real, imaginary = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
                z = torch.complex(x[..., real], x[..., imaginary]) * unit
                x[..., real], x[..., imaginary] = z.real, z.imag
                if name == "q":
                    out[rows] = x.flatten(1)
                else:
                    keys[table[s, at // page], :, at % page] = x
            values[table[s, at // page], :, at % page] = state["v"][rows].double().view(-1, kv_heads, head)
        return {"q": out, "keys": keys, "values": values}
    out = state["out"].double()
    group = case["q_heads"] // kv_heads
    for s in range(case["sequences"]):
        total, n = int(length[s]), int(new[s])
        held = table[s, :-(-total // page)]
        for h in range(kv_heads):
            keys = state["keys"][held, h].reshape(-1, head)[:total].double()
            values = state["values"][held, h].reshape(-1, head)[:total].double()
            for first in range(0, n, 1024):
                count = min(1024, n - first)
                rows = slice(int(begin[s]) + first, int(begin[s]) + first + count)
                q = state["q"][rows].double().view(count, kv_heads, group, head)[:, h].reshape(count * group, head)
                at = torch.arange(total - n + first, total - n + first + count, device="cuda").repeat_interleave(group)[:, None]
                key = torch.arange(total, device="cuda")[None, :]
                hidden = key > at
                if case["window"]:
                    hidden = hidden | ((key <= at - case["window"]) & (key >= case["sinks"]))
                share = torch.softmax((q @ keys.T / math.sqrt(head)).masked_fill(hidden, -math.inf), -1)
                out[rows].view(count, kv_heads, group, head)[:, h] = (share @ values).view(count, group, head)
    return out
