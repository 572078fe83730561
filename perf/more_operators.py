"""Timed cases of the operators that serve and judge many continuations of a prompt (``llm_accelerator_b200.paged``).

A prompt is forked into continuations that are decoded together.  Their queries
attend to the prompt's keys, which they share, once for all of them
(``SharedAttention``), or, where the texts grow long, to a sliding window and the
first few tokens (``Attention`` with ``sinks``); the tokens that come out, and given
ones, are judged by their log probabilities, with the entropy and the likeliest
alternatives at each place (``TokenLogprobs``).

Each case has a plain form in elementary torch operations, in 32 bits and rounded
once, and ``exact`` gives the values of the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoded token of a text that has outgrown its window: latency is all there is
        {"name": "sinks one token", "op": "sinks", "seqs": 1, "max_q": 1, "max_ctx": 4500, "window": 1024, "sinks": 4,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": False, "spread": 1},
        # batched decode at contexts of all lengths, most of them past the window
        {"name": "sinks decode batch", "op": "sinks", "seqs": 64, "max_q": 1, "max_ctx": 8704, "window": 2048,
         "sinks": 4, "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": True,
         "spread": 2},
        # one serving step that mixes decodes and prompt chunks, seven query heads a key head, odd sizes
        {"name": "sinks mixed chunks", "op": "sinks", "seqs": 24, "max_q": 700, "max_ctx": 4500, "window": 777,
         "sinks": 37, "q_heads": 28, "kv_heads": 4, "dim": 64, "page": 32, "dtype": "f16", "ragged": True,
         "spread": 3},
        # a long prompt's last large chunk through a window
        {"name": "sinks long chunk", "op": "sinks", "seqs": 1, "max_q": 8192, "max_ctx": 16384, "window": 4096,
         "sinks": 64, "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": False,
         "spread": 4},
        # the first steps of a conversation that was branched once
        {"name": "shared two", "op": "shared", "groups": 1, "seqs": 2, "max_q": 1, "max_prefix": 256, "max_own": 20,
         "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": False, "spread": 5},
        # four prompts with a few tokens of a speculative step each, seven query heads a key head
        {"name": "shared speculative", "op": "shared", "groups": 4, "seqs": 21, "max_q": 5, "max_prefix": 2500,
         "max_own": 333, "q_heads": 28, "kv_heads": 4, "dim": 64, "page": 32, "dtype": "f16", "ragged": True,
         "spread": 6},
        # sampling of many continuations of a few prompts
        {"name": "shared prompts", "op": "shared", "groups": 12, "seqs": 48, "max_q": 1, "max_prefix": 4096,
         "max_own": 256, "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": True,
         "spread": 7},
        # sampling of many continuations of one long prompt
        {"name": "shared one prompt", "op": "shared", "groups": 1, "seqs": 64, "max_q": 1, "max_prefix": 8192,
         "max_own": 512, "q_heads": 16, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "ragged": True,
         "spread": 8},
        # the next token of one sequence, with the alternative that came second
        {"name": "logprobs one row", "op": "logprobs", "rows": 1, "vocab": 151936, "pad": 0, "dtype": "f32", "top": 2,
         "masked": 0.0},
        # tokens of a small vocabulary of which a grammar allows some, rows cut from a padded product
        {"name": "logprobs small vocabulary", "op": "logprobs", "rows": 700, "vocab": 4099, "pad": 29, "dtype": "f16",
         "top": 0, "masked": 0.3},
        # a decode step's rows with the usual number of alternatives
        {"name": "logprobs decode batch", "op": "logprobs", "rows": 64, "vocab": 151936, "pad": 0, "dtype": "f32",
         "top": 20, "masked": 0.0},
        # a prompt's tokens
        {"name": "logprobs prompt", "op": "logprobs", "rows": 2048, "vocab": 151936, "pad": 0, "dtype": "bf16",
         "top": 5, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sinks", "shared", "logprobs"])
    if op == "logprobs":
        vocab, dtype = _log(rng, 256, 262144), rng.choice(["bf16", "f16", "f32"])
        most = 2048 * 151936 // (2 if dtype == "f32" else 1) // vocab
        return {"op": op, "rows": _log(rng, 1, min(8192, most)), "vocab": vocab,
                "pad": rng.choice([0, 0, rng.randrange(1, 128)]), "dtype": dtype,
                "top": rng.choice([0, 1, 5, 20, 32]), "masked": rng.choice([0.0, 0.0, 0.5])}
    dim = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 8])
    case = {"op": op, "q_heads": kv * rng.choice([1, 2, 3, 4, 7, 8]), "kv_heads": kv, "dim": dim,
            "page": rng.choice([16, 32, 64, 128]), "dtype": rng.choice(["bf16", "f16"]), "ragged": rng.random() < 0.7,
            "spread": rng.randrange(1 << 20)}
    heads = case["q_heads"]
    seqs = _log(rng, 1 if op == "sinks" else 2, 64)
    if op == "sinks":
        max_q = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        before = _log(rng, 1, 16384)
    else:
        max_q = 1 if rng.random() < 0.6 else _log(rng, 2, 32)
        before = _log(rng, 64, 16384)
    # the padded score matrix and the gathered cache stay below the largest listed cases'
    while seqs > 2 and (seqs * heads * max_q * (max_q + before) > 1 << 30 or
                        seqs * kv * (max_q + before) * dim > 1 << 28):
        seqs //= 2
    while seqs * heads * max_q * (max_q + before) > 1 << 30:
        max_q = max(1, max_q // 2)
        before = max(1, before // 2)
    if op == "sinks":
        return {**case, "seqs": seqs, "max_q": max_q, "max_ctx": max_q + before, "window": _log(rng, 16, 4096),
                "sinks": _log(rng, 1, 128)}
    longest = max(case["page"], before)
    return {**case, "seqs": seqs, "groups": rng.randint(1, max(1, seqs // 2)), "max_q": max_q, "max_prefix": longest,
            "max_own": max_q + _log(rng, 1, max(1, min(1024, longest // 2)))}


def _spread(rng, n, most, ragged):
    """n lengths up to `most`: all of them `most`, or spread over the logarithm, the first the longest."""
    return [most if i == 0 or not ragged else max(1, min(most, _log(rng, 1, most))) for i in range(n)]


def _lens(case):
    """(new tokens, tokens stored once they are in) of every sequence."""
    rng = random.Random(case["spread"])
    new = _spread(rng, case["seqs"], case["max_q"], case["ragged"])
    if case["op"] == "shared":
        prefix, members = _groups(case)
        more = _spread(rng, case["seqs"], case["max_own"] - case["max_q"], case["ragged"]) \
            if case["max_own"] > case["max_q"] else [0] * case["seqs"]
        common = [p for p, m in zip(prefix, members) for _ in range(m)]
        return new, [p + a + b for p, a, b in zip(common, new, more)]
    before = case["max_ctx"] - case["max_q"]
    old = _spread(rng, case["seqs"], before, case["ragged"]) if before else [0] * case["seqs"]
    if case["ragged"] and case["seqs"] > 3:
        old[2] = 0  # a sequence that begins
    if case["ragged"] and case["max_q"] > 1 and case["seqs"] > 4:
        new[3] = 0  # a sequence without new tokens in this step
    return new, [a + b for a, b in zip(new, old)]


def _groups(case):
    """(shared keys, sequences) of every group: whole pages, as a fork shares them."""
    rng = random.Random(case["spread"] + 1)
    prefix = [max(1, p // case["page"]) * case["page"]
              for p in _spread(rng, case["groups"], case["max_prefix"], case["ragged"])]
    if case["ragged"] and case["groups"] > 3:
        prefix[2] = 0  # sequences that share nothing
    cuts = sorted(rng.sample(range(1, case["seqs"]), case["groups"] - 1)) if case["ragged"] else \
        [g * case["seqs"] // case["groups"] for g in range(1, case["groups"])]
    return prefix, [b - a for a, b in zip([0] + cuts, cuts + [case["seqs"]])]


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ends(counts):
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        # rows from flat to certain: a spread of their own, and a favourite in every second one
        x = torch.randn(rows, vocab + case["pad"], device="cuda", generator=g)
        x *= torch.empty(rows, 1, device="cuda").uniform_(1.0, 4.0, generator=g)
        best = torch.randint(0, vocab, (rows,), device="cuda", generator=g)
        lift = torch.empty(rows, device="cuda").uniform_(0.0, 20.0, generator=g)
        lift[1::2] = 0.0
        x[torch.arange(rows, device="cuda"), best] += lift
        if case["masked"]:
            x[torch.rand(x.shape, device="cuda", generator=g) < case["masked"]] = -math.inf
        s["logits"] = x.to(dt)[:, :vocab]
        # a token drawn from each row's distribution
        chance = torch.empty(rows, vocab, device="cuda").exponential_(generator=g).log_()
        s["targets"] = (x[:, :vocab] - chance).argmax(-1)
        if own:
            from llm_accelerator_b200 import paged
            s["plan"] = paged.TokenLogprobs(top=case["top"])
            s["out"] = s["plan"].empty(rows)
        return s

    new, stored = _lens(case)
    page = case["page"]
    need = [-(-n // page) for n in stored]
    prefix, members = _groups(case) if case["op"] == "shared" else ([0] * case["seqs"], [1] * case["seqs"])
    common = [p // page for p in prefix]
    first, total = [], sum(common)  # where a sequence's own pages begin in the order of all pages
    for i, c in enumerate(c for c, m in zip(common, members) for _ in range(m)):
        first.append(total - c)
        total += need[i] - c
    pool = torch.empty(total + 1, 1, 2, case["kv_heads"], page, case["dim"], dtype=dt, device="cuda")
    pool.normal_(generator=g)
    s["k_cache"], s["v_cache"] = pool[:, 0, 0], pool[:, 0, 1]
    ids = torch.randperm(total + 1, device="cuda", generator=g)[:total].tolist()
    table, i = [], 0
    for at, c, m in zip(_ends(common), common, members):
        for _ in range(m):
            table.append(ids[at:at + c] + ids[first[i] + c:first[i] + need[i]] + [-1] * (max(need) - need[i]))
            i += 1
    s["table"], s["lens"] = _i32(table), _i32(stored)
    s["cu_q"] = _i32(_ends(new))
    s["q"] = torch.randn(sum(new), case["q_heads"], case["dim"], device="cuda", generator=g).to(dt)
    s["out"] = torch.empty_like(s["q"])
    s["lse"] = torch.empty(s["q"].shape[:2], dtype=torch.float32, device="cuda")
    if case["op"] == "shared":
        s["cu_group"], s["prefix_lens"] = _i32(_ends(members)), _i32(prefix)
    s["max_ctx"], s["max_prefix"] = max(stored), max(prefix)
    if own:
        from llm_accelerator_b200 import paged
        where = s["k_cache"], s["v_cache"], s["table"], s["lens"], case["q_heads"]
        s["plan"] = paged.SharedAttention(*where) if case["op"] == "shared" else \
            paged.Attention(*where, window=case["window"], sinks=case["sinks"])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_attention(s):
    case = s["case"]
    n, hk, d, page = case["seqs"], case["kv_heads"], case["dim"], case["page"]
    group = case["q_heads"] // hk
    lens, cu = s["lens"].long(), s["cu_q"].long()
    new = cu[1:] - cu[:-1]
    width = s["table"].shape[1]
    ids = s["table"].long().clamp(min=0)

    def gathered(cache):  # [n, hk, width * page, d]
        return cache[ids].permute(0, 2, 1, 3, 4).reshape(n, hk, width * page, d).float()

    step = torch.arange(case["max_q"], device="cuda")
    there = step[None, :] < new[:, None]
    token = (cu[:-1, None] + step[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][token].float().view(n, case["max_q"], hk, group, d)
    q = q.permute(0, 2, 3, 1, 4).reshape(n, hk, group * case["max_q"], d)
    place = (lens - new)[:, None] + step[None, :]
    key = torch.arange(width * page, device="cuda")
    seen = (key[None, None, :] <= place[:, :, None]) & (key[None, None, :] < lens[:, None, None])
    if case["op"] == "sinks":
        seen &= (key[None, None, :] > (place - case["window"])[:, :, None]) | (key < case["sinks"])
    score = torch.matmul(q, gathered(s["k_cache"]).transpose(-1, -2))
    score = score.view(n, hk, group, case["max_q"], -1).mul_(d ** -0.5)
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    value = torch.where((key[None, :] < lens[:, None])[:, None, :, None], gathered(s["v_cache"]), 0.0)
    out = torch.matmul(p.view(n, hk, group * case["max_q"], -1), value).view(n, hk, group, case["max_q"], d)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log()).squeeze(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, case["max_q"], case["q_heads"], d)[there]
    lse = lse.permute(0, 3, 1, 2).reshape(n, case["max_q"], case["q_heads"])[there]
    return {"out": out.to(s["q"].dtype), "lse": lse}


def _plain_logprobs(s):
    x = s["logits"].float()
    place = torch.arange(x.shape[1], device="cuda")
    top, best = x.max(-1, keepdim=True)
    e = (x - top).exp_()
    held = torch.where(e > 0, e * (x - top), 0.0).sum(-1, keepdim=True)
    # the sum but for the largest one, whose 1 would take the digits of a certain row's sum
    rest = torch.where(place == best, 0.0, e).sum(-1, keepdim=True)
    norm = rest.log1p()
    given = x.gather(1, s["targets"][:, None])
    ahead = (x > given) | ((x == given) & (place < s["targets"][:, None]))
    got = {"logprob": (given - top - norm).squeeze(1), "entropy": (norm - held / (1.0 + rest)).squeeze(1),
           "rank": (ahead.sum(-1) + 1).to(torch.int32)}
    if s["case"]["top"]:
        # numbers that order like (value, lower index first)
        bits = x.view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff), bits) * (1 << 32) - place
        index = order.topk(s["case"]["top"], -1).indices
        got |= {"top_logprob": x.gather(1, index) - top - norm, "top_index": index.to(torch.int32)}
    return got


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    case, plan = s["case"], s["plan"]
    if case["op"] == "logprobs":
        plan(s["logits"], s["targets"], s["out"])
        got = {"logprob": s["out"].logprob, "entropy": s["out"].entropy, "rank": s["out"].rank}
        if case["top"]:
            got |= {"top_logprob": s["out"].top_logprob, "top_index": s["out"].top_index}
        return got
    if case["op"] == "shared":
        plan(s["q"], s["out"], s["cu_q"], s["cu_group"], s["prefix_lens"], max_q=case["max_q"], max_ctx=s["max_ctx"],
             max_prefix=s["max_prefix"], lse=s["lse"])
    else:
        plan(s["q"], s["out"], s["cu_q"], max_q=case["max_q"], max_ctx=s["max_ctx"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def run(state):
    if own:
        return _own(state)
    return _plain_logprobs(state) if state["case"]["op"] == "logprobs" else _plain_attention(state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "logprobs":
        size = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
        values = case["rows"] * case["vocab"]
        # an exponential, its two sums and what leads to it
        return {"bytes": values * size + case["rows"] * (20 + 8 * case["top"]), "flops": 6 * values}
    new, stored = _lens(case)
    keys = seen = 0
    for n, ctx in zip(new, stored):
        if not n:
            continue
        first = ctx - n  # keys before the first query's own
        if case["op"] == "shared":
            keys += ctx
            seen += n * first + n * (n + 1) // 2
            continue
        w, sinks = case["window"], case["sinks"]
        low = max(0, first - w + 1)
        keys += ctx - low + min(sinks, low)
        # query i sees min(first + i + 1, w) keys through the window, and the sinks before those
        for i in range(n):
            low = max(0, first + i - w + 1)
            seen += first + i + 1 - low + min(sinks, low)
    if case["op"] == "shared":  # once for a group
        keys -= sum(p * (m - 1) for p, m in zip(*_groups(case)))
    kv = keys * case["kv_heads"] * case["dim"] * 2 * 2
    return {"bytes": kv + sum(new) * case["q_heads"] * (case["dim"] * 4 + 4),
            "flops": 4 * case["q_heads"] * case["dim"] * seen}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _exact_logprobs(s):
    k = s["case"]["top"]
    rows, vocab = s["logits"].shape
    got = {"logprob": [], "entropy": [], "rank": [], "top_logprob": [], "top_index": []}
    for lo in range(0, rows, 256):
        x, t = s["logits"][lo:lo + 256].double(), s["targets"][lo:lo + 256]
        at = torch.arange(x.shape[0], device="cuda")
        logp = torch.log_softmax(x, -1)
        got["logprob"].append(logp[at, t])
        got["entropy"].append(-torch.xlogy(logp.exp(), logp.exp()).sum(-1))
        before = torch.arange(vocab, device="cuda")[None, :] < t[:, None]
        mine = x[at, t][:, None]
        got["rank"].append(torch.where(before, x >= mine, x > mine).sum(-1).to(torch.int32) + 1)
        places = []
        for _ in range(k):  # the first of the largest that are left
            places.append(x.argmax(-1))
            x[at, places[-1]] = -math.inf
        if k:
            places = torch.stack(places, -1)
            got["top_index"].append(places.to(torch.int32))
            got["top_logprob"].append(logp.gather(1, places))
    return {name: torch.cat(parts) for name, parts in got.items() if parts}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    new, stored = _lens(case)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, ctx) in enumerate(zip(new, stored)):
        ids = s["table"][i, :-(-ctx // case["page"])].long()
        place = torch.arange(ctx - n, ctx, device="cuda")
        key = torch.arange(ctx, device="cuda")
        for h in range(case["kv_heads"] if n else 0):
            k = s["k_cache"][ids, h].reshape(-1, case["dim"])[:ctx].double()
            v = s["v_cache"][ids, h].reshape(-1, case["dim"])[:ctx].double()
            heads = slice(h * group, (h + 1) * group)
            for lo in range(0, n, 1024):
                rows = slice(lo, min(n, lo + 1024))
                hidden = key[None, :] > place[rows, None]
                if case["op"] == "sinks":
                    hidden |= (key[None, :] <= place[rows, None] - case["window"]) & (key[None, :] >= case["sinks"])
                a = torch.einsum("thd,kd->htk", s["q"][at + lo:at + rows.stop, heads].double(), k) / math.sqrt(case["dim"])
                a.masked_fill_(hidden, -math.inf)
                lse[at + lo:at + rows.stop, heads] = torch.logsumexp(a, -1).T
                out[at + lo:at + rows.stop, heads] = torch.einsum("htk,kd->thd", torch.softmax(a, -1), v)
        at += n
    return {"out": out, "lse": lse}
