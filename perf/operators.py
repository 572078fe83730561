"""Timed cases of the 16-bit paged serving operators (``llm_accelerator_b200.paged``).

Per layer, a serving loop adds the residual and norms it (``AddRmsNorm``), rotates
the new queries and keys and stores the keys and values in the pages of their
sequences (``RopeAppend``), and attends from the new tokens to everything stored
(``Attention``); between steps it forks sequences that share a prompt and packs
the pages that are in use (``Pages.fork``, ``Pages.compact``).

Each case has a plain form in elementary torch operations, in 32 bits and rounded
once, and ``exact`` gives the values of the definition in 64 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
THETA = 1.0e6
YARN_LO, YARN_HI = 1.0, 32.0


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one decoded token of one sequence: latency is all there is
        {"name": "norm one token", "op": "norm", "rows": 1, "n": 1024, "dtype": "bf16", "residual": True,
         "out": "same", "group": 0},
        # a prompt's activations, normed into 8 bits for the next product, one scale per 64 columns
        {"name": "norm prompt 8 bit", "op": "norm", "rows": 8192, "n": 4096, "dtype": "bf16", "residual": True,
         "out": "e4m3", "group": 64},
        # five tokens of a speculative step, interleaved pairs over half of each head
        {"name": "rope few tokens", "op": "rope", "tokens": 5, "q_heads": 16, "kv_heads": 8, "dim": 128, "rot": 64,
         "page": 64, "dtype": "f16", "interleaved": True, "head_norm": False, "factor": 1.0, "positions": 2048},
        # a prompt's tokens with the q/k head norm, positions stretched to four times the trained length
        {"name": "rope prompt", "op": "rope", "tokens": 8192, "q_heads": 16, "kv_heads": 8, "dim": 128, "rot": 128,
         "page": 64, "dtype": "bf16", "interleaved": False, "head_norm": True, "factor": 4.0, "positions": 131072},
        # the first decode steps of one sequence
        {"name": "attn one token", "op": "attn", "seqs": 1, "max_q": 1, "max_ctx": 257, "q_heads": 16, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "window": 0, "ragged": False, "spread": 1},
        # batched decode at contexts of all lengths
        {"name": "attn decode batch", "op": "attn", "seqs": 64, "max_q": 1, "max_ctx": 8704, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0, "ragged": True, "spread": 2},
        # one serving step that mixes decodes and prompt chunks, seven query heads a key head, a sliding window
        {"name": "attn mixed chunks", "op": "attn", "seqs": 24, "max_q": 700, "max_ctx": 4500, "q_heads": 28,
         "kv_heads": 4, "dim": 64, "page": 32, "dtype": "f16", "window": 1500, "ragged": True, "spread": 3},
        # a long prompt's last large chunk
        {"name": "attn long chunk", "op": "attn", "seqs": 1, "max_q": 8192, "max_ctx": 16384, "q_heads": 16,
         "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "window": 0, "ragged": False, "spread": 4},
        # one conversation branches
        {"name": "fork two", "op": "fork", "forks": 2, "layers": 4, "kv_heads": 8, "dim": 128, "page": 16,
         "max_ctx": 700, "dtype": "bf16", "spread": 5},
        # sampling of many continuations of a few prompts
        {"name": "fork many", "op": "fork", "forks": 48, "layers": 28, "kv_heads": 8, "dim": 128, "page": 64,
         "max_ctx": 8704, "dtype": "bf16", "spread": 6},
        # a small pool after a few sequences ended
        {"name": "compact small", "op": "compact", "pages": 96, "live": 0.4, "seqs": 5, "layers": 2, "kv_heads": 2,
         "dim": 64, "page": 16, "dtype": "f16", "spread": 7},
        # a fragmented pool of many sequences
        {"name": "compact pool", "op": "compact", "pages": 300, "live": 0.5, "seqs": 40, "layers": 28, "kv_heads": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "spread": 8},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "rope", "attn", "attn", "fork", "compact"])
    dtype = rng.choice(sorted(DTYPES))
    spread = rng.randrange(1 << 20)
    if op == "norm":
        n = _log(rng, 64, 16384)
        group = rng.choice([0, 64, 128])
        out = rng.choice(["same", "e4m3"])
        if out == "same":
            group = 0
        if group:
            n = max(group, n // group * group)
        return {"op": op, "rows": _log(rng, 1, max(1, min(32768, 8192 * 4096 // n))), "n": n, "dtype": dtype,
                "residual": rng.random() < 0.7, "out": out, "group": group}
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    kv = rng.choice([1, 2, 4, 8])
    if op == "rope":
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        rot = rng.choice([dim, dim // 2])
        return {"op": op, "tokens": _log(rng, 1, 8192), "q_heads": min(heads, 16), "kv_heads": min(kv, 8), "dim": dim,
                "rot": rot, "page": page, "dtype": dtype, "interleaved": rng.random() < 0.5,
                "head_norm": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0, 8.0]),
                "positions": _log(rng, 8192, 131072)}
    if op == "attn":
        heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
        max_q = 1 if rng.random() < 0.4 else _log(rng, 2, 4096)
        seqs = _log(rng, 1, 64)
        max_ctx = max_q + _log(rng, 1, 16384)
        # the padded score matrix and the gathered cache stay below the largest listed case's
        while seqs > 1 and (seqs * heads * max_q * max_ctx > 1 << 30 or seqs * kv * max_ctx * dim > 1 << 29):
            seqs = seqs // 2
        while heads * max_q * max_ctx > 1 << 30:
            max_ctx = max_q + max(1, (max_ctx - max_q) // 2)
            if max_ctx <= max_q + 1:
                max_q //= 2
                max_ctx = max_q + 1
        return {"op": op, "seqs": seqs, "max_q": max_q, "max_ctx": max_ctx, "q_heads": heads, "kv_heads": kv,
                "dim": dim, "page": page, "dtype": dtype, "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]),
                "ragged": rng.random() < 0.7, "spread": spread}
    layers = rng.choice([1, 2, 4, 12, 28])
    if op == "fork":
        return {"op": op, "forks": _log(rng, 1, 48), "layers": layers, "kv_heads": kv, "dim": dim, "page": page // 2
                if page == 128 else page, "max_ctx": _log(rng, 1, 8192), "dtype": dtype, "spread": spread}
    page = min(page, 64)
    page_values = layers * 2 * kv * page * dim
    most = max(8, min(4096, 300 * 28 * 2 * 8 * 64 * 128 // page_values))
    return {"op": op, "pages": _log(rng, 8, most), "live": round(rng.uniform(0.1, 0.9), 3), "seqs": _log(rng, 1, 64),
            "layers": layers, "kv_heads": kv, "dim": dim, "page": page, "dtype": dtype, "spread": spread}


def _spread(rng, n, most, ragged):
    """n lengths up to `most`: all of them `most`, or spread over the logarithm, the first the longest."""
    return [most if i == 0 or not ragged else max(1, min(most, _log(rng, 1, most))) for i in range(n)]


def _lens(case):
    """(new tokens, tokens stored once they are in) of every sequence of an attention case."""
    rng = random.Random(case["spread"])
    new = _spread(rng, case["seqs"], case["max_q"], case["ragged"])
    before = case["max_ctx"] - case["max_q"]
    old = _spread(rng, case["seqs"], before, case["ragged"]) if before else [0] * case["seqs"]
    if case["ragged"] and case["seqs"] > 3:
        old[2] = 0  # a sequence that begins
    if case["ragged"] and case["max_q"] > 1 and case["seqs"] > 4:
        new[3] = 0  # a sequence without new tokens in this step
    return new, [a + b for a, b in zip(new, old)]


def _fork_lens(case):
    """Lengths of the forked sequences: one parent for every four children."""
    rng = random.Random(case["spread"])
    parents = max(1, (case["forks"] + 3) // 4)
    return _spread(rng, parents, case["max_ctx"], True)


def _compact_plan(case):
    """Page ids of every sequence, scattered over the pool; the last two sequences share their first page."""
    rng = random.Random(case["spread"])
    live = max(1, min(case["pages"] - 1, int(case["pages"] * case["live"])))
    ids = rng.sample(range(case["pages"]), live)
    rows = [[] for _ in range(case["seqs"])]
    for i, p in enumerate(ids):
        rows[i % case["seqs"]].append(p)
    if case["seqs"] > 1 and rows[-1] and rows[-2]:
        rows[-1][0] = rows[-2][0]
    fill = [len(r) * case["page"] - (rng.randrange(case["page"]) if r else 0) for r in rows]
    return rows, fill


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _angles(case):
    """cos and sin [positions, rot / 2] in 64 bits: YaRN's by-part frequencies where `factor` is above 1."""
    half = case["rot"] // 2
    i = torch.arange(half, dtype=torch.float64, device="cuda")
    inv = THETA ** (-2.0 * i / case["rot"])
    scale = 1.0
    if case["factor"] > 1.0:
        turns = (case["positions"] / case["factor"]) * inv / (2.0 * math.pi)
        keep = ((turns - YARN_LO) / (YARN_HI - YARN_LO)).clamp(0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / case["factor"])
        scale = 0.1 * math.log(case["factor"]) + 1.0
    a = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return a.cos() * scale, a.sin() * scale


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32) * std).to(dt)

    def pool_of(pages, layers):
        p = torch.empty(pages, layers, 2, case["kv_heads"], case["page"], case["dim"], dtype=dt, device="cuda")
        return p.normal_(generator=g)

    s = {"case": case}
    if case["op"] == "norm":
        rows, n = case["rows"], case["n"]
        s["x"] = randn(rows, n)
        s["residual"] = randn(rows, n, std=3.0) if case["residual"] else None
        s["weight"] = 1.0 + randn(n, std=0.1)
        s["out"] = torch.empty(rows, n, dtype=torch.float8_e4m3fn if case["out"] == "e4m3" else dt, device="cuda")
        s["sum"] = torch.empty(rows, n, dtype=dt, device="cuda")
        groups = n // case["group"] if case["group"] else 1
        s["scale"] = torch.empty(rows, groups, dtype=torch.float32, device="cuda") if case["out"] == "e4m3" else None
        if own:
            from llm_accelerator_b200 import paged
            s["plan"] = paged.AddRmsNorm(s["weight"], eps=EPS, out_dtype=s["out"].dtype, group=case["group"])
        return s
    if case["op"] == "rope":
        t, d, hq, hk = case["tokens"], case["dim"], case["q_heads"], case["kv_heads"]
        qkv = randn(t, (hq + 2 * hk) * d)  # the fused projection's rows
        s["q"] = qkv[:, :hq * d].view(t, hq, d)
        s["k"] = qkv[:, hq * d:(hq + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
        pages = -(-t // case["page"]) + 1
        pool = pool_of(pages, 1)
        s["k_cache"], s["v_cache"] = pool[:, 0, 0], pool[:, 0, 1]
        s["rows"] = torch.randperm(pages * case["page"], device="cuda", generator=g)[:t].contiguous()
        first = max(0, case["positions"] - t)
        s["positions"] = (first + torch.arange(t, device="cuda") % (case["positions"] - first)).to(torch.int32)
        cos, sin = _angles(case)
        s["cos"], s["sin"] = cos.float(), sin.float()
        s["q_gamma"] = 1.0 + randn(d, std=0.1) if case["head_norm"] else None
        s["k_gamma"] = 1.0 + randn(d, std=0.1) if case["head_norm"] else None
        s["q_out"] = torch.empty(t, hq, d, dtype=dt, device="cuda")
        if own:
            from llm_accelerator_b200 import paged
            s["plan"] = paged.RopeAppend(s["cos"], s["sin"], interleaved=case["interleaved"], q_gamma=s["q_gamma"],
                                         k_gamma=s["k_gamma"], eps=EPS)
        return s
    if case["op"] == "attn":
        new, stored = _lens(case)
        need = [-(-n // case["page"]) for n in stored]
        total, width = sum(need), max(need)
        pool = pool_of(total + 1, 1)
        s["k_cache"], s["v_cache"] = pool[:, 0, 0], pool[:, 0, 1]
        ids = torch.randperm(total + 1, device="cuda", generator=g)[:total].tolist()
        table, at = [], 0
        for n in need:
            table.append(ids[at:at + n] + [-1] * (width - n))
            at += n
        s["table"], s["lens"] = _i32(table), _i32(stored)
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        s["cu_q"] = _i32(cu)
        s["q"] = randn(cu[-1], case["q_heads"], case["dim"])
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(cu[-1], case["q_heads"], dtype=torch.float32, device="cuda")
        if own:
            from llm_accelerator_b200 import paged
            s["plan"] = paged.Attention(s["k_cache"], s["v_cache"], s["table"], s["lens"], q_heads=case["q_heads"],
                                        window=case["window"])
        return s
    if case["op"] == "fork":
        lens = _fork_lens(case)
        need = [-(-n // case["page"]) for n in lens]
        width, slots = max(need) + 1, len(lens) + case["forks"]
        # the pages of a prompt besides its last one are only named in the table
        pages = len(lens) + case["forks"] + 1
        s["pool"] = pool_of(pages, case["layers"])
        order = torch.randperm(pages, device="cuda", generator=g).tolist()
        table = [[order[i]] * n + [-1] * (width - n) for i, n in enumerate(need)]
        table += [[-1] * width for _ in range(case["forks"])]
        s["table"], s["lens"] = _i32(table), _i32(lens + [0] * case["forks"])
        s["parents"] = _i32([i % len(lens) for i in range(case["forks"])])
        s["children"] = _i32([len(lens) + i for i in range(case["forks"])])
        s["fresh"] = _i32(order[len(lens):len(lens) + case["forks"]])
        assert slots == s["table"].shape[0]
    else:
        rows, fill = _compact_plan(case)
        width = max(len(r) for r in rows) + 1
        s["pool"] = pool_of(case["pages"], case["layers"])
        # the pages' order in the pool is the seed's
        perm = torch.randperm(case["pages"], device="cuda", generator=g).tolist()
        s["table"] = _i32([[perm[p] for p in r] + [-1] * (width - len(r)) for r in rows])
        s["lens"] = _i32(fill)
        s["new_table"] = torch.empty_like(s["table"])
        s["remap"] = torch.empty(case["pages"], dtype=torch.int32, device="cuda")
        s["n_live"] = torch.empty(1, dtype=torch.int32, device="cuda")
    if own:
        from llm_accelerator_b200 import paged
        s["plan"] = paged.Pages(s["pool"], s["table"], s["lens"], page_tokens=case["page"])
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    total = h.to(s["x"].dtype)
    if case["out"] == "same":
        return {"y": y.to(s["x"].dtype), "sum": total}
    rows, n = y.shape
    yg = y.view(rows, -1, case["group"] or n)
    most = yg.abs().amax(-1, keepdim=True)
    inv = torch.where(most > 0, 448.0 / most, torch.zeros_like(most))
    return {"y": (yg * inv).view(rows, n).to(torch.float8_e4m3fn), "sum": total, "scale": (most / 448.0).squeeze(-1)}


def _turn(x, cos, sin, rot, interleaved):
    cos, sin = cos[:, None, :], sin[:, None, :]
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((r, rest), -1)


def _plain_rope(s):
    case = s["case"]
    at = s["positions"].long()
    cos, sin = s["cos"][at], s["sin"][at]

    def head(x, gamma):
        x = x.float()
        if gamma is not None:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * gamma.float()
        return _turn(x, cos, sin, case["rot"], case["interleaved"])

    page, off = s["rows"] // case["page"], s["rows"] % case["page"]
    s["k_cache"][page, :, off] = head(s["k"], s["k_gamma"]).to(s["k"].dtype)
    s["v_cache"][page, :, off] = s["v"]
    return {"q": head(s["q"], s["q_gamma"]).to(s["q"].dtype), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


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
    if case["window"]:
        seen = seen & (key[None, None, :] > (place - case["window"])[:, :, None])
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


def _plain_fork(s):
    page = s["case"]["page"]
    par, chi = s["parents"].long(), s["children"].long()
    n = s["lens"].long()[par]
    rows = s["table"][par]
    last, part = (n - 1) // page, n % page
    width = rows.shape[1]
    col = torch.arange(width, device="cuda")[None, :]
    source = rows.gather(1, last[:, None]).squeeze(1).long()
    mine = (part > 0)[:, None] & (col == last[:, None])
    rows = torch.where(mine, s["fresh"][:, None], rows)
    rows = torch.where(col <= last[:, None], rows, -1)
    s["table"][chi] = rows
    s["lens"][chi] = n.to(torch.int32)
    fresh = s["fresh"].long()
    filled = torch.arange(page, device="cuda")[None, :] < part[:, None]
    s["pool"][fresh] = torch.where(filled[:, None, None, None, :, None], s["pool"][source], s["pool"][fresh])
    return {"pool": s["pool"].view(torch.int16), "table": s["table"], "lens": s["lens"]}


def _plain_compact(s):
    pages, page = s["case"]["pages"], s["case"]["page"]
    used = torch.arange(s["table"].shape[1], device="cuda")[None, :] < ((s["lens"] + page - 1) // page)[:, None]
    live = torch.zeros(pages, dtype=torch.bool, device="cuda")
    live[s["table"][used].long()] = True
    n_live = live.sum()
    at = torch.arange(pages, device="cuda")
    movers = at[live & (at >= n_live)]
    holes = at[~live & (at < n_live)]
    remap = torch.where(live, at, -1)
    remap[movers] = holes
    s["pool"][holes] = s["pool"][movers]
    table = torch.where(used, remap[s["table"].long().clamp(min=0)], -1)
    return {"pool": s["pool"].view(torch.int16), "table": table.to(torch.int32), "remap": remap.to(torch.int32),
            "n_live": n_live.to(torch.int32).view(1)}


PLAIN = {"norm": _plain_norm, "rope": _plain_rope, "attn": _plain_attention, "fork": _plain_fork,
         "compact": _plain_compact}


# ---------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------
def _own(s):
    case, plan = s["case"], s["plan"]
    if case["op"] == "norm":
        plan(s["x"], s["out"], residual=s["residual"], residual_out=s["sum"], scale=s["scale"])
        got = {"y": s["out"], "sum": s["sum"]}
        return got if s["scale"] is None else {**got, "scale": s["scale"]}
    if case["op"] == "rope":
        plan(s["q"], s["k"], s["v"], s["positions"], s["rows"], s["k_cache"], s["v_cache"], s["q_out"])
        return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attn":
        plan(s["q"], s["out"], s["cu_q"], max_q=case["max_q"], max_ctx=case["max_ctx"], lse=s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] == "fork":
        plan.fork(s["parents"], s["children"], s["fresh"])
        return {"pool": s["pool"].view(torch.int16), "table": s["table"], "lens": s["lens"]}
    plan.compact(s["new_table"], s["remap"], s["n_live"])
    return {"pool": s["pool"].view(torch.int16), "table": s["new_table"], "remap": s["remap"], "n_live": s["n_live"]}


def run(state):
    return _own(state) if own else PLAIN[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        values = case["rows"] * case["n"]
        per = 2 + 2 + (2 if case["residual"] else 0) + (1 if case["out"] == "e4m3" else 2)
        scales = case["rows"] * (case["n"] // case["group"] if case["group"] else 1) * 4 if case["out"] == "e4m3" else 0
        return {"bytes": values * per + scales + 2 * case["n"], "flops": 6 * values}
    if case["op"] == "rope":
        heads = case["q_heads"] + 2 * case["kv_heads"]
        table = min(case["tokens"], case["positions"]) * case["rot"] * 4
        return {"bytes": case["tokens"] * (heads * case["dim"] * 4 + 12) + table,
                "flops": 3 * case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["dim"]}
    if case["op"] == "attn":
        new, stored = _lens(case)
        flops = keys = 0
        for n, ctx in zip(new, stored):
            if not n:
                continue
            first = ctx - n
            w = case["window"] or ctx
            low = max(0, first - w + 1)
            keys += ctx - low
            # keys seen by query i: min(first + i + 1, w)
            short = max(0, min(n, w - first))
            seen = short * first + short * (short + 1) // 2 + (n - short) * w
            flops += 4 * case["q_heads"] * case["dim"] * seen
        kv = keys * case["kv_heads"] * case["dim"] * 2 * 2
        return {"bytes": kv + sum(new) * case["q_heads"] * (case["dim"] * 4 + 4), "flops": flops}
    page_bytes = case["layers"] * 2 * case["kv_heads"] * case["dim"] * 2 * case["page"]
    if case["op"] == "fork":
        lens = _fork_lens(case)
        width = -(-max(lens) // case["page"]) + 1
        part = [n % case["page"] / case["page"] for n in lens]
        read = sum(part[:case["forks"]]) * page_bytes
        written = sum(part[i % len(lens)] for i in range(case["forks"])) * page_bytes
        return {"bytes": int(read + written) + 4 * width * (len(lens) + case["forks"]), "flops": 0}
    rows, _ = _compact_plan(case)
    # how many live pages lie past the packed end is up to the seed: its expected number
    live = len({p for r in rows for p in r})
    moves = live * (case["pages"] - live) / case["pages"]
    return {"bytes": int(2 * moves * page_bytes) + 4 * (2 * sum(map(len, rows)) + case["pages"]), "flops": 0}


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def _e4m3(x):
    """The nearest e4m3 value (ties to even) of 64-bit numbers within +-448."""
    e = torch.frexp(x)[1].clamp(min=-5) - 1  # smallest normal exponent -6
    step = torch.pow(2.0, (e - 3).double())
    return torch.round(x / step) * step


def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # copies and page numbers: nothing is computed in floating point
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0.0)
        y = h * (h.square().sum(-1, keepdim=True) / case["n"] + EPS).rsqrt() * s["weight"].double()
        if case["out"] == "same":
            return {"y": y, "sum": h}
        y = y.unflatten(-1, (-1, case["group"] or case["n"]))
        scale = y.abs().amax(-1) / 448.0
        return {"y": _e4m3(y / scale[..., None]).flatten(-2), "sum": h, "scale": scale}
    if case["op"] == "rope":
        cos, sin = _angles(case)
        turn = torch.complex(cos, sin)[s["positions"].long()][:, None, :]

        def head(x, gamma):
            x = x.double()
            if gamma is not None:
                x = x * (x.square().sum(-1, keepdim=True) / case["dim"] + EPS).rsqrt() * gamma.double()
            pair = x[..., :case["rot"]]
            pair = pair.unflatten(-1, (-1, 2)) if case["interleaved"] else pair.unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            z = z if case["interleaved"] else z.transpose(-1, -2)
            return torch.cat((z.flatten(-2), x[..., case["rot"]:]), -1)

        k, v = s["k_cache"].double(), s["v_cache"].double()
        where = (s["rows"] // case["page"], slice(None), s["rows"] % case["page"])
        k[where] = head(s["k"], s["k_gamma"])
        v[where] = s["v"].double()
        return {"q": head(s["q"], s["q_gamma"]), "k_cache": k, "v_cache": v}
    new, stored = _lens(case)
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["lse"].shape, -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, ctx) in enumerate(zip(new, stored)):
        ids = s["table"][i, :-(-ctx // case["page"])].long()
        place = torch.arange(ctx - n, ctx, device="cuda")
        key = torch.arange(ctx, device="cuda")
        for h in range(case["q_heads"] if n else 0):
            k = s["k_cache"][ids, h // group].reshape(-1, case["dim"])[:ctx].double()
            v = s["v_cache"][ids, h // group].reshape(-1, case["dim"])[:ctx].double()
            for lo in range(0, n, 2048):
                rows = slice(lo, min(n, lo + 2048))
                hidden = key[None, :] > place[rows, None]
                if case["window"]:
                    hidden |= key[None, :] <= place[rows, None] - case["window"]
                a = s["q"][at + lo:at + rows.stop, h].double() @ k.T / math.sqrt(case["dim"])
                a[hidden] = -math.inf
                lse[at + lo:at + rows.stop, h] = torch.logsumexp(a, -1)
                out[at + lo:at + rows.stop, h] = torch.softmax(a, -1) @ v
        at += n
    return {"out": out, "lse": lse}
