"""16-bit paged serving operators against plain 64-bit forms.

Bounds.  u is the unit roundoff of the result's type (bf16 2^-8, f16 2^-11,
f32 2^-24); every result is rounded once, from values held in 32 bits:

* norm: the 32-bit part (a sum of up to 32768 squares, a reciprocal root, two
  products) stays within 1e-5 relative.  An 8-bit value is within half a step
  of its scaled value (e4m3: 2^-4 relative or half its smallest step 2^-9; s8:
  half a unit).
* rope: two products and a sum, 1e-5 of |a| + |b|.
* attention: a weight may be rounded to the cache's type (u of it), and a score
  of `dim` products in 32 bits is off by at most dim 2^-23 sum|q k| scale, which
  for the unit-normal inputs here is below 1.3e-4 and moves a weight by twice
  that; so |error| <= u |out| + (u + 3e-4) sum_j p_j |v_j|, and the log-sum is
  off by at most 3e-4.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}
BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def rnd(shape, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def within(got, ref, tol):
    bad = ~((got.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(got.double() - ref).abs().max():.3g}"


# ---------------------------------------------------------------------------
# norm
# ---------------------------------------------------------------------------
def norm_ref(x, r, w, eps):
    h = x.double() + (0 if r is None else r.double())
    return h, h * (h.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,n", [(1, 1), (1, 1024), (3, 7), (5, 33), (2, 4097), (700, 1023), (900, 1024),
                                    (3, 8200), (2, 32768), (1300, 264), (0, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(dtype, rows, n, residual):
    x, w = rnd((rows, n), dtype, 1, 2.0), rnd((n,), dtype, 2) + 1
    r = rnd((rows, n), dtype, 3) if residual else None
    total = torch.empty_like(x)
    y = paged.AddRmsNorm(w, eps=1e-5)(x, residual=r, residual_out=total)
    h, ref = norm_ref(x, r, w, 1e-5)
    within(y, ref, (U[dtype] + 1e-5) * ref.abs() + TINY[dtype])
    within(total, h, (U[dtype] + 1e-7) * h.abs() + TINY[dtype])


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("rows,n,group", [(1, 64, 64), (3, 1024, 0), (5, 1024, 64), (7, 4160, 64), (2, 256, 256),
                                          (9, 72, 8), (650, 2048, 128), (700, 333, 0), (3, 1001, 0), (2, 16384, 128)])
def test_norm_8bit(dtype, out, rows, n, group):
    x, w, r = rnd((rows, n), dtype, 1), rnd((n,), dtype, 2) + 1, rnd((rows, n), dtype, 3, 4.0)
    q, s = paged.AddRmsNorm(w, out_dtype=out, group=group)(x, residual=r)
    _, ref = norm_ref(x, r, w, 1e-6)
    g = ref.unflatten(-1, (-1, group or n))
    most = 448.0 if out == torch.float8_e4m3fn else 127.0
    want = g.abs().amax(-1) / most
    within(s, want, 2e-5 * want)
    value = q.double().unflatten(-1, (-1, group or n)) * s.double()[..., None]
    step = 2.0 ** -4 * g.abs() + 2.0 ** -10 * want[..., None] if out == torch.float8_e4m3fn else 0.5 * want[..., None]
    within(value, g, step * (1 + 1e-4) + 3e-5 * g.abs())


def test_norm_in_place_strided_and_zero_rows():
    base = rnd((6, 2080), BF, 4)
    x, r = base[:, 8:1032], base[:, 1040:2064]  # rows of a wider matrix
    x[2] = 0
    r[2] = 0
    w = rnd((1024,), BF, 5)
    h, ref = norm_ref(x.clone(), r.clone(), w, 1e-6)
    paged.AddRmsNorm(w)(x, out=x, residual=r, residual_out=r)
    within(x, ref, (U[BF] + 1e-5) * ref.abs())
    within(r, h, (U[BF] + 1e-7) * h.abs())
    z = torch.zeros(2, 128, dtype=HF, device="cuda")
    for out in (torch.float8_e4m3fn, torch.int8):
        q, s = paged.AddRmsNorm(torch.ones(128, dtype=HF, device="cuda"), eps=0.5, out_dtype=out, group=64)(z)
        assert not q.double().any() and not s.any()


def test_norm_nan_and_inf_stay_in_their_row():
    x, w = rnd((4, 512), BF, 6), rnd((512,), BF, 7)
    clean = paged.AddRmsNorm(w)(x)
    x[1, 17], x[3, 500] = math.nan, math.inf
    y = paged.AddRmsNorm(w)(x)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[2], clean[2])
    assert y[1].isnan().all() and y[3, 500].isnan()
    q, s = paged.AddRmsNorm(w, out_dtype=torch.int8, group=128)(x)
    assert s[1].isnan().all() and s[0].isfinite().all() and s[2].isfinite().all()


# ---------------------------------------------------------------------------
# rope
# ---------------------------------------------------------------------------
def angles(n, rot, theta=1e4):
    inv = theta ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv
    return a.cos().float(), a.sin().float()


def rope_ref(x, gamma, cos, sin, pos, inter, eps):
    x = x.double()
    if gamma is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * gamma.double()
    half = cos.shape[1]
    c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
    y, m = x.clone(), x.abs()
    ia = torch.arange(half, device="cuda") * 2 if inter else torch.arange(half, device="cuda")
    ib = ia + (1 if inter else half)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    m[..., ia] = m[..., ib] = a.abs() + b.abs()
    return y, m


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rot,page", [(1, 16, 8, 128, 128, 64), (5, 4, 2, 64, 32, 16),
                                                       (33, 7, 1, 72, 48, 3), (300, 6, 6, 128, 64, 32),
                                                       (9, 2, 1, 512, 512, 16), (4, 3, 3, 40, 0, 8)])
def test_rope_append(dtype, inter, normed, tokens, hq, hk, dim, rot, page):
    qkv = rnd((tokens, hq + 2 * hk, dim), dtype, 1)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
    pages = -(-tokens // page) + 2
    pool = rnd((pages, 2, hk, page, dim), dtype, 2)
    kc, vc = pool[:, 0], pool[:, 1]
    cos, sin = angles(500, rot) if rot else (torch.empty(500, 0, device="cuda"),) * 2
    pos = torch.randint(0, 500, (tokens,), device="cuda", dtype=torch.int32)
    rows = torch.randperm(pages * page, device="cuda")[:tokens].contiguous()
    rows[tokens // 2] = -1  # a padding token
    gq, gk = (rnd((dim,), dtype, 3) + 1, rnd((dim,), dtype, 4) + 1) if normed else (None, None)
    before = pool.clone()
    op = paged.RopeAppend(cos, sin, interleaved=inter, q_gamma=gq, k_gamma=gk, eps=1e-6)
    got = op(q, k, v, pos, rows, kc, vc, torch.empty_like(q))
    op.check()
    want, m = rope_ref(q, gq, cos, sin, pos.long(), inter, 1e-6)
    within(got, want, U[dtype] * want.abs() + 1e-5 * m + TINY[dtype])
    want, m = rope_ref(k, gk, cos, sin, pos.long(), inter, 1e-6)
    there = rows >= 0
    pg, off = rows[there] // page, rows[there] % page
    within(kc[pg, :, off], want[there], (U[dtype] * want.abs() + 1e-5 * m)[there] + TINY[dtype])
    assert torch.equal(vc[pg, :, off], v[there])
    kc[pg, :, off] = before[:, 0][pg, :, off]
    vc[pg, :, off] = before[:, 1][pg, :, off]
    assert torch.equal(pool, before)  # nothing else was written


def test_rope_parts_and_in_place():
    cos, sin = angles(64, 128)
    q, k = rnd((3, 2, 128), BF, 1), rnd((3, 1, 128), BF, 2)
    pos, rows = i32([0, 63, 5]), torch.tensor([2, 0, 1], device="cuda")
    cache = torch.zeros(1, 1, 16, 128, dtype=BF, device="cuda")
    want = rope_ref(q, None, cos, sin, pos.long(), False, 0)
    op = paged.RopeAppend(cos, sin)
    got = op(q, None, None, pos, None, None, None)
    assert got.data_ptr() == q.data_ptr()
    within(q, want[0], U[BF] * want[0].abs() + 1e-5 * want[1])
    op(None, k, None, pos, rows, cache, None)
    assert cache[0, 0, :3].any() and not cache[0, 0, 3:].any()
    op(None, None, k, None, rows, None, cache)
    assert torch.equal(cache[0, 0, rows], k[:, 0])


def test_rope_out_of_range_is_reported_and_skipped():
    cos, sin = angles(64, 128)
    k = rnd((4, 1, 128), BF, 2)
    cache = torch.zeros(1, 1, 16, 128, dtype=BF, device="cuda")
    op = paged.RopeAppend(cos, sin)
    for pos, rows in (([0, 64, 1, 2], [0, 1, 2, 3]), ([0, -1, 1, 2], [0, 1, 2, 3]), ([0, 1, 1, 2], [0, 16, 2, 3])):
        cache.zero_()
        op(None, k, k, i32(pos), torch.tensor(rows, device="cuda"), cache, torch.zeros_like(cache))
        with pytest.raises(_native.Q4GpuError):
            op.check()
        op.check()  # the word was cleared
        assert cache[0, 0, 0].any() and cache[0, 0, 3].any() and not cache[0, 0, 1].any()


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def make(new, old, hq, hk, dim, page, dtype, seed=0, extra=0):
    """Sequences with `old` stored and `new` query tokens over shuffled pages; page tails and unused pages are NaN."""
    g = torch.Generator().manual_seed(seed)
    lens = [a + b for a, b in zip(new, old)]
    need = [-(-max(n, 0) // page) for n in lens]
    total = sum(need) + 2 + extra
    pool = torch.full((total, 2, hk, page, dim), math.nan, dtype=dtype, device="cuda")
    ids = torch.randperm(total, generator=g)[:sum(need)].tolist()
    table, at = [], 0
    for n in need:
        table.append(ids[at:at + n] + [-1] * (max(need + [1]) - n))
        at += n
    for s, n in enumerate(lens):
        for j in range(need[s]):
            rows = min(page, n - j * page)
            pool[table[s][j], :, :, :rows] = rnd((2, hk, rows, dim), dtype, seed * 1000 + 37 * s + j)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = rnd((cu[-1], hq, dim), dtype, seed + 5)
    return pool, i32(table), i32(lens), i32(cu), q


def attn_ref(pool, table, lens, cu, q, scale, window=0, seq_ids=None):
    hk, page, dim = pool.shape[2], pool.shape[3], pool.shape[4]
    hq = q.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    cu, lens_h, tab = cu.tolist(), lens.tolist(), table.tolist()
    for i in range(len(cu) - 1):
        n = cu[i + 1] - cu[i]
        s = i if seq_ids is None else int(seq_ids[i])
        ctx = lens_h[s]
        if n == 0 or ctx <= 0:
            continue
        rows = tab[s][:-(-ctx // page)]
        ok = torch.tensor([0 <= p < pool.shape[0] for p in rows], device="cuda").repeat_interleave(page)[:ctx]
        ids = torch.tensor([max(0, min(p, pool.shape[0] - 1)) for p in rows], device="cuda")
        kv = pool[ids].double().permute(1, 2, 0, 3, 4).reshape(2, hk, -1, dim)[:, :, :ctx]
        kv = torch.where(ok[None, None, :, None], kv, 0.0)
        pos = torch.arange(ctx - n, ctx, device="cuda")[:, None]
        key = torch.arange(ctx, device="cuda")[None]
        seen = (key <= pos) & ok[None]
        if window:
            seen &= key > pos - window
        qs = q[cu[i]:cu[i + 1]].double().permute(1, 0, 2)
        k, v = kv[0].repeat_interleave(hq // hk, 0), kv[1].repeat_interleave(hq // hk, 0)
        sc = (qs @ k.transpose(1, 2) * scale).masked_fill(~seen, -math.inf)
        some = seen.any(-1)
        l = torch.logsumexp(sc, -1)
        p = torch.where(seen & some[:, None], (sc - torch.where(some, l, 0.0)[..., None]).exp(), 0.0)
        out[cu[i]:cu[i + 1]] = (p @ v).permute(1, 0, 2)
        mag[cu[i]:cu[i + 1]] = (p @ v.abs()).permute(1, 0, 2)
        lse[cu[i]:cu[i + 1]] = l.permute(1, 0)
    return out, mag, lse


def attend(pool, table, lens, cu, q, window=0, scale=None, seq_ids=None, max_ctx=0, out=None):
    new = (cu[1:] - cu[:-1]).max().item() if cu.numel() > 1 else 0
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=q.shape[1], window=window, scale=scale)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    out = op(q, out, cu, max_q=new, max_ctx=max_ctx or max(int(lens.max()), 1), lse=lse, seq_ids=seq_ids)
    return out, lse


def check_attn(pool, table, lens, cu, q, window=0, scale=None, seq_ids=None, **kw):
    out, lse = attend(pool, table, lens, cu, q, window, scale, seq_ids, **kw)
    ref, mag, rl = attn_ref(pool, table, lens, cu, q, scale or q.shape[2] ** -0.5, window, seq_ids)
    u = U[q.dtype]
    within(out, ref, u * ref.abs() + (u + 3e-4) * mag + TINY[q.dtype])
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none)
    within(lse[~none], rl[~none], 3e-4 + 1e-6 * rl[~none].abs())
    return out, lse


HEADS = [(16, 8, 128, 64), (4, 4, 64, 16), (7, 1, 128, 32), (24, 8, 64, 128), (8, 1, 64, 64), (6, 2, 128, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
def test_attention_single_tokens(dtype, hq, hk, dim, page):
    old = [0, 1, 2, 14, 15, 16, 17, 62, 63, 64, 65, 127, 128, 129, 500, 1023, 1500]
    check_attn(*make([1] * len(old), old, hq, hk, dim, page, dtype, 1))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
def test_attention_chunks(dtype, hq, hk, dim, page):
    new = [1, 2, 3, 0, 15, 16, 17, 63, 64, 65, 100, 129, 300, 1]
    old = [0, 0, 500, 70, 1, 31, 200, 64, 63, 0, 129, 1000, 0, 700]
    check_attn(*make(new, old, hq, hk, dim, page, dtype, 2))


@pytest.mark.parametrize("hq,hk,dim,page", [(16, 8, 128, 64), (7, 1, 64, 16), (3, 3, 128, 32)])
@pytest.mark.parametrize("window", [1, 5, 64, 130, 1000])
def test_attention_window(hq, hk, dim, page, window):
    check_attn(*make([1, 40, 200, 1, 9], [900, 600, 0, 3, 64], hq, hk, dim, page, BF, 3), window=window)


@pytest.mark.parametrize("new,old", [([1], [9000]), ([3], [5000]), ([200], [4000]), ([1, 600], [2500, 7000])])
@pytest.mark.parametrize("hq,hk,dim,page", [(2, 1, 128, 64), (8, 1, 64, 32), (16, 8, 128, 128)])
def test_attention_few_rows_long_context(new, old, hq, hk, dim, page):
    a = check_attn(*make(new, old, hq, hk, dim, page, BF, 4))
    b = check_attn(*make(new, old, hq, hk, dim, page, BF, 4))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # the joining order is fixed


def test_attention_long_prompt():
    check_attn(*make([2300], [0], 4, 2, 128, 64, BF, 5))
    check_attn(*make([1111, 900], [700, 1], 4, 1, 64, 16, HF, 5))


@pytest.mark.parametrize("new", [1, 40, 300])
def test_attention_empty_rows(new):
    """A slot that holds fewer keys than it has query tokens (or none), an unknown slot and a missing page."""
    pool, table, lens, cu, q = make([new] * 4, [130, 100, 0, 200], 4, 2, 64, 32, BF, 6)
    lens[1] = max(0, new - 3)
    lens[2] = 0
    table[3, 1] = -1
    table[3, 2] = pool.shape[0]
    out, lse = check_attn(pool, table, lens, cu, q)
    assert not out[cu[2]:cu[3]].any()
    ids = i32([3, 0, 0, 1])
    check_attn(pool, table, lens, cu, q, seq_ids=ids)
    out, lse = attend(pool, table, lens, cu, q, seq_ids=i32([3, -1, 4, 1]))
    assert not out[cu[1]:cu[3]].any() and (lse[cu[1]:cu[3]] == -math.inf).all()


@pytest.mark.parametrize("new,old", [(1, 300), (50, 300), (400, 300)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_attention_unseen_rows_do_not_reach_results(new, old, what):
    """Rows that a query does not see may hold anything: later tokens of its own chunk, keys before its window."""
    args = make([new], [old], 4, 2, 128, 64, BF, 7)
    pool, table, lens, cu, q = args
    clean, _ = attend(*args)
    page = pool.shape[3]
    if new > 1:
        at = old + new // 2  # this key is unseen by the first half of the queries
        pool[table[0, at // page], :, :, at % page] = what
        out, _ = attend(*args)
        assert torch.equal(out[:new // 2], clean[:new // 2])
        assert not out[new // 2:].isfinite().all()
    args = make([new], [old], 4, 2, 128, 64, BF, 7)
    pool = args[0]
    want, _ = attend(*args, window=20)
    for at in (0, 5, old - 20 - 1):  # before every query's window
        pool[args[1][0, at // page], :, :, at % page] = what
    assert torch.equal(attend(*args, window=20)[0], want)


@pytest.mark.parametrize("hq,hk,dim,page", [(32, 1, 128, 64), (17, 1, 64, 16), (40, 2, 64, 32), (48, 1, 128, 128)])
def test_attention_many_heads_a_key_head(hq, hk, dim, page):
    check_attn(*make([1, 2, 40, 0, 1], [0, 700, 100, 5, 64], hq, hk, dim, page, HF, 14))


@pytest.mark.parametrize("most", [1, 3, 40])
def test_attention_many_sequences(most):
    g = torch.Generator().manual_seed(most)
    new = torch.randint(0 if most > 1 else 1, most + 1, (300,), generator=g).tolist()
    old = torch.randint(0, 90, (300,), generator=g).tolist()
    old[7], old[250] = 1500, 900
    check_attn(*make(new, old, 4, 2, 64, 16, BF, 15))


def test_attention_workspace_serves_calls_of_all_shapes():
    """One operator, one workspace: splits, joins and chunks of different batches one after the other."""
    pool, table, lens, cu, q = make([1] * 40 + [70, 130], [3000] * 3 + [200] * 39, 8, 4, 128, 64, BF, 16)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=8)
    batches = [[0], list(range(40)), [40], [0, 1, 2], list(range(42)), [2], list(range(3, 40)), [1, 41], [0]]
    first = cu.tolist()
    for _ in range(2):
        for ids in batches:
            rows = torch.cat([torch.arange(first[i], first[i + 1], device="cuda") for i in ids])
            new = [first[i + 1] - first[i] for i in ids]
            c = i32([0] + torch.tensor(new).cumsum(0).tolist())
            got = op(q[rows], None, c, max_q=max(new), max_ctx=3200, seq_ids=i32(ids))
            ref, mag, _ = attn_ref(pool, table, lens, c, q[rows], 128 ** -0.5, 0, ids)
            within(got, ref, U[BF] * ref.abs() + (U[BF] + 3e-4) * mag)
    op.check()


def test_attention_extreme_scores():
    """Scores of +-1e4: weights are 0 or 1, nothing overflows."""
    pool, table, lens, cu, q = make([1, 150], [300, 200], 4, 2, 64, 64, BF, 8)
    out, lse = attend(pool, table, lens, cu, q, scale=300.0)
    ref, mag, rl = attn_ref(pool, table, lens, cu, q, 300.0)
    assert out.isfinite().all() and lse.isfinite().all()
    within(lse, rl, 1e-4 * rl.abs() + 1.0)
    out, _ = attend(pool, table, lens, cu, q, scale=1e-30)
    ref, mag, _ = attn_ref(pool, table, lens, cu, q, 1e-30)
    within(out, ref, U[BF] * ref.abs() + (U[BF] + 3e-4) * mag)


def test_attention_masked_infinities_in_queries():
    pool, table, lens, cu, q = make([130], [60], 4, 2, 64, 16, BF, 9)
    clean, _ = attend(pool, table, lens, cu, q)
    q[7, 1] = math.nan
    out, _ = attend(pool, table, lens, cu, q)
    assert out[7, 1].isnan().all()
    out[7, 1] = clean[7, 1]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new,old", [(1, 300), (50, 300), (400, 300)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 1, 2, 130])
def test_attention_seen_infinities_and_nans(new, old, what, at):
    """A key that is not finite makes every query that sees it NaN, wherever it stands in a step; the others keep
    their results."""
    args = make([new], [old], 4, 2, 128, 64, BF, 13)
    pool, table = args[:2]
    at += old if new > 200 else 0
    clean, _ = attend(*args)
    pool[table[0, at // 64], 0, 1, at % 64] = what  # key head 1: query heads 2 and 3
    out, lse = attend(*args)
    sees = torch.arange(old, old + new, device="cuda") >= at
    assert out[sees][:, 2:].isnan().all() and lse[sees][:, 2:].isnan().all()
    assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[~sees], clean[~sees])


@pytest.mark.parametrize("new,old", [([1, 1], [100, 900]), ([70, 3], [100, 900])])
def test_attention_strides_and_stream(new, old):
    """Queries inside a fused projection, an output with its own strides, another stream, and max_ctx left open."""
    pool, table, lens, cu, q = make(new, old, 4, 2, 64, 32, HF, 10)
    want, _ = attend(pool, table, lens, cu, q)
    wide = torch.zeros(q.shape[0], 9, 64, dtype=HF, device="cuda")
    wide[:, 3:7] = q
    out = torch.zeros(4, q.shape[0], 72, dtype=HF, device="cuda").permute(1, 0, 2)[..., :64]
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = op(wide[:, 3:7], out, cu, max_q=max(new))
    s.synchronize()
    bound = 3 * U[HF] * want.abs().double() + 2e-3
    within(got, want.double(), bound)


def test_attention_offsets_past_32_bits():
    """Pages whose byte and element offsets pass 2^32."""
    page, hk, dim = 64, 8, 128
    pages = (1 << 33) // (2 * hk * page * dim * 2) + 40  # over 8 GiB
    pool = torch.empty(pages, 2, hk, page, dim, dtype=BF, device="cuda")
    small, table, lens, cu, q = make([1, 200], [300, 50], 16, 8, 128, 64, BF, 11)
    where = torch.arange(small.shape[0], device="cuda") + pages - small.shape[0]
    pool[where] = small
    moved = torch.where(table >= 0, table + (pages - small.shape[0]), table).to(torch.int32)
    got, _ = attend(pool, moved, lens, cu, q)
    want, _ = attend(small, table, lens, cu, q)
    assert torch.equal(got, want)


def test_attention_nothing_to_do():
    pool, table, lens, cu, q = make([1], [10], 4, 2, 64, 32, HF, 12)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=4)
    assert op(q[:0], None, i32([0, 0])).shape == (0, 4, 64)
    assert op(q[:0], None, i32([0])).shape == (0, 4, 64)


# ---------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------
def pages_of(n_pages, blocks, page, dim, slots, width, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    pool = torch.randint(-9999, 9999, (n_pages, blocks, page, dim), dtype=torch.int16, device="cuda", generator=g)
    return pool, torch.full((slots, width), -1, dtype=torch.int32, device="cuda"), i32([0] * slots)


@pytest.mark.parametrize("page,dim,blocks", [(1, 8, 1), (16, 64, 3), (48, 8, 7), (64, 128, 40)])
def test_fork(page, dim, blocks):
    pool, table, lens = pages_of(40, blocks, page, dim, 9, 6)
    held = [0, 1, page, page + 1, 3 * page - 1, 5 * page]
    free = iter(range(39, -1, -1))
    for s, n in enumerate(held):
        for j in range(-(-n // page)):
            table[s, j] = next(free)
        lens[s] = n
    before, tb = pool.clone(), table.clone()
    op = paged.Pages(pool, table, lens, page)
    parents, children, fresh = [4, 0, 3], [6, 7, 8], [0, -1, 1]
    op.fork(i32(parents), i32(children), i32(fresh))
    op.check()
    for p, c, f in zip(parents, children, fresh):
        n, full, part = held[p], held[p] // page, held[p] % page
        want = tb[p].tolist()[:full] + ([f] if part else [])
        assert table[c].tolist() == want + [-1] * (6 - len(want)) and int(lens[c]) == n
        if part:
            before[f, :, :part] = before[int(tb[p, full]), :, :part]
    assert torch.equal(pool, before) and torch.equal(table[:6], tb[:6])


def test_fork_of_bad_ids_changes_nothing():
    pool, table, lens = pages_of(8, 2, 16, 8, 4, 3)
    table[0, 0], lens[0] = 5, 7
    table[1, 0], lens[1] = 8, 7  # a page outside the pool
    op = paged.Pages(pool, table, lens, 16)
    before, tb = pool.clone(), table.clone()
    for par, chi, fr in ((0, 4, 1), (-1, 2, 1), (0, 2, 8), (0, 2, -1), (1, 2, 3), (0, 0, 1), (0, 2, 5)):
        op.fork(i32([par]), i32([chi]), i32([fr]))
        with pytest.raises(_native.Q4GpuError):
            op.check()
    assert torch.equal(pool, before) and torch.equal(table, tb) and lens.tolist() == [7, 7, 0, 0]


@pytest.mark.parametrize("n_pages,page,blocks,live,seed", [(1, 4, 1, 1, 0), (1, 4, 1, 0, 0), (33, 4, 3, 20, 1),
                                                           (64, 16, 5, 64, 2), (257, 4, 2, 100, 3), (2000, 1, 1, 900, 4),
                                                           (96, 16, 900, 40, 5), (400000, 1, 1, 30000, 6)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(n_pages, page, blocks, live, seed, in_place):
    g = torch.Generator().manual_seed(seed)
    slots, dim = 5, 8
    width = live // 4 + 3
    pool, table, lens = pages_of(n_pages, blocks, page, dim, slots, width, seed)
    ids = torch.randperm(n_pages, generator=g)[:live].tolist()
    rows = [ids[s * (width - 2):(s + 1) * (width - 2)] for s in range(slots)]
    if rows[0] and rows[1]:
        rows[1][0] = rows[0][0]  # a shared page
    used = sorted({p for r in rows for p in r})
    table.copy_(i32([r + [7 if n_pages > 7 else 0] * (width - len(r)) for r in rows]))  # stale entries past the end
    lens.copy_(i32([len(r) * page - (s % page if r else 0) for s, r in enumerate(rows)]))
    before = pool.clone()
    op = paged.Pages(pool, table, lens, page)
    new = table if in_place else torch.empty_like(table)
    remap, n_live = torch.empty(n_pages, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32,
                                                                                       device="cuda")
    op.compact(new, remap, n_live)
    op.check()
    n = len(used)
    assert int(n_live) == n
    mapped = [p for p in used if p < n]
    low = set(mapped)
    holes = [p for p in range(n) if p not in low]
    want = {**{p: p for p in mapped}, **dict(zip([p for p in used if p >= n], holes))}
    rm = [-1] * n_pages
    for a, b in want.items():
        rm[a] = b
    assert remap.tolist() == rm
    assert new.tolist() == [[want[p] for p in r] + [-1] * (width - len(r)) for r in rows]
    for_src = torch.tensor(list(want), dtype=torch.long, device="cuda")
    for_dst = torch.tensor(list(want.values()), dtype=torch.long, device="cuda")
    assert torch.equal(pool[for_dst], before[for_src])
    if n < n_pages:
        assert torch.equal(pool[n:], before[n:])


def test_compact_reports_bad_pages():
    pool, table, lens = pages_of(8, 1, 4, 8, 2, 3)
    table[0], lens[0] = i32([6, 8, -1]), 8
    op = paged.Pages(pool, table, lens, 4)
    new, remap, n = torch.empty_like(table), torch.empty(8, dtype=torch.int32, device="cuda"), i32([0])
    want = pool[6].clone()
    op.compact(new, remap, n)
    with pytest.raises(_native.Q4GpuError):
        op.check()
    assert new.tolist() == [[0, -1, -1], [-1] * 3] and int(n) == 1 and torch.equal(pool[0], want)


# ---------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------
def test_refusals():
    w = torch.ones(64, dtype=BF, device="cuda")
    x = torch.zeros(2, 64, dtype=BF, device="cuda")
    norm = paged.AddRmsNorm(w)
    for bad in (lambda: norm(x.half()), lambda: norm(x[:, :32]), lambda: norm(x.cpu()), lambda: norm(x.t()),
                lambda: norm(x, residual=x[:1]), lambda: norm(x, out=torch.empty(2, 64, device="cuda")),
                lambda: paged.AddRmsNorm(w.cpu()), lambda: paged.AddRmsNorm(w, out_dtype=torch.int32)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_native.Q4GpuError, match="SHAPE"):
        paged.AddRmsNorm(w, out_dtype=torch.int8, group=48)(x)
    with pytest.raises(_native.Q4GpuError, match="SHAPE"):
        paged.AddRmsNorm(w, group=64)(x)
    with pytest.raises(_native.Q4GpuError, match="ALIGN"):
        wide = torch.zeros(2, 65, dtype=BF, device="cuda")
        paged.AddRmsNorm(w, out_dtype=torch.int8, group=64)(wide[:, 1:])
    with pytest.raises(_native.Q4GpuError, match="ARG"):
        paged.AddRmsNorm(w, out_dtype=HF)(x)

    cos, sin = angles(8, 64)
    op = paged.RopeAppend(cos, sin)
    q = torch.zeros(2, 4, 64, dtype=BF, device="cuda")
    pos, rows = i32([0, 1]), torch.tensor([0, 1], device="cuda")
    kc = torch.zeros(1, 4, 16, 64, dtype=BF, device="cuda")
    for bad in (lambda: op(q.float(), None, None, pos, None, None, None),
                lambda: op(q, None, None, pos.long(), None, None, None),
                lambda: op(q, q, q, pos, rows.int(), kc, kc), lambda: op(q, q, q, pos, rows, kc, kc[:, :2]),
                lambda: op(None, None, None, pos, rows, kc, kc), lambda: op(q, q, q, None, rows, kc, kc, q),
                lambda: op(q, q, q, pos, None, kc, kc, q), lambda: op(q, q, q, pos, rows, kc, None, q),
                lambda: paged.RopeAppend(cos, sin, q_gamma=w.float())(q, None, None, pos, None, None, None)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_native.Q4GpuError, match="SHAPE"):
        op(torch.zeros(2, 4, 32, dtype=BF, device="cuda"), None, None, pos, None, None, None)
    with pytest.raises(_native.Q4GpuError, match="ALIGN"):
        op(torch.zeros(2, 4, 65, dtype=BF, device="cuda")[..., 1:], None, None, pos, None, None, None)

    pool, table, lens, cu, q = make([1], [10], 4, 2, 64, 32, HF, 12)
    k, v = pool[:, 0], pool[:, 1]
    at = paged.Attention(k, v, table, lens, q_heads=4)
    for bad in (lambda: at(q.bfloat16(), None, cu), lambda: at(q, None, None), lambda: at(q, None, cu.long()),
                lambda: at(q, None, i32([0, 1, 1])), lambda: at(q, None, cu, lse=torch.empty(1, 4, device="cuda").half()),
                lambda: paged.Attention(k, v[:, :1], table, lens, q_heads=4),
                lambda: paged.Attention(k, v, table.long(), lens, q_heads=4),
                lambda: paged.Attention(k.float(), v.float(), table, lens, q_heads=4)):
        with pytest.raises(ValueError):
            bad()
    for kw in (dict(q_heads=5), dict(q_heads=0)):
        with pytest.raises(_native.Q4GpuError, match="SHAPE"):
            paged.Attention(k, v, table, lens, **kw)(torch.zeros(1, kw["q_heads"], 64, dtype=HF, device="cuda"), None, cu)
    odd = torch.zeros(2, 2, 24, 64, dtype=HF, device="cuda")
    with pytest.raises(_native.Q4GpuError, match="SHAPE"):
        paged.Attention(odd, odd, table, lens, q_heads=4)(q, None, cu)

    pool, table, lens = pages_of(8, 1, 4, 8, 2, 3)
    pages = paged.Pages(pool, table, lens, 4)
    with pytest.raises(ValueError):
        pages.fork(i32([0]), i32([1, 1]), i32([2]))
    with pytest.raises(ValueError):
        pages.compact(table[:1], i32([0] * 8), i32([0]))
    with pytest.raises(ValueError):
        paged.Pages(pool, table, lens, 5)
    with pytest.raises(_native.Q4GpuError, match="ALIGN"):
        narrow = torch.zeros(8, 4, 4, dtype=torch.int16, device="cuda")
        paged.Pages(narrow, table, lens, 4).fork(i32([0]), i32([1]), i32([2]))
