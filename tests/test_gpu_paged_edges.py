"""Corners of the 16-bit paged operators: degenerate scales and magnitudes, what only the device can see, layouts of
the cache and of calls, streams and graphs.

Bounds are those of the ordinary cases (``test_gpu_paged``): an attention result is within u |out| + (u + 3e-4)
sum p |v| of the 64-bit form and its log-sum within 3e-4 + 1e-6 |lse|; with the scale 0 the weights are exactly 1
and the same bounds hold."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402
from test_gpu_paged import (BF, HF, SF, TINY, U, angles, attn_ref, i32, make, norm_ref, pages_of, rnd,  # noqa: E402
                            rope_ref, within)


def operator(pool, table, lens, hq, **kw):
    return paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=hq, **kw)


def close(got, lse, ref, mag, rl, dtype):
    u = U[dtype]
    within(got, ref, u * ref.abs() + (u + 3e-4) * mag + TINY[dtype])
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none)
    within(lse[~none], rl[~none], 3e-4 + 1e-6 * rl[~none].abs())


def check(op, pool, table, lens, cu, q, scale, window=0, max_q=None, seq_ids=None):
    """One call against the 64-bit form; returns what it gave."""
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = torch.full_like(q, 5.0)
    most = int((cu[1:] - cu[:-1]).max()) if max_q is None else max_q
    op(q, out, cu, max_q=most, max_ctx=max(1, int(lens.max())), lse=lse, seq_ids=seq_ids)
    close(out, lse, *attn_ref(pool, table, lens, cu, q, scale, window, seq_ids), q.dtype)
    return out, lse


@pytest.mark.parametrize("hq,hk", [(4, 2), (32, 1)])
@pytest.mark.parametrize("max_q", [1, 64, 4096])
def test_attention_of_an_empty_step(hq, hk, max_q):
    pool, table, lens, cu, q = make([1], [10], hq, hk, 64, 32, BF, 20)
    op = operator(pool, table, lens, hq)
    assert op(q[:0], None, i32([0, 0]), max_q=max_q).shape == (0, hq, 64)
    assert op(q[:0], None, i32([0]), max_q=max_q).shape == (0, hq, 64)
    check(op, pool, table, lens, cu, q, 64 ** -0.5)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,old", [([1, 2], [300, 0]), ([200], [300]), ([3, 40, 300, 1], [500, 0, 20, 70]),
                                     ([70], [4000])])
@pytest.mark.parametrize("window", [0, 70])
def test_attention_scale_zero_is_the_mean(dtype, dim, new, old, window):
    args = make(new, old, 4, 2, dim, 32, dtype, 21)
    for scale in (0.0, -0.0, 1e-44):
        check(operator(*args[:3], 4, scale=scale, window=window), *args, scale, window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,old", [([1, 2], [300, 0]), ([3, 40, 300, 1], [500, 0, 20, 70])])
def test_attention_negative_scale(dim, new, old):
    args = make(new, old, 4, 2, dim, 32, BF, 22)
    check(operator(*args[:3], 4, scale=-dim ** -0.5), *args, -dim ** -0.5)


def reported(op):
    try:
        op.check()
    except _native.Q4GpuError as e:
        assert "out of range" in str(e)
        return True
    return False


@pytest.mark.parametrize("new", [1, 40, 300])
def test_attention_reports_what_is_out_of_range(new):
    pool, table, lens, cu, q = make([new] * 4, [130, 100, 0, 200], 4, 2, 64, 32, BF, 23)
    op = operator(pool, table, lens, 4)
    room = table.shape[1] * 32

    def run(ids=None, c=cu):
        out = op(q, torch.zeros_like(q), c, max_q=new, max_ctx=512, seq_ids=ids)
        return out, reported(op)

    def rest(out, rows):  # the other sequences (whose work may be split in other places) keep their results
        within(out[rows], ref[rows], U[BF] * ref[rows].abs() + (U[BF] + 3e-4) * mag[rows])

    ref, mag, _ = attn_ref(pool, table, lens, cu, q, 64 ** -0.5)
    good, said = run()
    assert not said
    for bad in (-1, 4, 2 ** 31 - 1, -2 ** 31):
        out, said = run(i32([0, bad, 2, 3]))
        assert said and not out[new:2 * new].any()
        rest(out, slice(2 * new, None))
    for s, n in ((1, room + 1), (0, -1), (3, 2 ** 31 - 1)):
        kept = int(lens[s])
        lens[s] = n
        assert run()[1]
        lens[s] = kept
    for page in (pool.shape[0], -1, 2 ** 31 - 1):
        kept = int(table[3, 1])
        table[3, 1] = page
        out, said = run()
        assert said
        rest(out, slice(0, 3 * new))
        table[3, 1] = kept
    for c in ([0, new, 2 * new, 3 * new, 4 * new + 1], [-1, new, 2 * new, 3 * new, 4 * new],
              [0, new, new - 1, 3 * new, 4 * new]):
        assert run(c=i32(c))[1]
    out, said = run()
    assert not said and torch.equal(out, good)


@pytest.mark.parametrize("new", [1, 3, 40])
def test_attention_does_not_report_what_nothing_reads(new):
    """Sequences without queries may name any slot (padding); pages before every query's window may be gone."""
    pool, table, lens, cu, q = make([new] * 2, [700, 300], 4, 2, 64, 32, BF, 24)
    op = operator(pool, table, lens, 4, window=100)
    want = op(q, None, cu, max_q=new)
    assert not reported(op)
    table[0, :(700 - 100 + 1) // 32] = -1  # the first query sees the keys from 601 on
    assert torch.equal(op(q, None, cu, max_q=new), want) and not reported(op)
    padded = torch.cat((cu, cu[-1:], cu[-1:]))
    assert torch.equal(op(q, None, padded, max_q=new, seq_ids=i32([0, 1, -1, 99])), want) and not reported(op)


@pytest.mark.parametrize("hq,hk,max_q", [(4, 2, 1), (4, 2, 8), (7, 1, 2), (16, 1, 1), (32, 1, 0), (4, 2, 0)])
def test_attention_of_a_sequence_longer_than_max_q(hq, hk, max_q):
    """A sequence with more queries than promised is reported and its rows are zeros or complete, never left over."""
    new = [1, 40, max_q, 0, 300]
    args = make(new, [30, 200, 500, 10, 0], hq, hk, 64, 32, BF, 25)
    pool, table, lens, cu, q = args
    op = operator(pool, table, lens, hq)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    op(q, out, cu, max_q=max_q, lse=lse)
    assert reported(op)
    ref, mag, rl = attn_ref(pool, table, lens, cu, q, 64 ** -0.5)
    for i, n in enumerate(new):
        rows = slice(int(cu[i]), int(cu[i + 1]))
        if n > max_q and not out[rows].any():
            assert (lse[rows] == -math.inf).all()
        else:
            close(out[rows], lse[rows], ref[rows], mag[rows], rl[rows], BF)
    check(op, *args, 64 ** -0.5)  # and the next call is as ever
    assert not reported(op)


def test_rope_stores_nothing_of_a_token_without_a_position():
    cos, sin = angles(64, 128)
    k, v = rnd((4, 2, 128), BF, 1), rnd((4, 2, 128), BF, 2)
    rows = torch.tensor([3, 2, 1, 0], device="cuda")
    for bad in (-1, 64, 2 ** 31 - 1):
        op = paged.RopeAppend(cos, sin)
        kc, vc = (torch.full((1, 2, 16, 128), 3.0, dtype=BF, device="cuda") for _ in range(2))
        op(None, k, v, i32([0, bad, 5, 63]), rows, kc, vc)
        with pytest.raises(_native.Q4GpuError):
            op.check()
        assert (kc[0, :, 2] == 3).all() and (vc[0, :, 2] == 3).all()
        assert torch.equal(vc[0][:, [3, 1, 0]].transpose(0, 1), v[[0, 2, 3]])
    op = paged.RopeAppend(cos, sin)
    op(None, None, v, None, rows, None, vc)  # values alone have no position
    op.check()
    assert torch.equal(vc[0][:, rows].transpose(0, 1), v)


def grown_args():
    """Forty decodes, a short chunk and a longer one; the split of long decodes and of chunks both need workspace."""
    return make([1] * 40 + [70, 130], [3000] * 3 + [200] * 39, 8, 4, 128, 64, BF, 27)


def part_of(args, ids):
    cu, q = args[3].tolist(), args[4]
    new = [cu[i + 1] - cu[i] for i in ids]
    rows = torch.cat([q[cu[i]:cu[i + 1]] for i in ids])
    return rows, i32([0] + torch.tensor(new).cumsum(0).tolist()), max(new), i32(ids)


def test_attention_captured_decodes_survive_larger_calls():
    """A decode step captured in a graph, then calls that need more workspace, then replays over new inputs; and a
    graph captured by an operator that had no workspace yet."""
    args = grown_args()
    pool, table, lens, cu, q = args
    few, c, most, ids = part_of(args, [0, 1, 7])
    big = part_of(args, list(range(42)))
    fresh = rnd(few.shape, BF, 77)
    for warm in (True, False):
        op = operator(pool, table, lens, 8)
        x, out, lse = few.clone(), torch.empty_like(few), torch.empty(few.shape[:2], device="cuda")
        if warm:
            op(x, out, c, max_q=most, max_ctx=3200, lse=lse, seq_ids=ids)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op(x, out, c, max_q=most, max_ctx=3200, lse=lse, seq_ids=ids)
        for step in (few, fresh):
            x.copy_(step)
            got = op(big[0], None, big[1], max_q=big[2], max_ctx=3200, seq_ids=big[3])
            filler = [torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda") for _ in range(8)]
            graph.replay()
            close(out, lse, *attn_ref(pool, table, lens, c, step, 128 ** -0.5, 0, ids.tolist()), BF)
            ref, mag, _ = attn_ref(pool, table, lens, big[1], big[0], 128 ** -0.5, 0, big[3].tolist())
            within(got, ref, U[BF] * ref.abs() + (U[BF] + 3e-4) * mag)
            assert all((f == 255).all() for f in filler)
        assert not reported(op)


def test_operators_captured_together():
    """A decode step of all operators as one graph."""
    heads, kv, dim, page = 8, 4, 128, 16
    cache = paged.PagedCache(1, 40, page, kv, dim, max_seqs=3, max_ctx=200)
    cos, sin = angles(200, dim)
    rope, attn = paged.RopeAppend(cos, sin), paged.Attention(cache.k(0), cache.v(0), cache.table, cache.lens, heads)
    norm = paged.AddRmsNorm(torch.ones(heads * dim, dtype=BF, device="cuda"))
    cache.pool.normal_()
    cache.extend([0, 1, 2], [100, 17, 1])
    step = cache.extend([0, 1, 2], [1, 1, 1])
    qkv = rnd((3, heads + 2 * kv, dim), BF, 5)
    y, out = torch.empty(3, heads * dim, dtype=BF, device="cuda"), torch.empty(3, heads, dim, dtype=BF, device="cuda")
    turned = torch.empty(3, heads, dim, dtype=BF, device="cuda")

    def run():
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
        rope(q, k, v, step.positions, step.rows, cache.k(0), cache.v(0), turned)
        attn(turned, out, step.cu_q, max_q=1, max_ctx=200, seq_ids=step.seq_ids)
        norm(out.view(3, -1), out=y)

    run()
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)
    qkv.mul_(-0.5)
    graph.replay()
    replayed = y.clone()
    run()
    assert torch.equal(y, replayed) and not torch.equal(y, want)


def test_attention_moves_to_another_stream_and_grows_there():
    args = grown_args()
    pool, table, lens, cu, q = args
    op = operator(pool, table, lens, 8)
    small, big = part_of(args, [0, 1]), part_of(args, list(range(42)))
    op(small[0], None, small[1], max_q=small[2], max_ctx=3200, seq_ids=small[3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(3):
            got = op(big[0], None, big[1], max_q=big[2], max_ctx=3200, seq_ids=big[3])
            op(small[0], None, small[1], max_q=small[2], max_ctx=3200, seq_ids=small[3])
    torch.cuda.current_stream().wait_stream(s)
    ref, mag, _ = attn_ref(pool, table, lens, big[1], big[0], 128 ** -0.5, 0, big[3].tolist())
    within(got, ref, U[BF] * ref.abs() + (U[BF] + 3e-4) * mag)
    assert not reported(op)


@pytest.mark.parametrize("out", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("group,n", [(0, 512), (64, 512), (0, 333)])
@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("size", [3e38, 1e38, 5e-35, 1e-36, 3e-37])
def test_norm_8bit_of_any_magnitude(out, group, n, dtype, size):
    """Groups whose largest value lies near either end of float32.  A scale below 2^-126 is a subnormal number, off by
    up to 2^-150: the tolerance has that times the largest factor."""
    w = (torch.linspace(-1, 1, n, device="cuda", dtype=torch.float64) * size).to(dtype)
    x = torch.ones(3, n, device="cuda", dtype=dtype)
    q, s = paged.AddRmsNorm(w, eps=0.0, out_dtype=out, group=group)(x)
    _, ref = norm_ref(x, None, w, 0.0)
    g = ref.unflatten(-1, (-1, group or n))
    most = 448.0 if out == torch.float8_e4m3fn else 127.0
    want = g.abs().amax(-1) / most
    within(s, want, 2e-5 * want + 2.0 ** -149)
    value = q.double().unflatten(-1, (-1, group or n)) * s.double()[..., None]
    step = 2.0 ** -4 * g.abs() + 2.0 ** -10 * want[..., None] if out == torch.float8_e4m3fn else 0.5 * want[..., None]
    within(value, g, step * (1 + 1e-4) + 3e-5 * g.abs() + most * 2.0 ** -149)


@pytest.mark.parametrize("new", [1, 3, 40, 300])
def test_attention_over_columns_of_a_wider_table(new):
    """A slot's row is as long as the table is wide, whatever lies between the rows."""
    pool, table, lens, cu, q = make([new] * 3, [100, 300, 40], 4, 2, 64, 32, BF, 26)
    pool.nan_to_num_(0.5)  # the unfilled rows of last pages are seen below
    w = table.shape[1]
    wide = torch.zeros(4, 2 * w + 1, dtype=torch.int32, device="cuda")  # its other entries name page 0
    wide[:3, w - 2:2 * w - 2] = table
    part = wide[:3, w - 2:2 * w - 2]
    op = operator(pool, part, lens, 4)
    check(op, pool, table, lens, cu, q, 64 ** -0.5)
    assert not reported(op)
    for s in range(3):
        kept = lens.clone()
        lens[s] = 32 * w + 50  # more than the slot's entries can name: cut off there
        cut = lens.clamp(max=32 * w)
        out, lse = torch.full_like(q, 5.0), torch.full(q.shape[:2], 5.0, device="cuda")
        op(q, out, cu, max_q=new, lse=lse)
        close(out, lse, *attn_ref(pool, table, cut, cu, q, 64 ** -0.5), BF)
        assert reported(op)
        lens.copy_(kept)


@pytest.mark.parametrize("new,held", [(3, 1), (3, 0), (40, 30), (300, 100), (300, 1), (1, 200), (40, 300)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 2, 2 ** 30, 100000])
def test_attention_windows_wider_than_any_context(new, held, window):
    """Also where a slot holds fewer keys than it has queries: differences of positions pass 31 bits."""
    pool, table, lens, cu, q = make([new] * 2, [held, 50], 4, 2, 64, 32, BF, 28)
    lens[0] = held
    out, lse = check(operator(pool, table, lens, 4, window=window), pool, table, lens, cu, q, 64 ** -0.5)
    want = check(operator(pool, table, lens, 4), pool, table, lens, cu, q, 64 ** -0.5)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.parametrize("hq,hk,dim,page", [(16, 8, 128, 64), (7, 1, 64, 16), (8, 4, 64, 128)])
@pytest.mark.parametrize("order", ["page", "split", "one page"])
def test_attention_cache_orders(hq, hk, dim, page, order):
    """Positions before heads in memory ([pages, page_tokens, kv_heads, dim]), K and V in rows of one wider tensor, and
    a pool of one page."""
    one = order == "one page"
    new, old = ([1, 5], [0, 0]) if one else ([1, 3, 40, 300], [300, 17, 5, 200])
    pool, table, lens, cu, q = make(new[:1] if one else new, old[:1] if one else old, hq, hk, dim, page, BF, 29)
    if order == "page":
        kv = [pool[:, i].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for i in (0, 1)]
    elif order == "split":
        wide = torch.empty(pool.shape[0], page, hk, 2, dim, dtype=BF, device="cuda")
        kv = [wide[:, :, :, i].permute(0, 2, 1, 3) for i in (0, 1)]
        for i in (0, 1):
            kv[i].copy_(pool[:, i])
    else:
        page_at = int(table[0, 0])
        table.zero_()
        pool = pool[page_at:page_at + 1].clone()
        kv = [pool[:, 0], pool[:, 1]]
    op = paged.Attention(kv[0], kv[1], table, lens, q_heads=hq)
    check(op, pool, table, lens, cu, q, dim ** -0.5)
    assert not reported(op)


@pytest.mark.parametrize("new", [1, 5, 40, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_heads_that_share_their_keys(new, dim):
    """One key head expanded to four (a head stride of 0)."""
    pool, table, lens, cu, q = make([new] * 2, [300, 20], 8, 1, dim, 32, BF, 30)
    k, v = (pool[:, i].expand(-1, 4, -1, -1) for i in (0, 1))
    op = paged.Attention(k, v, table, lens, q_heads=8)
    check(op, pool, table, lens, cu, q, dim ** -0.5)


@pytest.mark.parametrize("new,old", [(1, 300), (3, 300), (50, 300), (400, 300), (40, 3000)])
@pytest.mark.parametrize("what", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("window", [0, 90])
def test_attention_infinite_values_reach_the_queries_that_see_them(new, old, what, window):
    """Keys stay finite; one value of one key is not.  The queries that see it have it in that column (its weight is far
    above the least bf16 number), and nothing else changes."""
    args = make([new], [old], 4, 2, 128, 64, BF, 31)
    pool, table, lens, cu, q = args
    op = operator(pool, table, lens, 4, window=window)
    clean, base = check(op, *args, 128 ** -0.5, window)
    for at in sorted({old + new // 2, old, max(0, old - 60), old + new - 1}):
        kept = pool[table[0, at // 64], 1, 1, at % 64, 5].item()
        pool[table[0, at // 64], 1, 1, at % 64, 5] = what  # key head 1: query heads 2 and 3
        lse = torch.empty_like(base)
        out = op(q, None, cu, max_q=new, max_ctx=old + new, lse=lse)
        pos = torch.arange(old, old + new, device="cuda")
        sees = (pos >= at) & ((pos - window < at) if window else (pos >= 0))
        hit = out[sees][:, 2:, 5]
        assert hit.isnan().all() if math.isnan(what) else (hit == what).all()
        out[:, 2:, 5] = torch.where(sees[:, None], clean[:, 2:, 5], out[:, 2:, 5])
        assert torch.equal(out, clean) and torch.equal(lse, base)
        pool[table[0, at // 64], 1, 1, at % 64, 5] = kept


def test_rope_remembers_a_layout_not_its_tensors():
    """One object called again and again: the same layout at other addresses, other layouts between, errors between."""
    cos, sin = angles(300, 128)
    g = rnd((128,), BF, 3) + 1
    op = paged.RopeAppend(cos, sin, q_gamma=g, k_gamma=g)

    def one(tokens, hq, hk, page, seed, wide=0, q_out=True):
        qkv = rnd((tokens, hq + 2 * hk + wide, 128), BF, seed)
        q, k, v = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:hq + 2 * hk]
        kc, vc = (torch.zeros(8, hk, page, 128, dtype=BF, device="cuda") for _ in range(2))
        pos = torch.randint(0, 300, (tokens,), device="cuda", dtype=torch.int32)
        rows = torch.randperm(8 * page, device="cuda")[:tokens].contiguous()
        want = [rope(t.clone(), pos) for t in (q, k)] + [v.clone()]
        got = op(q, k, v, pos, rows, kc, vc, torch.empty_like(q) if q_out else None)
        turned(got, *want[0])
        turned(kc[rows // page, :, rows % page], *want[1])
        assert torch.equal(vc[rows // page, :, rows % page], want[2])

    def rope(x, pos):
        return rope_ref(x, g, cos, sin, pos.long(), False, 1e-6)

    def turned(got, want, m):
        within(got, want, U[BF] * want.abs() + 1e-5 * m + TINY[BF])

    for seed in range(3):
        one(5, 4, 2, 16, seed)
        one(5, 4, 2, 16, 10 + seed)
        one(5, 4, 2, 16, 20 + seed, wide=1)  # other strides
        one(5, 4, 2, 16, 30 + seed, q_out=False)
        with pytest.raises(ValueError):
            op(rnd((5, 4, 128), BF, 1), rnd((5, 2, 128), HF, 1), None, None, None, None, None)
        one(5, 4, 2, 16, 40 + seed)
        one(6, 2, 4, 32, 50 + seed)
    op.check()


def test_attention_mixed_step_captured():
    """Decodes, a short chunk and a split chunk in one call: both kernels and the join, replayed over new queries."""
    args = grown_args()
    pool, table, lens, cu, q = args
    for ids in (list(range(42)), [0, 41], [41], [2]):
        x, c, most, slots = part_of(args, ids)
        op = operator(pool, table, lens, 8)
        out, lse = torch.empty_like(x), torch.empty(x.shape[:2], device="cuda")
        op(x, out, c, max_q=most, max_ctx=3200, lse=lse, seq_ids=slots)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op(x, out, c, max_q=most, max_ctx=3200, lse=lse, seq_ids=slots)
        for seed in (61, 62):
            x.copy_(rnd(x.shape, BF, seed))
            out.zero_()
            graph.replay()
            close(out, lse, *attn_ref(pool, table, lens, c, x, 128 ** -0.5, 0, ids), BF)
        assert not reported(op)


@pytest.mark.parametrize("n", [-1, 3 * 16 + 1, 2 ** 31 - 1])
def test_pages_report_lengths_that_no_row_of_the_table_holds(n):
    pool, table, lens = pages_of(8, 2, 16, 8, 4, 3)
    table[0, 0], lens[0] = 5, 7
    table[1] = i32([1, 2, 3])
    lens[1] = n
    before, tb, kept = pool.clone(), table.clone(), lens.clone()
    op = paged.Pages(pool, table, lens, 16)
    op.fork(i32([1]), i32([2]), i32([4]))
    assert reported(op)
    assert torch.equal(pool, before) and torch.equal(table, tb) and torch.equal(lens, kept)
    op.fork(i32([0]), i32([2]), i32([4]))
    assert not reported(op) and int(lens[2]) == 7
    for new in (torch.empty_like(table), table):
        op.compact(new, torch.empty(8, dtype=torch.int32, device="cuda"), i32([0]))
        assert reported(op)
    lens[1] = 0
    op.compact(torch.empty_like(table), torch.empty(8, dtype=torch.int32, device="cuda"), i32([0]))
    assert not reported(op)
