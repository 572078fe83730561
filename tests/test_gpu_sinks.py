"""Attention through a window with sinks against a plain 64-bit form.

Bounds are those of ``test_gpu_paged``: |error| <= u |out| + (u + 3e-4) sum_j p_j |v_j|
with the unit roundoff u of the result's type, and 3e-4 for the log-sum.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402
from test_gpu_paged import BF, HF, TINY, U, i32, make, within  # noqa: E402


def ref(pool, table, lens, cu, q, window, sinks, scale=None):
    hk, page, dim = pool.shape[2], pool.shape[3], pool.shape[4]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    mag, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    cu, lens, tab = cu.tolist(), lens.tolist(), table.tolist()
    for i in range(len(cu) - 1):
        n, ctx = cu[i + 1] - cu[i], lens[i]
        if n == 0 or ctx <= 0:
            continue
        rows = tab[i][:-(-ctx // page)]
        ok = torch.tensor([0 <= p < pool.shape[0] for p in rows], device="cuda").repeat_interleave(page)[:ctx]
        ids = torch.tensor([max(0, min(p, pool.shape[0] - 1)) for p in rows], device="cuda")
        kv = pool[ids].double().permute(1, 2, 0, 3, 4).reshape(2, hk, -1, dim)[:, :, :ctx]
        pos = torch.arange(ctx - n, ctx, device="cuda")[:, None]
        key = torch.arange(ctx, device="cuda")[None]
        seen = (key <= pos) & ok[None] & ((key > pos - window) | (key < sinks))
        kv = torch.where(seen.any(0)[None, None, :, None], kv, 0.0)
        k, v = (x.repeat_interleave(q.shape[1] // hk, 0) for x in kv)
        sc = q[cu[i]:cu[i + 1]].double().permute(1, 0, 2) @ k.transpose(1, 2) * (scale or dim ** -0.5)
        sc.masked_fill_(~seen, -math.inf)
        some = seen.any(-1)
        l = torch.logsumexp(sc, -1)
        p = torch.where(seen & some[:, None], (sc - torch.where(some, l, 0.0)[..., None]).exp(), 0.0)
        out[cu[i]:cu[i + 1]] = (p @ v).permute(1, 0, 2)
        mag[cu[i]:cu[i + 1]] = (p @ v.abs()).permute(1, 0, 2)
        lse[cu[i]:cu[i + 1]] = l.permute(1, 0)
    return out, mag, lse


def attend(pool, table, lens, cu, q, window, sinks, scale=None, err=0):
    new = (cu[1:] - cu[:-1]).max().item()
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=q.shape[1], window=window, sinks=sinks,
                         scale=scale)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device="cuda")
    out = op(q, None, cu, max_q=new, max_ctx=max(int(lens.max()), 1), lse=lse)
    assert int(op.err.item()) == err
    return out, lse


def check(pool, table, lens, cu, q, window, sinks, scale=None, err=0):
    out, lse = attend(pool, table, lens, cu, q, window, sinks, scale, err)
    want, mag, rl = ref(pool, table, lens, cu, q, window, sinks, scale)
    u = U[q.dtype]
    within(out, want, u * want.abs() + (u + 3e-4) * mag + TINY[q.dtype])
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none)
    within(lse[~none], rl[~none], 3e-4 + 1e-6 * rl[~none].abs())
    return out, lse


def off(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


HEADS = [(16, 8, 128, 64), (4, 4, 64, 16), (7, 1, 128, 32), (8, 1, 64, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 1), (16, 4), (100, 37), (128, 128), (500, 130), (33, 1000)])
def test_single_tokens(dtype, hq, hk, dim, page, window, sinks):
    old = [0, 1, 15, 16, 17, 40, 63, 64, 127, 128, 129, 160, 300, 639, 640, 1023, 1500, 2000]
    check(*make([1] * len(old), old, hq, hk, dim, page, dtype, 1), window, sinks)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
@pytest.mark.parametrize("window,sinks", [(1, 1), (64, 4), (129, 37), (300, 128), (200, 500)])
def test_chunks(dtype, hq, hk, dim, page, window, sinks):
    new = [1, 2, 0, 17, 63, 64, 130, 300, 1, 5]
    old = [0, 900, 70, 200, 640, 0, 129, 1000, 1500, 333]
    check(*make(new, old, hq, hk, dim, page, dtype, 2), window, sinks)


@pytest.mark.parametrize("new,old", [([1], [9000]), ([200], [9000]), ([1, 600], [2500, 7000]), ([2300], [0])])
@pytest.mark.parametrize("window,sinks", [(4000, 4), (5000, 700), (100, 2000)])
def test_long(new, old, window, sinks):
    """One sequence or two, whose walk over the keys is split and joined."""
    args = make(new, old, 4, 2, 128, 64, BF, 3)
    a = check(*args, window, sinks)
    b = attend(*args, window, sinks)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("new", [1, 40, 300])
def test_everything_visible_is_plain_attention(new):
    """A window or sinks that leave nothing out: the same numbers as without them."""
    pool, table, lens, cu, q = make([new, new], [130, 700], 4, 2, 64, 32, BF, 4)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=4)
    want = op(q, None, cu, max_q=new, max_ctx=int(lens.max()))  # which decides how the keys are split
    assert torch.equal(attend(pool, table, lens, cu, q, 2 ** 31 - 1, 5)[0], want)
    check(pool, table, lens, cu, q, 10, 2 ** 31 - 1)


@pytest.mark.parametrize("new", [1, 40, 300])
def test_pages_between_are_not_read(new):
    """Pages between the sinks and every window may be gone; missing pages of seen keys hold none and are reported."""
    pool, table, lens, cu, q = make([new, new], [2000, 1900], 4, 2, 64, 32, BF, 5)
    want, _ = check(pool, table, lens, cu, q, 100, 40)
    gone = table.clone()
    gone[:, 2:(1900 - 100) // 32] = -1
    pool[table[:, 2:(1900 - 100) // 32].flatten().long()] = math.nan
    assert torch.equal(attend(pool, gone, lens, cu, q, 100, 40)[0], want)
    gone[1, 1] = -1  # keys 32 .. 39 are sinks
    check(pool, gone, lens, cu, q, 100, 40, err=1)
    gone[0, 0] = pool.shape[0]
    gone[1, 60] = -1
    check(pool, gone, lens, cu, q, 100, 40, err=1)


@pytest.mark.parametrize("new", [1, 50, 400])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_unseen_and_seen_infinities(new, what):
    args = make([new], [1000], 4, 2, 128, 64, BF, 7)
    pool, table = args[:2]
    want, _ = attend(*args, 20, 6)
    for at in (6, 7, 63, 64, 500, 1000 - 20):  # neither a sink nor in any window
        pool[table[0, at // 64], :, :, at % 64] = what
    assert torch.equal(attend(*args, 20, 6)[0], want)
    pool[table[0, 0], 1, 1, 5] = what  # the value of a sink that all queries see, of the second key head
    out, _ = attend(*args, 20, 6)
    assert torch.equal(out[:, :2], want[:, :2])
    assert not out[:, 2:].isfinite().any()
    if what == what:
        assert (out[:, 2:] == what).all()


@pytest.mark.parametrize("new", [1, 3, 40])
def test_empty_rows(new):
    """Fewer stored keys than queries, none at all."""
    pool, table, lens, cu, q = make([new] * 3, [200, 100, 50], 4, 2, 64, 32, BF, 6)
    lens[1], lens[2] = max(0, new - 3), 0
    out, _ = check(pool, table, lens, cu, q, 7, 3)
    assert not out[cu[2]:].any()


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("seqs", [3, 200])  # more than the kernels keep in shared memory
def test_out_of_range_is_reported(new, seqs):
    """Unknown slots, lengths that the table cannot hold, more queries than max_q, offsets past the tokens."""
    def fresh():
        return make([new] * seqs, [90] * seqs, 4, 2, 64, 32, BF, 11)

    def call(max_q=new, seq_ids=None, cu=None, lens=None):
        pool, table, lens0, cu0, q = fresh()
        lens = lens0 if lens is None else lens
        op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=4, window=20, sinks=3)
        lse = torch.full(q.shape[:2], 5.0, device="cuda")
        out = op(q, torch.full_like(q, 5.0), cu0 if cu is None else cu, max_q=max_q, max_ctx=512, lse=lse,
                 seq_ids=seq_ids)
        return out, lse, int(op.err.item())

    pool, table, lens, cu, q = fresh()
    want, lse = attend(pool, table, lens, cu, q, 20, 3)
    ids = list(range(seqs))
    for bad in (-1, seqs):
        out, l, err = call(seq_ids=i32([ids[0], bad] + ids[2:]))
        assert err == 1 and not out[new:2 * new].any() and (l[new:2 * new] == -math.inf).all()
        assert off(out[:new], want[:new]) < 0.01 and off(out[2 * new:], want[2 * new:]) < 0.01
    long = lens.clone()
    long[1] = 10 ** 6
    out, _, err = call(lens=long)
    assert err == 1 and off(out[:new], want[:new]) < 0.01 and out.isfinite()[:new].all()
    ends = cu.clone()
    ends[-1] += 5
    out, _, err = call(cu=ends)
    assert err == 1 and off(out, want) < 0.01
    if new > 1:
        out, l, err = call(max_q=new - 1)
        assert err == 1 and all(off(out[a:b], want[a:b]) < 0.01 or not out[a:b].any()
                                for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()))


def test_captured_with_growing_lengths():
    """One graph, replayed as the sequences grow past their window."""
    pool, table, lens, cu, q = make([1, 1], [300, 900], 8, 2, 128, 64, BF, 8)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=8, window=64, sinks=4)
    out = torch.empty_like(q)
    op(q, out, cu, max_q=1, max_ctx=1024)
    full = lens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(q, out, cu, max_q=1, max_ctx=1024)
    for a, b in ((1, 5), (64, 65), (70, 200), (300, 901)):
        lens.copy_(i32([min(a, int(full[0])), b]))
        graph.replay()
        want, mag, _ = ref(pool, table, lens, cu, q, 64, 4)
        within(out, want, U[BF] * want.abs() + (U[BF] + 3e-4) * mag)
    op.check()


def test_refusals():
    pool, table, lens, cu, q = make([1], [100], 4, 2, 64, 32, BF, 9)
    where = pool[:, 0], pool[:, 1], table, lens, 4
    for bad in (dict(window=0, sinks=1), dict(window=4, sinks=-1), dict(window=4, sinks=2 ** 31)):
        with pytest.raises(ValueError):
            paged.Attention(*where, **bad)
    a = paged.Attention(*where, window=4, sinks=2)
    a(q, None, cu)
    assert a.lib.q4gpu_sink_attention(a.args, -1, None) == -1001
    a.args.workspace_bytes = 16
    assert a.lib.q4gpu_sink_attention(a.args, 2, None) == -1005
    with pytest.raises(_native.Q4GpuError):
        paged.Attention(*where, window=-1)(q, None, cu)
