"""Attention of sequences that share their first keys against a plain 64-bit form.

Bounds are those of ``test_gpu_paged``: |error| <= u |out| + (u + 3e-4) sum_j p_j |v_j| with the unit
roundoff u of the result's type, and 3e-4 for the log-sum; joining the two parts of a row adds a few
roundings in 32 bits, far below that.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402
from test_gpu_paged import BF, HF, TINY, U, i32, rnd, within  # noqa: E402


class Case:
    """Groups of (shared keys, [(queries, own keys, those of the queries included), ..]).  Pages are shuffled; rows
    that nobody may read are NaN: page tails, and the shared rows of all but a group's first sequence (whose
    pages of shared keys alone are not there at all)."""

    def __init__(self, groups, hq, hk, dim, page, dtype, seed=0):
        g = torch.Generator().manual_seed(seed)
        members = [(p, first == 0, n, own) for p, seqs in groups for first, (n, own) in enumerate(seqs)]
        self.lens_h = [p + own for p, _, _, own in members]
        need = [-(-n // page) for n in self.lens_h]
        total = sum(need) + 2
        self.pool = torch.full((total, 2, hk, page, dim), math.nan, dtype=dtype, device="cuda")
        ids = torch.randperm(total, generator=g).tolist()
        table, self.kv, shared = [], [], None
        for i, (p, first, n, own) in enumerate(members):
            if first:
                shared = rnd((2, hk, p, dim), dtype, seed * 1000 + 500 + i)
            kv = torch.cat((shared, rnd((2, hk, own, dim), dtype, seed * 1000 + i)), 2)
            self.kv.append(kv)
            mine = ids[:need[i]]
            ids = ids[need[i]:]
            lo = 0 if first else p
            for j in range(lo // page, need[i]):
                a, b = max(lo, j * page), min(self.lens_h[i], (j + 1) * page)
                self.pool[mine[j], :, :, a - j * page:b - j * page] = kv[:, :, a:b]
            table.append([-1] * (lo // page) + mine[lo // page:] + [-1] * (max(need + [1]) - need[i]))
        self.new = [n for _, _, n, _ in members]
        self.table, self.lens = i32(table), i32(self.lens_h)
        self.cu_h = [0]
        for n in self.new:
            self.cu_h.append(self.cu_h[-1] + n)
        self.cu = i32(self.cu_h)
        ends = [0]
        for _, seqs in groups:
            ends.append(ends[-1] + len(seqs))
        self.ends, self.prefix = i32(ends), i32([p for p, _ in groups])
        self.q = rnd((self.cu_h[-1], hq, dim), dtype, seed + 5)
        self.page, self.max_ctx = page, max(self.lens_h + [1])

    def op(self, **kw):
        return paged.SharedAttention(self.pool[:, 0], self.pool[:, 1], self.table, self.lens, self.q.shape[1], **kw)

    def run(self, op=None, err=0, **kw):
        op = op or self.op()
        lse = torch.full(self.q.shape[:2], 5.0, device="cuda")
        out = torch.full_like(self.q, 5.0)
        args = dict(max_q=max(self.new + [1]), max_ctx=self.max_ctx, lse=lse) | kw
        assert op(self.q, out, self.cu, self.ends, self.prefix, **args) is out
        assert int(op.err.item()) == err
        return out, lse

    def ref(self, scale=None):
        q = self.q
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        mag, lse = torch.zeros_like(out), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
        for i, n in enumerate(self.new):
            ctx, at = self.lens_h[i], slice(self.cu_h[i], self.cu_h[i + 1])
            if n == 0 or ctx == 0:
                continue
            k, v = (x.double().repeat_interleave(q.shape[1] // x.shape[0], 0) for x in self.kv[i])
            pos = torch.arange(ctx - n, ctx, device="cuda")[:, None]
            unseen = torch.arange(ctx, device="cuda")[None] > pos
            sc = (q[at].double().permute(1, 0, 2) @ k.transpose(1, 2) * (scale or q.shape[2] ** -0.5)).masked_fill(
                unseen, -math.inf)
            p = torch.softmax(sc, -1).nan_to_num(0.0)
            out[at], mag[at] = (p @ v).permute(1, 0, 2), (p @ v.abs()).permute(1, 0, 2)
            lse[at] = torch.logsumexp(sc, -1).permute(1, 0)
        return out, mag, lse

    def check(self, op=None, scale=None, **kw):
        got = self.run(op, **kw)
        close(*got, *self.ref(scale))
        return got


def close(out, lse, want, mag, rl):
    u = U[out.dtype]
    within(out, want, u * want.abs() + (u + 3e-4) * mag + TINY[out.dtype])
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none)
    within(lse[~none], rl[~none], 3e-4 + 1e-6 * rl[~none].abs())


HEADS = [(16, 8, 128, 64), (4, 4, 64, 16), (7, 1, 128, 32), (28, 4, 64, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
@pytest.mark.parametrize("prefix", [0, 1, 16, 63, 64, 100, 128, 1000, 1024])
def test_one_group_of_single_tokens(dtype, hq, hk, dim, page, prefix):
    own = [1, 2, 15, 16, 17, 40, 64, 65, 130, 600, 1, 1]
    Case([(prefix, [(1, n) for n in own])], hq, hk, dim, page, dtype, 1).check()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hk,dim,page", HEADS)
@pytest.mark.parametrize("tokens", [2, 9, 17, 150])
def test_groups_of_all_kinds(dtype, hq, hk, dim, page, tokens):
    """Several queries a sequence; groups of one, without shared keys, of many; sequences without queries."""
    t = tokens
    Case([(500, [(t, t + 3), (1, 1), (t, t), (0, 77)]), (0, [(1, 30), (t, t + 200)]), (130, [(1, 5)]),
          (64, [(1, 1)] * 30), (2000, [(0, 5), (0, 9)]), (33, [(t, t + 700), (0, 0), (1, 900), (2, 2)])],
         hq, hk, dim, page, dtype, 2).check()


@pytest.mark.parametrize("hq,hk,dim,page", [(16, 8, 128, 64), (8, 1, 64, 32), (2, 1, 128, 128), (40, 1, 64, 64)])
@pytest.mark.parametrize("prefix,seqs", [(9000, 2), (5000, 9), (4096, 64), (700, 300), (10, 100)])
def test_long_prefixes_and_many_sequences(hq, hk, dim, page, prefix, seqs):
    case = Case([(prefix, [(1, 1 + 7 * i % 50) for i in range(seqs)])], hq, hk, dim, page, BF, 3)
    a = case.check()
    b = case.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # the joining order is fixed


@pytest.mark.parametrize("seqs", [1, 3])
def test_long_chunks_after_a_prefix(seqs):
    """Own keys that are split over CTAs as well."""
    Case([(3000, [(300, 2500)] * seqs)], 4, 1, 64, 32, HF, 4).check()
    Case([(3000, [(40, 6000)] * seqs)], 4, 2, 128, 64, BF, 4).check()


def test_the_same_numbers_as_separate_attention():
    """Against the operator that reads every sequence's keys for itself, over tables that name the same pages."""
    case = Case([(640, [(1, 20), (3, 70), (1, 1)]), (128, [(2, 9), (1, 400)])], 16, 8, 128, 64, BF, 5)
    out, lse = case.check()
    table = case.table.clone()
    table[1:3, :10], table[4:, :2] = table[0, :10], table[3, :2]
    plain = paged.Attention(case.pool[:, 0], case.pool[:, 1], table, case.lens, 16)
    l2 = torch.empty_like(lse)
    want = plain(case.q, None, case.cu, max_q=3, lse=l2)
    close(out, lse, want.double(), want.double().abs() + 1.0, l2.double())


@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_infinities_reach_only_those_who_see_them(new, what):
    groups = [(200, [(new, new + 30), (new, new + 3)]), (70, [(new, new)])]
    case = Case(groups, 4, 2, 64, 32, BF, 6)
    clean, _ = case.run()
    first = case.table[0]
    case.pool[first[100 // 32], 1, 1, 100 % 32] = what  # the value of a shared key, of the second key head
    out, _ = case.run()
    a, b = case.cu_h[2], case.cu_h[1]
    assert torch.equal(out[a:], clean[a:]) and torch.equal(out[:, :2], clean[:, :2])
    assert not out[:a, 2:].isfinite().any()
    case = Case(groups, 4, 2, 64, 32, BF, 6)
    case.pool[case.table[1, 202 // 32], 1, :, 202 % 32] = what  # the last own key of the second sequence, if new is 1
    out, _ = case.run()
    assert torch.equal(out[:b], clean[:b]) and torch.equal(out[a:], clean[a:])
    assert not out[a - 1].isfinite().any()


@pytest.mark.parametrize("group,hk", [(2, 2), (1, 1), (20, 1)])
@pytest.mark.parametrize("new", [1, 30])
def test_out_of_range_is_reported(group, hk, new):
    """Queries among the shared keys, unknown slots, missing pages, more queries than max_q, offsets out of order."""
    def fresh():
        return Case([(200, [(new, new + 10), (new, new + 1), (new, new + 40)]), (64, [(new, new)])], group * hk, hk, 64,
                    32, BF, 7)

    def others(case, got, gone):
        want, mag, rl = case.ref()
        for i in range(4):
            at = slice(case.cu_h[i], case.cu_h[i + 1])
            if i in gone:
                assert not got[0][at].any() and (got[1][at] == -math.inf).all()
            else:
                close(got[0][at], got[1][at], want[at], mag[at], rl[at])

    case = fresh()
    case.lens[1] = 200 + new - 1  # a query among the shared keys
    others(case, case.run(err=1), [1])
    case = fresh()
    others(case, case.run(err=1, seq_ids=i32([0, 1, 9, 3])), [2])
    others(case, case.run(err=1, seq_ids=i32([0, -1, 2, 3])), [1])
    if new > 1:
        case = fresh()
        case.cu_h = [0, new, 2 * new, 3 * new, 4 * new]
        got = case.run(err=1, max_q=new - 1)
        assert not got[0].any() and (got[1] == -math.inf).all()
    for bad in ([0, 3, 2], [0, 3, 5], [-1, 3, 4], [2, 1, 4]):
        case = fresh()
        case.ends = i32(bad)
        got = case.run(err=1)
        assert not got[0].any() and (got[1] == -math.inf).all()
    case = fresh()
    case.cu = i32([0, new, 0, 3 * new, 4 * new])
    got = case.run(err=1)
    assert not got[0][:1].any()
    case = fresh()
    case.prefix[1] = -5  # nothing shared, the fourth sequence's pages hold all its keys
    others(case, case.run(err=1), [])
    case = fresh()
    case.table[3, 0] = case.pool.shape[0]  # keys 0 .. 31 of the second group: not there
    case.kv[3] = case.kv[3][:, :, 32:]
    case.lens_h[3] -= 32
    others(case, case.run(err=1), [])
    op = case.op()
    case.run(op, err=1)
    with pytest.raises(_native.Q4GpuError):
        op.check()


def test_first_sequence_without_enough_keys():
    """The shared keys that are there count."""
    case = Case([(200, [(0, 0), (1, 40)])], 4, 2, 64, 32, BF, 8)
    case.lens[0] = 130
    got = case.run(err=1)
    case.kv[1] = torch.cat((case.kv[1][:, :, :130], case.kv[1][:, :, 200:]), 2)
    case.lens_h[1] -= 70
    close(*got, *case.ref())


def test_sequences_in_no_group_and_slots_out_of_order():
    case = Case([(100, [(1, 20)]), (300, [(1, 7), (2, 9)]), (50, [(1, 60)])], 8, 2, 128, 32, HF, 9)
    case.table[3, :2] = case.table[3, :2].clamp(min=0)
    case.ends, case.prefix = i32([1, 3]), i32([300])  # the first and the last stand alone
    case.check()
    perm = [2, 0, 3, 1]  # slot of each sequence
    where = torch.tensor(perm, device="cuda")
    table, lens = torch.empty_like(case.table), torch.empty_like(case.lens)
    table[where], lens[where] = case.table, case.lens
    case.table, case.lens = table, lens
    case.check(seq_ids=i32(perm))
    case.ends, case.prefix = i32([0]), i32([])  # no groups at all
    got = case.op()(case.q, None, case.cu, case.ends, case.prefix, max_q=2, seq_ids=i32(perm))
    assert torch.isfinite(got[:1]).all()


def test_rows_behind_the_last_sequence_stay():
    case = Case([(100, [(1, 20), (1, 3)])], 4, 2, 64, 32, BF, 10)
    q = torch.cat((case.q, case.q[:1]))
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    case.op()(q, out, case.cu, case.ends, case.prefix, lse=lse)
    assert (out[2:] == 7.0).all() and (lse[2:] == 7.0).all()
    close(out[:2], lse[:2], *case.ref())


def test_strides_streams_and_scales():
    case = Case([(333, [(2, 20), (1, 3), (30, 31)])], 8, 2, 64, 32, HF, 11)
    tokens = case.q.shape[0]
    wide = torch.full((tokens, 10, 192), math.nan, dtype=HF, device="cuda")
    q, out = wide[:, :8, :64], wide[:, 1:9, 64:128]
    q.copy_(case.q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for scale in (0.3, -0.2):
        op = case.op(scale=scale)
        with torch.cuda.stream(side):
            lse = torch.empty(tokens, 8, device="cuda")
            op(q, out, case.cu, case.ends, case.prefix, max_q=30, lse=lse)
        torch.cuda.current_stream().wait_stream(side)
        close(out, lse, *case.ref(scale))


def test_one_operator_for_calls_of_all_shapes():
    """The workspace grows and is left as the next call needs it."""
    case = Case([(900, [(1, 5)] * 40), (64, [(150, 200)])], 8, 2, 128, 64, BF, 12)
    op = case.op()
    for _ in range(2):
        case.check(op)
        few, n = i32(case.cu_h[:3]), 2
        lse = torch.empty(n, 8, device="cuda")
        out = op(case.q[:n], None, few, i32([0, 2]), i32([900]), lse=lse)
        close(out, lse, *(x[:n] for x in case.ref()))


def test_captured_with_growing_lengths():
    case = Case([(256, [(1, 60), (1, 64), (1, 20)]), (0, [(1, 70)])], 8, 2, 128, 64, BF, 13)
    op, full = case.op(), case.lens.clone()
    out, lse = torch.empty_like(case.q), torch.empty(case.q.shape[:2], device="cuda")
    kv = list(case.kv)

    def call():
        op(case.q, out, case.cu, case.ends, case.prefix, max_ctx=384, max_prefix=256, lse=lse)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for left in (59, 19, 1, 0):
        case.lens.copy_(torch.clamp(full - left, min=i32([257, 257, 257, 1])))
        case.lens_h = case.lens.tolist()
        case.kv = [x[:, :, :n] for x, n in zip(kv, case.lens_h)]
        graph.replay()
        close(out, lse, *case.ref())
    op.check()


def test_first_call_captured():
    """A graph whose call wants more workspace than there is."""
    case = Case([(700, [(1, 60)] * 30)], 8, 2, 64, 64, BF, 14)
    op = case.op()
    out, lse = torch.empty_like(case.q), torch.empty(case.q.shape[:2], device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(case.q, out, case.cu, case.ends, case.prefix, lse=lse)
    case.check(op)
    for _ in range(2):
        out.zero_()
        graph.replay()
        close(out, lse, *case.ref())


def test_nothing_to_do():
    case = Case([(100, [(1, 20)])], 4, 2, 64, 32, BF, 15)
    op = case.op()
    assert op(case.q[:0], None, i32([0, 0]), case.ends, case.prefix).shape == (0, 4, 64)
    assert op(case.q[:0], None, i32([0]), i32([0]), i32([])).shape == (0, 4, 64)
    case.check(op)


def test_refusals():
    case = Case([(100, [(1, 20), (1, 1)])], 4, 2, 64, 32, BF, 16)
    op = case.op()
    q, cu, ends, pre = case.q, case.cu, case.ends, case.prefix
    for bad in (lambda: op(q, None, cu), lambda: op(q, None, cu, ends), lambda: op(q, None, None, ends, pre),
                lambda: op(q, None, cu, ends.long(), pre), lambda: op(q, None, cu, ends, pre.long()),
                lambda: op(q, None, cu, ends.cpu(), pre), lambda: op(q, None, cu, ends, i32([1, 2])),
                lambda: op(q, None, cu, ends[:0], pre), lambda: op(q[:, :2], None, cu, ends, pre),
                lambda: op(q.float(), None, cu, ends, pre), lambda: op(q, q.float(), cu, ends, pre),
                lambda: op(q, None, i32([0, 1, 2, 2]), ends, pre)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_native.Q4GpuError):
        op(q, None, cu, ends, pre, max_prefix=-1)
    case.check(op)
