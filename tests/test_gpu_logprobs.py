"""Token log probabilities, entropy, ranks and likeliest tokens against plain 64-bit forms.

With m a row's largest logit, S the sum of e^(x - m) over the others and T = sum e^(x - m) (x - m):
log p_t = (x_t - m) - log1p(S) and H = log1p(S) - T / (1 + S).  In 32 bits a term e^d is off by at most
2^-22 + |d| 2^-22 of itself (the exponential's, and two roundings of its argument), and a sum of n terms by n
threads' shares, at most n / 128 + 64 additions one after another, by 2^-24 for each.  So with
s = sum e^d (1 + |d|) 2^-22 + (n / 128 + 64) 2^-24 S over the others and t likewise with the weights |d|:
  |error of log1p(S)| <= s / (1 + S) + 2^-22 log1p(S),
  |error of log p|    <= that + 2^-22 |x_t - m|,
  |error of H|        <= that + t / (1 + S) + 2 |T| s / (1 + S)^2 + 2^-22 |T| / (1 + S).
Whole numbers are exact."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def rnd(shape, dtype, seed=0, std=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def targets_of(rows, vocab, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(0, vocab, (rows,), device="cuda", generator=g)


def order(x):
    """Numbers by which logits are ranked: NaN above all."""
    return torch.where(x.isnan(), torch.full_like(x, math.inf), x), x.isnan()


def ref(x, targets, top):
    """(logprob, its bound, entropy, its bound, rank, top_logprob, bound, top_index) of finite or -infinite rows."""
    n = x.shape[1]
    x = x.double()
    m, best = x.max(-1, keepdim=True)
    none = (m == -math.inf).squeeze(1)
    d = torch.where(none[:, None], 0.0, x - m)
    e = d.exp()
    dd = torch.where(e > 0, d, 0.0)
    others = torch.arange(n, device="cuda")[None] != best
    S = torch.where(others, e, 0.0).sum(-1)
    T = (e * dd).sum(-1)
    more = (n / 128 + 64) * 2.0 ** -24
    s = torch.where(others, e * (1 + dd.abs()), 0.0).sum(-1) * 2.0 ** -22 + more * S
    t = (e * dd.abs() * (1 + dd.abs())).sum(-1) * 2.0 ** -22 + more * T.abs()
    norm = S.log1p()
    tol = s / (1 + S) + 2.0 ** -22 * norm
    H = torch.where(none, 0.0, norm - T / (1 + S))
    tol_h = tol + t / (1 + S) + 2 * T.abs() * s / (1 + S) ** 2 + 2.0 ** -22 * T.abs() / (1 + S)

    def logp(at):
        v = x.gather(1, at) - torch.where(none[:, None], 0.0, m)
        return v - norm[:, None], tol[:, None] + 2.0 ** -22 * torch.where(v == -math.inf, 0.0, v).abs()

    sure = targets.clamp(0, n - 1)[:, None]
    known = (targets >= 0) & (targets < n)
    lp, lp_tol = (torch.where(known, v.squeeze(1), 0.0) for v in logp(sure))
    mine = x.gather(1, sure)
    place = torch.arange(n, device="cuda")[None]
    rank = torch.where(known, 1 + ((x > mine) | ((x == mine) & (place < sure))).sum(-1), 0)
    index = x.sort(stable=True, dim=-1, descending=True).indices[:, :top]
    return lp, lp_tol, H, tol_h, rank, *logp(index), index


def within(got, want, tol):
    same = (got == want.float()) | ((got.double() - want).abs() <= tol)
    assert same.all(), f"{int((~same).sum())} of {same.numel()} off"


def check(x, targets, top, op=None, out=None, err=0):
    op = op or paged.TokenLogprobs(top=top)
    got = op(x, targets, out)
    lp, lp_tol, H, tol_h, rank, tlp, tlp_tol, index = ref(x, targets, top)
    assert torch.equal(got.rank.long(), rank)
    assert torch.equal(got.top_index.long(), index)
    within(got.logprob, lp, lp_tol)
    within(got.entropy, H, tol_h)
    within(got.top_logprob, tlp, tlp_tol)
    assert int(op.err.item()) == err
    return got


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (1, 31), (5, 32), (2, 33), (7, 257), (300, 1000), (1, 4096),
                                        (4, 4099), (150, 8191), (2, 32768), (17, 32001), (1, 151936), (9, 151936),
                                        (70, 50257), (500, 12345)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows(dtype, rows, vocab, top):
    check(rnd((rows, vocab), dtype, rows + vocab), targets_of(rows, vocab), min(top, vocab))


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("std", [1e-3, 0.3, 30.0, 1000.0])
def test_flat_and_certain_rows(dtype, std):
    """From rows without a preference to rows whose entropy is far below the type's step at 1."""
    x = rnd((40, 5000), dtype, 3, std)
    x[::2, 77] = x[::2].amax(-1) + torch.tensor([2.0 ** (i - 6) for i in range(20)], device="cuda").to(dtype)
    check(x, targets_of(40, 5000), 20)
    check(x, torch.full((40,), 77, device="cuda"), 3)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("vocab", [40, 3000, 151936])
@pytest.mark.parametrize("values", [1, 2, 40])
def test_ties_go_to_the_lowest_index(dtype, vocab, values):
    g = torch.Generator(device="cuda")
    g.manual_seed(values)
    x = torch.randint(0, values, (4, vocab), device="cuda", generator=g).to(dtype)
    x[1] = -0.0 * x[1]  # zeros of both signs are equal
    check(x, targets_of(4, vocab), 32)


@pytest.mark.parametrize("vocab", [100, 20011])
@pytest.mark.parametrize("rising", [True, False])
def test_sorted_rows(vocab, rising):
    x = torch.linspace(-20, 20, vocab, device="cuda").expand(3, vocab)
    x = x if rising else x.flip(-1)
    check(x, torch.tensor([0, vocab // 2, vocab - 1], device="cuda"), 32)
    check(x.contiguous(), torch.tensor([0, vocab // 2, vocab - 1], device="cuda"), 7)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("vocab", [50, 5000, 40000])
def test_masked_logits(dtype, vocab):
    """Masks of -infinity and of the type's lowest value, rows where few, one or no token is left."""
    low = torch.finfo(dtype).min
    x = rnd((12, vocab), dtype, 5)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    some = torch.rand(vocab, device="cuda", generator=g) < 0.5
    x[0, some], x[1, some] = -math.inf, low
    x[2], x[3] = -math.inf, low
    x[4], x[5] = -math.inf, low
    x[4, vocab - 1], x[5, vocab - 1] = 3.0, 3.0
    x[6, 10:], x[7, 10:] = -math.inf, low
    x[8, :vocab - 3], x[9, :vocab - 3] = -math.inf, low
    x[10, 1::2] = -math.inf
    x[11, :vocab // 2], x[11, vocab // 2:] = low, -math.inf
    t = torch.tensor([0, 0, 3, 3, vocab - 1, 1, 4, 30, vocab - 2, vocab - 2, 1, 0], device="cuda")
    check(x, t, 32)
    assert torch.isfinite(check(x[3:4], t[3:4], 2).logprob).all()
    none = check(x[2:3], t[2:3], 5)
    assert none.entropy.item() == 0 and (none.top_logprob == -math.inf).all()
    assert none.top_index[0].tolist() == [0, 1, 2, 3, 4] and none.logprob.item() == -math.inf


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("vocab", [60, 30000])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_infinities_and_nans_stay_in_their_row(dtype, vocab, what):
    x, t = rnd((9, vocab), dtype, 6), targets_of(9, vocab)
    clean = check(x, t, 8)
    for r, at in ((0, 0), (4, vocab // 2), (8, vocab - 1)):
        x[r, at] = what
    x[4, 3] = x[4, vocab - 2] = what
    op = paged.TokenLogprobs(top=8)
    got = op(x, t)
    bad = torch.zeros(9, dtype=torch.bool, device="cuda")
    bad[[0, 4, 8]] = True
    for name in ("logprob", "entropy", "top_logprob"):
        g, c = getattr(got, name), getattr(clean, name)
        assert g[bad].isnan().all() and torch.equal(g[~bad], c[~bad])
    assert torch.equal(got.top_index[~bad], clean.top_index[~bad]) and torch.equal(got.rank[~bad], clean.rank[~bad])
    assert got.top_index[0, 0].item() == 0 and got.top_index[8, 0].item() == vocab - 1
    assert got.top_index[4, :3].tolist() == sorted((3, vocab // 2, vocab - 2))
    assert torch.equal(got.top_index[0, 1:], clean.top_index[0][clean.top_index[0] != 0][:7])


def test_extremes():
    """Logits at both ends of float32: differences that pass its range."""
    big = torch.finfo(SF).max
    x = torch.full((4, 700), -big, device="cuda")
    x[0, 5] = big
    x[1, 5:9] = big
    x[2, ::2] = 0.0
    x[3] = big
    check(x, torch.tensor([5, 7, 1, 699], device="cuda"), 6)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("pad,first", [(0, 0), (1, 0), (7, 1), (29, 3), (64, 8)])
@pytest.mark.parametrize("vocab", [4, 1000, 20003])
def test_rows_cut_from_others(dtype, pad, first, vocab):
    """Strides and starts of any alignment; what stands between rows does not reach them."""
    store = torch.full((6, vocab + pad + first), math.nan, dtype=dtype, device="cuda")
    x = store[:, first:first + vocab]
    x.copy_(rnd((6, vocab), dtype, 7))
    check(x, targets_of(6, vocab), min(vocab, 9))
    check(x[::2], targets_of(3, vocab), min(vocab, 9))


def test_rows_that_share_their_memory():
    x = rnd((1, 5000), HF, 8).expand(5, 5000)
    check(x, targets_of(5, 5000), 4)


def test_targets():
    """Without a target, past the vocabulary, none at all."""
    x = rnd((5, 3000), BF, 9)
    t = torch.tensor([-1, 2999, -100, 0, 7], device="cuda")
    got = check(x, t, 2)
    assert got.logprob[0].item() == 0 and got.rank[2].item() == 0
    op = paged.TokenLogprobs(top=2)
    bad = torch.tensor([3000, 2 ** 40, 1, 2 ** 31 + 5, -(2 ** 40)], device="cuda")
    got = check(x, bad, 2, op, err=1)
    with pytest.raises(_native.Q4GpuError):
        op.check()
    op.check()
    none = op(x)
    assert torch.equal(none.top_index, got.top_index) and torch.equal(none.entropy, got.entropy)


def test_offsets_past_32_bits():
    """Rows that begin beyond 2^31 elements."""
    store = torch.empty(2 ** 31 + 200000, dtype=BF, device="cuda")
    x = store.as_strided((2, 100000), (2 ** 31 + 50000, 1))
    x.copy_(rnd((2, 100000), BF, 10))
    check(x, targets_of(2, 100000), 10)


def test_output_given_stream_and_graph():
    x, t = rnd((30, 20000), SF, 11), targets_of(30, 20000)
    op = paged.TokenLogprobs(top=5)
    out = op.empty(30)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        check(x, t, 5, op, out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op(x, t, out)
        late = op(x, t)  # results of its own
    for seed in range(3):
        x.copy_(rnd((30, 20000), SF, seed))
        t.copy_(targets_of(30, 20000, seed))
        graph.replay()
        want = paged.TokenLogprobs(top=5)(x, t)
        for name in ("logprob", "entropy", "rank", "top_logprob", "top_index"):
            assert torch.equal(getattr(out, name), getattr(want, name))
            assert torch.equal(getattr(late, name), getattr(want, name))
    op.check()


def test_one_operator_for_calls_of_all_shapes():
    op = paged.TokenLogprobs(top=3)
    for rows, vocab, dtype in ((1, 151936, SF), (200, 100, BF), (0, 5000, HF), (3, 3, BF), (64, 151936, BF), (1, 100, SF)):
        check(rnd((rows, vocab), dtype, 12), targets_of(rows, vocab), 3, op)


def test_same_numbers_in_any_batch():
    """A row's results do not depend on the rows beside it (but for the split that their number decides)."""
    x, t = rnd((400, 30000), BF, 13), targets_of(400, 30000)
    a, b = paged.TokenLogprobs(top=7)(x, t), paged.TokenLogprobs(top=7)(x, t)
    for name in ("logprob", "entropy", "rank", "top_logprob", "top_index"):
        assert torch.equal(getattr(a, name), getattr(b, name))


def test_refusals():
    op = paged.TokenLogprobs(top=3)
    x, t = rnd((4, 100), BF), targets_of(4, 100)
    for bad in (lambda: paged.TokenLogprobs(top=33), lambda: paged.TokenLogprobs(top=-1),
                lambda: paged.TokenLogprobs(device="cpu"), lambda: op(x[0], t), lambda: op(x.cpu(), t),
                lambda: op(x.double(), t), lambda: op(x.t(), t), lambda: op(x, t.int()), lambda: op(x, t[:3]),
                lambda: op(x, t.cpu()), lambda: op(x[:, :0], t), lambda: op(x, t, op.empty(5)),
                lambda: op(x, t, paged.TokenLogprobs(top=2).empty(4))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(_native.Q4GpuError):
        op(x[:, :2], t)  # fewer tokens than alternatives
    check(x, t, 3, op)
