"""Rows of logits whose likeliest tokens are hard to tell apart.  Whole numbers are exact: falling logits, NaN before
all, equal ones by rising index."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged  # noqa: E402

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32


def likeliest(x, top):
    """The order by definition: a stable sort, NaN as more than everything."""
    v = x.double()
    first = v.isnan().double().sort(stable=True, dim=-1, descending=True).indices  # NaNs, then the others
    nans = v.isnan().sum(-1)
    rest = torch.where(v.isnan(), -math.inf, v)
    # (a NaN's place in `rest` counts as the lowest; the others' order is cut behind the NaNs)
    order = rest.sort(stable=True, dim=-1, descending=True).indices
    out = torch.empty(x.shape[0], top, dtype=torch.int64, device="cuda")
    for r in range(x.shape[0]):
        n = int(nans[r])
        mine = order[r][~v[r].isnan()[order[r]]]
        out[r] = torch.cat((first[r][:min(n, top)], mine[:max(0, top - n)]))
    return out


def normal(rows, vocab, dtype, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)


def check(x, top):
    op = paged.TokenLogprobs(top=top)
    got = op(x)
    assert torch.equal(got.top_index.long(), likeliest(x, top))
    op.check()
    return got


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows", [1, 64, 300])
@pytest.mark.parametrize("top", [1, 2, 5, 32])
def test_rows_of_nan(dtype, rows, top):
    x = normal(rows, 151936, dtype)
    x[0] = math.nan
    x[-1, : 5000] = math.nan
    got = check(x, top)
    assert got.top_index[0].tolist() == list(range(top))
    assert got.top_logprob[0].isnan().all() and got.entropy[0].isnan()


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("what", [math.nan, 50.0])
@pytest.mark.parametrize("top", [5, 32])
def test_many_large_ones_in_a_few_threads(dtype, what, top):
    """Every 512th unit of 16 and the three behind it: more than 1024 logits of four threads."""
    x = normal(300, 151936, dtype)
    x[7].view(-1, 16)[torch.arange(151936 // 16, device="cuda") % 512 < 4] = what
    check(x, top)


@pytest.mark.parametrize("first", [0, 1, 7])
def test_vocabularies_next_to_2_to_the_31(first):
    """Equal logits but for three: sums and ranks of the last unit of 16 and of what stands behind it."""
    vocab = 2 ** 31 - 1
    store = torch.zeros(vocab + 16, dtype=BF, device="cuda")
    x = store[first:first + vocab].view(1, vocab)
    lp = paged.TokenLogprobs()
    for t in (vocab - 1, vocab - 15, vocab - 16, vocab - 17, vocab - 30, 2 ** 30, 0):
        got = lp(x, torch.tensor([t], device="cuda"))
        assert got.rank.item() == t + 1
        # 2^31 - 2 ones in 32 bits: each of the few additions a warp and its partners make is off by 2^-24 at most
        assert abs(got.logprob.item() + math.log(vocab)) < 1e-4 and abs(got.entropy.item() - math.log(vocab)) < 1e-4
    best = {vocab - 1: 32.0, vocab - 17: 31.0, 0: 30.0}
    for at, v in best.items():
        x[0, at] = v
    got = paged.TokenLogprobs(top=3)(x, torch.tensor([vocab - 2], device="cuda"))
    assert got.top_index[0].tolist() == list(best) and got.rank.item() == vocab
    want = torch.tensor(list(best.values()), dtype=torch.float64)
    norm = math.log(vocab - 3 + sum(math.exp(v) for v in best.values()))
    assert (got.top_logprob[0].double().cpu() - (want - norm)).abs().max() < 1e-4
    lp.check()


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("rows", [1, 20, 64])
def test_candidates_of_single_lanes(dtype, rows):
    """Rows over clusters whose candidates lie in one lane of a warp, in one warp, in the last CTA: lanes that have no
    more to look at wait for the others before the CTAs meet."""
    x = normal(rows, 151936, dtype)
    units = x.view(rows, -1, 16)
    units[0, 5::512, 3] = 40.0
    units[rows // 2, 32:64, 0] = 41.0
    units[-1, -7:, 9] = 42.0
    for _ in range(3):
        check(x, 20)


@pytest.mark.parametrize("rows,every,width", [(1, 512, 24), (64, 512, 8), (300, 512, 4)])
@pytest.mark.parametrize("what", [math.nan, 50.0])
def test_many_large_ones_in_a_few_threads_of_a_cluster(rows, every, width, what):
    """Likewise where 8, 2 or one CTA share a row, and in other rows not."""
    x = normal(rows, 151936, SF, 1)
    for r in {0, rows // 2}:
        x[r].view(-1, 16)[torch.arange(151936 // 16, device="cuda") % every < width] = what
    check(x, 5)
    check(x, 32)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,vocab", [(1, 151936), (64, 151936), (300, 151936), (1, 1100), (40, 32001), (700, 4099)])
@pytest.mark.parametrize("left", [0, 1, 3, 10, 40])
@pytest.mark.parametrize("low", ["infinity", "lowest"])
def test_masks_that_leave_few(dtype, rows, vocab, left, low):
    """Fewer tokens are allowed than alternatives are asked for: what is masked follows by rising index."""
    x = torch.full((rows, vocab), -math.inf if low == "infinity" else torch.finfo(dtype).min, dtype=dtype, device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(left)
    for r in range(min(rows, 8)):
        at = torch.randperm(vocab, device="cuda", generator=g)[:left]
        x[r, at] = torch.randn(left, device="cuda", generator=g).to(dtype)
    for top in (1, 5, 20, 32):
        check(x, top)


@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("rows", [1, 64, 300])
@pytest.mark.parametrize("kind", ["block", "rising", "falling", "constant", "stairs", "two values"])
def test_likeliest_that_stand_together(dtype, rows, kind):
    """A block of allowed tokens, logits in order, equal ones: many threads reach what a group's largest bounds."""
    vocab = 151936
    x = normal(rows, vocab, dtype, 2)
    at = torch.arange(vocab, device="cuda")
    if kind == "block":
        x[:, :5000], x[:, 9000:] = -math.inf, -math.inf
    elif kind == "constant":
        x[:] = 1.5
    elif kind == "stairs":
        x[:] = (at // 1000).to(dtype)
    elif kind == "two values":
        x[:] = (x > 0).to(dtype)
    else:
        x[:] = (at if kind == "rising" else -at).float().mul(1e-4).to(dtype)
    for top in (1, 5, 20, 32):
        check(x, top)


@pytest.mark.parametrize("dtype,ints,patterns", [
    (BF, torch.int16, (0x7fc0, 0x7fff, 0x7f81, -0x40, -1)), (HF, torch.int16, (0x7e00, 0x7fff, 0x7c01, -0x200, -1)),
    (SF, torch.int32, (0x7fc00000, 0x7fffffff, 0x7f800001, -0x400000, -1))])
@pytest.mark.parametrize("rows,vocab", [(40, 570), (3, 40), (64, 5000), (1, 151936)])
def test_targets_that_are_nan(dtype, ints, patterns, rows, vocab):
    """NaN of any bits comes first in the order: its rank counts the NaNs before it and nothing else."""
    for bits in patterns:
        x = normal(rows, vocab, dtype, 3)
        at = sorted({vocab // 7, vocab // 2, vocab - 1})
        for i in at:
            x.view(ints)[:, i] = bits
        assert x[0, at].isnan().all()
        op = paged.TokenLogprobs()
        for k, i in enumerate(at):
            got = op(x, torch.full((rows,), i, device="cuda"))
            assert (got.rank == k + 1).all() and got.logprob.isnan().all()
        rest = op(x, torch.zeros(rows, dtype=torch.int64, device="cuda"))  # and before every number
        v = x.double()
        assert torch.equal(rest.rank.long(), 1 + ((v > v[:, :1]) | v.isnan()).sum(-1))
