"""Rows and sequences do not depend on what is beside them: the same ones among others, in another order, bit for bit.

(The work is split by a call's sizes, so the calls that are compared have the same.)"""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged  # noqa: E402

BF, HF, SF = torch.bfloat16, torch.float16, torch.float32
NAMES = ("logprob", "entropy", "rank", "top_logprob", "top_index")


def normal(rows, vocab, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(rows, vocab, device="cuda", generator=g) * 3).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, SF])
@pytest.mark.parametrize("rows,vocab", [(400, 30000), (64, 151936), (7, 151936), (900, 4096)])
def test_rows_of_logits(dtype, rows, vocab):
    x = normal(rows, vocab, dtype, 1)
    t = torch.arange(rows, device="cuda") * 7 % vocab
    op = paged.TokenLogprobs(top=7)
    want = op(x, t)
    order = torch.randperm(rows, device="cuda")
    got = op(x[order], t[order])
    for name in NAMES:
        assert torch.equal(getattr(got, name), getattr(want, name)[order])
    # every second row among strangers: masked, certain, NaN
    other = normal(rows, vocab, dtype, 2)
    other[::4], other[1::4, 5:] = math.nan, -math.inf
    mixed = torch.where((torch.arange(rows, device="cuda") % 2 == 0)[:, None], x, other)
    got = op(mixed, t)
    for name in NAMES:
        assert torch.equal(getattr(got, name)[::2], getattr(want, name)[::2])


@pytest.mark.parametrize("threads", [2])
def test_one_operator_on_two_streams(threads):
    """No workspace: calls may overlap."""
    op = paged.TokenLogprobs(top=20)
    xs = [normal(64, 151936, SF, 3 + i) for i in range(threads)]
    want = [op(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    for _ in range(5):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append([op(x) for _ in range(4)])
        torch.cuda.synchronize()
        for mine, w in zip(got, want):
            for g in mine:
                assert all(torch.equal(getattr(g, n), getattr(w, n)) for n in ("entropy", "top_logprob", "top_index"))
