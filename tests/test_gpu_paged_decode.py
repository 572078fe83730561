"""The 16-bit paged decoder: its logits against the float32 forward of the same weights, and what must
not change them (chunk sizes, company in the batch, forks, compaction).

Bound of the logits: each layer adds a handful of roundings of the residual stream to bf16 (2^-9 of it,
uncorrelated); over 3 layers and the final product the relative 2-norm error stays below 16 * 2^-9 = 3.2 %
(8-bit gate/up products add 2^-4 / sqrt(3) of the MLP's share at most: 8 %)."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import fp32_diag, paged, paged_decode  # noqa: E402

VOCAB, LAYERS = 1000, 3


class Shape:
    vocab, n_layers = VOCAB, LAYERS


@pytest.fixture(scope="module")
def weights():
    return fp32_diag.float_weights(Shape, seed=3, gamma_std=0.05)


def tokens(n, seed=0):
    return torch.randint(0, VOCAB, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def off(a, b):
    return float((a - b).norm() / b.norm())


@pytest.mark.parametrize("dtype,eight_bit,bound", [(torch.bfloat16, False, 0.032), (torch.float16, False, 0.032),
                                                   (torch.bfloat16, True, 0.08)])
def test_logits_match_the_float32_forward(weights, dtype, eight_bit, bound):
    d = paged_decode.PagedDecoder(weights, max_seqs=2, max_ctx=128, page_tokens=16, dtype=dtype, eight_bit=eight_bit)
    toks = tokens(70)
    want = torch.from_numpy(fp32_diag.float_logits(weights, toks)).cuda()
    got = [d.forward([1], [toks[:33]])[0], d.forward([1], [toks[33:34]])[0], d.forward([1], [toks[34:]])[0]]
    for x, at in zip(got, (32, 33, 69)):
        assert off(x, want[at]) < bound


def test_chunks_and_company_do_not_matter(weights):
    d = paged_decode.PagedDecoder(weights, max_seqs=3, max_ctx=512, page_tokens=32)
    a, b = tokens(300, 1), tokens(45, 2)
    one = d.prefill(0, a, 512)
    two = d.prefill(1, a, 77)
    d.forward([2], [b[:44]])
    assert off(one, two) < 0.02
    both = d.forward([2, 0], [b[44:], [5]])
    alone = paged_decode.PagedDecoder(weights, max_seqs=3, max_ctx=512, page_tokens=32)
    want = alone.prefill(0, b, 44)
    assert off(both[:1], want) < 0.02
    assert off(both[1:], d.forward([1], [[5]])) < 0.02


def test_forks_continue_like_their_parent_and_compaction_changes_nothing(weights):
    d = paged_decode.PagedDecoder(weights, max_seqs=5, max_ctx=256, page_tokens=16)
    d.prefill(0, tokens(100, 1))
    d.prefill(4, tokens(130, 2))
    free = d.cache.free_pages
    d.cache.fork(4, [1, 2])
    assert d.cache.free_pages == free - 2  # 130 = 8 full pages and one partly filled
    x = d.forward([1, 2, 4], [[7], [7], [7]])
    assert torch.equal(x[0], x[1]) and torch.equal(x[0], x[2])
    y = d.forward([1, 2, 4], [[8], [9], [8]])
    assert torch.equal(y[0], y[2]) and not torch.equal(y[0], y[1])
    d.cache.fork(1, [3])
    d.cache.free(0)
    d.cache.free(4)
    used = d.cache.pool.shape[0] - d.cache.free_pages
    assert d.cache.compact() == used
    assert sorted({p for h in d.cache._held for p in h}) == list(range(used))
    assert d.cache.free_pages == d.cache.pool.shape[0] - used
    z = d.forward([1, 3], [[11], [11]])
    assert torch.equal(z[0], z[1])
    d.cache.pages.check()
    for lay in d.layers:
        lay["rope"].check()
        lay["attn"].check()


def test_the_command_runs():
    r = paged_decode.run(prompt_tokens=200, continuations=3, new_tokens=3, n_layers=2, vocab=500)
    assert len(r["continuations"]) == 3 and r["pages_after_compaction"] <= r["pages_used"] and len(r["continued"]) == 3


def test_cache_refusals():
    c = paged.PagedCache(1, 4, 16, 1, 64, max_seqs=3, max_ctx=48)
    c.extend([0], [33])
    for bad in (lambda: c.extend([0], [16]), lambda: c.extend([0, 0], [1, 1]), lambda: c.extend([1], [-1]),
                lambda: c.fork(0, [0]), lambda: c.fork(0, [1, 1]), lambda: c.extend([], [])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="full"):
        c.extend([1], [17])
    with pytest.raises(RuntimeError, match="full"):
        c.fork(0, [1, 2])
    assert c.free_pages == 1 and c.length(1) == 0
    c.fork(0, [2])
    assert c.free_pages == 0
    c.free(0)
    assert c.free_pages == 1  # two of its pages are shared with its fork
    c.free(2)
    assert c.free_pages == 4


def test_stretched_tables():
    from llm_accelerator_b200 import tables
    cos, sin = tables.rope_float_tables(64, 128)
    inv = 1e6 ** (-torch.arange(0, 128, 2, dtype=torch.float64) / 128)
    a = torch.arange(64, dtype=torch.float64)[:, None] * inv
    assert (cos.double() - a.cos()).abs().max() < 1e-7 and (sin.double() - a.sin()).abs().max() < 1e-7
    cos, sin = tables.rope_float_tables(8192, 128, factor=4.0)
    m = 0.1 * torch.log(torch.tensor(4.0, dtype=torch.float64)) + 1
    assert ((cos.double() ** 2 + sin.double() ** 2).sqrt() - m).abs().max() < 1e-6
    fast, slow = torch.atan2(sin[1, 0], cos[1, 0]), torch.atan2(sin[1, -1], cos[1, -1])
    assert abs(float(fast) - 1.0) < 1e-6 and abs(float(slow) / float(inv[-1]) - 0.25) < 1e-3
    with pytest.raises(ValueError):
        tables.rope_float_tables(8, 7)
