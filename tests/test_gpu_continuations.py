"""The decoder on the operators that serve and judge continuations: forks of a long prompt decoded together, texts
past a window with sinks, log probabilities of given and of chosen tokens; one run of them all.

Bounds: as for the decoder's other logits, what differs in summation order alone stays below 2 % (2-norm) over these
layers.  A log probability moves by at most twice the largest change of a logit: 2 (0.02 + 2^-8) of the largest, the
second term for logits that are judged in bf16."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged, paged_decode  # noqa: E402
from test_gpu_paged_decode import VOCAB, off, tokens, weights  # noqa: E402, F401


def decoder(weights, **kw):  # noqa: F811
    return paged_decode.PagedDecoder(weights, **(dict(max_seqs=6, max_ctx=1600, page_tokens=64) | kw))


def forked(weights, prompt=1100, kids=(1, 2, 3, 4), **kw):  # noqa: F811
    d = decoder(weights, **kw)
    d.prefill(0, tokens(prompt, 1))
    d.prefill(5, tokens(40, 2))
    d.cache.fork(0, list(kids))
    return d


@pytest.mark.parametrize("prompt", [1088, 1100])  # whole pages, a partly filled last one
def test_forks_attend_together(weights, monkeypatch, prompt):  # noqa: F811
    d = forked(weights, prompt)
    step = [[7, 8], [9], [10, 11, 12], [13], [14]]
    seqs = [1, 2, 3, 4, 5]  # four forks and a stranger
    got = d.forward(seqs, step)
    more = d.forward(seqs, [[t] for t in range(5)])
    assert all("shared" in lay for lay in d.layers)
    monkeypatch.setattr(paged.PagedCache, "SHARED_KEYS", 1 << 40)
    monkeypatch.setattr(paged.PagedCache, "SAVED_KEYS", 1 << 40)
    alone = forked(weights, prompt)
    want = alone.forward(seqs, step)
    assert not any("shared" in lay for lay in alone.layers)
    assert off(got, want) < 0.02 and off(more, alone.forward(seqs, [[t] for t in range(5)])) < 0.02
    for lay in d.layers:
        lay["shared"].check()
        lay["rope"].check()


def test_steps_name_their_groups(weights):  # noqa: F811
    d = forked(weights)
    c = d.cache
    c.extend([5], [1])
    s = c.extend([1, 2, 5, 3, 4], [1] * 5)
    assert s.cu_group.tolist() == [0, 2, 3, 5] and s.prefix_lens.tolist() == [1088, 0, 1088] and s.max_prefix == 1088
    assert c.extend([1, 5, 2], [1] * 3).cu_group is None  # no neighbours share anything
    c.free(0), c.free(2), c.free(3), c.free(4)
    assert c.extend([1, 5], [1, 1]).cu_group is None


def test_window_with_sinks(weights):  # noqa: F811
    text = tokens(700, 3)
    full = decoder(weights).prefill(0, text)
    wide = decoder(weights, window=1600, sinks=4).prefill(0, text)
    assert off(wide, full) < 0.02
    d = decoder(weights, window=100, sinks=5)
    one, two = d.prefill(0, text, 700), d.prefill(1, text, 77)
    assert off(one, two) < 0.02 and off(one, full) > 0.1
    d.cache.fork(0, [2, 3])
    x = d.forward([2, 3], [[1], [1]])  # forks step through their windows, each for itself
    assert torch.equal(x[0], x[1]) and not any("shared" in lay for lay in d.layers)
    # what stands between the sinks and the window has no say: other tokens there change nothing but through the
    # layers' reach (3 layers x 99 positions), which ends before the last 300
    other = text[:5] + tokens(300, 4) + text[305:]
    far = decoder(weights, window=100, sinks=5)
    assert off(far.prefill(0, other), one) < 0.02
    none = decoder(weights, window=100)
    assert off(none.prefill(0, text), one) > 0.01  # the sinks do


def test_scores_of_given_tokens(weights):  # noqa: F811
    text = tokens(150, 5)
    d = decoder(weights)
    scores = d.score(0, text, chunk=64, top=4)
    assert [s.logprob.shape[0] for s in scores] == [64, 64, 22]
    logprob, rank = torch.cat([s.logprob for s in scores]), torch.cat([s.rank for s in scores])
    entropy, best = torch.cat([s.entropy for s in scores]), torch.cat([s.top_index for s in scores])
    assert logprob[-1].item() == 0 and rank[-1].item() == 0 and (rank[:-1] > 0).all()
    one = decoder(weights)
    logits = torch.cat([one.forward([0], [[t]]) for t in text])
    p = torch.log_softmax(logits.double(), -1)
    tol = 2 * (0.02 + 2.0 ** -8) * logits.abs().max().item()
    follow = torch.tensor(text[1:], device="cuda")[:, None]
    assert (logprob[:-1] - p[:-1].gather(1, follow).squeeze(1)).abs().max() < tol
    h = -(p.exp() * p).sum(-1)
    # an entropy moves by at most (range of log p) x the change of the probabilities, each of them by a factor e^tol
    assert (entropy - h).abs().max() < tol * (1 + p.abs().max().item())
    top = torch.cat([s.top_logprob for s in scores])
    assert (top - p.gather(1, best.long())).abs().max() < tol
    assert (top[:, :-1] >= top[:, 1:]).all() and ((rank[:-1, None] == 1) == (best[:-1, :1] == follow)).all()
    again = d.forward([0], [[3]])  # the sequence goes on behind the text
    assert off(again, one.forward([0], [[3]])) < 0.02


def test_scores_of_chosen_tokens(weights):  # noqa: F811
    d = decoder(weights)
    logits = [d.prefill(s, tokens(50, 6 + s)) for s in (0, 1)]
    texts, scores = d.generate_scored([0, 1], torch.cat(logits), 5)
    e = decoder(weights)
    logits = torch.cat([e.prefill(s, tokens(50, 6 + s)) for s in (0, 1)])
    for i in range(5):
        p = torch.log_softmax(logits.double(), -1)
        assert [t[i] for t in texts] == logits.argmax(-1).tolist()
        want = p.max(-1).values.tolist()
        assert all(abs(s[i] - w) < 1e-4 for s, w in zip(scores, want))
        logits = e.forward([0, 1], [[t[i]] for t in texts])
    assert e.generate([0], logits[:1], 0) == [[]]


def test_score_refusals(weights):  # noqa: F811
    d = decoder(weights)
    for bad in (lambda: d.score(0, []), lambda: d.score(0, [1], chunk=0), lambda: d.score(0, [1, VOCAB], chunk=1),
                lambda: d.score(0, [1], top=33), lambda: decoder(weights, sinks=3)):
        with pytest.raises(ValueError):
            bad()
    assert d.cache.length(0) == 0


def test_a_run_of_them_together():
    r = paged_decode.run(prompt_tokens=1200, continuations=4, new_tokens=5, n_layers=2, vocab=500)
    assert len(r["logprobs"]) == 4 and all(-20 < v <= 0 for v in r["logprobs"].values())
    assert len(r["continued"]) == 5
