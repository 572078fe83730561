"""Greedy tokens of the decoder from logits of any kind that argmax takes."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged_decode  # noqa: E402
from test_gpu_paged_decode import tokens, weights  # noqa: E402, F401


def start(weights):  # noqa: F811
    d = paged_decode.PagedDecoder(weights, max_seqs=2, max_ctx=256)
    return d, torch.cat([d.prefill(s, tokens(40, 30 + s)) for s in (0, 1)])


KINDS = {"float32": lambda x: x, "float64": lambda x: x.double(), "host": lambda x: x.cpu(),
         "columns apart": lambda x: x.t().contiguous().t(), "bf16": lambda x: x.bfloat16().float().bfloat16()}


@pytest.mark.parametrize("kind", KINDS)
def test_logits_of_any_kind(weights, kind):  # noqa: F811
    d, logits = start(weights)
    given = KINDS[kind](logits)
    got = d.generate([0, 1], given, 4)
    e, same = start(weights)
    first = given.argmax(-1).tolist()
    want = [[t] for t in first]
    for _ in range(3):
        nxt = e.forward([0, 1], [[w[-1]] for w in want]).argmax(-1).tolist()
        for w, t in zip(want, nxt):
            w.append(t)
    assert got == want


def test_with_and_without_scores(weights):  # noqa: F811
    d, logits = start(weights)
    e, same = start(weights)
    plain = d.generate([0, 1], logits, 5)
    texts, scores = e.generate_scored([0, 1], same, 5)
    assert texts == plain and [len(s) for s in scores] == [5, 5] and all(v <= 0 for s in scores for v in s)
    assert d.generate([0, 1], logits, 0) == [[], []] and e.generate_scored([0], same[:1], 0) == ([[]], [[]])
