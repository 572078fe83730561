"""Attention operators that share a workspace: layers one after another, growing, captured, on other streams.
Bounds: ``test_gpu_shared``."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged, paged_decode  # noqa: E402
from test_gpu_paged import BF  # noqa: E402
from test_gpu_paged_decode import tokens, weights  # noqa: E402, F401
from test_gpu_shared import Case, close  # noqa: E402


def test_layers_that_share():
    cases = [Case([(700, [(1, 30)] * 6), (64, [(2, 9), (1, 1)])], 8, 2, 128, 64, BF, seed) for seed in (1, 2, 3)]
    first = cases[0].op()
    ops = [first] + [c.op(share=first) for c in cases[1:]]
    refs = [c.ref() for c in cases]
    for c, op, r in zip(cases, ops, refs):
        close(*c.run(op), *r)
    assert len({op.workspace.data_ptr() for op in ops}) == 1
    got = [(torch.empty_like(c.q), torch.empty(c.q.shape[:2], device="cuda")) for c in cases]

    def step():
        for c, op, (out, lse) in zip(cases, ops, got):
            op(c.q, out, c.cu, c.ends, c.prefix, max_q=2, max_ctx=c.max_ctx, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    big = Case([(700, [(40, 90)] * 6)], 8, 2, 128, 64, BF, 9)
    wide = big.op(share=first)
    close(*big.run(wide), *big.ref())  # grows; the graph keeps what it knows
    assert wide.workspace.data_ptr() != ops[1].workspace.data_ptr() and len(first.room) == 2
    side = torch.cuda.Stream()
    for _ in range(3):
        for out, lse in got:
            out.zero_(), lse.zero_()
        graph.replay()
        for (out, lse), r in zip(got, refs):
            close(out, lse, *r)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            close(*big.run(wide), *big.ref())
            step()
            for (out, lse), r in zip(got, refs):
                close(out, lse, *r)
        torch.cuda.current_stream().wait_stream(side)
    plain = paged.Attention(big.pool[:, 0], big.pool[:, 1], big.table.clamp(min=0), big.lens, 8, share=first)
    assert plain.room is first.room
    for op in ops + [wide]:
        op.check()


def test_a_decoder_has_one_for_all_layers(weights):  # noqa: F811
    d = paged_decode.PagedDecoder(weights, max_seqs=6, max_ctx=1600)
    d.prefill(0, tokens(1100, 1))
    d.cache.fork(0, [1, 2, 3, 4])
    d.forward([1, 2, 3, 4], [[5]] * 4)
    d.forward([1, 2, 3, 4], [[5, 6, 7]] * 4)
    assert len(d.layers) > 1
    assert len({id(lay["shared"].room) for lay in d.layers}) == 1
    assert all(any(lay["shared"].workspace is t for t in lay["shared"].room) for lay in d.layers)
    for lay in d.layers:
        lay["shared"].check()
