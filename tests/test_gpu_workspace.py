"""Attention in a workspace of exactly the size it asks for, with a guard behind it, whatever bound of the lengths it
was given.  Bounds of the results are those of ``test_gpu_sinks`` and ``test_gpu_shared``."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged  # noqa: E402
from test_gpu_paged import BF, TINY, U, make, within  # noqa: E402
from test_gpu_shared import Case, close  # noqa: E402
from test_gpu_sinks import ref  # noqa: E402

GUARD = 1 << 20


def guarded(need):
    room = torch.zeros(need + GUARD, dtype=torch.uint8, device="cuda")
    room[need:] = 0x5a
    return room


@pytest.mark.parametrize("max_ctx", [0, 1, 300, 5000])
@pytest.mark.parametrize("window,sinks", [(0, 0), (700, 0), (700, 5)])
@pytest.mark.parametrize("hq,hk,dim", [(16, 8, 128), (4, 4, 64), (8, 1, 64)])
@pytest.mark.parametrize("new", [1, 40])
def test_exactly_enough(hq, hk, dim, window, sinks, new, max_ctx):
    pool, table, lens, cu, q = make([new, 1, new], [4000, 3, 900], hq, hk, dim, 64, BF, 3)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, lens, hq, window=window, sinks=sinks)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    op(q, out, cu, max_q=new, max_ctx=5000, lse=lse)
    out.fill_(5.0), lse.fill_(5.0)
    a, lib = op.args, op.lib
    a.max_ctx = max_ctx
    need = lib.q4gpu_sink_attention_workspace_bytes(a, sinks)
    room = guarded(need)
    a.workspace, a.workspace_bytes = room.data_ptr(), need
    assert lib.q4gpu_sink_attention(a, sinks, torch.cuda.current_stream().cuda_stream) == 0
    assert (room[need:] == 0x5a).all()
    want, mag, rl = ref(pool, table, lens, cu, q, window or 1 << 30, sinks)
    u = U[BF]
    within(out, want, u * want.abs() + (u + 3e-4) * mag + TINY[BF])
    within(lse, rl, 3e-4 + 1e-6 * rl.abs())
    op.check()


@pytest.mark.parametrize("max_ctx,max_prefix", [(0, 0), (1, 1), (400, 1000), (5000, 3000)])
@pytest.mark.parametrize("hq,hk,dim", [(16, 8, 128), (4, 4, 64), (40, 1, 64)])
@pytest.mark.parametrize("new", [1, 70])
def test_exactly_enough_with_shared_keys(hq, hk, dim, new, max_ctx, max_prefix):
    case = Case([(3000, [(new, 900), (1, 20), (new, 100)]), (64, [(1, 1)])], hq, hk, dim, 64, BF, 4)
    op = case.op()
    case.run(op)
    out, lse = torch.full_like(case.q, 5.0), torch.full(case.q.shape[:2], 5.0, device="cuda")
    a, g, lib = op.args, op.groups, op.lib
    a.q, a.out, a.lse = case.q.data_ptr(), out.data_ptr(), lse.data_ptr()
    a.max_ctx, g.max_prefix = max_ctx, max_prefix
    need = lib.q4gpu_shared_attention_workspace_bytes(a, g)
    room = guarded(need)
    a.workspace, a.workspace_bytes = room.data_ptr(), need
    assert lib.q4gpu_shared_attention(a, g, torch.cuda.current_stream().cuda_stream) == 0
    assert (room[need:] == 0x5a).all()
    close(out, lse, *case.ref())
    op.check()
