"""Shared-key attention where its kernels' order in the stream and its refusals count.  Bounds: ``test_gpu_shared``."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from test_gpu_paged import BF, i32  # noqa: E402
from test_gpu_shared import Case, close  # noqa: E402


@pytest.mark.parametrize("seqs", [3, 200])
@pytest.mark.parametrize("new", [1, 40])
def test_a_call_without_queries_ends_before_what_follows(seqs, new):
    """Rows behind the last sequence stay as they are although the next kernels in the stream name them as queries."""
    case = Case([(300, [(new, new + 20)] * seqs)], 4, 2, 64, 32, BF, 1)
    op, full = case.op(), case.cu.clone()
    case.run(op)
    out, lse = torch.empty_like(case.q), torch.empty(case.q.shape[:2], device="cuda")
    want = case.ref()
    for _ in range(20):
        case.cu.zero_()
        out.fill_(7.0), lse.fill_(7.0)
        op(case.q, out, case.cu, case.ends, case.prefix, max_q=new, max_ctx=case.max_ctx, lse=lse)
        case.cu.copy_(full)
        assert (out == 7.0).all() and (lse == 7.0).all()
        op(case.q, out, case.cu, case.ends, case.prefix, max_q=new, max_ctx=case.max_ctx, lse=lse)
        close(out, lse, *want)
    op.check()


@pytest.mark.parametrize("seqs", [4, 150])
@pytest.mark.parametrize("bad", ["falls", "negative", "past", "groups"])
def test_every_row_of_a_call_out_of_order_is_zero(seqs, bad):
    """Offsets that do not ascend: zeros and -infinity in all rows of all sequences, with few and with many of them."""
    case = Case([(200, [(2, 12)] * seqs)], 4, 2, 64, 32, BF, 2)
    cu = list(case.cu_h)
    if bad == "falls":
        cu[2] = 0
    elif bad == "negative":
        cu[0] = -1
    elif bad == "past":
        cu[-1] += 1
    else:
        case.ends = i32([seqs, 0])
    case.cu = i32(cu)
    out, lse = case.run(err=1)
    assert not out.any() and (lse == -math.inf).all()
