"""Sequences of about 2^30 keys: a table that names one page again and again."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import paged  # noqa: E402
from test_gpu_paged import BF, TINY, U, i32, rnd, within  # noqa: E402

MOST, PAGE = 2 ** 30, 128


@pytest.fixture(scope="module")
def table():
    return torch.zeros(1, 2 ** 31 // PAGE, dtype=torch.int32, device="cuda")


def ref(pool, q, length, window, sinks):
    """Key j stands in row j % PAGE; those that no query sees are left out."""
    n, hq, dim = q.shape
    pos = torch.arange(length - n, length, device="cuda")[:, None]
    low = max(0, length - n - window + 1)
    key = torch.cat((torch.arange(min(sinks, low), device="cuda"), torch.arange(low, length, device="cuda")))
    seen = (key[None] <= pos) & ((key[None] > pos - window) | (key[None] < sinks))
    k, v = (pool[0, i][:, key % PAGE].double().repeat_interleave(hq // pool.shape[2], 0) for i in (0, 1))
    sc = (q.double().permute(1, 0, 2) @ k.transpose(1, 2) * dim ** -0.5).masked_fill(~seen, -math.inf)
    p = torch.softmax(sc, -1)
    return (p @ v).permute(1, 0, 2), (p @ v.abs()).permute(1, 0, 2), torch.logsumexp(sc, -1).permute(1, 0)


@pytest.mark.parametrize("length", [MOST, MOST - 1, MOST + 1, 2 ** 31 - 1])
@pytest.mark.parametrize("new", [1, 2, 300])
@pytest.mark.parametrize("window,sinks", [(100, 0), (700, 5)])
def test_windows_at_the_end(table, length, new, window, sinks):
    """Up to 2^30 keys are there; what lies behind is cut off and reported."""
    pool, q = rnd((1, 2, 2, PAGE, 64), BF, 1), rnd((new, 8, 64), BF, 2)
    op = paged.Attention(pool[:, 0], pool[:, 1], table, i32([length]), 8, window=window, sinks=sinks)
    lse = torch.empty(new, 8, device="cuda")
    out = op(q, None, i32([0, new]), max_q=new, lse=lse)
    want, mag, rl = ref(pool, q, min(length, MOST), window, sinks)
    u = U[BF]
    within(out, want, u * want.abs() + (u + 3e-4) * mag + TINY[BF])
    within(lse, rl, 3e-4 + 1e-6 * rl.abs())
    assert int(op.err.item()) == (length > MOST)


@pytest.mark.parametrize("length,prefix", [(MOST, MOST - 700), (2 ** 31 - 1, MOST - 700), (MOST - 3, MOST - 9)])
def test_own_keys_behind_a_long_prefix(table, length, prefix):
    """Two sequences of whose shared keys only one is there for real: a first sequence without any is reported."""
    pool, q = rnd((1, 2, 2, PAGE, 64), BF, 1), rnd((1, 8, 64), BF, 2)
    op = paged.SharedAttention(pool[:, 0], pool[:, 1], table.repeat(2, 1), i32([0, length]), 8)
    lse = torch.empty(1, 8, device="cuda")
    out = op(q, None, i32([0, 0, 1]), i32([0, 2]), i32([prefix]), lse=lse)
    end = min(length, MOST)
    want, mag, rl = ref(pool, q, end, end - prefix, 0)
    u = U[BF]
    within(out, want, u * want.abs() + (u + 3e-4) * mag + TINY[BF])
    within(lse, rl, 3e-4 + 1e-6 * rl.abs())
    assert int(op.err.item()) == 1
