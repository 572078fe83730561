"""Corners of the 16-bit paged operators: degenerate scales and magnitudes, what only the device can see, layouts of
the cache and of calls, streams and graphs.

Bounds are those of the ordinary cases (``test_gpu_paged``): an attention result is within u |out| + (u + 3e-4)
sum p |v| of the 64-bit form and its log-sum within 3e-4 + 1e-6 |lse|; with the scale 0 the weights are exactly 1
and the same bounds hold."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("needs a CUDA device", allow_module_level=True)

from llm_accelerator_b200 import _native, paged  # noqa: E402
from test_gpu_paged import BF, HF, SF, TINY, U, angles, attn_ref, i32, make, norm_ref, rnd, within  # noqa: E402


def operator(pool, table, lens, hq, **kw):
    return paged.Attention(pool[:, 0], pool[:, 1], table, lens, q_heads=hq, **kw)


def close(got, lse, ref, mag, rl, dtype):
    u = U[dtype]
    within(got, ref, u * ref.abs() + (u + 3e-4) * mag + TINY[dtype])
    none = rl == -math.inf
    assert torch.equal(lse == -math.inf, none)
    within(lse[~none], rl[~none], 3e-4 + 1e-6 * rl[~none].abs())


def check(op, pool, table, lens, cu, q, scale, window=0, max_q=None, seq_ids=None):
    """One call against the 64-bit form; returns what it gave."""
    lse = torch.full(q.shape[:2], 5.0, device="cuda")
    out = torch.full_like(q, 5.0)
    most = int((cu[1:] - cu[:-1]).max()) if max_q is None else max_q
    op(q, out, cu, max_q=most, max_ctx=max(1, int(lens.max())), lse=lse, seq_ids=seq_ids)
    close(out, lse, *attn_ref(pool, table, lens, cu, q, scale, window, seq_ids), q.dtype)
    return out, lse


@pytest.mark.parametrize("hq,hk", [(4, 2), (32, 1)])
@pytest.mark.parametrize("max_q", [1, 64, 4096])
def test_attention_of_an_empty_step(hq, hk, max_q):
    pool, table, lens, cu, q = make([1], [10], hq, hk, 64, 32, BF, 20)
    op = operator(pool, table, lens, hq)
    assert op(q[:0], None, i32([0, 0]), max_q=max_q).shape == (0, hq, 64)
    assert op(q[:0], None, i32([0]), max_q=max_q).shape == (0, hq, 64)
    check(op, pool, table, lens, cu, q, 64 ** -0.5)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,old", [([1, 2], [300, 0]), ([200], [300]), ([3, 40, 300, 1], [500, 0, 20, 70]),
                                     ([70], [4000])])
@pytest.mark.parametrize("window", [0, 70])
def test_attention_scale_zero_is_the_mean(dtype, dim, new, old, window):
    args = make(new, old, 4, 2, dim, 32, dtype, 21)
    for scale in (0.0, -0.0, 1e-44):
        check(operator(*args[:3], 4, scale=scale, window=window), *args, scale, window)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,old", [([1, 2], [300, 0]), ([3, 40, 300, 1], [500, 0, 20, 70])])
def test_attention_negative_scale(dim, new, old):
    args = make(new, old, 4, 2, dim, 32, BF, 22)
    check(operator(*args[:3], 4, scale=-dim ** -0.5), *args, -dim ** -0.5)
