"""The workspace that attention asks for is what its launch lays out (no GPU needed)."""
import pytest

from llm_accelerator_b200 import _native
from test_paged_capi import attn

WORKSPACE = -1005


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def laid_out(n_seqs, kv_heads, dim, max_ctx):
    """Bytes of a call of single tokens without sinks: a counter a CTA, and two tiles of 16 rows a CTA, of `dim` sums and
    a maximum and a sum each.  A CTA has at least one (sequence, head) or six units of 128 keys, three more of which stand
    for the start of each."""
    units = -(-max_ctx // 128) + 3
    ctas = min(n_seqs * kv_heads * max(1, -(-units // 6) + 1), 148 * (2 if dim == 64 else 1))
    return -(-(4096 * 4 + ctas * 2 * 16 * (8 + 4 * dim)) // 16) * 16


@pytest.mark.parametrize("max_ctx", [0, 1, 127, 128, 129, 1024, 8192, 2 ** 31 - 1])
@pytest.mark.parametrize("n_seqs", [1, 2, 4, 20, 256])
@pytest.mark.parametrize("kv_heads,dim", [(1, 64), (2, 128), (8, 64), (8, 128)])
@pytest.mark.parametrize("window", [0, 1, 600])
def test_sizes_without_sinks(lib, n_seqs, kv_heads, dim, max_ctx, window):
    a = attn(n_seqs=n_seqs, n_slots=n_seqs, tokens=n_seqs, q_heads=2 * kv_heads, kv_heads=kv_heads, dim=dim,
             max_ctx=max_ctx, table_stride=1 << 12, window=window)
    want = laid_out(n_seqs, kv_heads, dim, max_ctx)
    assert lib.q4gpu_paged_attention_workspace_bytes(a) == want
    assert lib.q4gpu_sink_attention_workspace_bytes(a, 0) == want
    if window == 0:  # nothing for sinks to add to
        assert lib.q4gpu_sink_attention_workspace_bytes(a, 4) == want
    a.workspace, a.workspace_bytes = 256, want - 1
    assert lib.q4gpu_paged_attention(a, None) == WORKSPACE


def test_a_bound_of_nothing_does_not_shrink_it_below_a_launch(lib):
    """One sequence of 8 key heads of 128, max_ctx = 0: 16 CTAs."""
    a = attn(n_seqs=1, tokens=1, q_heads=16, kv_heads=8, dim=128, max_ctx=0)
    assert lib.q4gpu_paged_attention_workspace_bytes(a) == 16384 + 16 * 32 * 520
