"""The operators that serve and judge continuations refuse wrong arguments before any device work (no GPU needed)."""
import ctypes as C

import pytest

from llm_accelerator_b200 import _native
from test_paged_capi import attn

ARG, SHAPE, ALIGN, WORKSPACE = -1001, -1002, -1003, -1005


@pytest.fixture(scope="module")
def lib():
    return _native.load()


@pytest.mark.parametrize("kw,sinks,rc", [
    (dict(window=4), -1, ARG), (dict(window=-1), 4, ARG), (dict(window=4, dim=96), 4, SHAPE),
    (dict(window=4, q=264), 4, ALIGN), (dict(window=4), 4, WORKSPACE), (dict(window=4, cu_q=None), 4, ARG)])
def test_sink_refusals(lib, kw, sinks, rc):
    assert lib.q4gpu_sink_attention(attn(**kw), sinks, None) == rc
    assert lib.q4gpu_last_error().startswith(b"attention")


def test_sink_sizes(lib):
    """Sinks lengthen what is split over the GPU; a size without refusal for any number of them."""
    big = dict(window=600, tokens=64, max_q=64, max_ctx=1 << 20, table_stride=1 << 16, q_heads=8)
    plain = lib.q4gpu_paged_attention_workspace_bytes(attn(**big))
    sizes = [lib.q4gpu_sink_attention_workspace_bytes(attn(**big), n) for n in (0, 4, 5000, 2 ** 31 - 1)]
    assert sizes[0] == plain and sizes == sorted(sizes) and sizes[-1] < 1 << 28
    assert lib.q4gpu_sink_attention_workspace_bytes(attn(**big), -1) == 0
    assert lib.q4gpu_sink_attention(None, 4, None) == ARG
    assert lib.q4gpu_sink_attention(attn(window=4, tokens=0), 4, None) == 0
