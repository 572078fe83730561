"""The host side of the 16-bit paged operators, without a GPU."""
import subprocess
import sys

import pytest

from conftest import REPO

# ---------------------------------------------------------------------------
# workspace sizes
# ---------------------------------------------------------------------------
ATTN = """
from llm_accelerator_b200 import _native
lib = _native.load()
def attn(**kw):
    a = dict(q=256, k_cache=256, v_cache=256, out=256, table=256, lens=256, cu_q=256, q_token_stride=64,
             q_head_stride=64, out_token_stride=64, out_head_stride=64, page_stride=1024, head_stride=1024, row_stride=64,
             table_stride=1, n_seqs=1, n_slots=1, tokens=1, max_q=1, max_ctx=16, q_heads=1, kv_heads=1, dim=64,
             page_tokens=16, n_pages=1, dtype=2, scale=0.125)
    a.update(kw)
    return _native.AttnArgs(**a)
def size(**kw):
    return lib.q4gpu_paged_attention_workspace_bytes(attn(**kw))
"""


def child(code: str) -> None:
    """Runs in a process of its own: a crash of the library fails one test, not the session."""
    r = subprocess.run([sys.executable, "-c", ATTN + code], cwd=REPO, capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


@pytest.mark.parametrize("n_seqs,tokens,max_q,q_heads", [(0, 0, 1, 1), (1, 0, 1, 1), (1, 0, 64, 1), (0, 0, 64, 1),
                                                         (0, 0, 1, 32), (1, 0, 1, 32), (0, 5, 64, 1), (7, 0, 64, 1),
                                                         (0, 300, 512, 256), (1, 0, 2 ** 31 - 1, 256)])
def test_empty_calls_have_a_workspace_size(n_seqs, tokens, max_q, q_heads):
    child(f"""
kw = dict(n_seqs={n_seqs}, tokens={tokens}, max_q={max_q}, q_heads={q_heads}, max_ctx=4096)
n = size(**kw)
assert 0 < n < 1 << 26, n
assert lib.q4gpu_paged_attention(attn(**kw), None) == 0  # no work
""")
