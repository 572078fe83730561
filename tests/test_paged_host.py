"""The host side of the 16-bit paged operators, without a GPU."""
import subprocess
import sys
import threading

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


# ---------------------------------------------------------------------------
# operators on CPU tensors with a stand-in for the library
# ---------------------------------------------------------------------------
torch = pytest.importorskip("torch")

from llm_accelerator_b200 import _native, paged  # noqa: E402

CPU = torch.device("cpu")


class Lib:
    """Records what each call was given; `during` runs inside a call, where the library has let other threads run."""

    def __init__(self):
        self.calls, self.during, self.need = [], lambda: None, 0

    def _call(self, a, *fields):
        before = [getattr(a, f) for f in fields]
        self.during()
        self.calls.append(before)
        assert before == [getattr(a, f) for f in fields], "another thread's call changed this one's arguments"
        return 0

    def q4gpu_add_rmsnorm(self, a, stream):
        return self._call(a, "x", "out", "rows")

    def q4gpu_rope_append(self, a, stream):
        return self._call(a, "q", "q_out", "positions", "tokens")

    def q4gpu_paged_attention_workspace_bytes(self, a):
        return self.need

    def q4gpu_paged_attention(self, a, stream):
        return self._call(a, "q", "out", "cu_q", "tokens", "workspace", "workspace_bytes")

    def q4gpu_pages_compact_workspace_bytes(self, n):
        return 64

    def q4gpu_pages_fork(self, *a):
        return 0


@pytest.fixture
def lib(monkeypatch):
    fake = Lib()
    monkeypatch.setattr(_native, "load", lambda: fake)
    monkeypatch.setattr(paged, "_cuda", lambda t, name: CPU)
    monkeypatch.setattr(paged, "_stream", lambda index: 7)
    return fake


def make_norm():
    op = paged.AddRmsNorm(torch.ones(8))
    return op, lambda n: op(torch.zeros(n, 8))


def make_rope():
    op = paged.RopeAppend(torch.ones(4, 8), torch.ones(4, 8))
    return op, lambda n: op(torch.zeros(n, 2, 16, dtype=torch.half), None, None, torch.zeros(n, dtype=torch.int32), None,
                            None, None)


def make_attn():
    c = torch.zeros(2, 1, 16, 64, dtype=torch.half)
    op = paged.Attention(c, c, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), q_heads=2)
    return op, lambda n: op(torch.zeros(n, 2, 64, dtype=torch.half), None, torch.tensor([0, n], dtype=torch.int32))


@pytest.mark.parametrize("make", [make_norm, make_rope, make_attn])
def test_two_threads_with_one_operator(lib, make):
    """A second thread calls the operator while the first is inside the library."""
    op, call = make()
    inside, errors, others = threading.Event(), [], []

    def other():
        inside.wait(5)
        try:
            call(5)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)

    second = threading.Thread(target=other)

    def during():
        if not inside.is_set():
            inside.set()
            second.join(0.3)  # long enough for the other call, if nothing holds it up

    lib.during = during
    second.start()
    call(3)
    second.join()
    assert not errors
    assert len(lib.calls) == 2 and [c[2] if len(c) == 3 else c[3] for c in lib.calls] == [3, 5]
