"""The host side of the 16-bit paged operators, without a GPU."""
import subprocess
import sys
import threading
import weakref

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
    monkeypatch.setattr(paged, "_current", lambda: CPU.index)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
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


def test_workspaces_outlive_the_calls_that_used_them(lib):
    """A captured graph and queued work keep the address of a workspace that has become too small."""
    op, call = make_attn()
    held = []
    for need in (100, 101, 5000, 90000, 90001):
        lib.need = need
        call(len(held) + 1)
        assert op.workspace.numel() >= need and op.args.workspace == op.workspace.data_ptr()
        assert op.args.workspace_bytes == op.workspace.numel() and not op.workspace.any()
        if not held or held[-1]() is not op.workspace:
            held.append(weakref.ref(op.workspace))
    assert all(w() is not None for w in held)
    assert sum(w().numel() for w in held) <= 2 * held[-1]().numel() and len(held) == 5
    ws = held[-1]
    del op, call
    assert ws() is None


def test_workspaces_know_the_streams_that_use_them(lib, monkeypatch):
    """A workspace comes from the pool of the stream of its first call: its memory must not go back there while a
    later stream's work is queued."""
    told = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: told.append((t.data_ptr(), s)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "other")
    raw = {"stream": 7}
    monkeypatch.setattr(paged, "_stream", lambda index: raw["stream"])
    op, call = make_attn()
    lib.need = 100
    call(1)
    call(1)
    assert not told
    raw["stream"] = 9
    call(1)  # laid out like the last call
    call(2)
    assert {(op.workspace.data_ptr(), "other"), (op.err.data_ptr(), "other")} <= set(told)

    lib.q4gpu_pages_compact = lambda *a: 0
    pool = torch.zeros(4, 16, 8, dtype=torch.int16)
    table, lens = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    raw["stream"] = 7
    pages = paged.Pages(pool, table, lens, 16)
    del told[:]
    remap, n = torch.zeros(4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    pages.compact(table, remap, n)
    pages.fork(n, n, n)
    assert not told
    raw["stream"] = 9
    pages.compact(table, remap, n)
    assert (pages.workspace.data_ptr(), "other") in told


def test_a_call_under_capture_leaves_the_workspace_alone(lib, monkeypatch):
    """What is allocated under capture is zeroed by the graph's replays only, so it serves that call and no other."""
    op, call = make_attn()
    lib.need = 100
    call(1)
    own = op.workspace.data_ptr()
    capturing = {"now": True}
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing["now"])
    lib.need = 5000
    call(2)
    assert lib.calls[-1][4] not in (None, own) and lib.calls[-1][5] >= 5000
    assert op.workspace.data_ptr() == own and op.args.workspace == own
    call(2)  # the same layout: the small workspace must not serve it
    assert lib.calls[-1][4] != own and lib.calls[-1][5] >= 5000
    capturing["now"] = False
    call(2)
    assert lib.calls[-1][4] == op.workspace.data_ptr() and op.workspace.numel() >= 5000


# ---------------------------------------------------------------------------
# the cache's bookkeeping
# ---------------------------------------------------------------------------
def make_cache(lib, monkeypatch):
    monkeypatch.setattr(paged.PagedCache, "_up", lambda self, a: torch.from_numpy(a))
    return paged.PagedCache(1, 8, 16, 1, 8, max_seqs=3, max_ctx=64, device=CPU)


def state(c):
    return (c._held.copy(), [list(h) for h in c._held], list(c._len), list(c._users), sorted(c._free), c.table.tolist(),
            c.lens.tolist())


@pytest.mark.parametrize("bad", [-1, 3, -3, 2 ** 31])
def test_cache_refuses_unknown_sequences(lib, monkeypatch, bad):
    c = make_cache(lib, monkeypatch)
    c.extend([0, 2], [20, 5])
    before = state(c)
    for call in (lambda: c.extend([bad], [1]), lambda: c.extend([0, bad], [1, 1]), lambda: c.extend([bad, 2], [1, 1]),
                 lambda: c.fork(bad, [1]), lambda: c.fork(0, [bad]), lambda: c.fork(0, [1, bad]), lambda: c.free(bad),
                 lambda: c.length(bad)):
        with pytest.raises(ValueError):
            call()
        assert state(c) == before
    c.extend([1], [1])
    c.free(2)
    assert c.lens.tolist() == [20, 1, 0] and c.length(0) == 20 and c.free_pages == 5


def make_decoder(lib, monkeypatch, vocab=10, **kw):
    from llm_accelerator_b200 import fp32_diag as F
    from llm_accelerator_b200 import paged_decode
    T, h = _native, 64
    monkeypatch.setattr(paged.PagedCache, "_up", lambda self, a: torch.from_numpy(a))
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    z = torch.zeros
    layer = {T.T_Q: z(F.HEADS * F.HEAD_DIM, h), T.T_K: z(F.KV_HEADS * F.HEAD_DIM, h),
             T.T_V: z(F.KV_HEADS * F.HEAD_DIM, h), T.T_O: z(h, F.HEADS * F.HEAD_DIM), T.T_GATE: z(F.INTER, h),
             T.T_UP: z(F.INTER, h), T.T_DOWN: z(h, F.INTER), T.T_INPUT_GAMMA: z(h), T.T_POST_GAMMA: z(h),
             T.T_Q_GAMMA: z(F.HEAD_DIM), T.T_K_GAMMA: z(F.HEAD_DIM)}
    return paged_decode.PagedDecoder({"embed": z(vocab, h), "final": z(h), "layers": [layer]}, max_seqs=2, max_ctx=64,
                                     page_tokens=16, dtype=torch.half, **kw)


@pytest.mark.parametrize("tokens", [[[3, 10]], [[-1]], [[1], [2 ** 40]]])
def test_decoder_refuses_tokens_outside_the_vocabulary(lib, monkeypatch, tokens):
    d = make_decoder(lib, monkeypatch)
    before = state(d.cache)
    with pytest.raises(ValueError, match="token"):
        d.forward(list(range(len(tokens))), tokens)
    assert state(d.cache) == before


def test_decoder_refuses_empty_prompts(lib, monkeypatch):
    d = make_decoder(lib, monkeypatch)
    for call in (lambda: d.prefill(0, []), lambda: d.prefill(0, [1, 2], -1), lambda: d.forward([0], [[]]),
                 lambda: d.forward([], []), lambda: d.forward([0, 1], [[1]])):
        with pytest.raises(ValueError):
            call()
    assert d.cache.free_pages == 8 and d.cache.length(0) == 0


@pytest.mark.parametrize("max_ctx", [2 ** 31 - 1, 2 ** 31 - 100])
@pytest.mark.parametrize("kw", [dict(), dict(dim=128), dict(n_seqs=3, tokens=3, q_heads=4, kv_heads=2)])
def test_contexts_near_the_largest_are_split_like_long_ones(max_ctx, kw):
    """One decode over a context of unknown length is spread over the GPU, whatever bound stands for 'unknown'."""
    child(f"""
kw = dict({kw!r}, table_stride=1 << 27)
assert size(max_ctx={max_ctx}, **kw) == size(max_ctx=1 << 26, **kw) > size(max_ctx=16, **kw)
""")


@pytest.mark.parametrize("make", [make_norm, make_rope, make_attn])
def test_calls_while_another_device_is_current_are_refused(lib, monkeypatch, make):
    """The default stream's handle is the same on every device: a launch would go to the current one."""
    op, call = make()
    call(2)
    monkeypatch.setattr(paged, "_current", lambda: 1)
    for _ in range(2):
        with pytest.raises(ValueError, match="current device"):
            call(2)
    assert len(lib.calls) == 1


def test_page_calls_while_another_device_is_current_are_refused(lib, monkeypatch):
    table, lens, remap = (torch.zeros(n, dtype=torch.int32) for n in (2, 1, 4))
    pages = paged.Pages(torch.zeros(4, 16, 8, dtype=torch.int16), table[None], lens, 16)
    lib.q4gpu_pages_fork = lib.q4gpu_pages_compact = lambda *a: pytest.fail("launched")
    monkeypatch.setattr(paged, "_current", lambda: 1)
    with pytest.raises(ValueError, match="current device"):
        pages.fork(lens, lens, lens)
    with pytest.raises(ValueError, match="current device"):
        pages.compact(table[None], remap, lens)


def test_decoder_8bit_weights_with_rows_of_zeros(lib, monkeypatch):
    d = make_decoder(lib, monkeypatch, eight_bit=True)
    lay = d.layers[0]
    assert lay["gu8_scale"].isfinite().all()
    assert not (lay["gu8"].float() * lay["gu8_scale"].t()).isnan().any()


def test_table_pages_refusals_and_default():
    child("""
assert lib.q4gpu_paged_attention(attn(table_pages=-1), None) == -1001 and size(table_pages=-1) == 0
assert size(table_pages=5) == size() > 0
""")
