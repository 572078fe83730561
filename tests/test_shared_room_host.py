"""Attention operators that share a workspace, without a GPU (a stand-in for the library)."""
import threading

import pytest

torch = pytest.importorskip("torch")

from llm_accelerator_b200 import paged  # noqa: E402
from test_paged_host import lib  # noqa: E402, F401


def make(share=None):
    c = torch.zeros(2, 1, 16, 64, dtype=torch.half)
    op = paged.Attention(c, c, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), q_heads=2,
                         share=share)
    return op, lambda n: op(torch.zeros(n, 2, 64, dtype=torch.half), None, torch.tensor([0, n], dtype=torch.int32))


@pytest.fixture
def told(monkeypatch):
    seen = []
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda t, s: seen.append((t.data_ptr(), s)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: "now")
    return seen


def test_layers_share_one_workspace(lib, told):  # noqa: F811
    ops = [make()]
    ops += [make(ops[0][0]) for _ in range(3)]
    lib.need = 1000
    for _, call in ops:
        call(1)
    assert len({op.workspace.data_ptr() for op, _ in ops}) == 1 and len(ops[0][0].room) == 1
    assert {(ops[0][0].workspace.data_ptr(), "now")} == set(told) and len(told) == 3  # (memory of the first one's call)
    old = ops[0][0].workspace
    lib.need = 3000
    ops[2][1](2)  # grows for all, and leaves the others what they have until they need more
    assert lib.calls[-1][4] == ops[2][0].workspace.data_ptr() != old.data_ptr()
    ops[1][1](1)
    assert lib.calls[-1][4] in (old.data_ptr(), ops[2][0].workspace.data_ptr())
    ops[1][1](2)
    assert lib.calls[-1][4] == ops[2][0].workspace.data_ptr() and lib.calls[-1][5] >= 3000
    assert [t.data_ptr() for t in ops[3][0].room] == [old.data_ptr(), ops[2][0].workspace.data_ptr()]
    assert any(t is old for t in ops[0][0].own)  # graphs may know it


def test_captured_call_takes_what_another_made(lib, told, monkeypatch):  # noqa: F811
    (a, first), lib.need = make(), 500
    first(1)
    b, second = make(a)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    second(1)
    assert lib.calls[-1][4] == a.workspace.data_ptr()
    lib.need = 5000
    second(2)  # more than there is: memory of the graph's own
    assert lib.calls[-1][4] != a.workspace.data_ptr() and lib.calls[-1][5] == 5000 and len(a.room) == 1


def test_threads_with_operators_that_share(lib, told):  # noqa: F811
    """One at a time: the library's launches of a call are not mixed with another's."""
    (a, first), lib.need = make(), 100
    b, second = make(a)
    first(1)
    inside, during, errors = threading.Event(), [], []

    def other():
        inside.wait(5)
        try:
            second(3)
        except BaseException as e:  # noqa: BLE001
            errors.append(e)
    t = threading.Thread(target=other)

    def hold():
        if not inside.is_set():
            n = len(lib.calls)
            inside.set()
            t.join(0.3)
            during.append(len(lib.calls) - n)
    lib.during = hold
    t.start()
    first(2)
    t.join(5)
    assert during == [0] and not errors


def test_refusals(lib):  # noqa: F811
    a, _ = make()
    a.device = torch.device("meta")
    with pytest.raises(ValueError, match="one device"):
        make(a)
