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


def logprob(**kw):
    a = _native.LogprobArgs(logits=256, targets=256, logprob=256, entropy=256, top_logprob=256, rank=256, top_index=256,
                            rows=1, stride=64, vocab=64, top=5, dtype=2)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(logits=None), ARG), (dict(entropy=None), ARG), (dict(logprob=None), ARG), (dict(rank=None), ARG),
    (dict(top_logprob=None), ARG), (dict(top_index=None), ARG), (dict(dtype=3), ARG), (dict(rows=-1), SHAPE),
    (dict(rows=2 ** 31), SHAPE), (dict(vocab=0), SHAPE), (dict(top=-1), SHAPE), (dict(top=33), SHAPE),
    (dict(top=5, vocab=4), SHAPE), (dict(logits=257), ALIGN), (dict(logits=258, dtype=0), ALIGN)])
def test_logprob_refusals(lib, kw, rc):
    assert lib.q4gpu_token_logprobs(logprob(**kw), None) == rc
    assert lib.q4gpu_last_error().startswith(b"logprobs")


def test_logprobs_of_no_rows(lib):
    assert lib.q4gpu_token_logprobs(logprob(rows=0, logits=None), None) == 0
    assert lib.q4gpu_token_logprobs(None, None) == ARG


def test_logprob_structure(tmp_path):
    """ctypes and the header agree on the arguments' layout."""
    import subprocess

    from conftest import REPO
    src = "#include <stddef.h>\n#include <stdio.h>\n#include \"q4gpu.h\"\nint main(void) {\n"
    for name, _ in _native.LogprobArgs._fields_:
        src += f'  printf("{name} %zu\\n", offsetof(q4gpu_logprob_args, {name}));\n'
    src += '  printf("size %zu\\n", sizeof(q4gpu_logprob_args));\n  return 0;\n}\n'
    (tmp_path / "t.c").write_text(src)
    subprocess.run(["gcc", "-I", str(REPO / "include"), "-o", str(tmp_path / "t"), str(tmp_path / "t.c")], check=True)
    out = dict(line.split() for line in subprocess.run([str(tmp_path / "t")], capture_output=True, text=True,
                                                       check=True).stdout.splitlines())
    assert int(out.pop("size")) == C.sizeof(_native.LogprobArgs)
    assert {k: int(v) for k, v in out.items()} == {n: getattr(_native.LogprobArgs, n).offset
                                                   for n, _ in _native.LogprobArgs._fields_}


def shared(**kw):
    return _native.SharedArgs(**(dict(cu_group=256, prefix_lens=256, n_groups=1, max_prefix=16) | kw))


@pytest.mark.parametrize("kw,sh,rc", [
    (dict(), dict(cu_group=None), ARG), (dict(), dict(prefix_lens=None), ARG), (dict(), dict(n_groups=-1), ARG),
    (dict(), dict(n_groups=65536), ARG), (dict(), dict(max_prefix=-1), ARG), (dict(window=5), dict(), ARG),
    (dict(dim=96), dict(), SHAPE), (dict(q=264), dict(), ALIGN), (dict(), dict(), WORKSPACE),
    (dict(workspace=264, workspace_bytes=1 << 30), dict(), ALIGN),
    (dict(tokens=2 ** 31 - 1, max_q=2 ** 31 - 1, q_heads=256, workspace=256, workspace_bytes=1 << 62), dict(), SHAPE)])
def test_shared_refusals(lib, kw, sh, rc):
    assert lib.q4gpu_shared_attention(attn(**kw), shared(**sh), None) == rc
    assert lib.q4gpu_last_error().startswith(b"attention")


def test_shared_sizes(lib):
    size = lib.q4gpu_shared_attention_workspace_bytes
    assert lib.q4gpu_shared_attention(attn(), None, None) == ARG and size(attn(), None) == 0
    assert lib.q4gpu_shared_attention(attn(tokens=0), shared(), None) == 0
    assert size(attn(window=3), shared()) == 0
    one = size(attn(q_heads=16, kv_heads=8, dim=128, max_ctx=8192), shared())
    # both sets of a row's unnormalised sums and statistics, beside the few-row kernel's own
    many = dict(q_heads=16, kv_heads=8, dim=128, max_ctx=8192, n_seqs=64, tokens=64)
    assert 0 < one < size(attn(**many), shared(max_prefix=8000)) < 1 << 26
    assert size(attn(**many), shared()) >= 2 * 64 * 16 * (128 + 2) * 4
    assert size(attn(tokens=2 ** 31 - 1, max_q=2 ** 31 - 1, q_heads=256), shared(n_groups=65535)) > 1 << 40
