"""The paged serving operators' C entry points refuse wrong arguments before any device work (no GPU needed),
and the ctypes structures have the header's layout."""
import ctypes as C
import re
import subprocess

import pytest

from conftest import REPO
from llm_accelerator_b200 import _native

ARG, SHAPE, ALIGN, WORKSPACE = -1001, -1002, -1003, -1005


@pytest.fixture(scope="module")
def lib():
    return _native.load()


def norm(**kw):
    a = _native.NormArgs(x=256, weight=256, out=256, rows=1, x_stride=64, out_stride=64, n=64, dtype=2, out_dtype=2,
                         eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), ARG), (dict(weight=None), ARG), (dict(out=None), ARG), (dict(n=0), SHAPE),
    (dict(n=32769), SHAPE), (dict(rows=-1), SHAPE), (dict(dtype=3), ARG), (dict(out_dtype=1), ARG),
    (dict(out_dtype=4), ARG), (dict(group=64), SHAPE), (dict(out_dtype=4, scale=256, group=12), SHAPE),
    (dict(out_dtype=4, scale=256, group=128), SHAPE), (dict(out_dtype=4, scale=256, group=64, x=258), ALIGN),
    (dict(out_dtype=4, scale=256, group=64, residual=256, residual_stride=3), ALIGN)])
def test_norm_refusals(lib, kw, rc):
    assert lib.q4gpu_add_rmsnorm(norm(**kw), None) == rc
    assert lib.q4gpu_last_error().startswith(b"norm")


def test_no_rows_is_no_work(lib):
    assert lib.q4gpu_add_rmsnorm(norm(rows=0), None) == 0
    assert lib.q4gpu_add_rmsnorm(None, None) == ARG


def rope(**kw):
    a = _native.RopeArgs(q=256, k=256, v=256, q_out=256, k_cache=256, v_cache=256, cos=256, sin=256, positions=256,
                         rows=256, q_token_stride=64, q_head_stride=64, k_token_stride=64, k_head_stride=64,
                         v_token_stride=64, v_head_stride=64, q_out_token_stride=64, q_out_head_stride=64,
                         page_stride=64, head_stride=64, row_stride=64, n_rows=16, tokens=1, q_heads=1, kv_heads=1,
                         dim=64, rot_dim=64, dtype=2, page_tokens=16, table_positions=4, eps=1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None, k=None, v=None), ARG), (dict(q_out=None), ARG), (dict(k_cache=None), ARG), (dict(v_cache=None), ARG),
    (dict(cos=None), ARG), (dict(positions=None), ARG), (dict(rows=None), ARG), (dict(tokens=-1), ARG),
    (dict(dtype=0), ARG), (dict(dim=0), SHAPE), (dict(dim=520), SHAPE), (dict(dim=60), SHAPE), (dict(rot_dim=80), SHAPE),
    (dict(rot_dim=8), SHAPE), (dict(table_positions=0), ARG), (dict(page_tokens=0), ARG), (dict(q=264), ALIGN),
    (dict(k_head_stride=4), ALIGN), (dict(row_stride=4), ALIGN), (dict(page_stride=1), ALIGN), (dict(q_gamma=258), ALIGN)])
def test_rope_refusals(lib, kw, rc):
    assert lib.q4gpu_rope_append(rope(**kw), None) == rc
    assert lib.q4gpu_last_error().startswith(b"rope")


def attn(**kw):
    a = _native.AttnArgs(q=256, k_cache=256, v_cache=256, out=256, table=256, lens=256, cu_q=256, q_token_stride=64,
                         q_head_stride=64, out_token_stride=64, out_head_stride=64, page_stride=1024, head_stride=1024,
                         row_stride=64, table_stride=1, n_seqs=1, n_slots=1, tokens=1, max_q=1, max_ctx=16, q_heads=1,
                         kv_heads=1, dim=64, page_tokens=16, n_pages=1, dtype=2, scale=0.125)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(q=None), ARG), (dict(k_cache=None), ARG), (dict(out=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG),
    (dict(cu_q=None), ARG), (dict(dtype=0), ARG), (dict(dim=96), SHAPE), (dict(page_tokens=8), SHAPE),
    (dict(page_tokens=48), SHAPE), (dict(q_heads=3, kv_heads=2), SHAPE), (dict(kv_heads=0), SHAPE),
    (dict(q_heads=512), SHAPE), (dict(n_seqs=-1), ARG), (dict(n_seqs=65536), ARG), (dict(window=-1), ARG),
    (dict(n_pages=0), ARG), (dict(n_slots=0), ARG), (dict(table_stride=0), ARG), (dict(scale=float("nan")), ARG),
    (dict(q=264), ALIGN), (dict(row_stride=68), ALIGN), (dict(out_head_stride=4), ALIGN), (dict(k_cache=264), ALIGN)])
def test_attention_refusals(lib, kw, rc):
    assert lib.q4gpu_paged_attention(attn(**kw), None) == rc
    assert lib.q4gpu_last_error().startswith(b"attention")


def test_attention_without_work_or_workspace(lib):
    assert lib.q4gpu_paged_attention(attn(n_seqs=0), None) == 0
    assert lib.q4gpu_paged_attention(attn(tokens=0), None) == 0
    assert lib.q4gpu_paged_attention_workspace_bytes(None) == 0
    assert lib.q4gpu_paged_attention_workspace_bytes(attn(dim=96)) == 0
    long = attn(max_ctx=100000)
    if lib.q4gpu_paged_attention_workspace_bytes(long):
        assert lib.q4gpu_paged_attention(long, None) == WORKSPACE


def pages(**kw):
    a = _native.PagesArgs(pool=256, table=256, lens=256, page_bytes=4096, block_bytes=2048, table_stride=4, n_pages=4,
                          page_tokens=16, n_slots=2)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,rc", [
    (dict(pool=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG), (dict(n_pages=0), ARG),
    (dict(page_tokens=0), ARG), (dict(n_slots=0), ARG), (dict(table_stride=0), ARG), (dict(page_bytes=5000), SHAPE),
    (dict(block_bytes=2040), SHAPE), (dict(page_tokens=15), SHAPE), (dict(pool=264), ALIGN),
    (dict(page_tokens=256), ALIGN)])
def test_pages_refusals(lib, kw, rc):
    assert lib.q4gpu_pages_fork(pages(**kw), 256, 256, 256, 1, None) == rc
    assert lib.q4gpu_pages_compact(pages(**kw), 256, 256, 256, 256, 1 << 20, None) == rc
    assert lib.q4gpu_last_error().startswith(b"pages")


def test_pages_more_refusals(lib):
    assert lib.q4gpu_pages_fork(pages(), 256, 256, 256, 0, None) == 0
    assert lib.q4gpu_pages_fork(pages(), 256, 256, 256, -1, None) == ARG
    assert lib.q4gpu_pages_fork(pages(), None, 256, 256, 1, None) == ARG
    need = lib.q4gpu_pages_compact_workspace_bytes(4)
    assert need >= 4 * 8 and lib.q4gpu_pages_compact_workspace_bytes(0) == 0
    assert lib.q4gpu_pages_compact(pages(), 256, 256, 256, 256, need - 1, None) == WORKSPACE
    assert lib.q4gpu_pages_compact(pages(), 256, 256, 256, 264, need, None) == ALIGN
    assert lib.q4gpu_pages_compact(pages(), 256, None, 256, 256, need, None) == ARG


def test_structures_match_the_header(tmp_path):
    names = {"q4gpu_norm_args": _native.NormArgs, "q4gpu_rope_args": _native.RopeArgs,
             "q4gpu_attn_args": _native.AttnArgs, "q4gpu_pages_args": _native.PagesArgs}
    lines = []
    for c, py in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include "q4gpu.h"\nint main(void) {' + "\n".join(lines) + "return 0;}\n")
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", str(REPO / "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        what, at = re.fullmatch(r"(\S+) (\d+)", line).groups()
        name, _, field = what.partition(".")
        py = names[name]
        assert int(at) == (getattr(py, field).offset if field else C.sizeof(py)), what
