"""16-bit paged serving operators on torch CUDA tensors.

The floating-point companions of the fixed-point kernels, for callers that
hold activations in bf16 or f16: the operators of one layer step over a paged
K/V cache, and what happens to the cache's pages between steps.

* ``AddRmsNorm``  residual addition + RMS norm, 16-bit or 8-bit output with scales
* ``RopeAppend``  q/k head norm, rotary positions, K/V stored in their pages
* ``Attention``   a chunk of new tokens per sequence (or one) over the pages
* ``SharedAttention``  the same where groups of sequences share their first keys
* ``TokenLogprobs``  log probabilities of given tokens, entropy, likeliest tokens
* ``Pages``       forking sequences, packing the pages in use
* ``PagedCache``  a pool with its tables, and which pages are free

Each operator is an object that holds what a serving loop keeps (weights,
tables, cache, workspace) and is called with the step's tensors.  Calls
enqueue on torch's current stream and do not synchronise; a workspace belongs
to its object, so one object's calls run on one stream at a time (and a captured
graph that holds them needs the object as long as it is replayed).  Threads may
share an object: a lock keeps the arguments of a call together until the library
has taken them.  Nothing has a reference counterpart (the reference decodes one
token at a time in fixed point with a flat cache of 256 positions,
``FPGA_Project/software/qmap_one_token_runtime/qmap_one_token_runtime.h:369-500``).
Wrong arguments raise ``ValueError`` here or ``_native.Q4GpuError`` from the
library, both before any device work; there is no CPU fallback.
"""
from __future__ import annotations

import heapq
import threading
from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from . import _native

_DTYPES = {torch.float32: _native.DT_F32, torch.float16: _native.DT_F16, torch.bfloat16: _native.DT_BF16,
           torch.float8_e4m3fn: _native.DT_E4M3, torch.int8: _native.DT_S8}


# torch's current stream of a device as a cudaStream_t.  The public accessor builds a Stream
# object first (3 us on the host, as long as a small kernel); this is the call inside it.
_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                  lambda index: torch.cuda.current_stream(index).cuda_stream)
_current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _at(index: int) -> int:
    """The current stream of device `index`, which has to be the current device: a launch goes to that one, and the
    default stream's handle is the same on all."""
    if _current() != index:
        raise ValueError(f"the operator is on cuda:{index}, the current device is cuda:{_current()}")
    return _stream(index)


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _on(t: torch.Tensor, device: torch.device, name: str, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """`t`, if it is a CUDA tensor of this device (and type)."""
    if t is None:
        raise ValueError(f"{name} is needed")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{name} is {t.dtype}, expected {dtype}")
    return t


def _cuda(t: torch.Tensor, name: str) -> torch.device:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU fallback)")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{name} is on {t.device}, the current device is cuda:{torch.cuda.current_device()}")
    return t.device


class AddRmsNorm:
    """h = x + residual; y = h / sqrt(mean(h^2) + eps) * weight, per row.

    ``out_dtype`` is the weight's type (default), ``torch.float8_e4m3fn`` or
    ``torch.int8``; an 8-bit output has one float32 scale per ``group`` columns
    (0: per row), y = out * scale.
    """

    def __init__(self, weight: torch.Tensor, eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
                 group: int = 0):
        self.lib = _native.load()
        self.device = _cuda(weight, "weight")
        self.index = self.device.index
        _need(weight.dim() == 1 and weight.is_contiguous(), "weight must be a contiguous vector")
        _need(weight.dtype in (torch.float32, torch.float16, torch.bfloat16), f"weight is {weight.dtype}")
        self.weight, self.n, self.dtype = weight, weight.shape[0], weight.dtype
        self.lock = threading.Lock()
        self.out_dtype = out_dtype or weight.dtype
        _need(self.out_dtype in _DTYPES, f"unsupported output type {self.out_dtype}")
        self.narrow = self.out_dtype in (torch.float8_e4m3fn, torch.int8)
        self.groups = self.n // group if group else 1
        self.args = _native.NormArgs(weight=weight.data_ptr(), n=self.n, group=group, dtype=_DTYPES[weight.dtype],
                                     out_dtype=_DTYPES[self.out_dtype], eps=eps)

    def _rows(self, t: torch.Tensor, rows: int, name: str, dtype: torch.dtype) -> int:
        if t.dtype != dtype or t.device != self.device:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {dtype} on {self.device}")
        if t.shape != (rows, self.n):
            raise ValueError(f"{name} must be [{rows}, {self.n}], got {tuple(t.shape)}")
        row, one = t.stride()
        if one != 1 and self.n > 1:
            raise ValueError(f"{name} must have contiguous rows")
        return row

    def __call__(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                 residual_out: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None):
        """x, residual, residual_out, out: [rows, n]; returns out, or (out, scale) for 8 bits."""
        with self.lock:
            a, dtype = self.args, self.dtype
            if x.dim() != 2:
                raise ValueError("x must be [rows, n]")
            a.rows = rows = len(x)
            a.x_stride = self._rows(x, rows, "x", dtype)
            a.x = x.data_ptr()
            if out is None:
                out = torch.empty(rows, self.n, dtype=self.out_dtype, device=self.device)
            a.out_stride = self._rows(out, rows, "out", self.out_dtype)
            a.out = out.data_ptr()
            a.residual = a.residual_out = a.scale = None
            if residual is not None:
                a.residual_stride = self._rows(residual, rows, "residual", dtype)
                a.residual = residual.data_ptr()
            if residual_out is not None:
                a.residual_out_stride = self._rows(residual_out, rows, "residual_out", dtype)
                a.residual_out = residual_out.data_ptr()
            if self.narrow:
                if scale is None:
                    scale = torch.empty(rows, self.groups, dtype=torch.float32, device=self.device)
                _on(scale, self.device, "scale", torch.float32)
                _need(scale.shape == (rows, self.groups) and scale.is_contiguous(),
                      f"scale must be contiguous [{rows}, {self.groups}]")
                a.scale = scale.data_ptr()
            rc = self.lib.q4gpu_add_rmsnorm(a, _at(self.index))
            if rc:
                _native.check(rc, "q4gpu_add_rmsnorm")
            return (out, scale) if self.narrow else out


class _Err:
    """The device error word of an operator: `check` waits for the stream and raises once.

    ``own`` is the memory that the operator itself allocated.  torch keeps freed memory back for work queued on the
    stream it came from only, so a call on another stream is made known to it.
    """

    def _new_err(self) -> None:
        self.err = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.index = self.device.index
        self.own, self.stream = [self.err], _stream(self.index)

    def _here(self) -> int:
        """The current stream, which may use what the operator owns."""
        now = _at(self.index)
        if now != self.stream:
            self.stream = now
            for t in self.own:
                t.record_stream(torch.cuda.current_stream(self.device))
        return now

    def check(self) -> None:
        what = int(self.err.item())
        if what:
            self.err.zero_()
        if what == 2:
            raise _native.Q4GpuError(f"{type(self).__name__}: a wait inside a kernel ran out; its output is incomplete")
        if what:
            raise _native.Q4GpuError(f"{type(self).__name__}: a position, row, page, slot, length, query range or "
                                     "token was out of range; what it named was left untouched")


class RopeAppend(_Err):
    """Rotary positions of new tokens, keys and values stored in their pages.

    ``cos`` / ``sin`` float32 [positions, rot_dim / 2] (``tables.rope_float_tables``);
    ``q_gamma`` / ``k_gamma`` [dim] norm each head vector first.
    """

    def __init__(self, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False,
                 q_gamma: Optional[torch.Tensor] = None, k_gamma: Optional[torch.Tensor] = None, eps: float = 1e-6):
        self.lib = _native.load()
        self.device = _cuda(cos, "cos")
        for t, name in ((cos, "cos"), (sin, "sin")):
            _on(t, self.device, name, torch.float32)
            _need(t.dim() == 2 and t.is_contiguous() and t.shape == cos.shape, f"{name} must be [positions, rot / 2]")
        self.cos, self.sin, self.q_gamma, self.k_gamma = cos, sin, q_gamma, k_gamma
        self.layout, self.lock = None, threading.Lock()
        self._new_err()
        a = self.args = _native.RopeArgs(cos=cos.data_ptr(), sin=sin.data_ptr(), table_positions=cos.shape[0],
                                         rot_dim=2 * cos.shape[1], interleaved=int(interleaved), eps=eps,
                                         err_flag=self.err.data_ptr())
        self.gamma_dim = None
        for g, name in ((q_gamma, "q_gamma"), (k_gamma, "k_gamma")):
            if g is not None:
                _on(g, self.device, name)
                _need(g.dim() == 1 and g.is_contiguous(), f"{name} must be a contiguous vector")
                _need(self.gamma_dim in (None, (g.shape[0], g.dtype)), "q_gamma and k_gamma differ in size or type")
                self.gamma_dim = (g.shape[0], g.dtype)
                setattr(a, name, g.data_ptr())

    def __call__(self, q: Optional[torch.Tensor], k: Optional[torch.Tensor], v: Optional[torch.Tensor],
                 positions: torch.Tensor, rows: Optional[torch.Tensor], k_cache: Optional[torch.Tensor],
                 v_cache: Optional[torch.Tensor], q_out: Optional[torch.Tensor] = None):
        """q [tokens, q_heads, dim], k / v [tokens, kv_heads, dim] (any of them None);
        positions int32 [tokens]; rows int64 [tokens], the cache row of each token
        (page * page_tokens + offset, negative: not stored); k_cache / v_cache
        [pages, kv_heads, page_tokens, dim].  Returns q_out (default: q in place)."""
        with self.lock:
            layout = None
            if not any(t is None for t in (q, k, v, q_out, positions, rows, k_cache, v_cache)):
                # what the checks below look at: tensors laid out like the last call's need only their addresses
                layout = (q.shape, q.stride(), q.dtype, q.device,
                          q_out.shape, q_out.stride(), q_out.dtype, q_out.device,
                          k.shape, k.stride(), k.dtype, k.device, v.shape, v.stride(), v.dtype, v.device,
                          positions.shape, positions.stride(), positions.dtype, positions.device,
                          rows.shape, rows.stride(), rows.dtype, rows.device,
                          k_cache.shape, k_cache.stride(), k_cache.dtype, k_cache.device,
                          v_cache.shape, v_cache.stride(), v_cache.dtype, v_cache.device)
                if layout == self.layout:
                    a = self.args
                    a.q, a.q_out, a.k, a.v = q.data_ptr(), q_out.data_ptr(), k.data_ptr(), v.data_ptr()
                    a.k_cache, a.v_cache = k_cache.data_ptr(), v_cache.data_ptr()
                    a.positions, a.rows = positions.data_ptr(), rows.data_ptr()
                    return self._launch(q_out)
            self.layout = None
            ref = q if q is not None else k if k is not None else v
            _need(ref is not None, "one of q, k, v is needed")
            tokens, _, dim = ref.shape
            dtype, a = ref.dtype, self.args
            if dtype not in (torch.float16, torch.bfloat16):
                raise ValueError(f"head vectors are {dtype}, expected float16 or bfloat16")
            if self.gamma_dim is not None and self.gamma_dim != (dim, dtype):
                raise ValueError(f"gamma does not match head vectors of {dim} x {dtype}")
            a.tokens, a.dim, a.dtype, a.q_heads, a.kv_heads = tokens, dim, _DTYPES[dtype], 0, 0
            a.q = a.k = a.v = a.q_out = a.k_cache = a.v_cache = a.positions = a.rows = None
            if q is not None or k is not None:
                _on(positions, self.device, "positions", torch.int32)
                if positions.shape != (tokens,) or not positions.is_contiguous():
                    raise ValueError(f"positions must be a contiguous vector of {tokens}")
                a.positions = positions.data_ptr()
            if q is not None:
                q_out = q if q_out is None else q_out
                a.q_heads = q.shape[1]
                a.q, a.q_token_stride, a.q_head_stride = self._heads(q, tokens, a.q_heads, dim, dtype, "q")
                a.q_out, a.q_out_token_stride, a.q_out_head_stride = self._heads(q_out, tokens, a.q_heads, dim, dtype,
                                                                                 "q_out")
            if k is not None or v is not None:
                _on(rows, self.device, "rows", torch.int64)
                if rows.shape != (tokens,) or not rows.is_contiguous():
                    raise ValueError(f"rows must be a contiguous vector of {tokens}")
                a.rows = rows.data_ptr()
                a.kv_heads = heads = (k if k is not None else v).shape[1]
                cache = k_cache if k is not None else v_cache
                if cache is None:
                    raise ValueError("keys and values need their caches")
                shape, strides = cache.shape, cache.stride()
                for t, c, name in ((k, k_cache, "k"), (v, v_cache, "v")):
                    if t is None:
                        continue
                    if c is None or c.dtype != dtype or c.device != self.device or c.shape != shape or \
                            c.stride() != strides:
                        raise ValueError(f"{name}_cache must be {tuple(shape)} {dtype}, K and V laid out alike")
                if len(shape) != 4 or strides[3] != 1 or shape[1] != heads or shape[3] != dim:
                    raise ValueError(f"the caches must be [pages, {heads}, page_tokens, {dim}] with contiguous head "
                                     "vectors")
                if k is not None:
                    a.k, a.k_token_stride, a.k_head_stride = self._heads(k, tokens, heads, dim, dtype, "k")
                    a.k_cache = k_cache.data_ptr()
                if v is not None:
                    a.v, a.v_token_stride, a.v_head_stride = self._heads(v, tokens, heads, dim, dtype, "v")
                    a.v_cache = v_cache.data_ptr()
                a.page_stride, a.head_stride, a.row_stride, _ = strides
                a.page_tokens, a.n_rows = shape[2], shape[0] * shape[2]
            self.layout = layout
            return self._launch(q_out)

    def _launch(self, q_out: Optional[torch.Tensor]):
        rc = self.lib.q4gpu_rope_append(self.args, self._here())
        if rc:
            _native.check(rc, "q4gpu_rope_append")
        return q_out

    def _heads(self, t: torch.Tensor, tokens: int, heads: int, dim: int, dtype: torch.dtype, name: str):
        if t.device != self.device or t.dtype != dtype:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {dtype} on {self.device}")
        ts, hs, ds = t.stride()
        if t.shape != (tokens, heads, dim) or ds != 1:
            raise ValueError(f"{name} must be [{tokens}, {heads}, {dim}] with contiguous head vectors")
        return t.data_ptr(), ts, hs


class Attention(_Err):
    """Attention of each sequence's newest tokens to its pages.

    ``k_cache`` / ``v_cache`` [pages, kv_heads, page_tokens, dim] (bf16 or f16, K and
    V laid out alike), ``table`` int32 [slots, pages per slot], ``lens`` int32 [slots]:
    the keys a slot holds, the new ones included.  ``scale`` defaults to
    dim ** -0.5; with ``window`` a query sees the last ``window`` keys up to its own, and
    the first ``sinks`` keys of its sequence up to its own (pages that hold neither are
    not read).  ``share``: another of them (a layer before, say) whose workspace this one
    uses as well; their calls then follow one another like those of one object.
    """

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                 q_heads: int, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                 share: Optional["Attention"] = None):
        self.lib = _native.load()
        self.device = _cuda(k_cache, "k_cache")
        self.dtype = k_cache.dtype
        _need(self.dtype in (torch.float16, torch.bfloat16), f"the cache is {self.dtype}")
        _on(v_cache, self.device, "v_cache", self.dtype)
        _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride() and
              k_cache.stride(3) == 1, "k_cache and v_cache must be [pages, kv_heads, page_tokens, dim], laid out alike")
        _on(table, self.device, "table", torch.int32)
        _on(lens, self.device, "lens", torch.int32)
        _need(table.dim() == 2 and table.stride(1) == 1 and lens.dim() == 1 and lens.is_contiguous() and
              lens.shape[0] == table.shape[0], "table must be [slots, pages] and lens [slots]")
        pages, kv_heads, page_tokens, dim = k_cache.shape
        _need(0 <= sinks < 2 ** 31, f"{sinks} sinks")
        _need(window > 0 or sinks == 0, "sinks need a window")
        self.q_heads, self.dim, self.slots, self.sinks = q_heads, dim, table.shape[0], sinks
        self.k_cache, self.v_cache, self.table, self.lens = k_cache, v_cache, table, lens
        _need(share is None or share.device == self.device, "a workspace is shared on one device")
        self.workspace = self.layout = None
        # workspaces, the newest last.  The old ones stay: captured graphs know their addresses (each is at least twice
        # the last, so all together are less than two of the newest)
        self.room: list[torch.Tensor] = [] if share is None else share.room
        self.lock = threading.Lock() if share is None else share.lock
        self._new_err()
        self.args = _native.AttnArgs(
            k_cache=k_cache.data_ptr(), v_cache=v_cache.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr(),
            page_stride=k_cache.stride(0), head_stride=k_cache.stride(1), row_stride=k_cache.stride(2),
            table_stride=table.stride(0) if self.slots > 1 else table.shape[1], table_pages=table.shape[1],
            n_slots=self.slots, q_heads=q_heads,
            kv_heads=kv_heads, dim=dim, page_tokens=page_tokens, n_pages=pages, window=window,
            dtype=_DTYPES[self.dtype], scale=dim ** -0.5 if scale is None else scale,
            err_flag=self.err.data_ptr())

    def __call__(self, q: torch.Tensor, out: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None,
                 max_q: int = 1, max_ctx: int = 0, lse: Optional[torch.Tensor] = None,
                 seq_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """q [tokens, q_heads, dim]; cu_q int32 [sequences + 1]: sequence i has the query
        tokens cu_q[i] .. cu_q[i + 1] - 1, at most max_q; seq_ids int32 [sequences]: their
        slots (default: 0, 1, ..); max_ctx: no lens is larger (0: the table's width).  A
        sequence with more than max_q tokens is an error that `check` reports.
        lse (optional) float32 [tokens, q_heads] receives log sum exp of the scores."""
        with self.lock:
            a = self.args
            if cu_q is None:
                raise ValueError("cu_q is needed")
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
            # what the checks below look at: tensors laid out like the last call's need only their addresses
            layout = (q.shape, q.stride(), q.dtype, q.device, out.shape, out.stride(), out.dtype, out.device,
                      cu_q.shape, cu_q.stride(), cu_q.dtype, cu_q.device, max_q, max_ctx,
                      None if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.device),
                      None if seq_ids is None else (seq_ids.shape, seq_ids.stride(), seq_ids.dtype, seq_ids.device))
            if layout == self.layout:
                a.q, a.out, a.cu_q = q.data_ptr(), out.data_ptr(), cu_q.data_ptr()
                if lse is not None:
                    a.lse = lse.data_ptr()
                if seq_ids is not None:
                    a.seq_ids = seq_ids.data_ptr()
                return self._launch(out)
            self.layout = None
            self._bind(q, out, cu_q, max_q, max_ctx, lse, seq_ids)
            return self._run(out, layout)

    def _bind(self, q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, max_q: int, max_ctx: int,
              lse: Optional[torch.Tensor], seq_ids: Optional[torch.Tensor]) -> None:
        """Checks a call's tensors and puts them into the arguments."""
        a, tokens = self.args, q.shape[0]
        a.q, a.q_token_stride, a.q_head_stride = self._heads(q, tokens, "q")
        a.out, a.out_token_stride, a.out_head_stride = self._heads(out, tokens, "out")
        a.cu_q, n = self._ends(cu_q, "cu_q")
        a.n_seqs, a.tokens, a.max_q = n, tokens, max_q
        a.max_ctx = max_ctx or min(a.table_pages * a.page_tokens, 2 ** 31 - 1)
        a.seq_ids = a.lse = None
        if seq_ids is not None:
            _on(seq_ids, self.device, "seq_ids", torch.int32)
            _need(seq_ids.shape == (n,) and seq_ids.is_contiguous(), f"seq_ids must be [{n}]")
            a.seq_ids = seq_ids.data_ptr()
        elif n > self.slots:
            raise ValueError(f"{n} sequences over {self.slots} slots")
        if lse is not None:
            _on(lse, self.device, "lse", torch.float32)
            if lse.shape != (tokens, self.q_heads) or not lse.is_contiguous():
                raise ValueError(f"lse must be contiguous [{tokens}, {self.q_heads}]")
            a.lse = lse.data_ptr()

    def _ends(self, cu: torch.Tensor, name: str) -> tuple[int, int]:
        if cu.dtype != torch.int32 or cu.device != self.device or cu.dim() != 1 or cu.shape[0] < 1 or \
                not cu.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector on {self.device}")
        return cu.data_ptr(), cu.shape[0] - 1

    def _run(self, out: torch.Tensor, layout: tuple) -> torch.Tensor:
        """Launches the checked call, with enough workspace; later calls of this layout need no checks."""
        a = self.args
        need = self._workspace_bytes(a)
        if need > a.workspace_bytes:
            if not self.room or self.room[-1].numel() < need:
                if torch.cuda.is_current_stream_capturing():
                    return self._launch_captured(out, need)
                held = self.room[-1].numel() if self.room else 0
                self.room.append(torch.zeros(max(need, 2 * held), dtype=torch.uint8, device=self.device))
            else:  # made by a call of another operator, on whatever stream
                self.room[-1].record_stream(torch.cuda.current_stream(self.device))
            self.workspace = self.room[-1]
            self.own.append(self.workspace)
            a.workspace, a.workspace_bytes = self.workspace.data_ptr(), self.workspace.numel()
        self.layout = layout
        return self._launch(out)

    def _launch_captured(self, out: torch.Tensor, need: int) -> torch.Tensor:
        """A captured call that wants more workspace than there is: what is allocated now is zeroed by the graph's
        replays only, so it serves this call and no other."""
        a, once = self.args, torch.zeros(need, dtype=torch.uint8, device=self.device)
        kept = a.workspace, a.workspace_bytes
        a.workspace, a.workspace_bytes = once.data_ptr(), need
        try:
            return self._launch(out)
        finally:
            a.workspace, a.workspace_bytes = kept

    def _launch(self, out: torch.Tensor) -> torch.Tensor:
        if self.sinks:
            rc = self.lib.q4gpu_sink_attention(self.args, self.sinks, self._here())
        else:
            rc = self.lib.q4gpu_paged_attention(self.args, self._here())
        if rc:
            _native.check(rc, "q4gpu_sink_attention" if self.sinks else "q4gpu_paged_attention")
        return out

    def _workspace_bytes(self, a: _native.AttnArgs) -> int:
        if self.sinks:
            return self.lib.q4gpu_sink_attention_workspace_bytes(a, self.sinks)
        return self.lib.q4gpu_paged_attention_workspace_bytes(a)

    def _heads(self, t: torch.Tensor, tokens: int, name: str):
        if t.device != self.device or t.dtype != self.dtype:
            raise ValueError(f"{name} is {t.dtype} on {t.device}, expected {self.dtype} on {self.device}")
        if t.shape != (tokens, self.q_heads, self.dim) or t.stride(2) != 1:
            raise ValueError(f"{name} must be [{tokens}, {self.q_heads}, {self.dim}] with contiguous head vectors")
        return t.data_ptr(), t.stride(0), t.stride(1)


class SharedAttention(Attention):
    """``Attention`` of sequences that share their first keys: those are read once for all of a group.

    Group g is the sequences cu_group[g] .. cu_group[g + 1] - 1 of a call and shares its
    first prefix_lens[g] keys, which are read from the pages of the group's first
    sequence.  Every query stands behind them.
    """

    def __init__(self, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                 q_heads: int, scale: Optional[float] = None, share: Optional[Attention] = None):
        super().__init__(k_cache, v_cache, table, lens, q_heads, scale, share=share)
        self.groups = _native.SharedArgs()

    def __call__(self, q: torch.Tensor, out: Optional[torch.Tensor] = None, cu_q: Optional[torch.Tensor] = None,
                 cu_group: Optional[torch.Tensor] = None, prefix_lens: Optional[torch.Tensor] = None, max_q: int = 1,
                 max_ctx: int = 0, max_prefix: int = 0, lse: Optional[torch.Tensor] = None,
                 seq_ids: Optional[torch.Tensor] = None) -> torch.Tensor:
        """As ``Attention``, with cu_group int32 [groups + 1] and prefix_lens int32 [groups]; sequences in no
        group share nothing; max_prefix: no prefix is longer (0: max_ctx).  A sequence whose queries do not
        stand behind the shared keys is an error that `check` reports, and so are offsets that do not ascend."""
        with self.lock:
            a, g = self.args, self.groups
            if cu_q is None or cu_group is None or prefix_lens is None:
                raise ValueError("cu_q, cu_group and prefix_lens are needed")
            if out is None:
                out = torch.empty_like(q, memory_format=torch.contiguous_format)
            # what the checks below look at: tensors laid out like the last call's need only their addresses
            layout = (q.shape, q.stride(), q.dtype, q.device, out.shape, out.stride(), out.dtype, out.device,
                      cu_q.shape, cu_q.stride(), cu_q.dtype, cu_q.device, max_q, max_ctx, max_prefix,
                      cu_group.shape, cu_group.stride(), cu_group.dtype, cu_group.device,
                      prefix_lens.shape, prefix_lens.stride(), prefix_lens.dtype, prefix_lens.device,
                      None if lse is None else (lse.shape, lse.stride(), lse.dtype, lse.device),
                      None if seq_ids is None else (seq_ids.shape, seq_ids.stride(), seq_ids.dtype, seq_ids.device))
            if layout == self.layout:
                a.q, a.out, a.cu_q = q.data_ptr(), out.data_ptr(), cu_q.data_ptr()
                g.cu_group, g.prefix_lens = cu_group.data_ptr(), prefix_lens.data_ptr()
                if lse is not None:
                    a.lse = lse.data_ptr()
                if seq_ids is not None:
                    a.seq_ids = seq_ids.data_ptr()
                return self._launch(out)
            self.layout = None
            self._bind(q, out, cu_q, max_q, max_ctx, lse, seq_ids)
            g.cu_group, g.n_groups = self._ends(cu_group, "cu_group")
            _on(prefix_lens, self.device, "prefix_lens", torch.int32)
            _need(prefix_lens.shape == (g.n_groups,) and prefix_lens.is_contiguous(),
                  f"prefix_lens must be [{g.n_groups}]")
            g.prefix_lens, g.max_prefix = prefix_lens.data_ptr(), max_prefix or a.max_ctx
            return self._run(out, layout)

    def _workspace_bytes(self, a: _native.AttnArgs) -> int:
        return self.lib.q4gpu_shared_attention_workspace_bytes(a, self.groups)

    def _launch(self, out: torch.Tensor) -> torch.Tensor:
        rc = self.lib.q4gpu_shared_attention(self.args, self.groups, self._here())
        if rc:
            _native.check(rc, "q4gpu_shared_attention")
        return out


class TokenScores:
    """What ``TokenLogprobs`` gives for each row, as contiguous device tensors.

    ``logprob`` / ``entropy`` float32 [rows], ``rank`` int32 [rows], ``top_logprob`` float32 and
    ``top_index`` int32 [rows, top].  Made by ``TokenLogprobs.empty``.
    """

    __slots__ = ("logprob", "entropy", "rank", "top_logprob", "top_index", "_made", "_room", "_at")

    def __init__(self, rows: int, top: int, device: torch.device):
        def room(dtype, *shape):
            return torch.empty(*shape, dtype=dtype, device=device)
        self.logprob, self.entropy = room(torch.float32, rows), room(torch.float32, rows)
        self.rank = room(torch.int32, rows)
        self.top_logprob, self.top_index = room(torch.float32, rows, top), room(torch.int32, rows, top)
        self._made = rows, top, device
        # (kept, so that the addresses hold whatever becomes of the names above)
        self._room = self.logprob, self.entropy, self.rank, self.top_logprob, self.top_index
        self._at = tuple(t.data_ptr() for t in self._room)


class TokenLogprobs(_Err):
    """Log probabilities of given tokens, the entropy and the ``top`` likeliest tokens of rows of logits.

    logprob = log softmax(x)[t]; rank: 1 + the tokens before t by falling logit (equal ones by
    rising index), the order of top_logprob / top_index; entropy in nats.
    """

    MOST = 32  # of the likeliest tokens

    def __init__(self, top: int = 0, device: Optional[torch.device] = None):
        self.lib = _native.load()
        _need(0 <= top <= self.MOST, f"top = {top}, at most {self.MOST}")
        self.device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        _need(self.device.type == "cuda" and self.device.index is not None, f"{self.device} is not a CUDA device")
        self.top, self.layout, self.lock = top, None, threading.Lock()
        self._new_err()
        self.args = _native.LogprobArgs(top=top, err_flag=self.err.data_ptr())

    def empty(self, rows: int) -> TokenScores:
        """Room for the results of ``rows`` rows."""
        return TokenScores(rows, self.top, self.device)

    def __call__(self, logits: torch.Tensor, targets: Optional[torch.Tensor] = None,
                 out: Optional[TokenScores] = None) -> TokenScores:
        """logits [rows, vocab] float32, float16 or bfloat16 with contiguous rows; targets int64 [rows],
        negative: no token (logprob 0, rank 0; without targets they are not written).  A target past the
        vocabulary counts as none and is an error that ``check`` reports."""
        with self.lock:
            a = self.args
            layout = (logits.shape, logits.stride(), logits.dtype, logits.device,
                      None if targets is None else (targets.shape, targets.stride(), targets.dtype, targets.device))
            if layout != self.layout:
                self.layout = None
                if logits.dim() != 2 or logits.device != self.device or \
                        logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                    raise ValueError(f"logits must be [rows, vocab] float32, float16 or bfloat16 on {self.device}")
                rows, vocab = logits.shape
                _need(vocab > 0 and (logits.stride(1) == 1 or vocab == 1), "logits must have contiguous rows")
                _need(vocab < 2 ** 31, f"a vocabulary of {vocab}")
                if targets is not None:
                    _on(targets, self.device, "targets", torch.int64)
                    _need(targets.shape == (rows,) and targets.is_contiguous(),
                          f"targets must be a contiguous vector of {rows}")
                a.rows, a.vocab, a.stride, a.dtype = rows, vocab, logits.stride(0), _DTYPES[logits.dtype]
                self.layout = layout
            if out is None:
                out = TokenScores(a.rows, self.top, self.device)
            elif out._made != (a.rows, self.top, self.device):
                raise ValueError(f"out must be what empty({a.rows}) of this operator makes")
            a.logits, a.targets = logits.data_ptr(), None if targets is None else targets.data_ptr()
            a.logprob, a.entropy, a.rank, a.top_logprob, a.top_index = out._at
            rc = self.lib.q4gpu_token_logprobs(a, self._here())
            if rc:
                _native.check(rc, "q4gpu_token_logprobs")
            return out


class Pages(_Err):
    """A pool of pages [pages, ..blocks.., page_tokens, dim] and the tables that name them.

    ``table`` int32 [slots, pages per slot], ``lens`` int32 [slots]; slot s holds lens[s]
    tokens in the pages of its first ceil(lens[s] / page_tokens) entries.
    """

    def __init__(self, pool: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, page_tokens: int):
        self.lib = _native.load()
        self.device = _cuda(pool, "pool")
        _need(pool.dim() >= 3 and pool.is_contiguous() and pool.shape[-2] == page_tokens,
              "pool must be contiguous [pages, .., page_tokens, dim]")
        _on(table, self.device, "table", torch.int32)
        _on(lens, self.device, "lens", torch.int32)
        _need(table.dim() == 2 and table.is_contiguous() and lens.is_contiguous() and
              lens.shape == (table.shape[0],), "table must be contiguous [slots, pages] and lens [slots]")
        self.pool, self.table, self.lens = pool, table, lens
        self._new_err()
        es = pool.element_size()
        self.args = _native.PagesArgs(pool=pool.data_ptr(), table=table.data_ptr(), lens=lens.data_ptr(),
                                      err_flag=self.err.data_ptr(), page_bytes=pool.stride(0) * es,
                                      block_bytes=page_tokens * pool.shape[-1] * es, table_stride=table.shape[1],
                                      n_pages=pool.shape[0], page_tokens=page_tokens, n_slots=table.shape[0])
        self.workspace = torch.empty(self.lib.q4gpu_pages_compact_workspace_bytes(pool.shape[0]), dtype=torch.uint8,
                                     device=self.device)
        self.own.append(self.workspace)

    def _ids(self, t: torch.Tensor, n: int, name: str) -> int:
        if t.dtype != torch.int32 or t.device != self.device or t.shape != (n,) or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous int32 vector of {n} on {self.device}")
        return t.data_ptr()

    def fork(self, parents: torch.Tensor, children: torch.Tensor, fresh: torch.Tensor) -> None:
        """Slot children[i] gets the pages of slot parents[i]; a partly filled last page is
        copied (its filled rows) to page fresh[i].  int32 [n] each."""
        n = parents.shape[0]
        rc = self.lib.q4gpu_pages_fork(self.args, self._ids(parents, n, "parents"), self._ids(children, n, "children"),
                                       self._ids(fresh, n, "fresh"), n, self._here())
        if rc:
            _native.check(rc, "q4gpu_pages_fork")

    def compact(self, new_table: torch.Tensor, remap: torch.Tensor, n_live: torch.Tensor) -> None:
        """Moves the pages in use into the first n_live pages.  new_table (may be the table
        itself) int32 [slots, pages per slot], remap int32 [pages] (old -> new, -1 unused),
        n_live int32 [1]."""
        _on(new_table, self.device, "new_table", torch.int32)
        if new_table.shape != self.table.shape or not new_table.is_contiguous():
            raise ValueError(f"new_table must be contiguous {tuple(self.table.shape)}")
        rc = self.lib.q4gpu_pages_compact(self.args, new_table.data_ptr(), self._ids(remap, self.args.n_pages, "remap"),
                                          self._ids(n_live, 1, "n_live"), self.workspace.data_ptr(),
                                          self.workspace.numel(), self._here())
        if rc:
            _native.check(rc, "q4gpu_pages_compact")


@dataclass
class Step:
    """One step's new tokens over a ``PagedCache``, as the operators take them (device tensors)."""
    seq_ids: torch.Tensor    # int32 [sequences]
    cu_q: torch.Tensor       # int32 [sequences + 1]
    positions: torch.Tensor  # int32 [tokens]
    rows: torch.Tensor       # int64 [tokens]
    max_q: int
    max_ctx: int
    # where groups of neighbouring sequences share enough of their first keys, what SharedAttention takes
    cu_group: Optional[torch.Tensor] = None     # int32 [groups + 1]
    prefix_lens: Optional[torch.Tensor] = None  # int32 [groups]
    max_prefix: int = 0


def shared_runs(held: Sequence[Sequence[int]], users: Sequence[int]) -> list[tuple[int, int]]:
    """(sequences, first pages that they share) of each run of neighbours in `held`, their pages in order.

    ``users[p]``: how many sequences hold page p.  A run goes on as long as the first page is the same.
    """
    runs: list[tuple[int, int]] = []
    first: Sequence[int] = ()
    for pages in held:
        if runs and first and pages and pages[0] == first[0]:
            n = runs[-1][1]
            if pages[:n] != first[:n]:
                n = next((i for i, (a, b) in enumerate(zip(pages, first)) if a != b), min(len(pages), len(first)))
            runs[-1] = runs[-1][0] + 1, n
            continue
        first = pages
        n = next((i for i, p in enumerate(pages) if users[p] < 2), len(pages))
        runs.append((1, n))
    return [(n, pages if n > 1 else 0) for n, pages in runs]


class PagedCache:
    """16-bit K/V pages of all layers for up to ``max_seqs`` sequences.

    The pool is [pages, layers, K/V, kv_heads, page_tokens, head_dim]: a page holds
    page_tokens positions of every layer, so a fork copies one run of memory.  Which
    pages are free and whose they are is kept on the host; ``table`` and ``lens`` are the
    device's view, updated in stream order.  Full pages can belong to several sequences
    and are never written again; a partly filled last page belongs to one.
    """

    # Whether a step's neighbouring forks attend together (us a layer of 16 heads on 8 of 128, then of 28 on 4 of 64, one
    # new token each, alone and together).  A few sequences do from SHARED_KEYS on: alone their keys are cut into many
    # pieces (2 forks of 256 keys 9.3 and 10.3, 8.2 and 10.0; of 1024 15.0 and 11.8, 13.6 and 10.6; 8 of 1024 16.5 and 15.5, 13.9
    # and 13.5; 12 of 1024 18.5 and 17.0, 14.4 and 19.1).  Otherwise they do where enough is not read again: SAVED_KEYS
    # of 8 heads of 128, of smaller ones more by the square of a key's values, as those are read in less time but joined in
    # the same (16 of 256 10.0 and 15.4; 32 of 256 20.3 and 15.9; 64 of 256 27.1 and 18.4, 10.3 and 21.1; 64 of 1024 50.5 and
    # 21.6, 22.1 and 25.3; 64 of 8192 261 and 31, 80 and 35), and more by the new tokens of a sequence (16 of 512 keys
    # 17.9 and 16.5 with one, 18.5 and 22.1 with 4; 32 of 1024 33.4 and 27.8 with 4).
    SHARED_KEYS, SAVED_KEYS = 1024, 7500
    FEW = 8, 4  # sequences, new tokens of each
    # New tokens of a sequence up to which it can pay: longer chunks fill tiles by themselves, so that sharing
    # saves no time and joining costs some (alone against together, 16 of 8192 keys: 112 and 59 us with 16 tokens, 113 and
    # 173 with 64; 64 of 1024: 94 and 71 with 16, 94 and 142 with 32, 243 and 750 with 256).
    NEW_TOKENS = 16

    def __init__(self, n_layers: int, n_pages: int, page_tokens: int, kv_heads: int, head_dim: int, max_seqs: int,
                 max_ctx: int, dtype: torch.dtype = torch.bfloat16, device: Optional[torch.device] = None):
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        self.page_tokens, self.max_ctx, self.device = page_tokens, max_ctx, dev
        self.pool = torch.empty(n_pages, n_layers, 2, kv_heads, page_tokens, head_dim, dtype=dtype, device=dev)
        self.table = torch.full((max_seqs, -(-max_ctx // page_tokens)), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(max_seqs, dtype=torch.int32, device=dev)
        self.pages = Pages(self.pool, self.table, self.lens, page_tokens)
        self._held: list[list[int]] = [[] for _ in range(max_seqs)]
        self._len = [0] * max_seqs
        self._users = [0] * n_pages
        self._free = list(range(n_pages))  # a heap: the lowest free page is taken first

    def k(self, layer: int) -> torch.Tensor:
        return self.pool[:, layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.pool[:, layer, 1]

    def _known(self, seqs: Sequence[int]) -> None:
        for s in seqs:  # a negative number would mean another sequence on the host and none on the device
            if not 0 <= s < len(self._len):
                raise ValueError(f"sequence {s} is not one of {len(self._len)}")

    def length(self, seq: int) -> int:
        self._known((seq,))
        return self._len[seq]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise RuntimeError(f"the cache is full: {n} pages wanted, {len(self._free)} free")
        got = [heapq.heappop(self._free) for _ in range(n)]
        for p in got:
            self._users[p] += 1
        return got

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            self._users[p] -= 1
            if self._users[p] == 0:
                heapq.heappush(self._free, p)

    def _up(self, a: np.ndarray) -> torch.Tensor:
        return torch.from_numpy(a).pin_memory().to(self.device, non_blocking=True)

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> Step:
        """Room for counts[i] new tokens of sequence seqs[i]; returns the step's index tensors.
        Nothing changes if the pages do not suffice."""
        _need(len(seqs) == len(counts) and len(set(seqs)) == len(seqs) and len(seqs) > 0, "one count per sequence")
        self._known(seqs)
        need = []
        for s, n in zip(seqs, counts):
            if n < 0 or self._len[s] + n > self.max_ctx:
                raise ValueError(f"sequence {s}: {self._len[s]} + {n} tokens, at most {self.max_ctx}")
            need.append(-(-(self._len[s] + n) // self.page_tokens) - len(self._held[s]))
        got = self._take(sum(need))
        pos, rows = [], []
        table = np.full((len(seqs), self.table.shape[1]), -1, dtype=np.int32)
        for i, (s, n) in enumerate(zip(seqs, counts)):
            self._held[s] += got[:need[i]]
            got = got[need[i]:]
            held = np.asarray(self._held[s], dtype=np.int64)
            table[i, :held.size] = held
            p = np.arange(self._len[s], self._len[s] + n, dtype=np.int64)
            pos.append(p)
            rows.append(held[p // self.page_tokens] * self.page_tokens + p % self.page_tokens if n else p)
            self._len[s] += n
        runs = shared_runs([self._held[s] for s in seqs], self._users) if len(seqs) > 1 else []
        prefix = self._together(runs, counts)
        groups = {}
        if prefix:
            ends = np.cumsum([0] + [n for n, _ in runs])
            groups = dict(cu_group=self._up(ends.astype(np.int32)), max_prefix=prefix,
                          prefix_lens=self._up(np.asarray([p * self.page_tokens for _, p in runs], dtype=np.int32)))
        ids = self._up(np.asarray(seqs, dtype=np.int32))
        at = ids.long()
        self.table.index_copy_(0, at, self._up(table))
        lens = [self._len[s] for s in seqs]
        self.lens.index_copy_(0, at, self._up(np.asarray(lens, dtype=np.int32)))
        return Step(ids, self._up(np.concatenate(([0], np.cumsum(counts))).astype(np.int32)),
                    self._up(np.concatenate(pos).astype(np.int32)), self._up(np.concatenate(rows)), max(counts),
                    max(max(lens), 1), **groups)

    def _together(self, runs: Sequence[tuple[int, int]], counts: Sequence[int]) -> int:
        """The most keys that a run of a step shares, if its runs are worth attending to together, else 0."""
        new = max(1, *counts)
        if new > self.NEW_TOKENS:
            return 0
        prefix = max((p for _, p in runs), default=0) * self.page_tokens
        saved = sum((n - 1) * p for n, p in runs) * self.page_tokens
        values = self.pool.shape[3] * self.pool.shape[5]  # of a key
        few = len(counts) <= self.FEW[0] and new <= self.FEW[1]
        enough = saved * values ** 2 >= self.SAVED_KEYS * new * 1024 ** 2
        return prefix if few and prefix >= self.SHARED_KEYS or enough else 0

    def fork(self, parent: int, children: Sequence[int]) -> None:
        """Empty sequences `children` continue `parent`: full pages are shared, its last one copied."""
        self._known((parent, *children))
        _need(all(self._len[c] == 0 and c != parent for c in children) and len(set(children)) == len(children),
              "children must be empty sequences")
        n, held = self._len[parent], self._held[parent]
        full = n // self.page_tokens
        part = bool(n % self.page_tokens)
        fresh = self._take(len(children) if part else 0)
        for i, c in enumerate(children):
            for p in held[:full]:
                self._users[p] += 1
            self._held[c] = held[:full] + ([fresh[i]] if part else [])
            self._len[c] = n
        if children:
            self.pages.fork(self._up(np.full(len(children), parent, dtype=np.int32)),
                            self._up(np.asarray(children, dtype=np.int32)),
                            self._up(np.asarray(fresh or [-1] * len(children), dtype=np.int32)))

    def free(self, seq: int) -> None:
        """Ends a sequence; pages that nobody else uses become free."""
        self._known((seq,))
        self._drop(self._held[seq])
        self._held[seq], self._len[seq] = [], 0
        self.lens[seq:seq + 1].zero_()
        self.table[seq].fill_(-1)

    def compact(self) -> int:
        """Packs the pages in use into the first ones and returns their number (waits for the stream)."""
        remap = torch.empty(self.pool.shape[0], dtype=torch.int32, device=self.device)
        n_live = torch.empty(1, dtype=torch.int32, device=self.device)
        self.pages.compact(self.table, remap, n_live)
        to, live = remap.tolist(), int(n_live.item())
        self._held = [[to[p] for p in held] for held in self._held]
        users = [0] * len(to)
        for p, n in enumerate(self._users):
            if n:
                users[to[p]] = n
        self._users = users
        self._free = [p for p, n in enumerate(users) if n == 0]
        return live
