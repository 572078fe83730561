"""Host-built tables of the fixed-point path: RoPE cos/sin in Q1.15, the
softmax exp LUT and the SwiGLU sigmoid LUT.

The RoPE table is built the way the reference builds it: HF's default
inverse frequencies (float32), ``freqs = inv_freq @ positions`` and
``cos/sin`` in float32 torch (``Qwen3-0.6B-Base/python_each_module/common.py:155-170``),
then ``rint(x * 2^15)`` clipped to signed 16 bit
(``22_export_qk_norm_rope_fixed_vectors.py:75-83`` as called at
``56_export_persistent_multitoken_layer_golden.py:942-956``).  The device
never evaluates trigonometry; both LUTs come from the library's host
builder (``q4gpu_build_tables``).
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import torch

from . import _native

ROPE_THETA = 1.0e6
HEAD_DIM = 128


def rope_inv_freq(theta: float = ROPE_THETA, dim: int = HEAD_DIM) -> torch.Tensor:
    """HF Qwen3 default-RoPE inverse frequencies (float32)."""
    return 1.0 / (theta ** (torch.arange(0, dim, 2, dtype=torch.int64).to(dtype=torch.float) / dim))


def rope_tables(n_positions: int, theta: float = ROPE_THETA) -> tuple[np.ndarray, np.ndarray]:
    """int32 [n_positions, 128] cos and sin in Q1.15."""
    inv = rope_inv_freq(theta)
    pos = torch.arange(n_positions, dtype=torch.long).float()
    # the reference forms freqs with a k=1 float32 matmul (one rounding per
    # product); an elementwise float32 product is that same rounding without
    # depending on which BLAS path the matmul takes
    freqs = pos[:, None] * inv[None, :]
    emb = torch.cat((freqs, freqs), dim=-1)

    def q115(t: torch.Tensor) -> np.ndarray:
        v = np.rint(t.numpy().astype(np.float64) * 32768.0)
        return np.clip(v, -32768, 32767).astype(np.int32)

    return q115(emb.cos()), q115(emb.sin())


def rope_float_tables(n_positions: int, rot_dim: int = HEAD_DIM, theta: float = ROPE_THETA, factor: float = 1.0,
                      original: int | None = None, device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """float32 [n_positions, rot_dim / 2] cos and sin for ``paged.RopeAppend``, from float64 angles.

    With ``factor`` above 1 the frequencies are stretched by parts (YaRN): pair i turns
    ``original * inv_freq_i / 2 pi`` times over the ``original`` (trained) positions, by default
    n_positions / factor; pairs that turn more than 32 times keep their frequency, those below
    one turn are slowed by ``factor``, in between the two are mixed in proportion, and both
    tables are scaled by 0.1 ln(factor) + 1.  That is the published formula, a mix in proportion to
    the number of turns; a checkpoint that was stretched by a mix in proportion to the pair's index
    between the two limits has other frequencies in between (16 of 64, by up to 42 %, for 128
    values, theta 1e6, 32768 trained positions, factor 4) and needs tables of its own, which ``paged.RopeAppend`` takes as
    they are.  (The reference has 256 positions and no scaling.)
    """
    if rot_dim < 2 or rot_dim % 2 or n_positions < 1 or factor < 1.0:
        raise ValueError(f"no rotary table of {n_positions} positions x {rot_dim}, factor {factor}")
    inv = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    scale = 1.0
    if factor > 1.0:
        turns = (original or n_positions / factor) * inv / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        inv = inv * (keep + (1.0 - keep) / factor)
        scale = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(n_positions, dtype=torch.float64, device=device)[:, None] * inv
    return (angle.cos() * scale).float(), (angle.sin() * scale).float()


def luts() -> tuple[np.ndarray, np.ndarray]:
    """(exp LUT int32[257], sigmoid LUT int32[1025])."""
    e = np.zeros(257, dtype=np.int32)
    s = np.zeros(1025, dtype=np.int32)
    _native.load().q4gpu_build_tables(e.ctypes.data_as(C.c_void_p), s.ctypes.data_as(C.c_void_p))
    return e, s
