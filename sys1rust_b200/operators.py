"""Token-step operators of ``libs1c.so`` on device pointers: what a host needs beside the encoder to
generate an answer token by token.

* ``nibble_gemm``: a few rows times 4-bit weights with group scales; ``nibble_pack`` makes the codes.
* ``Cache``, ``cache_write``, ``cache_read``: a paged cache of keys and values in 8 bits, a scale for each
  page and head.
* ``cache_attention``: causal attention of new rows over that cache.
* ``sample``: one token for each row of logits under temperature, top-k, top-p and min-p.

As with ``backend.gemm`` and ``backend.attention``, arguments are raw device pointers (``tensor.data_ptr()``) and
element strides, 0 standing for an absent tensor; a call enqueues its work on ``stream`` (a raw
``cudaStream_t``) and raises ``BackendError`` for arguments the library refuses. ``include/s1c.h`` has
each operator's definition.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from .backend import DT_BF16, DT_F16, DT_F32, S1C_OK, BackendError, CCache, S1C_ERR_ARG, _raise, lib

__all__ = ["Cache", "cache_attention", "cache_attention_workspace", "cache_read", "cache_write", "nibble_gemm", "nibble_pack",
           "sample", "DT_BF16", "DT_F16", "DT_F32"]


def _done(rc: int) -> None:
    if rc != S1C_OK:
        _raise(rc, lib().s1c_create_error().decode())


def nibble_pack(w: np.ndarray, group: int, scale_dtype=np.float32):
    """4-bit codes and group scales of a matrix ``[N, K]``, on the host: ``scale = max |w| / 7`` of each
    group of columns (rounded to ``scale_dtype``), ``code = round(w / scale) + 8`` in 1..15. Returns
    ``(codes [N, pitch] uint8, scales [N, ceil(K / group)])``; columns past K hold code 8 (zero)."""
    w = np.ascontiguousarray(w, dtype=np.float32)
    if w.ndim != 2 or group not in (32, 64, 128) or not np.isfinite(w).all():
        raise BackendError(S1C_ERR_ARG, "nibble_pack takes a finite matrix [N, K] and a group of 32, 64 or 128")
    N, K = w.shape
    groups = -(-K // group)
    padded = np.zeros((N, groups * group), dtype=np.float32)
    padded[:, :K] = w
    parts = padded.reshape(N, groups, group)
    with np.errstate(over="ignore"):
        scales = (np.abs(parts).max(2) / 7).astype(scale_dtype)
    if not np.isfinite(scales).all():
        raise BackendError(S1C_ERR_ARG, "nibble_pack: a group's scale does not fit scale_dtype")
    div = np.where(scales > 0, scales, 1).astype(np.float64)
    codes = np.clip(np.rint(parts / div[:, :, None]), -7, 7).astype(np.int8).reshape(N, -1) + 8
    pitch = -(-K // 32) * 16
    codes = codes.astype(np.uint8)[:, : 2 * pitch]
    return np.ascontiguousarray(codes[:, 0::2] | (codes[:, 1::2] << 4)), scales


def nibble_gemm(dtype: int, x_ptr: int, x_stride: int, codes_ptr: int, code_pitch: int, scales_ptr: int, scale_stride: int,
                out_ptr: int, out_stride: int, M: int, N: int, K: int, group: int, zeros_ptr: int = 0, bias_ptr: int = 0,
                act: int = 0, out_f32: bool = False, stream: int = 0) -> None:
    """``out[M, N] = act(x[M, K] W[N, K]^T + bias)``, W from 4-bit codes (``s1c_nibble_gemm``). ``dtype``
    (``DT_F16`` or ``DT_BF16``) is that of x, scales, zeros and, unless ``out_f32``, out."""
    _done(lib().s1c_nibble_gemm(dtype, x_ptr or None, x_stride, codes_ptr or None, code_pitch, scales_ptr or None,
                                zeros_ptr or None, scale_stride, group, out_ptr or None, out_stride, M, N, K,
                                bias_ptr or None, act, 1 if out_f32 else 0, stream or None))


class Cache(CCache):
    """A layer's paged 8-bit cache: int8 codes ``[num_pages, kv_heads, page, head_dim]`` of keys and values
    and their fp32 scales ``[num_pages, kv_heads]``. Holds the pointers only; the buffers are the caller's."""

    def __init__(self, k_codes_ptr: int, v_codes_ptr: int, k_scales_ptr: int, v_scales_ptr: int, num_pages: int, page: int,
                 kv_heads: int, head_dim: int):
        super().__init__(k_codes_ptr or None, v_codes_ptr or None, k_scales_ptr or None, v_scales_ptr or None, num_pages,
                         page, kv_heads, head_dim)


def cache_write(cache: Cache, dtype: int, k_ptr: int, k_stride: int, v_ptr: int, v_stride: int, cu_ptr: int, start_ptr: int,
                pages_ptr: int, max_pages: int, n: int, max_new: int, stream: int = 0) -> None:
    """Quantise and append new rows (``s1c_cache_write``): sequence i's rows ``cu[i] .. cu[i + 1]`` go to
    positions ``start[i] ..`` of the pages its table row names."""
    _done(lib().s1c_cache_write(C.byref(cache), dtype, k_ptr or None, k_stride, v_ptr or None, v_stride, cu_ptr or None,
                                start_ptr or None, pages_ptr or None, max_pages, n, max_new, stream or None))


def cache_read(cache: Cache, dtype: int, k_ptr: int, k_stride: int, v_ptr: int, v_stride: int, cu_ptr: int, start_ptr: int,
               pages_ptr: int, max_pages: int, n: int, max_rows: int, stream: int = 0) -> None:
    """Read rows back as 16-bit values (``s1c_cache_read``): positions ``start[i] ..`` of sequence i into
    rows ``cu[i] .. cu[i + 1]``."""
    _done(lib().s1c_cache_read(C.byref(cache), dtype, k_ptr or None, k_stride, v_ptr or None, v_stride, cu_ptr or None,
                               start_ptr or None, pages_ptr or None, max_pages, n, max_rows, stream or None))


def cache_attention_workspace(cache: Cache, heads: int, n: int, max_q: int, max_kv: int) -> int:
    """Bytes of device workspace that serve every ``cache_attention`` with bounds up to these."""
    return int(lib().s1c_cache_attention_workspace(C.byref(cache), heads, n, max_q, max_kv))


def cache_attention(cache: Cache, dtype: int, q_ptr: int, q_stride: int, out_ptr: int, out_stride: int, heads: int,
                    cu_ptr: int, len_ptr: int, pages_ptr: int, max_pages: int, n: int, max_q: int, max_kv: int, scale: float,
                    window: int = -1, lse_ptr: int = 0, workspace_ptr: int = 0, workspace_bytes: int = 0,
                    stream: int = 0) -> None:
    """Causal attention of new rows over the cache (``s1c_cache_attention``): sequence i's query rows
    ``cu[i] .. cu[i + 1]`` are the last of its ``len[i]`` cached positions."""
    _done(lib().s1c_cache_attention(C.byref(cache), dtype, q_ptr or None, q_stride, out_ptr or None, out_stride,
                                    lse_ptr or None, heads, cu_ptr or None, len_ptr or None, pages_ptr or None, max_pages, n,
                                    max_q, max_kv, window, scale, workspace_ptr or None, workspace_bytes, stream or None))


def sample(dtype: int, logits_ptr: int, row_stride: int, rows: int, vocab: int, token_ptr: int, uniform_ptr: int,
           temperature_ptr: int = 0, top_k_ptr: int = 0, top_p_ptr: int = 0, min_p_ptr: int = 0, prob_ptr: int = 0,
           stream: int = 0) -> None:
    """One token for each row of logits (``s1c_sample``), chosen by a given uniform number; ``dtype`` is
    ``DT_F32``, ``DT_F16`` or ``DT_BF16``."""
    _done(lib().s1c_sample(dtype, logits_ptr or None, row_stride, rows, vocab, temperature_ptr or None, top_k_ptr or None,
                           top_p_ptr or None, min_p_ptr or None, uniform_ptr or None, token_ptr or None, prob_ptr or None,
                           stream or None))
