"""Operators of a differential-attention block over boards and their history.

Torch CUDA tensors in and out (torch only allocates); every computation runs in
``libkatab200.so``:

=======================  ===================================================
:func:`rope_axes`        rotary positions with several axes (time, row, column)
:func:`diff_attention`   the difference of two softmax maps, prompts to single tokens
:func:`norm_residual`    the norms around a block with gate and residual scale
:func:`diff_lambda`      the maps' weights from their learned vectors (CPU)
=======================  ===================================================

Tensors may have any strides as long as the innermost dimension is contiguous
(:func:`diff_attention` needs multiples of 8 elements).  Work goes to the
current stream of the tensors' device, or to ``stream``; outputs and scratch
that a call allocates belong to that stream.  Wrong arguments raise
``ValueError`` / ``TypeError`` here or :class:`rust_katago_b200._capi.KbError`
from the library.  No reference counterparts: the reference's trunk has one
softmax map over 361 tokens.
"""

from __future__ import annotations

import contextlib
import ctypes

import numpy as np
import torch

from . import _capi
from ._capi import call
from .int8 import _ptr, _stream

_DTYPES = {torch.float32: _capi.DT_F32, torch.float16: _capi.DT_F16, torch.bfloat16: _capi.DT_BF16}
_LAYOUTS = {"pairs": _capi.ROPE_PAIRS, "halves": _capi.ROPE_HALVES}
_NORMS = {None: _capi.NORM_NONE, "rms": _capi.NORM_RMS, "layer": _capi.NORM_LAYER}
_GATES = {"linear": _capi.GATE_LINEAR, "sigmoid": _capi.GATE_SIGMOID, "tanh": _capi.GATE_TANH}


def _on(stream, device):
    """The context in which tensors are allocated for a call on `stream`."""
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else stream)


def _lookup(table, key, what):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise ValueError(f"{what} must be one of {list(table)}, got {key!r}") from None


def _check(t, what, shape, dtype, device, inner=True):
    """Raise unless `t` has this shape (None: any extent), type and device and a contiguous last dimension."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{what} must be on {device}, got {t.device}")
    if len(t.shape) != len(shape) or any(w is not None and w != g for w, g in zip(shape, t.shape)):
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if inner and t.shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{what}'s last dimension must be contiguous")


def _cuda(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{what} must be a CUDA tensor")
    if t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what} must be on the current device")
    return t.device


def rope_axes(x, positions, freqs, out=None, *, rotary_heads=None, layout="pairs", slots=None, stream=None):
    """Rotate x [tokens, heads, head_dim] by angle sum_a positions[a, t] * freqs[h, p, a].

    positions int32 [axes, tokens], freqs fp32 [1 or rotary_heads, pairs, axes];
    heads from rotary_heads on (default: none) and elements from 2 * pairs on
    are copied.  layout: "pairs" mixes (2p, 2p + 1), "halves" (p, p + pairs).
    With slots (int64 [tokens]) token t goes to row slots[t] of out [rows,
    heads, head_dim] (a cache), rows outside it are skipped.  Returns out.
    """
    device = _cuda(x, "x")
    dtype = _lookup(_DTYPES, x.dtype, "x's dtype")
    _check(x, "x", (None, None, None), x.dtype, device)
    tokens, heads, head_dim = x.shape
    rotary = heads if rotary_heads is None else rotary_heads
    _check(positions, "positions", (None, tokens), torch.int32, device)
    axes = positions.shape[0]
    _check(freqs, "freqs", (None, None, axes), torch.float32, device)
    if not positions.is_contiguous() or not freqs.is_contiguous():
        raise ValueError("positions and freqs must be contiguous")
    if out is None:
        if slots is not None:
            raise ValueError("slots need an out to write to")
        with _on(stream, device):
            out = torch.empty((tokens, heads, head_dim), dtype=x.dtype, device=device)
    _check(out, "out", (None if slots is not None else tokens, heads, head_dim), x.dtype, device)
    if slots is not None:
        _check(slots, "slots", (tokens,), torch.int64, device)
    xs, os = x.stride(), out.stride()
    call("kb_rope_axes", x.data_ptr(), dtype, tokens, heads, head_dim, xs[0], xs[1], positions.data_ptr(), axes,
         freqs.data_ptr(), freqs.shape[0], freqs.shape[1], rotary, _lookup(_LAYOUTS, layout, "layout"), _ptr(slots),
         out.shape[0], out.data_ptr(), os[0], os[1], _stream(stream))
    return out


def norm_residual(x, y=None, *, post=None, pre=None, post_gamma=None, post_beta=None, pre_gamma=None, pre_beta=None,
                  gate=None, gate_act="linear", mod_scale=None, mod_shift=None, rows_per_cond=1, res_scale=1.0,
                  branch_scale=1.0, eps=1e-6, x_out=None, h=None, h_dtype=None, stream=None):
    """The norms around a block in one pass over the stream x and the block's output y [rows, width]:

    r = res_scale * x + branch_scale * gate_act(gate) * post_norm(y), returned rounded to x's type, and
    h = pre_norm(r) * (1 + mod_scale) + mod_shift, the next block's input.

    post / pre: None, "rms" or "layer"; gammas and betas fp32 [width] or None;
    gate, mod_scale, mod_shift [ceil(rows / rows_per_cond), width] in y's type
    (h_dtype without y) or None, row r using row r // rows_per_cond.  x_out may
    be x and h may be y (in place); False leaves an output out.  Returns (x_out, h).
    """
    device = _cuda(x, "x")
    _check(x, "x", (None, None), x.dtype, device)
    rows, width = x.shape
    stream_dtype = _lookup(_DTYPES, x.dtype, "x's dtype")
    if y is not None:
        if h_dtype is not None and h_dtype != y.dtype:
            raise TypeError("h has y's type")
        h_dtype = y.dtype
        _check(y, "y", (rows, width), h_dtype, device)
    elif h_dtype is None:
        h_dtype = x.dtype
    branch_dtype = _lookup(_DTYPES, h_dtype, "h's dtype")
    if rows_per_cond < 1:
        raise ValueError("rows_per_cond must be positive")
    for t, what in ((post_gamma, "post_gamma"), (post_beta, "post_beta"), (pre_gamma, "pre_gamma"), (pre_beta, "pre_beta")):
        if t is not None:
            _check(t, what, (width,), torch.float32, device)
    cond_stride = None
    for t, what in ((gate, "gate"), (mod_scale, "mod_scale"), (mod_shift, "mod_shift")):
        if t is not None:
            _check(t, what, (-(-rows // rows_per_cond), width), h_dtype, device)
            stride = t.stride(0) if t.shape[0] > 1 else 0
            if cond_stride is not None and stride != cond_stride:
                raise ValueError("gate, mod_scale and mod_shift must have equal strides")
            cond_stride = stride
    with _on(stream, device):
        if x_out is None:
            x_out = torch.empty((rows, width), dtype=x.dtype, device=device)
        if h is None:
            h = torch.empty((rows, width), dtype=h_dtype, device=device)
    x_out = None if x_out is False else x_out
    h = None if h is False else h
    if x_out is not None:
        _check(x_out, "x_out", (rows, width), x.dtype, device)
    if h is not None:
        _check(h, "h", (rows, width), h_dtype, device)

    def row_stride(t):  # rows of a single-row tensor never step
        return 0 if t is None else t.stride(0) if rows > 1 else width

    desc = _capi.NormResidualDesc(
        rows, width, stream_dtype, branch_dtype, _lookup(_NORMS, post, "post"), _lookup(_NORMS, pre, "pre"),
        _lookup(_GATES, gate_act, "gate_act"), rows_per_cond, res_scale, branch_scale, eps, row_stride(x), row_stride(y),
        row_stride(x_out), row_stride(h), cond_stride or 0)
    call("kb_norm_residual", ctypes.byref(desc), x.data_ptr(), _ptr(y), _ptr(post_gamma), _ptr(post_beta),
         _ptr(pre_gamma), _ptr(pre_beta), _ptr(gate), _ptr(mod_scale), _ptr(mod_shift), _ptr(x_out), _ptr(h),
         _stream(stream))
    return x_out, h


def diff_attention(q, k, v, lam, *, gamma=None, out_scale=1.0, eps=1e-5, scale=None, causal=False, window=0,
                   kv_lens=None, key_mask=None, out=None, status=None, stream=None):
    """softmax(q1 k1^T scale) v - lam softmax(q2 k2^T scale) v per head, then RMS-normed by gamma and scaled.

    q [batch, q_len, heads, 2, d], k [batch, kv_len, kv_heads, 2, d], v [batch,
    kv_len, kv_heads, 2 d], d 32 or 64, bf16 or fp16; lam fp32 [heads]; gamma
    fp32 [2 d] or None (no norm); scale defaults to d ** -0.5.  Keys: below
    kv_lens[b] (int32 [batch]) and with key_mask[b, j] set (bool or uint8
    [batch, kv_len]); causal puts the queries at the end of the keys, window
    keeps the last `window` keys of each.  Queries that see no key give zeros.
    Returns out [batch, q_len, heads, 2 d].
    """
    device = _cuda(q, "q")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"q must be float16 or bfloat16, got {q.dtype}")
    _check(q, "q", (None, None, None, 2, None), q.dtype, device)
    batch, q_len, heads, _, d = q.shape
    _check(k, "k", (batch, None, None, 2, d), q.dtype, device)
    kv_len, kv_heads = k.shape[1:3]
    _check(v, "v", (batch, kv_len, kv_heads, 2 * d), q.dtype, device)
    _check(lam, "lam", (heads,), torch.float32, device)
    if gamma is not None:
        _check(gamma, "gamma", (2 * d,), torch.float32, device)
    if kv_lens is not None:
        _check(kv_lens, "kv_lens", (batch,), torch.int32, device)
    mask_batch = 0
    if key_mask is not None:
        if key_mask.dtype != torch.bool:
            _check(key_mask, "key_mask", (batch, kv_len), torch.uint8, device)
        else:
            _check(key_mask, "key_mask", (batch, kv_len), torch.bool, device)
        mask_batch = key_mask.stride(0)
    if out is None:
        with _on(stream, device):
            out = torch.empty((batch, q_len, heads, 2 * d), dtype=q.dtype, device=device)
    _check(out, "out", (batch, q_len, heads, 2 * d), q.dtype, device)
    desc = _capi.DiffAttentionDesc(
        _DTYPES[q.dtype], batch, q_len, kv_len, heads, kv_heads, d, bool(causal), window,
        d**-0.5 if scale is None else scale, out_scale, eps, *q.stride()[:4], *k.stride()[:4], *v.stride()[:3],
        *out.stride()[:3], mask_batch)
    ref, need = ctypes.byref(desc), ctypes.c_size_t()
    call("kb_diff_attention_workspace", ref, ctypes.byref(need))
    work = None
    if need.value:
        with _on(stream, device):
            work = torch.empty(need.value, dtype=torch.uint8, device=device)
    call("kb_diff_attention", ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _ptr(gamma),
         _ptr(kv_lens), _ptr(key_mask), out.data_ptr(), _ptr(work), need.value, _ptr(status), _stream(stream))
    return out


def diff_lambda(q1, k1, q2, k2, lambda_init):
    """fp32 [heads] weights exp(q1 . k1) - exp(q2 . k2) + lambda_init from learned vectors [heads, d] (CPU)."""
    vectors = [np.ascontiguousarray(t, dtype=np.float32) for t in (q1, k1, q2, k2)]
    if any(t.ndim != 2 or t.shape != vectors[0].shape for t in vectors):
        raise ValueError("the four vectors must have one shape [heads, d]")
    heads, d = vectors[0].shape
    lam = np.empty(heads, np.float32)
    call("kb_diff_lambda", *[t.ctypes.data for t in vectors], heads, d, lambda_init, lam.ctypes.data)
    return lam
