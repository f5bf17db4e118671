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
from the library.  Inference only: nothing is recorded for autograd, and the
outputs carry no gradient even where an input requires one.  No reference
counterparts: the reference's trunk has one softmax map over 361 tokens.
"""

from __future__ import annotations

import contextlib
import ctypes
import functools
import operator
import struct

import numpy as np
import torch

from . import _capi
from ._capi import call, check, load

_DTYPES = {torch.float32: _capi.DT_F32, torch.float16: _capi.DT_F16, torch.bfloat16: _capi.DT_BF16}
_LAYOUTS = {"pairs": _capi.ROPE_PAIRS, "halves": _capi.ROPE_HALVES}
_NORMS = {None: _capi.NORM_NONE, "rms": _capi.NORM_RMS, "layer": _capi.NORM_LAYER}
_GATES = {"linear": _capi.GATE_LINEAR, "sigmoid": _capi.GATE_SIGMOID, "tanh": _capi.GATE_TANH}

# kb_norm_residual_desc and kb_diff_attention_desc as bytes: packing them takes a
# third of the time of filling a ctypes structure, and a call on one token is
# mostly this file's time.
_NORM_DESC = struct.Struct("@8i3f5q")
_DIFF_DESC = struct.Struct("@9i3f15q")
assert _NORM_DESC.size == ctypes.sizeof(_capi.NormResidualDesc)
assert _DIFF_DESC.size == ctypes.sizeof(_capi.DiffAttentionDesc)


# What torch.cuda.current_device() and current_stream().cuda_stream return, without
# the 10 us of their wrappers (through those where a torch names them otherwise).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


def _raw(stream, device):
    """The cudaStream_t of `stream` (None: the current stream) as an integer."""
    if stream is None:
        return _current_stream(device)
    return stream if isinstance(stream, int) else _cuda_stream(stream).cuda_stream


def _cuda_stream(stream):
    if not isinstance(stream, torch.cuda.Stream):
        raise TypeError(f"stream must be a torch.cuda.Stream or a cudaStream_t as an integer, got {stream!r}")
    return stream


def _lookup(table, key, what):
    try:
        return table[key]
    except (KeyError, TypeError):
        raise ValueError(f"{what} must be one of {list(table)}, got {key!r}") from None


def _device(t, what):
    """The device index of a CUDA tensor on the current device."""
    index = _tensor(t, what).get_device()
    if index < 0:
        raise ValueError(f"{what} must be a CUDA tensor")
    if index != _current_device():
        raise ValueError(f"{what} must be on the current device")
    return index


def _tensor(t, what):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a tensor")
    return t


def _pack(form, *values):
    """A descriptor as bytes."""
    try:
        return form.pack(*values)
    except struct.error as e:
        raise ValueError(f"an argument is no 32-bit integer or no number: {e}") from None


def _check(t, what, shape, dtype, device):
    """The address of `t`; raises unless it has this shape, type and device and a contiguous last dimension."""
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device
            and (t.stride(-1) == 1 or shape[-1] < 2)):
        return t.data_ptr()
    _tensor(t, what)
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.get_device() != device:
        raise ValueError(f"{what} must be on device {device}, got {t.device}")
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    raise ValueError(f"{what}'s last dimension must be contiguous")


def _status(t, device):
    """The address of a status word [flags, first_layer] (None: 0)."""
    if t is None:
        return 0
    if not isinstance(t, torch.Tensor) or t.dtype not in (torch.int32, torch.uint32):
        raise TypeError("status must be an int32 or uint32 tensor")
    if t.get_device() != device or t.dim() != 1 or t.shape[0] < 2 or not t.is_contiguous():
        raise ValueError(f"status must be two contiguous elements on device {device}")
    return t.data_ptr()


@functools.cache
def _native(name):
    """A function of the library (loaded at the first call), without the lookups of a call by name."""
    return getattr(load(), name)


def _on(stream, device):
    """The context in which tensors are allocated for a call on `stream`."""
    if stream is None:
        return contextlib.nullcontext()
    return torch.cuda.stream(
        torch.cuda.ExternalStream(stream, device=device) if isinstance(stream, int) else _cuda_stream(stream))


def _empty(like, shape, dtype, stream, device):
    if stream is None:
        return like.new_empty(shape) if like.dtype is dtype else like.new_empty(shape, dtype=dtype)
    with _on(stream, device):
        return like.new_empty(shape, dtype=dtype)


def rope_axes(x, positions, freqs, out=None, *, rotary_heads=None, layout="pairs", slots=None, stream=None):
    """Rotate x [tokens, heads, head_dim] by angle sum_a positions[a, t] * freqs[h, p, a].

    positions int32 [axes, tokens], freqs fp32 [1 or rotary_heads, pairs, axes];
    heads from rotary_heads on (default: none) and elements from 2 * pairs on
    are copied.  layout: "pairs" mixes (2p, 2p + 1), "halves" (p, p + pairs).
    With slots (int64 [tokens]) token t goes to row slots[t] of out [rows,
    heads, head_dim] (a cache), rows outside it are skipped (two tokens with one
    slot: either may stay).  A NaN or infinite frequency makes its pair NaN.  Returns out.
    """
    device = _device(x, "x")
    dtype, shape = x.dtype, x.shape
    kind = _lookup(_DTYPES, dtype, "x's dtype")
    if len(shape) != 3 or _tensor(freqs, "freqs").dim() != 3:
        raise ValueError("x must be [tokens, heads, head_dim] and freqs [heads, pairs, axes]")
    tokens, heads, head_dim = shape
    freq_shape = freqs.shape
    freq_heads, pairs, axes = freq_shape
    rotary = heads
    if rotary_heads is not None:
        rotary = operator.index(rotary_heads)
        if rotary < 0 or rotary > heads:
            raise ValueError(f"rotary_heads must be 0..{heads}, got {rotary}")
    if (tokens | heads | head_dim | freq_heads | pairs | axes) >> 31:
        raise ValueError("no dimension may pass 2^31 - 1")
    xp = _check(x, "x", shape, dtype, device)
    pp = _check(positions, "positions", (axes, tokens), torch.int32, device)
    fp = _check(freqs, "freqs", freq_shape, torch.float32, device)
    if not positions.is_contiguous() or not freqs.is_contiguous():
        raise ValueError("positions and freqs must be contiguous")
    sp = rows = 0
    if out is None:
        if slots is not None:
            raise ValueError("slots need an out to write to")
        out = _empty(x, shape, dtype, stream, device)
        op = out.data_ptr()
    else:
        rows = out.shape[0] if _tensor(out, "out").dim() else 0
        op = _check(out, "out", shape if slots is None else (rows, heads, head_dim), dtype, device)
        if slots is not None:
            sp = _check(slots, "slots", (tokens,), torch.int64, device)
    xs, os = x.stride(), out.stride()
    code = _native("kb_rope_axes")(
        xp, kind, tokens, heads, head_dim, xs[0], xs[1], pp, axes, fp, freq_heads, pairs,
        rotary, _lookup(_LAYOUTS, layout, "layout"), sp, rows, op, os[0],
        os[1], _raw(stream, device))
    if code:
        check(code)
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
    device = _device(x, "x")
    dtype = x.dtype
    stream_kind = _lookup(_DTYPES, dtype, "x's dtype")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must be [rows, width]")
    rows, width = shape
    xp = _check(x, "x", shape, dtype, device)
    yp = y_stride = 0
    if y is not None:
        if h_dtype is not None and h_dtype != _tensor(y, "y").dtype:
            raise TypeError("h has y's type")
        h_dtype = _tensor(y, "y").dtype
        yp = _check(y, "y", shape, h_dtype, device)
        y_stride = y.stride(0)
    elif h_dtype is None:
        h_dtype = dtype
    branch_kind = _lookup(_DTYPES, h_dtype, "h's dtype")
    if rows_per_cond < 1:
        raise ValueError("rows_per_cond must be positive")
    row, f32 = (width,), torch.float32
    affine = (0 if post_gamma is None else _check(post_gamma, "post_gamma", row, f32, device),
              0 if post_beta is None else _check(post_beta, "post_beta", row, f32, device),
              0 if pre_gamma is None else _check(pre_gamma, "pre_gamma", row, f32, device),
              0 if pre_beta is None else _check(pre_beta, "pre_beta", row, f32, device))
    cond, cond_stride = (0, 0, 0), None
    if gate is not None or mod_scale is not None or mod_shift is not None:
        cond = []
        cond_rows = -(-rows // rows_per_cond)
        for t, what in ((gate, "gate"), (mod_scale, "mod_scale"), (mod_shift, "mod_shift")):
            cond.append(0 if t is None else _check(t, what, (cond_rows, width), h_dtype, device))
            if t is not None:
                if cond_stride is not None and t.stride(0) != cond_stride and cond_rows > 1:
                    raise ValueError("gate, mod_scale and mod_shift must have equal strides")
                cond_stride = t.stride(0)
    xo_p = xo_stride = h_p = h_stride = 0
    if x_out is None:
        x_out = _empty(x, shape, dtype, stream, device)
        xo_p, xo_stride = x_out.data_ptr(), width
    elif x_out is False:
        x_out = None
    else:
        xo_p, xo_stride = _check(x_out, "x_out", shape, dtype, device), x_out.stride(0)
    if h is None:
        h = _empty(x, shape, h_dtype, stream, device)
        h_p, h_stride = h.data_ptr(), width
    elif h is False:
        h = None
    else:
        h_p, h_stride = _check(h, "h", shape, h_dtype, device), h.stride(0)
    x_stride = x.stride(0)
    if rows <= 1:  # the strides of single rows are never used
        x_stride = y_stride = xo_stride = h_stride = width
    desc = _pack(
        _NORM_DESC, rows, width, stream_kind, branch_kind, _lookup(_NORMS, post, "post"), _lookup(_NORMS, pre, "pre"),
        _lookup(_GATES, gate_act, "gate_act"), rows_per_cond, res_scale, branch_scale, eps, x_stride, y_stride,
        xo_stride, h_stride, cond_stride or 0)
    code = _native("kb_norm_residual")(desc, xp, yp, *affine, *cond, xo_p, h_p, _raw(stream, device))
    if code:
        check(code)
    return x_out, h


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(desc, device):
    """Scratch that a descriptor needs on a device (its number of SMs matters)."""
    need = ctypes.c_size_t()
    call("kb_diff_attention_workspace", desc, ctypes.byref(need))
    return need.value


def diff_attention(q, k, v, lam, *, gamma=None, out_scale=1.0, eps=1e-5, scale=None, causal=False, window=0,
                   kv_lens=None, key_mask=None, out=None, status=None, stream=None):
    """softmax(q1 k1^T scale) v - lam softmax(q2 k2^T scale) v per head, then RMS-normed by gamma and scaled.

    q [batch, q_len, heads, 2, d], k [batch, kv_len, kv_heads, 2, d], v [batch,
    kv_len, kv_heads, 2 d], d 32 or 64, bf16 or fp16; lam fp32 [heads]; gamma
    fp32 [2 d] or None (no norm); scale defaults to d ** -0.5.  Keys: below
    kv_lens[b] (int32 [batch]) and with key_mask[b, j] set (bool or uint8
    [batch, kv_len]); causal puts the queries at the end of the sequence (of
    kv_lens[b] tokens, of which k and v may hold only the first kv_len), window
    keeps the last `window` positions of each.  Queries that see no key give zeros.
    status: a status word (int32 or uint32 [flags, first_layer], two elements),
    zero flags and first_layer -1 to begin with; a kernel that gives up one of its
    waits (two seconds: a fault) sets KB_STATUS_TIMEOUT there and leaves out
    partial, and without a status word nothing tells.  Returns out [batch, q_len,
    heads, 2 d].
    """
    device = _device(q, "q")
    dtype = q.dtype
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise TypeError(f"q must be float16 or bfloat16, got {dtype}")
    q_shape, k_shape = q.shape, _tensor(k, "k").shape
    if len(q_shape) != 5 or len(k_shape) != 5 or q_shape[3] != 2:
        raise ValueError("q and k must be [batch, tokens, heads, 2, d]")
    batch, q_len, heads, _, d = q_shape
    kv_len, kv_heads = k_shape[1], k_shape[2]
    qp = _check(q, "q", q_shape, dtype, device)
    kp = _check(k, "k", (batch, kv_len, kv_heads, 2, d), dtype, device)
    vp = _check(v, "v", (batch, kv_len, kv_heads, 2 * d), dtype, device)
    lp = _check(lam, "lam", (heads,), torch.float32, device)
    gp = 0 if gamma is None else _check(gamma, "gamma", (2 * d,), torch.float32, device)
    np_ = 0 if kv_lens is None else _check(kv_lens, "kv_lens", (batch,), torch.int32, device)
    mp = mask_batch = 0
    if key_mask is not None:
        mp = _check(key_mask, "key_mask", (batch, kv_len),
                    torch.bool if _tensor(key_mask, "key_mask").dtype is torch.bool else torch.uint8, device)
        mask_batch = key_mask.stride(0)
    if out is None:
        out = _empty(q, (batch, q_len, heads, 2 * d), dtype, stream, device)
        op = out.data_ptr()
    else:
        op = _check(out, "out", (batch, q_len, heads, 2 * d), dtype, device)
    qs, ks, vs, os = q.stride(), k.stride(), v.stride(), out.stride()
    desc = _pack(
        _DIFF_DESC, _DTYPES[dtype], batch, q_len, kv_len, heads, kv_heads, d, bool(causal), window,
        d**-0.5 if scale is None else scale, out_scale, eps, qs[0], qs[1], qs[2], qs[3], ks[0], ks[1], ks[2], ks[3],
        vs[0], vs[1], vs[2], os[0], os[1], os[2], mask_batch)
    sp = _status(status, device)
    need, wp = _workspace_bytes(desc, device), 0
    if need:
        work = _empty(q, need, torch.uint8, stream, device)
        wp = work.data_ptr()
    code = _native("kb_diff_attention")(desc, qp, kp, vp, lp, gp, np_, mp, op, wp, need,
                                        sp, _raw(stream, device))
    if code:
        check(code)
    return out


def diff_lambda(q1, k1, q2, k2, lambda_init):
    """fp32 [heads] weights exp(q1 . k1) - exp(q2 . k2) + lambda_init from learned vectors [heads, d] (CPU)."""
    vectors = [np.ascontiguousarray(t, dtype=np.float32) for t in (q1, k1, q2, k2)]
    if any(t.ndim != 2 or t.shape != vectors[0].shape for t in vectors):
        raise ValueError("the four vectors must have one shape [heads, d]")
    heads, d = vectors[0].shape
    lam = np.empty(heads, np.float32)
    call("kb_diff_lambda", *[t.ctypes.data for t in vectors], heads, d, float(lambda_init), lam.ctypes.data)
    return lam
