"""CPU tests of the block operators: the lambda weights and the refusals that the
library makes before it touches a device (fake, never dereferenced pointers)."""

import ctypes

import numpy as np
import pytest

from rust_katago_b200 import _capi, block

P = 0x10000  # aligned, never dereferenced


def invalid(code):
    assert code == _capi.KB_E_INVALID, code
    assert _capi.load().kb_last_error()


@pytest.mark.parametrize("heads,d", [(1, 1), (6, 64), (7, 33)])
def test_diff_lambda(heads, d):
    rng = np.random.default_rng(heads * 100 + d)
    v = [(0.1 * rng.standard_normal((heads, d))).astype(np.float32) for _ in range(4)]
    w = [t.astype(np.float64) for t in v]
    ref = np.exp((w[0] * w[1]).sum(1)) - np.exp((w[2] * w[3]).sum(1)) + np.float64(np.float32(0.35))
    # sums in 64 bits, one rounding to fp32 (values below 4: half an ulp is 2^-23)
    assert np.abs(block.diff_lambda(*v, 0.35) - ref).max() <= 2.0**-23


def test_diff_lambda_refusals():
    a = np.zeros((2, 4), np.float32)
    with pytest.raises(ValueError):
        block.diff_lambda(a, a, a, np.zeros((2, 5), np.float32), 0.5)
    with pytest.raises(_capi.KbError):
        block.diff_lambda(*[np.zeros((0, 4), np.float32)] * 4, 0.5)


def rope(**kw):
    a = dict(x=P, dtype=_capi.DT_BF16, tokens=3, heads=4, head_dim=64, x_token=256, x_head=64, positions=P, axes=2,
             freqs=P, freq_heads=1, pairs=32, rotary_heads=4, layout=0, slots=0, out_rows=3, out=2 * P, out_token=256,
             out_head=64)
    a.update(kw)
    return _capi.load().kb_rope_axes(*a.values(), 0)


@pytest.mark.parametrize("kw", [
    dict(dtype=3), dict(tokens=-1), dict(heads=0), dict(head_dim=63), dict(axes=0), dict(axes=5), dict(pairs=33),
    dict(pairs=0), dict(rotary_heads=5), dict(freq_heads=3), dict(layout=2), dict(x=0), dict(out=0), dict(freqs=0),
    dict(positions=0), dict(x=P + 1), dict(x_token=-8), dict(out_token=255), dict(out_head=63), dict(out_token=0),
    dict(out_head=0), dict(out=P, out_token=512), dict(out=P, slots=P), dict(slots=P, out_rows=-1)])
def test_rope_refusals(kw):
    invalid(rope(**kw))


def test_nothing_to_do_needs_no_device():
    assert rope(tokens=0, x=0, out=0) == _capi.KB_OK
    assert norm(rows=0) == _capi.KB_OK
    assert attn(batch=0) == _capi.KB_OK and attn(q_len=0) == _capi.KB_OK


def norm(ptr=None, **kw):
    a = dict(rows=5, width=96, stream_dtype=_capi.DT_F32, branch_dtype=_capi.DT_BF16, post_norm=1, pre_norm=1,
             gate_act=0, rows_per_cond=1, res_scale=1.0, branch_scale=1.0, eps=1e-6, x_stride=96, y_stride=96,
             x_out_stride=96, h_stride=96, cond_stride=96)
    a.update(kw)
    p = dict(x=P, y=2 * P, pg=0, pb=0, qg=0, qb=0, gate=0, ms=0, mt=0, x_out=3 * P, h=4 * P)
    p.update(ptr or {})
    return _capi.load().kb_norm_residual(ctypes.byref(_capi.NormResidualDesc(**a)), *p.values(), 0)


@pytest.mark.parametrize("ptr,kw", [
    ({}, dict(width=0)), ({}, dict(width=16385)), ({}, dict(rows=-1)), ({}, dict(stream_dtype=7)),
    ({}, dict(branch_dtype=-1)), ({}, dict(post_norm=3)), ({}, dict(pre_norm=-1)), ({}, dict(gate_act=3)),
    ({}, dict(eps=-1.0)), ({}, dict(eps=float("nan"))), (dict(gate=P), dict(rows_per_cond=0)), (dict(x=0), {}),
    (dict(x_out=0, h=0), {}), (dict(y=0, gate=P), {}), ({}, dict(x_stride=-96)), ({}, dict(x_out_stride=95)),
    ({}, dict(h_stride=8)), (dict(x_out=P), dict(x_out_stride=128)), (dict(h=2 * P), dict(h_stride=128)),
    (dict(h=P), {}), (dict(h=3 * P), {}), (dict(x_out=2 * P), {})])
def test_norm_refusals(ptr, kw):
    invalid(norm(ptr, **kw))


def attn(ptr=None, bytes_=1 << 40, **kw):
    d = kw.get("head_dim", 64)
    a = dict(dtype=_capi.DT_BF16, batch=2, q_len=8, kv_len=16, heads=4, kv_heads=2, head_dim=d, causal=1, window=0,
             scale=0.125, out_scale=1.0, eps=1e-5, q_batch=8 * 4 * 2 * d, q_token=4 * 2 * d, q_head=2 * d, q_map=d,
             k_batch=16 * 2 * 2 * d, k_token=2 * 2 * d, k_head=2 * d, k_map=d, v_batch=16 * 2 * 2 * d,
             v_token=2 * 2 * d, v_head=2 * d, out_batch=8 * 4 * 2 * d, out_token=4 * 2 * d, out_head=2 * d, mask_batch=16)
    a.update(kw)
    p = dict(q=P, k=2 * P, v=3 * P, lam=P, gamma=P, kv_lens=0, key_mask=0, out=4 * P, work=P)
    p.update(ptr or {})
    desc = _capi.DiffAttentionDesc(**a)
    return _capi.load().kb_diff_attention(ctypes.byref(desc), *p.values(), bytes_, 0, 0)


@pytest.mark.parametrize("ptr,kw", [
    ({}, dict(dtype=_capi.DT_F32)), ({}, dict(head_dim=48)), ({}, dict(head_dim=128)), ({}, dict(heads=3)),
    ({}, dict(kv_heads=0)), ({}, dict(q_len=-1)), ({}, dict(kv_len=-1)), ({}, dict(batch=70000)),
    ({}, dict(window=-1)), ({}, dict(causal=0, window=4)), ({}, dict(scale=float("inf"))), ({}, dict(eps=float("nan"))),
    ({}, dict(q_token=511)), ({}, dict(k_token=-512)), ({}, dict(v_head=132)), ({}, dict(out_head=64)),
    ({}, dict(out_token=0)), ({}, dict(mask_batch=-1)), (dict(q=0), {}), (dict(k=0), {}), (dict(v=0), {}),
    (dict(lam=0), {}), (dict(out=0), {}), (dict(q=P + 8), {}), (dict(k=P + 2), {}), (dict(out=P + 4), {}),
    (dict(out=2 * P), {})])
def test_attention_refusals(ptr, kw):
    invalid(attn(ptr, **kw))


def test_attention_needs_its_workspace():
    d = 64
    desc = _capi.DiffAttentionDesc(
        dtype=_capi.DT_BF16, batch=1, q_len=1, kv_len=65536, heads=2, kv_heads=2, head_dim=d, causal=1, scale=0.125,
        out_scale=1.0, eps=1e-5, k_token=4 * d, k_head=2 * d, k_map=d, q_head=2 * d, q_map=d, v_token=4 * d,
        v_head=2 * d, out_head=2 * d)
    need = ctypes.c_size_t()
    lib = _capi.load()
    assert lib.kb_diff_attention_workspace(ctypes.byref(desc), ctypes.byref(need)) == _capi.KB_OK
    invalid(lib.kb_diff_attention_workspace(None, ctypes.byref(need)))
    invalid(lib.kb_diff_attention_workspace(ctypes.byref(desc), None))
    if need.value:
        args = (ctypes.byref(desc), P, P * 2, P * 3, P, 0, 0, 0, P * 4)
        invalid(lib.kb_diff_attention(*args, P, need.value - 1, 0, 0))
        invalid(lib.kb_diff_attention(*args, 0, need.value, 0, 0))


def test_wrappers_refuse_cpu_tensors():
    import torch

    x = torch.zeros(2, 2, 8)
    with pytest.raises(ValueError):
        block.rope_axes(x, torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 4, 1))
    with pytest.raises(ValueError):
        block.norm_residual(x[0])
    with pytest.raises(TypeError):
        block.diff_attention(None, x, x, x)


@pytest.mark.parametrize("kw", [dict(positions=P + 2), dict(freqs=P + 1), dict(slots=P + 4)])
def test_rope_refuses_misaligned_tensors(kw):
    invalid(rope(**kw))


@pytest.mark.parametrize("ptr", [dict(x=P + 2), dict(y=P + 1), dict(pg=P + 2), dict(pb=P + 3), dict(qg=P + 1), dict(qb=P + 2),
                                 dict(gate=P + 1), dict(ms=P + 1), dict(mt=P + 3), dict(x_out=3 * P + 2), dict(h=4 * P + 1)])
def test_norm_refuses_misaligned_tensors(ptr):
    invalid(norm(ptr))


@pytest.mark.parametrize("ptr", [dict(lam=P + 2), dict(gamma=P + 1), dict(kv_lens=P + 2), dict(status=P + 2)])
def test_attention_refuses_misaligned_tensors(ptr):
    status = ptr.pop("status", 0)
    if status:
        d = 64
        desc = _capi.DiffAttentionDesc(dtype=_capi.DT_BF16, batch=1, q_len=1, kv_len=1, heads=1, kv_heads=1, head_dim=d,
                                       scale=1.0, out_scale=1.0, q_map=d, k_map=d)
        invalid(_capi.load().kb_diff_attention(ctypes.byref(desc), P, P, P, P, 0, 0, 0, 2 * P, 0, 0, status, 0))
    else:
        invalid(attn(ptr))


@pytest.mark.parametrize("ptr,kw", [
    (dict(gate=4 * P), dict(rows_per_cond=5)), (dict(ms=4 * P), dict(rows_per_cond=2)), (dict(mt=4 * P), dict(cond_stride=0)),
    (dict(gate=4 * P), dict(cond_stride=192)), (dict(gate=3 * P), {}), (dict(ms=3 * P), dict(stream_dtype=_capi.DT_BF16)),
    (dict(mt=3 * P), dict(rows_per_cond=5)), (dict(pg=4 * P), {}), (dict(pb=3 * P), {}), (dict(qg=3 * P), dict(rows=1)),
    (dict(qb=4 * P), dict(rows=1))])
def test_norm_refuses_outputs_over_what_rows_share(ptr, kw):
    invalid(norm(ptr, **kw))


@pytest.mark.parametrize("kw", [
    dict(out_token=128, out_head=128), dict(out_batch=512, out_token=512), dict(out_batch=128, out_token=512, out_head=128),
    dict(out_token=128, out_head=8 * 128 - 8), dict(out_batch=8 * 512 - 8), dict(out_batch=128, out_token=248, out_head=8 * 512)])
def test_attention_refuses_outputs_that_overlap(kw):
    invalid(attn(**kw))


@pytest.mark.parametrize("kw", [
    dict(out_token=128, out_head=8 * 128), dict(out_token=520, out_batch=7 * 520 + 512), dict(out_batch=136, out_token=272, out_head=8 * 272),
    dict(out_batch=128, out_token=4 * 256, out_head=256), dict(q_len=1, out_token=0), dict(batch=1, out_batch=8)])
def test_attention_takes_any_nested_output(kw):
    """A descriptor that is right (asked for its workspace: no device needed)."""
    need = ctypes.c_size_t()
    d = dict(dtype=_capi.DT_BF16, batch=2, q_len=8, kv_len=16, heads=4, kv_heads=2, head_dim=64, causal=1, scale=0.125,
             out_scale=1.0, eps=1e-5, q_batch=4096, q_token=512, q_head=128, q_map=64, k_batch=4096, k_token=256, k_head=128,
             k_map=64, v_batch=4096, v_token=256, v_head=128, out_batch=4096, out_token=512, out_head=128)
    desc = _capi.DiffAttentionDesc(**{**d, **kw})
    assert _capi.load().kb_diff_attention_workspace(ctypes.byref(desc), ctypes.byref(need)) == _capi.KB_OK


@pytest.mark.parametrize("init", [None, "half", [0.5, 0.5]])
def test_diff_lambda_refuses_what_is_no_number(init):
    with pytest.raises((TypeError, ValueError)):
        block.diff_lambda(*[np.zeros((2, 4), np.float32)] * 4, init)


@pytest.mark.parametrize("limit,status", [(0, P), (2_000_000_001, P), (5, 0)])
def test_wait_limits_of_no_use_are_refused(limit, status):
    d = 64
    desc = _capi.DiffAttentionDesc(dtype=_capi.DT_BF16, batch=1, q_len=1, kv_len=1, heads=1, kv_heads=1, head_dim=d,
                                   scale=1.0, out_scale=1.0, q_map=d, k_map=d)
    invalid(_capi.load().kb_test_diff_attention_wait_limit(ctypes.byref(desc), P, P, P, P, 2 * P, 0, 0, limit, status, 0))


def test_wrappers_load_without_torch_private_names(monkeypatch):
    import importlib.util

    import torch

    for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("rust_katago_b200._block_copy", block.__file__)
    copy = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(copy)
    assert copy._current_device is torch.cuda.current_device and callable(copy._current_stream)
    with pytest.raises(ValueError):
        copy.norm_residual(torch.zeros(1, 8))
