"""GPU tests of the block operators against their definitions in 64 bits.

Every tolerance is an error bound derived from the kernels' roundings: u is half
an ulp of the 16-bit type relative to the value (2^-8 for bfloat16, 2^-11 for
binary16 plus half its smallest subnormal), e = 2^-24 that of fp32.
"""

import ctypes

import pytest
import torch

from rust_katago_b200 import _capi, block

pytestmark = pytest.mark.gpu

E = 2.0**-24
U = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0**-25, torch.float32: 0.0}


def rounding(ref, dtype):
    return U[dtype] * ref.abs() + TINY[dtype]


def close(got, ref, bound):
    assert got.shape == ref.shape
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(ref))
    over = (got - ref).abs() - bound
    over = over[~torch.isnan(ref)]
    assert over.numel() == 0 or float(over.max()) <= 0, f"off by {float(over.max())} over the bound"


# ------------------------------------------------------------------ rotary positions
def rope_ref(x, positions, freqs, rotary, layout):
    """(result, |u| + |v| of each element's pair) in 64 bits."""
    x = x.double()
    pairs = freqs.shape[1]
    ang = torch.einsum("at,hpa->thp", positions.double(), freqs.double())
    c, s = ang.cos(), ang.sin()
    out, size = x.clone(), torch.zeros_like(x)
    at = torch.arange(pairs, device=x.device)
    lo, hi = (2 * at, 2 * at + 1) if layout == "pairs" else (at, at + pairs)
    u, v = x[:, :rotary, lo], x[:, :rotary, hi]
    out[:, :rotary, lo], out[:, :rotary, hi] = u * c - v * s, u * s + v * c
    size[:, :rotary, lo] = size[:, :rotary, hi] = u.abs() + v.abs()
    return out, size


def rope_bound(ref, size, dtype):
    # 16-bit: sine and cosine good to 2^-20 absolute.  fp32: 2 ulp of sincospif, pi e of the rounded turns, 3 e of the
    # products and the sum.
    return rounding(ref, dtype) + size * (12 * E if dtype == torch.float32 else 2.0**-20)


def rope_inputs(tokens, heads, head_dim, pairs, axes, freq_heads, dtype, span, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, heads, head_dim, generator=g, device="cuda").to(dtype)
    pos = torch.randint(-span, span, (axes, tokens), generator=g, device="cuda", dtype=torch.int32)
    freqs = 2 * torch.rand(freq_heads, pairs, axes, generator=g, device="cuda") - 1
    return x, pos, freqs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("tokens,heads,head_dim,pairs,rotary,axes,shared", [
    (1, 1, 2, 1, 1, 1, True), (1, 36, 64, 32, 24, 3, True), (361, 18, 64, 32, 12, 2, False),
    (37, 5, 32, 8, 3, 4, False), (7, 3, 40, 14, 3, 3, False), (1000, 2, 128, 64, 0, 1, True),
    (2888, 12, 32, 16, 12, 2, False), (5, 700, 8, 4, 650, 2, True), (129, 4, 96, 5, 4, 1, True)])
def test_rope(cuda, dtype, layout, tokens, heads, head_dim, pairs, rotary, axes, shared):
    x, pos, freqs = rope_inputs(tokens, heads, head_dim, pairs, axes, 1 if shared else max(rotary, 1), dtype, 400)
    got = block.rope_axes(x, pos, freqs, rotary_heads=rotary, layout=layout)
    ref, size = rope_ref(x, pos, freqs, rotary, layout)
    close(got, ref, rope_bound(ref, size, dtype))
    assert torch.equal(got[:, rotary:], x[:, rotary:]) and torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rope_long_positions_keep_their_accuracy(cuda, dtype):
    x, pos, freqs = rope_inputs(300, 2, 64, 32, 3, 2, dtype, 2**31 - 1, seed=3)
    ref, size = rope_ref(x, pos, freqs, 2, "pairs")
    # the 64-bit angle itself: 3 * 2^31 * 2^-52 of reduction error on either side
    close(block.rope_axes(x, pos, freqs), ref, rope_bound(ref, size, dtype) + size * 2.0**-17)


def test_rope_strides_in_place_and_slots(cuda):
    x, pos, freqs = rope_inputs(100, 6, 64, 32, 2, 1, torch.bfloat16, 50, seed=1)
    plain = block.rope_axes(x, pos, freqs)
    # heads outer, odd offsets (single elements), a piece of wider rows
    outer = x.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(block.rope_axes(outer, pos, freqs), plain)
    wide = torch.zeros(100, 6 * 64 + 11, dtype=x.dtype, device="cuda")
    odd = wide[:, 3:3 + 384].unflatten(1, (6, 64))
    odd.copy_(x)
    assert torch.equal(block.rope_axes(odd, pos, freqs), plain)
    assert torch.equal(block.rope_axes(odd, pos, freqs, out=odd), plain)
    assert (wide[:, :3] == 0).all() and (wide[:, 387:] == 0).all()
    # into a cache by slot; rows outside it are skipped
    slots = torch.randperm(150, device="cuda")[:100]
    slots[5], slots[17], slots[40] = -1, 150, 2**40
    cache = torch.full((150, 6, 64), 7.0, dtype=x.dtype, device="cuda")
    block.rope_axes(x, pos, freqs, out=cache, slots=slots)
    want = torch.full_like(cache, 7.0)
    keep = (slots >= 0) & (slots < 150)
    want[slots[keep]] = plain[keep]
    assert torch.equal(cache, want)


def test_rope_copies_non_finite_values_and_keeps_them_in_their_pair(cuda):
    x, pos, freqs = rope_inputs(4, 2, 32, 8, 1, 1, torch.float16, 9, seed=2)
    x[1, 0, 20], x[2, 1, 31], x[3, 0, 2] = float("nan"), float("inf"), float("nan")
    got = block.rope_axes(x, pos, freqs)
    ref, size = rope_ref(x, pos, freqs, 2, "pairs")
    bad = torch.isnan(got)
    assert bad.sum() == 3 and bad[1, 0, 20] and bad[3, 0, 2] and bad[3, 0, 3] and got[2, 1, 31] == float("inf")


# ------------------------------------------------------------------ norms around a block
def norm_ref(v, kind, gamma, beta, eps):
    if kind is None:
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / ((v * v).mean(-1, keepdim=True) + eps).sqrt()
    v = v * (1 if gamma is None else gamma.double())
    return v + (0 if beta is None else beta.double())


ACTS = {"linear": lambda t: t, "sigmoid": torch.sigmoid, "tanh": torch.tanh}


@pytest.mark.parametrize("xdt,ydt", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.bfloat16),
                                     (torch.float16, torch.float16), (torch.float32, torch.float32),
                                     (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,width,post,pre,act,per,affine", [
    (1, 768, "rms", "rms", None, 1, True), (1, 1, "layer", "rms", "tanh", 1, True), (361, 384, "layer", "layer", "linear", 361, True),
    (50, 17, "rms", "layer", "sigmoid", 7, False), (33, 1000, None, "rms", "tanh", 1, True),
    (9, 1024, "rms", None, None, 1, False), (6, 1032, "layer", "layer", "linear", 2, True),
    (5, 5121, "rms", "layer", "sigmoid", 5, True), (3, 16384, "layer", "rms", "tanh", 2, True),
    (4000, 256, "rms", "rms", "linear", 100, True), (2, 16383, "rms", "rms", None, 1, False)])
def test_norm_residual(cuda, xdt, ydt, rows, width, post, pre, act, per, affine):
    g = torch.Generator(device="cuda").manual_seed(rows * 31 + width)

    def normal(*shape, dtype=torch.float32, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    x, y = normal(rows, width, dtype=xdt, std=2.0), normal(rows, width, dtype=ydt, mean=0.3)
    pg, pb, qg, qb = (normal(width, std=0.2, mean=m) if affine else None for m in (1.0, 0.1, 0.9, -0.1))
    gate = ms = mt = None
    if act:
        n = -(-rows // per)
        gate, ms, mt = (normal(n, width, dtype=ydt, std=0.5) for _ in range(3))
    xo, h = block.norm_residual(x, y, post=post, pre=pre, post_gamma=pg, post_beta=pb, pre_gamma=qg, pre_beta=qb,
                                gate=gate, gate_act=act or "linear", mod_scale=ms, mod_shift=mt, rows_per_cond=per,
                                res_scale=0.75, branch_scale=1.25, eps=1e-3)
    eps = float(torch.tensor(1e-3))
    yd = y.double()
    n = norm_ref(yd, post, pg, pb, eps)
    row = torch.arange(rows, device="cuda") // per
    if act:
        n = n * ACTS[act](gate.double()[row])
    r = 0.75 * x.double() + 1.25 * n
    # fp32 roundings on the way to r: at most 32 terms in a thread's chain, 5 + 32 steps of the reduction, 10 more; a
    # centred value also carries the mean's error, relative to the row's largest value over its deviation.
    steps = 96 * E
    yrms = (yd.square().mean(-1, keepdim=True) + eps).sqrt()
    spread = 1 if post != "layer" else yrms / (yd.var(-1, correction=0, keepdim=True) + eps).sqrt()
    gpost = 1 if pg is None or post is None else pg.double().abs()
    gact = ACTS[act](gate.double()[row]).abs() if act else 1
    # |post_norm| without its shift is at most |y| / deviation; + 1 for the mean's share, + |beta|
    size_n = gact * (gpost * (((yd.abs() / yrms + 1) * spread) if post else yd.abs()) + (pb.double().abs() if pb is not None and post else 0))
    rerr = steps * (0.75 * x.double().abs() + 1.25 * size_n * (spread if post else 1))
    close(xo, r, rounding(r, xdt) + rerr)
    m = norm_ref(r, pre, qg, qb, eps)
    scale = 1 + ms.double()[row] if act else torch.ones_like(m)
    ref = m * scale + (mt.double()[row] if act else 0)
    rrms = (r.square().mean(-1, keepdim=True) + eps).sqrt()
    dev = rrms if pre != "layer" else (r.var(-1, correction=0, keepdim=True) + eps).sqrt()
    gpre = 1 if qg is None or pre is None else qg.double().abs()
    top = rerr.amax(-1, keepdim=True)
    if pre:
        # r's error, its effect on mean and deviation (at most its largest, relative to the deviation), own roundings
        herr = gpre * ((rerr + top + top * (r.abs() + rrms) / dev) / dev + steps * (r.abs() + rrms) / dev * (rrms / dev))
        herr = herr + steps * (qb.double().abs() if qb is not None else 0)
    else:
        herr = rerr + steps * r.abs()
    herr = herr * (scale.abs() + (1 + scale.abs()) * 2 * E) + 4 * E * ref.abs() + (2 * E * mt.double()[row].abs() if act else 0)
    close(h, ref, rounding(ref, ydt) + herr)


@pytest.mark.parametrize("width", [1032, 2560, 2568, 2680, 3584, 3592, 4096, 4100, 5120, 5128, 6144, 8192, 8200, 12000])
@pytest.mark.parametrize("shifts", [0, 1, 2])
def test_norm_wide_rows_of_every_shared_size(cuda, width, shifts):
    g = torch.Generator(device="cuda").manual_seed(width)
    x, y = (torch.randn(3, width, generator=g, device="cuda") for _ in range(2))
    b = torch.randn(width, generator=g, device="cuda")
    kw = dict(pre_beta=b if shifts else None, post_beta=b if shifts == 2 else None)
    xo, h = block.norm_residual(x, y, post="rms", pre="layer", **kw)
    r = x.double() + norm_ref(y.double(), "rms", None, kw["post_beta"], 1e-6)
    ref = norm_ref(r, "layer", None, kw["pre_beta"], 1e-6)
    # values and deviations near 1: 96 roundings of fp32 on the way to r, twice that to h
    close(xo, r, 96 * E * (1 + r.abs()))
    close(h, ref, 192 * E * (2 + ref.abs() + b.abs()))


def test_norm_forms_without_parts_in_place_and_strided(cuda):
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(70, 200, generator=g, device="cuda")
    y = torch.randn(70, 200, generator=g, device="cuda").bfloat16()
    full = block.norm_residual(x, y, post="rms", pre="rms", res_scale=0.5)
    only_x, none = block.norm_residual(x, y, post="rms", pre="rms", res_scale=0.5, h=False)
    assert none is None and torch.equal(only_x, full[0])
    none, only_h = block.norm_residual(x, y, post="rms", pre="rms", res_scale=0.5, x_out=False)
    assert none is None and torch.equal(only_h, full[1])
    xi, yi = x.clone(), y.clone()
    a, b = block.norm_residual(xi, yi, post="rms", pre="rms", res_scale=0.5, x_out=xi, h=yi)
    assert a is xi and b is yi and torch.equal(xi, full[0]) and torch.equal(yi, full[1])
    # rows of wider buffers at odd offsets take the kernel of single elements; its sums run in another order
    wx = torch.zeros(70, 209, device="cuda")
    wx[:, 5:205] = x
    sx, sh = block.norm_residual(wx[:, 5:205], y, post="rms", pre="rms", res_scale=0.5)
    assert (sx - full[0]).abs().max() <= 96 * E * 8
    assert (sh.float() - full[1].float()).abs().max() <= 2.0**-7 * full[1].float().abs().max()
    # the first block's norm: no branch
    xo, h = block.norm_residual(x, pre="layer", h_dtype=torch.float16)
    assert torch.equal(xo, x) and h.dtype == torch.float16
    ref = norm_ref(x.double(), "layer", None, None, 1e-6)
    close(h, ref, rounding(ref, torch.float16) + 200 * E * (1 + ref.abs()))


def test_norm_rows_of_zeros_and_non_finite_rows(cuda):
    x, y = torch.zeros(6, 96, device="cuda"), torch.zeros(6, 96, device="cuda", dtype=torch.float16)
    y[2, 3], y[4, 5] = float("nan"), float("inf")
    xo, h = block.norm_residual(x, y, post="rms", pre="rms")
    fine = [0, 1, 3, 5]
    assert (xo[fine] == 0).all() and (h[fine] == 0).all()
    assert torch.isnan(xo[2]).all() and torch.isnan(h[2]).all() and torch.isnan(xo[4, 5]) and torch.isnan(h[4]).all()


# ------------------------------------------------------------------ differential attention
def attn_inputs(batch, q_len, kv_len, heads, kv_heads, d, dtype, seed=0, qstd=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    return (normal(batch, q_len, heads, 2, d, std=qstd), normal(batch, kv_len, kv_heads, 2, d),
            normal(batch, kv_len, kv_heads, 2 * d), torch.rand(heads, generator=g, device="cuda") + 0.1,
            torch.randn(2 * d, generator=g, device="cuda") * 0.2 + 1)


def visible(batch, q_len, kv_len, causal, window, kv_lens, key_mask):
    at = torch.arange(kv_len, device="cuda")
    n = torch.full((batch,), kv_len, device="cuda") if kv_lens is None else kv_lens.long().clamp(0, kv_len)
    see = (at < n[:, None])[:, None].expand(batch, q_len, kv_len).clone()
    if key_mask is not None:
        see &= key_mask.bool()[:, None]
    if causal:
        pos = n[:, None, None] - q_len + torch.arange(q_len, device="cuda")[:, None]
        see &= at <= pos
        if window:
            see &= at > pos - window
    return see


def attn_ref(q, k, v, lam, gamma, see, out_scale, eps, scale):
    """(result, error bound) in 64 bits.  P is rounded to the 16-bit type (u) after an exponential good to 2^-12 and a
    logit good to d e of its terms' size; both maps' errors add, and the norm scales them and its own relative error."""
    b, q_len, heads, _, d = q.shape
    dtype = q.dtype
    g = heads // k.shape[2]
    hidden_k, hidden_v = ~see.any(1), ~see.any(1)
    k = k.double().masked_fill(hidden_k[:, :, None, None, None], 0).repeat_interleave(g, 2)
    v = v.double().masked_fill(hidden_v[:, :, None, None], 0).repeat_interleave(g, 2)
    q = q.double()
    logit = torch.einsum("bihmd,bjhmd->bhmij", q, k) * scale
    size = torch.einsum("bihmd,bjhmd->bhmij", q.abs(), k.abs()) * abs(scale)
    logit = logit.masked_fill(~see[:, None, None], float("-inf"))
    p = torch.nan_to_num(torch.softmax(logit, -1))
    o = torch.einsum("bhmij,bjhe->bihme", p, v)
    rel = U[dtype] + 2.0**-11 + 2 * (d + 4) * E * size.masked_fill(~see[:, None, None], 0).amax(-1)  # bhmi
    # binary16: probabilities below its normal range lose up to half a subnormal each
    small = (2.0**-25 if dtype == torch.float16 else 0.0) * torch.einsum("bij,bjhe->bihe", see.double(), v.abs())
    mass = torch.einsum("bhmij,bjhe->bihme", p, v.abs()) * rel.permute(0, 3, 1, 2)[..., None]
    w = lam.double()[None, None, :, None]
    diff = o[:, :, :, 0] - w * o[:, :, :, 1]
    err = mass[:, :, :, 0] + w * mass[:, :, :, 1] + small * (1 + w)
    if gamma is not None:
        rms = (diff.square().mean(-1, keepdim=True) + eps).sqrt()
        err_rms = err.square().mean(-1, keepdim=True).sqrt()
        f = gamma.double() * out_scale / rms
        ref = diff * f
        bound = f.abs() * (err + (diff.abs() + err) * err_rms / rms)
    else:
        ref, bound = diff * out_scale, err * abs(out_scale)
    return ref, bound + rounding(ref, dtype) + 16 * E * ref.abs()


CASES = [
    # batch, q_len, kv_len, heads, kv_heads, d, causal, window, lens, mask
    (1, 1, 1, 1, 1, 64, True, 0, None, None),
    (1, 1, 1, 1, 1, 32, False, 0, None, None),
    (2, 1, 63, 6, 6, 64, True, 0, None, None),
    (3, 1, 1000, 12, 4, 64, True, 0, [1000, 0, 17], None),
    (2, 1, 777, 6, 1, 32, True, 100, [777, 300], None),
    (2, 3, 515, 4, 2, 64, True, 0, [515, 2], None),
    (1, 16, 200, 3, 3, 32, False, 0, None, "random"),
    (2, 17, 17, 2, 2, 64, True, 0, None, None),
    (2, 40, 33, 2, 1, 64, True, 0, [33, 20], None),
    (2, 361, 361, 6, 6, 64, False, 0, None, None),
    (3, 361, 361, 6, 6, 32, False, 0, None, "boards"),
    (2, 361, 361, 2, 2, 64, False, 0, [361, 0], "empty"),
    (1, 127, 129, 2, 2, 64, True, 0, None, None),
    (1, 129, 128, 2, 2, 32, True, 0, None, None),
    (1, 300, 300, 4, 2, 64, True, 50, None, "random"),
    (1, 700, 700, 2, 2, 32, True, 129, None, None),
    (1, 257, 2500, 2, 2, 64, True, 0, [2301], None),
    (4, 130, 1300, 3, 1, 64, True, 300, [1300, 131, 64, 1], None),
    (1, 5, 4097, 8, 1, 64, True, 0, None, None),
    (1, 33, 9000, 4, 4, 32, True, 0, [8999], "random"),
    (1, 1, 20000, 2, 2, 64, True, 0, None, "random"),
    (2, 1, 5000, 16, 1, 64, True, 700, [5000, 512], "random"),
    # several tiles of queries for every SM
    (40, 361, 361, 6, 6, 32, False, 0, None, "random"),
    (24, 300, 333, 8, 2, 64, True, 150, None, None),
]


def make_mask(kind, batch, kv_len):
    if kind is None:
        return None
    g = torch.Generator(device="cuda").manual_seed(kv_len)
    if kind == "random":
        return torch.rand(batch, kv_len, generator=g, device="cuda") < 0.6
    if kind == "empty":
        return torch.zeros(batch, kv_len, dtype=torch.bool, device="cuda")
    at = torch.arange(kv_len, device="cuda")
    side = torch.tensor([19, 9, 13], device="cuda")[:batch, None]
    return (at // 19 < side) & (at % 19 < side)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c[:8]))
def test_diff_attention(cuda, dtype, case):
    batch, q_len, kv_len, heads, kv_heads, d, causal, window, lens, mask = case
    q, k, v, lam, gamma = attn_inputs(batch, q_len, kv_len, heads, kv_heads, d, dtype, seed=q_len + kv_len)
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    key_mask = make_mask(mask, batch, kv_len)
    see = visible(batch, q_len, kv_len, causal, window, kv_lens, key_mask)
    for norm in (gamma, None):
        got = block.diff_attention(q, k, v, lam, gamma=norm, out_scale=0.6, eps=1e-4, causal=causal, window=window,
                                   kv_lens=kv_lens, key_mask=key_mask)
        ref, bound = attn_ref(q, k, v, lam, norm, see, float(torch.tensor(0.6)), float(torch.tensor(1e-4)), d**-0.5)
        close(got, ref, bound)
        assert (got[~see.any(-1)] == 0).all()


HIDDEN = [c for c in CASES if c[8] is not None or c[9] is not None]


@pytest.mark.parametrize("fill", [float("nan"), float("inf")])
@pytest.mark.parametrize("case", HIDDEN, ids=lambda c: "-".join(str(x) for x in c[:8]))
def test_hidden_keys_and_values_are_never_used(cuda, case, fill):
    batch, q_len, kv_len, heads, kv_heads, d, causal, window, lens, mask = case
    q, k, v, lam, gamma = attn_inputs(batch, q_len, kv_len, heads, kv_heads, d, torch.bfloat16)
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    key_mask = make_mask(mask, batch, kv_len)
    kw = dict(gamma=gamma, causal=causal, window=window, kv_lens=kv_lens, key_mask=key_mask)
    before = block.diff_attention(q, k, v, lam, **kw)
    hidden = ~visible(batch, 1, kv_len, False, 0, kv_lens, key_mask)[:, 0]
    k[hidden], v[hidden] = fill, -fill
    assert torch.equal(block.diff_attention(q, k, v, lam, **kw), before)
    assert torch.isfinite(before).all()


def test_visible_non_finite_values_reach_the_output(cuda):
    for q_len in (1, 200):
        q, k, v, lam, _ = attn_inputs(1, q_len, 200, 2, 2, 64, torch.bfloat16)
        v[0, 7, 1, 5] = float("nan")
        got = block.diff_attention(q, k, v, lam)
        assert torch.isnan(got[0, :, 1, 5]).all() and torch.isnan(got).sum() == q_len
        v[0, 7, 1, 5] = 0
        q[0, 0, 0, 0, 3] = float("nan")
        got = block.diff_attention(q, k, v, lam)
        assert torch.isnan(got[0, 0, 0]).all() and torch.isnan(got).sum() == 128


@pytest.mark.parametrize("q_len,kv_len", [(1, 900), (200, 333)])
def test_large_and_constant_logits(cuda, q_len, kv_len):
    q, k, v, lam, gamma = attn_inputs(2, q_len, kv_len, 2, 2, 64, torch.bfloat16, qstd=40.0)
    see = visible(2, q_len, kv_len, False, 0, None, None)
    ref, bound = attn_ref(q, k, v, lam, gamma, see, 1.0, 1e-5, 0.125)
    close(block.diff_attention(q, k, v, lam, gamma=gamma), ref, bound)
    # one growing logit after another: every key is the new maximum
    ramp = torch.linspace(-30, 30, kv_len, device="cuda").bfloat16()
    k[:] = 0
    k[..., 0] = ramp[None, :, None, None]
    q[:] = 0
    q[..., 0] = 16.0
    ref, bound = attn_ref(q, k, v, lam, gamma, see, 1.0, 1e-5, 0.125)
    close(block.diff_attention(q, k, v, lam, gamma=gamma), ref, bound)
    q[:] = 0  # all logits equal: means
    ref, bound = attn_ref(q, k, v, lam, None, see, 1.0, 1e-5, 0.125)
    close(block.diff_attention(q, k, v, lam), ref, bound)


@pytest.mark.parametrize("q_len,kv_len,kv_heads", [(1, 700, 2), (150, 260, 2), (90, 2000, 4)])
def test_strides_and_layouts(cuda, q_len, kv_len, kv_heads):
    q, k, v, lam, gamma = attn_inputs(2, q_len, kv_len, 4, kv_heads, 32, torch.float16, seed=9)
    kw = dict(gamma=gamma, causal=True)
    ref = block.diff_attention(q, k, v, lam, **kw)
    hf = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # heads before tokens
    maps = lambda t: t.permute(3, 0, 1, 2, 4).contiguous().permute(1, 2, 3, 0, 4)  # the two maps far apart
    assert torch.equal(block.diff_attention(hf(q), hf(k), hf(v), lam, **kw), ref)
    assert torch.equal(block.diff_attention(maps(q), maps(k), v, lam, **kw), ref)
    row = torch.zeros(2, kv_len, 2 * kv_heads * 64 + 24, dtype=torch.float16, device="cuda")  # a fused cache row
    row[..., 8:8 + kv_heads * 64], row[..., 16 + kv_heads * 64:-8] = k.flatten(2), v.flatten(2)
    kk, vv = row[..., 8:8 + kv_heads * 64].unflatten(-1, (kv_heads, 2, 32)), row[..., 16 + kv_heads * 64:-8].unflatten(-1, (kv_heads, 64))
    out = torch.full((2, 4, q_len, 72), 5.0, dtype=torch.float16, device="cuda")
    got = block.diff_attention(q, kk, vv, lam, out=out[..., :64].transpose(1, 2), **kw)
    assert torch.equal(got, ref) and (out[..., 64:] == 5).all()
    # broadcast: one sequence's keys for all, one key head for both maps
    ks, vs = k[:1].expand_as(k), v[:1].expand_as(v)
    assert torch.equal(block.diff_attention(q, ks, vs, lam, **kw), block.diff_attention(q, ks.clone(), vs.clone(), lam, **kw))
    km = k[..., :1, :].expand_as(k)
    assert torch.equal(block.diff_attention(q, km, v, lam, **kw), block.diff_attention(q, km.clone(), v, lam, **kw))
    with pytest.raises(_capi.KbError):
        block.diff_attention(q, row[..., 4:4 + kv_heads * 64].unflatten(-1, (kv_heads, 2, 32)), v, lam, **kw)


@pytest.mark.parametrize("q_len", [1, 130])
def test_offsets_past_32_bits(cuda, q_len):
    q, k, v, lam, gamma = attn_inputs(1, q_len, 160, 2, 2, 64, torch.bfloat16, seed=4)
    step = (1 << 25) + 264
    room = torch.empty(160 * step, dtype=torch.bfloat16, device="cuda")
    kf = room.as_strided(k.shape, (0, step, 128, 64, 1))
    vf = room.as_strided(v.shape, (0, step, 128, 1), 256)
    kf.copy_(k)
    vf.copy_(v)
    kw = dict(gamma=gamma, causal=True)
    assert torch.equal(block.diff_attention(q, kf, vf, lam, **kw), block.diff_attention(q, k, v, lam, **kw))


def test_window_wider_than_the_keys_hides_nothing(cuda):
    for q_len, kv_len in ((1, 300), (140, 140)):
        q, k, v, lam, gamma = attn_inputs(1, q_len, kv_len, 2, 2, 64, torch.bfloat16)
        ref = block.diff_attention(q, k, v, lam, gamma=gamma, causal=True)
        for window in (kv_len, 2**31 - 1):
            assert torch.equal(block.diff_attention(q, k, v, lam, gamma=gamma, causal=True, window=window), ref)


def test_empty_lengths(cuda):
    q, k, v, lam, gamma = attn_inputs(2, 5, 8, 2, 2, 64, torch.bfloat16)
    got = block.diff_attention(q, k[:, :0], v[:, :0], lam, gamma=gamma)
    assert (got == 0).all() and got.shape == (2, 5, 2, 128)
    assert block.diff_attention(q[:, :0], k, v, lam).shape == (2, 0, 2, 128)
    assert block.diff_attention(q[:0], k[:0], v[:0], lam).shape == (0, 5, 2, 128)
    far = torch.tensor([99, -4], dtype=torch.int32, device="cuda")  # clamped to [0, kv_len]
    got = block.diff_attention(q, k, v, lam, kv_lens=far)
    assert torch.equal(got[0], block.diff_attention(q, k, v, lam)[0]) and (got[1] == 0).all()


@pytest.mark.parametrize("batch,q_len,kv_len", [(1, 1, 30000), (1, 361, 361), (1, 100, 6000), (130, 361, 361), (1, 9000, 9000)])
def test_repeats_are_bitwise_equal_on_any_stream(cuda, batch, q_len, kv_len):
    q, k, v, lam, gamma = attn_inputs(batch, q_len, kv_len, 2, 2, 64, torch.bfloat16)
    ref = block.diff_attention(q, k, v, lam, gamma=gamma, causal=True)
    status = torch.tensor([0, -1], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [block.diff_attention(q, k, v, lam, gamma=gamma, causal=True, status=status, stream=side) for _ in range(3)]
    with torch.cuda.stream(side):
        outs.append(block.diff_attention(q, k, v, lam, gamma=gamma, causal=True))
    outs.append(block.diff_attention(q, k, v, lam, gamma=gamma, causal=True, stream=side.cuda_stream))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs) and status.tolist() == [0, -1]


@pytest.mark.parametrize("q_len,kv_len", [(1, 5000), (200, 1000)])
def test_graph_capture(cuda, q_len, kv_len):
    q, k, v, lam, gamma = attn_inputs(1, q_len, kv_len, 2, 2, 64, torch.bfloat16)
    lens = torch.tensor([kv_len], dtype=torch.int32, device="cuda")
    run = lambda: block.diff_attention(q, k, v, lam, gamma=gamma, causal=True, kv_lens=lens)  # noqa: E731
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    lens.fill_(kv_len - 300)  # replays read the lengths of the day
    q.mul_(0.5)
    graph.replay()
    assert torch.equal(out, run())


def test_wrapper_refusals(cuda):
    q, k, v, lam, gamma = attn_inputs(2, 5, 8, 2, 2, 64, torch.bfloat16)
    for bad in (dict(q=q.float()), dict(k=k[:1]), dict(v=v[..., :64]), dict(lam=lam[:1]), dict(lam=lam.double()),
                dict(k=k.half()), dict(v=v.cpu()), dict(q=q.transpose(-1, -2).contiguous().transpose(-1, -2))):
        with pytest.raises((TypeError, ValueError)):
            block.diff_attention(**{**dict(q=q, k=k, v=v, lam=lam), **bad})
    with pytest.raises((TypeError, ValueError)):
        block.diff_attention(q, k, v, lam, kv_lens=torch.zeros(2, device="cuda"))
    with pytest.raises((TypeError, ValueError)):
        block.diff_attention(q, k, v, lam, key_mask=torch.zeros(2, 7, dtype=torch.bool, device="cuda"))
    with pytest.raises(_capi.KbError):
        block.diff_attention(q, k, v, lam, window=3)
    x = torch.zeros(4, 96, device="cuda")
    with pytest.raises(ValueError):
        block.norm_residual(x, x, post="rms", gate=x[:2], rows_per_cond=3, pre="batch")
    with pytest.raises(ValueError):
        block.norm_residual(x, x, gate=x[:3], rows_per_cond=2)
    with pytest.raises(ValueError):
        block.rope_axes(x.view(4, 3, 32), torch.zeros(1, 3, dtype=torch.int32, device="cuda"), torch.zeros(1, 16, 1, device="cuda"))


def test_status_word_is_checked(cuda):
    q, k, v, lam, _ = attn_inputs(1, 2, 8, 2, 2, 64, torch.bfloat16)
    word = lambda *a, **kw: torch.zeros(*a, device="cuda", **{"dtype": torch.int32, **kw})  # noqa: E731
    for status in (word(2, dtype=torch.float32), word(2, dtype=torch.int64), word(2, dtype=torch.int16), [0, 0], 5,
                   word(2).cpu(), word(1), word(0), word(()), word(4)[::2], word(2, 2)):
        with pytest.raises((TypeError, ValueError)):
            block.diff_attention(q, k, v, lam, status=status)
    ref = block.diff_attention(q, k, v, lam)
    for status in (None, word(2), word(2, dtype=torch.uint32), word(6)[2:5]):
        assert torch.equal(block.diff_attention(q, k, v, lam, status=status), ref)
        assert status is None or status.cpu().view(torch.int32).tolist() == [0] * len(status)


@pytest.mark.parametrize("width,ydt", [(256, torch.bfloat16), (1100, torch.float16), (9000, torch.bfloat16)])
@pytest.mark.parametrize("name", ["gate", "mod_scale", "mod_shift"])
def test_norm_output_in_place_of_a_condition_per_row(cuda, width, ydt, name):
    g = torch.Generator(device="cuda").manual_seed(width)
    x = torch.randn(700, width, generator=g, device="cuda")
    y, gate, ms, mt = (torch.randn(700, width, generator=g, device="cuda").to(ydt) for _ in range(4))
    cond = dict(gate=gate, mod_scale=ms, mod_shift=mt)
    kw = dict(post="rms", pre="layer", rows_per_cond=1)
    xo, h = block.norm_residual(x, y, **cond, **kw)
    xi, hi = block.norm_residual(x, y, **cond, h=cond[name], **kw)
    assert hi is cond[name] and torch.equal(xi, xo) and torch.equal(hi, h)
    with pytest.raises(_capi.KbError):
        block.norm_residual(x[:1], y[:1], pre="rms", pre_gamma=x[0], x_out=x[:1])


# batch, q_len, kv_len, heads, kv_heads, lens, mask: rows without keys through every end of both kernels (one block,
# a cluster, parts in the workspace; tiles of 128 queries with and without keys)
UNSEEN = [(2, 1, 40, 2, 2, [40, 0], None), (1, 3, 1000, 2, 2, [2], None), (2, 1, 60000, 1, 1, [60000, 0], None),
          (2, 200, 200, 2, 2, None, "empty"), (2, 300, 300, 2, 2, [20, 0], None), (1, 160, 6000, 1, 1, [90], None)]


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (32, torch.float16)])
@pytest.mark.parametrize("case", UNSEEN, ids=lambda c: "-".join(str(x) for x in c[:5]))
def test_queries_without_keys_are_zero_for_any_eps_and_gamma(cuda, d, dtype, case):
    batch, q_len, kv_len, heads, kv_heads, lens, mask = case
    q, k, v, lam, gamma = attn_inputs(batch, q_len, kv_len, heads, kv_heads, d, dtype, seed=q_len)
    kv_lens = None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")
    key_mask = make_mask(mask, batch, kv_len)
    see = visible(batch, q_len, kv_len, True, 0, kv_lens, key_mask)
    hidden = ~see.any(-1)
    assert hidden.any()
    kw = dict(causal=True, kv_lens=kv_lens, key_mask=key_mask, eps=0.0)
    got = block.diff_attention(q, k, v, lam, gamma=gamma, **kw)
    ref, bound = attn_ref(q, k, v, lam, gamma, see, 1.0, 0.0, d**-0.5)
    assert (got[hidden] == 0).all()
    seen = ~hidden
    close(got[seen], ref[seen], bound[seen])
    gamma[3] = float("inf")
    assert (block.diff_attention(q, k, v, lam, gamma=gamma, **kw)[hidden] == 0).all()


@pytest.mark.parametrize("d,dtype", [(64, torch.bfloat16), (32, torch.float16)])
@pytest.mark.parametrize("q_len,kv_len,lens,window", [
    (6, 4, [6, 4, 0], 0), (1, 300, [300, 301, 2**31 - 1], 0), (5, 1000, [1003, 1200, 40], 30), (1, 900, [930, 1500, 900], 700),
    (200, 150, [200, 230, 90], 0), (300, 400, [460, 700, 900], 350), (140, 5000, [5100, 9000, 77], 5000)])
def test_positions_of_sequences_longer_than_their_keys(cuda, d, dtype, q_len, kv_len, lens, window):
    q, k, v, lam, gamma = attn_inputs(3, q_len, kv_len, 2, 1, d, dtype, seed=q_len)
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    at = torch.arange(kv_len, device="cuda")
    pos = kv_lens.long()[:, None, None] - q_len + torch.arange(q_len, device="cuda")[:, None]
    see = (at <= pos) & (at < kv_lens[:, None, None])
    if window:
        see &= at > pos - window
    got = block.diff_attention(q, k, v, lam, gamma=gamma, eps=1e-4, causal=True, window=window, kv_lens=kv_lens)
    ref, bound = attn_ref(q, k, v, lam, gamma, see, 1.0, float(torch.tensor(1e-4)), d**-0.5)
    close(got, ref, bound)
    assert (got[~see.any(-1)] == 0).all()


@pytest.mark.parametrize("dtype,head_dim", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 20)])
@pytest.mark.parametrize("layout", ["pairs", "halves"])
@pytest.mark.parametrize("shared", [True, False])
def test_rope_shows_non_finite_frequencies(cuda, dtype, head_dim, layout, shared):
    pairs = head_dim // 2 - 2 if head_dim == 20 else head_dim // 4
    x, pos, freqs = rope_inputs(300, 5, head_dim, pairs, 2, 1 if shared else 3, dtype, 100, seed=6)
    clean = block.rope_axes(x, pos, freqs, rotary_heads=3, layout=layout)
    freqs[0, 1, 0], freqs[0, 4, 1], freqs[-1, 7, 0] = float("nan"), float("inf"), -float("inf")
    bad = torch.zeros(5, head_dim, dtype=torch.bool, device="cuda")
    for h, p in ((0, 1), (0, 4), (2, 7)) if not shared else [(h, p) for h in range(3) for p in (1, 4, 7)]:
        bad[h, [2 * p, 2 * p + 1] if layout == "pairs" else [p, p + pairs]] = True
    for out in (None, x):  # x last: in place
        got = block.rope_axes(x, pos, freqs, out, rotary_heads=3, layout=layout)
        assert torch.isnan(got[:, bad]).all() and torch.equal(got[:, ~bad], clean[:, ~bad])
    # a cache row that is skipped stays as it is
    y, pos, _ = rope_inputs(4, 5, head_dim, pairs, 2, 1, dtype, 100, seed=7)
    cache = torch.full((4, 5, head_dim), 3.0, dtype=dtype, device="cuda")
    block.rope_axes(y, pos, freqs, cache, rotary_heads=3, layout=layout, slots=torch.tensor([2, -1, 9, 0], device="cuda"))
    assert (cache[[1, 3]] == 3).all() and torch.isnan(cache[[0, 2]][:, bad]).all() and not torch.isnan(cache[:, ~bad]).any()


@pytest.mark.parametrize("kw", [dict(window=2**31), dict(window=-2**40), dict(window="wide"), dict(window=2.5), dict(scale=1e39),
                                dict(eps="small"), dict(out_scale=None), dict(key_mask=[True]), dict(k=None), dict(v=3),
                                dict(out=[0]), dict(gamma=2.0), dict(kv_lens=7)])
def test_attention_arguments_of_no_use_are_refused(cuda, kw):
    q, k, v, lam, _ = attn_inputs(2, 5, 8, 2, 2, 64, torch.bfloat16)
    with pytest.raises((TypeError, ValueError, _capi.KbError)):
        block.diff_attention(**{**dict(q=q, k=k, v=v, lam=lam, causal=True), **kw})


@pytest.mark.parametrize("kw", [dict(rows_per_cond=2**31), dict(rows_per_cond="all"), dict(eps=None),
                                dict(y=[1.0]), dict(x_out=3), dict(h="h"), dict(gate=1.0, rows_per_cond=4)])
def test_norm_arguments_of_no_use_are_refused(cuda, kw):
    x = torch.zeros(4, 96, device="cuda")
    with pytest.raises((TypeError, ValueError, _capi.KbError)):
        block.norm_residual(x, **{**dict(y=x, pre="rms"), **kw})


@pytest.mark.parametrize("kw", [dict(rotary_heads=2**32 + 1), dict(rotary_heads=2.0), dict(rotary_heads=-(2**32) + 2),
                                dict(freqs=None), dict(positions=[1]), dict(out=[0]), dict(slots=1, out=True)])
def test_rope_arguments_of_no_use_are_refused(cuda, kw):
    x, pos, freqs = rope_inputs(3, 2, 32, 16, 1, 1, torch.float32, 9)
    if kw.get("out") is True:
        kw = dict(kw, out=torch.empty_like(x))
    with pytest.raises((TypeError, ValueError, _capi.KbError)):
        block.rope_axes(**{**dict(x=x, positions=pos, freqs=freqs), **kw})


def test_streams_of_no_use_are_refused(cuda):
    q, k, v, lam, _ = attn_inputs(1, 2, 8, 2, 2, 64, torch.bfloat16)
    for stream in ("side", 1.5, q):
        with pytest.raises(TypeError):
            block.diff_attention(q, k, v, lam, stream=stream)
        with pytest.raises(TypeError):
            block.norm_residual(q[0, 0, 0], pre="rms", stream=stream, h=torch.empty_like(q[0, 0, 0]), x_out=False)


@pytest.mark.parametrize("limit_ns", [1, 3_000, 20_000])
@pytest.mark.parametrize("q_len,kv_len,heads,d,dtype", [
    (4096, 4096, 4, 64, torch.bfloat16), (4096, 4096, 4, 32, torch.float16), (256, 300_000, 2, 64, torch.float16)])
def test_waits_that_run_out_are_reported_and_leave_the_device_usable(cuda, limit_ns, q_len, kv_len, heads, d, dtype):
    q, k, v, lam, _ = attn_inputs(1, q_len, kv_len, heads, heads, d, dtype)
    ref = block.diff_attention(q, k, v, lam, causal=True)
    out = torch.empty_like(ref)
    desc = _capi.DiffAttentionDesc(
        dtype=block._DTYPES[dtype], batch=1, q_len=q_len, kv_len=kv_len, heads=heads, kv_heads=heads, head_dim=d, causal=1,
        scale=d**-0.5, out_scale=1.0, eps=1e-5, q_token=q.stride(1), q_head=q.stride(2), q_map=d, k_token=k.stride(1),
        k_head=k.stride(2), k_map=d, v_token=v.stride(1), v_head=v.stride(2), out_token=out.stride(1), out_head=out.stride(2))
    need = ctypes.c_size_t()
    _capi.call("kb_diff_attention_workspace", ctypes.byref(desc), ctypes.byref(need))
    work = torch.zeros(max(need.value, 1), dtype=torch.uint8, device="cuda")

    def run(limit):
        status = torch.tensor([0, -1], dtype=torch.int32, device="cuda")
        _capi.call("kb_test_diff_attention_wait_limit", ctypes.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                   lam.data_ptr(), out.data_ptr(), work.data_ptr(), need.value, limit, status.data_ptr(),
                   torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return status.tolist()

    assert run(limit_ns) == [_capi.STATUS_TIMEOUT, -1]  # items of 30 tiles and more take 60 us and more
    # shared and tensor memory of every SM are free again, nothing is in flight
    for _ in range(2):
        assert run(2_000_000_000) == [0, -1] and torch.equal(out, ref)
        assert torch.equal(block.diff_attention(q, k, v, lam, causal=True), ref)


def both_operators(g):
    """Calls of the rotary operator and of the norms on inputs of their own: run(stream) -> tensors."""
    x, pos, freqs = rope_inputs(500, 6, 64, 32, 3, 1, torch.bfloat16, 300, seed=21)
    s, y = (torch.randn(700, 768, generator=g, device="cuda") for _ in range(2))
    gate = torch.randn(70, 768, generator=g, device="cuda").bfloat16()

    def run(stream=None):
        return (block.rope_axes(x, pos, freqs, stream=stream),
                *block.norm_residual(s, y.bfloat16() if stream is None else yb, post="rms", pre="layer", gate=gate,
                                     rows_per_cond=10, stream=stream))

    yb = y.bfloat16()
    return run, (x, s, yb)


def test_rope_and_norms_repeat_on_any_stream_and_in_graphs(cuda):
    run, inputs = both_operators(torch.Generator(device="cuda").manual_seed(20))
    ref = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = [run(side), run(side.cuda_stream)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(torch.cuda.current_stream())
    graph.replay()
    for got in (*outs, captured):
        assert all(torch.equal(a, b) for a, b in zip(got, ref))
    for t in inputs:
        t.mul_(0.5)
    graph.replay()
    for a, b in zip(captured, run(torch.cuda.current_stream())):
        assert torch.equal(a, b)


def test_rope_and_norm_offsets_past_32_bits(cuda):
    step = (1 << 25) + 264
    room = torch.empty(160 * step, dtype=torch.bfloat16, device="cuda")
    x, pos, freqs = rope_inputs(160, 4, 64, 32, 2, 4, torch.bfloat16, 99, seed=22)
    far, to = (room.as_strided((160, 4, 64), (step, 64, 1), at) for at in (0, 256))
    far.copy_(x)
    ref = block.rope_axes(x, pos, freqs)
    assert torch.equal(block.rope_axes(far, pos, freqs), ref)
    assert torch.equal(block.rope_axes(x, pos, freqs, out=to), ref)
    slots = torch.arange(159, -1, -1, device="cuda")
    assert torch.equal(block.rope_axes(x, pos, freqs, out=to, slots=slots), ref.flip(0))
    kw = dict(post="rms", pre="layer", gate=x[:16].flatten(1), rows_per_cond=10)
    y = ref.flatten(1)
    fx, fy = (room.as_strided((160, 256), (step, 1), at) for at in (0, 1024))
    fy.copy_(y)
    a = block.norm_residual(x.flatten(1), y, **kw)
    b = block.norm_residual(fx, fy, x_out=room.as_strided((160, 256), (step, 1), 2048),
                            h=room.as_strided((160, 256), (step, 1), 4096), **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
