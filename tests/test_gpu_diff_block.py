"""GPU test of the differential-attention block: against the same block in 64 bits, and one token or board at a
time against all at once."""

import pytest
import torch

from rust_katago_b200 import diff_block

pytestmark = pytest.mark.gpu


def reference(net, x, positions, see):
    """The block in 64 bits from the bf16 weights and input; returns (x, h)."""
    batch, new, width = x.shape
    d, hq, hk = net.head_dim, net.heads, net.kv_heads

    def rms(v, gamma, eps):
        return v / (v.square().mean(-1, keepdim=True) + eps).sqrt() * gamma.double()

    def turn(v, freqs):
        ang = torch.einsum("at,hpa->thp", positions.double(), freqs.double()).view(batch, new, -1, d // 2)
        a, b = v[..., 0::2], v[..., 1::2]
        return torch.stack([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()], -1).flatten(-2)

    xd = x.double()
    heads = (rms(xd, net.pre_gamma, net.eps) @ net.wqkv.double().T).view(batch, new, -1, d)
    q = turn(heads[:, :, : 2 * hq], net.q_freqs).view(batch, new, hq, 2, d)
    k = turn(heads[:, :, 2 * hq : 2 * (hq + hk)], net.k_freqs).view(batch, new, hk, 2, d)
    v = heads[:, :, 2 * (hq + hk) :].reshape(batch, new, hk, 2 * d)
    k, v = k.repeat_interleave(hq // hk, 2), v.repeat_interleave(hq // hk, 2)
    logit = torch.einsum("bihmd,bjhmd->bhmij", q, k) * d**-0.5
    p = torch.softmax(logit.masked_fill(~see, float("-inf")), -1).nan_to_num()
    o = torch.einsum("bhmij,bjhe->bihme", p, v)
    o = o[..., 0, :] - net.lam.double()[:, None] * o[..., 1, :]
    a = rms(o, net.sub_gamma, 1e-5) * net.out_scale
    y = a.flatten(-2) @ net.wout.double().T
    out = xd + net.gate.double() * rms(y, net.post_gamma, net.eps)
    return out, rms(out, net.pre_gamma, net.eps)


def off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


# Seven roundings to bfloat16 (2^-8 at most, a third of that on average) lie between x and y, each of which passes on
# what came before at about its size: sqrt(7) 2^-8 in the norm of a result that the residual dominates.
BOUND = 7**0.5 * 2.0**-8


@pytest.mark.parametrize("heads,kv_heads,d,width", [(6, 6, 64, 768), (6, 2, 32, 384)])
def test_boards_against_64_bits(cuda, heads, kv_heads, d, width):
    batch, n = 3, 361
    net = diff_block.DiffBlock.random(width, heads, kv_heads, d, depth=2, seed=heads + d)
    x = torch.randn(batch, n, width, generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    pos = diff_block.board_positions(batch, 1)
    side = torch.tensor([19, 13, 9], device="cuda")[:, None]
    at = torch.arange(n, device="cuda")
    mask = (at // 19 < side) & (at % 19 < side)
    cache = diff_block.Cache(batch, n, kv_heads, d)
    out, h = net(x, pos, cache, key_mask=mask, causal=False)
    ref, ref_h = reference(net, x, pos, mask[:, None, None, None, :])
    assert off(out, ref) <= BOUND and off(h, ref_h) <= BOUND
    assert cache.lens.tolist() == [n] * batch


def test_pieces_follow_the_whole(cuda):
    batch, width, n = 2, 768, 2 * 361 + 3
    net = diff_block.DiffBlock.random(width, 6, 2, 64, seed=5)
    x = torch.randn(batch, n, width, generator=torch.Generator("cuda").manual_seed(2), device="cuda").bfloat16()
    pos = diff_block.board_positions(1, 3)[:, :n].repeat(1, batch).contiguous()
    see = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
    ref, _ = reference(net, x, pos, see)
    whole, _ = net(x, pos, diff_block.Cache(batch, n, 2, 64))
    assert off(whole, ref) <= BOUND
    cache = diff_block.Cache(batch, n, 2, 64)
    outs, at = [], 0
    for new in (361, 361, 1, 1, 1):  # two boards, then token by token
        p = pos.view(3, batch, n)[:, :, at : at + new].reshape(3, -1).contiguous()
        outs.append(net(x[:, at : at + new].contiguous(), p, cache)[0])
        at += new
    assert off(torch.cat(outs, 1), ref) <= BOUND
    assert cache.lens.tolist() == [n] * batch


def test_full_cache_drops_further_tokens(cuda):
    net = diff_block.DiffBlock.random(384, 6, 6, 32, seed=7)
    cache = diff_block.Cache(1, 4, 6, 32)
    x = torch.randn(1, 6, 384, device="cuda").bfloat16()
    out, _ = net(x, torch.zeros(3, 6, dtype=torch.int32, device="cuda"), cache)
    assert torch.isfinite(out).all() and cache.slots(1).tolist() == [-1]


def test_tokens_that_do_not_fit_leave_the_others_right(cuda):
    width, d, capacity, n = 384, 32, 5, 9
    net = diff_block.DiffBlock.random(width, 6, 6, d, seed=8)
    x = torch.randn(2, n, width, generator=torch.Generator("cuda").manual_seed(3), device="cuda").bfloat16()
    pos = diff_block.board_positions(1, 1)[:, :n].repeat(1, 2).contiguous()
    at = torch.arange(n, device="cuda")
    ref, _ = reference(net, x, pos, (at <= at[:, None]) & (at < capacity))  # tokens past the capacity see all that fitted
    for pieces in ((9,), (3, 4, 1, 1), (5, 1, 3)):
        cache = diff_block.Cache(2, capacity, 6, d)
        outs, first = [], 0
        for new in pieces:
            p = pos.view(3, 2, n)[:, :, first : first + new].reshape(3, -1).contiguous()
            outs.append(net(x[:, first : first + new].contiguous(), p, cache)[0])
            first += new
        got = torch.cat(outs, 1)
        for i in range(n):
            assert off(got[:, i], ref[:, i]) <= BOUND, (pieces, i)
        assert cache.lens.tolist() == [n, n]


@pytest.mark.parametrize("batch,new", [(2, 0), (0, 3), (0, 0)])
def test_calls_without_tokens_do_nothing(cuda, batch, new):
    net = diff_block.DiffBlock.random(384, 6, 2, 32, seed=9)
    cache = diff_block.Cache(batch, 8, 2, 32)
    x = torch.zeros(batch, new, 384, dtype=torch.bfloat16, device="cuda")
    out, h = net(x, torch.zeros(3, batch * new, dtype=torch.int32, device="cuda"), cache)
    assert out.shape == h.shape == (batch, new, 384) and cache.lens.tolist() == [0] * batch


def test_kernels_that_do_not_finish_show(cuda, monkeypatch):
    net = diff_block.DiffBlock.random(384, 6, 6, 32, seed=10)
    seen = []
    attention = diff_block.block.diff_attention
    monkeypatch.setattr(diff_block.block, "diff_attention", lambda *a, **kw: seen.append(kw["status"]) or attention(*a, **kw))
    net(torch.zeros(1, 2, 384, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 2, dtype=torch.int32, device="cuda"),
        diff_block.Cache(1, 4, 6, 32))
    assert seen[0] is net.status and net.status.tolist() == [0, -1]
    net.check()
    net.status[0] = 32  # what a kernel leaves that gave up a wait
    with pytest.raises(RuntimeError):
        net.check()
