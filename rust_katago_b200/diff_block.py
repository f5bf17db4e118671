"""A differential-attention block over boards and their history, on the library's operators.

The attention half of a trunk block in the form that differential transformers
give it, for tokens that are the points of one board or of a sequence of boards:

    h = pre_norm(x)                                       kb_norm_residual
    q, k, v = h Wqkv^T                                    kb_bf16_linear
    q, k rotated by (time, row, column)                   kb_rope_axes, K and V straight into the cache
    a = differential attention of q over the cache        kb_diff_attention
    y = a Wout^T                                          kb_bf16_linear
    x = x + gate * post_norm(y); h = next pre_norm(x)     kb_norm_residual

One call takes any number of new tokens per sequence: whole boards, a board
appended to a history, or one token.  ``python -m rust_katago_b200.diff_block``
evaluates a few boards with random weights, then steps token by token.
"""

from __future__ import annotations

import numpy as np
import torch

from . import _capi, block, int8

BOARD = 19


class Cache:
    """Rotated keys and the values of `batch` sequences, `capacity` tokens each: one row per token, [K | V].

    lens counts the tokens that every sequence has had.  Those past the capacity get no row: they see the tokens
    that have one and are seen by none.
    """

    def __init__(self, batch: int, capacity: int, kv_heads: int, head_dim: int):
        self.batch, self.capacity = batch, capacity
        self.rows = torch.zeros(batch * capacity, 4 * kv_heads, head_dim, dtype=torch.bfloat16, device="cuda")
        self.lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
        split = self.rows.view(batch, capacity, 2, 2 * kv_heads, head_dim)
        self.k = split[:, :, 0].unflatten(2, (kv_heads, 2))
        self.v = split[:, :, 1].unflatten(2, (kv_heads, 2)).flatten(-2)

    def slots(self, new: int) -> torch.Tensor:
        """Cache rows of the next `new` tokens of every sequence (past the capacity: none), [batch * new]."""
        at = self.lens.long()[:, None] + torch.arange(new, device="cuda")
        base = torch.arange(self.batch, device="cuda")[:, None] * self.capacity
        return torch.where(at < self.capacity, base + at, -1).flatten()


class DiffBlock:
    """One block's weights: bf16 wqkv [(2 heads + 4 kv_heads) * d, width] ([Q | K | V], a head's two maps side by
    side, values 2 d wide), wout [width, heads * 2 d]; fp32 freqs [2 heads + 2 kv_heads, d / 2, axes], lam [heads],
    sub_gamma [2 d], pre_gamma, post_gamma [width]; bf16 gate [1, width].

    status (int32 [flags, first_layer], on the device) is sticky: a flag says that a kernel of some call gave up a wait
    and that its results are partial.  :meth:`check` reads it."""

    def __init__(self, heads: int, kv_heads: int, wqkv, wout, freqs, lam, sub_gamma, pre_gamma, post_gamma, gate,
                 lambda_init: float, eps: float = 1e-6):
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, sub_gamma.shape[0] // 2
        self.width = wqkv.shape[1]
        self.wqkv, self.wout, self.lam, self.sub_gamma = wqkv, wout, lam, sub_gamma
        self.q_freqs, self.k_freqs = freqs[: 2 * heads].contiguous(), freqs[2 * heads:].contiguous()
        self.pre_gamma, self.post_gamma, self.gate = pre_gamma, post_gamma, gate
        self.out_scale, self.eps = 1.0 - lambda_init, eps
        self.status = torch.tensor([0, -1], dtype=torch.int32, device=wqkv.device)

    def check(self) -> None:
        """Raise RuntimeError if a kernel of an earlier call gave up a wait (waits for the calls on the current stream)."""
        if flags := int(self.status[0]):
            raise RuntimeError(f"a kernel of the block did not finish (status flags {flags})")

    @classmethod
    def random(cls, width: int, heads: int, kv_heads: int, head_dim: int, axes: int = 3, depth: int = 0, seed: int = 0):
        """Random weights in the manner of an initialised network."""
        g = torch.Generator().manual_seed(seed)

        def normal(*shape, std, mean=0.0):
            return (torch.randn(*shape, generator=g) * std + mean).cuda()

        lambda_init = 0.8 - 0.6 * float(np.exp(-0.3 * depth))
        vectors = [0.1 * torch.randn(heads, head_dim, generator=g).numpy() for _ in range(4)]
        lam = torch.from_numpy(block.diff_lambda(*vectors, lambda_init)).cuda()
        std = width**-0.5
        return cls(
            heads, kv_heads, normal((2 * heads + 4 * kv_heads) * head_dim, width, std=2 * std).bfloat16(),
            normal(width, heads * 2 * head_dim, std=std).bfloat16(),
            normal(2 * (heads + kv_heads), head_dim // 2, axes, std=0.3), lam, normal(2 * head_dim, std=0.1, mean=1.0),
            normal(width, std=0.1, mean=1.0), normal(width, std=0.1, mean=1.0),
            normal(1, width, std=0.3).bfloat16(), lambda_init)

    def __call__(self, x, positions, cache: Cache, key_mask=None, causal: bool = True, next_gamma=None):
        """x bf16 [batch, new, width] and int32 positions [axes, batch * new] of the tokens that follow what the
        cache holds.  Returns (x, h): the residual stream after the block and its norm by `next_gamma` (the next
        block's pre-norm, default this one's).  key_mask [batch, capacity] hides cache rows (points off a smaller
        board); causal lets a token see only itself and what came before."""
        batch, new, width = x.shape
        rows, d = batch * new, self.head_dim
        if rows == 0:
            return x.clone(), x.clone()
        flat = x.reshape(rows, width)
        _, h = block.norm_residual(flat, pre="rms", pre_gamma=self.pre_gamma, eps=self.eps, x_out=False)
        qkv = self._linear(h, self.wqkv)
        heads = qkv.view(rows, -1, d)
        q = block.rope_axes(heads[:, : 2 * self.heads], positions, self.q_freqs)
        block.rope_axes(heads[:, 2 * self.heads:], positions, self.k_freqs, rotary_heads=2 * self.kv_heads,
                        out=cache.rows, slots=cache.slots(new))
        cache.lens += new
        a = block.diff_attention(q.view(batch, new, self.heads, 2, d), cache.k, cache.v, self.lam, gamma=self.sub_gamma,
                                 out_scale=self.out_scale, causal=causal, kv_lens=cache.lens, key_mask=key_mask,
                                 status=self.status)
        y = self._linear(a.view(rows, -1), self.wout)
        out, h = block.norm_residual(
            flat, y, post="rms", post_gamma=self.post_gamma, gate=self.gate, rows_per_cond=rows, pre="rms",
            pre_gamma=self.pre_gamma if next_gamma is None else next_gamma, eps=self.eps)
        return out.view(batch, new, width), h.view(batch, new, width)

    @staticmethod
    def _linear(a, w):
        m, k, n = a.shape[0], a.shape[1], w.shape[0]
        out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
        int8.bf16_linear(a, w, None, m, n, k, _capi.EPI_16, out, n)
        return out


def board_positions(batch: int, boards: int, first: int = 0) -> torch.Tensor:
    """(time, row, column) of the points of `boards` boards of every sequence, int32 [3, batch * boards * 361]."""
    t, r, c = torch.meshgrid(torch.arange(first, first + boards), torch.arange(BOARD), torch.arange(BOARD), indexing="ij")
    one = torch.stack([t.flatten(), r.flatten(), c.flatten()])
    return one.repeat(1, batch).int().cuda()


def main() -> None:
    batch, boards = 4, 2
    new = boards * BOARD * BOARD
    net = DiffBlock.random(768, 6, 6, 64)
    cache = Cache(batch, new + 8, 6, 64)
    x, _ = net(torch.randn(batch, new, 768, device="cuda").bfloat16(), board_positions(batch, boards), cache)
    print(f"{boards} boards of {batch} games: {tuple(x.shape)}, cache at {cache.lens.tolist()}")
    for step in range(4):
        pos = torch.tensor([[boards], [0], [step]], dtype=torch.int32, device="cuda").repeat(1, batch)
        x, _ = net(torch.randn(batch, 1, 768, device="cuda").bfloat16(), pos, cache)
    net.check()
    print(f"one token at a time: {tuple(x.shape)}, cache at {cache.lens.tolist()}, mean square {x.float().square().mean():.3f}")


if __name__ == "__main__":
    main()
