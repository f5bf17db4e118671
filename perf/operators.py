"""Cases of the block operators: multi-axis rotary positions, differential attention
and the norms around a block, each as its plain form (elementary torch operations in
32 bits) and through the framework's entry points (``rust_katago_b200.block``)."""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
BOARD = 19
BOARD_TOKENS = BOARD * BOARD


# ------------------------------------------------------------------ the cases
def _rope(name, tokens, heads, rotary_heads, head_dim, pairs, axes, freq_heads, layout, dtype, span):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "rotary_heads": rotary_heads,
            "head_dim": head_dim, "pairs": pairs, "axes": axes, "freq_heads": freq_heads, "layout": layout,
            "dtype": dtype, "span": span}


def _attn(name, batch, q_len, kv_len, heads, kv_heads, head_dim, dtype, causal=False, window=0, ragged=False,
          boards=False):
    return {"name": name, "op": "attn", "batch": batch, "q_len": q_len, "kv_len": kv_len, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype, "causal": causal, "window": window,
            "ragged": ragged, "boards": boards}


def _norm(name, rows, width, kind, stream, branch, gate_act, rows_per_cond):
    return {"name": name, "op": "norm", "rows": rows, "width": width, "kind": kind, "stream": stream,
            "branch": branch, "gate_act": gate_act, "rows_per_cond": rows_per_cond}


def listed():
    return [
        # One token of one sequence, queries and keys of 12 heads of 64, on its way into a step of decoding: latency.
        _rope("rope_one_token", 1, 36, 24, 64, 32, 3, 1, "halves", "bf16", 4096),
        # 256 positions of 361 points: the trunk's own learned row and column frequencies per head and pair.
        _rope("rope_boards_256", 256 * BOARD_TOKENS, 36, 24, 64, 32, 2, 24, "pairs", "bf16", BOARD),
        # A long history of boards (time, row, column), narrow heads, a 32-bit stream, an odd number of tokens.
        _rope("rope_history_f32", 91 * BOARD_TOKENS - 6, 12, 12, 32, 16, 3, 1, "halves", "f32", 91),
        # One position: the latency of a search that evaluates leaf by leaf.
        _attn("attn_board_1", 1, BOARD_TOKENS, BOARD_TOKENS, 6, 6, 64, "bf16"),
        # 64 positions of several board sizes in 19 x 19 frames, points off the board hidden; the narrow heads.
        _attn("attn_boards_64", 64, BOARD_TOKENS, BOARD_TOKENS, 6, 6, 32, "f16", boards=True),
        # A prompt: every token sees those before it; grouped key and value heads.
        _attn("attn_prompt_8192", 1, 8192, 8192, 12, 4, 64, "bf16", causal=True),
        # One new board appended to caches of different lengths.
        _attn("attn_chunk_on_cache", 3, BOARD_TOKENS, 16001, 6, 6, 64, "bf16", causal=True, ragged=True),
        # One token on a cache of three boards: latency.
        _attn("attn_token_short", 1, 1, 3 * BOARD_TOKENS, 6, 6, 64, "bf16", causal=True),
        # Serving: one token each of 64 sequences on long caches of different lengths.
        _attn("attn_tokens_64", 64, 1, 8192, 12, 4, 64, "bf16", causal=True, ragged=True),
        # One token: latency.
        _norm("norm_one_token", 1, 768, "rms", "bf16", "bf16", "none", 1),
        # 256 positions at the trunk's width, a bf16 stream, a gate per position.
        _norm("norm_boards_256", 256 * BOARD_TOKENS, 768, "rms", "bf16", "bf16", "linear", BOARD_TOKENS),
        # A wider model with layer norms, a 32-bit stream and gates and modulations per sequence; odd row count.
        _norm("norm_wide_f32", 8191, 5120, "layer", "f32", "bf16", "tanh", 1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "norm"])
    if op == "rope":
        head_dim = rng.choice([32, 64, 128])
        pairs = rng.choice([head_dim // 2, head_dim // 2, head_dim // 4])
        dtype = rng.choice(["bf16", "f16", "f32"])
        heads = rng.randint(1, 36)
        rotary = rng.randint((heads + 1) // 2, heads)
        tokens = _log(rng, 1, min(90000, 200_000_000 // (heads * head_dim * BYTES[dtype])))
        span = _log(rng, 16, 256) if dtype == "f32" else _log(rng, 16, 30000)
        return _rope("drawn", tokens, heads, rotary, head_dim, pairs, rng.randint(1, 4), rng.choice([1, rotary]),
                     rng.choice(["pairs", "halves"]), dtype, span)
    if op == "norm":
        width = _log(rng, 64, 8192)
        width -= width % rng.choice([1, 8, 64])
        stream = rng.choice(["bf16", "f16", "f32"])
        rows = _log(rng, 1, 28_000_000 // width)
        return _norm("drawn", rows, width, rng.choice(["rms", "layer"]), stream,
                     stream if stream != "f32" else rng.choice(["bf16", "f16", "f32"]),
                     rng.choice(["none", "linear", "sigmoid", "tanh"]), rng.choice([1, rng.randint(2, 500), rows]))
    head_dim, dtype = rng.choice([32, 64]), rng.choice(["bf16", "f16"])
    kv_heads = rng.choice([1, 2, 3, 4, 6])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4])
    kind = rng.choice(["boards", "prompt", "chunk", "token"])
    if kind == "boards":
        return _attn("drawn", _log(rng, 1, 64), BOARD_TOKENS, BOARD_TOKENS, kv_heads, kv_heads, head_dim, dtype,
                     boards=rng.random() < 0.7)
    if kind == "prompt":
        length = _log(rng, 65, min(6000, int(8000 / math.sqrt(heads / 12))))
        return _attn("drawn", 1, length, length, heads, kv_heads, head_dim, dtype, causal=True,
                     window=rng.choice([0, 0, length // 3 + 1]))
    batch = _log(rng, 1, 4) if kind == "chunk" else _log(rng, 1, 48)
    most = 64 * 8192 * 4 // (batch * kv_heads)
    if kind == "chunk":
        q_len = _log(rng, 2, 512)
        kv_len = max(q_len, _log(rng, 128, min(most, 16000)))
    else:
        q_len, kv_len = 1, _log(rng, 2, min(most, 30000))
    window = rng.choice([0, 0, _log(rng, 16, 4096)])
    return _attn("drawn", batch, q_len, kv_len, heads, kv_heads, head_dim, dtype, causal=True, window=window,
                 ragged=rng.random() < 0.5)


# ------------------------------------------------------------------ what a case fixes besides its sizes
def _lens(case):
    """Keys of each sequence: all, or lengths spread over the upper half of the cache."""
    b, n = case["batch"], case["kv_len"]
    return [n - (i * 1009 % (n // 2 + 1)) if case["ragged"] else n for i in range(b)]


def _sides(case):
    return [(19, 13, 9, 19)[i % 4] if case["boards"] else 0 for i in range(case["batch"])]


def _visible_pairs(case):
    """(query, key) pairs that the masks leave, over the batch, and keys read."""
    pairs = keys = 0
    for n, side in zip(_lens(case), _sides(case)):
        q = case["q_len"]
        if side:
            n = side * side
        if not case["causal"]:
            pairs, keys = pairs + q * n, keys + n
            continue
        first, w = n - q, case["window"]
        seen = [max(0, p + 1 - (max(0, p + 1 - w) if w else 0)) for p in range(first, n)]
        pairs += sum(seen)
        keys += min(n, w + q - 1) if w else n
    return pairs, keys


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["head_dim"]
        small = case["tokens"] * case["axes"] * 4 + case["freq_heads"] * case["pairs"] * case["axes"] * 4
        return {"bytes": 2 * n * BYTES[case["dtype"]] + small, "flops": 6 * case["tokens"] * case["rotary_heads"] * case["pairs"]}
    if case["op"] == "norm":
        n, s, b = case["rows"] * case["width"], BYTES[case["stream"]], BYTES[case["branch"]]
        cond = -(-case["rows"] // case["rows_per_cond"]) * case["width"] * 3 * b if case["gate_act"] != "none" else 0
        return {"bytes": n * (2 * s + 2 * b) + cond, "flops": 14 * n}
    d, e = case["head_dim"], BYTES[case["dtype"]]
    pairs, keys = _visible_pairs(case)
    rows = case["batch"] * case["q_len"]
    return {"bytes": keys * case["kv_heads"] * 4 * d * e + rows * case["heads"] * 4 * d * e,
            "flops": pairs * case["heads"] * 12 * d}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = dict(case)
    if case["op"] == "rope":
        t, axes, pairs = case["tokens"], case["axes"], case["pairs"]
        s["x"] = normal(t, case["heads"], case["head_dim"], dtype=DTYPES[case["dtype"]])
        s["positions"] = torch.randint(0, case["span"], (axes, t), generator=g, device="cuda", dtype=torch.int32)
        # A geometric ladder of frequencies, dealt out to the axes, with learned deviations.
        ladder = 10000.0 ** (-torch.arange(pairs, device="cuda") / pairs)
        own_axis = torch.arange(pairs, device="cuda")[:, None] % axes == torch.arange(axes, device="cuda")
        s["freqs"] = (ladder[:, None] * (own_axis + 0.1 * normal(case["freq_heads"], pairs, axes))).contiguous()
        return s
    if case["op"] == "norm":
        n, c, b = case["rows"], case["width"], DTYPES[case["branch"]]
        s["x"] = normal(n, c, std=2.0, dtype=DTYPES[case["stream"]])
        s["y"] = normal(n, c, std=0.5, mean=0.1, dtype=b)
        s["post_gamma"], s["pre_gamma"] = normal(c, std=0.1, mean=0.3), normal(c, std=0.1, mean=1.0)
        layer = case["kind"] == "layer"
        s["post_beta"], s["pre_beta"] = (normal(c, std=0.02), normal(c, std=0.02)) if layer else (None, None)
        s["gate"] = s["mod_scale"] = s["mod_shift"] = None
        if case["gate_act"] != "none":
            m = -(-n // case["rows_per_cond"])
            s["gate"], s["mod_scale"], s["mod_shift"] = (normal(m, c, std=0.3, dtype=b) for _ in range(3))
        s["res_scale"], s["branch_scale"], s["eps"] = 0.9, 1.1, 1e-6
        return s
    dt, d, b = DTYPES[case["dtype"]], case["head_dim"], case["batch"]
    # Logits of standard deviation 2 (trained maps are peaked), keys and values side by side in one cache row.
    s["q"] = normal(b, case["q_len"], case["heads"], 2, d, std=2.0, dtype=dt)
    cache = normal(b, case["kv_len"], 2, case["kv_heads"] * 2 * d, dtype=dt)
    s["k"] = cache[:, :, 0].unflatten(-1, (case["kv_heads"], 2, d))
    s["v"] = cache[:, :, 1].unflatten(-1, (case["kv_heads"], 2 * d))
    s["lam"] = torch.rand(case["heads"], generator=g, device="cuda") * 0.6 + 0.2
    s["gamma"] = normal(2 * d, std=0.1, mean=1.0)
    s["out_scale"], s["eps"], s["scale"] = 0.4, 1e-5, d**-0.5
    s["kv_lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
    s["key_mask"] = None
    if case["boards"]:
        side = torch.tensor(_sides(case), device="cuda")[:, None]
        at = torch.arange(case["kv_len"], device="cuda")
        s["key_mask"] = (at // BOARD < side) & (at % BOARD < side)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_rope(s):
    x = s["x"].float()
    r, pairs = s["rotary_heads"], s["pairs"]
    angle = (s["positions"].float().T[:, None, None, :] * s["freqs"][None]).sum(-1)  # [tokens, freq heads, pairs]
    c, n = torch.cos(angle), torch.sin(angle)
    out = x.clone()
    if s["layout"] == "pairs":
        lo, hi = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
    else:
        lo, hi = slice(0, pairs), slice(pairs, 2 * pairs)
    a, b = x[:, :r, lo], x[:, :r, hi]
    out[:, :r, lo] = a * c - b * n
    out[:, :r, hi] = a * n + b * c
    return out.to(s["x"].dtype)


def _plain_normed(v, kind, gamma, beta, eps):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + eps) * gamma
    return v if beta is None else v + beta


def _plain_norm(s):
    n = _plain_normed(s["y"].float(), s["kind"], s["post_gamma"], s["post_beta"], s["eps"])
    modulated = s["gate"] is not None
    if modulated:
        row = torch.arange(s["x"].shape[0], device="cuda") // s["rows_per_cond"]
        gate = s["gate"].float()[row]
        act = s["gate_act"]
        n = n * (torch.sigmoid(gate) if act == "sigmoid" else torch.tanh(gate) if act == "tanh" else gate)
    r = s["res_scale"] * s["x"].float() + s["branch_scale"] * n
    h = _plain_normed(r, s["kind"], s["pre_gamma"], s["pre_beta"], s["eps"])
    if modulated:
        h = h * (1 + s["mod_scale"].float()[row]) + s["mod_shift"].float()[row]
    return r.to(s["x"].dtype), h.to(s["y"].dtype)


def _plain_attention(s):
    b, q_len, heads, _, d = s["q"].shape
    kv_len, kv_heads = s["k"].shape[1:3]
    g = heads // kv_heads
    q = s["q"].float().reshape(b, q_len, kv_heads, g, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b, kv_heads, 2, g * q_len, d)
    k = s["k"].float().permute(0, 2, 3, 4, 1)
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    score = (q @ k).mul_(s["scale"]).reshape(b, kv_heads, 2, g, q_len, kv_len)
    hidden = _hidden(s, b, q_len, kv_len)
    if hidden is not None:
        score.masked_fill_(hidden[:, None, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1.0, total)).reshape(b, kv_heads, 2, g * q_len, kv_len)
    o = (p @ v).reshape(b, kv_heads, 2, g, q_len, 2 * d)
    o = o[:, :, 0] - s["lam"].reshape(kv_heads, g, 1, 1) * o[:, :, 1]
    o = o * torch.rsqrt((o * o).mean(-1, keepdim=True) + s["eps"]) * s["gamma"] * s["out_scale"]
    return o.permute(0, 3, 1, 2, 4).reshape(b, q_len, heads, 2 * d).to(s["q"].dtype)


def _hidden(s, b, q_len, kv_len):
    """[batch, q_len or 1, kv_len]: keys that a query does not see; None where it sees all."""
    at = torch.arange(kv_len, device="cuda")
    hidden = None
    if s["kv_lens"] is not None:
        hidden = (at >= s["kv_lens"][:, None])[:, None]
    if s["key_mask"] is not None:
        off = ~s["key_mask"][:, None]
        hidden = off if hidden is None else hidden | off
    if s["causal"]:
        n = s["kv_lens"] if s["kv_lens"] is not None else torch.full((b,), kv_len, device="cuda")
        pos = n[:, None, None] - q_len + torch.arange(q_len, device="cuda")[:, None]
        off = at > pos
        if s["window"]:
            off = off | (at <= pos - s["window"])
        hidden = off if hidden is None else hidden | off
    return hidden


def run(state):
    s = state
    if own:
        from rust_katago_b200 import block

        if s["op"] == "rope":
            return block.rope_axes(s["x"], s["positions"], s["freqs"], rotary_heads=s["rotary_heads"], layout=s["layout"])
        if s["op"] == "norm":
            return block.norm_residual(
                s["x"], s["y"], post=s["kind"], pre=s["kind"], post_gamma=s["post_gamma"], post_beta=s["post_beta"],
                pre_gamma=s["pre_gamma"], pre_beta=s["pre_beta"], gate=s["gate"], gate_act="linear" if s["gate"] is None else s["gate_act"],
                mod_scale=s["mod_scale"], mod_shift=s["mod_shift"], rows_per_cond=s["rows_per_cond"],
                res_scale=s["res_scale"], branch_scale=s["branch_scale"], eps=s["eps"])
        return block.diff_attention(
            s["q"], s["k"], s["v"], s["lam"], gamma=s["gamma"], out_scale=s["out_scale"], eps=s["eps"],
            scale=s["scale"], causal=s["causal"], window=s["window"], kv_lens=s["kv_lens"], key_mask=s["key_mask"])
    if s["op"] == "rope":
        return _plain_rope(s)
    if s["op"] == "norm":
        return _plain_norm(s)
    return _plain_attention(s)


# ------------------------------------------------------------------ the definitions in 64 bits
def _exact_norm_row(v, layer, gamma, beta, eps):
    if layer:
        root = (v.var(-1, correction=0, keepdim=True) + eps).sqrt()
        v = v - v.mean(-1, keepdim=True)
    else:
        root = (v.square().sum(-1, keepdim=True) / v.shape[-1] + eps).sqrt()
    v = v / root * gamma.double()
    return v if beta is None else v + beta.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        x, p, r = s["x"].double(), case["pairs"], case["rotary_heads"]
        turn = torch.einsum("at,hpa->thp", s["positions"].double(), s["freqs"].double())
        turn = torch.polar(torch.ones_like(turn), turn)
        part = x[:, :r, : 2 * p]
        if case["layout"] == "pairs":
            z = torch.view_as_complex(part.unflatten(-1, (p, 2)).contiguous()) * turn
            part = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(part[..., :p].contiguous(), part[..., p:].contiguous()) * turn
            part = torch.cat([z.real, z.imag], -1)
        return torch.cat([torch.cat([part, x[:, :r, 2 * p :]], -1), x[:, r:]], 1)
    if case["op"] == "norm":
        rs, hs, n, per = [], [], case["rows"], case["rows_per_cond"]
        for at in range(0, n, 8192):
            rows = slice(at, min(n, at + 8192))
            y = _exact_norm_row(s["y"][rows].double(), case["kind"] == "layer", s["post_gamma"], s["post_beta"], s["eps"])
            cond = None
            if s["gate"] is not None:
                cond = [c[torch.arange(rows.start, rows.stop, device="cuda") // per].double()
                        for c in (s["gate"], s["mod_scale"], s["mod_shift"])]
                y = y * {"linear": lambda u: u, "sigmoid": lambda u: 1 / (1 + torch.exp(-u)), "tanh": torch.tanh}[
                    case["gate_act"]](cond[0])
            r = s["x"][rows].double() * s["res_scale"] + y * s["branch_scale"]
            h = _exact_norm_row(r, case["kind"] == "layer", s["pre_gamma"], s["pre_beta"], s["eps"])
            rs.append(r)
            hs.append(h if cond is None else torch.addcmul(cond[2], h, 1 + cond[1]))
        return torch.cat(rs), torch.cat(hs)
    q_len, heads, d = case["q_len"], case["heads"], case["head_dim"]
    out = torch.zeros(case["batch"], q_len, heads, 2 * d, dtype=torch.float64, device="cuda")
    share = heads // case["kv_heads"]
    for b, (n, side) in enumerate(zip(_lens(case), _sides(case))):
        key = torch.arange(n, device="cuda")
        if side:
            key = key[(key // BOARD < side) & (key % BOARD < side)]
        see = None
        if case["causal"]:
            ahead = (n - q_len + torch.arange(q_len, device="cuda"))[:, None] - key
            see = ahead >= 0
            if case["window"]:
                see &= ahead < case["window"]
        for h in range(heads):
            maps = []
            for m in (0, 1):
                logit = s["q"][b, :, h, m].double() @ s["k"][b, key, h // share, m].double().T * s["scale"]
                if see is not None:
                    logit = torch.where(see, logit, -torch.inf)
                maps.append(torch.nan_to_num(torch.softmax(logit, -1)))
            o = (maps[0] - s["lam"][h].double() * maps[1]) @ s["v"][b, key, h // share].double()
            size = (o.square().mean(-1, keepdim=True) + s["eps"]).sqrt()
            out[b, :, h] = o / size * s["gamma"].double() * s["out_scale"]
    return out
