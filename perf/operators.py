"""Measured calls of the operators around a key/value cache held in 4 or 8 bits.

Three operators of a decoder's attention block, in the order a block runs them:

- "rope": rotary positions with several axes (time, height, width, one more) over the heads of q or
  k, ggml's modes MROPE (sections of pairs, one axis each), VISION (sections that restart the
  frequencies, the whole head rotated) and IMROPE (axes interleaved pair by pair);
- "cache": f32 rows quantised into Q4_0 / Q8_0 rows of a cache at given indices as they are written,
  then rows of that cache read back to f32 at other indices (a window that covers new and old rows);
- "attn": attention of q over a Q4_0 cache, grouped heads, additive f16 mask, from one token a
  sequence to long prompts.

Every case's sizes are a Llama-3-8B layer's (32 query heads, 8 key/value heads, head size 128, 1024
values a cache row, 512-token ubatches) or generic odd ones.
"""
import math
import os
import sys

import torch

own = False

MROPE, VISION, IMROPE = 8, 24, 40          # ggml's rope modes with sections
Q4_0, Q8_0 = 2, 8                          # ggml's type numbers
BLOCK_BYTES = {Q4_0: 18, Q8_0: 34}         # a block of 32 values: f16 scale, then the codes
NEG = float("-inf")


def _lib():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ggml-rocket_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ggml_b200
    return ggml_b200


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFFFFFF)
    return g


# ---- the cases ---------------------------------------------------------------------------------------


def listed():
    return [
        # the next token of eight sequences: q of every head, one launch of a few microseconds
        {"name": "rope_next_tokens", "op": "rope", "mode": MROPE, "tokens": 8, "heads": 32, "dim": 128, "f16": False},
        # q of a long prompt of text and images
        {"name": "rope_prompt", "op": "rope", "mode": IMROPE, "tokens": 4096, "heads": 32, "dim": 128, "f16": False},
        # the patches of one picture (73 x 73) in a vision tower, an odd head size, half precision
        {"name": "rope_picture", "op": "rope", "mode": VISION, "tokens": 5329, "heads": 16, "dim": 80, "f16": True},
        # one new token's K row into the cache, and a small window of the cache read
        {"name": "cache_token", "op": "cache", "kind": Q4_0, "width": 1024, "rows": 8192, "write": 1, "read": 64},
        # a 512-token ubatch written, and a window of 4096 rows read back
        {"name": "cache_ubatch", "op": "cache", "kind": Q4_0, "width": 1024, "rows": 16384, "write": 512, "read": 4096},
        # many sequences' rows scattered over a long cache, odd counts, 8 bits
        {"name": "cache_scattered", "op": "cache", "kind": Q8_0, "width": 1024, "rows": 40000, "write": 1999, "read": 12345},
        # a chat's next token early on: latency
        {"name": "attn_token_short", "op": "attn", "seqs": 1, "tokens": 1, "kv": 512, "heads": 32, "kv_heads": 8, "dim": 128, "f16": False},
        # a chat's next token late in a long document
        {"name": "attn_token_long", "op": "attn", "seqs": 1, "tokens": 1, "kv": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "f16": False},
        # a served batch: 32 sequences of unequal length, one token each
        {"name": "attn_batch", "op": "attn", "seqs": 32, "tokens": 1, "kv": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "f16": True},
        # three drafted tokens checked at once in four sequences, small heads, an odd length
        {"name": "attn_draft", "op": "attn", "seqs": 4, "tokens": 3, "kv": 5003, "heads": 32, "kv_heads": 8, "dim": 64, "f16": True},
        # a 512-token ubatch of a prompt, 4096 tokens into it
        {"name": "attn_ubatch", "op": "attn", "seqs": 1, "tokens": 512, "kv": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "f16": True},
        # a large ubatch far into a long prompt
        {"name": "attn_prompt", "op": "attn", "seqs": 1, "tokens": 2048, "kv": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "f16": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attn"])
    if op == "rope":
        heads, dim = rng.choice([1, 4, 8, 14, 16, 28, 32]), rng.choice([64, 80, 96, 128])
        most = 4096 * 32 * 128 // (heads * dim)
        return {"op": op, "mode": rng.choice([MROPE, VISION, IMROPE]), "tokens": _log_int(rng, 1, min(most, 16384)),
                "heads": heads, "dim": dim, "f16": rng.random() < 0.5}
    if op == "cache":
        kind, width = rng.choice([Q4_0, Q8_0]), rng.choice([64, 128, 256, 512, 1024])
        rows = _log_int(rng, 256, 40000)
        return {"op": op, "kind": kind, "width": width, "rows": rows, "write": _log_int(rng, 1, min(rows, 2048)),
                "read": _log_int(rng, 1, min(rows, 12000))}
    dim, kv_heads, group = rng.choice([64, 128]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    if rng.random() < 0.6:   # single tokens, and a few drafted ones
        tokens, seqs = rng.choice([1, 1, 1, 2, 3, 5]), _log_int(rng, 1, 32)
        kv = _log_int(rng, max(64, tokens), max(128, min(40000, 32 * 16384 // seqs)))
        return {"op": op, "seqs": seqs, "tokens": tokens, "kv": kv, "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": dim, "f16": tokens * group > 8 or rng.random() < 0.5}
    tokens = _log_int(rng, 16, 2048)
    return {"op": op, "seqs": rng.choice([1, 1, 2]), "tokens": tokens, "kv": _log_int(rng, max(64, tokens), 8192),
            "heads": kv_heads * min(group, 4), "kv_heads": kv_heads, "dim": dim, "f16": True}


def _sections(case):
    """Pairs for time, height, width and the fourth axis; VISION counts two axes over the whole head."""
    half = case["dim"] // 2
    if case["mode"] == VISION:
        return [half // 2, half - half // 2, 0, 0]
    t = half // 4
    h = (half - t) // 2
    return [t, h, half - t - h, 0]


def _lengths(case):
    """How many keys each sequence holds: from half of kv to kv, uneven."""
    n, kv, t = case["seqs"], case["kv"], case["tokens"]
    return [max(t, kv - (kv * ((7 * i) % n)) // (2 * n)) for i in range(n)]


# ---- inputs ------------------------------------------------------------------------------------------


def prepare(case, seed):
    dev = "cuda"
    s = dict(case)
    s["err"] = torch.zeros(1, dtype=torch.int32, device=dev)
    if case["op"] == "rope":
        g = _gen(seed, 1)
        dtype = torch.float16 if case["f16"] else torch.float32
        s["x"] = torch.randn(case["tokens"], case["heads"], case["dim"], device=dev, generator=g).to(dtype)
        # positions of a text that pictures interrupt: one base that grows, and small offsets in a picture
        base = torch.randint(0, 100000, (1,), device=dev, generator=g) + torch.arange(case["tokens"], device=dev)
        off = torch.randint(0, 73, (4, case["tokens"]), device=dev, generator=g)
        pos = off if case["mode"] == VISION else base // 2 + off
        s["pos"] = pos.to(torch.int32).contiguous()
        s["sections"] = _sections(case)
        s["n_dims"] = case["dim"] // 2 if case["mode"] == VISION else case["dim"]
        s["base"] = 10000.0 if case["mode"] == VISION else 1000000.0
        s["out"] = torch.empty_like(s["x"])
        return s
    if case["op"] == "cache":
        g = _gen(seed, 2)
        n = case["width"]
        # channels of unequal size, as keys have them
        gain = torch.exp(torch.randn(n, device=dev, generator=g))
        old = torch.randn(case["rows"], n, device=dev, generator=g) * gain
        s["cache"] = _quantise(old, case["kind"]).contiguous()
        s["rows_in"] = torch.randn(case["write"], n, device=dev, generator=g) * gain
        s["where"] = torch.randperm(case["rows"], device=dev, generator=g)[: case["write"]].to(torch.int64).contiguous()
        s["read_at"] = torch.randint(0, case["rows"], (case["read"],), device=dev, generator=g).to(torch.int32)
        k = min(case["write"], (case["read"] + 1) // 2)      # half of the window is what was just written
        s["read_at"][:k] = s["where"][:k].to(torch.int32)
        s["out"] = torch.empty(case["read"], n, device=dev)
        return s
    S, T, KV, H, HK, D = (case[k] for k in ("seqs", "tokens", "kv", "heads", "kv_heads", "dim"))
    g = _gen(seed, 3)
    dtype = torch.float16 if case["f16"] else torch.float32
    s["q"] = (1.5 * torch.randn(S, T, H, D, device=dev, generator=g)).to(dtype)
    s["k"] = torch.empty(S, KV, HK, D // 32 * 18, dtype=torch.uint8, device=dev)
    s["v"] = torch.empty_like(s["k"])
    for i in range(S):
        for c in (s["k"], s["v"]):
            c[i] = _quantise(torch.randn(KV, HK * D, device=dev, generator=g), Q4_0).view(KV, HK, -1)
    # token t of a sequence of n keys sees its keys 0 .. n - T + t, as a causal mask has it
    at = torch.arange(KV, device=dev)
    last = torch.tensor([[n - T + t for t in range(T)] for n in _lengths(case)], device=dev)
    mask = torch.zeros(S, T, KV, dtype=torch.float16, device=dev)
    mask.masked_fill_(at > last[..., None], NEG)
    s["mask"] = mask
    s["scale"] = 1.0 / math.sqrt(D)
    s["out"] = torch.empty(S, T, H, D, dtype=dtype, device=dev)
    if own:
        s["ws"] = torch.empty(_lib().flash_attn_kvq_workspace_size(D, T, H, KV, HK, S), dtype=torch.uint8, device=dev)
    return s


# ---- one pass ------------------------------------------------------------------------------------------


def run(s):
    if own:
        g = _lib()
        if s["op"] == "rope":
            g.rope_multi(s["x"], s["pos"], s["out"], s["n_dims"], s["mode"], s["sections"], freq_base=s["base"])
        elif s["op"] == "cache":
            g.set_rows(s["rows_in"], s["where"], s["cache"], s["kind"], s["err"])
            g.get_rows(s["cache"], s["kind"], s["read_at"], s["out"], s["err"])
        else:
            g.flash_attn_kvq(Q4_0, s["q"], s["k"], s["v"], s["mask"], s["out"], s["scale"], s["ws"], s["err"])
        return s["out"]
    if s["op"] == "rope":
        return _rope(s["x"], s["pos"], s["n_dims"], s["mode"], s["sections"], s["base"])
    if s["op"] == "cache":
        s["cache"][s["where"]] = _quantise(s["rows_in"], s["kind"])
        return _dequantise(s["cache"][s["read_at"].long()], s["kind"])
    return _attention(s["q"], s["k"], s["v"], s["mask"], s["scale"])


def _rope(x, pos, n_dims, mode, sections, base):
    """y = x rotated pair by pair by pos[axis(pair)] * base^(-2 step(pair) / n_dims); the angles in 64 bits."""
    pairs = x.shape[-1] // 2 if mode == VISION else n_dims // 2
    gap = n_dims if mode == VISION else n_dims // 2
    i = torch.arange(pairs, device=x.device)
    s0, s1, s2, s3 = sections
    sector = i % (s0 + s1 + s2 + s3)
    if mode == IMROPE:
        turn = sector % 3
        axis = torch.where((turn == 0) & (sector < 3 * s0), 0, 3)
        axis = torch.where((turn == 1) & (sector < 3 * s1), 1, axis)
        axis = torch.where((turn == 2) & (sector < 3 * s2), 2, axis)
        step = i
    else:
        axis = (sector >= s0).long() + (sector >= s0 + s1).long() + (sector >= s0 + s1 + s2).long()
        start = (sector >= s0).long() * s0 + (sector >= s0 + s1).long() * s1 + (sector >= s0 + s1 + s2).long() * s2
        step = sector - start if mode == VISION else i
    freq = torch.pow(torch.tensor(base, dtype=torch.float64, device=x.device), -2.0 * step.double() / n_dims)
    angle = pos.t()[:, axis].double() * freq
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    x32 = x.float()
    a, b = x32[..., :pairs], x32[..., gap:gap + pairs]
    y = x32.clone()
    y[..., :pairs] = a * cos - b * sin
    y[..., gap:gap + pairs] = a * sin + b * cos
    return y.to(x.dtype)


def _quantise(x, kind):
    """Rows of f32 as ggml's Q4_0 or Q8_0 blocks: uint8 [rows, width / 32 * block bytes]."""
    v = x.reshape(x.shape[0], -1, 32)
    size = v.abs()
    amax = size.amax(-1, keepdim=True)
    if kind == Q8_0:
        d = amax / torch.full_like(amax, 127.0)   # a true division: by a plain number torch multiplies with its inverse
        inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        t = v * inv
        q = (torch.sign(t) * torch.floor(t.abs().double() + 0.5)).to(torch.int8)
        codes = q.view(torch.uint8)
    else:
        lane = torch.arange(32, device=x.device).expand_as(v)
        first = torch.where(size == amax, lane, 32).amin(-1, keepdim=True)   # ties: the lowest index
        d = torch.gather(v, -1, first) / -8.0
        inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
        q = torch.trunc(v.double() * inv.double() + 8.5).clamp(0, 15).to(torch.uint8)   # next to a border: 64 bits
        codes = q[..., :16] | (q[..., 16:] << 4)
    return torch.cat([d.half().view(torch.uint8), codes], -1).reshape(x.shape[0], -1)


def _dequantise(rows, kind):
    """Rows of blocks as f32: [..., row bytes] -> [..., width]."""
    b = rows.reshape(*rows.shape[:-1], -1, BLOCK_BYTES[kind])
    d = b[..., :2].contiguous().view(torch.float16).float()
    q = b[..., 2:].contiguous()
    if kind == Q8_0:
        v = q.view(torch.int8).float()
    else:
        v = torch.cat([q & 15, q >> 4], -1).float() - 8.0
    return (v * d).reshape(*rows.shape[:-1], -1)


def _attention(q, k, v, mask, scale):
    """softmax(scale q k^T + mask) v over the decoded cache, a group of query heads per key/value head."""
    S, T, H, D = q.shape
    HK = k.shape[2]
    kf = _dequantise(k, Q4_0).permute(0, 2, 3, 1)                     # [S, HK, D, KV]
    vf = _dequantise(v, Q4_0).permute(0, 2, 1, 3)                     # [S, HK, KV, D]
    qf = q.float().reshape(S, T, HK, H // HK, D).permute(0, 2, 3, 1, 4)   # [S, HK, G, T, D]
    x = torch.matmul(qf.reshape(S, HK, -1, D), kf).reshape(S, HK, H // HK, T, -1)
    x = x.mul_(scale).add_(mask.float()[:, None, None])
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == NEG, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(S, HK, -1, p.shape[-1]), vf).reshape(S, HK, H // HK, T, D)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    return o.permute(0, 3, 1, 2, 4).reshape(S, T, H, D).to(q.dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (2 if case["f16"] else 4) + 16 * case["tokens"], "flops": 3 * n}
    if case["op"] == "cache":
        row = case["width"] // 32 * BLOCK_BYTES[case["kind"]]
        return {"bytes": case["write"] * (4 * case["width"] + row + 8) + case["read"] * (row + 4 * case["width"] + 4),
                "flops": 4 * case["write"] * case["width"] + 2 * case["read"] * case["width"]}
    S, T, H, HK, D = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim"))
    held = sum(_lengths(case))                                        # keys that some token sees
    seen = sum(n * T - T * (T - 1) // 2 for n in _lengths(case))      # (token, key) pairs
    size = 2 if case["f16"] else 4
    return {"bytes": 2 * held * HK * (D // 32 * 18) + 2 * S * T * H * D * size + 2 * S * T * case["kv"],
            "flops": 4 * seen * H * D}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        x, pos = s["x"].double(), s["pos"].double()
        n, mode, out = s["n_dims"], s["mode"], s["x"].double().clone()
        start = [0]
        for w in s["sections"]:
            start.append(start[-1] + w)
        for i in range(case["dim"] // 2 if mode == VISION else n // 2):
            sec = i % start[4]
            ax = max(a for a in range(4) if start[a] <= sec and s["sections"][a] > 0)
            if mode == IMROPE:
                ax = sec % 3 if sec < 3 * s["sections"][sec % 3] else 3
            e = sec - start[ax] if mode == VISION else i
            th = pos[ax] * s["base"] ** (-2.0 * e / n)
            j = i + (n if mode == VISION else n // 2)
            c, w = torch.cos(th)[:, None], torch.sin(th)[:, None]
            out[..., i], out[..., j] = x[..., i] * c - x[..., j] * w, x[..., i] * w + x[..., j] * c
        return out
    if case["op"] == "cache":
        kind, n = case["kind"], case["width"]
        blocks = s["rows_in"].double().reshape(-1, 32)
        if kind == Q8_0:
            d = (blocks.abs().max(1, keepdim=True).values / 127.0).float()
            inv = (1.0 / d.double()).float().double()                 # the format's inverse is an f32 number,
            t = (blocks * inv).float().double()                       # and so are the scaled values
            val = torch.where(t < 0, torch.ceil(t - 0.5), torch.floor(t + 0.5))
        else:
            hi, lo = blocks.max(1, keepdim=True).values, blocks.min(1, keepdim=True).values
            d = (torch.where(hi > -lo, hi, lo) / -8.0).float()
            inv = (1.0 / d.double()).float().double()                 # the format's inverse is an f32 number
            val = torch.floor(blocks * inv + 8.5).clamp(max=15.0) - 8.0
        new = (val * d.half().double()).reshape(-1, n)
        slot = torch.full((case["rows"],), -1, dtype=torch.long, device="cuda")
        slot[s["where"]] = torch.arange(case["write"], device="cuda")
        at = s["read_at"].long()
        raw = s["cache"][at].reshape(case["read"], n // 32, BLOCK_BYTES[kind]).int()
        bits = raw[..., 0] | (raw[..., 1] << 8)
        scale = bits.to(torch.int16).view(torch.float16).double()[..., None]
        body = raw[..., 2:]
        code = torch.where(body > 127, body - 256, body) if kind == Q8_0 else torch.cat([body % 16, body // 16], -1) - 8
        out = (code.double() * scale).reshape(case["read"], n)
        fresh = slot[at] >= 0
        out[fresh] = new[slot[at[fresh]]]
        return out
    S, T, H, HK, D, KV = (case[k] for k in ("seqs", "tokens", "heads", "kv_heads", "dim", "kv"))
    out = torch.zeros(S, T, H, D, dtype=torch.float64, device="cuda")
    lengths = _lengths(case)
    for i in range(S):
        for h in range(HK):
            kv = []
            for c in (s["k"], s["v"]):
                raw = c[i, :, h].reshape(KV, D // 32, 18).int()
                d = (raw[..., 0] | (raw[..., 1] << 8)).to(torch.int16).view(torch.float16).double()
                body = raw[..., 2:]
                kv.append((torch.cat([body % 16, body // 16], -1) - 8).double().mul_(d[..., None]).reshape(KV, D))
            hidden = torch.arange(KV, device="cuda")[None, :] > torch.arange(T, device="cuda")[:, None] + lengths[i] - T
            for j in range(h * (H // HK), (h + 1) * (H // HK)):
                x = (s["q"][i, :, j].double() @ kv[0].T) / math.sqrt(D)
                x = x.masked_fill_(hidden, NEG).sub_(x.amax(1, keepdim=True)).exp_()
                out[i, :, j] = (x @ kv[1]) / x.sum(1, keepdim=True)
    return out
