"""Attention over a Q4_0 cache (b200_flash_attn_kvq) on the GPU against its definition in 64 bits.

Tolerance. Let A be the largest scale * sum_i |q_i k_i| of a row and V the largest |v|. The row kernel
holds q to 2^-22 of its row's largest value, adds exact products in fp32 (at most 16 roundings of 2^-23
of A, the tensor core truncating) and forms the exponent with |s| log2(e) rounded at 2^-24 and ex2 at
2^-22: a weight is within e = A 2^-18 + 2^-20 of its value, relative. Outputs are ratios of sums of such
weights, each added in fp32 over at most a few hundred steps (2^-15 at the worst, far less in truth):
|dO| <= (2 e + 2^-15) V. An f16 result adds the rounding of P (2^-11 of each weight) and of itself
(2^-11): |dO| <= (2 e + 2^-15 + 2^-11) V + 2^-11 |O| + 2^-25.

More than 32 query rows a KV head take the tcgen05 kernel over fp16 tiles: q, the decoded keys, the
decoded values and P each round to fp16 (2^-11 of a value), and a score plus its mask M to fp32 (2^-24 of
1.45 M in log2 units, 2^-24 M of the weight; 2^-23 allowed), so e = 2 * 2^-11 A + A 2^-18 + 2^-23 M + 2^-20, and |dO| <= (2 e + 2^-15 + 2 * 2^-11) V for the rest, the maximum taken over V."""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

NEG = float("-inf")
Q4_0 = 2
LOWEST = -65504.0


def quantise(x):
    """f32 [.., n] -> uint8 [.., n / 32 * 18]; any valid blocks serve."""
    import torch
    v = x.reshape(*x.shape[:-1], -1, 32)
    i = v.abs().argmax(-1, keepdim=True)
    d = torch.gather(v, -1, i) / -8
    c = torch.where(d != 0, torch.trunc(v / torch.where(d != 0, d, torch.ones_like(d)) + 8.5), torch.full_like(v, 8))
    c = c.clamp(0, 15).to(torch.uint8)
    q = c[..., :16] | (c[..., 16:] << 4)
    h = d.half().contiguous().view(torch.uint8).reshape(*d.shape[:-1], 2)
    return torch.cat([h, q], -1).reshape(*x.shape[:-1], -1).contiguous()


def decode64(b):
    import torch
    r = b.reshape(*b.shape[:-1], -1, 18)
    d = r[..., :2].contiguous().view(torch.float16).double()
    q = r[..., 2:]
    return ((torch.cat([q & 15, q >> 4], -1).double() - 8) * d).reshape(*b.shape[:-1], -1)


def reference(q, k, v, mask, scale, softcap=0.0):
    """64-bit outputs [S, T, H, D], A per row and V; a key whose mask is -inf takes no part."""
    import torch
    S, T, H, D = q.shape
    HK = k.shape[2]
    kd, vd = decode64(k), decode64(v)
    out = torch.zeros(S, T, H, D, dtype=torch.float64, device=q.device)
    A = torch.zeros(S, T, H, 1, dtype=torch.float64, device=q.device)
    vmax = 0.0
    for s in range(S):
        m = torch.zeros(T, k.shape[1], dtype=torch.float64, device=q.device) if mask is None else \
            mask[s if mask.shape[0] == S else 0, :T, :k.shape[1]].double()
        gone = m == NEG
        used = ~gone.all(0)
        for h in range(H):
            hk = h // (H // HK)
            kk, vv = kd[s, used, hk], vd[s, used, hk]
            if not used.any():
                continue
            vmax = max(vmax, float(vv[torch.isfinite(vv)].abs().max()))
            qq = q[s, :, h].double()
            x = qq @ kk.T * scale
            fin = torch.where(torch.isfinite(kk), kk, torch.zeros_like(kk))
            A[s, :, h, 0] = (qq.abs() @ fin.abs().T * abs(scale)).amax(1)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            x = (x + m[:, used]).masked_fill(gone[:, used], NEG)
            top = x.amax(1, keepdim=True)
            p = torch.exp(x - torch.where(top == NEG, torch.zeros_like(top), top))
            p = torch.where(gone[:, used], torch.zeros_like(p), p)
            num = torch.where((p == 0)[..., None] & gone[:, used][..., None], 0.0, p[..., None] * vv[None]).sum(1) \
                if not torch.isfinite(vv).all() else p @ vv
            den = p.sum(1, keepdim=True)
            out[s, :, h] = torch.where(den == 0, torch.zeros_like(num), num / den)
    return out, A, vmax


def workspace(D, T, H, KV, HK, S):
    import torch
    import ggml_b200 as g
    return torch.empty(g.flash_attn_kvq_workspace_size(D, T, H, KV, HK, S), dtype=torch.uint8, device="cuda")


def run(q, k, v, mask, scale, f16=False, softcap=0.0, stream=None, ws=None):
    import torch
    import ggml_b200 as g
    S, T, H, D = q.shape
    out = torch.full(q.shape, 7.0, dtype=torch.float16 if f16 else torch.float32, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = workspace(D, T, H, k.shape[1], k.shape[2], S) if ws is None else ws
    g.flash_attn_kvq(Q4_0, q, k, v, mask, out, scale, ws, err, softcap=softcap, stream=stream)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    return out


def check(out, q, k, v, mask, scale, softcap=0.0):
    import torch
    want, A, vmax = reference(q, k, v, mask, scale, softcap)
    prompt = q.shape[1] * (q.shape[2] // k.shape[2]) > 32
    e = A * (2.0 ** -18 + (2 * 2.0 ** -11 if prompt else 0)) + 2.0 ** -20
    if prompt and mask is not None:      # score + mask rounded to fp32
        fin = mask[torch.isfinite(mask)]
        e = e + (float(fin.abs().max()) * 2.0 ** -23 if fin.numel() else 0.0)
    tol = (2 * e + 2.0 ** -15 + (2 * 2.0 ** -11 if prompt else 0)) * vmax
    if out.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * vmax + 2.0 ** -11 * want.abs() + 2.0 ** -25
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    d = torch.where(torch.isnan(want), torch.zeros_like(want), (out.double() - want).abs())
    assert bool((d <= tol).all()), float((d - tol).max())


def inputs(S, T, H, HK, D, KV, seed=0, q_f16=False, gain=1.0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed + S * 7 + T * 11 + KV * 13 + D)
    q = 1.5 * torch.randn(S, T, H, D, device="cuda", generator=gen)
    k = quantise(torch.randn(S, KV, HK, D, device="cuda", generator=gen))
    v = quantise(gain * torch.randn(S, KV, HK, D, device="cuda", generator=gen))
    return (q.half() if q_f16 else q), k, v


def causal(S, T, KV, lengths=None):
    import torch
    m = torch.zeros(S, T, KV, dtype=torch.float16, device="cuda")
    for s in range(S):
        n = KV if lengths is None else lengths[s]
        last = torch.arange(T, device="cuda") + n - T
        m[s].masked_fill_(torch.arange(KV, device="cuda")[None] > last[:, None], NEG)
    return m


SHAPES = [
    # S, T, H, HK, D, KV
    (1, 1, 1, 1, 64, 1),
    (1, 1, 8, 8, 128, 31),
    (1, 1, 32, 8, 128, 33),
    (1, 1, 32, 8, 128, 257),
    (1, 1, 7, 1, 64, 1000),
    (2, 1, 64, 4, 128, 515),       # sixteen rows a head
    (3, 2, 14, 2, 64, 130),
    (1, 3, 8, 2, 128, 4099),
    (2, 5, 24, 3, 64, 96),         # a row tile that spans tokens
    (1, 9, 4, 4, 128, 64),         # one row a token
    (5, 1, 32, 8, 128, 2048),
    (1, 1, 32, 8, 128, 40000),
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", SHAPES)
def test_rows_against_definition(cuda, S, T, H, HK, D, KV, f16):
    q, k, v = inputs(S, T, H, HK, D, KV, q_f16=f16)
    scale = 1 / math.sqrt(D)
    m = causal(S, T, max(KV, T)) if KV >= T else None
    m = m[:, :, :KV] if m is not None else None
    check(run(q, k, v, m, scale, f16), q, k, v, m, scale)
    check(run(q, k, v, None, scale, f16), q, k, v, None, scale)


PROMPTS = [
    # S, T, H, HK, D, KV
    (1, 33, 1, 1, 64, 33),
    (1, 40, 4, 1, 128, 129),
    (1, 200, 32, 8, 128, 1000),
    (2, 130, 14, 2, 64, 700),        # seven heads a group: one query head a tile
    (3, 17, 8, 2, 128, 2000),        # parts of the keys over several CTAs
    (1, 512, 8, 2, 128, 4096),
    (1, 9, 32, 4, 64, 20000),
    (1, 300, 32, 8, 128, 5000),      # an odd number of token blocks
    (2, 1100, 8, 8, 64, 1100),
    (1, 700, 64, 8, 128, 900),       # more tiles than a wave: whole ones, then cut ones
]


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", PROMPTS)
def test_prompts_against_definition(cuda, S, T, H, HK, D, KV, f16):
    q, k, v = inputs(S, T, H, HK, D, KV, q_f16=f16)
    scale = 1 / math.sqrt(D)
    m = causal(S, T, KV, [KV - (KV - T) * s // (S + 1) for s in range(S)])
    out = run(q, k, v, m, scale, f16)
    check(out, q, k, v, m, scale)
    want = reference(q, k, v, m, scale)[0]
    assert float((out.double() - want).norm() / want.norm()) < 2e-3     # random roundings: far below the bound
    check(run(q, k, v, None, scale, f16), q, k, v, None, scale)
    check(run(q, k, v, None, scale, f16, softcap=5.0), q, k, v, None, scale, softcap=5.0)
    check(run(q, k, v, m, -3 * scale, f16), q, k, v, m, -3 * scale)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("T", [1, 6, 50])
def test_masks(cuda, T, f16):
    """Rows that see nothing, one key, only keys of fp16's lowest value, that value beside visible keys,
    finite biases, a gap of more than a tile, and a mask row wider and off alignment."""
    import torch
    S, H, HK, D, KV = 2, 8, 2, 128, 700
    q, k, v = inputs(S, T, H, HK, D, KV)
    scale = 1 / math.sqrt(D)
    wide = torch.zeros(S, T + 2, KV + 3, dtype=torch.float16, device="cuda")
    m = wide[:, :T, 1:KV + 1]
    gen = torch.Generator(device="cuda").manual_seed(1)
    kinds = ["none", "one", "lowest", "beside", "bias", "gap", "tail", "big"]
    for i in range(0, len(kinds), T * S):
        m.zero_()
        for j, kind in enumerate(kinds[i:i + T * S]):
            row = m[j // T, j % T]
            if kind == "none":
                row.fill_(NEG)
            elif kind == "one":
                row.fill_(NEG)
                row[333] = 0
            elif kind == "lowest":
                row.fill_(LOWEST)
            elif kind == "beside":
                row[::2] = LOWEST
            elif kind == "bias":
                row.copy_(-8 * torch.rand(KV, device="cuda", generator=gen))
            elif kind == "gap":
                row[40:600] = NEG
            elif kind == "tail":
                row[65:] = NEG
            elif kind == "big":
                row.fill_(-30000)
                row[100:300] = -30016
                row[5] = NEG
        check(run(q, k, v, m, scale, f16), q, k, v, m, scale)


def test_lowest_over_many_splits(cuda):
    """All keys at the lowest value: as if there were no mask, also when CTAs share the keys."""
    import torch
    q, k, v = inputs(1, 1, 8, 2, 128, 9000)
    m = torch.full((1, 1, 9000), LOWEST, dtype=torch.float16, device="cuda")
    check(run(q, k, v, m, 0.09), q, k, v, m, 0.09)
    m[..., 4000:] = 0
    check(run(q, k, v, m, 0.09), q, k, v, m, 0.09)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_garbage_behind_the_mask(cuda, T):
    """Bytes that decode to NaN and infinity in keys no row sees, and in keys only later rows see."""
    import torch
    S, H, HK, D, KV = 2, 8, 2, 64, 300
    q, k, v = inputs(S, T, H, HK, D, KV)
    m = causal(S, T, KV, [200, 290])
    clean = run(q, k, v, m, 0.125)
    k2, v2 = k.clone(), v.clone()
    for s, n in ((0, 200), (1, 290)):
        k2[s, n:], v2[s, n:] = 0xff, 0xff
        k2[s, n:, :, 1::18], v2[s, n:, :, 1::18] = 0x7c, 0x7c
    assert torch.equal(run(q, k2, v2, m, 0.125), clean)
    if T > 1:
        # the last token alone sees key n - 1: its scales become no numbers
        k2, v2 = k.clone(), v.clone()
        for s, n in ((0, 200), (1, 290)):
            v2[s, n - 1, :, 0], v2[s, n - 1, :, 1] = 0xff, 0x7f
            k2[s, n - 1, 0, 0], k2[s, n - 1, 0, 1] = 0x00, 0x7e
        got = run(q, k2, v2, m, 0.125)
        assert bool(torch.isfinite(got[:, :T - 1]).all())
        assert torch.allclose(got[:, :T - 1], clean[:, :T - 1], rtol=0, atol=1e-3)
        assert bool(torch.isnan(got[:, T - 1, :H // HK, 0]).all())


@pytest.mark.parametrize("gain", [1e-4, 300.0])
def test_value_sizes(cuda, gain):
    """Values far from 1, and keys whose scales differ by orders of magnitude."""
    import torch
    q, k, v = inputs(1, 1, 16, 4, 128, 600, gain=gain)
    check(run(q, k, v, None, 0.1, False), q, k, v, None, 0.1)
    q, k, v = inputs(1, 2, 16, 4, 128, 600, gain=gain)
    vv = decode64(v) * torch.logspace(-2, 2, 600, device="cuda", dtype=torch.float64)[None, :, None, None]
    v = quantise(vv.float())
    check(run(q, k, v, None, 0.1, False), q, k, v, None, 0.1)


def test_scores_and_queries_far_from_one(cuda):
    """Large and tiny q, a softcap, a negative scale."""
    import torch
    q, k, v = inputs(1, 1, 8, 2, 128, 300)
    for mul, scale in ((1e4, 1e-5), (1e-6, 1e5), (1.0, -0.2), (3e38, 1e-39)):
        check(run(q * mul if mul < 1e38 else q.sign() * mul, k, v, None, scale),
              q * mul if mul < 1e38 else q.sign() * mul, k, v, None, scale)
    check(run(q, k, v, None, 0.3, softcap=20.0), q, k, v, None, 0.3, softcap=20.0)
    check(run(torch.zeros_like(q), k, v, None, 0.3), torch.zeros_like(q), k, v, None, 0.3)


@pytest.mark.parametrize("T", [1, 4])
def test_strides(cuda, T):
    """q by heads outside tokens, cache rows inside wider ones, K and V side by side, a mask shared by
    the streams, streams in another order in memory."""
    import torch
    S, H, HK, D, KV = 3, 8, 2, 128, 150
    q, k, v = inputs(S, T, H, HK, D, KV)
    m = causal(1, T, KV)
    check(run(q, k, v, m.expand(S, T, KV).contiguous(), 0.1), q, k, v, m, 0.1)
    qh = q.transpose(1, 2).contiguous().transpose(1, 2)
    both = torch.zeros(KV, S, HK, 2, 88, dtype=torch.uint8, device="cuda")
    both[..., 0, 8:80], both[..., 1, 8:80] = k.transpose(0, 1), v.transpose(0, 1)
    ks, vs = both[..., 0, 8:80].transpose(0, 1), both[..., 1, 8:80].transpose(0, 1)
    check(run(qh, ks, vs, m, 0.1), q, k, v, m, 0.1)     # another copy route: another split, other roundings


def test_repeats_exactly_on_streams_and_in_graphs(cuda):
    import torch
    import ggml_b200 as g
    S, T, H, HK, D, KV = 1, 1, 32, 8, 128, 5000
    q, k, v = inputs(S, T, H, HK, D, KV)
    m = causal(S, T, KV, [4321])
    want = run(q, k, v, m, 0.1)
    for _ in range(3):
        assert torch.equal(run(q, k, v, m, 0.1), want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    assert torch.equal(run(q, k, v, m, 0.1, stream=st), want)
    out = torch.empty_like(q)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = workspace(D, T, H, KV, HK, S)
    ws.fill_(0xff)                                       # nothing is expected of the workspace's bytes
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.flash_attn_kvq(Q4_0, q, k, v, m, out, 0.1, ws, err)
    q2, k2, v2 = inputs(S, T, H, HK, D, KV, seed=5)
    q.copy_(q2), k.copy_(k2), v.copy_(v2)
    m.copy_(causal(S, T, KV, [4999]))
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run(q, k, v, m, 0.1))


def test_cache_past_32_bits(cuda):
    """Keys more than 2^32 bytes into a cache view: the last of a long shared buffer."""
    import torch
    S, T, H, HK, D, KV = 1, 1, 4, 1, 128, 64
    q, k, v = inputs(S, T, H, HK, D, KV)
    stride = 1 << 27                                      # bytes between keys: 64 keys span 8.6 GB
    big = torch.zeros(KV * stride, dtype=torch.uint8, device="cuda")
    kv = big.as_strided((S, KV, HK, 72), (KV * stride, stride, 72, 1))
    vv = big.as_strided((S, KV, HK, 72), (KV * stride, stride, 72, 1), 4096)
    kv.copy_(k), vv.copy_(v)
    check(run(q, kv, vv, None, 0.1), q, k, v, None, 0.1)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", [
    (1, 1, 40, 1, 128, 777),         # single tokens whose KV head serves more rows than the row kernel takes
    (1, 1, 256, 1, 64, 300),
    (2, 1, 33, 1, 64, 5),
    (300, 1, 4, 1, 64, 40),          # more streams than SMs
    (70, 2, 64, 2, 64, 129),
    (1, 16, 2, 1, 128, 1),           # as many rows as the row kernel takes, one key; and two more
    (1, 17, 2, 1, 128, 1),
    (1, 64, 6, 3, 64, 20),           # more tokens than keys
    (2, 1, 4, 2, 128, 127),
    (1, 12, 8, 2, 128, 700),         # either side of the row kernels' last size
    (1, 13, 8, 2, 128, 700),
    (2, 16, 14, 2, 64, 900),         # a group of seven: rows for longer
    (1, 100, 7, 1, 128, 300),
])
def test_shapes_at_the_ends(cuda, S, T, H, HK, D, KV, f16):
    """A random mask, its first row of every stream hidden whole, its last key of every other row visible."""
    import torch
    q, k, v = inputs(S, T, H, HK, D, KV, seed=5, q_f16=f16)
    scale = 1 / math.sqrt(D)
    gen = torch.Generator(device="cuda").manual_seed(S + T + KV)
    m = torch.randn(S, T, KV, device="cuda", generator=gen).half()
    m[torch.rand(S, T, KV, device="cuda", generator=gen) < 0.5] = NEG
    m[:, 1:, -1] = 0.0
    m[:, 0] = NEG
    check(run(q, k, v, m, scale, f16), q, k, v, m, scale)
    check(run(q, k, v, None, scale, f16), q, k, v, None, scale)
