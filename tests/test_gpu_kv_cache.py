"""SET_ROWS into F32 / F16 / Q8_0 / Q4_0 rows and GET_ROWS out of Q8_0 / Q4_0 rows on the GPU.

Both are exact: the encoders follow ggml's reference bit for bit (Q4_0 with the product and sum before
the truncation unrounded, in 64 bits here; Q8_0 with an f32 product rounded half away from zero), and a
decoded value is one f32 product."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

Q4_0, Q8_0, F32, F16 = 2, 8, 0, 1


def encode(x, kind):
    """x f32 [rows, n] -> uint8 [rows, n / 32 * block bytes]."""
    v = x.reshape(x.shape[0], -1, 32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        if kind == Q8_0:
            d = np.abs(v).max(-1, keepdims=True) / np.float32(127)
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
            t = (v * inv).astype(np.float64)
            q = np.clip(np.sign(t) * np.floor(np.abs(t) + 0.5), -127, 127).astype(np.int8).view(np.uint8)
        else:
            at = np.abs(v).argmax(-1)[..., None]          # the first of equals
            d = np.take_along_axis(v, at, -1) / np.float32(-8)
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0))
            c = np.clip(np.trunc(v.astype(np.float64) * inv.astype(np.float64) + 8.5), 0, 15).astype(np.uint8)
            q = c[..., :16] | (c[..., 16:] << 4)
        h = d.astype(np.float16).view(np.uint8).reshape(*d.shape[:2], 2)
    return np.concatenate([h, q], -1).reshape(x.shape[0], -1)


def decode(rows, kind):
    b = rows.reshape(*rows.shape[:-1], -1, 34 if kind == Q8_0 else 18)
    d = b[..., :2].copy().view(np.float16).astype(np.float32)
    q = b[..., 2:]
    c = q.view(np.int8).astype(np.float32) if kind == Q8_0 else np.concatenate([q & 15, q >> 4], -1).astype(np.float32) - 8
    return (c * d).reshape(*rows.shape[:-1], -1)


def values(rng, rows, n):
    """Rows with ties for the largest size, zero blocks, tiny, subnormal and huge values among them."""
    x = (rng.standard_normal((rows, n)) * np.exp(rng.standard_normal((1, n)))).astype(np.float32)
    if rows > 5 and n >= 64:
        x[0, :32] = 0
        x[1, 3], x[1, 20] = 7.5, -7.5
        x[2, 3], x[2, 20] = -7.5, 7.5
        x[3, :32] *= np.float32(1e-38)
        x[4, :32] *= np.float32(1e-42)
        x[5, 32:64] *= np.float32(1e5)
        x[4, 32:64] = np.round(x[4, 32:64] * 4) / 2           # many values on a border
    return x


@pytest.mark.parametrize("kind", [Q4_0, Q8_0])
@pytest.mark.parametrize("n,n_rows,total", [(32, 1, 1), (64, 7, 9), (96, 33, 50), (1024, 1, 300), (1024, 512, 700),
                                            (128, 3000, 3001), (2080, 65, 80), (480, 21, 40), (5120, 3, 4)])
def test_write_and_read_back(cuda, kind, n, n_rows, total):
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(n + n_rows)
    x = values(rng, n_rows, n)
    where = rng.permutation(total)[:n_rows]
    row = n // 32 * (34 if kind == Q8_0 else 18)
    cache = rng.integers(0, 256, (total, row), dtype=np.uint8)
    cache.reshape(total, -1, row // (n // 32))[..., 1] &= 0x3b     # finite scales
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    for idt in (np.int64, np.int32):
        d = torch.from_numpy(cache).cuda()
        g.set_rows(torch.from_numpy(x).cuda(), torch.from_numpy(where.astype(idt)).cuda(), d, kind, err)
        want = cache.copy()
        want[where] = encode(x, kind)
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        assert np.array_equal(d.cpu().numpy(), want)               # rows no index names stay as they were
    at = rng.integers(0, total, 2 * n_rows + 1).astype(np.int32)
    out = torch.empty(len(at), n, device="cuda")
    g.get_rows(d, kind, torch.from_numpy(at).cuda(), out, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    # a scale past fp16's range is infinite, and code 0 of it reads as NaN on both sides
    assert np.array_equal(out.cpu().numpy(), decode(want, kind)[at], equal_nan=True)


@pytest.mark.parametrize("kind,n", [(F32, 5), (F32, 128), (F16, 1), (F16, 100), (F16, 256)])
def test_plain_rows(cuda, kind, n):
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(n)
    x = rng.standard_normal((6, n)).astype(np.float32) * 1000
    dt = np.float32 if kind == F32 else np.float16
    cache = rng.standard_normal((9, n)).astype(dt)
    where = rng.permutation(9)[:6]
    d = torch.from_numpy(cache).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), torch.from_numpy(where).cuda(), d, kind, err)
    cache[where] = x.astype(dt)
    torch.cuda.synchronize()
    assert np.array_equal(d.cpu().numpy(), cache)


@pytest.mark.parametrize("kind", [Q4_0, Q8_0, F16])
@pytest.mark.parametrize("n_rows", [40, 5000])
def test_the_last_of_equal_indices_stays(cuda, kind, n_rows):
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(4)
    n = 64
    x = rng.standard_normal((n_rows, n)).astype(np.float32)
    where = rng.integers(0, 17, n_rows)
    enc = x.astype(np.float16) if kind == F16 else encode(x, kind)
    cache = np.zeros((20, enc.shape[1]), dtype=enc.dtype)
    d = torch.from_numpy(cache).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), torch.from_numpy(where).cuda(), d, kind, err)
    for i, r in enumerate(where):
        cache[r] = enc[i]
    torch.cuda.synchronize()
    assert np.array_equal(d.cpu().numpy(), cache)


@pytest.mark.parametrize("kind", [Q4_0, Q8_0])
def test_strided_views_and_slices(cuda, kind):
    """[streams, kv, width] views inside wider rows, source rows off 16-byte alignment, an index per
    slice and one shared by slices."""
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(6)
    size = 34 if kind == Q8_0 else 18
    S, KV, n, T = 4, 30, 96, 7
    wide = rng.integers(0, 256, (S, KV, 3 * size + 2 * size + 6), dtype=np.uint8)
    for per_slice in (4, 2, 1):
        x = rng.standard_normal((S, T, n + 5)).astype(np.float32)
        where = np.stack([rng.permutation(KV)[:T] for _ in range(per_slice)]).astype(np.int64)
        d = torch.from_numpy(wide).cuda()
        view = d[:, :, 4:4 + 3 * size]
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        g.set_rows(torch.from_numpy(x).cuda()[:, :, 1:1 + n], torch.from_numpy(where).cuda(), view, kind, err)
        want = wide.copy()
        for s in range(S):
            want[s, where[s % per_slice], 4:4 + 3 * size] = encode(np.ascontiguousarray(x[s, :, 1:1 + n]), kind)
        torch.cuda.synchronize()
        assert int(err.item()) == 0
        assert np.array_equal(d.cpu().numpy(), want)
        back = torch.empty(S, T, n, device="cuda")
        at = torch.from_numpy(np.stack([where[s % per_slice] for s in range(S)]).astype(np.int32)).cuda()
        g.get_rows(view, kind, at, back, err)
        torch.cuda.synchronize()
        for s in range(S):
            fin = decode(np.ascontiguousarray(want[s, where[s % per_slice], 4:4 + 3 * size]), kind)
            assert np.array_equal(back[s].cpu().numpy(), fin, equal_nan=True)


@pytest.mark.parametrize("kind", [Q4_0, Q8_0])
def test_bad_indices_are_reported_and_not_written(cuda, kind):
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(7)
    size = 34 if kind == Q8_0 else 18
    x = rng.standard_normal((4, 64)).astype(np.float32)
    cache = rng.integers(0, 256, (10, 2 * size), dtype=np.uint8)
    d = torch.from_numpy(cache).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), torch.tensor([3, -1, 10, 1 << 40]).cuda(), d, kind, err)
    torch.cuda.synchronize()
    with pytest.raises(g.B200Error, match="bad_index"):
        g.check_device(err, "set_rows")
    cache[3] = encode(x[:1], kind)[0]
    assert np.array_equal(d.cpu().numpy(), cache)
    err.zero_()
    out = torch.full((3, 64), 5.0, device="cuda")
    g.get_rows(d, kind, torch.tensor([3, -2, 10], dtype=torch.int32).cuda(), out, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 6
    o = out.cpu().numpy()
    assert np.array_equal(o[0], decode(cache[3:4], kind)[0]) and not o[1:].any()


@pytest.mark.parametrize("kind", [Q4_0, Q8_0])
def test_values_that_are_no_numbers(cuda, kind):
    import torch
    import ggml_b200 as g
    x = np.ones((3, 96), dtype=np.float32)
    x[0, 40], x[1, 0], x[2, 95] = np.nan, np.inf, -np.inf
    cache = torch.zeros(3, 3 * (34 if kind == Q8_0 else 18), dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), torch.arange(3, device="cuda"), cache, kind, err)
    out = torch.empty(3, 96, device="cuda")
    g.get_rows(cache, kind, torch.arange(3, dtype=torch.int32, device="cuda"), out, err)
    got = torch.isnan(out).cpu().numpy().reshape(3, 3, 32)
    assert np.array_equal(got.all(-1), np.array([[0, 1, 0], [1, 0, 0], [0, 0, 1]], dtype=bool))
    assert np.array_equal(got.any(-1), got.all(-1))


def test_offsets_past_32_bits(cuda):
    """Rows that lie more than 2^32 bytes into the cache."""
    import torch
    import ggml_b200 as g
    rows, n = 10_000_000, 1024
    cache = torch.zeros(rows, 576, dtype=torch.uint8, device="cuda")       # 5.8 GB
    x = np.random.default_rng(8).standard_normal((3, n)).astype(np.float32)
    where = np.array([rows - 1, 7_500_000, 5])
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), torch.from_numpy(where).cuda(), cache, Q4_0, err)
    out = torch.empty(3, n, device="cuda")
    g.get_rows(cache, Q4_0, torch.from_numpy(where.astype(np.int32)).cuda(), out, err)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), decode(encode(x, Q4_0), Q4_0))
    assert int(cache[where].count_nonzero().item()) == int(cache.count_nonzero().item())


def test_replayed_graph_and_side_stream(cuda):
    import torch
    import ggml_b200 as g
    x = torch.randn(5, 128, device="cuda")
    idx = torch.arange(5, device="cuda")
    cache = torch.zeros(16, 72, dtype=torch.uint8, device="cuda")
    out = torch.empty(5, 128, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    idx32 = idx.to(torch.int32)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.set_rows(x, idx, cache, Q4_0, err)
        g.get_rows(cache, Q4_0, idx32, out, err)
    x.copy_(torch.randn_like(x))
    idx.add_(9)
    idx32.add_(9)
    graph.replay()
    torch.cuda.synchronize()
    want = encode(x.cpu().numpy(), Q4_0)
    assert np.array_equal(cache[9:14].cpu().numpy(), want)
    assert np.array_equal(out.cpu().numpy(), decode(want, Q4_0))
    st = torch.cuda.Stream()
    side = torch.zeros_like(cache)
    st.wait_stream(torch.cuda.current_stream())
    g.set_rows(x, idx, side, Q4_0, err, stream=st)
    st.synchronize()
    assert np.array_equal(side[9:14].cpu().numpy(), want)


@pytest.mark.parametrize("kind", [Q4_0, Q8_0])
@pytest.mark.parametrize("n,n_rows,total", [(16384, 3, 4), (1 << 20, 1, 1), (32, 70000, 70001)])
def test_widest_and_most_rows(cuda, kind, n, n_rows, total):
    """Rows of many CTAs, many rows of one block; indices every second element of a longer vector."""
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(n_rows)
    x = rng.standard_normal((n_rows, n)).astype(np.float32)
    where = rng.permutation(total)[:n_rows].astype(np.int32)
    idx = torch.from_numpy(np.repeat(where, 2)).cuda()[::2]
    blocks = np.zeros((total, n // 32 * (34 if kind == Q8_0 else 18)), np.uint8)
    d = torch.from_numpy(blocks).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), idx, d, kind, err)
    blocks[where] = encode(x, kind)
    back = torch.empty(n_rows, n, device="cuda")
    g.get_rows(d, kind, idx, back, err)
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert np.array_equal(d.cpu().numpy(), blocks)
    assert np.array_equal(back.cpu().numpy(), decode(blocks[where], kind), equal_nan=True)
    with pytest.raises(g.B200Error, match="dev_err"):
        g.set_rows(torch.from_numpy(x).cuda(), idx, d, kind, err.float())
