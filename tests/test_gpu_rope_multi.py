"""ROPE with several position axes (b200_rope_multi) on the GPU against its formula in 64 bits.

Tolerance, per element: the kernel rounds the reduced angle (in half turns, at most 1) to f32, off by
pi 2^-25 < 1e-7, its sine and cosine are within 2 ulp (1.2e-7) and take attn_factor with one rounding
(6e-8); the two products and their sum round three times (2^-24 each). Each factor is so within 3.5e-7
of the exact one (times attn_factor), and y within 6e-7 attn (|x0| + |x1|). f16 results add half a step:
2^-11 of the value, 2^-25 in the subnormal range."""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def reference(x, pos, n_dims, mode, sections, base, freq_scale, attn):
    """x [batch, tokens, heads, dim] f64, pos [4, tokens]; y and |x0| + |x1| per element."""
    y, mag = x.copy(), np.zeros_like(x)
    starts = np.concatenate([[0], np.cumsum(sections)])
    pairs = n_dims if mode == 24 else n_dims // 2
    for i in range(pairs):
        sec = i % starts[4]
        if mode == 40:
            axis = sec % 3
            axis = axis if sec < 3 * sections[axis] else 3
        else:
            axis = int(np.searchsorted(starts, sec, side="right")) - 1
        step = sec - starts[axis] if mode == 24 else i
        th = pos[axis].astype(np.float64) * freq_scale * float(base) ** (-2.0 * step / n_dims)
        c, s = attn * np.cos(th)[None, :, None], attn * np.sin(th)[None, :, None]
        x0, x1 = x[..., i], x[..., i + pairs]
        y[..., i], y[..., i + pairs] = x0 * c - x1 * s, x0 * s + x1 * c
        mag[..., i] = mag[..., i + pairs] = np.abs(x0) + np.abs(x1)
    return y, mag


def run(x, pos, n_dims, mode, sections, base, freq_scale=1.0, attn=1.0, out=None, stream=None):
    import torch
    import ggml_b200 as g
    out = torch.empty(x.shape, dtype=x.dtype, device="cuda") if out is None else out
    g.rope_multi(x, pos, out, n_dims, mode, sections, freq_base=base, freq_scale=freq_scale, attn_factor=attn,
                 stream=stream)
    torch.cuda.synchronize()
    return out


def check(got, x, pos, n_dims, mode, sections, base, freq_scale=1.0, attn=1.0):
    x64 = x.double().cpu().numpy()
    x64 = x64.reshape((1,) * (4 - x64.ndim) + x64.shape)
    y, mag = reference(x64, pos.cpu().numpy(), n_dims, mode, sections, base, freq_scale, attn)
    half = str(x.dtype) == "torch.float16"
    tol = 6e-7 * abs(attn) * mag + (2.0 ** -11 * np.abs(y) + 2.0 ** -25 if half else 0)
    got = got.double().cpu().numpy().reshape(y.shape)
    assert np.all(np.abs(got - y) <= tol), float(np.max(np.abs(got - y) - tol))


CASES = [
    # tokens, heads, dim, n_dims, mode, sections
    (1, 1, 64, 64, 8, [8, 12, 12, 0]),
    (7, 3, 128, 128, 8, [16, 24, 24, 0]),
    (300, 32, 128, 128, 40, [24, 20, 20, 0]),
    (129, 8, 128, 64, 8, [8, 8, 8, 8]),            # values past n_dims copied, all four axes
    (33, 5, 96, 80, 40, [10, 10, 10, 10]),
    (73, 16, 80, 40, 24, [20, 20, 0, 0]),
    (5, 2, 72, 36, 24, [9, 9, 9, 9]),              # four sections, frequencies restart in each
    (17, 3, 66, 62, 8, [5, 7, 3, 0]),              # sections shorter than the head: they repeat; odd alignment
    (2, 1, 4096, 2048, 8, [300, 400, 324, 0]),     # the widest head and the most pairs
    (1500, 1, 2, 2, 8, [1, 0, 0, 0]),              # one pair a head
]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,n_dims,mode,sections", CASES)
def test_against_formula(cuda, tokens, heads, dim, n_dims, mode, sections, half):
    import torch
    gen = torch.Generator().manual_seed(tokens * 31 + dim)
    x = torch.randn(tokens, heads, dim, generator=gen).to(torch.float16 if half else torch.float32).cuda()
    pos = torch.randint(0, 1 << 20, (4, tokens), generator=gen).to(torch.int32).cuda()
    got = run(x, pos, n_dims, mode, sections, 1e6)
    check(got, x, pos, n_dims, mode, sections, 1e6)


def test_scales_negative_and_largest_positions(cuda):
    import torch
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(6, 4, 64, generator=gen).cuda()
    pos = torch.tensor([[0, 1, -5, 2147483647, -2147483648, 99]] * 4, dtype=torch.int32).cuda()
    got = run(x, pos, 64, 8, [10, 10, 12, 0], 10000.0, freq_scale=0.25, attn=1.5)
    check(got, x, pos, 64, 8, [10, 10, 12, 0], 10000.0, freq_scale=0.25, attn=1.5)


@pytest.mark.parametrize("half", [False, True])
def test_strides_batch_in_place_and_streams(cuda, half):
    import torch
    gen = torch.Generator().manual_seed(5)
    dt = torch.float16 if half else torch.float32
    pos = torch.randint(0, 5000, (4, 9), generator=gen).to(torch.int32).cuda()
    sec = [16, 24, 24, 0]
    wide = torch.randn(2, 9, 6, 200, generator=gen).to(dt).cuda()
    view = wide[:, :, 1:5, 3:131]                                  # rows off 16-byte alignment, heads inside a wider row
    check(run(view, pos, 128, 40, sec, 1e4), view, pos, 128, 40, sec, 1e4)
    by_head = torch.randn(2, 4, 9, 128, generator=gen).to(dt).cuda().transpose(1, 2)   # heads outside tokens
    check(run(by_head, pos, 128, 40, sec, 1e4), by_head, pos, 128, 40, sec, 1e4)
    x = torch.randn(2, 9, 4, 128, generator=gen).to(dt).cuda()
    want = run(x, pos, 128, 8, sec, 1e4)
    inplace = x.clone()
    run(inplace, pos, 128, 8, sec, 1e4, out=inplace)
    assert torch.equal(inplace, want)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    assert torch.equal(run(x, pos, 128, 8, sec, 1e4, stream=st), want)
    with torch.cuda.stream(st):
        assert torch.equal(run(x, pos, 128, 8, sec, 1e4), want)


def test_nan_and_inf_stay_in_their_pair(cuda):
    import torch
    x = torch.ones(2, 2, 64, device="cuda")
    x[0, 1, 5], x[1, 0, 40] = float("nan"), float("inf")
    pos = torch.full((4, 2), 7, dtype=torch.int32, device="cuda")
    got = run(x, pos, 64, 8, [10, 10, 12, 0], 1e4)
    bad = ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    want[0, 1, 5] = want[0, 1, 37] = want[1, 0, 40] = want[1, 0, 8] = True
    assert torch.equal(bad, want)


def test_replayed_graph_reads_new_inputs(cuda):
    import torch
    import ggml_b200 as g
    x = torch.randn(11, 4, 128, device="cuda")
    pos = torch.arange(44, dtype=torch.int32, device="cuda").reshape(4, 11).contiguous()
    out = torch.empty_like(x)
    run(x, pos, 128, 8, [16, 24, 24, 0], 1e4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.rope_multi(x, pos, out, 128, 8, [16, 24, 24, 0], freq_base=1e4)
    x.copy_(torch.randn_like(x))
    pos.add_(1000)
    graph.replay()
    torch.cuda.synchronize()
    check(out, x, pos, 128, 8, [16, 24, 24, 0], 1e4)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,n_dims,mode,sections", [
    (1, 700, 64, 64, 40, [11, 11, 10, 0]),         # many heads of one token
    (20000, 1, 32, 32, 8, [6, 5, 5, 0]),           # many tokens of one head
    (2, 2, 4096, 64, 8, [16, 8, 8, 0]),            # nearly all of the head copied
    (9, 3, 2048, 1024, 24, [512, 512, 0, 0]),
])
def test_sizes_at_the_ends(cuda, tokens, heads, dim, n_dims, mode, sections, half):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(tokens + dim)
    x = torch.randn(tokens, heads, dim, device="cuda", generator=gen)
    x = x.half() if half else x
    pos = torch.randint(0, 200000, (4, tokens), device="cuda", generator=gen, dtype=torch.int32)
    check(run(x, pos, n_dims, mode, sections, 1e6), x, pos, n_dims, mode, sections, 1e6)
