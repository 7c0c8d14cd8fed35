"""How near b200_flash_attn_kvq comes to its definition in 64 bits, whichever kernel takes the call.

Tolerance, per element. Let A be the largest scale * sum_i |q_i k_i| of a row, B the same with the row's
largest |q| in the place of q_i, V the largest |v|, N the number of keys.
- q lies in two fp16 halves: what they leave is 2^-22 of the row's largest value, B 2^-22 of a score.
- The exact products are added in fp32, the tensor core truncating: at most 32 steps of 2^-23 of A, with the
  product of the two low halves left out (2^-22 A) and the roundings of scale, cap and log2(e) well inside.
- ex2 is within 2^-22; a weight's two halves leave 2^-22 of it; the row's sum rounds a few times.
So a weight is off by e = A 2^-18 + B 2^-22 + 2^-20, relative. Outputs are ratios of two sums of such weights:
2 e V, and the sums are added in at most 3 N / 16 + 32 steps of 2^-23 of V. An f16 result adds its own rounding,
half a step: 2^-11 of the value, 2^-25 in the subnormal range."""
import math

import pytest

from test_gpu_flash_attn_kvq import check as loose
from test_gpu_flash_attn_kvq import causal, decode64, inputs, reference, run

pytestmark = pytest.mark.gpu


def check(out, q, k, v, mask, scale, softcap=0.0, key=None):
    import torch
    want, A, vmax = reference(q, k, v, mask, scale, softcap)
    G = q.shape[2] // k.shape[2]
    ks = decode64(k).abs().sum(-1).amax(1).repeat_interleave(G, 1)          # [S, H]: sum |k_i| of the largest key
    B = abs(scale) * q.double().abs().amax(-1) * ks[:, None]                # [S, T, H]
    e = A * 2.0 ** -18 + B[..., None] * 2.0 ** -22 + 2.0 ** -20
    tol = (2 * e + (3 * k.shape[1] / 16 + 32) * 2.0 ** -23) * vmax
    if out.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -25
    d = (out.double() - want).abs()
    assert bool((d <= tol).all()), (float((d - tol).max()), float((d / tol).max()))


@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", [
    (40, 1, 8, 2, 128, 3),
    (40, 1, 8, 2, 64, 9),
    (40, 2, 8, 2, 128, 8),           # rows of two tokens in a tile
    (40, 1, 3, 1, 128, 5),           # a head alone in its cache row
])
def test_f16_results_of_few_rows_lose_their_own_rounding_alone(cuda, S, T, H, HK, D, KV, q_f16):
    """Few keys, so that the softmax weights' rounding does not average out."""
    q, k, v = inputs(S, T, H, HK, D, KV, seed=3, q_f16=q_f16)
    check(run(q, k, v, None, 1 / 128, True), q, k, v, None, 1 / 128)


@pytest.mark.parametrize("T", [1, 60])
def test_queries_at_the_end_of_f32(cuda, T):
    """The largest |q| at 2^127 and above, and among f32's smallest, with a scale that brings them back."""
    q, k, v = inputs(1, T, 8, 2, 128, 300)
    for qq, scale in ((q.sign() * 3e38, 1e-39), (q / q.abs().max() * 3.4e38, 2e-39), (q * 1e-38, 1e37)):
        loose(run(qq, k, v, None, scale), qq, k, v, None, scale)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("q_f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", [
    (1, 100, 4, 1, 128, 5),
    (2, 60, 4, 2, 64, 9),
    (1, 64, 8, 2, 128, 129),
    (1, 200, 32, 8, 128, 1000),
    (2, 130, 14, 2, 64, 700),        # a head a tile
    (3, 17, 8, 2, 128, 2000),        # the keys of a tile over several CTAs
    (1, 700, 64, 8, 128, 900),       # whole tiles, then cut ones
    (1, 512, 8, 2, 128, 4096),
])
def test_prompts_keep_what_the_row_kernels_keep(cuda, S, T, H, HK, D, KV, q_f16, f16):
    q, k, v = inputs(S, T, H, HK, D, KV, seed=3, q_f16=q_f16)
    m = causal(S, T, KV) if T <= KV else None
    for scale in (1 / 128, 1 / math.sqrt(D)):
        check(run(q, k, v, m, scale, f16), q, k, v, m, scale)
    check(run(q, k, v, None, -0.02, f16), q, k, v, None, -0.02)


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("cap", [1e5, 1000.0, 30.0, 2.0])
def test_softcap(cuda, T, cap):
    """tanhf is within 2^-22 of its value, the cap far above the scores too."""
    q, k, v = inputs(2, T, 8, 2, 128, 20, seed=4)
    for scale in (1 / 128, 0.3):
        check(run(q, k, v, None, scale, softcap=cap), q, k, v, None, scale, softcap=cap)


@pytest.mark.parametrize("T,KV", [(1, 700), (70, 700), (40, 9000)])
def test_masks_far_from_zero(cuda, T, KV):
    """Mask values whose sum with a score is no f32 number: a row's weights are those of the differences."""
    import torch
    q, k, v = inputs(1, T, 8, 2, 128, KV, seed=6)
    m = torch.full((1, T, KV), -65504.0, dtype=torch.float16, device="cuda")
    check(run(q, k, v, m, 0.05), q, k, v, m, 0.05)
    gen = torch.Generator(device="cuda").manual_seed(T)
    m[:, :, ::3] = float("-inf")
    m[:, 1::4, 100:300] = -65472.0                       # 32 above the lowest
    m[:, 2::4] = -30000 - 16 * torch.randint(0, 3, (KV,), device="cuda", generator=gen).half()
    m[:, 3::4, 400:] = 0
    check(run(q, k, v, m, 0.05), q, k, v, m, 0.05)


@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("S,T,H,HK,D,KV", [
    (1, 1, 40, 1, 128, 777),
    (1, 33, 1, 1, 64, 33),
    (2, 1, 33, 1, 64, 5),
    (1, 17, 2, 1, 128, 1),
    (1, 12, 8, 2, 128, 700),         # 48 rows a KV head, the last size whatever the group
    (2, 16, 14, 2, 64, 900),         # 112 of them in groups of seven
    (1, 5, 56, 8, 128, 3000),
    (1, 13, 8, 2, 128, 700),         # 52: the prompt kernel
    (3, 1, 32, 8, 128, 2500),
    (1, 3, 24, 3, 64, 5003),
])
def test_either_side_of_the_row_kernels_last_size(cuda, S, T, H, HK, D, KV, f16):
    """One bound for both kernels, whichever takes the call."""
    import torch
    q, k, v = inputs(S, T, H, HK, D, KV, seed=5, q_f16=f16)
    gen = torch.Generator(device="cuda").manual_seed(S + T + KV)
    m = torch.randn(S, T, KV, device="cuda", generator=gen).half()
    m[torch.rand(S, T, KV, device="cuda", generator=gen) < 0.5] = float("-inf")
    m[:, 1:, -1] = 0.0
    m[:, 0] = float("-inf")
    for mask in (m, None):
        check(run(q, k, v, mask, 1 / math.sqrt(D), f16), q, k, v, mask, 1 / math.sqrt(D))


def test_streams_inside_keys(cuda):
    """A cache whose streams lie side by side in a key's row: the stride of a stream below that of a key."""
    S, T, H, HK, D, KV = 3, 1, 8, 2, 128, 300
    q, k, v = inputs(S, T, H, HK, D, KV)
    kk, vv = (c.transpose(0, 1).contiguous().transpose(0, 1) for c in (k, v))
    assert kk.stride(0) < kk.stride(1)
    check(run(q, kk, vv, None, 0.1), q, k, v, None, 0.1)
    q, _, _ = inputs(S, 70, H, HK, D, KV)
    check(run(q, kk, vv, None, 0.1), q, k, v, None, 0.1)


@pytest.mark.parametrize("S,T,H,HK,D,KV", [(1, 70, 8, 2, 128, 3000), (2, 300, 32, 8, 64, 700)])
def test_prompts_repeat_exactly_and_replay(cuda, S, T, H, HK, D, KV):
    """Whole tiles, and tiles whose keys CTAs share; nothing is expected of the workspace's bytes."""
    import torch
    import ggml_b200 as g
    from test_gpu_flash_attn_kvq import workspace
    q, k, v = inputs(S, T, H, HK, D, KV)
    m = causal(S, T, KV)
    want = run(q, k, v, m, 0.1)
    assert all(torch.equal(run(q, k, v, m, 0.1), want) for _ in range(3))
    out, ws = torch.empty_like(q), workspace(D, T, H, KV, HK, S)
    ws.fill_(0xff)
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.flash_attn_kvq(2, q, k, v, m, out, 0.1, ws, err)
    for seed in (5, 6):
        for a, b in zip((q, k, v), inputs(S, T, H, HK, D, KV, seed=seed)):
            a.copy_(b)
        m.copy_(causal(S, T, KV, [KV - 100 * s - seed for s in range(S)]))
        graph.replay()
        torch.cuda.synchronize()
        assert int(err.item()) == 0 and torch.equal(out, run(q, k, v, m, 0.1))
        check(out, q, k, v, m, 0.1)
