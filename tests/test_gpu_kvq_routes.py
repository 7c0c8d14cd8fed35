"""Which kernel graph_compute gives FLASH_ATTN_EXT over a Q4_0 cache in device memory, and what it holds meanwhile.

Long prompts of one stream run, as over a Q8_0 cache, on the fp16 kernel over tiles made by b200_kv_to_f16, bit for
bit; shorter ones on b200_flash_attn_kvq, and so do several streams, a few at a time where their tiles are large."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

_CHILD = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/ggml-rocket_b200", sys.argv[1] + "/tests"]
import math
import torch
import ggml_b200 as g
from test_gpu_flash_attn_kvq import causal, inputs, run

be = g.Backend()
def node(q, k, v, m, out, scale):
    S, T, H, D = q.shape
    KV, HK = k.shape[1:3]
    row = HK * D // 32 * 18
    tq = g.make_tensor(g.F32, [D, T, H, S], q.data_ptr(), nb=[4, 4 * H * D, 4 * D, 4 * T * H * D], on_device=True)
    tk, tv = [g.make_tensor(g.Q4_0, [D, KV, HK, S], c.data_ptr(), nb=[18, row, D // 32 * 18, row * KV], on_device=True) for c in (k, v)]
    tm = g.make_tensor(g.F16, [KV, T, 1, S], m.data_ptr(), on_device=True)
    return g.make_tensor(g.F32, [D, H, T, S], out.data_ptr(), op=g.OP_FLASH_ATTN_EXT, srcs=[tq, tk, tv, tm],
                         op_params=[scale, 0.0, 0.0, 10], on_device=True)
def routes():
    return [be.route_ops(r) for r in ("fa", "fa_kvq", "fa_quant_kv")]
def graph(q, k, v, m, scale=0.09):
    out = torch.full(q.shape, 3.0, device="cuda")
    n = node(q, k, v, m, out, scale)
    assert g.supports_op(n)
    torch.cuda.synchronize()
    before = routes()
    assert be.graph_compute([n]) == g.STATUS_SUCCESS
    torch.cuda.synchronize()
    return out, [b - a for a, b in zip(before, routes())]
def fp16(q, k, v, m, scale=0.09):
    S, T, H, D = q.shape
    KV, HK = k.shape[1:3]
    t16 = torch.empty(2, HK, KV, D, dtype=torch.float16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    for i, c in enumerate((k, v)):
        assert g.lib().b200_kv_to_f16(2, c.data_ptr(), D, KV, HK, HK * D // 32 * 18, D // 32 * 18, t16[i].data_ptr(), st) == 0
    out, err = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = torch.empty(g.flash_attn_workspace_size(D, D, T, H, KV, HK), dtype=torch.uint8, device="cuda")
    g.flash_attn_ext(q, 4 * H * D, 4 * D, t16[0], 2 * D, 2 * KV * D, t16[1], 2 * D, 2 * KV * D, m, 2 * KV, out, D, D, T, H, KV,
                     HK, scale, 0.0, ws, err)
    torch.cuda.synchronize()
    return out

if sys.argv[2] == "routes":
    for T, H, HK, D, KV in ((512, 32, 8, 128, 2048), (300, 32, 8, 128, 1024), (64, 32, 8, 128, 1000 + 24), (2048, 14, 2, 64, 2048)):
        q, k, v = inputs(1, T, H, HK, D, KV)
        m = causal(1, T, KV)
        out, by = graph(q, k, v, m)
        assert by == [1, 0, 1], (T, H, KV, by)
        assert torch.equal(out, fp16(q, k, v, m))
    for S, T, H, HK, D, KV in ((1, 1, 32, 8, 128, 300), (1, 40, 8, 2, 128, 1024), (1, 64, 32, 8, 128, 4096), (2, 600, 32, 8, 64, 1100),
                               (1, 512, 32, 8, 128, 1023)):
        q, k, v = inputs(S, T, H, HK, D, KV)
        m = causal(S, T, KV)
        out, by = graph(q, k, v, m)
        assert by == [1, 1, 0], (S, T, H, KV, by)
        assert torch.equal(out, run(q, k, v, m, 0.09))
elif sys.argv[2] == "garbage":
    # cells no row sees, and one the last token alone does, of bytes that decode to NaN and infinity
    T, H, HK, D, KV = 512, 32, 8, 128, 2048
    q, k, v = inputs(1, T, H, HK, D, KV)
    m = causal(1, T, KV, [1500])
    clean, by = graph(q, k, v, m)
    assert by == [1, 0, 1]
    k[:, 1500:], v[:, 1500:] = 0xff, 0xff
    k[:, 1600:1700, :, 1::18], v[:, 1600:1700, :, 1::18] = 0x7c, 0x7c
    v[:, 1700:1800, :, 1::18] = 0x7a               # scales of fp16's largest size: code * scale is past its range
    assert torch.equal(graph(q, k, v, m)[0], clean)
    v[0, 1499, 2, 0], v[0, 1499, 2, 1] = 0xff, 0x7f
    got = graph(q, k, v, m)[0]
    assert torch.equal(got[:, :T - 1], clean[:, :T - 1])
    assert bool(torch.isnan(got[0, T - 1, 8:12]).all())
    got[0, T - 1, 8:12] = clean[0, T - 1, 8:12]
    assert torch.equal(got, clean)
else:
    # sixteen streams whose tiles would take 4.4 GB
    S, T, H, HK, D, KV = 16, 13, 32, 8, 128, 32768
    q, k, v = inputs(S, T, H, HK, D, KV)
    m = causal(S, T, KV, [KV - 1000 * s for s in range(S)])
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    out, by = graph(q, k, v, m)
    held = free - torch.cuda.mem_get_info()[0]
    assert by == [1, 1, 0] and held < (3 << 30), (by, held)
    for s in (0, 7, 8, 15):
        one = run(q[s:s + 1], k[s:s + 1], v[s:s + 1], m[s:s + 1], 0.09)
        assert float((one - out[s:s + 1]).abs().max()) < 2e-5 * 4
be.close()
print("DONE")
"""


@pytest.mark.parametrize("what", ["routes", "garbage", "memory"])
def test_routes_and_memory(cuda, what):
    env = {k: v for k, v in os.environ.items() if not k.startswith("B200_")}
    env.update(B200_FA_QUANT_KV="1")
    p = subprocess.run([sys.executable, "-c", _CHILD, ROOT, what], env=env, capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-3000:]
    assert "DONE" in p.stdout
