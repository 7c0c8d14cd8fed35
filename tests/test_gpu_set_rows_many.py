"""SET_ROWS of many rows: the last of equal indices in linear time, with a workspace."""
import numpy as np
import pytest

from test_gpu_kv_cache import F16, F32, Q4_0, Q8_0, encode

pytestmark = pytest.mark.gpu


def last_rows(where, x, cache):
    """cache after its rows `where` are written in order."""
    rows, at = np.unique(where[::-1], return_index=True)
    cache[rows] = x[len(where) - 1 - at]
    return cache


def workspace(idx, dst):
    import torch
    import ggml_b200 as g
    return torch.full((g.set_rows_workspace_size(idx, dst),), 0x7f, dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("n,n_rows,total,kind", [(1, 524288, 300000, F16), (1, 200000, 1 << 20, F32), (32, 150001, 150, Q8_0),
                                                 (1024, 5000, 4096, Q4_0), (64, 2048, 1, Q4_0), (96, 2047, 3000, Q8_0)])
def test_the_last_of_equal_indices_stays(cuda, n, n_rows, total, kind):
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(n_rows)
    x = rng.standard_normal((n_rows, n)).astype(np.float32)
    where = rng.integers(0, total, n_rows)
    enc = encode(x, kind) if kind in (Q4_0, Q8_0) else x.astype(np.float16 if kind == F16 else np.float32)
    cache = np.zeros((total, enc.shape[1]), enc.dtype)
    d, idx = torch.from_numpy(cache).cuda(), torch.from_numpy(where).cuda()
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x).cuda(), idx, d, kind, err, workspace=workspace(idx, d))
    torch.cuda.synchronize()
    assert int(err.item()) == 0
    assert np.array_equal(d.cpu().numpy(), last_rows(where, enc, cache))


def test_slices_bad_indices_and_replays(cuda):
    """Index rows shared by slices, indices outside the cache, a captured call whose indices change."""
    import torch
    import ggml_b200 as g
    rng = np.random.default_rng(2)
    S, T, KV, n = 6, 3000, 2500, 32
    x = torch.from_numpy(rng.standard_normal((S, T, n)).astype(np.float32)).cuda()
    idx = torch.zeros(2, T, dtype=torch.int32, device="cuda")
    d = torch.zeros(S, KV, 18, dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    ws = workspace(idx, d)
    assert ws.numel() == 2 * KV * 4
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        g.set_rows(x, idx, d, Q4_0, err, workspace=ws)
    for k in range(3):
        where = rng.integers(0, KV, (2, T))
        if k == 2:
            where[0, 7], where[1, -1] = -1, KV
        idx.copy_(torch.from_numpy(where.astype(np.int32)))
        d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for s in range(S):
            ok = (where[s % 2] >= 0) & (where[s % 2] < KV)
            want = last_rows(where[s % 2][ok], encode(x[s].cpu().numpy(), Q4_0)[ok], np.zeros((KV, 18), np.uint8))
            assert np.array_equal(d[s].cpu().numpy(), want)
        assert int(err.item()) == (6 if k == 2 else 0)


def test_through_the_backend(cuda):
    """A transposed V cache: a row a value, 512 tokens of 256 values."""
    import os
    import subprocess
    import sys
    from conftest import ROOT
    child = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/ggml-rocket_b200"]
import numpy as np
import torch
import ggml_b200 as g
T, n, kv = 512, 256, 1024
be = g.Backend()
rng = np.random.default_rng(1)
x = torch.from_numpy(rng.standard_normal((T, n)).astype(np.float32)).cuda()
cells = rng.permutation(kv)[:T]
idx = torch.from_numpy((np.arange(n)[None] * kv + cells[:, None]).astype(np.int64)).cuda()
v = torch.zeros(n, kv, dtype=torch.float16, device="cuda")
a = g.make_tensor(g.F32, [1, T * n], x.data_ptr(), on_device=True)
i = g.make_tensor(g.I64, [T * n], idx.data_ptr(), on_device=True)
c = g.make_tensor(g.F16, [1, n * kv], v.data_ptr(), on_device=True)
node = g.make_tensor(g.F16, [1, n * kv], v.data_ptr(), op=g.OP_SET_ROWS, srcs=[a, i, c], on_device=True)
torch.cuda.synchronize()
assert g.supports_op(node) and be.graph_compute([node]) == g.STATUS_SUCCESS
want = np.zeros((n, kv), np.float16)
want[:, cells] = x.cpu().numpy().T.astype(np.float16)
assert np.array_equal(v.cpu().numpy(), want) and be.device_errors() == 0
be.close()
print("DONE")
"""
    env = {k: v for k, v in os.environ.items() if not k.startswith("B200_")}
    env.update(B200_GLUE="1")
    p = subprocess.run([sys.executable, "-c", child, ROOT], env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "DONE" in p.stdout, p.stdout[-2000:] + p.stderr[-2000:]
