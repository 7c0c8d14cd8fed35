"""Q4_0 codes next to a border: SET_ROWS takes the code of the exact x / d + 8.5 (1 / d an f32 number), which an
encoder that rounds the product and the sum to f32 misses by one for a few values in ten million."""
import numpy as np
import pytest

from test_gpu_kv_cache import Q4_0, encode

pytestmark = pytest.mark.gpu


def test_codes_next_to_a_border(cuda):
    import torch
    import ggml_b200 as g
    x = np.random.default_rng(11).standard_normal((1 << 18, 64)).astype(np.float32)      # 16.8 million values
    v = x.reshape(-1, 32)
    m = np.take_along_axis(v, np.abs(v).argmax(1)[:, None], 1)
    inv = np.float32(1) / (m / np.float32(-8))
    exact = np.minimum(np.trunc(v.astype(np.float64) * inv.astype(np.float64) + 8.5), 15)
    rounded = np.minimum(np.trunc((v * inv) + np.float32(8.5)), 15)
    apart = exact != rounded
    assert 0 < apart.sum() < 100 and np.abs(exact - rounded).max() == 1
    rows = np.unique(np.nonzero(apart)[0] // 2)
    d = torch.zeros(len(rows), 36, dtype=torch.uint8, device="cuda")
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    g.set_rows(torch.from_numpy(x[rows]).cuda(), torch.arange(len(rows), device="cuda"), d, Q4_0, err)
    assert np.array_equal(d.cpu().numpy(), encode(x[rows], Q4_0))
    # the exact code is the nearer one where both are representable
    at = np.nonzero(apart)
    t = v[at].astype(np.float64) * inv[at[0], 0].astype(np.float64) + 8
    assert np.all(np.abs(t - exact[at]) <= np.abs(t - rounded[at]))
