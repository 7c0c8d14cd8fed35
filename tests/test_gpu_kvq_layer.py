"""A decoder layer over a Q4_0 cache with sectioned rotary positions, through graph_compute: a prompt,
then single tokens. Norm, Q/K/V, ROPE (MROPE) of q and k, SET_ROWS of the new K / V rows into scattered
cells of the cache, FLASH_ATTN_EXT over the cache as it is stored, output projection, FFN.

Each of the run's stages is checked against its definition on what the stage before it left in the device
buffer: rotated rows within the rope's f32 bound, the cache bytes exactly, attention against 64 bits over
the cache's own bytes; then the layer's output against the oracle composed from that attention (cosine >=
0.999, max |err| / max |ref| <= 1e-2, the layer bar of the repository's other layer test)."""
import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

_CHILD = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/ggml-rocket_b200", sys.argv[1] + "/tests"]
import numpy as np
import ggml_b200 as g
import oracle
from ggml_b200 import quants
from ggml_b200.graph import llama_layer
from conftest import rel_err, rk_compare
from test_gpu_kv_cache import encode, decode
from test_gpu_rope_multi import reference as rope_ref

E, F, H, HK, D, n_kv = 1024, 2816, 8, 2, 128, 1024
eps, base, sections = 1e-5, 500000.0, [16, 24, 24, 0]
be = g.Backend()
buf = g.DeviceBuffer(be, 256 << 20)
top = [0]
def alloc(n):
    off = top[0]
    top[0] += (n + 255) // 256 * 256
    assert top[0] <= buf.size
    return buf.base + off, True
off = lambda t: t.data - buf.base
def get(t, shape, dtype=np.float32):
    a = np.zeros(shape, dtype)
    assert buf.get(off(t), a) == 0
    return a
rng = np.random.default_rng(0xCAC4E)
W = {}
cache = {k: np.full((n_kv, HK * D // 32 * 18), 0xff, np.uint8) for k in "kv"}      # never written: no numbers
order = rng.permutation(n_kv)                                                      # the cells, in the order they fill
used = 0
for T in (40, 1, 1, 3):
    L = llama_layer(T, E=E, F=F, H=H, HK=HK, D=D, n_kv=n_kv, wtype=g.Q4_K, eps=eps, rope_base=base, alloc=alloc,
                    rope_mode=g.ROPE_MROPE, rope_sections=sections, kv_type=g.Q4_0)
    for nd in L.nodes:
        assert g.supports_op(nd), nd.name
    by = {nd.name.decode(): nd for nd in L.nodes}
    x = rng.standard_normal((T, E), dtype=np.float32)
    pos = rng.integers(0, 40000, (4, T)).astype(np.int32)
    cells = order[used:used + T].astype(np.int64)
    used += T
    mask = np.full((L.inputs["mask"].ne[1], n_kv), -np.inf, np.float32)
    for t in range(T):
        mask[t, order[:used - T + t + 1]] = 0.0
    m16 = mask.astype(np.float16)
    for name, a in (("x", x), ("pos", pos), ("mask", m16.view(np.uint16)), ("kv_cells", cells)):
        assert buf.set(off(L.inputs[name]), a) == 0
    for k in "kv":
        assert buf.set(off(L.caches[k]), cache[k]) == 0
    for name, t in L.weights.items():
        if name not in W:
            W[name] = (1.0 + 0.1 * rng.standard_normal(t.ne[0])).astype(np.float32) if t.type == g.F32 else \
                quants.quantize(g.Q4_K, (rng.standard_normal((t.ne[1], t.ne[0])) * 0.02).astype(np.float32))
        assert buf.set(off(t), W[name]) == 0
    assert be.graph_compute(L.nodes) == g.STATUS_SUCCESS
    # rotary positions
    rot = {}
    for raw, out, heads in (("Qcur", "Qcur_rope", H), ("Kcur", "Kcur_rope", HK)):
        src = get(by[raw], (T, heads, D)).astype(np.float64)
        y, mag = rope_ref(src[None], pos, D, g.ROPE_MROPE, sections, base, 1.0, 1.0)
        rot[raw] = get(by[out], (T, heads, D))
        assert np.all(np.abs(rot[raw] - y[0]) <= 6e-7 * mag[0])
    # the cache
    v = get(by["Vcur"], (T, HK * D))
    for k, rows in (("k", rot["Kcur"].reshape(T, -1)), ("v", v)):
        cache[k][cells] = encode(rows, 2)
        assert np.array_equal(get(L.caches[k], cache[k].shape, np.uint8), cache[k])
    # attention over what the cache holds
    att = get(by["kqv_out"], (T, H, D))
    want = np.zeros((T, H, D))
    live = np.sort(order[:used])
    kd = decode(cache["k"][live], 2).astype(np.float64).reshape(-1, HK, D)
    vd = decode(cache["v"][live], 2).astype(np.float64).reshape(-1, HK, D)
    for h in range(H):
        s = rot["Qcur"][:, h].astype(np.float64) @ kd[:, h // (H // HK)].T / np.sqrt(D) + mask[:T, live]
        p = np.exp(s - s.max(1, keepdims=True))
        want[:, h] = p @ vd[:, h // (H // HK)] / p.sum(1, keepdims=True)
    # at most 32 rows a KV head: fp32 accuracy; the prompt: fp16 operands (2^-11 of every value, twice over)
    tol = (2e-5 if T * H // HK <= 32 else 4e-3) * np.abs(vd).max()
    assert np.abs(att - want).max() <= tol, (T, np.abs(att - want).max(), tol)
    # the rest of the layer
    def mm(name, a):
        t = L.weights[name]
        return oracle.mul_mat(g.Q4_K, W[name], t.ne[1], t.ne[0], a)
    h = mm("attn_output", att.reshape(T, E)) + x
    fn = oracle.rms_norm(h, eps) * W["ffn_norm"][None, :]
    ref = mm("ffn_down", oracle.swiglu(mm("ffn_gate", fn), mm("ffn_up", fn))) + h
    got = get(L.out, (T, E))
    cos, bad = rk_compare(ref, got)
    assert rel_err(got, ref) <= 1e-2 and cos >= 0.999 and bad == 0, (T, rel_err(got, ref), cos, bad)
assert be.cpu_fallbacks() == 0 and be.device_errors() == 0
print("ROUTES", be.route_ops("fa_kvq"), be.route_ops("fa"))
# an index past the cache fails the graph and leaves the cache alone
assert buf.set(off(L.inputs["kv_cells"]), np.array([3, n_kv, 5], np.int64)) == 0
nodes = [by["k_cache_set"]]
before = get(L.caches["k"], cache["k"].shape, np.uint8)
assert be.graph_compute(nodes) == g.STATUS_FAILED and be.device_errors() == 1
after = get(L.caches["k"], cache["k"].shape, np.uint8)
keep = np.ones(n_kv, bool)
keep[[3, 5]] = False
assert np.array_equal(before[keep], after[keep])
# cache rows read back through GET_ROWS
idx = np.array([order[0], order[5], order[0]], np.int32)
data, _ = alloc(idx.nbytes)
ti = g.make_tensor(g.I32, [3], data, on_device=True)
data, _ = alloc(3 * HK * D * 4)
to = g.make_tensor(g.F32, [HK * D, 3], data, op=g.OP_GET_ROWS, srcs=[L.caches["v"], ti], on_device=True)
assert buf.set(off(ti), idx) == 0
assert g.supports_op(to) and be.graph_compute([to]) == g.STATUS_SUCCESS
assert np.array_equal(get(to, (3, HK * D)), decode(cache["v"][idx], 2))
buf.free()
be.close()
print("DONE")
"""


def test_layer_over_a_q4_0_cache(cuda):
    env = {k: v for k, v in os.environ.items() if not k.startswith("B200_")}
    env.update(B200_GLUE="1", B200_FA_QUANT_KV="1", B200_DECODE="1")
    p = subprocess.run([sys.executable, "-c", _CHILD, ROOT], env=env, capture_output=True, text=True, timeout=600)
    assert p.returncode == 0, p.stdout[-3000:] + p.stderr[-3000:]
    kvq, fa = [int(v) for v in p.stdout.split("ROUTES")[1].split()[:2]]
    assert kvq == 4 and fa == 4
    assert "DONE" in p.stdout
