"""The claim rules of the sectioned ROPE modes, SET_ROWS, quantised GET_ROWS and FLASH_ATTN_EXT over a Q4_0
cache: declined by default, claimed under their knobs for what the kernels take (descriptors only, no GPU)."""
import json
import os
import subprocess
import sys

from conftest import ROOT

_CHILD = r"""
import json, sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/ggml-rocket_b200"]
import ggml_b200 as g
from ggml_b200.graph import llama_layer
T = g.make_tensor
DEV = 1 << 40
def rope(mode=8, sections=(16, 24, 24, 0), n_dims=128, ptokens=12, t=g.F32, dt=None, ext=0.0, src2=None):
    x = T(t, [128, 8, 3])
    return T(t if dt is None else dt, [128, 8, 3], op=g.OP_ROPE, srcs=[x, T(g.I32, [ptokens]), src2],
             op_params=[0, n_dims, mode, 0, 4096, 10000.0, 1.0, ext, 1.0, 32.0, 1.0] + list(sections))
def set_rows(dt=g.Q4_0, n=256, rows=5, it=g.I64, dev=True, n_idx=None, st=g.F32, data=DEV, nb=None):
    a, i = T(st, [n, rows]), T(it, [rows if n_idx is None else n_idx])
    c = T(dt, [n, 100], data, on_device=dev)
    return T(dt, [n, 100], data, nb=nb, op=g.OP_SET_ROWS, srcs=[a, i, c], on_device=dev)
def get_rows(t=g.Q4_0, dev=True, n=256):
    return T(g.F32, [n, 4], op=g.OP_GET_ROWS, srcs=[T(t, [n, 100], DEV if dev else None, on_device=dev), T(g.I32, [4])])
def fa(tokens=1, kv=64, D=128, H=8, HK=2, S=1, kt=g.Q4_0, vt=g.Q4_0, dev=True, mask=True, sinks=False, bias=0.0, data=DEV, qt=g.F32, ms=None):
    be, bb = g.BLOCK[kt]
    row = D * HK // be * bb
    nb = [bb, row, D // be * bb, row * kv]
    bv, bvb = g.BLOCK[vt]
    rv = D * HK // bv * bvb
    q = T(qt, [D, tokens, H, S])
    k = T(kt, [D, kv, HK, S], data if dev else None, nb=nb, on_device=dev)
    v = T(vt, [D, kv, HK, S], data if dev else None, nb=[bvb, rv, D // bv * bvb, rv * kv], on_device=dev)
    m = T(g.F16, [kv, (tokens + 63) // 64 * 64, 1, S if ms is None else ms]) if mask else None
    return T(g.F32, [D, H, tokens, S], op=g.OP_FLASH_ATTN_EXT, srcs=[q, k, v, m, T(g.F32, [H]) if sinks else None], op_params=[0.1, bias, 0.0, 10])
r = {
    "rope": [rope(), rope(40), rope(24, (32, 32, 0, 0), 64), rope(t=g.F16)],
    "rope_no": [rope(ptokens=3), rope(sections=(0, 0, 0, 0)), rope(24), rope(ext=1.0), rope(9), rope(t=g.BF16), rope(n_dims=130),
                rope(sections=(-1, 24, 24, 0)), rope(src2=T(g.F32, [64])), rope(dt=g.F16)],
    "set": [set_rows(), set_rows(g.Q8_0), set_rows(g.F16), set_rows(g.F32, n=7), set_rows(it=g.I32),
            set_rows(nb=[18, 162, 16200, 16200])],
    "set_no": [set_rows(dev=False), set_rows(n=48), set_rows(g.Q4_K), set_rows(n_idx=4), set_rows(it=g.F32), set_rows(st=g.F16),
               set_rows(data=DEV + 1), set_rows(nb=[18, 126, 14400, 14400])],
    "get": [get_rows(), get_rows(g.Q8_0)],
    "get_no": [get_rows(dev=False), get_rows(g.Q4_K), get_rows(g.Q8_0, dev=False)],
    "fa": [fa(), fa(tokens=7, kv=1), fa(D=64, S=5), fa(tokens=600, kv=700, S=2, ms=1), fa(qt=g.F16)],
    "fa_no": [fa(D=96), fa(dev=False), fa(sinks=True), fa(bias=2.0), fa(mask=False), fa(H=7), fa(kt=g.Q8_0), fa(kt=g.F16, vt=g.F16),
              fa(data=DEV + 4), fa(S=3, ms=2)],
}
out = {k: [bool(g.supports_op(x)) for x in v] for k, v in r.items()}
top = [DEV]
def alloc(n):
    a = top[0]
    top[0] += (n + 255) // 256 * 256
    return a, True
L = llama_layer(1, alloc=alloc, rope_mode=8, rope_sections=[16, 24, 24, 0], kv_type=g.Q4_0)
out["layer"] = {x.name.decode(): bool(g.supports_op(x)) for x in L.nodes}
out["name"] = g.lib().ggml_backend_b200_op_from_name(b"SET_ROWS") == g.OP_SET_ROWS
print(json.dumps(out))
"""


def claims(**knobs):
    env = {k: v for k, v in os.environ.items() if not k.startswith("B200_")}
    env.update(knobs)
    p = subprocess.run([sys.executable, "-c", _CHILD, ROOT], env=env, capture_output=True, text=True, timeout=120)
    assert p.returncode == 0, p.stderr[-2000:]
    return json.loads(p.stdout.strip().splitlines()[-1])


def test_declined_by_default():
    r = claims()
    for kind in ("rope", "rope_no", "set", "set_no", "get", "get_no", "fa", "fa_no"):
        assert not any(r[kind]), kind
    assert r["name"]


def test_glue_claims_rope_and_rows():
    r = claims(B200_GLUE="1")
    for kind in ("rope", "set", "get"):
        assert all(r[kind]), (kind, r[kind])
        assert not any(r[kind + "_no"]), (kind, r[kind + "_no"])
    assert not any(r["fa"])


def test_quantised_cache_attention_claim():
    r = claims(B200_FA_QUANT_KV="1")
    assert all(r["fa"]) and not any(r["fa_no"]), (r["fa"], r["fa_no"])
    assert not any(r["set"])


def test_a_decode_layer_over_a_q4_0_cache_is_claimed_whole():
    r = claims(B200_GLUE="1", B200_FA_QUANT_KV="1", B200_DECODE="1")
    assert all(r["layer"].values()), r["layer"]
