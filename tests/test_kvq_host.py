"""Refusals of the rope-with-sections, cache-write and 4-bit attention entry points: arguments are checked
before any CUDA call, so a malformed call gets its status on a host without a GPU."""
import ctypes

import ggml_b200 as g

P = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 1)
BAD, NO, WS = g.B200_E_INVALID, g.B200_E_UNSUPPORTED, g.B200_E_WORKSPACE


def ne(*v):
    return (ctypes.c_int64 * 4)(*(list(v) + [1] * (4 - len(v))))


def nb(*v):
    return (ctypes.c_size_t * 4)(*v)


def test_rope_multi():
    lib = g.lib()

    def call(type=0, x=P, shape=(128, 4, 3), strides=(4, 512, 2048, 6144), pos=P, n_dims=128, mode=8,
             sections=(16, 24, 24, 0), base=1e4, dst=P):
        s = None if sections is None else (ctypes.c_int32 * 4)(*sections)
        return lib.b200_rope_multi(type, x, ne(*shape), nb(*strides), pos, n_dims, mode, s, base, 1.0, 1.0, dst, None)

    assert call(x=None) == BAD and call(pos=None) == BAD and call(dst=None) == BAD and call(sections=None) == BAD
    assert call(shape=(128, 0, 3)) == BAD and call(n_dims=0) == BAD and call(n_dims=3) == BAD
    assert call(n_dims=130) == BAD and call(base=0.0) == BAD and call(sections=(0, 0, 0, 0)) == BAD
    assert call(sections=(16, -1, 24, 0)) == BAD
    assert call(mode=24) == BAD                                # VISION rotates the whole head
    assert call(mode=0) == NO and call(mode=2) == NO           # b200_rope's modes
    assert call(type=8) == NO and call(x=ODD) == NO and call(dst=ODD) == NO
    assert call(strides=(8, 512, 2048, 6144)) == NO and call(strides=(4, 514, 2048, 6144)) == NO
    assert call(shape=(8192, 4, 3), n_dims=4096) == NO         # more pairs than a CTA's table holds


def test_set_rows_and_get_rows():
    lib = g.lib()

    def call(src=P, sne=(64, 5), snb=(4, 256, 1280, 1280), it=27, idx=P, ine=(5,), inb=(8, 40, 40, 40), dt=2, dst=P,
             dne=(64, 9), dnb=(18, 36, 324, 324), err=P):
        return lib.b200_set_rows(src, ne(*sne), nb(*snb), it, idx, ne(*ine), nb(*inb), dt, dst, ne(*dne), nb(*dnb), err, None)

    assert call(src=None) == BAD and call(idx=None) == BAD and call(dst=None) == BAD and call(err=None) == BAD
    assert call(sne=(64, 0)) == BAD and call(dne=(96, 9)) == BAD and call(ine=(4,)) == BAD
    assert call(sne=(48, 5), dne=(48, 9)) == BAD               # whole blocks
    assert call(sne=(64, 5, 3), dne=(64, 9, 3), ine=(5, 2)) == BAD   # three slices, two index rows
    assert call(dt=12) == NO and call(dt=30) == NO and call(it=1) == NO
    assert call(dnb=(2, 36, 324, 324)) == NO and call(dnb=(18, 37, 324, 324)) == NO and call(dst=ODD) == NO
    assert call(snb=(8, 256, 1280, 1280)) == NO and call(src=ctypes.c_void_p((1 << 20) + 2)) == NO
    assert call(inb=(4, 40, 40, 40)) == NO

    def get(t=2, sne=(64, 9), snb=(18, 36, 324, 324), src=P):
        return lib.b200_get_rows(t, src, ne(*sne), nb(*snb), P, ne(5), nb(4, 20, 20, 20), P, P, None)

    assert get(sne=(48, 9)) == BAD and get(t=12) == NO and get(snb=(34, 36, 324, 324)) == NO and get(src=ODD) == NO
    assert get(t=8) == NO and get(snb=(18, 35, 324, 324)) == NO


def test_flash_attn_kvq():
    lib = g.lib()
    size = lib.b200_flash_attn_kvq_workspace_size
    assert size(128, 1, 32, 4096, 8, 1) > 0 and size(96, 1, 32, 4096, 8, 1) == 0 and size(128, 1, 30, 4096, 8, 1) == 0
    assert size(128, 0, 32, 4096, 8, 1) == 0 and size(128, 1, 32, 0, 8, 1) == 0

    def call(kt=2, qt=0, q=P, qne=(128, 1, 32, 1), qnb=(4, 16384, 512, 16384), k=P, kne=(128, 64, 8, 1),
             knb=(18, 576, 72, 36864), v=P, vne=(128, 64, 8, 1), vnb=(18, 576, 72, 36864), mask=P,
             mnb=(2, 128, 128, 128), dt=0, dst=P, ws=P, wsb=1 << 30, err=P):
        return lib.b200_flash_attn_kvq(kt, qt, q, ne(*qne), nb(*qnb), k, ne(*kne), nb(*knb), v, ne(*vne), nb(*vnb), mask,
                                       nb(*mnb), dt, dst, 0.1, 0.0, ws, wsb, err, None)

    for name in ("q", "k", "v", "dst", "err"):
        assert call(**{name: None}) == BAD
    assert call(qne=(128, 0, 32, 1)) == BAD and call(kne=(128, 0, 8, 1)) == BAD and call(kne=(64, 64, 8, 1)) == BAD
    assert call(vne=(128, 65, 8, 1)) == BAD and call(vne=(128, 64, 4, 1)) == BAD and call(kne=(128, 64, 8, 2)) == BAD
    assert call(qne=(128, 1, 30, 1)) == BAD and call(vne=(64, 64, 8, 1)) == BAD
    assert call(kt=8) == NO and call(kt=1) == NO and call(qt=30) == NO and call(dt=30) == NO
    assert call(qne=(96, 1, 32, 1), kne=(96, 64, 8, 1), vne=(96, 64, 8, 1)) == NO
    assert call(qnb=(8, 16384, 512, 16384)) == NO and call(q=ctypes.c_void_p((1 << 20) + 2)) == NO
    assert call(knb=(18, 574, 72, 36864)) == NO and call(v=ctypes.c_void_p((1 << 20) + 4)) == NO
    assert call(mnb=(4, 128, 128, 128)) == NO and call(mask=ODD) == NO and call(dst=ctypes.c_void_p((1 << 20) + 2)) == NO
    assert call(kne=(128, 1 << 31, 8, 1), vne=(128, 1 << 31, 8, 1)) == NO
    assert call(ws=None) == WS and call(wsb=16) == WS and call(ws=ctypes.c_void_p((1 << 20) + 16)) == WS


def test_sizes_past_the_counters():
    """Sizes whose grids or 32-bit counters would not hold the work have no workspace and are refused."""
    size = g.lib().b200_flash_attn_kvq_workspace_size
    assert size(64, 65536, 1, (1 << 22) - 128, 1, 1) > 0      # 2^31 - 2^16 mask blocks of a token and 128 keys
    assert size(64, 65536, 1, 1 << 22, 1, 1) == 0              # 2^31
    assert size(64, 1, 1, 1 << 30, 1, 65535) > 0               # few rows: no such blocks
    assert size(64, 65537, 1, 64, 1, 1) == 0 and size(64, 1, 1, (1 << 30) + 1, 1, 1) == 0
    assert size(64, 1, 1, 64, 1, 65536) == 0 and size(128, 1, 65536 * 32, 64, 65536, 1) == 0


def test_more_refusals():
    """A misaligned position tensor, rows of a cache that lie in one another, sizes past 32 bits."""
    lib = g.lib()
    s = (ctypes.c_int32 * 4)(16, 24, 24, 0)
    assert lib.b200_rope_multi(0, P, ne(128, 4, 3), nb(4, 512, 2048, 6144), ctypes.c_void_p((1 << 20) + 2), 128, 8, s, 1e4,
                               1.0, 1.0, P, None) == NO

    def call(sne=(64, 5), snb=(4, 256, 1280, 1280), dne=(64, 9), dnb=(18, 36, 324, 324)):
        return lib.b200_set_rows(P, ne(*sne), nb(*snb), 27, P, ne(sne[1]), nb(8, 0, 0, 0), 2, P, ne(*dne), nb(*dnb), P, None)

    assert call(dnb=(18, 18, 324, 324)) == BAD and call(dnb=(18, 0, 324, 324)) == BAD
    assert call(sne=(64, 5, 2), dne=(64, 9, 2), dnb=(18, 36, 0, 0)) == BAD
    assert call(sne=(64, 1 << 62)) == NO and call(sne=(1 << 40, 1 << 30), dne=(1 << 40, 9), dnb=(18, 1 << 40, 1 << 50, 0)) == NO


def test_wrapper_types():
    """The wrappers name a type they do not take, before any CUDA call."""
    import pytest
    import torch
    with pytest.raises(g.B200Error, match="type 99"):
        g._dims_q(torch.zeros(2, 36, dtype=torch.uint8), 99, "set_rows")
    with pytest.raises(g.B200Error, match="whole blocks"):
        g._dims_q(torch.zeros(2, 35, dtype=torch.uint8), g.Q4_0, "set_rows")
