"""Cache layouts of SET_ROWS: rows that share bytes are refused whichever dims share them, others are not, checked
before any CUDA call."""
import ctypes

import pytest

import ggml_b200 as g

P = ctypes.c_void_p(1 << 20)


def call(dne, dnb):
    """SET_ROWS of Q4_0 rows of 64 values; a call that is not refused fails at its launch, here without a GPU."""
    ne = (ctypes.c_int64 * 4)
    nb = (ctypes.c_size_t * 4)
    n2, n3 = dne[2], dne[3]
    return g.lib().b200_set_rows(P, ne(64, 5, n2, n3), nb(4, 256, 1280, 1280 * n2), 27, P, ne(5, 1, 1, 1), nb(8, 40, 40, 40),
                                 2, P, ne(*dne), nb(*dnb), P, None)


@pytest.mark.parametrize("dne,dnb", [
    ((64, 9, 2, 1), (18, 36, 36, 72)),                # a slice begins at the other's second row
    ((64, 9, 2, 1), (18, 36, 288, 576)),              # at its last
    ((64, 9, 2, 1), (18, 70, 36, 72)),                # rows of two slices in turn, two bytes short
    ((64, 9, 2, 3), (18, 72, 36, 72)),                # the streams at each other's rows
    ((64, 9, 1, 2), (18, 36, 0, 0)),
    ((64, 9, 1, 2), (18, 36, 324, 323)),
])
def test_rows_that_share_bytes_are_refused(dne, dnb):
    assert call(dne, dnb) == g.B200_E_INVALID


@pytest.mark.parametrize("dne,dnb", [
    ((64, 9, 2, 1), (18, 36, 324, 648)),              # slice behind slice
    ((64, 9, 2, 1), (18, 72, 36, 648)),               # the slices' rows in turn
    ((64, 9, 2, 3), (18, 216, 36, 72)),               # those of the streams too
    ((64, 9, 1, 1), (18, 36, 0, 0)),                  # strides of dims of one mean nothing
    ((64, 1, 2, 1), (18, 0, 36, 72)),
])
def test_rows_apart_are_taken(dne, dnb):
    import torch
    if torch.cuda.is_available():
        pytest.skip("the call would launch, on made-up addresses")
    assert call(dne, dnb) == -3                          # B200_E_CUDA


def test_many_rows_need_a_workspace():
    """Without one the time grows by the square of the rows."""
    ne, nb = (ctypes.c_int64 * 4), (ctypes.c_size_t * 4)

    def many(rows, ws=None, wsb=0):
        return g.lib().b200_set_rows_ws(P, ne(64, rows, 1, 1), nb(4, 256, 256 * rows, 256 * rows), 27, P, ne(rows, 1, 1, 1),
                                        nb(8, 0, 0, 0), 2, P, ne(64, 1 << 20, 1, 1), nb(18, 36, 0, 0), ws, wsb, P, None)

    size = g.lib().b200_set_rows_workspace_size
    assert size(ne(2047, 1, 1, 1), ne(64, 9, 1, 1)) == 0 and size(ne(2048, 3, 2, 1), ne(64, 9, 6, 2)) == 9 * 6 * 4
    assert many(131073) == g.B200_E_WORKSPACE
    assert many(131073, P, (1 << 22) - 1) == g.B200_E_WORKSPACE and many(5000, ctypes.c_void_p((1 << 20) + 2), 1 << 22) == g.B200_E_WORKSPACE
    assert g.lib().b200_set_rows(P, ne(64, 1 << 20, 1, 1), nb(4, 256, 1 << 28, 1 << 28), 27, P, ne(1 << 20, 1, 1, 1),
                                 nb(8, 0, 0, 0), 2, P, ne(64, 1 << 20, 1, 1), nb(18, 36, 0, 0), P, None) == g.B200_E_WORKSPACE


def test_wrappers_name_shapes_they_do_not_take():
    """As B200Error, before any CUDA call."""
    import torch
    with pytest.raises(g.B200Error, match="5 dims"):
        g._dims(torch.zeros(1, 1, 1, 1, 1))
    with pytest.raises(g.B200Error, match="four sections"):
        g._sections([16, 24, 24])
    assert g._sections([16, 24, 24, 0]) == b"".join(v.to_bytes(4, "little") for v in (16, 24, 24, 0))
