"""Argument checks of the operators on learned and compressed rows: they come before any call to the GPU."""
import ctypes as C

import pytest

import legion_ibp_b200 as L

A = 1 << 20   # an address that no check looks behind


def _calls(**change):
    """The four operators with good arguments, but for `change`."""
    d = dict(ids=A, id_bytes=4, n_ids=0, n_nodes=10, dim=8, dtype=L.F32, stride=8, table=A, table_dtype=L.F32, table_stride=8, weight=A,
             weight_dtype=L.F32, eps=1e-6, n_rows=0, codec=0, out=A, out_stride=8, ws=A, ws_bytes=1 << 20, m=0, n=0, k=8, row_stride=16, count=A)
    d.update(change)
    l = L.lib()
    return dict(
        lookup=lambda: l.legion_embedding_lookup(0, d["table"], d["table_dtype"], d["table_stride"], d["n_nodes"], d["ids"], d["id_bytes"], d["n_ids"],
                                                 d["dim"], 1.0, d["out"], d["dtype"], d["out_stride"], None),
        grad=lambda: l.legion_embedding_grad(0, d["ids"], d["id_bytes"], d["n_ids"], d["out"], d["dtype"], d["stride"], d["dim"], 1.0, d["table"],
                                             d["table_dtype"], d["table_stride"], d["n_nodes"], 0, d["ws"], d["ws_bytes"], None),
        rows=lambda: l.legion_embedding_grad_rows(0, d["ids"], d["id_bytes"], d["n_ids"], d["out"], d["dtype"], d["stride"], d["dim"], 1.0, d["n_nodes"],
                                                  d["ids"], d["table"], d["table_stride"], d["count"], d["ws"], d["ws_bytes"], None),
        norm=lambda: l.legion_rms_norm(0, d["table"], d["dtype"], d["stride"], None, 0, d["weight"], d["weight_dtype"], d["eps"], d["n_rows"], d["dim"],
                                       d["codec"], d["out"], d["out_stride"], None, 0, None),
        norm_grad=lambda: l.legion_rms_norm_grad(0, d["out"], d["stride"], d["table"], d["stride"], d["dtype"], None, 0, d["weight"], d["weight_dtype"],
                                                 d["eps"], d["n_rows"], d["dim"], d["out"], d["out_stride"], d["weight"], L.F32, d["ws"], d["ws_bytes"],
                                                 None),
        matmul=lambda: l.legion_matmul_rows(0, d["codec"] or 1, d["table"], d["m"], d["row_stride"], d["weight"], d["n"], d["row_stride"], d["k"],
                                            d["out"], d["dtype"], d["out_stride"], None))


BAD = [
    ("lookup grad rows", dict(id_bytes=2)), ("lookup grad rows", dict(n_ids=-1)), ("lookup grad rows", dict(n_ids=(1 << 28) + 1)),
    ("lookup grad rows", dict(n_nodes=0)), ("lookup grad rows", dict(n_nodes=1 << 31)), ("lookup grad rows norm norm_grad", dict(dim=0)),
    ("lookup grad rows", dict(dim=(1 << 16) + 1, stride=1 << 17, table_stride=1 << 17, out_stride=1 << 17)),
    ("lookup grad rows norm norm_grad matmul", dict(dtype=3)), ("lookup grad", dict(table_dtype=-1)), ("lookup grad rows", dict(table_stride=7)),
    ("lookup norm norm_grad", dict(out_stride=7)), ("grad rows norm norm_grad", dict(stride=7)), ("lookup grad rows", dict(ids=A + 2, n_ids=1)),
    ("lookup grad rows", dict(ids=None, n_ids=1)), ("lookup grad", dict(table=None)), ("lookup", dict(out=None, n_ids=1)),
    ("lookup norm norm_grad matmul", dict(out=A + 2)), ("lookup grad rows norm", dict(table=A + 1)), ("grad rows", dict(ws_bytes=100, n_ids=5)),
    ("grad rows", dict(ws=None, n_ids=5)), ("grad rows", dict(ws=A + 8, n_ids=5)), ("rows", dict(count=None)), ("rows", dict(count=A + 2)),
    ("norm norm_grad", dict(eps=-1.0)), ("norm norm_grad", dict(eps=float("nan"))), ("norm norm_grad", dict(weight_dtype=L.F16)),
    ("norm norm_grad", dict(n_rows=-1)), ("norm norm_grad", dict(n_rows=1 << 31)), ("norm norm_grad", dict(dim=16388, stride=16388, out_stride=16388)),
    ("norm norm_grad", dict(weight=A + 2)), ("norm norm_grad", dict(weight=None, n_rows=1)), ("norm", dict(codec=3)), ("norm", dict(codec=-1)),
    ("norm", dict(codec=1)), ("norm", dict(codec=1, out_stride=24)), ("norm", dict(codec=2, out_stride=16, out=A + 8)),
    ("norm", dict(codec=1, dim=6, out_stride=16)), ("norm_grad", dict(ws_bytes=31, n_rows=1)), ("norm_grad", dict(ws=None, n_rows=1)),
    ("matmul", dict(codec=3)), ("matmul", dict(k=0)), ("matmul", dict(k=6)), ("matmul", dict(row_stride=24)), ("matmul", dict(row_stride=0)),
    ("matmul", dict(k=16)), ("matmul", dict(m=-1)), ("matmul", dict(n=-1)), ("matmul", dict(table=A + 4)), ("matmul", dict(weight=A + 8)),
    ("lookup grad rows", dict(n_ids=1)), ("norm", dict(n_rows=1, codec=2, out_stride=16)), ("norm_grad", dict(n_rows=1)), ("matmul", dict(m=1, n=1)),   # outputs that are inputs
    ("lookup", dict(n_ids=1 << 28, dim=1 << 16, stride=1 << 16, table_stride=1 << 16, out_stride=1 << 16, out=2 * A)),
    ("matmul", dict(n=9, m=1)), ("matmul", dict(m=1, n=1, table=None)), ("matmul", dict(k=131072, row_stride=1 << 18)),
]


@pytest.mark.parametrize("names,change", BAD)
def test_bad_arguments_are_refused(names, change):
    for name in names.split():
        rc = _calls(**change)[name]()
        assert rc in (-1, -4), (name, rc)
        assert L.lib().legion_last_error()


@pytest.mark.parametrize("output", ["out", "residual_out", "grad_x"])
@pytest.mark.parametrize("input", [0, 1, 2])
def test_rows_in_place_keep_their_stride(output, input):
    """An output in an input's place but with other distances between its rows would be written over rows not read yet."""
    l, at, n = L.lib(), (A, 2 * A, 3 * A), 2
    if output == "grad_x":
        rc = l.legion_rms_norm_grad(0, at[0], 8, at[1], 8, L.F32, at[2], 8, 9 * A, L.F32, 1e-6, n, 8, at[input], 16, 5 * A, L.F32, 6 * A, 1 << 20, None)
    elif input == 2:
        return
    else:
        out, other = (at[input], 7 * A) if output == "out" else (7 * A, at[input])
        rc = l.legion_rms_norm(0, at[0], L.F32, 8, at[1], 8, 9 * A, L.F32, 1e-6, n, 8, 0, out, 16, other, 16, None)
    assert rc == -1 and b"stride" in l.legion_last_error()


def test_blocks_have_the_size_of_the_structs():
    """A block of another size, or of no operator, is refused; one of the right size reaches the operator's own checks."""
    call, error = L.lib().legion_operator_call, L.lib().legion_last_error
    for op, s in ((1, L._LOOKUP), (2, L._GRAD), (3, L._GRAD_ROWS), (4, L._NORM), (5, L._NORM_GRAD), (6, L._MATMUL)):
        empty = lambda size: op.to_bytes(4, "little") + size.to_bytes(4, "little") + bytes(s.size - 8)
        assert call(empty(s.size + 8)) == -1 and b"size" in error()
        assert call(empty(s.size)) == -1 and b"block" not in error()
    assert call((99).to_bytes(4, "little") + bytes(100)) == -1 and b"unknown" in error()
    assert call(None) == -1


def test_nothing_to_do_is_no_error_without_a_gpu():
    for name in ("lookup", "norm", "matmul"):
        assert _calls()[name]() == 0


def test_workspace_sizes():
    """Pairs twice, and from two stretches on two sums a stretch; the norm: one row of sums per CTA at most."""
    assert L.embedding_grad_workspace(0, 64, 10) >= 0
    one, many = L.embedding_grad_workspace(32, 64, 10), L.embedding_grad_workspace(33, 64, 10)
    assert many - one >= 2 * 2 * 64 * 4
    assert L.embedding_grad_workspace(100000, 64, 10) >= 100000 * 16
    assert L.rms_norm_grad_workspace(0, 64) == 0 and L.rms_norm_grad_workspace(3, 64) == 3 * 64 * 4
    assert L.rms_norm_grad_workspace(1 << 20, 64) == L.rms_norm_grad_workspace(1 << 21, 64)
    for bad in (lambda: L.embedding_grad_workspace(-1, 8, 10), lambda: L.embedding_grad_workspace(1, 0, 10), lambda: L.embedding_grad_workspace(1, 8, 0),
                lambda: L.rms_norm_grad_workspace(-1, 8), lambda: L.rms_norm_grad_workspace(1, 1 << 15)):
        with pytest.raises(L.LegionError):
            bad()
    b = C.c_int64()
    assert L.lib().legion_embedding_grad_workspace(1, 8, 10, None) == -1 and L.lib().legion_rms_norm_grad_workspace(1, 8, C.byref(b)) == 0


def test_limits_of_waits():
    try:
        for good in (0, 1, 60000000):
            L.operator_wait_limit(good)
        for bad in (-1, 60000001):
            with pytest.raises(L.LegionError):
                L.operator_wait_limit(bad)
    finally:
        L.operator_wait_limit(2000000)
