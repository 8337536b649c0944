"""RMS norm, its compressed output and its gradient against 64-bit formulas.

Tolerances: an fp32 operation is off by at most u = 2^-24.  A thread adds at most 32 squares one after the other, lanes and
warps add in ten more steps: the mean square is off by at most 43 u, its root's inverse by 22 u and three more for
the root, the quotient and eps; h, h * w and * s add one each: 28 u, taken as 32 u.  The last rounding is half a step of the output's
type.  Codes: half a step of the code (int8: half a scale; e4m3: 2^-4, or half of its smallest number) on top."""
import numpy as np
import pytest

import legion_ibp_b200 as L
from test_gpu_embedding import U32, _close, _strided, _types

pytestmark = pytest.mark.gpu
SHAPES = [(1, 1), (3, 4), (5, 7), (257, 32), (130, 75), (1000, 128), (17, 256), (19, 260), (301, 602), (64, 1000), (9, 1024), (700, 2048), (3, 4096),
          (310, 4100), (2, 8191), (5, 8192), (400, 8200), (2, 16383), (3, 16384), (300, 16384)]


def _inputs(n, dim, t, wt, residual, pad=0, shift=0, seed=0):
    import torch
    torch.manual_seed(n * 31 + dim + seed)
    x = _strided(n, dim, t, pad, shift)[1]
    x.copy_(torch.randn(n, dim, device="cuda") * torch.exp(torch.randn(n, 1, device="cuda")))
    r = None
    if residual:
        r = _strided(n, dim, t, pad, shift)[1]
        r.copy_(3 * torch.randn(n, dim, device="cuda"))
    return x, (1 + 0.2 * torch.randn(dim, device="cuda")).to(wt), r


def _exact(x, w, r, eps):
    import torch
    h = x.double() + (r.double() if r is not None else 0.0)
    return h, h * w.double() / torch.sqrt((h * h).mean(1, keepdim=True) + eps)


@pytest.mark.parametrize("n,dim", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(n, dim, dtype, residual):
    import torch
    t = _types()[dtype]
    for pad, shift, wt in ((0, 0, torch.float32), (8, 8, t), (3, 1, t)):
        x, w, r = _inputs(n, dim, t, wt, residual, pad, shift)
        whole, out = _strided(n, dim, t, pad, shift)
        total = _strided(n, dim, t, pad, shift)[1] if residual else None
        L.rms_norm(0, x, w, out, 1e-5, r, total)
        h, y = _exact(x, w, r, 1e-5)
        _close(out, y, y.abs() * (32 * U32))
        if residual:
            _close(total, h, h.abs() * U32)
        rest = whole.clone()
        torch.as_strided(rest, (n, dim), (dim + pad, 1), shift).fill_(7.0)
        assert bool((rest == 7.0).all())
    # in place: the sum over the residual, the result over the rows
    a, b = _strided(n, dim, t, pad, shift)[1], None if r is None else _strided(n, dim, t, pad, shift)[1]
    a.copy_(x)
    if residual:
        b.copy_(r)
    L.rms_norm(0, a, w, a, 1e-5, b, b)
    assert torch.equal(a, out) and (b is None or torch.equal(b, total))


@pytest.mark.parametrize("codec", [L.CODEC_INT8, L.CODEC_E4M3])
@pytest.mark.parametrize("n,dim", [(n, d) for n, d in SHAPES if d % 4 == 0] + [(33, 12), (50, 36), (5, 772)])
def test_codes_are_those_of_the_quantiser(oracle_mod, codec, n, dim):
    """fp32 rows: the bytes that quantize_table makes of the uncompressed output, padding included."""
    import torch
    for residual in (False, True):
        x, w, r = _inputs(n, dim, torch.float32, torch.float32, residual)
        if n > 4:
            x[1], x[2, 0], x[3] = 0.0, float("nan"), torch.randn(dim, device="cuda") * 1e-30
            x[4, dim // 2] = float("inf")
        plain = torch.empty(n, dim, device="cuda")
        L.rms_norm(0, x, w, plain, 1e-6, r)
        slot = oracle_mod.quant_row_bytes(dim)
        want = torch.zeros(n, slot, dtype=torch.uint8, device="cuda")
        L.quantize_table(0, codec, plain, n, dim, want)
        got = torch.full((n, slot + 16), 9, dtype=torch.uint8, device="cuda")
        L.rms_norm(0, x, w, got, 1e-6, r, None, codec)
        assert torch.equal(got[:, :slot], want) and bool((got[:, slot:] == 9).all())


@pytest.mark.parametrize("codec", [L.CODEC_INT8, L.CODEC_E4M3])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("n,dim", [(1, 4), (3, 12), (70, 132), (301, 768), (40, 2052), (5, 8192), (300, 16384)])
def test_codes_of_short_types(codec, dtype, n, dim):
    import torch
    t = _types()[dtype]
    for pad in (0, 4, 1):
        x, w, r = _inputs(n, dim, t, t, True, pad, pad)
        total = torch.empty(n, dim, dtype=t, device="cuda")
        slot = (dim + 19) // 16 * 16
        out = torch.full((n, slot), 9, dtype=torch.uint8, device="cuda")
        L.rms_norm(0, x, w, out, 1e-6, r, total, codec)
        h, y = _exact(x, w, r, 1e-6)
        _close(total, h, h.abs() * U32)
        top = 127.0 if codec == L.CODEC_INT8 else 448.0
        scale = out.view(torch.float32)[:, dim // 4].double()
        want = y.abs().amax(1) / top
        assert bool(((scale - want).abs() <= want * (34 * U32)).all())
        codes = out[:, :dim].contiguous().view(torch.int8 if codec == L.CODEC_INT8 else torch.float8_e4m3fn).double()
        step = 0.5 * scale[:, None] if codec == L.CODEC_INT8 else torch.maximum(y.abs() * 2 ** -4, scale[:, None] * 2 ** -10)
        assert bool(((codes * scale[:, None] - y).abs() <= step * (1 + 2 ** -10) + y.abs() * (40 * U32)).all())
        assert bool((out[:, dim + 4:] == 0).all())


@pytest.mark.parametrize("n,dim", SHAPES + [(5000, 40), (3000, 300)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("residual", [False, True])
def test_gradient(n, dim, dtype, residual):
    """dx: s is off by 25 u, s^3 by 75 u, the dot product by 43 u of the sum of its terms' magnitudes and 3 u a term; at most
    130 u of the magnitudes of the three terms in all.  dw: n terms of at most 30 u each, added in some order."""
    import torch
    t = _types()[dtype]
    for pad, shift, wt in ((0, 0, torch.float32), (3, 1, t)):
        x, w, r = _inputs(n, dim, t, wt, residual, pad, shift)
        dy = _strided(n, dim, t, pad, shift)[1]
        dy.copy_(torch.randn(n, dim, device="cuda"))
        dx, dw = _strided(n, dim, t, pad, shift)[1], torch.zeros(dim, dtype=wt, device="cuda")
        ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda").fill_(0xFF)
        L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
        h, g = x.double(), dy.double() * w.double()
        s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
        first, second = s * g, h * s ** 3 * (g * h).mean(1, keepdim=True)
        extra = r.double() if residual else torch.zeros_like(h)
        mag = first.abs() + h.abs() * s ** 3 * (g * h).abs().mean(1, keepdim=True) + extra.abs()
        _close(dx, first - second + extra, mag * (130 * U32))
        terms = dy.double() * h * s
        _close(dw, terms.sum(0), terms.abs().sum(0) * ((n + 32) * U32))
        again, dw2 = _strided(n, dim, t, pad, shift)[1], torch.zeros_like(dw)
        L.rms_norm_grad(0, dy, x, w, again, dw2, ws, 1e-5, r)
        assert torch.equal(dw, dw2) and torch.equal(dx, again)
    # in place over the gradient that came in
    L.rms_norm_grad(0, dy, x, w, dy, dw2, ws, 1e-5, r)
    assert torch.equal(dy, again)


def test_gradient_against_differences():
    """Central differences in 64 bits of the formula that test_norm holds the kernel to."""
    import torch
    torch.manual_seed(0)
    n, dim, eps = 5, 36, 1e-3
    x, w, dy = (torch.randn(s, device="cuda") for s in ((n, dim), (dim,), (n, dim)))
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    L.rms_norm_grad(0, dy, x, w, dx, dw, torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda"), eps)

    def value(a, b):
        return (_exact(a, b, None, eps)[1] * dy.double()).sum()

    step = 1e-5
    for grad, at in ((dx, 0), (dw, 1)):
        base = [x.double(), w.double()]
        for k in range(grad.numel()):
            moved = [b.clone() for b in base], [b.clone() for b in base]
            moved[0][at].view(-1)[k] += step
            moved[1][at].view(-1)[k] -= step
            d = float((value(*moved[0]) - value(*moved[1])) / (2 * step))
            # third derivatives times step^2 / 6, and 64-bit cancellation over 2 * step: both below 1e-6 at these sizes
            assert abs(d - float(grad.view(-1)[k])) <= 1e-6 + 200 * U32 * (abs(d) + 10)


def test_rows_of_zeros_infinities_and_large_values():
    import torch
    x = torch.randn(6, 64, device="cuda")
    x[0], x[1, 3], x[2, 4], x[3] = 0.0, float("inf"), float("nan"), 1e18
    w, out = torch.ones(64, device="cuda"), torch.empty(6, 64, device="cuda")
    L.rms_norm(0, x, w, out, 1e-6)
    want = x / torch.sqrt((x.double() ** 2).mean(1, keepdim=True) + 1e-6)
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert bool((out[0] == 0).all()) and bool((out[1].nan_to_num(0.0) == 0).all())
    keep = [0, 3, 4, 5]
    _close(out[keep], want[keep], want[keep].abs() * (32 * U32))


@pytest.mark.parametrize("n,dim", [(300, 512), (1300, 2048)])
def test_captured_on_another_stream(n, dim):
    import torch
    x, w, r = _inputs(n, dim, torch.bfloat16, torch.float32, True)
    out, total = torch.empty_like(x), torch.empty_like(x)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    L.rms_norm(0, x, w, out, 1e-6, r, total)
    L.rms_norm_grad(0, out, total, w, dx, dw, ws, 1e-6, r)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s = torch.cuda.current_stream()
        L.rms_norm(0, x, w, out, 1e-6, r, total, stream=s)
        L.rms_norm_grad(0, out, total, w, dx, dw, ws, 1e-6, r, stream=s)
    for _ in range(2):
        x.copy_(torch.randn(n, dim, device="cuda"))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        want = [torch.empty_like(t) for t in (out, total, dx, dw)]
        L.rms_norm(0, x, w, want[0], 1e-6, r, want[1])
        L.rms_norm_grad(0, want[0], want[1], w, want[2], want[3], torch.empty_like(ws), 1e-6, r)
        assert all(torch.equal(a, b) for a, b in zip((out, total, dx, dw), want))


def test_no_rows_and_refusals():
    import torch
    x, w = torch.zeros(4, 8, device="cuda"), torch.ones(8, device="cuda")
    L.rms_norm(0, x[:0], w, x[:0])
    dw = torch.ones(8, device="cuda")
    L.rms_norm_grad(0, x[:0], x[:0], w, x[:0], dw, None)
    assert bool((dw == 0).all())
    big = torch.zeros(2, 16388, device="cuda")
    for bad in (lambda: L.rms_norm(0, x, w, x.half()), lambda: L.rms_norm(0, x, w[:7], x), lambda: L.rms_norm(0, x, w, x, -1.0),
                lambda: L.rms_norm(0, x, w.half(), x), lambda: L.rms_norm(0, x, w, x, 1e-6, x.half()),
                lambda: L.rms_norm(0, big, torch.ones(16388, device="cuda"), big), lambda: L.rms_norm(0, x.cpu(), w, x),
                lambda: L.rms_norm(0, x, w, x, codec=L.CODEC_INT8),
                lambda: L.rms_norm(0, x, w, torch.zeros(4, 8, dtype=torch.uint8, device="cuda"), codec=L.CODEC_INT8),
                lambda: L.rms_norm(0, x[:, :6], w[:6], torch.zeros(4, 16, dtype=torch.uint8, device="cuda"), codec=L.CODEC_INT8),
                lambda: L.rms_norm(0, x, w, torch.zeros(4, 24, dtype=torch.uint8, device="cuda"), codec=L.CODEC_E4M3),
                lambda: L.rms_norm(0, x, w, x, codec=3),
                lambda: L.rms_norm_grad(0, x, x, w, x, dw, None), lambda: L.rms_norm_grad(0, x, x, w, x, dw, x[:1]),
                lambda: L.rms_norm_grad(0, x, x, w, x, dw.half(), torch.zeros(1 << 12, device="cuda"))):
        with pytest.raises(L.LegionError):
            bad()


@pytest.mark.parametrize("n,dim,dtype", [(592, 1024, "bf16"), (593, 4096, "bf16"), (1000, 8192, "f16"), (700, 2052, "f32"), (2000, 512, "f32"), (595, 6000, "f32"),
                                         (600, 16384, "bf16"), (3000, 1032, "f16")])
@pytest.mark.parametrize("residual", [False, True])
def test_gradient_of_many_long_rows(n, dim, dtype, residual):
    """Rows that the copy engine brings: around the smallest number of them, rows per CTA that differ, one stage more and less."""
    import torch
    t = _types()[dtype]
    x, w, r = _inputs(n, dim, t, torch.float32, residual, 16 // t.itemsize, 0, 5)
    dy = torch.randn(n, dim, device="cuda").to(t)
    dx, dw = torch.empty_like(dy), torch.zeros(dim, device="cuda")
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda").fill_(0xFF)
    L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
    h, g = x.double(), dy.double() * w.double()
    s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    first, second = s * g, h * s ** 3 * (g * h).mean(1, keepdim=True)
    extra = r.double() if residual else torch.zeros_like(h)
    mag = first.abs() + h.abs() * s ** 3 * (g * h).abs().mean(1, keepdim=True) + extra.abs()
    _close(dx, first - second + extra, mag * (130 * U32))
    terms = dy.double() * h * s
    _close(dw, terms.sum(0), terms.abs().sum(0) * ((n + 32) * U32))
    assert L.operator_error(0) == 0
    dw2 = torch.zeros_like(dw)
    L.rms_norm_grad(0, dy, x, w, dy, dw2, ws, 1e-5, r)   # in place
    assert torch.equal(dy, dx) and torch.equal(dw, dw2)


@pytest.mark.parametrize("n,dim", [(1, 65), (7, 101), (2000, 129), (1300, 255), (600, 602), (50, 1022), (900, 1030), (300, 2047), (296, 1025), (297, 12289), (500, 1027), (700, 4097), (20, 8191), (3, 16383),
                                   (400, 16382)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (0, 3), (5, 1), (8, 2)])
def test_rows_that_start_anywhere(n, dim, dtype, pad, shift):
    """Rows that begin at every place of a 16-byte vector, all operands alike; forward, backward, in place; nothing beside the rows is touched."""
    import torch
    t = _types()[dtype]
    x, w, r = _inputs(n, dim, t, t, True, pad, shift, 2)
    whole, out = _strided(n, dim, t, pad, shift)
    wholes, total = _strided(n, dim, t, pad, shift)
    L.rms_norm(0, x, w, out, 1e-5, r, total)
    h, y = _exact(x, w, r, 1e-5)
    _close(out, y, y.abs() * (32 * U32))
    _close(total, h, h.abs() * U32)
    for mem in (whole, wholes):
        rest = mem.clone()
        torch.as_strided(rest, (n, dim), (dim + pad, 1), shift).fill_(7.0)
        assert bool((rest == 7.0).all())
    a = _strided(n, dim, t, pad, shift)[1]
    a.copy_(x)
    L.rms_norm(0, a, w, a, 1e-5, r)
    assert torch.equal(a, out)
    dy, (mem, dx), dw = _strided(n, dim, t, pad, shift)[1], _strided(n, dim, t, pad, shift), torch.zeros(dim, device="cuda")
    dy.copy_(torch.randn(n, dim, device="cuda"))
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda").fill_(0xFF)
    L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
    h, g = x.double(), dy.double() * w.double()
    s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
    first, second = s * g, h * s ** 3 * (g * h).mean(1, keepdim=True)
    mag = first.abs() + h.abs() * s ** 3 * (g * h).abs().mean(1, keepdim=True) + r.double().abs()
    _close(dx, first - second + r.double(), mag * (130 * U32))
    terms = dy.double() * h * s
    _close(dw, terms.sum(0), terms.abs().sum(0) * ((n + 32) * U32))
    rest = mem.clone()
    torch.as_strided(rest, (n, dim), (dim + pad, 1), shift).fill_(7.0)
    assert bool((rest == 7.0).all())
    dw2 = torch.zeros_like(dw)
    L.rms_norm_grad(0, dy, x, w, dy, dw2, ws, 1e-5, r)
    assert torch.equal(dy, dx) and torch.equal(dw, dw2)


@pytest.mark.parametrize("n,dim,dtype", [(593, 2048, "bf16"), (1185, 2048, "f16"), (1777, 2056, "bf16"), (4001, 1032, "f32"), (741, 4096, "bf16"), (887, 2044, "f32"),
                                         (1333, 12000, "bf16"), (2000, 8200, "f16"), (607, 16384, "f16"), (893, 5000, "f32"), (592, 8192, "f32")])
@pytest.mark.parametrize("arrays", [2, 3])
def test_gradient_of_rows_that_meet_in_pairs(n, dim, dtype, arrays):
    """Two rows a reduction where the second one may be missing, and wide rows that are read again; the bound is test_gradient's: the root's
    inverse has one rounding of a product and one of the result, no more than the root and the quotient that it takes the place of."""
    import torch
    t = _types()[dtype]
    x, w, r = _inputs(n, dim, t, torch.float32, arrays == 3, 0, 0, 7)
    dy = torch.randn(n, dim, device="cuda").to(t)
    dx, dw = torch.empty_like(dy), torch.zeros(dim, device="cuda")
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda").fill_(0xFF)
    for turn in range(2):
        L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
        h, g = x.double(), dy.double() * w.double()
        s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5)
        first, second = s * g, h * s ** 3 * (g * h).mean(1, keepdim=True)
        extra = r.double() if arrays == 3 else torch.zeros_like(h)
        mag = first.abs() + h.abs() * s ** 3 * (g * h).abs().mean(1, keepdim=True) + extra.abs()
        _close(dx, first - second + extra, mag * (130 * U32))
        terms = dy.double() * h * s
        _close(dw, terms.sum(0), terms.abs().sum(0) * ((n + 32) * U32))
        x.mul_(-0.5)
    assert L.operator_error(0) == 0


@pytest.mark.parametrize("n,dim", [(7, 100), (600, 2048), (600, 12000)])
def test_gradient_of_rows_without_a_norm(n, dim):
    """A row of zeros with eps: its gradient is dy w / sqrt(eps).  Squares that sum to infinity: the norm's inverse is 0, and so is the gradient by it."""
    import torch
    x = torch.zeros(n, dim, device="cuda")
    x[1::2] = 3e19
    w, dy = torch.ones(dim, device="cuda"), torch.full((n, dim), 0.5, device="cuda")
    dx, dw = torch.empty_like(x), torch.zeros(dim, device="cuda")
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda")
    L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 2.0 ** -10)
    assert bool(((dx[0::2] - 16.0).abs() <= 16.0 * 4 * U32).all())
    assert bool((dx[1::2] == 0).all()) and bool((dw == 0).all())


@pytest.mark.parametrize("n,dim,dtype", [(50, 24, "f32"), (9, 64, "bf16"), (700, 300, "f32"), (20, 4096, "f32"), (30, 1000, "bf16"), (600, 2048, "bf16"), (700, 2052, "f32"),
                                         (300, 4096, "f32"), (400, 12000, "bf16"), (200, 8192, "f32"), (400, 4097, "f32"), (500, 1027, "bf16")])
@pytest.mark.parametrize("size,eps", [(1e15, 1e-6), (1e17, 1e-6), (1e-14, 0.0), (1e-17, 0.0)])
def test_gradient_of_large_and_small_rows(n, dim, dtype, size, eps):
    """Rows whose squares' sum is an fp32 number, while the third power of the norm's inverse is not.  dx = s (dy w - (x s) (s mean(dy w x))), up
    to the order of the factors: s is off by 25 u, so s twice and x s by 76 u, the mean by 46 u, the products by 5 u: 127 u, within
    test_gradient's 130 u of the terms' magnitudes."""
    import torch
    t = _types()[dtype]
    torch.manual_seed(dim)
    x = (torch.randn(n, dim, device="cuda", dtype=torch.float64) * size).to(t)
    w = 1 + 0.2 * torch.randn(dim, device="cuda")
    dy = (torch.randn(n, dim, device="cuda") + 2 * x.double().sign()).to(t)   # rows that the second term does not leave alone
    dx, dw = torch.empty_like(x), torch.zeros(dim, device="cuda")
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda")
    L.rms_norm_grad(0, dy, x, w, dx, dw, ws, eps)
    h, g = x.double(), dy.double() * w.double()
    assert float((h * h).sum(1).max()) < 3.4e38
    s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    first, second = s * g, (h * s) * (s * (g * h * s).mean(1, keepdim=True))
    mag = first.abs() + (h * s).abs() * s * (g * h * s).abs().mean(1, keepdim=True)
    _close(dx, first - second, mag * (130 * U32))
    terms = dy.double() * h * s
    _close(dw, terms.sum(0), terms.abs().sum(0) * ((n + 32) * U32))


@pytest.fixture
def wait_limit():
    yield L.operator_wait_limit
    L.operator_wait_limit(2000000)


@pytest.mark.parametrize("n,dim,dtype", [(8000, 2048, "bf16"), (3000, 4096, "f32"), (3000, 12000, "bf16")])
@pytest.mark.parametrize("residual", [False, True])
def test_a_wait_that_is_given_up(wait_limit, n, dim, dtype, residual):
    """Limit 0: the rows behind the first stages are never brought, their waits run out, and the call ends with its error; limits about as long as a
    copy takes: the waits of some threads of a CTA may run out and those of others not, and the call ends with an error or is right."""
    import torch
    t = _types()[dtype]
    x, w, r = _inputs(n, dim, t, torch.float32, residual, 0, 0, 3)
    dy = torch.randn(n, dim, device="cuda").to(t)
    ws = torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda")
    want, want_w = torch.empty_like(dy), torch.zeros(dim, device="cuda")
    L.rms_norm_grad(0, dy, x, w, want, want_w, ws, 1e-5, r)
    assert L.operator_error(0) == 0
    for limit in (0, 1, 20, 40, 200):
        wait_limit(limit)
        dx, dw = torch.empty_like(dy), torch.zeros(dim, device="cuda")
        L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
        error = L.operator_error(0, reset=False)
        assert error == (-7 if limit == 0 else error) and error in (0, -7)
        assert L.operator_error(0) == error and L.operator_error(0) == 0   # kept until it is reset
        if error == 0:
            assert torch.equal(dx, want) and torch.equal(dw, want_w)
    wait_limit(2000000)
    dx, dw = torch.empty_like(dy), torch.zeros(dim, device="cuda")
    L.rms_norm_grad(0, dy, x, w, dx, dw, ws, 1e-5, r)
    assert L.operator_error(0) == 0 and torch.equal(dx, want) and torch.equal(dw, want_w)
