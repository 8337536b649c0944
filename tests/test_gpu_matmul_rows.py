"""Products of compressed rows against 64-bit sums over the codes.

Tolerances: int8 sums are exact; the sum becomes fp32 and meets two scales, three roundings of 2^-24, then one of the output's
type.  e4m3: products of two codes are exact in fp32, K of them are added with at most one step (2^-23) lost per
addition, relative to the sum of their magnitudes."""
import numpy as np
import pytest

import legion_ibp_b200 as L
from test_gpu_embedding import U32, _close, _strided, _types

pytestmark = pytest.mark.gpu
CODECS = [L.CODEC_INT8, L.CODEC_E4M3]


def _coded(n, k, codec, pad=0, seed=0, std=1.0):
    """Compressed rows (random codes of a normal distribution, one scale a row), bytes behind the scale filled with 0xFF."""
    import torch
    torch.manual_seed(seed + 7 * n + k)
    slot = (k + 19) // 16 * 16 + pad
    rows = torch.full((n, slot), 0xFF, dtype=torch.uint8, device="cuda")
    x = torch.randn(n, k, device="cuda") * std
    codes = (x * 40).round().clamp(-128, 127).to(torch.int8) if codec == L.CODEC_INT8 else (x * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
    rows[:, :k] = codes.view(torch.uint8)
    scale = torch.exp(torch.randn(n, device="cuda"))
    rows.view(torch.float32)[:, k // 4] = scale
    return rows, codes.double(), scale.double()


def _check(got, a, b, k, codec):
    (_, ca, sa), (_, cb, sb) = a, b
    outer = sa[:, None] * sb[None]
    want = (ca @ cb.t()) * outer
    slack = want.abs() * (3 * U32)
    if codec == L.CODEC_E4M3:
        slack = slack + (ca.abs() @ cb.abs().t()) * outer * (k * 2 * U32)
    _close(got, want, slack)


SHAPES = [(1, 1, 4), (1, 5, 16), (2, 33, 20), (3, 130, 36), (4, 64, 128), (5, 1000, 132), (7, 16, 2048), (1, 700, 4100), (2, 601, 508), (3, 5000, 1036), (6, 9500, 8), (8, 1203, 4108), (4, 4097, 520), (5, 40, 12), (8, 17, 1028), (9, 300, 64), (16, 128, 256),
          (17, 129, 260), (33, 500, 768), (64, 64, 516), (65, 257, 100), (127, 128, 128), (128, 1000, 384), (129, 100, 132), (200, 513, 1024),
          (300, 256, 640), (611, 1000, 768), (1030, 70, 40), (257, 2600, 4096), (5000, 260, 128), (2049, 9001, 260), (4096, 8192, 128), (3000, 9100, 1100)]


@pytest.mark.parametrize("codec", CODECS)
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
def test_product(codec, m, n, k, out_type):
    import torch
    t = _types()[out_type]
    for pad, out_pad, shift in ((0, 0, 0), (32, 3, 1)):
        a, b = _coded(m, k, codec, pad, 1), _coded(n, k, codec, pad, 2, 0.3 if out_type == "f16" else 1.0)
        if out_type == "f16":   # inside the range of the type
            a = (a[0], a[1], a[2] / 4096)
            a[0].view(torch.float32)[:, k // 4] = a[2].float()
        whole, out = _strided(m, n, t, out_pad, shift)
        L.matmul_rows(0, codec, a[0], b[0], k, out)
        _check(out, a, b, k, codec)
        rest = whole.clone()
        torch.as_strided(rest, (m, n), (n + out_pad, 1), shift).fill_(7.0)
        assert bool((rest == 7.0).all())
        assert L.operator_error(0) == 0


@pytest.mark.parametrize("m", [1, 9, 40, 300])
def test_int8_sums_are_exact_at_their_limits(m):
    """The longest rows, all codes -128 on both sides: the sum is 128 * 128 * K, close below 2^31."""
    import torch
    k = 131068
    rows = torch.zeros(m, k + 4, dtype=torch.uint8, device="cuda")
    rows[:, :k] = 128
    rows.view(torch.float32)[:, k // 4] = 1.0
    out = torch.zeros(m, m, device="cuda")
    L.matmul_rows(0, L.CODEC_INT8, rows, rows, k, out)
    assert bool((out == float(np.float32(128 * 128 * k))).all())


@pytest.mark.parametrize("codec", CODECS)
@pytest.mark.parametrize("m", [3, 20, 200])
def test_scales_of_zero_infinity_and_nan_stay_in_their_row(codec, m):
    import torch
    a, b = _coded(m, 64, codec, 0, 3), _coded(40, 64, codec, 0, 4)
    a[0].view(torch.float32)[1, 16] = 0.0
    b[0].view(torch.float32)[2, 16] = float("nan")
    out = torch.empty(m, 40, device="cuda")
    L.matmul_rows(0, codec, a[0], b[0], 64, out)
    bad = torch.isnan(out)
    assert bool(bad[:, 2].all()) and int(bad.sum()) == m
    assert bool((out[1].nan_to_num(0.0) == 0).all())


def test_rows_of_a_cache_partition(oracle_mod):
    """A compressed cache's partition is projected as it lies in memory: what decoding and multiplying gives."""
    import torch
    rng = np.random.default_rng(5)
    n, f, h = 900, 100, 48
    table = rng.standard_normal((n, f)).astype(np.float32)
    for codec in CODECS:
        cache = L.UnifiedCache(0, n, f * 4, n, codec=codec)
        order = torch.from_numpy(rng.permutation(n).astype(np.int32)).cuda()
        cache.fill_static(order, torch.from_numpy(table).pin_memory())
        torch.cuda.synchronize()
        weight = torch.randn(h, f, device="cuda")
        coded = torch.empty(h, oracle_mod.quant_row_bytes(f), dtype=torch.uint8, device="cuda")
        L.quantize_table(0, codec, weight, h, f, coded)
        stored = oracle_mod.quant_rows(table[order.cpu().numpy()], codec)
        ptr, nbytes = cache.partition()
        assert nbytes == stored.size
        rows = torch.empty(n, stored.shape[1], dtype=torch.uint8, device="cuda")
        L._check(L.lib().legion_copy(L._ptr(rows), L.C.c_void_p(ptr), L.C.c_int64(nbytes), L.C.c_int32(3)))
        out = torch.empty(n, h, device="cuda")
        L.matmul_rows(0, codec, rows, coded, f, out)
        a = oracle_mod.dequant_rows(stored, f, codec).astype(np.float64)
        b = oracle_mod.dequant_rows(coded.cpu().numpy(), f, codec).astype(np.float64)
        # decoding rounds each value once more (2^-24 of it)
        slack = (np.abs(a) @ np.abs(b).T) * ((2 * f + 8) * U32)
        assert (np.abs(out.cpu().numpy().astype(np.float64) - a @ b.T) <= slack + np.abs(a @ b.T) * U32).all()
        cache.close()


@pytest.mark.parametrize("codec", CODECS)
def test_lookup_norm_product_and_back(codec):
    """A run as it is used: learned rows, norm to compressed rows, product; the way back through norm and lookup."""
    import torch
    torch.manual_seed(2)
    n, nodes, dim, width = 777, 400, 256, 130
    table, w, weight = torch.randn(nodes, dim, device="cuda"), 1 + 0.1 * torch.randn(dim, device="cuda"), torch.randn(width, dim, device="cuda")
    ids = torch.randint(0, nodes, (n,), device="cuda", dtype=torch.int32)
    slot = (dim + 19) // 16 * 16
    coded_w = torch.empty(width, slot, dtype=torch.uint8, device="cuda")
    L.quantize_table(0, codec, weight, width, dim, coded_w)
    x, coded, out = torch.empty(n, dim, device="cuda"), torch.empty(n, slot, dtype=torch.uint8, device="cuda"), torch.empty(n, width, device="cuda")
    L.embedding_lookup(0, table, ids, x, 2.0)
    L.rms_norm(0, x, w, coded, 1e-6, codec=codec)
    L.matmul_rows(0, codec, coded, coded_w, dim, out)
    h = table.double()[ids.long()] * 2
    y = h * w.double() / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
    want = y @ weight.double().t()
    # both sides are off by half a step of their codes: int8 half of max / 127 each; e4m3 2^-4 of the value, or 2^-10 of max / 448
    if codec == L.CODEC_INT8:
        ey, ew = y.abs().amax(1, keepdim=True) / 254, weight.double().abs().amax(1, keepdim=True) / 254
        slack = ey * weight.double().abs().sum(1)[None] + y.abs().sum(1, keepdim=True) * ew.t() + dim * ey * ew.t()
    else:
        ey = y.abs() * 2 ** -4 + y.abs().amax(1, keepdim=True) / 448 * 2 ** -10
        ew = weight.double().abs() * 2 ** -4 + weight.double().abs().amax(1, keepdim=True) / 448 * 2 ** -10
        slack = ey @ weight.double().abs().t() + y.abs() @ ew.t() + ey @ ew.t()
    assert bool(((out.double() - want).abs() <= slack * 1.001 + 1e-4).all())
    dy, dx, dw, grad = torch.randn(n, dim, device="cuda"), torch.empty(n, dim, device="cuda"), torch.empty(dim, device="cuda"), torch.empty(nodes, dim, device="cuda")
    L.rms_norm_grad(0, dy, x, w, dx, dw, torch.empty(L.rms_norm_grad_workspace(n, dim), dtype=torch.uint8, device="cuda"))
    L.embedding_grad(0, ids, dx, grad, torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda"), 2.0)
    leaf = table.double().requires_grad_()
    hh = leaf[ids.long()] * 2
    ((hh * w.double() / torch.sqrt((hh * hh).mean(1, keepdim=True) + 1e-6)) * dy.double()).sum().backward()
    assert float((grad.double() - leaf.grad).abs().max()) <= 1e-4 * float(leaf.grad.abs().max())


def test_captured_with_other_rows():
    import torch
    for m in (2, 24, 300):
        a, b = _coded(m, 256, L.CODEC_INT8, 0, 5), _coded(200, 256, L.CODEC_INT8, 0, 6)
        out = torch.empty(m, 200, device="cuda")
        side = torch.cuda.Stream()
        L.matmul_rows(0, L.CODEC_INT8, a[0], b[0], 256, out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            L.matmul_rows(0, L.CODEC_INT8, a[0], b[0], 256, out, stream=torch.cuda.current_stream())
        c = _coded(m, 256, L.CODEC_INT8, 0, 9)
        a[0].copy_(c[0])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        _check(out, c, b, 256, L.CODEC_INT8)


def test_two_streams_at_once():
    """Kernels that fill the chip, each with all of an SM's tensor memory, on two streams: the same as one after the other."""
    import torch
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = [(_coded(m, k, L.CODEC_INT8, 0, 20 + m), _coded(n, k, L.CODEC_INT8, 0, 30 + n), k, torch.empty(m, n, device="cuda", dtype=torch.bfloat16))
            for m, n, k in ((2000, 4000, 512), (300, 3000, 1024))]
    torch.cuda.synchronize()
    for turn in range(4):
        for k, (a, b, width, out) in enumerate(work):
            L.matmul_rows(0, L.CODEC_INT8, a[0], b[0], width, out, stream=sides[k])
    torch.cuda.synchronize()
    for a, b, width, out in work:
        again = torch.empty_like(out)
        L.matmul_rows(0, L.CODEC_INT8, a[0], b[0], width, again)
        assert torch.equal(out, again)
    assert L.operator_error(0) == 0


def test_nothing_to_do_and_refusals():
    import torch
    a, b = _coded(4, 64, 1)[0], _coded(6, 64, 1)[0]
    out = torch.full((4, 6), 3.0, device="cuda")
    L.matmul_rows(0, 1, a[:0], b, 64, out[:0])
    for bad in (lambda: L.matmul_rows(0, 0, a, b, 64, out), lambda: L.matmul_rows(0, 1, a, b, 62, out), lambda: L.matmul_rows(0, 1, a, b, 128, out),
                lambda: L.matmul_rows(0, 1, a, b, 64, out[:, :5]), lambda: L.matmul_rows(0, 1, a.float(), b, 64, out),
                lambda: L.matmul_rows(0, 1, a, b, 64, out.double()), lambda: L.matmul_rows(0, 1, a, b, 0, out),
                lambda: L.matmul_rows(0, 1, a[:, 4:], b, 60, out), lambda: L.matmul_rows(0, 1, a, b.cpu(), 64, out)):
        with pytest.raises(L.LegionError):
            bad()
    long = torch.zeros(1, 131088, dtype=torch.uint8, device="cuda")
    with pytest.raises(L.LegionError, match="limit"):
        L.matmul_rows(0, 1, long, long, 131072, torch.zeros(1, 1, device="cuda"))
    assert bool((out == 3.0).all())


@pytest.mark.parametrize("codec", CODECS)
def test_scales_far_from_one(codec):
    """Scales whose product leaves fp32's range while the result does not, at every number of rows that is served in a way of its own: each
    result is the sum scaled, and int8 rows (whose sums are exact) give the same bits whatever other rows are in the call.  The sum meets the
    row's scale first, above 2^92 the weight's: a whole number times a subnormal one is exact or normal, so the three roundings of _check are all
    (e4m3 sums are multiples of 2^-18: scales from 1e-30 on keep them normal)."""
    import torch
    n, k, most = 1280, 64, 3712
    a, b = _coded(most, k, codec, 0, 11), _coded(n, k, codec, 0, 12)
    a[0][::7, :k] = 0
    a[1][::7] = 0
    low = -44.0 if codec == L.CODEC_INT8 else -30.0
    scales = []
    for rows in (a, b):
        s = (10.0 ** (low + (30.0 - low) * torch.rand(rows[0].shape[0], device="cuda", dtype=torch.float64))).float()
        s[0], s[1], s[2] = 1e25, 1e-22, 1e-23
        rows[0].view(torch.float32)[:, k // 4] = s
        scales.append(s.double())
    sums, outer = a[1] @ b[1].t(), scales[0][:, None] * scales[1][None]
    want = sums * outer
    slack = want.abs() * (3 * U32)
    if codec == L.CODEC_E4M3:
        slack = slack + (a[1].abs() @ b[1].abs().t()) * outer * (k * 2 * U32)
    over = want.abs() > 3.4e38
    near = over | (want.abs() + slack > 3.4e38)
    whole = None
    for m in (most, 2500, 1500, 300, 100, 50, 20, 9, 1):
        out = torch.empty(m, n, device="cuda")
        L.matmul_rows(0, codec, a[0][:m], b[0], k, out)
        assert not bool(torch.isnan(out).any())
        assert torch.equal(torch.isinf(out) | near[:m], near[:m])
        _close(torch.where(near[:m], 0.0, out), torch.where(near[:m], 0.0, want[:m]), torch.where(near[:m], 0.0, slack[:m]))
        assert bool((out[::7] == 0).all())
        if codec == L.CODEC_INT8:
            whole = out if whole is None else whole
            assert torch.equal(out, whole[:m])
    assert int(over.sum()) > 0


@pytest.mark.parametrize("m,n,k", [(1, 300, 64), (20, 1280, 4100), (100, 40, 260), (300, 1280, 4100), (1500, 1280, 64), (2500, 1280, 2052), (3712, 1280, 1028), (2500, 9001, 132)])
@pytest.mark.parametrize("codec", CODECS)
def test_a_wait_that_is_given_up(codec, m, n, k):
    """Limit 0: nothing is brought, the waits for it run out, and the call ends with its error; limits about as long as a tile takes: some waits may
    run out and others not, and the call ends with an error or is right.  (One row is worked out without waits.)"""
    import torch
    a, b = _coded(m, k, codec, 0, 1), _coded(n, k, codec, 0, 2)
    want = torch.empty(m, n, device="cuda")
    L.matmul_rows(0, codec, a[0], b[0], k, want)
    assert L.operator_error(0) == 0
    try:
        for limit in (0, 1, 20, 40, 100, 300):
            L.operator_wait_limit(limit)
            out = torch.empty(m, n, device="cuda")
            L.matmul_rows(0, codec, a[0], b[0], k, out)
            error = L.operator_error(0, reset=False)
            assert error in ((0,) if m == 1 else (-7,) if limit == 0 else (0, -7))
            assert L.operator_error(0) == error and L.operator_error(0) == 0   # kept until it is reset
            if error == 0:
                assert torch.equal(out, want)
    finally:
        L.operator_wait_limit(2000000)
    out = torch.empty(m, n, device="cuda")
    L.matmul_rows(0, codec, a[0], b[0], k, out)
    assert L.operator_error(0) == 0 and torch.equal(out, want)


@pytest.mark.parametrize("codec", CODECS)
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("m", [1, 20, 100, 131, 300, 1500, 2500, 3712])
@pytest.mark.parametrize("n", [1, 5, 66, 265, 1001, 1279, 1283])
def test_rows_that_end_inside_16_bytes(codec, out_type, m, n):
    """Rows of the output that start on 16-byte boundaries, whatever their length: what lies between them stays as it was."""
    import torch
    t, k = _types()[out_type], 64
    per = 16 // t.itemsize
    for pad in (-n % per, -n % per + per):
        a, b = _coded(m, k, codec, 0, 21), _coded(n, k, codec, 0, 22)
        a = (a[0], a[1], a[2] / 4096)
        a[0].view(torch.float32)[:, k // 4] = a[2].float()
        whole, out = _strided(m, n, t, pad, 0)
        L.matmul_rows(0, codec, a[0], b[0], k, out)
        # fp16: what lies beyond the type's largest number, whose last binade has steps of 2^-10, is infinite or that number
        want = (a[1] @ b[1].t()) * a[2][:, None] * b[2][None]
        over = want.abs() > torch.finfo(t).max * (1 - 2 ** -11)
        assert bool((out[over].abs() >= torch.finfo(t).max * (1 - 2 ** -10)).all())
        slack = want.abs() * (3 * U32)
        if codec == L.CODEC_E4M3:
            slack = slack + (a[1].abs() @ b[1].abs().t()) * a[2][:, None] * b[2][None] * (k * 2 * U32)
        _close(torch.where(over, 0.0, out), torch.where(over, 0.0, want), torch.where(over, 0.0, slack))
        rest = whole.clone()
        torch.as_strided(rest, (m, n), (n + pad, 1), 0).fill_(7.0)
        assert bool((rest == 7.0).all())
