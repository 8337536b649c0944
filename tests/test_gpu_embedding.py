"""Lookup of learned rows and its gradient against 64-bit sums.

Tolerances: a product or a sum in fp32 is off by at most half a step, 2^-24 relative; c terms added in any order by at
most (c - 1) of those relative to the sum of their magnitudes; the last rounding by half a step of the output's type (for a
subnormal result, by half of the smallest number)."""
import numpy as np
import pytest

import legion_ibp_b200 as L

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24


def _types():
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _half_step(dtype):
    import torch
    return torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _close(got, want, slack):
    """|got - want| <= half a step of got's type + slack (fp32 work)."""
    import torch
    rel, least = _half_step(got.dtype)
    bound = want.abs() * (rel * (1 + 2 ** -10)) + least + slack * (1 + rel)
    off = (got.double() - want).abs() - bound
    assert bool(torch.isfinite(got.double()).all())
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def _strided(n, width, dtype, pad, shift):
    """[n, width] rows with `pad` elements between them that start `shift` elements behind an aligned address; pad filled with 7."""
    import torch
    whole = torch.full((n * (width + pad) + shift + 8,), 7.0, dtype=dtype, device="cuda")
    return whole, torch.as_strided(whole, (n, width), (width + pad, 1), shift)


def _ids(rng, n, nodes, wide, skew=1.0):
    import torch
    ids = np.minimum((nodes * rng.random(n) ** skew).astype(np.int64), nodes - 1)
    return torch.from_numpy(ids.astype(np.int64 if wide else np.int32)).cuda()


def _exact_grad(ids, grad, nodes, scale):
    """(gradient, sum of magnitudes, rows per id) in 64 bits; ids outside the table are left out."""
    import torch
    ids = ids.long()
    keep = (ids >= 0) & (ids < nodes)
    g = grad.double()[keep] * scale
    total = torch.zeros((nodes, grad.shape[1]), dtype=torch.float64, device="cuda").index_add_(0, ids[keep], g)
    mag = torch.zeros_like(total).index_add_(0, ids[keep], g.abs())
    return total, mag, torch.bincount(ids[keep], minlength=nodes)


@pytest.mark.parametrize("table_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("out_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,dim,pad,shift", [(1, 1, 0, 0), (3, 7, 0, 0), (257, 128, 0, 0), (1000, 100, 4, 0), (65, 602, 0, 0),
                                             (4099, 75, 3, 1), (5, 4096, 8, 8), (33000, 48, 0, 0), (17, 65536, 0, 0)])
def test_lookup(table_type, out_type, n, dim, pad, shift):
    import torch
    t = _types()
    rng = np.random.default_rng(n + dim)
    nodes = 301
    _, table = _strided(nodes, dim, t[table_type], pad, shift)
    table.copy_(torch.randn(nodes, dim, device="cuda"))
    for wide in (False, True):
        ids = _ids(rng, n, nodes, wide)
        if n > 2:
            ids[1], ids[n // 2] = -1, nodes
        whole, out = _strided(n, dim, t[out_type], pad, shift)
        L.embedding_lookup(0, table, ids, out, 2.375)
        want = torch.where(((ids >= 0) & (ids < nodes))[:, None], table.double()[ids.long().clamp(0, nodes - 1)] * 2.375, 0.0)
        _close(out, want, want.abs() * U32)
        rest = whole.clone()
        torch.as_strided(rest, (n, dim), (dim + pad, 1), shift).fill_(7.0)
        assert bool((rest == 7.0).all())  # nothing between the rows is written


def test_lookup_keeps_bits_and_special_values():
    """Scale 1 and one type: the rows themselves, infinities and NaN among them; a row that is not asked for does not leak."""
    import torch
    for t in _types().values():
        table = torch.randn(50, 40, device="cuda").to(t)
        table[3, 5], table[4, 6], table[7] = float("inf"), -float("inf"), float("nan")
        ids = torch.tensor([4, 3, 0, 3, 49], device="cuda")
        out = torch.zeros(5, 40, dtype=t, device="cuda")
        L.embedding_lookup(0, table, ids, out)
        assert torch.equal(out, table[ids])


def test_lookup_far_row_offsets():
    """Rows behind 2^31 elements of the table."""
    import torch
    nodes, dim = 2200000, 1024
    table = torch.zeros((nodes, dim), dtype=torch.float16, device="cuda")
    far = torch.tensor([0, 2097151, 2097152, 2097153, nodes - 1, 1], device="cuda")
    table[far] = torch.randn(6, dim, device="cuda").half()
    out = torch.zeros(6, dim, dtype=torch.float16, device="cuda")
    L.embedding_lookup(0, table, far, out)
    assert torch.equal(out, table[far])


SHAPES = [(1, 1, 1, 1.0), (2, 5, 3, 1.0), (31, 40, 64, 2.0), (32, 3, 8, 1.0), (33, 1, 20, 1.0), (333, 5003, 602, 2.0), (1000, 300, 75, 3.0),
          (4096, 2, 100, 1.0), (8192, 700, 16, 2.0), (8193, 700, 16, 2.0), (20000, 40000, 33, 3.0), (70001, 1 << 20, 24, 3.0),
          (3000, 1 << 24, 4, 2.0), (1024, 65535, 12, 1.0), (1025, 65536, 12, 1.0), (90113, 255, 8, 1.0), (180224, 256, 5, 2.0),
          (180225, 4000, 6, 2.0), (600001, 70000, 4, 3.0)]


@pytest.mark.parametrize("n,nodes,dim,skew", SHAPES)
@pytest.mark.parametrize("grad_type,table_type", [("f32", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
def test_gradient_of_the_whole_table(n, nodes, dim, skew, grad_type, table_type):
    import torch
    t = _types()
    rng = np.random.default_rng(n)
    wide = n % 2 == 0
    ids = _ids(rng, n, nodes, wide, skew)
    if n > 100:
        ids[5], ids[77] = -1, nodes
    grad = torch.randn(n, dim, device="cuda").to(t[grad_type])
    want, mag, count = _exact_grad(ids, grad, nodes, 1.75)
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda").fill_(0xA5)
    out = torch.full((nodes, dim), 3.0, dtype=t[table_type], device="cuda")
    L.embedding_grad(0, ids, grad, out, ws, 1.75)
    slack = mag * ((count[:, None] + 2).double() * U32)
    _close(out, want, slack)
    # twice: the same bits; added to what is there
    again = torch.full_like(out, -1.0)
    L.embedding_grad(0, ids, grad, again, ws, 1.75)
    assert torch.equal(out, again)
    start = torch.randn(nodes, dim, device="cuda").to(t[table_type])
    more = start.clone()
    L.embedding_grad(0, ids, grad, more, ws, 1.75, accumulate=True)
    _close(more, want + start.double(), slack + (want.abs() + start.double().abs()) * (2 * U32))
    assert torch.equal(more[count == 0], start[count == 0])


@pytest.mark.parametrize("n,nodes,dim,skew", SHAPES)
@pytest.mark.parametrize("grad_type", ["f32", "bf16", "f16"])
def test_gradient_rows(n, nodes, dim, skew, grad_type):
    import torch
    rng = np.random.default_rng(n + 1)
    wide = n % 2 == 1
    ids = _ids(rng, n, nodes, wide, skew)
    if n > 100:
        ids[5], ids[77] = -1, nodes
    grad = torch.randn(n, dim, device="cuda").to(_types()[grad_type])
    want, mag, count = _exact_grad(ids, grad, nodes, 0.5)
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda").fill_(0xA5)
    unique = torch.full((n + 3,), -9, dtype=ids.dtype, device="cuda")
    rows = torch.full((n + 3, dim), -9.0, device="cuda")
    found = torch.full((1,), -9, dtype=torch.int32, device="cuda")
    L.embedding_grad_rows(0, ids, grad, nodes, unique, rows, found, ws, 0.5)
    occur = torch.nonzero(count).flatten()
    k = occur.numel()
    assert int(found) == k
    assert torch.equal(unique[:k].long(), occur)
    _close(rows[:k], want[occur], mag[occur] * ((count[occur][:, None] + 2).double() * U32))
    assert bool((unique[k:] == -9).all()) and bool((rows[k:] == -9.0).all())


@pytest.mark.parametrize("n", [40, 5000, 70000])
def test_gradient_of_one_id_and_of_none(n):
    """Every position names the same row (one sum over all stretches); every position is padding."""
    import torch
    nodes, dim = 9, 130
    ids = torch.full((n,), 4, dtype=torch.int32, device="cuda")
    grad = torch.randn(n, dim, device="cuda")
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda")
    out = torch.ones(nodes, dim, device="cuda")
    L.embedding_grad(0, ids, grad, out, ws)
    want, mag, count = _exact_grad(ids, grad, nodes, 1.0)
    _close(out, want, mag * ((count[:, None] + 2).double() * U32))
    out.fill_(1.0)
    L.embedding_grad(0, torch.full_like(ids, -1), grad, out, ws)
    assert bool((out == 0).all())
    unique, rows = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(n, dim, device="cuda")
    found = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    L.embedding_grad_rows(0, torch.full_like(ids, nodes), grad, nodes, unique, rows, found, ws)
    assert int(found) == 0 and bool((rows == 0).all())


def test_gradient_nan_stays_in_its_row_and_strides():
    import torch
    n, nodes, dim = 9000, 37, 50
    rng = np.random.default_rng(3)
    ids = _ids(rng, n, nodes, True)
    whole, grad = _strided(n, dim, torch.bfloat16, 6, 2)
    grad.copy_(torch.randn(n, dim, device="cuda"))
    grad[17, 3], grad[18, 4] = float("nan"), float("inf")
    ids[17], ids[18] = 5, 6
    ids[19] = -1
    grad[19] = float("nan")   # the gradient of padding is not read into any row
    outs, out = _strided(nodes, dim, torch.float32, 2, 2)
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda")
    L.embedding_grad(0, ids, grad, out, ws)
    want, mag, count = _exact_grad(ids, grad, nodes, 1.0)
    assert bool(torch.isnan(out[5, 3])) and float(out[6, 4]) == float("inf")
    ok = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out), ok) and int((~ok).sum()) == 2
    slack = torch.where(ok, mag * ((count[:, None] + 2).double() * U32), 0.0)
    _close(torch.where(ok, out, 0.0), torch.where(ok, want, 0.0), slack)
    rest = outs.clone()
    torch.as_strided(rest, (nodes, dim), (dim + 2, 1), 2).fill_(7.0)
    assert bool((rest == 7.0).all())


@pytest.mark.parametrize("table_type,pad,shift", [("f32", 1, 1), ("f16", 3, 1), ("bf16", 2, 2), ("f32", 4, 0), ("f16", 8, 0)])
@pytest.mark.parametrize("n,dim", [(5, 17), (700, 64), (3000, 130), (30000, 10)])
def test_gradient_of_tables_with_strides(n, dim, table_type, pad, shift):
    """Rows that no id names are zeroed, what lies between the rows is not."""
    import torch
    nodes = 900
    ids = _ids(np.random.default_rng(n), n, nodes, False, 2.0)
    grad = torch.randn(n, dim, device="cuda")
    whole, out = _strided(nodes, dim, _types()[table_type], pad, shift)
    L.embedding_grad(0, ids, grad, out, torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda"), 0.25)
    want, mag, count = _exact_grad(ids, grad, nodes, 0.25)
    _close(out, want, mag * ((count[:, None] + 2).double() * U32))
    rest = whole.clone()
    torch.as_strided(rest, (nodes, dim), (dim + pad, 1), shift).fill_(7.0)
    assert bool((rest == 7.0).all())


def test_two_streams_at_once():
    """Calls that share nothing but their inputs, on two streams, against the same calls one after the other."""
    import torch
    rng = np.random.default_rng(4)
    nodes, dim = 4000, 256
    table = torch.randn(nodes, dim, device="cuda").half()
    sides = [torch.cuda.Stream() for _ in range(2)]
    work = []
    for n in (15000, 40000):
        ids = _ids(rng, n, nodes, True, 3.0)
        work.append((ids, torch.randn(n, dim, device="cuda"), [torch.empty(n, dim, device="cuda", dtype=torch.half) for _ in range(2)],
                     [torch.empty(nodes, dim, device="cuda") for _ in range(2)],
                     [torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda") for _ in range(2)]))
    torch.cuda.synchronize()
    for turn in range(5):
        for k, (ids, grad, out, whole, ws) in enumerate(work):
            L.embedding_lookup(0, table, ids, out[0], 2.0, stream=sides[k])
            L.embedding_grad(0, ids, grad, whole[0], ws[0], stream=sides[k])
    torch.cuda.synchronize()
    for ids, grad, out, whole, ws in work:
        L.embedding_lookup(0, table, ids, out[1], 2.0)
        L.embedding_grad(0, ids, grad, whole[1], ws[1])
        assert torch.equal(out[0], out[1]) and torch.equal(whole[0], whole[1])


def test_gradient_against_differences():
    """The lookup is linear in the table: <grad, step> is the difference of <out, weights> over any step."""
    import torch
    torch.manual_seed(1)
    n, nodes, dim = 600, 50, 24
    ids = torch.randint(0, nodes, (n,), device="cuda")
    table, step, g = torch.randn(nodes, dim, device="cuda"), torch.randn(nodes, dim, device="cuda"), torch.randn(n, dim, device="cuda")
    out = [torch.empty(n, dim, device="cuda") for _ in range(2)]
    L.embedding_lookup(0, table, ids, out[0], 3.0)
    L.embedding_lookup(0, table + step, ids, out[1], 3.0)
    grad = torch.empty(nodes, dim, device="cuda")
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda")
    L.embedding_grad(0, ids, g, grad, ws, 3.0)
    difference = ((out[1].double() - out[0].double()) * g.double()).sum()
    # each output is off by two roundings of values up to |table| + |step|; each sum of n / nodes = 12 terms or a few more
    slack = 40 * U32 * float((3.0 * (table.abs() + step.abs()).double()[ids] * g.double().abs()).sum())
    assert abs(float((grad.double() * step.double()).sum() - difference)) <= slack


@pytest.mark.parametrize("n", [300, 9000, 50000])
def test_gradient_captured_and_replayed_on_another_stream(n):
    """Two captured gradients with workspaces of their own, replayed over changed inputs, side by side with an eager one."""
    import torch
    nodes, dim = 500, 64
    rng = np.random.default_rng(11)
    sides = [torch.cuda.Stream() for _ in range(2)]
    made = []
    for k in range(2):
        ids, grad = _ids(rng, n, nodes, False, 2.0), torch.randn(n, dim, device="cuda")
        out = torch.empty(nodes, dim, device="cuda")
        ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda")
        L.embedding_grad(0, ids, grad, out, ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=sides[k]):
            L.embedding_grad(0, ids, grad, out, ws, stream=torch.cuda.current_stream())
        made.append((ids, grad, out, ws, graph))
    for turn in range(3):
        for ids, grad, *_ in made:
            ids.copy_(_ids(rng, n, nodes, False, 2.0))
            grad.copy_(torch.randn(n, dim, device="cuda"))
        torch.cuda.synchronize()
        for k, (ids, grad, out, ws, graph) in enumerate(made):
            with torch.cuda.stream(sides[k]):
                graph.replay()
        torch.cuda.synchronize()
        for ids, grad, out, ws, graph in made:
            eager = torch.empty_like(out)
            L.embedding_grad(0, ids, grad, eager, torch.empty_like(ws))
            assert torch.equal(eager, out)


def test_no_rows():
    import torch
    none, table = torch.zeros(0, dtype=torch.int64, device="cuda"), torch.ones(5, 8, device="cuda")
    L.embedding_lookup(0, table, none, torch.zeros(0, 8, device="cuda"))
    grad = torch.ones(5, 8, device="cuda")
    L.embedding_grad(0, none, torch.zeros(0, 8, device="cuda"), grad, None, accumulate=True)
    assert bool((grad == 1).all())
    L.embedding_grad(0, none, torch.zeros(0, 8, device="cuda"), grad, None)
    assert bool((grad == 0).all())
    found = torch.full((1,), 7, dtype=torch.int32, device="cuda")
    L.embedding_grad_rows(0, none, torch.zeros(0, 8, device="cuda"), 5, none, torch.zeros(0, 8, device="cuda"), found, None)
    assert int(found) == 0


def test_refusals():
    import torch
    ids, table, out = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(5, 8, device="cuda"), torch.zeros(4, 8, device="cuda")
    for bad in (lambda: L.embedding_lookup(0, table, ids, out[:3]), lambda: L.embedding_lookup(0, table, ids, out.double()),
                lambda: L.embedding_lookup(0, table.cpu(), ids, out), lambda: L.embedding_lookup(0, table, ids.float(), out),
                lambda: L.embedding_lookup(0, table.t(), ids, torch.zeros(4, 5, device="cuda")),
                lambda: L.embedding_lookup(1, table, ids, out), lambda: L.embedding_lookup(0, table, ids.short(), out),
                lambda: L.embedding_lookup(0, table, ids, torch.zeros(1, 8, device="cuda").expand(4, 8)),
                lambda: L.embedding_grad(0, ids, out, table, None),
                lambda: L.embedding_grad(0, ids, out, table, torch.zeros(16, dtype=torch.uint8, device="cuda")),
                lambda: L.embedding_grad(0, ids, out[:, :4], table, torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")),
                lambda: L.embedding_grad_rows(0, ids, out, 5, ids, out.half(), ids[:1], torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")),
                lambda: L.embedding_grad_rows(0, ids, out, 5, ids.long(), out, ids[:1], torch.zeros(1 << 20, dtype=torch.uint8, device="cuda"))):
        with pytest.raises(L.LegionError):
            bad()


@pytest.mark.parametrize("scale", [float("inf"), -2.0, float("nan")])
@pytest.mark.parametrize("n,dim,dtype", [(5, 64, "f32"), (3000, 128, "bf16"), (50, 333, "f16"), (9, 7, "f32")])
def test_lookup_outside_the_table_is_zero_whatever_the_scale(n, dim, dtype, scale):
    import torch
    t = _types()[dtype]
    table = torch.ones(10, dim, dtype=t, device="cuda")
    ids = torch.arange(n, device="cuda") % 12 - 1   # -1 and 10 among them
    out = torch.full((n, dim), 3.0, dtype=t, device="cuda")
    L.embedding_lookup(0, table, ids, out, scale)
    none = (ids < 0) | (ids > 9)
    assert bool((out[none].view(torch.int32 if dtype == "f32" else torch.int16) == 0).all())
    assert torch.equal(out[~none].nan_to_num(7.0), torch.full_like(out[~none], scale).nan_to_num(7.0))


@pytest.mark.parametrize("n", [0, 40, 5000, 30000])
def test_gradient_of_a_table_with_far_rows(n):
    """Rows of the table that lie more than 2^31 bytes apart."""
    import torch
    nodes, dim, stride = 2, 64, (1 << 29) + 64
    whole = torch.full((stride + dim,), 7.0, device="cuda")
    out = torch.as_strided(whole, (nodes, dim), (stride, 1))
    ids, grad = torch.ones(n, dtype=torch.int32, device="cuda"), torch.ones(n, dim, device="cuda")
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda")
    L.embedding_grad(0, ids, grad, out, ws)
    assert bool((out[0] == 0).all()) and bool((out[1] == n).all())   # whole numbers: exact
    assert bool((whole[dim:stride] == 7.0).all())


@pytest.mark.parametrize("n,nodes,dim", [((1 << 20) + 5, 70000, 3), ((1 << 22) + 3, 1 << 20, 2), (30001, (1 << 24) + 9, 3)])
def test_gradient_of_the_longest_lists_and_largest_tables(n, nodes, dim):
    """Stretches of 64 and of 128 entries, four passes over long lists."""
    import torch
    rng = np.random.default_rng(n)
    ids = _ids(rng, n, nodes, False, 2.0)
    ids[5], ids[77] = -1, nodes
    grad = torch.randn(n, dim, device="cuda")
    want, mag, count = _exact_grad(ids, grad, nodes, 1.0)
    ws = torch.empty(L.embedding_grad_workspace(n, dim, nodes), dtype=torch.uint8, device="cuda").fill_(0xA5)
    out = torch.full((nodes, dim), 3.0, device="cuda")
    L.embedding_grad(0, ids, grad, out, ws)
    _close(out, want, mag * ((count[:, None] + 2).double() * U32))
    unique, rows = torch.full((n,), -9, dtype=torch.int32, device="cuda"), torch.full((n, dim), -9.0, device="cuda")
    found = torch.zeros(1, dtype=torch.int32, device="cuda")
    L.embedding_grad_rows(0, ids, grad, nodes, unique, rows, found, ws)
    occur = torch.nonzero(count).flatten()
    k = occur.numel()
    assert int(found) == k and torch.equal(unique[:k].long(), occur)
    assert torch.equal(rows[:k], out[occur])   # the same sums in the same order
    assert bool((unique[k:] == -9).all()) and bool((rows[k:] == -9.0).all())
