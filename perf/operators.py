"""The operators on learned and compressed rows, as cases that can be timed and compared.

A case is a dict of plain values.  Its "kind" is the call (or the calls) that a pass makes:

  lookup        embedding_lookup: rows of a learned table by id, scaled
  grad          embedding_grad: the gradient of the whole table
  grad_rows     embedding_grad_rows: the rows of the gradient that are not zero, by rising id
  norm          rms_norm, with or without the residual's addition, output in the type of its input
  norm_codes    rms_norm with the output as compressed rows (e4m3 codes and a scale per row)
  norm_grad     rms_norm_grad
  project       matmul_rows: compressed rows times compressed weight rows
  norm_project  rms_norm to compressed rows, then matmul_rows: a layer's first product, as it is served

Where `own` is false a pass computes the same from elementary torch operations.
"""
import functools
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32, "i64": torch.int64}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4, "i64": 8}
_TOP = {"int8": 127.0, "e4m3": 448.0}
_EPS = 1e-6


@functools.lru_cache(maxsize=None)
def _package():
    """The package directory is `legion-ibp_b200` (beside this folder); it is imported as legion_ibp_b200."""
    if "legion_ibp_b200" in sys.modules:
        return sys.modules["legion_ibp_b200"]
    pkg = os.path.join(os.getcwd(), "legion-ibp_b200")
    spec = importlib.util.spec_from_file_location("legion_ibp_b200", os.path.join(pkg, "__init__.py"),
                                                  submodule_search_locations=[pkg])
    mod = importlib.util.module_from_spec(spec)
    sys.modules["legion_ibp_b200"] = mod
    spec.loader.exec_module(mod)
    return mod


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # a decode step of 16 sequences: the ids of the last tokens, rows scaled by sqrt(width)
        dict(name="lookup-token", kind="lookup", n=16, nodes=32000, dim=4096, table="bf16", out="bf16", ids="i64", scale=64.0, skew=3.0),
        # learned rows of the nodes of a products-shaped batch, 400 bytes each
        dict(name="lookup-nodes", kind="lookup", n=200000, nodes=2449029, dim=100, table="f32", out="f32", ids="i32", scale=1.0, skew=1.0),
        # a training step's tokens, frequent ones thousands of times; the optimizer takes the whole gradient in fp32
        dict(name="grad-tokens", kind="grad", n=16384, nodes=32000, dim=2048, grad="bf16", table="f32", ids="i64", scale=45.25, skew=3.0),
        # a small batch over a small table, odd sizes, gradient kept in the type of the rows
        dict(name="grad-ragged", kind="grad", n=333, nodes=5003, dim=602, grad="f16", table="f16", ids="i32", scale=1.0, skew=2.0),
        # learned node rows, the nodes of four products-shaped batches: the optimizer touches the rows that occur
        dict(name="grad-nodes", kind="grad_rows", n=150000, nodes=2449029, dim=128, grad="f32", ids="i32", scale=1.0, skew=2.0),
        # a decode step of 8 sequences between two layers
        dict(name="norm-token", kind="norm", n=8, dim=4096, x="bf16", weight="bf16", residual=True),
        # feature rows normed before the first layer, 2408 bytes each, no residual yet
        dict(name="norm-ragged", kind="norm", n=12371, dim=602, x="f32", weight="f32", residual=False),
        # a prompt's rows between two layers, output as compressed rows for the next product
        dict(name="norm-e4m3", kind="norm_codes", n=8192, dim=4096, x="bf16", weight="bf16", residual=True, codec="e4m3"),
        # the way back through the norm of a training step, the gradient of the residual stream added
        dict(name="norm-grad", kind="norm_grad", n=16384, dim=2048, x="bf16", weight="f32", residual=True),
        # one token's product: all of the weights for one row
        dict(name="project-token", kind="project", m=1, n=16384, dim=4096, codec="int8", out="bf16"),
        # a prompt's product
        dict(name="project-prompt", kind="project", m=4096, n=16384, dim=4096, codec="int8", out="bf16"),
        # a few hundred rows of 768 features normed, encoded and projected to a ragged number of classes
        dict(name="norm-project", kind="norm_project", m=611, n=1000, dim=768, x="f16", weight="f32", residual=False, codec="int8", out="f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["lookup", "grad", "grad_rows", "norm", "norm_codes", "norm_grad", "project", "project", "norm_project"])
    if kind in ("lookup", "grad", "grad_rows"):
        dim = rng.choice([_spread(rng, 16, 8192), 8 * _spread(rng, 4, 1024)])
        case = dict(kind=kind, n=_spread(rng, 1, 300000), nodes=_spread(rng, 500, 3000000), dim=dim, ids=rng.choice(["i32", "i64"]),
                    scale=rng.choice([1.0, math.sqrt(dim)]), skew=rng.choice([1.0, 2.0, 3.0]))
        if kind == "lookup":
            elt = rng.choice(["f32", "f16", "bf16"])
            return dict(case, table=elt, out=rng.choice([elt, "f32", "bf16"]))
        if kind == "grad":
            elt = rng.choice(["f32", "f16", "bf16"])
            return dict(case, grad=elt, table=rng.choice([elt, "f32"]))
        return dict(case, grad=rng.choice(["f32", "f16", "bf16"]))
    x = rng.choice(["f32", "f16", "bf16", "bf16"])
    weight = rng.choice([x, "f32"])
    if kind in ("norm", "norm_grad"):
        return dict(kind=kind, n=_spread(rng, 1, 60000), dim=rng.choice([_spread(rng, 16, 8192), 8 * _spread(rng, 4, 1500)]), x=x,
                    weight=weight, residual=rng.random() < 0.6)
    if kind == "norm_codes":
        return dict(kind=kind, n=_spread(rng, 1, 60000), dim=4 * _spread(rng, 4, 3000), x=x, weight=weight,
                    residual=rng.random() < 0.6, codec="e4m3")
    codec = rng.choice(["int8", "int8", "e4m3"])
    out = rng.choice(["bf16", "f16", "f32"] if codec == "int8" and kind == "project" else ["bf16", "f16"])
    case = dict(kind=kind, m=_spread(rng, 1, 8192), n=_spread(rng, 16, 16384), dim=4 * _spread(rng, 4, 2048), codec=codec, out=out)
    return case if kind == "project" else dict(case, x=x, weight=weight, residual=rng.random() < 0.5)


def draw(rng):
    most = [work(c) for c in listed()]
    bytes_, flops = (max(w[k] for w in most) for k in ("bytes", "flops"))
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= bytes_ and w["flops"] <= flops and case.get("nodes", 0) * case["dim"] <= 320000000:
            return case


# ---- what a pass needs -------------------------------------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _expected_unique(n, nodes, skew):
    """Different ids among n draws of floor(nodes * u^skew)."""
    edge = (np.arange(nodes + 1, dtype=np.float64) / nodes) ** (1.0 / skew)
    return float((1.0 - (1.0 - np.minimum(np.diff(edge), 1.0)) ** n).sum())


def work(case):
    kind, dim = case["kind"], case["dim"]
    if kind in ("lookup", "grad", "grad_rows"):
        n, ids = case["n"], _SIZE[case["ids"]]
        if kind == "grad":
            return {"bytes": n * (ids + dim * _SIZE[case["grad"]]) + case["nodes"] * dim * _SIZE[case["table"]], "flops": 2 * n * dim}
        unique = _expected_unique(n, case["nodes"], case["skew"])
        if kind == "lookup":
            return {"bytes": n * (ids + dim * _SIZE[case["out"]]) + unique * dim * _SIZE[case["table"]], "flops": n * dim}
        return {"bytes": n * (ids + dim * _SIZE[case["grad"]]) + unique * (ids + dim * 4), "flops": 2 * n * dim}
    if kind == "project":
        m, n = case["m"], case["n"]
        return {"bytes": (m + n) * (dim + 4) + m * n * _SIZE[case["out"]], "flops": 2 * m * n * dim}
    x, w = _SIZE[case["x"]], _SIZE[case["weight"]]
    more = 2 * x if case["residual"] else 0   # the residual in, the sum out
    if kind == "norm":
        return {"bytes": case["n"] * dim * (2 * x + more) + dim * w, "flops": 5 * case["n"] * dim}
    if kind == "norm_codes":
        return {"bytes": case["n"] * (dim * (x + more + 1) + 4) + dim * w, "flops": 7 * case["n"] * dim}
    if kind == "norm_grad":
        return {"bytes": case["n"] * dim * (3 * x + more // 2) + dim * (w + 4), "flops": 12 * case["n"] * dim}
    m, n = case["m"], case["n"]
    return {"bytes": m * dim * (x + more) + dim * w + n * (dim + 4) + m * n * _SIZE[case["out"]], "flops": 2 * m * n * dim}


# ---- inputs ------------------------------------------------------------------------------------------------------

class _State:
    pass


def _slot(dim):
    """Bytes of a compressed row: codes, an fp32 scale, zeros up to a multiple of 16."""
    return (dim + 4 + 15) // 16 * 16


def _encoded(rows, codec):
    """Compressed rows of fp32 rows."""
    n, dim = rows.shape
    a = rows.abs().amax(1, keepdim=True)
    scaled = rows * (_TOP[codec] / a)
    out = torch.zeros((n, _slot(dim)), dtype=torch.uint8, device=rows.device)
    out[:, :dim] = (scaled.round().to(torch.int8) if codec == "int8" else scaled.to(torch.float8_e4m3fn)).view(torch.uint8)
    out.view(torch.float32)[:, dim // 4] = (a / _TOP[codec]).squeeze(1)
    return out


def prepare(case, seed):
    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 16 + 5)
    s = _State()
    s.case, kind, dim = case, case["kind"], case["dim"]

    def normal(n, width, elt, std=1.0):
        return (torch.randn(n, width, device="cuda", generator=g) * std).to(_DTYPE[elt])

    def empty(n, width, elt):
        return torch.zeros((n, width), dtype=_DTYPE[elt], device="cuda")

    if kind in ("lookup", "grad", "grad_rows"):
        n, nodes = case["n"], case["nodes"]
        # a few ids come often; which ones is scattered over the table
        ids = (nodes * torch.rand(n, device="cuda", generator=g, dtype=torch.float64) ** case["skew"]).long().clamp_(max=nodes - 1)
        s.ids = ((ids * 7919 + 13) % nodes).to(_DTYPE[case["ids"]])
        if kind == "lookup":
            s.table, s.out = normal(nodes, dim, case["table"], 0.02), empty(n, dim, case["out"])
            return s
        s.grad_out = normal(n, dim, case["grad"], 0.01)
        if kind == "grad":
            s.grad_table = empty(nodes, dim, case["table"])
        else:
            s.unique, s.rows = torch.zeros(n, dtype=s.ids.dtype, device="cuda"), empty(n, dim, "f32")
            s.count = torch.zeros(1, dtype=torch.int32, device="cuda")
        s.workspace = {}
        return s
    if kind == "project":
        # rows of different magnitude, and a few that stand out, as activations have them
        a = normal(case["m"], dim, "f32") * torch.exp(torch.randn(case["m"], 1, device="cuda", generator=g))
        s.rows = _encoded(a, case["codec"])
        s.weight_rows = _encoded(normal(case["n"], dim, "f32", 0.02), case["codec"])
        s.out = empty(case["m"], case["n"], case["out"])
        return s
    n = case["m"] if kind == "norm_project" else case["n"]
    s.x = normal(n, dim, case["x"])
    s.weight = (1.0 + 0.1 * torch.randn(dim, device="cuda", generator=g)).to(_DTYPE[case["weight"]])
    s.residual = normal(n, dim, case["x"], 3.0) if case["residual"] else None
    if kind == "norm_grad":
        s.grad_out = normal(n, dim, case["x"], 0.01)
        s.grad_x, s.grad_weight = empty(n, dim, case["x"]), torch.zeros(dim, dtype=torch.float32, device="cuda")
        s.workspace = {}
        return s
    s.residual_out = empty(n, dim, case["x"]) if case["residual"] else None
    if kind == "norm":
        s.out = empty(n, dim, case["x"])
        return s
    s.coded = torch.zeros((n, _slot(dim)), dtype=torch.uint8, device="cuda")
    if kind == "norm_codes":
        s.codes, s.scales = s.coded[:, :dim].view(torch.float8_e4m3fn), s.coded.view(torch.float32)[:, dim // 4]
        return s
    s.weight_rows = _encoded(normal(case["n"], dim, "f32", 0.02), case["codec"])
    s.out = empty(n, case["n"], case["out"])
    return s


# ---- a pass through the framework ----------------------------------------------------------------------------------

def _scratch(s, bytes_):
    """The workspace that a program keeps beside its buffers: made with the first call."""
    if "own" not in s.workspace:
        s.workspace["own"] = torch.empty(max(16, bytes_()), dtype=torch.uint8, device="cuda")
    return s.workspace["own"]


def _run_own(s):
    L, c = _package(), s.case
    kind = c["kind"]
    if kind == "lookup":
        L.embedding_lookup(0, s.table, s.ids, s.out, c["scale"])
        return s.out
    if kind == "grad":
        ws = _scratch(s, lambda: L.embedding_grad_workspace(c["n"], c["dim"], c["nodes"]))
        L.embedding_grad(0, s.ids, s.grad_out, s.grad_table, ws, c["scale"])
        return s.grad_table
    if kind == "grad_rows":
        ws = _scratch(s, lambda: L.embedding_grad_workspace(c["n"], c["dim"], c["nodes"]))
        L.embedding_grad_rows(0, s.ids, s.grad_out, c["nodes"], s.unique, s.rows, s.count, ws, c["scale"])
        return {"ids": s.unique, "rows": s.rows, "count": s.count}
    if kind == "norm_grad":
        ws = _scratch(s, lambda: L.rms_norm_grad_workspace(c["n"], c["dim"]))
        L.rms_norm_grad(0, s.grad_out, s.x, s.weight, s.grad_x, s.grad_weight, ws, _EPS, s.residual)
        return {"x": s.grad_x, "weight": s.grad_weight}
    if kind == "norm":
        L.rms_norm(0, s.x, s.weight, s.out, _EPS, s.residual, s.residual_out)
        return {"out": s.out, "sum": s.residual_out}
    codec = {"int8": L.CODEC_INT8, "e4m3": L.CODEC_E4M3}[c["codec"]]
    if kind == "project":
        L.matmul_rows(0, codec, s.rows, s.weight_rows, c["dim"], s.out)
        return s.out
    L.rms_norm(0, s.x, s.weight, s.coded, _EPS, s.residual, s.residual_out, codec)
    if kind == "norm_codes":
        return {"codes": s.codes, "scales": s.scales, "sum": s.residual_out}
    L.matmul_rows(0, codec, s.coded, s.weight_rows, c["dim"], s.out)
    return {"out": s.out, "sum": s.residual_out}


# ---- a pass in plain form ------------------------------------------------------------------------------------------

def _plain_norm(s):
    """The normed rows in fp32, and the sum with the residual in the type of the rows."""
    h = s.x.float()
    if s.residual is not None:
        h = h + s.residual.float()
    y = h * s.weight.float() * torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
    return y, h.to(s.x.dtype) if s.residual is not None else None


def _plain_codes(y, codec):
    """Codes as the values they stand for up to their row's scale, and the scales."""
    a = y.abs().amax(1, keepdim=True)
    scaled = y * (_TOP[codec] / a)
    return scaled.round() if codec == "int8" else scaled.to(torch.float8_e4m3fn), a / _TOP[codec]


def _plain_values(rows, dim, codec):
    codes = rows[:, :dim].view(torch.int8 if codec == "int8" else torch.float8_e4m3fn).float()
    return codes, rows.view(torch.float32)[:, dim // 4:dim // 4 + 1]


def _run_plain(s):
    c = s.case
    kind, dim = c["kind"], c["dim"]
    if kind == "lookup":
        return (s.table[s.ids].float() * c["scale"]).to(s.out.dtype)
    if kind == "grad":
        whole = torch.zeros((c["nodes"], dim), device="cuda").index_add_(0, s.ids, s.grad_out.float())
        return (whole * c["scale"]).to(s.grad_table.dtype)
    if kind == "grad_rows":
        ids, at = torch.sort(s.ids, stable=True)
        first = torch.ones(ids.numel(), dtype=torch.int32, device="cuda")
        first[1:] = ids[1:] != ids[:-1]
        segment = torch.cumsum(first, 0) - 1
        unique = torch.zeros_like(ids).index_copy_(0, segment, ids)
        rows = torch.zeros((c["n"], dim), device="cuda").index_add_(0, segment, s.grad_out[at].float())
        return {"ids": unique, "rows": rows * c["scale"], "count": (segment[-1:] + 1).to(torch.int32)}
    if kind == "norm_grad":
        h, dy = s.x.float(), s.grad_out.float()
        r = torch.rsqrt((h * h).mean(1, keepdim=True) + _EPS)
        g, normed = dy * s.weight.float(), h * r
        dx = r * (g - normed * (g * normed).mean(1, keepdim=True))
        if s.residual is not None:
            dx = dx + s.residual.float()
        return {"x": dx.to(s.x.dtype), "weight": (dy * normed).sum(0)}
    if kind == "project":
        a, sa = _plain_values(s.rows, dim, c["codec"])
        b, sb = _plain_values(s.weight_rows, dim, c["codec"])
        return ((a @ b.t()) * sa * sb.t()).to(s.out.dtype)
    y, total = _plain_norm(s)
    if kind == "norm":
        return {"out": y.to(s.x.dtype), "sum": total}
    codes, scales = _plain_codes(y, c["codec"])
    if kind == "norm_codes":
        return {"codes": codes, "scales": scales.squeeze(1), "sum": total}
    b, sb = _plain_values(s.weight_rows, dim, c["codec"])
    return {"out": ((codes.float() @ b.t()) * scales * sb.t()).to(s.out.dtype), "sum": total}


def run(state):
    if own:
        return _run_own(state)
    return _run_plain(state)


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind, dim = case["kind"], case["dim"]
    wide = torch.float64
    if kind == "lookup":
        return torch.index_select(s.table, 0, s.ids.long()).to(wide) * case["scale"]
    if kind in ("grad", "grad_rows"):
        where = s.ids.long()
        if kind == "grad_rows":
            found, where = torch.unique(where, sorted=True, return_inverse=True)
        rows = case["nodes"] if kind == "grad" else case["n"]
        total = torch.zeros((rows, dim), dtype=wide, device="cuda")
        total.scatter_add_(0, where[:, None].expand(-1, dim), s.grad_out.to(wide) * case["scale"])
        return total if kind == "grad" else {"ids": None, "rows": total, "count": None}

    def values(rows):
        kept = rows[:, :dim].contiguous().view(torch.int8 if case["codec"] == "int8" else torch.float8_e4m3fn)
        return kept.to(wide) * rows[:, dim:dim + 4].contiguous().view(torch.float32).to(wide)

    if kind == "project":
        return torch.einsum("mk,nk->mn", values(s.rows), values(s.weight_rows))
    x, w = s.x.to(wide), s.weight.to(wide)
    r = s.residual.to(wide) if s.residual is not None else None
    if kind == "norm_grad":
        root = torch.sqrt(x.pow(2).sum(1, keepdim=True) / dim + _EPS)
        dy = s.grad_out.to(wide)
        dot = (dy * w * x).sum(1, keepdim=True)
        dx = dy * w / root - x * dot / (dim * root ** 3)
        return {"x": dx if r is None else dx + r, "weight": torch.einsum("nd,nd->d", dy, x / root)}
    total = x if r is None else x + r
    y = total / torch.sqrt(total.pow(2).sum(1, keepdim=True) / dim + _EPS) * w
    shown = None if r is None else total
    if kind == "norm":
        return {"out": y, "sum": shown}
    scale = y.abs().amax(1, keepdim=True) / _TOP[case["codec"]]
    if kind == "norm_codes":
        return {"codes": y / scale, "scales": scale.squeeze(1), "sum": shown}
    codes = torch.round(y / scale) if case["codec"] == "int8" else (y / scale).to(torch.float8_e4m3fn).to(wide)
    return {"out": torch.einsum("mk,nk->mn", codes * scale, values(s.weight_rows)), "sum": shown}
