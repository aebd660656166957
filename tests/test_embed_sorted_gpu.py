"""cutie_embed_scaled_fwd and cutie_embed_grad_sorted against plain sums in f64: element types, row widths, strides, id
distributions (one id everywhere, all distinct, a document grid), ids outside the table, sizes on both sides of every
boundary of the sort, refusals, streams and graphs.

Tolerances.  The lookup rounds scale * row once to f32 and once to the output type: equal to torch's f32 product rounded.
The gradient adds the n_v rows of an id: a pair passes through at most L = 512 additions in its subgroup, 256 subgroups,
and (chunks of an id) / 8 + 8 joins; with u = 2^-24 the sum is off by at most (512 + 256 + n / 512 + 16) u sum |dout|, and the
product with the scale by one more rounding.  The inputs are exact in their type, so nothing else enters.
"""
import ctypes
import os
import sys

import pytest
import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if REPO not in sys.path:
    sys.path.insert(0, REPO)

from cutie_amd import capi, ops  # noqa: E402

DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def draw_ids(n, V, kind, g):
    if kind == "one":
        return torch.full((n,), V - 1, dtype=torch.int32)
    if kind == "uniform":
        return torch.randint(0, V, (n,), generator=g, dtype=torch.int32)
    if kind == "rising":
        return (torch.arange(n) % V).to(torch.int32)
    if kind == "falling":
        return (V - 1 - torch.arange(n) % V).to(torch.int32)
    ids = (V ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, V - 1)
    ids[torch.rand(n, generator=g) < 0.9] = 0
    if kind == "outside":
        ids[torch.rand(n, generator=g) < 0.2] = -1
        ids[torch.rand(n, generator=g) < 0.1] = V
        ids[torch.rand(n, generator=g) < 0.1] = 2 ** 31 - 1
        ids[torch.rand(n, generator=g) < 0.05] = -2 ** 31
    return ids.to(torch.int32)


def views(n, E, dtype, pad, off, g):
    flat = torch.zeros(n * (E + pad) + off + 8, dtype=dtype)
    flat[off:off + n * (E + pad)] = torch.randn(n * (E + pad), generator=g).to(dtype)
    return flat.to(DEV)[off:off + n * (E + pad)].view(n, E + pad)[:, :E]


def expect(ids, dout, V, scale):
    """(sum, sum of magnitudes) per id, f64"""
    keep = (ids >= 0) & (ids < V)
    i = ids[keep].long()
    d = dout.double()[keep]
    s = torch.zeros(V, dout.shape[1], dtype=torch.float64).index_add_(0, i, d)
    m = torch.zeros(V, dout.shape[1], dtype=torch.float64).index_add_(0, i, d.abs())
    return s * scale, m * abs(scale)


def check_grad(ids, dout, V, scale, got, base=None):
    n = ids.numel()
    s, m = expect(ids.cpu(), dout.cpu(), V, scale)
    tol = (512 + 256 + n / 512 + 17) * U * m
    if base is not None:
        s = s + base.double().cpu()
        tol = tol + 2 * U * s.abs()
    err = (got.cpu().double() - s).abs()
    assert bool((err <= tol).all()), "worst %.3g of its tolerance" % float((err / (tol + 1e-300)).max())


CASES = [
    # n, V, E, pad, off, kind
    (1, 1, 1, 0, 0, "one"), (1, 7, 4, 0, 0, "one"), (2, 3, 5, 1, 0, "uniform"),
    (63, 2, 8, 0, 0, "uniform"), (64, 1, 8, 0, 0, "one"), (65, 70000, 8, 0, 0, "uniform"),
    (513, 300, 128, 64, 0, "grid"), (4096, 11200, 99, 1, 0, "grid"), (4096, 11200, 128, 0, 1, "outside"),
    (8191, 1023, 12, 0, 0, "falling"), (8192, 1024, 12, 4, 0, "outside"), (8193, 1025, 12, 0, 0, "rising"),
    (8192, 5, 256, 0, 0, "one"), (10000, 5, 256, 0, 0, "one"),
    (20481, 511, 64, 0, 0, "uniform"), (20481, 18000, 64, 0, 0, "outside"), (20480, 18000, 4, 0, 0, "rising"),
    (65536, 3000, 40, 0, 0, "grid"), (65537, 1 << 20, 16, 0, 0, "uniform"), (65537, (1 << 20) + 1, 8, 0, 0, "uniform"),
    (131072, 18000, 128, 64, 0, "grid"), (262145, 18000, 24, 0, 0, "one"),
    (3000, 50, 2048, 0, 0, "grid"), (3000, 50, 2052, 0, 0, "grid"), (700, 50, 1031, 2, 0, "grid"),
    (30000, 50, 1, 0, 0, "uniform"), (30000, 2, 2, 0, 0, "grid"), (12288, 40, 8, 0, 0, "falling"), (12289, 1000, 8, 0, 0, "outside"),
    (524288, 3000, 4, 0, 0, "rising"), (524289, 3000, 4, 0, 0, "grid"), (700001, 70000, 4, 0, 0, "outside"),      # many tiles
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,E,pad,off,kind", CASES)
def test_gradient(n, V, E, pad, off, kind, dtype):
    g = torch.Generator().manual_seed(n + V + E)
    ids = draw_ids(n, V, kind, g).to(DEV)
    dout = views(n, E, dtype, pad, off, g)
    got = torch.full((V, E), 7.0, device=DEV)
    ops.embed_grad_sorted(ids, dout, got, scale=1.5)
    check_grad(ids, dout, V, 1.5, got)
    again = torch.full((V, E), 5.0, device=DEV)
    ops.embed_grad_sorted(ids, dout, again, scale=1.5)
    assert torch.equal(again, got)
    base = torch.randn(V, E, generator=g).to(DEV)
    acc = base.clone()
    ops.embed_grad_sorted(ids, dout, acc, scale=-0.5, accumulate=True)
    check_grad(ids, dout, V, -0.5, acc, base)
    absent = torch.ones(V, dtype=torch.bool)
    ok = (ids.cpu() >= 0) & (ids.cpu() < V)
    absent[ids.cpu()[ok].long()] = False
    assert torch.equal(acc.cpu()[absent], base.cpu()[absent])
    assert bool((got.cpu()[absent] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,V,E,pad,off,kind", CASES)
def test_lookup(n, V, E, pad, off, kind, dtype):
    g = torch.Generator().manual_seed(n + V + E)
    ids = draw_ids(n, V, kind, g)
    table = torch.randn(V, E, generator=g)
    flat = torch.full((n * (E + pad) + off,), 3.0, dtype=dtype, device=DEV)
    wide = flat[off:].view(n, E + pad)
    oob = torch.zeros(1, dtype=torch.int32, device=DEV)
    scale = float(E) ** 0.5
    ops.embed_scaled_fwd(ids.to(DEV), table.to(DEV), wide[:, :E], scale, oob)
    ok = (ids >= 0) & (ids < V)
    want = torch.zeros(n, E)
    want[ok] = table[ids[ok].long()] * torch.tensor(scale, dtype=torch.float32)
    assert torch.equal(wide[:, :E].cpu(), want.to(dtype))
    assert bool((wide[:, E:] == 3).all()) and int(oob) == int((~ok).sum())


@pytest.mark.gpu
def test_gradient_is_the_lookup_transposed():
    """sum(lookup(t) * d) == sum(t * gradient(d)) for every t: the gradient of a linear map, checked at random directions and
    against differences of the lookup (which are exact up to rounding)"""
    g = torch.Generator().manual_seed(4)
    n, V, E, scale = 3000, 400, 48, 2.5
    ids = draw_ids(n, V, "grid", g).to(DEV)
    d = torch.randn(n, E, generator=g).to(DEV)
    grad = torch.empty(V, E, device=DEV)
    ops.embed_grad_sorted(ids, d, grad, scale=scale)
    oob = torch.zeros(1, dtype=torch.int32, device=DEV)
    t = torch.randn(V, E, generator=g).to(DEV)

    def value(table):
        out = torch.empty(n, E, device=DEV)
        ops.embed_scaled_fwd(ids, table, out, scale, oob)
        return float((out.double() * d.double()).sum())
    h = 0.5
    got = float((grad.double() * t.double()).sum())
    zero = torch.zeros_like(t)
    want = (value(zero + h * t) - value(zero - h * t)) / (2 * h)
    mag = float((t.double().abs()[ids.long()] * d.double().abs()).sum()) * scale
    assert abs(got - want) <= (512 + 256 + 30) * U * mag


@pytest.mark.gpu
@pytest.mark.parametrize("n", [0, 5])
def test_no_cells_and_no_valid_cells(n):
    ids = torch.full((n,), -3, dtype=torch.int32, device=DEV)
    d = torch.ones((n, 6), device=DEV)
    out = torch.full((9, 6), 4.0, device=DEV)
    ops.embed_grad_sorted(ids, d, out, accumulate=True)
    assert bool((out == 4).all())
    ops.embed_grad_sorted(ids, d, out)
    assert bool((out == 0).all())


@pytest.mark.gpu
def test_non_finite_rows_stay_with_their_id():
    ids = torch.tensor([2, 1, 2, 0, 1, -1], dtype=torch.int32, device=DEV)
    d = torch.ones(6, 8, device=DEV)
    d[2, 3], d[5] = float("inf"), float("nan")       # the last row belongs to no id
    out = torch.empty(4, 8, device=DEV)
    ops.embed_grad_sorted(ids, d, out)
    want = torch.tensor([1.0, 2.0, 2.0, 0.0]).view(4, 1).repeat(1, 8)
    want[2, 3] = float("inf")
    assert torch.equal(out.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3000, 30000])
def test_side_stream_and_graph(n):
    g = torch.Generator().manual_seed(9)
    V, E = 777, 64
    ids = draw_ids(n, V, "grid", g).to(DEV)
    other = draw_ids(n, V, "uniform", g).to(DEV)
    d = torch.randn(n, E, generator=g).half().to(DEV)
    out = torch.empty(V, E, device=DEV)
    ws = torch.empty(ops.embed_grad_sorted_workspace_bytes(n, V, E), dtype=torch.uint8, device=DEV)
    ops.embed_grad_sorted(ids, d, out, workspace=ws)
    want = out.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out.zero_()
        ops.embed_grad_sorted(ids, d, out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.embed_grad_sorted(ids, d, out, workspace=ws)
    for r in range(4):
        ids.copy_(other if r % 2 == 0 else torch.flip(other, (0,)))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        eager = torch.empty_like(out)
        ops.embed_grad_sorted(ids, d, eager)
        assert torch.equal(got, eager), r


# ------------------------------------------------------------------------------------------------------------------ refusals
P = ctypes.c_void_p


@pytest.mark.parametrize("kw,word", [
    (dict(V=0), b"V=0"), (dict(E=0), b"E=0"), (dict(E=65537), b"E=65537"), (dict(n=-1), b"n_cells=-1"), (dict(n=(1 << 30) + 1), b"n_cells"),
    (dict(V=1 << 30), b"V="), (dict(ld=7), b"leading dimension"), (dict(dt=3), b"dtype"), (dict(ids=None), b"null"),
    (dict(rows=P(4097)), b"misaligned"), (dict(table=None), b"null")])
def test_refusals(kw, word):
    a = dict(ids=P(4096), n=4, table=P(8192), V=3, E=8, rows=P(4096), ld=8, dt=0)
    a.update(kw)
    lib = capi.lib()
    rc = lib.cutie_embed_scaled_fwd(a["ids"], a["n"], a["table"], a["V"], a["E"], 1.0, a["rows"], a["ld"], a["dt"], P(4096), None)
    assert rc == -1 and word in lib.cutie_last_error()
    rc = lib.cutie_embed_grad_sorted(a["ids"], a["n"], a["rows"], a["ld"], a["dt"], 1.0, a["table"], a["V"], a["E"], 0, P(4096), 1 << 40, None)
    assert rc == -1 and word in lib.cutie_last_error()


def test_workspace_refusals():
    lib = capi.lib()
    need = lib.cutie_embed_grad_sorted_workspace_bytes(10000, 300, 16)
    assert need > 10000 * 16
    for ws, n in ((None, need), (P(4096), need - 1), (P(4097), need)):
        assert lib.cutie_embed_grad_sorted(P(4096), 10000, P(4096), 16, 0, 1.0, P(4096), 300, 16, 0, ws, n, None) == -3
        assert b"workspace" in lib.cutie_last_error()
    assert lib.cutie_embed_grad_sorted_workspace_bytes(0, 3, 4) == 0 and lib.cutie_embed_grad_sorted_workspace_bytes(4, 0, 4) == 0


def test_wrapper_refusals():
    ids, t = torch.zeros(4, dtype=torch.int32), torch.zeros(3, 8)
    oob = torch.zeros(1, dtype=torch.int32)
    for bad in (lambda: ops.embed_scaled_fwd(ids.long(), t, torch.zeros(4, 8), 1.0, oob),
                lambda: ops.embed_scaled_fwd(ids, t.half(), torch.zeros(4, 8), 1.0, oob),
                lambda: ops.embed_scaled_fwd(ids, t, torch.zeros(4, 9), 1.0, oob),
                lambda: ops.embed_scaled_fwd(ids, t, torch.zeros(5, 8), 1.0, oob),
                lambda: ops.embed_scaled_fwd(ids, t, torch.zeros(4, 8), 1.0, oob.long()),
                lambda: ops.embed_grad_sorted(ids[::2], torch.zeros(2, 8), t),
                lambda: ops.embed_grad_sorted(ids, torch.zeros(4, 8), t)):      # the last one: not device tensors
        with pytest.raises(capi.CutieError):
            bad()
