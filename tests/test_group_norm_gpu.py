"""cutie_gn_fwd / cutie_gn_bwd against the definition in f64, over element types, group widths, strides and the two forms of
the kernels (a group held by one workgroup; sums over slices), their refusals, and the streams and graphs they run under.

Tolerances.  u = 2^-24 is half a step of f32, t half a step of the stored type (f32 2^-24, bf16 2^-8, f16 2^-11).  The
longest chain of f32 additions behind one sum: 16 vectors of 8 in a thread, 16 terms a lane, 6 in a wave, at most 256 slots
and 32 x ceil(B / 32) samples: below 512.  So a sum is off by at most 512 u times the sum of its terms' magnitudes, and a
value made from such sums by 512 u of the magnitudes it is made from, plus t of itself for the store.  The 16-bit types take
the hardware exponential and reciprocal: 2^-20 more of what the activation multiplies.
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
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def act64(z, act):
    s = torch.sigmoid(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).double()
    if act == "sigmoid":
        return s, s * (1 - s)
    if act == "silu":
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def gn64(x, groups, gamma, beta, act, eps=1e-5):
    """(y, mean, rstd, xhat, z) in f64 on the CPU"""
    B, H, W, C = x.shape
    xg = x.double().reshape(B, H * W, groups, C // groups)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(((xg - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
    xhat = ((xg - mean) * rstd).reshape(B, H, W, C)
    z = xhat * (gamma.double() if gamma is not None else 1.0) + (beta.double() if beta is not None else 0.0)
    return act64(z, act)[0], mean.reshape(B, groups), rstd.reshape(B, groups), xhat, z


def gn_bwd64(dy, x, stats, gamma, beta, act):
    """(dx, dgamma, dbeta) and the magnitudes behind each, from the formula and the stored statistics"""
    B, H, W, C = x.shape
    G = stats.shape[1]
    Cg = C // G
    ga = gamma.double() if gamma is not None else torch.ones(C, dtype=torch.float64)
    be = beta.double() if beta is not None else torch.zeros(C, dtype=torch.float64)
    mean, rstd = (stats.double()[..., k].reshape(B, 1, G, 1) for k in (0, 1))
    xh = ((x.double().reshape(B, H * W, G, Cg) - mean) * rstd).reshape(B, H, W, C)
    g = dy.double() * act64(xh * ga + be, act)[1]
    dgamma, dbeta = (g * xh).sum((0, 1, 2)), g.sum((0, 1, 2))
    h = (g * ga).reshape(B, H * W, G, Cg)
    xg = xh.reshape(B, H * W, G, Cg)
    m0, m1 = h.mean((1, 3), keepdim=True), (h * xg).mean((1, 3), keepdim=True)
    dx = (rstd * (h - m0 - xg * m1)).reshape(B, H, W, C)
    # with a smooth activation h itself is off by rounding of z: |dy gamma| (|xh gamma| + |beta| + 1) roundings of it
    soft = (dy.double().abs() * ga.abs() * ((xh * ga).abs() + be.abs() + 1)).reshape(B, H * W, G, Cg)
    mag = rstd * (soft + soft.mean((1, 3), keepdim=True) + xg.abs() * (soft * xg.abs()).mean((1, 3), keepdim=True))
    sg = soft.reshape(B, H, W, C) / ga.abs().clamp_min(1e-30)
    return dx, dgamma, dbeta, mag.reshape(B, H, W, C), (sg * (xh.abs() + 1e-3)).sum((0, 1, 2)), sg.sum((0, 1, 2))


def make(B, H, W, C, groups, dtype, pad=0, off=0, affine=True, seed=0, level=1.0):
    g = torch.Generator().manual_seed(seed)
    # `off` elements in front shift the base off its 16-byte boundary
    flat = torch.zeros(B * H * W * (C + pad) + off + 8, dtype=dtype)
    n = B * H * W * (C + pad)
    vals = torch.randn(n, generator=g).reshape(B, H, W, C + pad) * (0.5 + torch.rand(C + pad, generator=g))
    vals += level * torch.randn(C + pad, generator=g)
    flat[off:off + n] = vals.reshape(-1).to(dtype)
    x = flat.to(DEV)[off:off + n].view(B, H, W, C + pad)[..., :C]
    dy = (torch.randn(B, H, W, C, generator=g) * 0.1).to(dtype).to(DEV)
    gamma = (1 + 0.3 * torch.randn(C, generator=g)).to(DEV) if affine else None
    beta = (0.3 * torch.randn(C, generator=g)).to(DEV) if affine else None
    return x, dy, gamma, beta


def run_fwd(x, groups, gamma, beta, act):
    y = torch.full_like(x, 7.0, memory_format=torch.contiguous_format)
    stats = torch.full((x.shape[0], groups, 2), 7.0, device=DEV)
    ops.gn_fwd(x, y, stats, gamma=gamma, beta=beta, act=act)
    return y, stats


def cpu(t):
    return None if t is None else t.detach().cpu()


def check_fwd(x, groups, gamma, beta, act, y, stats):
    ref, mean, rstd, xh, z = gn64(cpu(x), groups, cpu(gamma), cpu(beta), act)
    B, H, W, C = x.shape
    xa = cpu(x).double().abs().reshape(B, H * W, groups, C // groups).mean((1, 3))
    t = HALF[x.dtype]
    got = cpu(stats).double()
    assert bool(((got[..., 0] - mean).abs() <= 2 * U * (xa + mean.abs())).all()) or \
        float(((got[..., 0] - mean).abs() / (xa + 1e-30)).max()) <= 512 * U
    assert float(((got[..., 1] - rstd).abs() / rstd).max()) <= 512 * U
    soft = (z - (cpu(beta).double() if beta is not None else 0)).abs() + (cpu(beta).double().abs() if beta is not None else 0) + 1
    tol = t * ref.abs() * (1 + t) + 512 * U * soft
    if x.dtype != torch.float32:
        tol = tol + 2.0 ** -20 * soft + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)     # half a step below f16's normals
    err = (cpu(y).double() - ref).abs()
    assert bool((err <= tol).all()), "worst %.3g of its tolerance" % float((err / tol).max())


def check_bwd(dy, x, stats, gamma, beta, act, dx, dgamma, dbeta):
    ref, rg, rb, mag, mg, mb = gn_bwd64(cpu(dy), cpu(x), cpu(stats), cpu(gamma), cpu(beta), act)
    t = HALF[x.dtype]
    soft = 512 * U + (2.0 ** -20 if x.dtype != torch.float32 else 0.0)
    tol = t * ref.abs() * (1 + t) + soft * mag + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    err = (cpu(dx).double() - ref).abs()
    assert bool((err <= tol).all()), "dx: worst %.3g of its tolerance" % float((err / tol).max())
    for name, got, want, m in (("dgamma", dgamma, rg, mg), ("dbeta", dbeta, rb, mb)):
        e = (cpu(got).double() - want).abs()
        assert bool((e <= soft * m + 1e-30).all()), "%s: worst %.3g of its tolerance" % (name, float((e / (soft * m + 1e-30)).max()))


SHAPES = [
    # B, H, W, C, groups, pad, off
    (2, 8, 8, 64, 8, 0, 0),          # 8 channels a group
    (1, 64, 64, 256, 32, 64, 0),     # a document, channel slice of a wider buffer
    (2, 40, 40, 256, 4, 0, 0),       # 64 channels a group
    (1, 1, 1, 8, 1, 0, 0),           # one pixel
    (3, 1, 1, 5, 5, 0, 0),           # one value a group
    (1, 1, 2, 3, 1, 1, 0),
    (2, 37, 53, 66, 6, 2, 0),        # eleven channels a group
    (2, 9, 7, 24, 2, 0, 0),          # twelve: 8-byte vectors of a 16-bit type, 16-byte of f32
    (2, 9, 7, 64, 8, 0, 1),          # base off its 16-byte boundary
    (2, 9, 7, 64, 8, 1, 0),          # odd leading dimension
    (1, 130, 130, 32, 2, 0, 0),      # a group too large for a workgroup
    (1, 130, 131, 33, 3, 0, 0),      # the same with single elements
    (1, 100, 90, 512, 1, 0, 0),      # one group of every channel
    (1, 3, 5, 4096, 2, 0, 0),        # many channels, few pixels
    (1, 3, 5, 1300, 1, 1, 0),        # more than 1024 single elements a pixel
    (70, 4, 4, 16, 2, 0, 0),         # many samples
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,W,C,groups,pad,off", SHAPES)
def test_forward_and_backward(B, H, W, C, groups, pad, off, dtype):
    for i, act in enumerate(("none", "relu", "sigmoid", "silu")):
        x, dy, gamma, beta = make(B, H, W, C, groups, dtype, pad, off, affine=i != 0, seed=i)
        y, stats = run_fwd(x, groups, gamma, beta, act)
        check_fwd(x, groups, gamma, beta, act, y, stats)
        dx = torch.full_like(dy, 7.0)
        dgamma, dbeta = torch.full((C,), 7.0, device=DEV), torch.full((C,), 7.0, device=DEV)
        ops.gn_bwd(dy, x, stats, dx, gamma=gamma, beta=beta, act=act, dgamma=dgamma, dbeta=dbeta)
        check_bwd(dy, x, stats, gamma, beta, act, dx, dgamma, dbeta)
        # same bits again, added to, and without the parameters' gradients
        dx2 = torch.full_like(dy, 7.0)
        dg2, db2 = dgamma.clone(), dbeta.clone()
        ops.gn_bwd(dy, x, stats, dx2, gamma=gamma, beta=beta, act=act, dgamma=dg2, dbeta=db2, accumulate=True)
        assert torch.equal(dx2, dx) and torch.equal(dg2, dgamma + dgamma) and torch.equal(db2, dbeta + dbeta)
        dx3 = torch.full_like(dy, 7.0)
        ops.gn_bwd(dy, x, stats, dx3, gamma=gamma, beta=beta, act=act)
        assert torch.equal(dx3, dx)
        db3 = torch.full((C,), 7.0, device=DEV)
        ops.gn_bwd(dy, x, stats, dx3, gamma=gamma, beta=beta, act=act, dbeta=db3)
        assert torch.equal(db3, dbeta)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,W,C,groups,pad,off", [
    (2, 128, 128, 16, 2, 0, 0),      # few groups of many pixels, which would fit: in slices all the same
    (3, 64, 65, 66, 33, 1, 1),       # two channels a group
    (24, 64, 64, 66, 33, 0, 0),      # and many of them
    (1, 130, 130, 36, 2, 3, 1),      # slices of vectors that begin anywhere, groups that end inside a vector
    (1, 61, 67, 1032, 4, 1, 0),      # wide rows: eight values a vector, more than one block of columns for f32
    (2, 90, 91, 20, 1, 2, 1),
])
def test_forms_and_alignments(B, H, W, C, groups, pad, off, dtype):
    x, dy, gamma, beta = make(B, H, W, C, groups, dtype, pad, off, seed=B + C)
    y, stats = run_fwd(x, groups, gamma, beta, "silu")
    check_fwd(x, groups, gamma, beta, "silu", y, stats)
    wide = torch.full((B, H, W, C + pad + 1), 3.0, dtype=dtype, device=DEV)      # dx beside columns that stay
    dgamma, dbeta = torch.full((C,), 7.0, device=DEV), torch.full((C,), 7.0, device=DEV)
    ops.gn_bwd(dy, x, stats, wide[..., 1:C + 1], gamma=gamma, beta=beta, act="silu", dgamma=dgamma, dbeta=dbeta)
    check_bwd(dy, x, stats, gamma, beta, "silu", wide[..., 1:C + 1], dgamma, dbeta)
    assert bool((wide[..., 0] == 3).all()) and bool((wide[..., C + 1:] == 3).all())
    again = torch.empty_like(dy)
    dg2, db2 = torch.empty_like(dgamma), torch.empty_like(dbeta)
    ops.gn_bwd(dy, x, stats, again, gamma=gamma, beta=beta, act="silu", dgamma=dg2, dbeta=db2)
    assert torch.equal(again, wide[..., 1:C + 1]) and torch.equal(dg2, dgamma) and torch.equal(db2, dbeta)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 16, 16, 32, 4), (1, 130, 130, 32, 2)])
def test_level_far_above_spread(shape):
    """mean = 4096 sigma: the second moment is taken about the mean (or in f64), so 1/sigma keeps its digits"""
    B, H, W, C, G = shape
    g = torch.Generator().manual_seed(3)
    x = (4096.0 + torch.randn(B, H, W, C, generator=g)).to(DEV)
    x[:, 0, 0] = 0.0          # and a first pixel that lies far off
    y, stats = run_fwd(x, G, None, None, "none")
    ref, mean, rstd, xh, _ = gn64(cpu(x), G, None, None, "none")
    assert float(((cpu(stats)[..., 1].double() - rstd).abs() / rstd).max()) <= 512 * U
    # x - mean is exact to a rounding of the mean's own residue: 2^-24 of the spread, not of the level
    assert float((cpu(y).double() - ref).abs().max()) <= 512 * U * float(ref.abs().max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2, 8, 8, 32, 4), (2, 130, 130, 32, 2)])
def test_nan_and_infinity_stay_in_their_group(shape, dtype):
    B, H, W, C, G = shape
    x, dy, gamma, beta = make(B, H, W, C, G, dtype, seed=5)
    clean, cs = run_fwd(x, G, gamma, beta, "relu")
    for bad in (float("nan"), float("inf"), float("-inf")):
        xb = x.clone()
        xb[1, 3, 3, 1] = bad
        y, stats = run_fwd(xb, G, gamma, beta, "relu")
        assert torch.isnan(y[1, ..., :C // G]).all()
        assert torch.equal(y[0], clean[0]) and torch.equal(y[1, ..., C // G:], clean[1, ..., C // G:])
        dx = torch.empty_like(dy)
        ops.gn_bwd(dy, xb, stats, dx, gamma=gamma, beta=beta, act="relu")
        assert torch.isnan(dx[1, ..., :C // G]).all() and torch.isfinite(dx[0].float()).all()
        assert torch.isfinite(dx[1, ..., C // G:].float()).all()


@pytest.mark.gpu
def test_output_is_written_and_nothing_else():
    """columns of a wider buffer beside the view stay as they were"""
    x, dy, gamma, beta = make(2, 5, 7, 24, 3, torch.float16, seed=7)
    wide = torch.full((2, 5, 7, 40), 3.0, dtype=torch.float16, device=DEV)
    stats = torch.empty((2, 3, 2), device=DEV)
    ops.gn_fwd(x, wide[..., 8:32], stats, gamma=gamma, beta=beta, act="silu")
    check_fwd(x, 3, gamma, beta, "silu", wide[..., 8:32], stats)
    assert bool((wide[..., :8] == 3).all()) and bool((wide[..., 32:] == 3).all())
    dw = torch.full((2, 5, 7, 40), 3.0, dtype=torch.float16, device=DEV)
    ops.gn_bwd(dy, x, stats, dw[..., 8:32], gamma=gamma, beta=beta, act="silu")
    assert bool((dw[..., :8] == 3).all()) and bool((dw[..., 32:] == 3).all())


@pytest.mark.gpu
def test_empty_batch():
    stats = torch.empty((0, 2, 2), device=DEV)
    x = torch.empty((0, 4, 4, 8), device=DEV)
    ops.gn_fwd(x, torch.empty_like(x), stats)
    dg, db = torch.ones(8, device=DEV), torch.ones(8, device=DEV)
    ops.gn_bwd(x, x, stats, torch.empty_like(x), dgamma=dg, dbeta=db, accumulate=True)
    assert bool((dg == 1).all())
    ops.gn_bwd(x, x, stats, torch.empty_like(x), dgamma=dg, dbeta=db)
    assert bool((dg == 0).all()) and bool((db == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 6, 6, 16, 4), (1, 130, 130, 16, 1)])
def test_gradient_against_differences(shape):
    """L = sum w y of the kernel's own forward, central differences of steps h and h / 2 combined (error of order h^4 per unit
    step).  The forward is off by at most 512 u (|z| + 1) an element in the worst case; its roundings are independent, so the
    quotient is off by about their root-sum-square over h."""
    B, H, W, C, G = shape
    x, dy, gamma, beta = make(B, H, W, C, G, torch.float32, seed=11)
    w = torch.randn(x.shape, generator=torch.Generator().manual_seed(12)).to(DEV)
    _, stats = run_fwd(x, G, gamma, beta, "silu")
    dx, dg, db = torch.empty_like(w), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.gn_bwd(w, x, stats, dx, gamma=gamma, beta=beta, act="silu", dgamma=dg, dbeta=db)

    def loss(xx, ga, be):
        return float((run_fwd(xx, G, ga, be, "silu")[0].double() * w.double()).sum())

    g = torch.Generator().manual_seed(13)
    h = 2.0 ** -5
    noise = 4 * 16 * U * float((w.double() ** 2).sum().sqrt()) * 4 / h
    for name in ("x", "gamma", "beta"):
        v = torch.randn(x.shape if name == "x" else (C,), generator=g).to(DEV)
        grad = {"x": dx, "gamma": dg, "beta": db}[name]

        def at(t):
            return loss(x + t * v if name == "x" else x, gamma + t * v if name == "gamma" else gamma,
                        beta + t * v if name == "beta" else beta)
        c1 = (at(h) - at(-h)) / (2 * h)
        c2 = (at(h / 2) - at(-h / 2)) / h
        want = (4 * c2 - c1) / 3
        got = float((grad.double() * v.double()).sum())
        scale = float((grad.double() ** 2).sum().sqrt()) * float((v.double() ** 2).sum().sqrt())
        assert abs(got - want) <= noise + abs(c2 - c1) / 3 + 1e-5 * scale, (name, got, want, noise)


def test_formula_against_autograd():
    """the f64 gradient the kernels are held to is the gradient of the f64 forward"""
    for act in ("none", "relu", "sigmoid", "silu"):
        g = torch.Generator().manual_seed(2)
        x = torch.randn(2, 3, 4, 12, generator=g, dtype=torch.float64, requires_grad=True)
        gamma = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
        beta = torch.randn(12, generator=g, dtype=torch.float64, requires_grad=True)
        dy = torch.randn(2, 3, 4, 12, generator=g, dtype=torch.float64)
        y, mean, rstd, _, _ = gn64(x, 3, gamma, beta, act)
        want = torch.autograd.grad((y * dy).sum(), (x, gamma, beta))
        stats = torch.stack([mean, rstd], -1).detach()
        got = gn_bwd64(dy, x.detach(), stats, gamma.detach(), beta.detach(), act)[:3]
        for a, b in zip(got, want):
            assert float((a - b).abs().max()) <= 1e-10


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(2, 16, 16, 64, 8), (1, 130, 130, 32, 2)])
def test_side_stream_and_graph(shape):
    B, H, W, C, G = shape
    x, dy, gamma, beta = make(B, H, W, C, G, torch.float16, seed=21)
    y0, s0 = run_fwd(x, G, gamma, beta, "silu")
    y, stats, dx = torch.empty_like(y0), torch.empty_like(s0), torch.empty_like(dy)
    dg, db = torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ws = torch.empty(ops.gn_workspace_bytes(B, H * W, C, G), dtype=torch.uint8, device=DEV)

    def step():
        ops.gn_fwd(x, y, stats, gamma=gamma, beta=beta, act="silu", workspace=ws)
        ops.gn_bwd(dy, x, stats, dx, gamma=gamma, beta=beta, act="silu", dgamma=dg, dbeta=db, workspace=ws)
    step()
    torch.cuda.synchronize()
    want = [t.clone() for t in (y, stats, dx, dg, db)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for t in (y, stats, dx, dg, db):
            t.zero_()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip((y, stats, dx, dg, db), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for r in range(4):
        x.mul_(0.75)
        for t in (y, stats, dx, dg, db):
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, stats, dx, dg, db)]
        step()
        assert all(torch.equal(a, b) for a, b in zip((y, stats, dx, dg, db), got)), r


# ------------------------------------------------------------------------------------------------------------------ refusals
FAKE = ctypes.c_void_p(4096)


def fwd_rc(**kw):
    a = dict(x=FAKE, ld_x=8, groups=2, eps=1e-5, act=0, y=ctypes.c_void_p(8192), ld_y=8, dt=0, stats=FAKE, B=1, HW=4, C=8, ws=None, n=0)
    a.update(kw)
    return capi.lib().cutie_gn_fwd(a["x"], a["ld_x"], None, None, a["groups"], a["eps"], a["act"], a["y"], a["ld_y"], a["dt"], a["stats"],
                                   a["B"], a["HW"], a["C"], a["ws"], a["n"], None)


def bwd_rc(**kw):
    a = dict(dy=FAKE, ld=8, x=ctypes.c_void_p(8192), groups=2, act=0, stats=FAKE, dx=ctypes.c_void_p(12288), dt=0, B=1, HW=4, C=8,
             ws=ctypes.c_void_p(16384), n=1 << 30)
    a.update(kw)
    return capi.lib().cutie_gn_bwd(a["dy"], a["ld"], a["x"], a["ld"], None, None, a["groups"], a["act"], a["stats"], a["dx"], a["ld"],
                                   a["dt"], None, None, 0, a["B"], a["HW"], a["C"], a["ws"], a["n"], None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(groups=3), -1, b"groups"), (dict(groups=0), -1, b"groups"), (dict(C=0), -1, b"C=0"), (dict(B=-1), -1, b"B=-1"),
    (dict(B=70000), -1, b"65535"), (dict(act=4), -1, b"activation"), (dict(dt=3), -1, b"dtype"), (dict(ld_x=7), -1, b"ld_x"),
    (dict(ld_y=7), -1, b"ld_y"), (dict(eps=0.0), -1, b"eps"), (dict(x=None), -1, b"null"), (dict(stats=None), -1, b"null"),
    (dict(y=FAKE), -1, b"y must not be x"), (dict(x=ctypes.c_void_p(4097)), -1, b"misaligned"),
    (dict(HW=1 << 20, ws=None), -3, b"workspace"), (dict(HW=1 << 20, ws=FAKE, n=16), -3, b"workspace")])
def test_forward_refusals(kw, rc, word):
    assert fwd_rc(**kw) == rc and word in capi.lib().cutie_last_error()


@pytest.mark.parametrize("kw,rc,word", [
    (dict(groups=3), -1, b"groups"), (dict(act=-1), -1, b"activation"), (dict(dt=9), -1, b"dtype"), (dict(ld=7), -1, b"ld_dy"),
    (dict(dy=None), -1, b"null"), (dict(dx=FAKE), -1, b"dx must be"), (dict(stats=None), -1, b"null"),
    (dict(ws=None), -3, b"workspace"), (dict(n=64), -3, b"workspace"), (dict(ws=ctypes.c_void_p(16385)), -3, b"workspace")])
def test_backward_refusals(kw, rc, word):
    assert bwd_rc(**kw) == rc and word in capi.lib().cutie_last_error()


def test_wrapper_refusals():
    x = torch.zeros(1, 2, 2, 8)
    st = torch.zeros(1, 2, 2)
    for bad in (lambda: ops.gn_fwd(x, x.clone(), torch.zeros(1, 2)), lambda: ops.gn_fwd(x, x.clone(), st, act="tanh"),
                lambda: ops.gn_fwd(x, x.half(), st), lambda: ops.gn_fwd(x, torch.zeros(1, 2, 2, 4), st),
                lambda: ops.gn_fwd(x, x.clone(), st.double()), lambda: ops.gn_fwd(x, x.clone(), st, gamma=torch.zeros(7)),
                lambda: ops.gn_fwd(x, x.clone(), st)):          # the last one: not a device tensor
        with pytest.raises(capi.CutieError):
            bad()


def test_workspace_size():
    n = capi.lib().cutie_gn_workspace_bytes
    assert n(1, 4, 8, 3) == 0 and n(0, 4, 8, 2) == 0
    assert n(32, 4096, 256, 32) >= 32 * 256 * 8


@pytest.mark.parametrize("y,ld_x,ld_y", [(4096 + 4, 64, 64), (4096 + 28, 64, 64), (4096 + 64 * 4 - 28, 64, 64), (4096 + 3 * 64 * 4, 64, 64),
                                         (4096 - 64 * 4 + 4, 64, 64), (4096 + 32, 64, 128)])
@pytest.mark.parametrize("HW", [4, 1 << 20])
def test_overlapping_views_are_refused(y, ld_x, ld_y, HW):
    """rows of 8 f32 channels: refused on the host, nothing is launched"""
    v = ctypes.c_void_p
    ws, n = v(1 << 40), 1 << 40
    assert fwd_rc(y=v(y), ld_x=ld_x, ld_y=ld_y, HW=HW, ws=ws, n=n) == -1 and b"overlaps" in capi.lib().cutie_last_error()
    for dy, x in ((4096, 1 << 36), (1 << 36, 4096)):
        rc = capi.lib().cutie_gn_bwd(v(dy), ld_x, v(x), ld_x, None, None, 2, 0, v(1 << 41), v(y), ld_y, 0, None, None, 0, 1, HW, 8, ws, n, None)
        assert rc == -1 and b"overlaps" in capi.lib().cutie_last_error()


def test_sizes_beyond_the_c_abi_are_refused():
    for shape in ((1, 1 << 16, 1 << 16, 1), (65536, 1, 1, 1), (1, 1, 1, 65536)):
        x = torch.empty(shape, device="meta")
        with pytest.raises(capi.CutieError, match="at most"):
            ops.gn_fwd(x, x, torch.empty(shape[0], 1, 2, device="meta"))
    x = torch.empty_strided((1, 1, 2, 1), (1 << 33, 1 << 33, 1 << 32, 1), device="meta")
    with pytest.raises(capi.CutieError, match="leading dimension"):
        capi.ld_of(x)
    with pytest.raises(capi.CutieError, match="below 2"):
        ops._check_ids("embed_grad_sorted", torch.empty(3, dtype=torch.int32, device="meta"), torch.empty(3, 1, device="meta"),
                       torch.empty((1 << 32) + 3, 1, device="meta"))


@pytest.mark.gpu
def test_slices_of_one_buffer_are_taken():
    """x, y and the gradients as neighbouring channel slices"""
    g = torch.Generator().manual_seed(4)
    wide = torch.randn(2, 5, 7, 48, generator=g).to(DEV)
    xs = wide[..., 8:16].clone()
    st, st2 = torch.empty(2, 2, 2, device=DEV), torch.empty(2, 2, 2, device=DEV)
    want = torch.empty(2, 5, 7, 8, device=DEV)
    ops.gn_fwd(xs, want, st, act="silu")
    ops.gn_fwd(wide[..., 8:16], wide[..., 16:24], st2, act="silu")
    assert torch.equal(wide[..., 16:24], want) and torch.equal(st, st2)
    dy = wide[..., 24:32].clone()
    ops.gn_bwd(dy, xs, st, want, act="silu")
    ops.gn_bwd(wide[..., 24:32], wide[..., 8:16], st, wide[..., 0:8], act="silu")
    assert torch.equal(wide[..., 0:8], want)
    with pytest.raises(capi.CutieError, match="overlaps"):
        ops.gn_fwd(wide[..., 8:16], wide[..., 12:20], st2)
