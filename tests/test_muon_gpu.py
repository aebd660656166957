"""cutie_orthogonalize_batched and cutie_muon_step against the iteration in f64: sizes from 1 x 1 over odd ones to several tiles
and K parts, tall and wide, batches, ranks and magnitudes, skipped steps, refusals, streams and graphs.

Tolerances.  An operand is held in 22 bits: stored X, A and B are each off by up to h = 2^-23 of themselves, and a product,
whose lo*lo part (2^-12 of each factor) is left out, by up to 2^-24 = h / 2 of the sum of its terms' magnitudes.  How much of
that reaches the result depends on the matrix: later steps amplify a rounding by up to 3.4445 each where a singular value is near
0 (2 x 2 with singular values 1 and 1e-3: h * 485 = 6e-5) and hardly at all elsewhere.  So the measure is the iteration in f64
with errors of just those sizes drawn at random, eight times: the kernel may be off by 4 times the largest of the eight.  (The
plain f32 iteration is no measure for small matrices: a 1 x 1 one is a single sequence of roundings, and may happen to be exact.)
The update: p and m are f32 elementwise; u32 = 2^-24: m off by at most 4 u32 of the magnitudes added, p by 4 u32 of its terms plus
lr k times the error of X.
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
NS = (3.4445, -4.7750, 2.0315)
H = 2.0 ** -23      # half a step of 22 bits


def iterate(u, steps=5, eps=1e-7):
    """the definition in u's own type (norm in f64)"""
    a, b, c = NS
    x = u / (torch.sqrt((u.double() ** 2).sum()) + eps).to(u.dtype)
    for _ in range(steps):
        if u.shape[0] <= u.shape[1]:
            m = x @ x.t()
            x = a * x + (b * m + c * (m @ m)) @ x
        else:
            m = x.t() @ x
            x = a * x + x @ (b * m + c * (m @ m))
    return x


def rounded(u, steps, eps, seed):
    """iterate() of an f64 matrix with the errors of the number format drawn at random"""
    g = torch.Generator(device=u.device).manual_seed(seed)

    def off(t, size):
        return t * (1 + size * (2 * torch.rand(t.shape, generator=g, device=t.device, dtype=torch.float64) - 1))

    def product(p, q):
        err = (2 * torch.rand((p.shape[0], q.shape[1]), generator=g, device=p.device, dtype=torch.float64) - 1) * (p.abs() @ q.abs())
        return p @ q + H / 2 * err
    a, b, c = NS
    x = u if u.shape[0] >= u.shape[1] else u.t()
    x = off(x / (u.norm() + eps), H)
    for _ in range(steps):
        m = off(product(x.t(), x), H)
        y = off(b * m + c * product(m, m), H)
        x = off(a * x + product(x, y), H)
    return x if u.shape[0] >= u.shape[1] else x.t()


def allowed(u, steps=5, eps=1e-7):
    """(f64 result, largest error in 2-norm over all values)"""
    u = u.double()
    want = iterate(u, steps, eps)
    return want, 4 * max(float((rounded(u, steps, eps, k) - want).norm()) for k in range(8))


def matrix(r, c, kind, g):
    if kind == "normal":
        return torch.randn(r, c, generator=g)
    if kind == "falling":
        k = min(r, c)
        q1 = torch.linalg.qr(torch.randn(r, k, generator=g, dtype=torch.float64))[0]
        q2 = torch.linalg.qr(torch.randn(c, k, generator=g, dtype=torch.float64))[0]
        return ((q1 * torch.logspace(0, -3, k, dtype=torch.float64)) @ q2.t()).float()
    if kind == "rank1":
        return torch.randn(r, 1, generator=g) @ torch.randn(1, c, generator=g)
    if kind == "one":
        m = torch.zeros(r, c)
        m[r // 2, c // 3] = -3.0
        return m
    raise ValueError(kind)


SIZES = [(1, 1), (1, 7), (9, 1), (2, 2), (18, 64), (64, 18), (63, 65), (64, 64), (65, 129), (128, 128), (300, 129), (256, 1000),
         (1920, 256), (130, 4000), (700, 700),
         (192, 64), (64, 192), (193, 64), (64, 193), (192, 65), (3000, 20), (520, 530), (1, 2500), (2500, 1)]      # both sides of the one-workgroup form


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "falling", "rank1", "one"])
@pytest.mark.parametrize("r,c", SIZES)
def test_one_matrix(r, c, kind):
    g = torch.Generator().manual_seed(r * 1000 + c)
    u = matrix(r, c, kind, g)
    want, tol = allowed(u)
    d = u.to(DEV)
    out = torch.full((r, c), 7.0, device=DEV)
    ops.orthogonalize_batched([(d, out)])
    err = float((out.cpu().double() - want).norm())
    assert err <= tol, "%.3g over %.3g" % (err, tol)
    assert torch.equal(d.cpu(), u)
    ops.orthogonalize_batched([(d, d)])      # in place, the same bits
    assert torch.equal(d, out)


@pytest.mark.gpu
@pytest.mark.parametrize("r,c", [(2048, 1100), (1100, 2500), (4608, 192)])
def test_many_tiles(r, c):
    u = matrix(r, c, "normal", torch.Generator().manual_seed(3)).to(DEV)
    out = torch.empty_like(u)
    ops.orthogonalize_batched([(u, out)])
    want, tol = allowed(u)      # f64 products on the device
    assert float((out.double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 3, 6, 12])
@pytest.mark.parametrize("r,c", [(70, 40), (300, 70)])
def test_steps(r, c, steps):
    u = matrix(r, c, "falling", torch.Generator().manual_seed(1))
    want, tol = allowed(u, steps)
    out = torch.empty(r, c, device=DEV)
    ops.orthogonalize_batched([(u.to(DEV), out)], steps=steps)
    assert float((out.cpu().double() - want).norm()) <= tol


@pytest.mark.gpu
def test_batch_of_every_shape():
    g = torch.Generator().manual_seed(5)
    shapes = (SIZES * 2)[:32]
    us = [matrix(r, c, ("normal", "falling")[i % 2], g) * 10.0 ** (i % 7 - 3) for i, (r, c) in enumerate(shapes)]
    ds = [u.to(DEV) for u in us]
    outs = [torch.full_like(d, 7.0) for d in ds]
    ops.orthogonalize_batched(list(zip(ds, outs)))
    again = [torch.empty_like(d) for d in ds]
    ops.orthogonalize_batched(list(zip(ds, again)))
    for i, (u, o, a) in enumerate(zip(us, outs, again)):
        want, tol = allowed(u)
        assert torch.equal(o, a)
        assert float((o.cpu().double() - want).norm()) <= tol, shapes[i]


@pytest.mark.gpu
def test_singular_values_and_shapes_of_filters():
    """a conv kernel [kh,kw,cin,cout] is the matrix [kh*kw*cin, cout]; five steps bring its singular values to 0.6 .. 1.25"""
    w = torch.randn(3, 5, 20, 24, generator=torch.Generator().manual_seed(2)).to(DEV)
    out = torch.empty_like(w)
    ops.orthogonalize_batched([(w, out)])
    flat = torch.empty(300, 24, device=DEV)
    ops.orthogonalize_batched([(w.view(300, 24), flat)])
    assert torch.equal(out.view(300, 24), flat)
    s = torch.linalg.svdvals(flat.cpu().double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.25


@pytest.mark.gpu
@pytest.mark.parametrize("mag", [1e-25, 1e-4, 1e25, 5e37])
@pytest.mark.parametrize("r,c", [(50, 80), (300, 200)])
def test_magnitudes(r, c, mag):
    """the squares of the values leave f32: the norm is f64, and the result does not depend on the scale"""
    u = matrix(r, c, "normal", torch.Generator().manual_seed(6)) * mag
    want, tol = allowed(u, eps=1e-30)
    assert bool(torch.isfinite(u).all())
    out = torch.empty(r, c, device=DEV)
    ops.orthogonalize_batched([(u.to(DEV), out)], eps=1e-30)
    assert float((out.cpu().double() - want).norm()) <= tol


@pytest.mark.gpu
def test_zero_small_and_not_finite():
    for shape in ((70, 30), (300, 70)):
        z = torch.zeros(shape, device=DEV)
        out = torch.full_like(z, 7.0)
        ops.orthogonalize_batched([(z, out)], eps=1e-38)
        assert bool((out == 0).all())
    bad = torch.randn(40, 40, device=DEV)
    bad[3, 3] = float("nan")
    good = torch.randn(66, 40, generator=torch.Generator().manual_seed(1)).to(DEV)
    inf = torch.randn(20, 40, device=DEV)
    inf[1, 2] = float("inf")
    ob, og, oi = torch.empty_like(bad), torch.empty_like(good), torch.empty_like(inf)
    ops.orthogonalize_batched([(z, out), (bad, ob), (good, og), (inf, oi)])
    assert bool((out == 0).all()) and bool(torch.isnan(ob).all()) and bool(torch.isnan(oi).any())
    want, tol = allowed(good.cpu())
    assert float((og.cpu().double() - want).norm()) <= tol
    # a norm of half of eps
    tiny = matrix(10, 5, "normal", torch.Generator().manual_seed(9))
    tiny = tiny / tiny.norm() * 5e-8
    ot = torch.empty(10, 5, device=DEV)
    ops.orthogonalize_batched([(tiny.to(DEV), ot)])
    want, tol = allowed(tiny)
    assert float((ot.cpu().double() - want).norm()) <= tol


def muon64(p, g, m, lr, mu, wd, l2, nesterov, k, scale):
    g1 = (g.double() + l2 * p.double()) * scale
    m1 = mu * m.double() + g1
    u = g1 + mu * m1 if nesterov else m1
    return u, m1, lambda x: p.double() * (1 - lr * wd) - lr * k * x


@pytest.mark.gpu
@pytest.mark.parametrize("nesterov,wd,l2,clip,S", [(True, 0.0, 0.0, 0.0, None), (False, 0.1, 0.0, 0.0, None), (True, 0.01, 5e-4, 1.0, None),
                                                   (True, 0.01, 5e-4, 0.5, 1024.0), (False, 0.0, 1e-2, 1e6, 8.0)])
def test_muon_step(nesterov, wd, l2, clip, S):
    gen = torch.Generator().manual_seed(8)
    lr, mu = 0.02, 0.95
    shapes = [(3, 5, 16, 40), (64, 18), (1, 1, 100, 70), (33, 200)]
    ents, host = [], []
    for sh in shapes:
        p, g, m = (torch.randn(sh, generator=gen) * s for s in (0.02, 1e-3, 5e-3))
        if S:
            g = g * S
        host.append((p, g, m))
        ents.append([t.to(DEV) for t in (p, g, m)])
    norm = torch.sqrt(sum(((g / (S or 1.0)).double() ** 2).sum() for _, g, _ in host))
    gn = (norm ** 2).float().reshape(1).to(DEV)
    state = ops.loss_scale_state(S, DEV) if S else None
    outs = [(torch.full_like(p, 7.0), torch.full_like(m, 7.0)) for p, _, m in ents]
    kw = dict(momentum=mu, nesterov=nesterov, weight_decay=wd, l2=l2, gnorm_sq=gn, clip=clip, grad_scale=0.5, loss_scale=state)
    ops.muon_step([(p, g, m, po, mo, 1.5) for (p, g, m), (po, mo) in zip(ents, outs)], lr, **kw)
    gscale = 0.5 * (clip / max(float(gn.double().sqrt()) * 0.5, clip) if clip else 1.0)
    for (p, g, m), (po, mo) in zip(host, outs):
        u, m1, step = muon64(p, g / (S or 1.0), m, lr, mu, wd, l2, nesterov, 1.5, gscale)
        mag = mu * m.double().abs() + (g.double().abs() / (S or 1.0) + l2 * p.double().abs()) * gscale
        assert bool(((mo.cpu().double() - m1).abs() <= 8 * U * mag).all())
        u2 = u.reshape(-1, u.shape[-1])
        x, off = allowed(u2)
        want = step(x.reshape(p.shape))
        tol = lr * 1.5 * off + 4 * U * (float(p.double().norm()) + lr * 1.5 * float(x.norm()))
        assert float((po.cpu().double() - want).norm()) <= tol
    # in place: the same bits
    ops.muon_step([(p, g, m, p, m, 1.5) for p, g, m in ents], lr, **kw)
    for (p, _, m), (po, mo) in zip(ents, outs):
        assert torch.equal(p, po) and torch.equal(m, mo)


@pytest.mark.gpu
def test_skipped_steps():
    gen = torch.Generator().manual_seed(8)
    p, g, m = (torch.randn(70, 40, generator=gen).to(DEV) for _ in range(3))
    g[2, 2] = float("inf")
    gn = torch.full((1,), float("inf"), device=DEV)
    one = torch.ones(1, dtype=torch.int32, device=DEV)
    ok = torch.ones(1, device=DEV)
    for kw in (dict(gnorm_sq=gn, clip=1.0), dict(gnorm_sq=gn), dict(gnorm_sq=gn * float("nan")), dict(invalid=one),
               dict(invalid=one, gnorm_sq=ok, clip=1.0)):
        po, mo = torch.full_like(p, 7.0), torch.full_like(m, 7.0)
        ops.muon_step([(p, g, m, po, mo, 1.0)], 0.1, **kw)
        assert torch.equal(po, p) and torch.equal(mo, m)
        p1, m1 = p.clone(), m.clone()
        ops.muon_step([(p1, g, m1, p1, m1, 1.0)], 0.1, **kw)
        assert torch.equal(p1, p) and torch.equal(m1, m)
    g[2, 2] = 1.0
    ops.muon_step([(p, g, m, p1, m1, 1.0)], 0.1, gnorm_sq=ok, clip=1.0, invalid=one * 0)
    assert not torch.equal(p1, p) and bool(torch.isfinite(p1).all())


@pytest.mark.gpu
def test_side_stream_and_graph():
    gen = torch.Generator().manual_seed(8)
    ents = [[(torch.randn(s, generator=gen) * 0.1).to(DEV) for _ in range(3)] for s in ((200, 64), (64, 18), (100, 300))]
    outs = [(torch.empty_like(p), torch.empty_like(p)) for p, _, _ in ents]
    plan = ops.muon_descs([(p, g, m, po, mo, 1.0) for (p, g, m), (po, mo) in zip(ents, outs)])
    ws = torch.empty(ops.orthogonalize_workspace_bytes(plan[1]), dtype=torch.uint8, device=DEV)
    gn = torch.ones(1, device=DEV)

    def step(workspace=ws):
        ops.muon_step(plan, 0.1, gnorm_sq=gn, clip=1.0, workspace=workspace)
    step()
    torch.cuda.synchronize()
    want = [t.clone() for o in outs for t in o]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for o in outs:
            o[0].zero_()
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip([t for o in outs for t in o], want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for r in range(4):
        for e in ents:
            e[1].mul_(-0.7).add_(0.01)
        for o in outs:
            o[0].fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for o in outs for t in o]
        step(None)
        assert all(torch.equal(a, b) for a, b in zip([t for o in outs for t in o], got)), r


def test_iteration_against_svd():
    """the f64 iteration the kernels are held to maps singular values by the quintic and leaves singular vectors alone"""
    g = torch.Generator().manual_seed(1)
    for r, c in ((6, 9), (9, 6)):
        u = torch.randn(r, c, generator=g, dtype=torch.float64)
        a, s, b = torch.linalg.svd(u, full_matrices=False)
        s = s / (s.norm() + 1e-7)
        for _ in range(5):
            s = NS[0] * s + NS[1] * s ** 3 + NS[2] * s ** 5
        assert float((iterate(u) - (a * s) @ b).abs().max()) <= 1e-12


# ------------------------------------------------------------------------------------------------------------------ refusals
P = ctypes.c_void_p


def orth_rc(rows=4, cols=3, n=1, steps=5, eps=1e-7, g=P(4096), out=P(8192), ws=P(1 << 20), nbytes=1 << 40):
    d = (capi.OrthDesc * 33)()
    for x in d:
        x.g, x.out, x.rows, x.cols = g, out, rows, cols
    return capi.lib().cutie_orthogonalize_batched(d, n, steps, eps, ws, nbytes, None)


@pytest.mark.parametrize("kw,rc,word", [
    (dict(rows=0), -1, b"0 x 3"), (dict(cols=-1), -1, b"4 x -1"), (dict(n=0), -1, b"0 matrices"), (dict(n=33), -1, b"33 matrices"),
    (dict(steps=0), -1, b"steps"), (dict(steps=33), -1, b"steps"), (dict(eps=0.0), -1, b"eps"), (dict(g=None), -1, b"null"),
    (dict(out=P(8193)), -1, b"misaligned"), (dict(rows=1 << 20, cols=1 << 10), -1, b"2^29"), (dict(ws=None), -3, b"workspace"),
    (dict(nbytes=255), -3, b"workspace"), (dict(ws=P((1 << 20) + 16)), -3, b"workspace"), (dict(rows=300, cols=200, nbytes=4096), -3, b"workspace")])
def test_orthogonalize_refusals(kw, rc, word):
    assert orth_rc(**kw) == rc and word in capi.lib().cutie_last_error()


def test_muon_refusals():
    lib = capi.lib()
    d = (capi.MuonDesc * 1)()
    d[0].p, d[0].g, d[0].m, d[0].p_out, d[0].m_out = (4096 * k for k in range(1, 6))
    d[0].rows, d[0].cols, d[0].out_scale = 4, 3, 1.0

    def rc(steps=5, gn=None, clip=0.0, ws=P(1 << 20), n=1 << 40):
        return lib.cutie_muon_step(d, 1, 0.1, 0.9, 1, 0.0, 0.0, steps, 1e-7, gn, clip, 1.0, None, None, ws, n, None)
    assert rc(steps=0) == -1 and b"steps" in lib.cutie_last_error()
    assert rc(clip=1.0) == -1 and b"gnorm_sq" in lib.cutie_last_error()
    assert rc(clip=-1.0, gn=P(4096)) == -1 and b"clip" in lib.cutie_last_error()
    assert rc(n=0) == -3 and b"workspace" in lib.cutie_last_error()
    d[0].m = None
    assert rc() == -1 and b"null" in lib.cutie_last_error()


def test_workspace_bytes():
    assert ops.orthogonalize_workspace_bytes([(64, 18)]) > 0
    assert ops.orthogonalize_workspace_bytes([(64, 18), (300, 200)]) >= 2 * 320 * 256 * 4
    assert ops.orthogonalize_workspace_bytes([(0, 18)]) == 0 and ops.orthogonalize_workspace_bytes([(4, 4)] * 33) == 0


def test_wrapper_refusals():
    w = torch.zeros(4, 6)
    big = torch.zeros(100)
    for bad in (lambda: ops.orthogonalize_batched([]), lambda: ops.orthogonalize_batched([(w, w)] * 33),
                lambda: ops.orthogonalize_batched([(w.half(), w)]), lambda: ops.orthogonalize_batched([(w.t(), w.t())]),
                lambda: ops.orthogonalize_batched([(w, torch.zeros(6, 4))]), lambda: ops.orthogonalize_batched([(torch.zeros(0, 4), w)]),
                lambda: ops.orthogonalize_batched([(torch.zeros(4), torch.zeros(4))]), lambda: ops.orthogonalize_batched([(w, w.clone())]),
                lambda: ops.muon_step([], 0.1), lambda: ops.muon_step([(w, w.clone(), w.clone(), w, torch.zeros(4, 5), 1.0)], 0.1),
                lambda: ops.muon_descs([(w, w.clone(), w.clone(), w, w, 1.0)]),
                lambda: ops.muon_descs([(big[:24].view(4, 6), w.clone(), w.clone(), big[6:30].view(4, 6), w, 1.0)])):
        with pytest.raises(capi.CutieError):
            bad()


@pytest.mark.gpu
def test_overlapping_outputs_are_refused():
    w = torch.zeros(400, device=DEV)
    g, m = torch.zeros(4, 6, device=DEV), torch.zeros(4, 6, device=DEV)
    p = w[:24].view(4, 6)
    for po, mo in ((w[6:30].view(4, 6), m), (g, m), (m, m), (p, p), (p, g), (p, w[12:36].view(4, 6))):
        with pytest.raises(capi.CutieError, match="overlaps"):
            ops.muon_descs([(p, g, m, po, mo, 1.0)])
    ops.muon_descs([(p, g, m, p, m, 1.0)])
    ops.muon_descs([(p, g, m, w[24:48].view(4, 6), m, 1.0)])


# sizes around the borders of the three forms: one workgroup, tiles of rows with S up to 64, the general one
TALL = [(352, 16), (353, 16), (1, 353), (3, 400), (273, 32), (193, 48), (113, 64), (64, 129), (2049, 33), (17, 2050), (4100, 64), (8192, 5), (8193, 5)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "falling", "rank1", "one"])
@pytest.mark.parametrize("r,c", TALL)
def test_tall(r, c, kind):
    g = torch.Generator().manual_seed(r + 7 * c)
    u = matrix(r, c, kind, g)
    want, tol = allowed(u)
    buf = torch.full((r * c + 2,), 7.0, device=DEV)      # a misaligned matrix, and what lies around it
    out = buf[1:-1].view(r, c)
    ops.orthogonalize_batched([(u.to(DEV), out)])
    assert float((out.cpu().double() - want).norm()) <= tol
    assert float(buf[0]) == 7.0 and float(buf[-1]) == 7.0
    out.copy_(u)
    first = torch.empty(r, c, device=DEV)
    ops.orthogonalize_batched([(out, first)])
    ops.orthogonalize_batched([(out, out)])      # in place: the same bits
    assert torch.equal(out, first)


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 2, 6])
@pytest.mark.parametrize("mag", [1e-25, 1.0, 1e37])
def test_tall_steps_and_magnitudes(steps, mag):
    """the tiles' parts are scaled by a power of two each: rows of very different sizes, tiles of zeros among them"""
    g = torch.Generator().manual_seed(steps)
    u = matrix(700, 20, "normal", g)
    u[:64] *= 1e-20
    u[128:192] = 0
    u[300:] *= 1e-3
    u = u * mag
    for m in (u, u.t().contiguous()):
        want, tol = allowed(m, steps, eps=1e-30)
        out = torch.empty(m.shape, device=DEV)
        ops.orthogonalize_batched([(m.to(DEV), out)], steps=steps, eps=1e-30)
        assert float((out.cpu().double() - want).norm()) <= tol


@pytest.mark.gpu
def test_tall_zero_and_not_finite():
    z, out = torch.zeros(900, 40, device=DEV), torch.full((900, 40), 7.0, device=DEV)
    ops.orthogonalize_batched([(z, out)], eps=1e-38)
    assert bool((out == 0).all())
    good = torch.randn(50, 600, generator=torch.Generator().manual_seed(1))
    bad = good.clone()
    bad[3, 599] = float("nan")
    inf = good.clone()
    inf[49, 0] = float("-inf")
    outs = [torch.empty(50, 600, device=DEV) for _ in range(3)]
    ops.orthogonalize_batched([(t.to(DEV), o) for t, o in zip((bad, good, inf), outs)])
    assert bool(torch.isnan(outs[0]).all()) and bool(torch.isnan(outs[2]).any())
    want, tol = allowed(good)
    assert float((outs[1].cpu().double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 8, 9, 32])
def test_tall_batches(n):
    """up to 256 workgroups 64 columns are taken in tiles, from there on in the general form; 16 waves a workgroup or 8; small
    and large matrices of the same call in between"""
    g = torch.Generator().manual_seed(n)
    shapes = [(2048, 64) if i % 4 != 3 else ((40, 2000), (300, 200), (20, 16))[i // 4 % 3] for i in range(n)]
    us = [matrix(r, c, "normal", g) for r, c in shapes]
    outs = [torch.empty(s, device=DEV) for s in shapes]
    ops.orthogonalize_batched([(u.to(DEV), o) for u, o in zip(us, outs)])
    for u, o in zip(us, outs):
        want, tol = allowed(u)
        assert float((o.cpu().double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("S", [None, 1024.0])
def test_tall_muon_step_graph_and_skip(S):
    gen = torch.Generator().manual_seed(8)
    lr, mu, wd, l2, clip = 0.02, 0.95, 0.01, 5e-4, 0.5
    shapes = [(3, 3, 64, 40), (30, 1000), (1027, 3)]
    host = [tuple(torch.randn(sh, generator=gen) * s for s in (0.02, 1e-3 * (S or 1.0), 5e-3)) for sh in shapes]
    ents = [[t.to(DEV) for t in h] for h in host]
    gn = sum(((g / (S or 1.0)).double() ** 2).sum() for _, g, _ in host).float().reshape(1).to(DEV)
    state = ops.loss_scale_state(S, DEV) if S else None
    invalid = torch.zeros(1, dtype=torch.int32, device=DEV)
    outs = [(torch.full_like(p, 7.0), torch.full_like(m, 7.0)) for p, _, m in ents]
    plan = ops.muon_descs([(p, g, m, po, mo, 1.5) for (p, g, m), (po, mo) in zip(ents, outs)])
    ws = torch.empty(ops.orthogonalize_workspace_bytes(plan[1]), dtype=torch.uint8, device=DEV)

    def step():
        ops.muon_step(plan, lr, momentum=mu, weight_decay=wd, l2=l2, gnorm_sq=gn, clip=clip, loss_scale=state, invalid=invalid, workspace=ws)
    step()
    gscale = clip / max(float(gn.double().sqrt()), clip)
    for (p, g, m), (po, mo) in zip(host, outs):
        u, m1, after = muon64(p, g / (S or 1.0), m, lr, mu, wd, l2, True, 1.5, gscale)
        mag = mu * m.double().abs() + (g.double().abs() / (S or 1.0) + l2 * p.double().abs()) * gscale
        assert bool(((mo.cpu().double() - m1).abs() <= 8 * U * mag).all())
        x, off = allowed(u.reshape(-1, u.shape[-1]))
        tol = lr * 1.5 * off + 4 * U * (float(p.double().norm()) + lr * 1.5 * float(x.norm()))
        assert float((po.cpu().double() - after(x.reshape(p.shape))).norm()) <= tol
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for r in range(3):
        for e in ents:
            e[1].mul_(-0.7).add_(0.01)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for o in outs for t in o]
        step()
        assert all(torch.equal(a, b) for a, b in zip([t for o in outs for t in o], got)), r
    invalid.fill_(1)
    graph.replay()
    for (p, _, m), (po, mo) in zip(ents, outs):
        assert torch.equal(po, p) and torch.equal(mo, m)


def test_call_overlaps_are_refused():
    """the same matrix twice, an output over another matrix's tensors: refused on the host, nothing is launched"""
    lib = capi.lib()

    def orth(*pairs):
        d = (capi.OrthDesc * len(pairs))()
        for x, (g, out) in zip(d, pairs):
            x.g, x.out, x.rows, x.cols = g, out, 16, 16      # 1024 bytes each
        rc = lib.cutie_orthogonalize_batched(d, len(pairs), 5, 1e-7, P(1 << 20), 1 << 40, None)
        return rc, lib.cutie_last_error()
    for pairs in (((4096, 4096), (4096, 4096)), ((4096, 8192), (8192, 16384)), ((4096, 8192), (12288, 8192)), ((4096, 4100),),
                  ((4096, 5116),), ((4096, 8192), (12288, 9212))):
        rc, err = orth(*pairs)
        assert rc == -1 and b"overlaps" in err, pairs

    def muon(*mats):
        d = (capi.MuonDesc * len(mats))()
        for x, t in zip(d, mats):
            x.p, x.g, x.m, x.p_out, x.m_out = (1024 * k for k in t)
            x.rows, x.cols, x.out_scale = 16, 16, 1.0
        rc = lib.cutie_muon_step(d, len(mats), 0.1, 0.9, 1, 0.0, 0.0, 5, 1e-7, None, 0.0, 1.0, None, None, P(1 << 20), 1 << 40, None)
        return rc, lib.cutie_last_error()
    for mats in (((1, 2, 3, 1, 3), (1, 4, 5, 1, 5)), ((1, 2, 3, 4, 5), (6, 4, 7, 6, 7)), ((1, 2, 3, 3, 1),), ((1, 2, 3, 4, 4),),
                 ((1, 2, 3, 2, 3),), ((1, 2, 3, 1, 3), (4, 5, 3, 4, 6))):
        rc, err = muon(*mats)
        assert rc == -1 and b"overlaps" in err, mats


def test_sizes_beyond_the_c_abi_are_refused():
    meta = torch.empty(((1 << 32) + 5, 1), device="meta")
    with pytest.raises(capi.CutieError, match="2\\^29"):
        ops.orthogonalize_batched([(meta, meta)])
    w = torch.zeros(4, 6)
    plan = (None, [(4, 6)], w.device)
    for kw in (dict(loss_scale=torch.zeros(1)), dict(gnorm_sq=torch.zeros(0)), dict(invalid=torch.zeros(1)), dict(gnorm_sq=torch.zeros(1).half())):
        with pytest.raises(capi.CutieError, match="must be"):
            ops.muon_step(plan, 0.1, **kw)


@pytest.mark.gpu
def test_shared_inputs_and_neighbours_are_taken():
    g = torch.randn(64, 16, generator=torch.Generator().manual_seed(1)).to(DEV)
    w = torch.empty(2 * g.numel(), device=DEV)
    a, b = w[:g.numel()].view(64, 16), w[g.numel():].view(64, 16)
    ops.orthogonalize_batched([(g, a), (g, b)])      # one input twice, outputs side by side
    assert torch.equal(a, b)
    want, tol = allowed(g.cpu())
    assert float((a.cpu().double() - want).norm()) <= tol
    with pytest.raises(capi.CutieError, match="overlaps"):
        ops.orthogonalize_batched([(g, a), (g, a)])
