"""The 128-wide tiles of the update's three products: matrices large enough for them, at odd multiples of 64 (half-empty edge tiles), K
cut and whole.  Which tiles a call takes shows in its workspace (the larger of the two symmetric products' slabs), whose size the first
test holds to the rule.

Tolerance.  That of test_muon_gpu.py - the iteration in f64 with the format's errors drawn at random, eight times, times four - with one
term more, since the sums are long here: a value of a product is n = 3 K / 32 additions in f32 (three matrix instructions for 32
terms), each off by at most half a step, 2^-24, of a partial sum that grows evenly to at most the sum of its terms' magnitudes (as it
does where they have one sign: rank 1).  Independent roundings add as the root of the sum of their squares: sqrt(n / 3) 2^-24 of it.
"""
import pytest
import torch

import test_muon_gpu as mu
from cutie_amd import ops

DEV = mu.DEV


def rounded(u, steps, eps, seed):
    """mu.rounded() with the roundings of the sums"""
    g = torch.Generator(device=u.device).manual_seed(seed)

    def draw(*shape):
        return 2 * torch.rand(shape, generator=g, device=u.device, dtype=torch.float64) - 1

    def off(t):
        return t * (1 + mu.H * draw(*t.shape))

    def product(p, q):
        size = p.abs() @ q.abs()
        return p @ q + mu.H / 2 * draw(*size.shape) * size + (p.shape[1] / 32) ** 0.5 * 2.0 ** -24 * draw(*size.shape) * size
    a, b, c = mu.NS
    x = u if u.shape[0] >= u.shape[1] else u.t()
    x = off(x / (u.norm() + eps))
    for _ in range(steps):
        m = off(product(x.t().contiguous(), x))
        y = off(b * m + c * product(m, m))
        x = off(a * x + product(x, y))
    return x if u.shape[0] >= u.shape[1] else x.t()


def allowed(u, steps=5, eps=1e-7):
    u = u.double()
    want = mu.iterate(u, steps, eps)
    return want, 4 * max(float((rounded(u, steps, eps, k) - want).norm()) for k in range(8))


def up(v, m):
    return -(-v // m) * m


def tri(S, f):
    nt = -(-S // (32 * f))
    return nt * (nt + 1) // 2


def workspace(shapes, fg, fs):
    """bytes of the general form with tiles of 32 fg (X^T X) and 32 fs (A A)"""
    pads = [(up(max(s), 64), up(min(s), 64)) for s in shapes]
    ng, nq = sum(tri(S, fg) for _, S in pads), sum(tri(S, fs) for _, S in pads)

    def cut(want, steps):
        return max(1, min(want, steps // 4, 64))
    total = 0
    for (r, c), (L, S) in zip(shapes, pads):
        gram = cut(512 // ng, L // 32) * tri(S, fg) * (32 * fg) ** 2 * 4
        square = (cut(512 // nq, S // 32) if S > 512 else 1) * tri(S, fs) * (32 * fs) ** 2 * 4
        total += sum(up(b, 256) for b in (L * S * 4, L * S * 4, S * S * 4, S * S * 4, max(gram, square), -(-r * c // 8192) * 8))
    return total


CASES = [
    # shapes, tile factor of X^T X, of A A
    ([(2240, 2300)], 4, 4),            # 35 blocks of 64; both K cut in two
    ([(2300, 2240)], 4, 4),
    ([(26300, 500)], 4, 2),            # K of X^T X cut in 51
    ([(1472, 1500)], 2, 4),            # 23 blocks; A A's K cut in six
    ([(448, 500)] * 32, 2, 4),         # 7 blocks; A A whole, straight to B with its mirror
    ([(500, 448)] * 32, 2, 4),
    ([(1088, 1100)] * 16, 4, 4),       # 17 blocks; nothing cut
]


@pytest.mark.parametrize("shapes,fg,fs", CASES)
def test_the_tiles_are_these(shapes, fg, fs):
    sizes = {(a, b): workspace(shapes, a, b) for a in (2, 4) for b in (2, 4)}
    got = ops.orthogonalize_workspace_bytes(shapes)
    assert got == sizes[fg, fs], (got, sizes)
    assert got != sizes[2, 2] and (fs == 4 or got != sizes[2, 4])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "rank1", "one"])
@pytest.mark.parametrize("shapes,fg,fs", CASES)
def test_against_f64(shapes, fg, fs, kind):
    g = torch.Generator().manual_seed(len(shapes) + shapes[0][0])
    us = [mu.matrix(r, c, kind, g).to(DEV) for r, c in shapes]
    outs = [torch.full_like(u, 7.0) for u in us]
    ops.orthogonalize_batched(list(zip(us, outs)))
    for k in sorted({0, len(us) // 2, len(us) - 1}):
        want, tol = allowed(us[k])
        err = float((outs[k].double() - want).norm())
        assert err <= tol, "matrix %d: %.3g over %.3g" % (k, err, tol)
    assert all(bool(torch.isfinite(o).all()) for o in outs)
    again = [torch.empty_like(u) for u in us]
    ops.orthogonalize_batched(list(zip(us, again)))
    assert all(torch.equal(a, o) for a, o in zip(again, outs))


@pytest.mark.gpu
def test_update_of_a_large_matrix():
    """the momentum step in place around the 128-wide tiles, rows of a length that is no multiple of four"""
    g = torch.Generator().manual_seed(1)
    p, grad, m = (torch.randn(2243, 2301, generator=g).to(DEV) * s for s in (0.02, 1e-3, 5e-3))
    p0, m0 = p.clone(), m.clone()
    ops.muon_step([(p, grad, m, p, m, 1.25)], 0.02, momentum=0.95, weight_decay=0.01, l2=5e-4)
    gd = grad.double() + 5e-4 * p0.double()
    m1 = 0.95 * m0.double() + gd
    mag = 0.95 * m0.double().abs() + grad.double().abs() + 5e-4 * p0.double().abs()
    assert bool(((m.double() - m1).abs() <= 8 * mu.U * mag).all())
    x, off = allowed((gd + 0.95 * m1).float())
    want = p0.double() * (1 - 0.02 * 0.01) - 0.02 * 1.25 * x
    tol = 0.02 * 1.25 * off + 4 * mu.U * (float(p0.double().norm()) + 0.02 * 1.25 * float(x.norm()))
    assert float((p.double() - want).norm()) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "rank1"])
@pytest.mark.parametrize("r,c", [(1 << 20, 1), (5, 100001), (8193, 64), (30001, 70)])
def test_long_and_thin(r, c, kind):
    """more rows than the form with one launch a step takes"""
    u = mu.matrix(r, c, kind, torch.Generator().manual_seed(r + c)).to(DEV)
    out = torch.full_like(u, 7.0)
    ops.orthogonalize_batched([(u, out)])
    want, tol = allowed(u)
    assert float((out.double() - want).norm()) <= tol
