"""Group norm at the ends of what it accepts: more (sample, group) pairs than one launch has threads for, planes whose sums are long,
levels far above the spread, several groups in a workgroup.  The f64 definitions, the tolerances and their derivation are those of
test_group_norm_gpu.py; where a case needs another one it is derived beside it.
"""
import pytest
import torch

import test_group_norm_gpu as gn
from cutie_amd import ops

DEV, U = gn.DEV, gn.U


@pytest.mark.gpu
def test_more_groups_than_a_launch_has_threads():
    """81.9 million (sample, group) pairs of eleven values: workgroups of 64 threads would be 5.2e9 threads"""
    B, G, C = 20000, 4093, 45023
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty((B, 1, 1, C), dtype=torch.float16, device=DEV)
    dy = torch.empty_like(x)
    for t in (x, dy):
        for lo in range(0, B, 2000):
            t[lo:lo + 2000] = torch.randn((2000, 1, 1, C), generator=g, device=DEV)
    y = torch.full_like(x, 7.0)
    stats = torch.full((B, G, 2), 7.0, device=DEV)
    ops.gn_fwd(x, y, stats)
    assert float(y.max()) < 4.0      # of eleven values none lies further than sqrt(10) from their mean: every one was written
    dx = torch.full_like(x, float("inf"))
    ops.gn_bwd(dy, x, stats, dx)
    assert bool(torch.isfinite(dx).all())
    at = torch.tensor([0, 1, 9999, 13107, 19998, 19999], device=DEV)
    xs, ys, ss = x[at], y[at], stats[at]
    gn.check_fwd(xs, G, None, None, "none", ys, ss)
    ref, _, _, mag, _, _ = gn.gn_bwd64(dy[at].cpu(), xs.cpu(), ss.cpu(), None, None, "none")
    tol = 2.0 ** -11 * ref.abs() * (1 + 2.0 ** -11) + (512 * U + 2.0 ** -20) * mag + 2.0 ** -25
    assert bool(((dx[at].cpu().double() - ref).abs() <= tol).all())


# a plane in slices (16 channels a group, 270400 values), eleven channels a group, one with 16-byte vectors that span groups
SLICED = [(1, 130, 130, 32, 2), (1, 130, 131, 33, 3), (2, 90, 91, 20, 1), (1, 130, 130, 36, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("level,spread", [(1e5, 1.0), (1e6, 0.25), (1e8, 100.0), (-3e6, 1.0), (1e6, 0.0)])
@pytest.mark.parametrize("shape", SLICED)
def test_plane_in_slices_far_above_its_spread(shape, level, spread):
    """Sums in f64 about the group's first value s: at most 2^13 roundings in a row, of sums that (s - mean)^2 <= N var keeps below
    N + 1 times the variance, N < 2^20: 2^(13 + 20 - 53) = 2^-20 of 1/sigma, and the f32 steps behind it: 512 u holds.  x - mean
    is exact (both lie within a factor of two) up to the mean's residue, which the kernel carries."""
    B, H, W, C, G = shape
    x = (level + spread * torch.randn(B, H, W, C, generator=torch.Generator().manual_seed(int(abs(level)) % 97))).to(DEV)
    y, stats = gn.run_fwd(x, G, None, None, "none")
    ref, mean, rstd, _, _ = gn.gn64(x.cpu(), G, None, None, "none")
    got = stats.cpu().double()
    assert float(((got[..., 1] - rstd).abs() / rstd).max()) <= 512 * U
    assert float(((got[..., 0] - mean).abs() / mean.abs()).max()) <= 2 * U
    assert float((y.cpu().double() - ref).abs().max()) <= 512 * U * max(1.0, float(ref.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,level,step", [(torch.float16, 4096.0, 4.0), (torch.float16, 60000.0, 32.0), (torch.bfloat16, 2.0 ** 20, 2.0 ** 13)])
@pytest.mark.parametrize("every", [2, 1000, 100000])
@pytest.mark.parametrize("shape", SLICED)
def test_sixteen_bit_plane_of_two_neighbouring_values(shape, every, dtype, level, step):
    """one value in `every` is one step of the type above the others: the sums are exact, and so is the variance up to the f64 steps
    behind them"""
    B, H, W, C, G = shape
    x = torch.full((B * H * W * C,), level)
    x[every // 2::every] += step
    x = x.to(dtype).view(B, H, W, C).to(DEV)
    assert x.unique().numel() == 2
    y, stats = gn.run_fwd(x, G, None, None, "none")
    ref, mean, rstd, _, _ = gn.gn64(x.cpu(), G, None, None, "none")
    got = stats.cpu().double()
    assert float(((got[..., 1] - rstd).abs() / rstd).max()) <= 4 * U
    assert float(((got[..., 0] - mean).abs() / mean).max()) <= 2 * U
    gn.check_fwd(x, G, None, None, "none", y, stats)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("dtype", gn.DTYPES)
def test_first_value_that_is_not_finite(dtype, bad):
    """the value that the sums are taken about: its group is NaN, its neighbours are what they were"""
    x, _, _, _ = gn.make(2, 130, 130, 32, 2, dtype, seed=3)
    clean, cs = gn.run_fwd(x, 2, None, None, "none")
    x[1, 0, 0, 16] = bad
    y, stats = gn.run_fwd(x, 2, None, None, "none")
    assert bool(torch.isnan(y[1, ..., 16:]).all()) and bool(torch.isnan(stats[1, 1, 1]))
    assert torch.equal(y[0], clean[0]) and torch.equal(y[1, ..., :16], clean[1, ..., :16]) and torch.equal(stats[0], cs[0])


@pytest.mark.gpu
@pytest.mark.parametrize("HW,C,G,dtype", [((16384, 16384), 1, 1, torch.float32), ((4096, 4096), 24, 2, torch.bfloat16), ((512, 512), 1024, 32, torch.float32)])
def test_backward_of_a_large_plane(HW, C, G, dtype):
    """2^28 values of one channel, 4096 pixels a thread.  f32 sums are of 64 pixels; theirs are in f64, a slice's is rounded to f32
    once, at most 256 slices of a channel are added in f32, in any order, and 16 more cover the terms' own roundings and a group's
    channels: 336 u of the magnitudes.  (One f32 chain of 4096 equal terms of 0.7 drifts by 679.)  dy is one value, with a little
    noise on half of the rows, so that roundings do not cancel."""
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.randn((1, *HW, C), generator=g, device=DEV).to(dtype)
    dy = torch.full_like(x, 0.7)
    dy[:, ::2] += 0.01 * torch.randn(dy[:, ::2].shape, generator=g, device=DEV).to(dtype)
    y, stats = gn.run_fwd(x, G, None, None, "none")
    del y
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.gn_bwd(dy, x, stats, dx, dgamma=dgamma, dbeta=dbeta)
    n = HW[0] * HW[1]
    half = gn.HALF[dtype]
    for k in range(0, C, max(1, C // G)):      # group by group, f64 on the device
        cut = slice(k, k + C // G)
        mean, rstd = (stats[0, k // (C // G), i].double() for i in (0, 1))
        xh = (x[0, ..., cut].double().reshape(n, -1) - mean) * rstd
        d = dy[0, ..., cut].double().reshape(n, -1)
        sg, sx, mg, mx = d.sum(0), (d * xh).sum(0), d.abs().sum(0), (d * xh).abs().sum(0)
        assert bool(((dbeta[cut].double() - sg).abs() <= 336 * U * mg).all())
        assert bool(((dgamma[cut].double() - sx).abs() <= 336 * U * mx).all())
        N = n * (C // G)
        ref = rstd * (d - sg.sum() / N - xh * (sx.sum() / N))
        mag = rstd * (d.abs() + mg.sum() / N + xh.abs() * (mx.sum() / N))
        err = (dx[0, ..., cut].double().reshape(n, -1) - ref).abs()
        assert bool((err <= half * ref.abs() + 336 * U * mag).all()), float((err / (half * ref.abs() + 336 * U * mag)).max())
        del xh, d, ref, mag, err


# batches of 256 (sample, group) pairs and more, whose workgroups take several groups of a pixel (their number in brackets, and the
# threads side by side in a pixel): both kinds of sums, and samples that share a workgroup's share of groups with no other
SEVERAL = [
    (64, 16, 16, 64, 8),      # [2] 4 or 2 threads: lane exchanges
    (64, 9, 7, 96, 8),        # [2] 6: through LDS
    (64, 9, 7, 36, 12),       # [3] 9 single elements
    (300, 5, 5, 40, 10),      # [10] 10
    (128, 8, 8, 512, 64),     # [4 or 8] 8
    (40, 31, 9, 264, 33),     # [3] 6 or 3
    (512, 3, 3, 96, 4),       # [4] 24 or 12
    (64, 16, 16, 192, 48),    # [4 or 8] vectors of four in a 16-bit type
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", gn.DTYPES)
@pytest.mark.parametrize("act", ["silu", "relu"])
@pytest.mark.parametrize("B,H,W,C,groups", SEVERAL)
def test_several_groups_in_a_workgroup(B, H, W, C, groups, act, dtype):
    check_both(B, H, W, C, groups, act, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", gn.DTYPES)
@pytest.mark.parametrize("B,H,W,act", [(16, 64, 64, "silu"), (16, 48, 40, "sigmoid")])
def test_the_widest_workgroups(B, H, W, act, dtype):
    """256 channels in 32 groups, two of them a workgroup: 8 to 16 vectors a thread, 128 KB of x in LDS on the way back"""
    check_both(B, H, W, 256, 32, act, dtype)


def check_both(B, H, W, C, groups, act, dtype):
    x, dy, gamma, beta = gn.make(B, H, W, C, groups, dtype, seed=B + C)
    y, stats = gn.run_fwd(x, groups, gamma, beta, act)
    gn.check_fwd(x, groups, gamma, beta, act, y, stats)
    dx, dgamma, dbeta = torch.full_like(dy, 7.0), torch.full((C,), 7.0, device=DEV), torch.full((C,), 7.0, device=DEV)
    ops.gn_bwd(dy, x, stats, dx, gamma=gamma, beta=beta, act=act, dgamma=dgamma, dbeta=dbeta)
    gn.check_bwd(dy, x, stats, gamma, beta, act, dx, dgamma, dbeta)
    # the whole batch is the samples one by one, which take another number of groups a workgroup: to the rounding of the sums
    for b in (0, B - 1):
        y1, s1 = gn.run_fwd(x[b:b + 1], groups, gamma, beta, act)
        gn.check_fwd(x[b:b + 1], groups, gamma, beta, act, y1, s1)
        assert float((s1[0] - stats[b]).abs().max()) <= 1024 * U * float(stats[b].abs().max() + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "silu"])
@pytest.mark.parametrize("shape", [(1, 16, 16, 32, 4), (1, 130, 130, 32, 2)])
def test_backward_at_a_level_far_above_the_spread(shape, act):
    """against the gradient at the values' own statistics.  The backward takes the mean as it is stored, rounded to f32: every xhat is
    off by one r <= 2^-24 |mean| / sigma (2.4e-4 here: 4096 sigma), and with it dgamma by r sum |g|, and dx by what r moves in
    xhat mean(h xhat) and, through act'' (at most 1/2), in h.  Nothing else is lost to the level."""
    B, H, W, C, G = shape
    g = torch.Generator().manual_seed(4)
    x = (4096.0 + torch.randn(B, H, W, C, generator=g)).to(DEV)
    dy = torch.randn(B, H, W, C, generator=g).to(DEV)
    gamma, beta = (1 + 0.3 * torch.randn(C, generator=g)).to(DEV), (0.3 * torch.randn(C, generator=g)).to(DEV)
    _, stats = gn.run_fwd(x, G, gamma, beta, act)
    dx, dgamma, dbeta = torch.empty_like(x), torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.gn_bwd(dy, x, stats, dx, gamma=gamma, beta=beta, act=act, dgamma=dgamma, dbeta=dbeta)
    _, mean, rstd, xh, z = gn.gn64(x.cpu(), G, gamma.cpu(), beta.cpu(), act)
    true = torch.stack([mean, rstd], dim=-1)
    ref, rg, rb, mag, mg, mb = gn.gn_bwd64(dy.cpu(), x.cpu(), true, gamma.cpu(), beta.cpu(), act)
    r = 2.0 ** -24 * float((mean.abs() * rstd).max())
    ga, d = gamma.cpu().double(), dy.cpu().double().abs()
    dh = 0.5 * r * d * ga ** 2 if act == "silu" else torch.zeros_like(d)      # h may be off by this
    grouped = lambda t: t.reshape(B, H * W, G, C // G)
    mean_of = lambda t: grouped(t).mean((1, 3), keepdim=True).expand(B, H * W, G, C // G).reshape(B, H, W, C)
    h = (1.1 * d * ga.abs())      # |act'| <= 1.1
    rs = rstd.reshape(B, 1, G, 1).expand(B, H * W, G, C // G).reshape(B, H, W, C)
    tol = 512 * U * mag + rs * (dh + mean_of(dh) + xh.abs() * mean_of(dh * xh.abs()) + 2 * r * (mean_of(h * xh.abs()) + xh.abs() * mean_of(h)))
    assert bool(((dx.cpu().double() - ref).abs() <= U * ref.abs() + tol).all())
    sg = (dh / ga.abs()).sum((0, 1, 2))
    assert bool(((dbeta.cpu().double() - rb).abs() <= 512 * U * mb + sg).all())
    assert bool(((dgamma.cpu().double() - rg).abs() <= 512 * U * mg + (dh / ga.abs() * xh.abs()).sum((0, 1, 2)) + 1.1 * r * d.sum((0, 1, 2)) + r * sg).all())


@pytest.mark.gpu
@pytest.mark.parametrize("B,H,W,C,groups", [
    (17000, 32, 32, 256, 32),      # whole groups in a workgroup
    (3, 8192, 8192, 24, 2),        # in slices
])
def test_offsets_beyond_32_bits(B, H, W, C, groups):
    """more than 2^32 values: the last sample alone, as a view of the same memory, gives the same bits or, where a batch takes another
    number of groups a workgroup, the same values to the rounding of the sums"""
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.empty((B, H, W, C), dtype=torch.bfloat16, device=DEV)
    assert x.numel() > 2 ** 32
    step = max(1, B // 16)
    for lo in range(0, B, step):
        x[lo:lo + step] = torch.randn(x[lo:lo + step].shape, generator=g, device=DEV, dtype=torch.bfloat16)
    dy = torch.flip(x, dims=(0,))
    y, stats, dx = torch.empty_like(x), torch.empty(B, groups, 2, device=DEV), torch.empty_like(x)
    dgamma, dbeta = torch.empty(C, device=DEV), torch.empty(C, device=DEV)
    ops.gn_fwd(x, y, stats, act="silu")
    ops.gn_bwd(dy, x, stats, dx, act="silu", dgamma=dgamma, dbeta=dbeta)
    for b in (0, B - 1):
        y1, s1, dx1 = torch.empty_like(x[b:b + 1]), torch.empty(1, groups, 2, device=DEV), torch.empty_like(x[b:b + 1])
        ops.gn_fwd(x[b:b + 1], y1, s1, act="silu")
        assert float((s1[0] - stats[b]).abs().max()) <= 1024 * U * float(stats[b].abs().max() + 1)
        ops.gn_bwd(dy[b:b + 1], x[b:b + 1], stats[b:b + 1].contiguous(), dx1, act="silu")
        # two roundings to bf16 of values that agree to f32 rounding: equal, or neighbours
        for got, want in ((y[b], y1[0]), (dx[b], dx1[0])):
            assert float((got.float() - want.float()).abs().max()) <= 2.0 ** -7 * float(want.float().abs().max())
            assert float((got != want).float().mean()) < 1e-3
    assert bool(torch.isfinite(dgamma).all()) and bool(torch.isfinite(dbeta).all())
