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
