"""The sorted embedding gradient where its sums are long: as many parts of one id as the cells make, wide rows that a workgroup takes one
at a time, long text.  With u = 2^-24, and s the pairs a thread adds in a row (at most 1024: a workgroup of one row of columns), r the
rows side by side in a workgroup (s r <= 1280), a part is off by at most (s + r) u of its terms' magnitudes; parts are added in f64,
and a part, the sum and the product with the scale are rounded once each: (s + r + 3) u, at most 1284 u.
"""
import pytest
import torch

import test_embed_sorted_gpu as es
from cutie_amd import ops

DEV, U = es.DEV, es.U


@pytest.mark.gpu
def test_parts_of_one_id_meet_in_f64():
    """8388608 equal rows of 516 columns on one id: 8192 parts of 1024.  A chain of f32 additions of the parts drifts by 1369 u (the
    parts themselves by 60)"""
    n, E = 1 << 23, 516
    ids = torch.full((n,), 1, dtype=torch.int32, device=DEV)
    dout = torch.full((n, E), 1.3, device=DEV)
    got = torch.empty(3, E, device=DEV)
    ops.embed_grad_sorted(ids, dout, got)
    want = float(torch.tensor(1.3).double()) * n
    assert not got[0].any() and not got[2].any()
    assert float((got[1].double() - want).abs().max()) <= (1024 + 1 + 3) * U * want


# rows that a workgroup takes one, two or more of, at every number of pairs a workgroup adds (64, 256, 1024), ids all one, most one
WIDE = [
    (300000, 3000, 512, "grid"), (300000, 3000, 512, "one"), (270000, 50, 1023, "grid"), (270000, 50, 1024, "one"), (270000, 50, 1024, "grid"),
    (270000, 7, 516, "one"), (262144, 900, 260, "grid"), (65537, 40, 1032, "grid"), (65536, 40, 1032, "one"), (20000, 11, 4100, "grid"),
    (5000, 3, 65536, "uniform"), (300000, 100000, 36, "uniform"), (300000, 300, 1, "grid"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", es.DTYPES)
@pytest.mark.parametrize("n,V,E,kind", WIDE)
def test_every_cell_counts_once(n, V, E, kind, dtype):
    """whole-number rows of up to 31 either way, whose sums of any part stay below 2^24: every f32 sum is exact, and the result is
    equal to the sum in whole numbers, scaled by a power of two"""
    g = torch.Generator().manual_seed(n + V + E)
    ids = es.draw_ids(n, V, kind, g).to(DEV)
    gd = torch.Generator(device=DEV).manual_seed(E)
    dout = torch.randint(-31, 32, (n, E), generator=gd, device=DEV, dtype=torch.int8).to(dtype)
    want = torch.zeros(V, E, device=DEV)
    for lo in range(0, n, 1 << 15):      # every addition is exact: the order is no matter
        want.index_add_(0, ids[lo:lo + (1 << 15)].long(), dout[lo:lo + (1 << 15)].float())
    assert float(want.abs().max()) < 2 ** 24
    got = torch.full((V, E), 7.0, device=DEV)
    ops.embed_grad_sorted(ids, dout, got, scale=0.25)
    assert torch.equal(got, want * 0.25)
    base = torch.randint(-99, 100, (V, E), generator=gd, device=DEV).float()
    acc = base.clone()
    ops.embed_grad_sorted(ids, dout, acc, scale=2.0, accumulate=True)
    assert torch.equal(acc, base + want * 2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", es.DTYPES)
@pytest.mark.parametrize("n,V,E,kind", [c for c in WIDE if c[0] * c[2] < 1.6e8])
def test_rounded_sums(n, V, E, kind, dtype):
    g = torch.Generator().manual_seed(n + V + E)
    ids = es.draw_ids(n, V, kind, g)
    dout = torch.randn(n, E, generator=torch.Generator(device=DEV).manual_seed(E), device=DEV).to(dtype)
    got = torch.empty(V, E, device=DEV)
    ops.embed_grad_sorted(ids.to(DEV), dout, got, scale=-1.5)
    s, m = es.expect(ids, dout.cpu(), V, -1.5)
    assert bool(((got.cpu().double() - s).abs() <= 1284 * U * m).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,E", [(torch.float16, 516), (torch.float32, 513)])
def test_lookup_beyond_32_bits_of_values(dtype, E):
    n, V = (1 << 23) + 5, 77
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(-1, V, (n,), generator=g, device=DEV, dtype=torch.int32)
    table = torch.randn(V, E, generator=g, device=DEV)
    out = torch.empty((n, E), dtype=dtype, device=DEV)
    assert out.numel() > 2 ** 32
    oob = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.embed_scaled_fwd(ids, table, out, 1.5, oob)
    assert int(oob) == int((ids < 0).sum())
    rows = torch.cat([table * 1.5, torch.zeros(1, E, device=DEV)]).to(dtype)      # an id outside the table: a row of zeros
    for lo in range(0, n, 1 << 20):
        i = ids[lo:lo + (1 << 20)].long()
        assert torch.equal(out[lo:lo + (1 << 20)], rows[torch.where(i < 0, V, i)]), lo
