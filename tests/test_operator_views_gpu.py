"""What views the group norm and the scaled embedding take: any whose leading axes collapse to one row index, an axis of one element
having no say.  The answer on a view is the answer on its dense copy, bit for bit where the form of the kernel does not depend on
the view (it never does: forms are chosen by sizes), and every other view is refused.
"""
import pytest
import torch

from cutie_amd import capi, ops

DEV = "cuda:0"
# slices of a [3, 8, 9, 24] tensor whose rows of pixels collapse, and the leading dimension they collapse to
VIEWS = [
    ("all of it", lambda w: w, 24),
    ("some channels", lambda w: w[..., 3:19], 24),
    ("pixels of one sample", lambda w: w[1:2, :5], 24),
    ("one row", lambda w: w[1:2, 2:3], 24),
    ("a part of a row", lambda w: w[2:3, 4:5, 2:6, 8:16], 24),
    ("one column", lambda w: w[:, :, 3:4], 9 * 24),
    ("one column of one sample", lambda w: w[:1, :, 8:, 1:2], 9 * 24),
    ("one pixel of each sample", lambda w: w[:, 7:, :1, :8], 8 * 9 * 24),
    ("every other row of pixels of one column", lambda w: w[:, ::2, 3:4], 2 * 9 * 24),
    ("one pixel", lambda w: w[2:, 3:4, 3:4, 5:6], 1),
    ("samples all the same way", lambda w: w[:, :1, :1].permute(1, 0, 2, 3), 8 * 9 * 24),
]
REFUSED = [
    ("rows of two samples", lambda w: w[:2, :5]), ("one row of two samples", lambda w: w[:2, 2:3]), ("columns", lambda w: w[:1, :, 2:5]),
    ("channels apart", lambda w: w[..., ::2]), ("transposed", lambda w: w.permute(0, 2, 1, 3)), ("a row of channels apart", lambda w: w[:1, :1, :1, ::2]),
]


@pytest.mark.parametrize("what,cut,ld", VIEWS)
def test_leading_dimension(what, cut, ld):
    w = torch.arange(3 * 8 * 9 * 24).view(3, 8, 9, 24)
    v = cut(w)
    rows = v.numel() // v.shape[-1]
    assert ops._rows_ld(v) == ld
    assert torch.equal(v.as_strided((rows, v.shape[-1]), (ld, 1)), v.reshape(rows, v.shape[-1]))


@pytest.mark.parametrize("what,cut", REFUSED)
def test_other_views_are_refused(what, cut):
    with pytest.raises(capi.CutieError):
        ops._rows_ld(cut(torch.zeros(3, 8, 9, 24)))


def test_rows_that_share_memory_keep_their_stride():
    """an expanded axis has the stride 0, which the C ABI refuses (below the row's width); it is no axis of one element"""
    assert ops._rows_ld(torch.zeros(1, 5).expand(4, 5)) == 0
    assert ops._rows_ld(torch.zeros(0, 5)) == 5 and ops._rows_ld(torch.zeros(5)) == 5
    with pytest.raises(capi.CutieError):
        ops._rows_ld(torch.zeros(10)[::2])


def group_count(C):
    return 2 if C % 2 == 0 else 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("what,cut,ld", VIEWS)
def test_group_norm_on_views(what, cut, ld, dtype):
    g = torch.Generator().manual_seed(1)
    wide = [torch.randn(3, 8, 9, 24, generator=g).to(dtype).to(DEV) for _ in range(2)]
    x, dy = (cut(t) for t in wide)
    B, H, W, C = x.shape
    y0, s0, d0 = (torch.empty(B, H, W, C, dtype=dtype, device=DEV), torch.empty(B, group_count(C), 2, device=DEV),
                  torch.empty(B, H, W, C, dtype=dtype, device=DEV))
    ops.gn_fwd(x.contiguous(), y0, s0, act="silu")
    ops.gn_bwd(dy.contiguous(), x.contiguous(), s0, d0, act="silu")
    out = [torch.full((3, 8, 9, 24), 3.0, dtype=dtype, device=DEV) for _ in range(2)]
    y, dx, st = cut(out[0]), cut(out[1]), torch.empty_like(s0)
    ops.gn_fwd(x, y, st, act="silu")
    ops.gn_bwd(dy, x, st, dx, act="silu")
    assert torch.equal(st, s0) and torch.equal(y, y0) and torch.equal(dx, d0)
    for t in out:      # and nothing else is written
        cut(t).fill_(3.0)
        assert bool((t == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("what,cut,ld", VIEWS)
def test_embedding_on_views(what, cut, ld):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(3, 8, 9, 24, generator=g).to(DEV)
    d = cut(wide)
    V, E = 7, d.shape[-1]
    ids = torch.randint(0, V, d.shape[:-1], generator=g, dtype=torch.int32).to(DEV)
    table = torch.randn(V, E, generator=g).to(DEV)
    oob = torch.zeros(1, dtype=torch.int32, device=DEV)
    out = torch.full((3, 8, 9, 24), 3.0, device=DEV)
    ops.embed_scaled_fwd(ids, table, cut(out), 2.0, oob)
    assert torch.equal(cut(out), table[ids.long()] * 2.0) and int(oob) == 0
    cut(out).fill_(3.0)
    assert bool((out == 3.0).all())
    got, want = torch.empty(V, E, device=DEV), torch.empty(V, E, device=DEV)
    ops.embed_grad_sorted(ids, d, got)
    ops.embed_grad_sorted(ids, d.contiguous(), want)
    assert torch.equal(got, want)
