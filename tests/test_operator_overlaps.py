"""Calls of the training operators in which an output shares memory with another tensor are refused on the host, before anything is
launched: made-up addresses, no GPU.  (Tensors that only lie in the gaps between the rows of a view are neighbours, not overlaps.)
"""
import ctypes

import pytest
import torch

from cutie_amd import capi, ops

A = ctypes.c_void_p
FAR = [1 << k for k in range(36, 46)]      # addresses that meet nothing


def refused(rc):
    return rc == -1 and b"overlaps" in capi.lib().cutie_last_error()


# ------------------------------------------------------------------------------------------------------------------ group norm
# B 2, HW 4, C 8 f32, 2 groups: rows of 32 bytes, 64 apart (ld 16): a view covers 64 * 7 + 32 = 480 bytes; stats 32, vectors 32
def gn_fwd(HW=4, **kw):
    a = dict(x=FAR[0], gamma=FAR[1], beta=FAR[2], y=FAR[3], stats=FAR[4], ws=FAR[5])
    a.update(kw)
    return capi.lib().cutie_gn_fwd(A(a["x"]), 16, A(a["gamma"]), A(a["beta"]), 2, 1e-5, 0, A(a["y"]), 16, 0, A(a["stats"]), 2, HW, 8,
                                   A(a["ws"]), 1 << 30, None)


def gn_bwd(**kw):
    a = dict(dy=FAR[0], x=FAR[1], gamma=FAR[2], beta=FAR[3], stats=FAR[4], dx=FAR[5], dgamma=FAR[6], dbeta=FAR[7], ws=FAR[8], B=2)
    a.update(kw)
    return capi.lib().cutie_gn_bwd(A(a["dy"]), 16, A(a["x"]), 16, A(a["gamma"]), A(a["beta"]), 2, 0, A(a["stats"]), A(a["dx"]), 16, 0,
                                   A(a["dgamma"]), A(a["dbeta"]), 0, a["B"], 4, 8, A(a["ws"]), 1 << 20, None)


VIEW_OFFSETS = (-28, 0, 28, 64, 448 + 28, 32 + 4)      # the last one begins in a gap and runs into the next row


@pytest.mark.parametrize("off", VIEW_OFFSETS)
@pytest.mark.parametrize("view", ["x", "y"])
def test_group_norm_forward_statistics_over_a_view(view, off):
    assert refused(gn_fwd(stats=FAR[0 if view == "x" else 3] + off))


@pytest.mark.parametrize("kw", [dict(stats=FAR[1] + 28), dict(stats=FAR[2] - 28), dict(gamma=FAR[3] + 64), dict(beta=FAR[3] - 4)])
def test_group_norm_forward_vectors(kw):
    assert refused(gn_fwd(**kw))


@pytest.mark.parametrize("over", ["x", "y", "gamma", "beta", "stats"])
def test_group_norm_forward_workspace(over):
    """the form that goes through the workspace"""
    assert refused(gn_fwd(HW=1 << 20, **{over: FAR[5] + 64}))


@pytest.mark.parametrize("off", VIEW_OFFSETS)
@pytest.mark.parametrize("view", ["dy", "x", "dx"])
@pytest.mark.parametrize("out", ["dgamma", "dbeta"])
def test_group_norm_backward_vectors_over_a_view(out, view, off):
    at = dict(dy=FAR[0], x=FAR[1], dx=FAR[5])
    assert refused(gn_bwd(**{out: at[view] + off}))


@pytest.mark.parametrize("out", ["dgamma", "dbeta"])
@pytest.mark.parametrize("other", ["gamma", "beta", "stats"])
def test_group_norm_backward_vectors(out, other):
    at = dict(gamma=FAR[2], beta=FAR[3], stats=FAR[4])
    assert refused(gn_bwd(**{out: at[other] + 28})) and refused(gn_bwd(**{out: at[other]}))
    assert refused(gn_bwd(**{other: FAR[5] + 64}))      # dx over it


def test_group_norm_backward_one_gradient_twice():
    assert refused(gn_bwd(dgamma=FAR[7])) and refused(gn_bwd(dbeta=FAR[6] + 28)) and refused(gn_bwd(dgamma=FAR[7], B=0))


@pytest.mark.parametrize("over", ["dy", "x", "gamma", "beta", "stats", "dx", "dgamma", "dbeta"])
def test_group_norm_backward_workspace(over):
    assert refused(gn_bwd(**{over: FAR[8] + 64}))


@pytest.mark.gpu
def test_group_norm_neighbours_are_taken():
    """statistics and gradients in the gaps between the rows of the views"""
    wide = torch.randn(2, 4, 1, 16, generator=torch.Generator().manual_seed(1)).to("cuda:0")
    x, dy = wide[..., :8].clone(), wide[..., 8:].clone()
    y, st, dx, dg, db = torch.empty_like(x), torch.empty(2, 2, 2, device="cuda:0"), torch.empty_like(x), torch.empty(8, device="cuda:0"), torch.empty(8, device="cuda:0")
    ops.gn_fwd(x, y, st)
    ops.gn_bwd(dy, x, st, dx, dgamma=dg, dbeta=db)
    s2 = wide.view(-1)[8:16].view(2, 2, 2)      # the gap behind the first row
    ops.gn_fwd(wide[..., :8], dx.clone(), s2)
    assert torch.equal(s2, st)
    g2, b2, out = wide.view(-1)[24:32], wide.view(-1)[40:48], torch.empty_like(dx)
    ops.gn_bwd(dy, wide[..., :8], st, out, dgamma=g2, dbeta=b2)
    assert torch.equal(out, dx) and torch.equal(g2, dg) and torch.equal(b2, db)


# ------------------------------------------------------------------------------------------------------------------ embedding
# 4 cells, rows of 8 f32 (32 bytes) 64 apart; a table of 3 x 8 (96 bytes), ids 16 bytes
def lookup(**kw):
    a = dict(ids=FAR[0], table=FAR[1], out=FAR[2], oob=FAR[3])
    a.update(kw)
    return capi.lib().cutie_embed_scaled_fwd(A(a["ids"]), 4, A(a["table"]), 3, 8, 1.0, A(a["out"]), 16, 0, A(a["oob"]), None)


def gradient(n=4, **kw):
    a = dict(ids=FAR[0], dout=FAR[1], dtable=FAR[2], ws=FAR[3])
    a.update(kw)
    return capi.lib().cutie_embed_grad_sorted(A(a["ids"]), n, A(a["dout"]), 16, 0, 1.0, A(a["dtable"]), 3, 8, 0, A(a["ws"]), 1 << 20, None)


@pytest.mark.parametrize("kw", [dict(ids=FAR[2] + 64), dict(ids=FAR[2] - 12), dict(table=FAR[2]), dict(table=FAR[2] - 92), dict(table=FAR[2] + 32),
                                dict(oob=FAR[2] + 28), dict(oob=FAR[0] + 12), dict(oob=FAR[1] + 92)])
def test_lookup(kw):
    assert refused(lookup(**kw))


@pytest.mark.parametrize("kw", [dict(dtable=FAR[0] + 12), dict(dtable=FAR[0] - 92), dict(dtable=FAR[1]), dict(dtable=FAR[1] + 32), dict(dtable=FAR[1] + 192 + 28),
                                dict(ids=FAR[3] + 16), dict(dout=FAR[3] + 16), dict(dtable=FAR[3] + 16), dict(dout=FAR[3] - 64)])
def test_gradient(kw):
    assert refused(gradient(**kw))


@pytest.mark.gpu
def test_embedding_neighbours_are_taken():
    """the gradient's table as columns beside the rows it is made from: a table of one row in one gap"""
    wide = torch.randn(4, 16, generator=torch.Generator().manual_seed(2)).to("cuda:0")
    ids = torch.tensor([0, 1, 0, -1], dtype=torch.int32, device="cuda:0")
    want = wide[0, :8] + wide[2, :8]
    got = wide[1:2, 8:]
    assert ops.embed_grad_sorted(ids, wide[:, :8], got) is got and torch.equal(got[0], want)
    oob = wide[3, 8:9].view(torch.int32)
    oob.zero_()
    ops.embed_scaled_fwd(ids, got, wide[:, :8], 2.0, oob)
    assert torch.equal(wide[0, :8], 2 * want) and torch.equal(wide[2, :8], 2 * want) and int(oob) == 2 and not wide[1, :8].any()


# ------------------------------------------------------------------------------------------------------------------ the update
def muon(scalars, ws=1 << 20, at=4096):
    d = capi.MuonDesc()
    d.p, d.g, d.m, d.p_out, d.m_out = (at + 1024 * k for k in range(5))
    d.rows, d.cols, d.out_scale = 16, 16, 1.0      # 1024 bytes each
    a = dict(gnorm_sq=FAR[0], loss_scale=FAR[1], invalid=FAR[2])
    a.update(scalars)
    return capi.lib().cutie_muon_step(ctypes.byref(d), 1, 0.1, 0.9, 1, 0.0, 0.0, 5, 1e-7, A(a["gnorm_sq"]), 1.0, 1.0, A(a["loss_scale"]),
                                      A(a["invalid"]), A(ws), 1 << 40, None)


@pytest.mark.parametrize("name", ["gnorm_sq", "loss_scale", "invalid"])
@pytest.mark.parametrize("off", [3 * 1024, 3 * 1024 + 1020, 4 * 1024, 5 * 1024 - 4])
def test_update_over_what_it_is_steered_by(name, off):
    assert refused(muon({name: 4096 + off}))


def test_update_workspace():
    for k in range(5):
        assert refused(muon({}, at=(1 << 20) - 1024 * k + 128 if k else (1 << 20) + 128))
    for name, size in (("gnorm_sq", 4), ("loss_scale", 8), ("invalid", 4)):
        assert refused(muon({name: (1 << 20) + 4})) and refused(muon({name: (1 << 20) + 4 - size}))


@pytest.mark.parametrize("g,out", [((1 << 20) + 128, FAR[0]), (FAR[0], (1 << 20) + 128), (FAR[0], (1 << 20) - 64)])
def test_orthogonalize_workspace(g, out):
    d = capi.OrthDesc()
    d.g, d.out, d.rows, d.cols = g, out, 16, 16
    assert refused(capi.lib().cutie_orthogonalize_batched(ctypes.byref(d), 1, 5, 1e-7, A(1 << 20), 1 << 40, None))
