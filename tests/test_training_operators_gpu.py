"""The scaled embedding with its sorted gradient, group-normalised layers and the orthogonalised update together, as a graph
and a train step use them: a small network against the same network in f64 (forward, losses, every gradient), one optimizer
step against the formula, skipped steps, and two runs bit for bit.

Bounds are those the framework's own layers are held to (test_model_gpu.py): f32 every layer within 1e-4 of the largest value,
gradients 1e-3 in relative 2-norm; f16 2e-2 and 3e-2.
"""
import math
import types

import pytest
import torch

from cutie_amd.model_cutie import CUTIE
from oracle import cutie_oracle as co

DEV = "cuda:0"
V, E, C, B, H, W = 400, 64, 18, 2, 24, 40
SCALE = math.sqrt(E)


class SmallNet(CUTIE):
    """embedding * scale -> two group-normalised layers -> an instance-normalised one -> concat -> decoder -> logits"""

    def __init__(self, scale=SCALE, g2_act="silu"):
        self.name = "small"
        self.scale, self.g2_act = scale, g2_act
        p = types.SimpleNamespace(embedding_size=E, weight_decay=5e-4, hard_negative_ratio=3, batch_size=B)
        self._init_common(V, C, p, True)
        self.setup()
        self.build_loss()

    def setup(self):
        (self.feed("data_grid").embed(V, E, name="embedding", scale=self.scale)
             .conv(3, 5, 128, 1, 1, name="g1", norm="group", groups=16, activation="silu")
             .dilate_conv(3, 5, 128, 1, 1, 2, name="g2", norm="group", groups=2, activation=self.g2_act)
             .conv(1, 1, 64, 1, 1, name="i1"))
        (self.feed("g1", "i1").concat(3, name="cat")
             .conv(3, 5, 64, 1, 1, name="d1", norm="group", groups=64, activation="none")
             .conv(1, 1, C, 1, 1, name="cls_logits").softmax(name="softmax"))


def inputs(seed=3):
    g = torch.Generator().manual_seed(seed)
    grid = torch.zeros((B, H, W), dtype=torch.int64)
    occ = torch.rand((B, H, W), generator=g) < 0.2
    grid[occ] = torch.randint(1, V, (int(occ.sum()),), generator=g)
    labels = torch.zeros((B, H, W), dtype=torch.int64)
    fg = occ & (torch.rand((B, H, W), generator=g) < 0.4)
    labels[fg] = torch.randint(1, C, (int(fg.sum()),), generator=g)
    return grid, labels


def params64(net, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = {}
    for s in net.param_specs:
        t = torch.randn(s.shape, generator=g, dtype=torch.float64)
        if s.name.endswith("/gamma"):
            t = 1 + 0.2 * t
        elif len(s.shape) == 4:
            t = t / math.sqrt(s.shape[0] * s.shape[1] * s.shape[2])
        else:
            t = 0.2 * t
        out[s.name] = t.float().double()
    return out


def group_norm(x, groups, gamma, beta, act):
    b, h, w, c = x.shape
    xg = x.reshape(b, h * w, groups, c // groups)
    mean = xg.mean(dim=(1, 3), keepdim=True)
    var = ((xg - mean) ** 2).mean(dim=(1, 3), keepdim=True)
    z = ((xg - mean) / torch.sqrt(var + 1e-5)).reshape(x.shape) * gamma + beta
    return {"silu": z * torch.sigmoid(z), "relu": torch.relu(z), "none": z, "sigmoid": torch.sigmoid(z)}[act]


def reference(net, params, grid, labels, weight, masks):
    """weight: the device's weight of each cell's cross-entropy (its hard-negative selection); masks: its ReLU patterns.  Both are
    steps: a logit or a pre-activation that 16 bits round across one changes a gradient by a whole cell, which says nothing about
    the gradient kernels (test_model_gpu.py gives its oracle both for the same reason)."""
    ps = {k: v.clone().requires_grad_(True) for k, v in params.items()}
    L = {"embedding": ps["embedding/weights"][grid] * net.scale}

    def grouped(x, name, rate=1):
        a = net.layers[name].attrs
        return group_norm(co.conv_raw(x, ps[name + "/weights"], rate), a["groups"], ps[name + "/gamma"], ps[name + "/beta"], a["activation"])
    L["g1"] = grouped(L["embedding"], "g1")
    L["g2"] = grouped(L["g1"], "g2", 2)
    L["i1"] = co.cbrn(L["g2"], ps["i1/weights"], ps["i1/biases"], mask=masks["i1"])
    L["d1"] = grouped(torch.cat([L["g1"], L["i1"]], dim=3), "d1")
    L["cls_logits"] = co.cbrn(L["d1"], ps["cls_logits/weights"], ps["cls_logits/biases"], mask=masks["cls_logits"])
    L["embedding"].retain_grad()
    ce = co.softmax_ce(L["cls_logits"].reshape(-1, C), labels.reshape(-1))
    loss = (ce * weight).sum()
    reg = 5e-4 * sum((ps[s.name] ** 2).sum() / 2 for s in net.param_specs if s.regularized)
    (loss + reg).backward()
    return L, float(loss.detach()), float(reg.detach()), {k: v.grad for k, v in ps.items()}, L["embedding"].grad


def engine(net, dtype, **kw):
    from cutie_amd.runtime import Engine
    return Engine(net, DEV, dtype=dtype, seed=0, **kw)


def rel2(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return float((a - b).norm() / b.norm().clamp_min(1e-300))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol,gtol", [("f32", 1e-4, 1e-3), ("f16", 2e-2, 3e-2)])
def test_graph_matches_f64(dtype, tol, gtol):
    net = SmallNet()
    grid, labels = inputs()
    params = params64(net)
    eng = engine(net, dtype)
    eng.load_params(params)
    P = eng.forward(grid.unsqueeze(-1), labels=labels)
    eng.check_inputs(P)
    eng.loss_backward(P)
    L, loss, reg, grads, d_emb = reference(net, params, grid, labels, P.weight.double().cpu(),
                                           {k: eng.relu_mask(P, k).double().cpu() for k in ("i1", "cls_logits")})
    if dtype == "f32":      # the selection itself, where nothing is rounded across its step
        w = co.hnm_loss(co.softmax_ce(L["cls_logits"].detach().reshape(-1, C), labels.reshape(-1)), labels, 3)[1]
        assert float((P.weight.double().cpu() - w).abs().max()) < 1e-6
    for name in ("embedding", "g1", "g2", "i1", "d1", "cls_logits"):
        got, want = eng.get(P, name).double().cpu(), L[name].detach()
        assert float((got - want).abs().max() / want.abs().max()) < tol, name
    got_loss = eng.losses(P)
    assert abs(got_loss[0] - loss) < tol * abs(loss) and abs(got_loss[1] - reg) < 1e-5 * reg
    for k, want in grads.items():
        assert rel2(eng.grads[k], want) < gtol, (k, rel2(eng.grads[k], want))
    # tf.clip_by_global_norm's norm: the embedding through its un-deduplicated rows, each scale times the gradient of the row
    dense = sum(float((grads[k] ** 2).sum()) for k in grads if k != "embedding/weights")
    want = dense + SCALE ** 2 * float((d_emb ** 2).sum())
    assert abs(float(eng.global_norm_sq(P)) - want) < 2 * gtol * want


@pytest.mark.gpu
def test_inference_equals_training_forward():
    net = SmallNet(g2_act="sigmoid")
    eng = engine(net, "f32")
    grid, labels = inputs(5)
    a = eng.get(eng.forward(grid, labels=labels), "cls_logits").clone()
    assert torch.equal(a, eng.get(eng.forward(grid), "cls_logits"))


@pytest.mark.gpu
def test_sorted_gradient_of_an_unscaled_embedding():
    """Engine(embed_grad='sorted') on a graph of the reference's: the same gradient as the atomic form to rounding, and the
    same bits run after run"""
    net = SmallNet(scale=1.0)
    grid, labels = inputs(6)
    got = []
    for kind in ("sorted", "sorted", "atomic"):
        eng = engine(net, "f16", embed_grad=kind)
        P = eng.forward(grid, labels=labels)
        eng.loss_backward(P)
        got.append(eng.grads["embedding/weights"].clone())
    assert torch.equal(got[0], got[1])
    # both add the same f32 rows, 2000 at most for one id: 2000 u of the sum of magnitudes, u = 2^-24, and the rows of one id
    # differ in sign and size (their sum is at least a hundredth of their magnitudes in 2-norm over the table)
    assert rel2(got[0], got[2]) < 2000 * 2.0 ** -24 * 100


def quintic(u, steps=5):
    x = u.double()
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        a = x.t() @ x if x.shape[0] >= x.shape[1] else x @ x.t()
        b = -4.7750 * a + 2.0315 * a @ a
        x = 3.4445 * x + (x @ b if x.shape[0] >= x.shape[1] else b @ x)
    return x


HP = {"lr": 0.02, "momentum": 0.95, "nesterov": True, "weight_decay": 0.01, "steps": 5}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_update_step(dtype):
    from cutie_amd import ops
    net = SmallNet()
    grid, labels = inputs(7)
    g = torch.Generator().manual_seed(1)
    runs = []
    for muon in (HP, None):
        eng = engine(net, dtype)
        eng.load_params(params64(net))
        m, v = torch.zeros_like(eng.params_flat), torch.zeros_like(eng.params_flat)
        for k in eng.params:
            eng._view(m, k).copy_(1e-3 * torch.randn(eng.params[k].shape, generator=g.manual_seed(1)))
        P = eng.forward(grid, labels=labels)
        eng.loss_backward(P, defer_l2=True)
        raw, p0, m0 = eng.grads_flat.clone(), eng.params_flat.clone(), m.clone()
        gn = float(eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0, t=1, muon=muon))
        runs.append((eng, m, v, raw, p0, m0, gn))
    (eng, m, v, raw, p0, m0, gn), other = runs
    assert torch.equal(raw, other[3]) and gn == other[6]
    S = eng.loss_scale_value()[0] if dtype == "f16" else 1.0
    conv = [k for k in eng.conv_w_names if k != "cls_logits/weights"]
    for k in eng.params:
        if k not in conv:      # Adam's share is what it was
            assert torch.equal(eng.params[k], other[0].params[k]), k
            assert torch.equal(eng._view(m, k), other[0]._view(other[1], k)), k
            continue
        off, n, shape = eng.offsets[k]
        cut = lambda t: t[off:off + n].double().cpu().view(-1, shape[-1])
        p, grad, mom = cut(p0), cut(raw), cut(m0)
        grad = (grad / S + 5e-4 * p) * (1.0 / max(math.sqrt(gn), 1.0))
        mom1 = 0.95 * mom + grad
        # f32 elementwise: four roundings of the magnitudes added
        assert bool(((cut(m) - mom1).abs() <= 8 * 2.0 ** -24 * (0.95 * mom.abs() + grad.abs() + 1e-12)).all()), k
        step = quintic(grad + 0.95 * mom1) * 0.02 * math.sqrt(max(1.0, shape[-1] / (n // shape[-1])))
        want = p * (1 - 0.02 * 0.01) - step
        # the orthogonalised matrix is held to f32's own error on it (test_muon_gpu.py, below 2e-5 of its norm), p to 4 roundings
        assert float((cut(eng.params_flat) - want).norm()) <= 2e-5 * float(step.norm()) + 4 * 2.0 ** -24 * float(p.norm()), k
        assert not eng._view(v, k).any()
    for k in eng.conv_w_names:      # operands are the pack of the new kernels
        wf, wd = ops.pack_weights(eng.params[k].contiguous(), eng.dt)
        assert torch.equal(eng.w_fwd[k], wf) and torch.equal(eng.w_dg[k], wd), k


@pytest.mark.gpu
def test_invalid_step_changes_nothing():
    net = SmallNet()
    eng = engine(net, "f16")
    grid, labels = inputs(8)
    m, v = torch.zeros_like(eng.params_flat), torch.zeros_like(eng.params_flat)
    P = eng.forward(grid, labels=labels)
    eng.loss_backward(P, defer_l2=True)
    P.late.fill_(1)
    p0, packed = eng.params_flat.clone(), {k: t.clone() for k, t in eng.w_fwd.items()}
    eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0, t=1, muon=HP)
    assert torch.equal(eng.params_flat, p0) and not m.any() and eng.steps_invalid() == 1
    assert all(torch.equal(eng.w_fwd[k], t) for k, t in packed.items())
    P = eng.forward(grid, labels=labels)      # an overflow: the loss scale made infinite gradients
    eng.loss_backward(P, defer_l2=True)
    eng.grads["g1/weights"][0, 0, 0, 0] = float("inf")
    eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0, t=2, muon=HP)
    assert torch.equal(eng.params_flat, p0) and not m.any()


@pytest.mark.gpu
def test_trainer_runs_the_same_twice():
    from cutie_amd.train import Trainer
    got = []
    for _ in range(2):
        net = SmallNet()
        eng = engine(net, "f16")
        tr = Trainer(eng, learning_rate=1e-3, optimizer="muon", muon_lr=0.01, gc_freeze=False)
        for k in range(4):
            grid, labels = inputs(20 + k)
            out = tr.step({"grid_table": grid.unsqueeze(-1), "gt_classes": labels})
            assert math.isfinite(out["total_loss"]) and math.isfinite(out["global_norm"])
        got.append(eng.params_flat.clone())
    assert bool(torch.isfinite(got[0]).all()) and torch.equal(got[0], got[1])


@pytest.mark.gpu
def test_cutie_aspp_with_the_orthogonalised_update():
    """the reference's graph under Trainer(optimizer='muon'): every filter but the logits layer's moves by about muon_lr times
    the 2-norm of an orthogonal matrix of its shape"""
    from cutie_amd.model_cutie_aspp import CUTIERes
    from cutie_amd.train import Trainer
    p = types.SimpleNamespace(embedding_size=E, weight_decay=5e-4, hard_negative_ratio=3, batch_size=B)
    net = CUTIERes(V, C, p)
    net.build_loss()
    eng = engine(net, "f16")
    before = {k: eng.params[k].clone() for k in eng.conv_w_names}
    grid, labels = inputs(30)
    Trainer(eng, optimizer="muon", muon_lr=0.01, gc_freeze=False).step({"grid_table": grid.unsqueeze(-1), "gt_classes": labels})
    for k in eng.conv_w_names:
        if k == "cls_logits/weights":
            continue
        w = eng.params[k]
        rows, cols = w.numel() // w.shape[-1], w.shape[-1]
        moved = float((w - before[k]).norm()) / (0.01 * math.sqrt(max(1.0, cols / rows)))
        # singular values after five steps lie in 0.68 .. 1.21 where they began above 1e-2 of the norm; smaller ones lag behind
        assert 0.05 * math.sqrt(min(rows, cols)) < moved < 1.21 * math.sqrt(min(rows, cols)) * 1.001, k


# ------------------------------------------------------------------------------------------------------------------ on the CPU
def test_graph_variables_and_refusals():
    net = SmallNet()
    shapes = {s.name: s.shape for s in net.param_specs}
    assert shapes["g1/gamma"] == (128,) and shapes["d1/beta"] == (64,) and "g1/biases" not in shapes and "i1/biases" in shapes
    assert net.layers["embedding"].attrs["scale"] == SCALE

    class Bad(SmallNet):
        def setup(self):
            self.feed("data_grid").embed(V, E, name="embedding").conv(3, 5, 64, 1, 1, name="x", **self.kw)

    for kw in (dict(norm="batch"), dict(norm="group", groups=7), dict(norm="group", groups=0), dict(norm="group", activation="gelu")):
        Bad.kw = kw
        with pytest.raises(ValueError):
            Bad()
    from cutie_amd.train import Trainer
    with pytest.raises(ValueError):
        Trainer(types.SimpleNamespace(params_flat=torch.zeros(1)), optimizer="sgd")


@pytest.mark.gpu
def test_engine_refusals():
    from cutie_amd.capi import CutieError

    class GroupLogits(SmallNet):
        def setup(self):
            (self.feed("data_grid").embed(V, E, name="embedding")
                 .conv(1, 1, C, 1, 1, name="cls_logits", norm="group", groups=2).softmax(name="softmax"))

    with pytest.raises(NotImplementedError):
        engine(GroupLogits(), "f16")
    with pytest.raises(CutieError):
        engine(SmallNet(), "f16", embed_grad="fast")

    class Pooled(SmallNet):
        def setup(self):
            (self.feed("data_grid").embed(V, E, name="embedding").conv(1, 1, 64, 1, 1, name="g", norm="group", groups=2)
                 .global_pool(name="pool").conv(1, 1, C, 1, 1, name="cls_logits").softmax(name="softmax"))
    eng = engine(Pooled(), "f16")
    grid, labels = inputs()
    P = eng.forward(grid, labels=labels)
    with pytest.raises(NotImplementedError):      # the pool's gradient vanishes behind an instance norm only
        eng.loss_backward(P)
    with pytest.raises(CutieError):
        eng.relu_mask(P, "g")
