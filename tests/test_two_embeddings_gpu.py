"""A graph with two embeddings of the grid: tables of different sizes, one of them scaled, under both forms of the gradient.  Each
takes its own work area, and the clip norm counts the rows of both.  The reference is the same network in f64, with the bounds of the
other networks (test_training_operators_gpu.py: f32 gradients 1e-3 in relative 2-norm, f16 3e-2).
"""
import types

import pytest
import torch

import test_training_operators_gpu as base
from cutie_amd.model_cutie import CUTIE
from oracle import cutie_oracle as co

V, C, B = base.V, base.C, base.B


class TwoNet(CUTIE):
    def __init__(self, large, small):
        """large, small: (rows, columns, factor); the backward pass meets the one named second first"""
        self.name = "two"
        self.large, self.small = large, small
        self._init_common(V, C, types.SimpleNamespace(embedding_size=64, weight_decay=5e-4, hard_negative_ratio=3, batch_size=B), True)
        self.setup()
        self.build_loss()

    def setup(self):
        for name, (rows, cols, scale) in (("large", self.large), ("small", self.small)):
            self.feed("data_grid").embed(rows, cols, name=name, scale=scale)
        (self.feed("large", "small").concat(3, name="cat").conv(1, 1, 64, 1, 1, name="i1")
             .conv(1, 1, C, 1, 1, name="cls_logits").softmax(name="softmax"))


def reference(net, params, grid, labels, weight, masks):
    ps = {k: v.clone().requires_grad_(True) for k, v in params.items()}
    rows = {k: ps[k + "/weights"][grid] * s for k, s in (("large", net.large[2]), ("small", net.small[2]))}
    for t in rows.values():
        t.retain_grad()
    x = co.cbrn(torch.cat([rows["large"], rows["small"]], dim=3), ps["i1/weights"], ps["i1/biases"], mask=masks["i1"])
    x = co.cbrn(x, ps["cls_logits/weights"], ps["cls_logits/biases"], mask=masks["cls_logits"])
    loss = (co.softmax_ce(x.reshape(-1, C), labels.reshape(-1)) * weight).sum()
    (loss + 5e-4 * sum((ps[s.name] ** 2).sum() / 2 for s in net.param_specs if s.regularized)).backward()
    return {k: v.grad for k, v in ps.items()}, {k: t.grad for k, t in rows.items()}


@pytest.mark.gpu
@pytest.mark.parametrize("embed_grad", ["sorted", "atomic"])
@pytest.mark.parametrize("large,small", [
    ((3 * V, 128, 1.0), (V, 64, 1.0)),      # the larger work area is asked for second
    ((3 * V, 128, 2.5), (V, 64, 1.0)),      # one scaled, one not
    ((3 * V, 128, 1.0), (V, 64, -0.5)),
    ((V, 64, 3.0), (3 * V, 128, 0.25)),
])
@pytest.mark.parametrize("dtype,gtol", [("f32", 1e-3), ("f16", 3e-2)])
def test_gradients_and_norm(large, small, embed_grad, dtype, gtol):
    net = TwoNet(large, small)
    grid, labels = base.inputs(9)
    params = base.params64(net)
    eng = base.engine(net, dtype, embed_grad=embed_grad)
    eng.load_params(params)
    P = eng.forward(grid.unsqueeze(-1), labels=labels)
    eng.check_inputs(P)
    eng.loss_backward(P)
    grads, rows = reference(net, params, grid, labels, P.weight.double().cpu(),
                            {k: eng.relu_mask(P, k).double().cpu() for k in ("i1", "cls_logits")})
    for k, want in grads.items():
        assert base.rel2(eng.grads[k], want) < gtol, (k, base.rel2(eng.grads[k], want))
    share = sum(s ** 2 * float((rows[k] ** 2).sum()) for k, s in (("large", large[2]), ("small", small[2])))
    want = share + sum(float((grads[k] ** 2).sum()) for k in grads if k not in ("large/weights", "small/weights"))
    assert abs(float(eng.embedding_rows_sumsq(P)) - share) < 2 * gtol * share
    assert abs(float(eng.global_norm_sq(P)) - want) < 2 * gtol * want
    # and what the optimizer clips by
    P = eng.forward(grid.unsqueeze(-1), labels=labels)
    eng.loss_backward(P, defer_l2=True)
    m, v = torch.zeros_like(eng.params_flat), torch.zeros_like(eng.params_flat)
    assert abs(float(eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0, t=1)) - want) < 2 * gtol * want
    assert not eng.grads_flat[eng.n_dense:].any()      # cleared behind itself, both tables


@pytest.mark.gpu
def test_before_any_backward_pass_the_rows_count_nothing():
    eng = base.engine(TwoNet((V, 64, 1.0), (V, 64, 2.0)), "f16")
    grid, labels = base.inputs(9)
    P = eng.forward(grid, labels=labels)
    assert float(eng.embedding_rows_sumsq(P)) == 0.0
