"""Calls of the orthogonalised update: matrices in a tuple, and a train step that is refused before anything of it is done."""
import types

import pytest
import torch

import test_training_operators_gpu as base
from cutie_amd import capi, ops
from cutie_amd.train import Trainer


@pytest.mark.parametrize("n", [1, 2, 3, 4])
def test_matrices_in_a_tuple_are_matrices(n):
    """(of three, one could be taken for a plan: descriptors, shapes, device) - host tensors are refused as such, not misread"""
    ents = tuple((torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6), torch.zeros(4, 6), 1.0) for _ in range(n))
    with pytest.raises(capi.CutieError, match="expected a device tensor"):
        ops.muon_step(ents, 0.1)


@pytest.mark.gpu
def test_tuple_and_list_are_the_same():
    g = torch.Generator().manual_seed(1)
    got = []
    for kind in (list, tuple):
        ents = [[torch.randn(40, 24, generator=g.manual_seed(k)).to(base.DEV) for k in range(3)] for _ in range(3)]
        ops.muon_step(kind((p, d, m, p, m, 1.0) for p, d, m in ents), 0.1)
        got.append([t for e in ents for t in (e[0], e[2])])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("kw", [dict(muon_steps=0), dict(muon_steps=33), dict(clip_norm=0.0), dict(clip_norm=-1.0), dict(clip_norm=float("nan"))])
def test_trainer_refuses(kw):
    with pytest.raises(ValueError):
        Trainer(types.SimpleNamespace(params_flat=torch.zeros(1)), optimizer="muon", **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("hp,clip", [(dict(base.HP, steps=0), 1.0), (dict(base.HP, steps=40), 1.0), (base.HP, 0.0)])
def test_refused_step_changes_nothing(hp, clip):
    eng = base.engine(base.SmallNet(), "f16")
    grid, labels = base.inputs(8)
    m, v = torch.zeros_like(eng.params_flat), torch.zeros_like(eng.params_flat)
    P = eng.forward(grid, labels=labels)
    eng.loss_backward(P, defer_l2=True)
    p0 = eng.params_flat.clone()
    with pytest.raises(ValueError):
        eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, clip, t=1, muon=hp)
    assert torch.equal(eng.params_flat, p0) and not m.any() and not v.any()
    eng.apply_update(P, m, v, 1e-3, 0.9, 0.999, 1e-8, 1.0, t=1, muon=base.HP)      # and the step can still be taken
    assert not torch.equal(eng.params_flat, p0)
