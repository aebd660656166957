"""Calls of the orthogonalised update: matrices in a tuple."""
import pytest
import torch

import test_training_operators_gpu as base
from cutie_amd import capi, ops


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
