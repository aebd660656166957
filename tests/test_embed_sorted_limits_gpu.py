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
