"""The network of test_training_operators_gpu.py (scaled embedding with its sorted gradient, group-normalised layers, the orthogonalised
update) in the engine's other modes: bf16, weight gradients on a second stream, and a train step of two ranks.

bf16 bounds are the framework's own for that type (test_model_gpu.py: 6e-2 on a layer, 1e-1 on gradients and norms).
"""
import math

import pytest
import torch

import test_training_operators_gpu as base
from cutie_amd.train import Trainer

pytestmark = pytest.mark.gpu
DEV, B = base.DEV, base.B


def test_bf16_graph_matches_f64():
    net = base.SmallNet()
    grid, labels = base.inputs()
    params = base.params64(net)
    eng = base.engine(net, "bf16")
    eng.load_params(params)
    P = eng.forward(grid.unsqueeze(-1), labels=labels)
    eng.check_inputs(P)
    eng.loss_backward(P)
    L, loss, reg, grads, d_emb = base.reference(net, params, grid, labels, P.weight.double().cpu(),
                                                {k: eng.relu_mask(P, k).double().cpu() for k in ("i1", "cls_logits")})
    for name in ("embedding", "g1", "g2", "i1", "d1", "cls_logits"):
        got, want = eng.get(P, name).double().cpu(), L[name].detach()
        assert float((got - want).abs().max() / want.abs().max()) < 6e-2, name
    for k, want in grads.items():
        assert base.rel2(eng.grads[k], want) < 1e-1, (k, base.rel2(eng.grads[k], want))
    want = sum(float((grads[k] ** 2).sum()) for k in grads if k != "embedding/weights") + base.SCALE ** 2 * float((d_emb ** 2).sum())
    assert abs(float(eng.global_norm_sq(P)) - want) < 2e-1 * want


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_weight_gradients_on_a_second_stream(dtype):
    """everything but the filters' gradients comes from the same launches: the same bits.  Those are summed layer by layer, in other
    parts: equal to the rounding of f32 sums of 1920 products, 1920 * 2^-24 of their magnitudes at most"""
    grid, labels = base.inputs(11)
    got = []
    for overlap in (False, True):
        net = base.SmallNet()
        eng = base.engine(net, dtype, overlap_wgrad=overlap)
        eng.load_params(base.params64(net))
        for _ in range(2):
            P = eng.forward(grid, labels=labels)
            eng.loss_backward(P)
        torch.cuda.synchronize()
        got.append({k: v.clone() for k, v in eng.grads.items()})
    for k in got[0]:
        if k.endswith("/weights") and k != "embedding/weights":
            assert base.rel2(got[1][k], got[0][k]) < 1e-4, k
        else:
            assert torch.equal(got[0][k], got[1][k]), k


class _Done(object):
    def wait(self):
        return True


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_two_ranks_with_the_orthogonalised_update(monkeypatch, dtype):
    """dist.all_reduce is replaced by a stub that records a rank's buffers or adds the other rank's recorded ones.  Nothing in this
    network adds in an order of its own (the embedding's gradient is sorted), so the replicas hold the same bits after every step;
    and a step is the formula on the two shards' raw gradients, each from an engine of its own."""
    import torch.distributed as dist
    from cutie_amd import train
    shards = [base.inputs(50 + r) for r in range(2)]
    mode = {"store": None, "k": None}

    def all_reduce(t, op=None, group=None, async_op=False):
        if mode["k"] is None:
            mode["store"].append(t.clone())
        else:
            t.add_(mode["store"][mode["k"]])
            mode["k"] += 1
        return _Done()

    monkeypatch.setattr(dist, "all_reduce", all_reduce)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "nccl")

    def make(rank):
        net = base.SmallNet()
        eng = base.engine(net, dtype)
        eng.load_params(base.params64(net))
        monkeypatch.setattr(train, "dist_info", lambda: (rank, 2))
        return Trainer(eng, learning_rate=1e-3, clip_norm=0.5, optimizer="muon", muon_lr=0.01, muon_weight_decay=0.02, gc_freeze=False)

    def batch(r):
        return {"grid_table": shards[r][0].unsqueeze(-1), "gt_classes": shards[r][1]}

    ranks, scratch = [make(0), make(1)], make(0)
    raw_net = base.SmallNet()
    raw_eng = base.engine(raw_net, dtype)
    for step in range(3):
        sent = []
        for r in range(2):      # what rank r sends: its step on the scratch engine, from the replicas' common state
            s, src = scratch, ranks[0]
            s.eng.params_flat.copy_(src.eng.params_flat)
            s.eng.repack()
            s.m.copy_(src.m)
            s.v.copy_(src.v)
            s.eng.opt_state.copy_(src.eng.opt_state)
            s.t, s.iter = src.t, src.iter
            mode.update(store=[], k=None)
            s.step(batch(r), fetch=False)
            sent.append(mode["store"])
        # the raw gradients of the two shards, without hook or collective
        raw_eng.params_flat.copy_(ranks[0].eng.params_flat)
        raw_eng.repack()
        raw_eng.opt_state.copy_(ranks[0].eng.opt_state)
        raw, rows = torch.zeros_like(raw_eng.grads_flat), 0.0
        for r in range(2):
            P = raw_eng.forward(shards[r][0], labels=shards[r][1])
            raw_eng.loss_backward(P, defer_l2=True)
            raw += raw_eng.grads_flat
            rows += float(raw_eng.embedding_rows_sumsq(P))
        S = raw_eng.loss_scale_value()[0] if dtype == "f16" else 1.0
        p0, m0 = ranks[0].eng.params_flat.clone(), ranks[0].m.clone()
        outs = []
        for r in range(2):
            mode.update(store=sent[1 - r], k=0)
            outs.append(ranks[r].step(batch(r)))
            assert mode["k"] == len(sent[1 - r]) and math.isfinite(outs[-1]["total_loss"])
        a, b = ranks[0], ranks[1]
        assert torch.equal(a.eng.params_flat, b.eng.params_flat) and torch.equal(a.m, b.m) and torch.equal(a.v, b.v), step
        assert outs[0]["global_norm"] == outs[1]["global_norm"]
        # the norm of the mean gradient, L2 terms and the embedding's rows in it
        dense = raw[:raw_eng.n_dense].double() / S
        dense[:raw_eng.n_conv_w] += 2 * 5e-4 * p0[:raw_eng.n_conv_w].double()
        gn = math.sqrt(float((dense ** 2).sum()) + rows)
        assert abs(outs[0]["global_norm"] - gn / 2) < 1e-3 * gn
        for k in raw_eng.conv_w_names:
            if k == "cls_logits/weights":
                continue
            off, n, shape = raw_eng.offsets[k]
            cut = lambda t: t[off:off + n].double().cpu().view(-1, shape[-1])
            g = cut(dense) * 0.5 * (0.5 / max(gn / 2, 0.5))
            p, mom = cut(p0), 0.95 * cut(m0) + g
            # the batched weight-gradient calls of a data-parallel step cut K otherwise than one call: f32 rounding of the sums
            assert float((cut(a.m) - mom).norm()) <= 1e-4 * float(mom.norm()), k
            u = g + 0.95 * cut(a.m)
            scale = 0.01 * math.sqrt(max(1.0, shape[-1] / (n // shape[-1])))
            moved = (cut(a.eng.params_flat) - p * (1 - 0.01 * 0.02)) / scale
            want = base.quintic(u)
            # small singular values are raised by up to 3.4445^5 = 485: 485 * 1e-4 of the smallest, seen against the whole
            assert float((moved + want).norm()) <= 2e-2 * float(want.norm()), (k, float((moved + want).norm() / want.norm()))
