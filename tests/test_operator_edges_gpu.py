"""Routing and packed attention where plain forms of their formulas lose everything: logits that are not finite, scores at
the ends of the sigmoid, query gradients under nearly uniform attention."""
import pytest
import torch

from oracle import ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -8


def native():
    from pippy_amd import _native
    return _native


def within(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    assert bool((err <= bound).all()), f"{what}: error exceeds its bound by {float((err - bound).max()):.3e}"


def selection(x, k, scoring, bias, n_group, topk_group, group_score):
    """The definition for rows with NaN and infinite logits, a token at a time: NaN ranks behind every number (in a group's
    score it counts as not there), lower indexes first, and infinite logits share all of the softmax."""
    T, E = x.shape
    out = torch.full((T, k), -1, dtype=torch.long)
    for t in range(T):
        row = x[t].double()
        known = ~row.isnan()
        num = torch.where(known, row, torch.full_like(row, float("-inf")))
        if scoring == "sigmoid":
            score = torch.sigmoid(row)
        elif bool((num == float("inf")).any()):
            score = (num == float("inf")).double() / (num == float("inf")).sum()
        else:
            score = torch.softmax(num, -1)
        there = row != float("-inf")
        choice = row if bias is None else score + bias.double()
        in_group = choice if group_score == "max" else score + (0 if bias is None else bias.double())
        order = sorted((e for e in range(E) if there[e] and known[e]), key=lambda e: (-float(choice[e]), e))
        order += [e for e in range(E) if not known[e]]
        if n_group > 1:
            rank = []
            for g in range(n_group):
                own = sorted((float(in_group[e]) for e in range(E) if there[e] and known[e] and e // (E // n_group) == g))
                own = own[-1:] if group_score == "max" else own[-2:]
                rank.append((-sum(own) if own else float("inf"), g))
            kept = {g for _, g in sorted(rank)[:topk_group]}
            order = [e for e in order if e // (E // n_group) in kept]
        out[t, :min(k, len(order))] = torch.tensor(order[:k])
    return out


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [True, False])
@pytest.mark.parametrize("E,k,groups", [(24, 4, 1), (24, 4, 4), (72, 5, 1), (72, 6, 9), (256, 8, 1), (256, 8, 8), (512, 12, 16)])
@pytest.mark.parametrize("group_score", ["max", "top2"])
def test_routing_ranks_a_nan_behind_every_number(scoring, biased, E, k, groups, group_score):
    N = native()
    g = torch.Generator().manual_seed(E + groups)
    x = torch.randn(12, E, generator=g)
    x[1, 3] = float("nan")
    x[2, ::2] = float("nan")
    x[3] = float("nan")
    x[4, E // 2] = float("inf")
    x[5, 5] = x[5, E - 2] = float("inf")
    x[6, 1] = float("inf")
    x[6, 2] = float("nan")
    x[7, 4] = float("-inf")
    x[7, 9] = float("nan")
    x[8, 2:] = float("nan")
    x[9, 2:] = float("nan")
    x[9, :2] = float("-inf")
    bias = torch.randn(E, generator=g) * 0.05 if biased else None
    how = dict(scoring=scoring, n_group=groups, topk_group=max(1, groups // 2), group_score=group_score)
    idx = torch.full((12, k), -7, dtype=torch.int32, device=DEV)
    gate = torch.full((12, k), -7.0, device=DEV)
    want = selection(x, k, bias=bias, **how)
    for renorm in (True, False):
        N.moe_route(x.to(DEV), idx, gate, bias=None if bias is None else bias.to(DEV), renorm=renorm, **how)
        assert torch.equal(idx.cpu().long(), want)
        clean = [0, 10, 11]
        assert bool(gate[clean].isfinite().all()) and bool((gate.cpu()[want < 0] == 0).all())
        hit = torch.gather(x, 1, want.clamp(min=0)).isnan() & (want >= 0)
        if scoring == "softmax":
            # renormalised weights are formed from the selected logits alone, the others from the whole row
            bad = hit.any(-1, keepdim=True) if renorm else x.isnan().any(-1, keepdim=True)
            bad = bad | (x == float("inf")).any(-1, keepdim=True)       # infinite ones are selected
            assert bool(gate.cpu()[(want >= 0) & bad].isnan().all())
        else:
            assert bool(gate.cpu()[hit].isnan().all())
