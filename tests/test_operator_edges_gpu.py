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


@pytest.mark.parametrize("base", [-60.0, -82.0, -85.5, -88.5, -95.0, -300.0, -700.0])
@pytest.mark.parametrize("k", [1, 3, 8])
def test_renormalised_sigmoid_weights_of_small_scores(base, k):
    """Scores far below what fp32 holds still have ratios.  The weights are quotients of exponentials of differences up to
    4: 4 x 2^-24 from the difference, 2^-23 from every exponential, 2^-22 from sums and quotients, 2^-20 in all; a gradient is two
    such products, and the fp32 sum of g dgate before it (K terms, 2^-21 of its absolute values)."""
    N = native()
    T, E = 40, 32
    g = torch.Generator().manual_seed(k)
    x = base - 4 * torch.rand(T, E, generator=g)
    dgate = torch.randn(T, k, generator=g) * 1000
    idx = torch.empty(T, k, dtype=torch.int32, device=DEV)
    gate = torch.empty(T, k, device=DEV)
    N.moe_route(x.to(DEV), idx, gate, scoring="sigmoid", scale=1.5)
    xr = x.double().requires_grad_(True)
    want_idx, want = O.moe_route(xr, k, scoring="sigmoid", scale=1.5)
    assert torch.equal(idx.cpu().long(), want_idx)
    want = want.detach()
    assert float(want.sum(-1).min()) > 1.49
    within(gate, want, 2.0 ** -20 * want, "gate")
    dl = torch.empty(T, E, device=DEV)
    N.moe_route_bwd(x.to(DEV), idx, dl, dgate=dgate.to(DEV), scoring="sigmoid", scale=1.5)
    # d gate_k / d x_k = gate_k (1 - g_k) (1 - s_k), formed without the quotient s / sum s that autograd would take
    s1, w = torch.sigmoid(-x.double()).gather(1, want_idx), want / 1.5
    d = dgate.double()
    dx = 1.5 * (d - (w * d).sum(-1, keepdim=True)) * w * s1
    size = 1.5 * (d.abs() + (w * d.abs()).sum(-1, keepdim=True)) * w * s1
    wanted = torch.zeros(T, E, dtype=torch.float64).scatter(1, want_idx, dx)
    bound = torch.zeros(T, E, dtype=torch.float64).scatter(1, want_idx, 2.0 ** -18 * size)
    within(dl, wanted, bound, "dlogits")


def test_scores_that_64_bits_hold_as_zero_give_no_weight():
    """Logits at the lowest value of their type, as masks are written: the sum of the scores is 0, the weights are 0."""
    N = native()
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.full((3, 8), torch.finfo(dtype).min, dtype=dtype)
        x[1, 2] = -750.0
        x[2, 5] = -2.0
        idx = torch.empty(3, 2, dtype=torch.int32, device=DEV)
        gate = torch.empty(3, 2, device=DEV)
        N.moe_route(x.to(DEV), idx, gate, scoring="sigmoid")
        want_idx, want = O.moe_route(x.double(), 2, scoring="sigmoid")
        assert torch.equal(idx.cpu().long(), want_idx) and torch.equal(gate.cpu().double(), want)
        dl = torch.full((3, 8), 9.0, dtype=dtype, device=DEV)
        N.moe_route_bwd(x.to(DEV), idx, dl, dgate=torch.tensor([[1.0, 2.0]] * 3, device=DEV), scoring="sigmoid")
        assert bool((dl == 0).all())


@pytest.mark.parametrize("renorm", [True, False])
def test_sigmoid_gradient_of_large_logits(renorm):
    """1 - s is formed as the sigmoid of -x, not by subtraction from 1.  Relative errors: 2^-23 each from the exponential, the sum and
    the quotient of s and of 1 - s, 2^-20 with the sums over the slots."""
    N = native()
    T, E, k = 50, 16, 3
    g = torch.Generator().manual_seed(5)
    x = torch.rand(T, E, generator=g) * 40 + torch.linspace(-20, 40, T)[:, None]
    dgate = torch.randn(T, k, generator=g)
    idx, _ = O.moe_route(x.double(), k, scoring="sigmoid")
    s = torch.sigmoid(x.double()).gather(1, idx)
    rest = torch.sigmoid(-x.double()).gather(1, idx)
    d = dgate.double()
    if renorm:
        w = s / s.sum(-1, keepdim=True)
        dx = (d - (w * d).sum(-1, keepdim=True)) * w * rest
        size = (d.abs() + (w * d.abs()).sum(-1, keepdim=True)) * w * rest
    else:
        dx = d * s * rest
        size = dx.abs()
    dl = torch.empty(T, E, device=DEV)
    N.moe_route_bwd(x.to(DEV), idx.int().to(DEV), dl, dgate=dgate.to(DEV), scoring="sigmoid", renorm=renorm)
    zero = torch.zeros(T, E, dtype=torch.float64)
    within(dl, zero.scatter(1, idx, dx), zero.scatter(1, idx, 2.0 ** -20 * size), "dlogits")


@pytest.mark.parametrize("D,H,Hkv,cu", [(64, 2, 2, [0, 70, 326, 590]), (128, 4, 1, [0, 70, 326, 590]),
                                        (64, 32, 32, [0, 2000, 2100]), (128, 32, 8, [0, 2000, 2100])])
@pytest.mark.parametrize("causal", [False, True])
def test_query_gradient_under_nearly_uniform_attention_with_a_common_part(D, H, Hkv, cu, causal):
    """Keys and values that share a large part: the gradient of a query is a small difference.  The common part of the keys
    meets the sum of a row of dS, which is zero, so only the rounding of the terms of dS (2^-8 of each), fp32 noise of the
    products (2^-16 of P |dP| and of its row's sum) and the result's own rounding may reach dQ.  The error of the stored
    output, (2^-8 + 2^-8) P |V|, which is large beside dS, may not, but for products with a second rounding: that of dS, which
    holds it, and that of P in its correction, 4 x 2^-16 |dO| P |V| together."""
    N = native()
    T = cu[-1]
    g = torch.Generator().manual_seed(D + H + T)
    q = (torch.randn(T, H, D, generator=g) * 0.05).to(torch.bfloat16)
    common = torch.randn(2, 1, Hkv, D, generator=g) * 8
    k, v = (torch.randn(2, T, Hkv, D, generator=g) * 0.5 + common).to(torch.bfloat16).unbind(0)
    do = (torch.randn(T, H, D, generator=g) * 0.1).to(torch.bfloat16)
    qd, kd, vd, dod = (t.to(DEV) for t in (q, k, v, do))
    o, dq, dk, dv = torch.empty_like(qd), torch.empty_like(qd), torch.empty_like(kd), torch.empty_like(vd)
    lse, delta = (torch.empty(H, T, device=DEV) for _ in range(2))
    plan = N.attn_packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), T)
    N.attn_packed_fwd(qd, kd, vd, o, lse, plan, causal=causal)
    N.attn_packed_bwd(qd, kd, vd, o, lse, dod, dq, dk, dv, delta, plan, causal=causal)
    scale = D ** -0.5
    for a, b in zip(cu[:-1], cu[1:]):
        for h in range(0, H, max(1, H // 2)):
            Q, dO = q[a:b, h].double(), do[a:b, h].double()
            K, V = k[a:b, h * Hkv // H].double(), v[a:b, h * Hkv // H].double()
            S = Q @ K.T * scale
            if causal:
                S = S.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), float("-inf"))
            P = torch.softmax(S, -1)
            dP = dO @ V.T
            dS = P * (dP - (P * dP).sum(-1, keepdim=True))
            want = dS @ K * scale
            noise = P * (dP.abs() + (P * dP.abs()).sum(-1, keepdim=True))
            stored = P * (dO.abs() * (P @ V.abs())).sum(-1, keepdim=True)
            bound = scale * (U * dS.abs() + 2.0 ** -16 * noise + 2.0 ** -14 * stored) @ K.abs() + U * want.abs()
            within(dq[a:b, h], want, 1.02 * bound + 1e-30, "dq")


@pytest.mark.parametrize("n", [4096, 4097, 65536, 65537, 300000, 524288, 524289, 1048576, 1048577])
@pytest.mark.parametrize("E", [2, 250])
def test_permutation_on_either_side_of_its_borders(n, E):
    """Numbers of slots from which on a work-group takes more of them."""
    N = native()
    slots = torch.randint(-1, E, (n,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    kept = slots >= 0
    seg = torch.full((E + 1,), -7, dtype=torch.int32, device=DEV)
    row_src, pos = (torch.full((n,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    ws = torch.full((N.moe_permute_workspace(n, E),), -9, dtype=torch.int32, device=DEV)
    N.moe_permute_ws(slots.to(DEV), E, seg, row_src, pos, ws)
    order = torch.sort(torch.where(kept, slots, torch.full_like(slots, E)), stable=True).indices[:int(kept.sum())]
    counts = torch.bincount(slots[kept], minlength=E)
    assert seg.tolist() == [0] + counts.cumsum(0).tolist()
    assert torch.equal(row_src[:len(order)].cpu().long(), order) and bool((row_src[len(order):] == -7).all())
    assert torch.equal(pos.cpu()[order].long(), torch.arange(len(order))) and bool((pos.cpu()[~kept] == -1).all())


def test_batches_without_tokens():
    N = native()
    q, k = torch.empty(0, 4, 64, dtype=torch.bfloat16, device=DEV), torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    stat = torch.empty(4, 0, device=DEV)
    for bounds in ([0], [0, 0, 0]):
        plan = N.attn_packed_plan(torch.tensor(bounds, dtype=torch.int32, device=DEV), 0)
        N.attn_packed_fwd(q, k, k, torch.empty_like(q), stat, plan)
        N.attn_packed_bwd(q, k, k, q, stat, q, torch.empty_like(q), torch.empty_like(k), torch.empty_like(k),
                          torch.empty_like(stat), plan)
    x, idx, gate = torch.empty(0, 16, device=DEV), torch.empty(0, 2, dtype=torch.int32, device=DEV), torch.empty(0, 2, device=DEV)
    rows = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    N.moe_route(x, idx, gate)
    N.moe_route_bwd(x, idx, torch.empty_like(x), dgate=gate)
    N.moe_route_bwd(x, idx, torch.empty_like(x), dout=rows, y=rows, pos=idx.view(-1))
    seg, none = torch.full((17,), 9, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV)
    N.moe_permute_ws(idx.view(-1), 16, seg, none, none, torch.empty(N.moe_permute_workspace(0, 16), dtype=torch.int32, device=DEV))
    assert bool((seg == 0).all())
    N.dropout_add(rows, torch.empty_like(rows), torch.zeros(2, dtype=torch.int64, device=DEV), 0.1, resid=rows)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[1, 1, 2, 3, 1], [40, 2, 130], [1, 300]])
@pytest.mark.parametrize("causal", [False, True])
def test_query_and_key_gradients_under_large_scores(D, lens, causal):
    """Scores of some thousands: fp32 holds a row's log-sum-exp to 2^-24 of that, so all its weights are off by one factor,
    which must not show: the row sum is of weights that sum to one.  What may show: fp32 errors of the single scores, e =
    (D + 8) 2^-24 of sum |q| |k|, which shift weights against each other and enter dS as P 2 e (|dP - D| + sum P |dP - D|); those
    of the products dP, (D + 8) 2^-24 of sum |dO| |V|, and of the row sum, 2^-20 of sum P |dP|; dS and the results in bf16."""
    N = native()
    H, T = 4, sum(lens)
    g = torch.Generator().manual_seed(T + D)
    common = torch.randn(2, 1, H, D, generator=g) * 4
    q = (torch.randn(T, H, D, generator=g) * 16).to(torch.bfloat16)
    k, v = (torch.randn(2, T, H, D, generator=g) + common).to(torch.bfloat16).unbind(0)
    q[:, 0] = (8 * common[0, :, 0]).to(torch.bfloat16)              # one head with scores far from zero on one side
    do = torch.randn(T, H, D, generator=g).to(torch.bfloat16)
    qd, kd, vd, dod = (t.to(DEV) for t in (q, k, v, do))
    o, dq, dk, dv = (torch.empty_like(qd) for _ in range(4))
    lse, delta = (torch.empty(H, T, device=DEV) for _ in range(2))
    cu = [0] + torch.tensor(lens).cumsum(0).tolist()
    plan = N.attn_packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), T)
    N.attn_packed_fwd(qd, kd, vd, o, lse, plan, causal=causal)
    N.attn_packed_bwd(qd, kd, vd, o, lse, dod, dq, dk, dv, delta, plan, causal=causal)
    scale = D ** -0.5
    for a, b in zip(cu[:-1], cu[1:]):
        Q, K, V, dO = (t[a:b].double().transpose(0, 1) for t in (q, k, v, do))
        hidden = torch.ones(b - a, b - a, dtype=torch.bool).triu(1) if causal else torch.zeros(b - a, b - a, dtype=torch.bool)
        P = torch.softmax((Q @ K.transpose(1, 2) * scale).masked_fill(hidden, float("-inf")), -1)
        dP = dO @ V.transpose(1, 2)
        off = dP - (P * dP).sum(-1, keepdim=True)
        dS = P * off
        e = ((D + 8) * 2.0 ** -24 * (Q.abs() @ K.abs().transpose(1, 2)) * scale).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
        dp_err = (D + 8) * 2.0 ** -24 * (dO.abs() @ V.abs().transpose(1, 2))
        err = U * dS.abs() + P * (2 * e * (off.abs() + dS.abs().sum(-1, keepdim=True)) + dp_err
                                  + (P * dp_err).sum(-1, keepdim=True) + 2.0 ** -20 * (P * dP.abs()).sum(-1, keepdim=True))
        for name, got, want, bound in (("dq", dq, dS @ K * scale, scale * err @ K.abs()),
                                       ("dk", dk, dS.transpose(1, 2) @ Q * scale, scale * err.transpose(1, 2) @ Q.abs())):
            within(got[a:b].transpose(0, 1), want, 1.02 * (bound + U * want.abs()) + 1e-30, f"{name} of rows {a} to {b - 1}")
