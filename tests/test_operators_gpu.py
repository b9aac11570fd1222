"""Packed attention, routing, permutation and dropout on the GPU against their definitions in 64 bits.

Tolerances count roundings.  A value stored or multiplied as bf16 is off by at most U = 2^-8 of itself, an fp32 one by
2^-24; sums of products with rounded factors are off by at most the sum of the factors' errors times the other
factors' absolute values, which the tests form element by element.
"""
import functools

import pytest
import torch

from oracle import ops as O

DEV = "cuda"
U = 2.0 ** -8


def native():
    from pippy_amd import _native
    return _native


def within(got, want, bound, what):
    err = (got.double().cpu() - want).abs()
    worst = (err - bound).max() if err.numel() else torch.tensor(-1.0)
    assert bool((err <= bound).all()), f"{what}: error exceeds its bound by {float(worst):.3e}"


# ---- attention over packed sequences ------------------------------------------------------------
def attention_reference(q, k, v, do, cu, causal, scale=None):
    """Outputs, gradients and the elementwise error bounds of all of them, in 64 bits."""
    T, H, D = q.shape
    rep = H // k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    q, k, v, do = (t.double() for t in (q, k, v, do))
    out = {n: torch.zeros_like(t) for n, t in (("o", q), ("dq", q), ("dk", k), ("dv", v))}
    out["lse"] = torch.zeros(H, T, dtype=torch.float64)
    tol = {n: torch.zeros_like(t) for n, t in out.items()}
    # fp32 work around the roundings to bf16: scores of size s are off by (D + 8) 2^-24 of sum |q||k|, which the
    # exponential turns into a relative error of P; sums of up to 2^13 terms add 2^-11 at the very most
    for r0, r1 in zip(cu[:-1], cu[1:]):
        for h in range(H if r1 > r0 else 0):
            at, g = slice(r0, r1), h // rep
            Q, K, V, dO = q[at, h], k[at, g], v[at, g], do[at, h]
            S = Q @ K.T * scale
            hidden = torch.ones(r1 - r0, r1 - r0, dtype=torch.bool).triu(1) if causal else None
            if causal:
                S = S.masked_fill(hidden, float("-inf"))
            lse = torch.logsumexp(S, -1)
            P = torch.exp(S - lse[:, None])
            s_err = (D + 8) * 2.0 ** -24 * (Q.abs() @ K.abs().T * scale)
            if causal:
                s_err = s_err.masked_fill(hidden, 0.0)
            lse_err = s_err.amax(-1) + 2.0 ** -20 * (1 + lse.abs())
            p_rel = s_err + lse_err[:, None]            # relative error of P in fp32
            o = P @ V
            o_tol = (P * (U + p_rel)) @ V.abs() * (1 + U) + (U + 2.0 ** -18) * o.abs() + p_rel.amax(-1, keepdim=True) * o.abs()
            out["o"][at, h], tol["o"][at, h] = o, o_tol
            out["lse"][h, at], tol["lse"][h, at] = lse, lse_err
            dP = dO @ V.T
            Dr = (P * dP).sum(-1, keepdim=True)
            dS = P * (dP - Dr)
            dp_err = (D + 8) * 2.0 ** -24 * (dO.abs() @ V.abs().T)
            # the dQ kernel takes rowsum(dO * O) of the stored output, the dK / dV kernel the sum of P dP in fp32
            d_sum_err = (P * (p_rel * dP.abs() + dp_err)).sum(-1, keepdim=True) + 2.0 ** -18 * (P * dP.abs()).sum(-1, keepdim=True)
            d_out_err = (dO.abs() * o_tol).sum(-1, keepdim=True) + 2.0 ** -18 * (dO.abs() * o.abs()).sum(-1, keepdim=True)
            ds_err = U * dS.abs() + P * (p_rel * (dP - Dr).abs() + dp_err)
            out["dv"][at, g] += P.T @ dO
            tol["dv"][at, g] += (P * (U + p_rel)).T @ dO.abs() * (1 + U)
            out["dq"][at, h] = scale * dS @ K
            tol["dq"][at, h] = scale * (ds_err + P * d_out_err) @ K.abs() * (1 + U) + (U + 2.0 ** -18) * out["dq"][at, h].abs()
            out["dk"][at, g] += scale * dS.T @ Q
            tol["dk"][at, g] += scale * (ds_err + P * d_sum_err).T @ Q.abs() * (1 + U)
    for n in ("dk", "dv"):
        tol[n] += (U + 2.0 ** -18) * out[n].abs()
    return out, {n: t + 1e-30 for n, t in tol.items()}


SENTINEL = 77.0


class Packed:
    """One packed batch on the device: q | k | v sections of one buffer, outputs preset to a sentinel."""

    def __init__(self, cu, rows, H, Hkv, D, seed=0, scale_q=1.0):
        N = native()
        g = torch.Generator().manual_seed(seed)
        self.cu, self.rows, self.H, self.Hkv, self.D = cu, rows, H, Hkv, D
        W = (H + 2 * Hkv) * D
        qkv = torch.randn(rows, W, generator=g)
        qkv[:, :H * D] *= scale_q
        self.qkv = qkv.to(torch.bfloat16).to(DEV)
        self.do = (torch.randn(rows, H, D, generator=g) * 0.1).to(torch.bfloat16).to(DEV)
        self.outputs()
        self.cu_dev = torch.tensor(cu, dtype=torch.int32, device=DEV)
        self.plan = N.attn_packed_plan(self.cu_dev, rows)

    def sections(self, t):
        H, Hkv, D = self.H, self.Hkv, self.D
        q, k, v = t.split([H * D, Hkv * D, Hkv * D], dim=-1)
        return q.unflatten(-1, (H, D)), k.unflatten(-1, (Hkv, D)), v.unflatten(-1, (Hkv, D))

    def outputs(self):
        self.o = torch.full((self.rows, self.H, self.D), SENTINEL, dtype=torch.bfloat16, device=DEV)
        self.lse = torch.full((self.H, self.rows), SENTINEL, device=DEV)
        self.delta = torch.full((self.H, self.rows), SENTINEL, device=DEV)
        self.dqkv = torch.full_like(self.qkv, SENTINEL)

    def run(self, causal, scale=None, backward=True):
        N = native()
        q, k, v = self.sections(self.qkv)
        N.attn_packed_fwd(q, k, v, self.o, self.lse, self.plan, causal=causal, scale=scale)
        if backward:
            N.attn_packed_bwd(q, k, v, self.o, self.lse, self.do, *self.sections(self.dqkv), self.delta, self.plan,
                              causal=causal, scale=scale)
        return self

    def check(self, causal, scale=None):
        q, k, v = (t.cpu() for t in self.sections(self.qkv))
        want, tol = attention_reference(q, k, v, self.do.cpu(), self.cu, causal, scale)
        inside = torch.zeros(self.rows, dtype=torch.bool)
        for r0, r1 in zip(self.cu[:-1], self.cu[1:]):
            inside[r0:r1] = True
        dq, dk, dv = self.sections(self.dqkv)
        for name, got in (("o", self.o), ("dq", dq), ("dk", dk), ("dv", dv)):
            within(got.cpu()[inside], want[name][inside], tol[name][inside], name)
            assert bool((got.cpu()[~inside] == SENTINEL).all()), f"{name}: a row outside every sequence was written"
        within(self.lse.cpu()[:, inside], want["lse"][:, inside], tol["lse"][:, inside], "lse")
        assert bool((self.lse.cpu()[:, ~inside] == SENTINEL).all())


CUTS = {
    "one token": [0, 1],
    "empty ones between": [0, 0, 1, 1, 64, 127, 127, 256],
    "tile edges": [0, 63, 127, 192, 257, 385, 512],
    "long and short": [0, 3, 703, 704, 1004],
    "gap in front": [5, 70, 200],
}


@pytest.mark.gpu
@pytest.mark.parametrize("cut", list(CUTS))
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (8, 2, 64), (3, 1, 128), (8, 8, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_forward_and_backward(cut, H, Hkv, D, causal):
    cu = CUTS[cut]
    b = Packed(cu, cu[-1] + 7, H, Hkv, D, seed=len(cut))
    # what lies outside the sequences may be anything
    b.qkv[cu[-1]:] = float("nan")
    b.do[cu[-1]:] = float("nan")
    b.qkv[:cu[0]] = float("inf")
    b.run(causal).check(causal)


@pytest.mark.gpu
@pytest.mark.parametrize("H,Hkv,D", [(48, 48, 64), (48, 6, 64), (32, 32, 128), (32, 4, 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_in_launches_that_fill_the_gpu(H, Hkv, D, causal):
    """Sizes from which on the kernels take blocks of 128 rows (and, with as many key / value heads, of 128 keys)."""
    cu = [0, 1, 130, 130, 386, 700, 1465, 1529, 2052]
    b = Packed(cu, 2060, H, Hkv, D, seed=31)
    b.qkv[cu[-1]:] = float("nan")
    b.do[cu[-1]:] = float("nan")
    b.run(causal).check(causal)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
def test_packed_attention_with_large_scores_and_a_scale_of_the_callers(D):
    cu = [0, 100, 230]
    Packed(cu, 230, 4, 2, D, seed=3, scale_q=8.0).run(True, scale=0.3).check(True, scale=0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("scale", [2.0 ** -60, 1e-3, 4.0])
def test_packed_attention_with_nearly_equal_and_nearly_single_weights(D, scale):
    cu = [0, 1, 65, 200]
    Packed(cu, 200, 4, 2, D, seed=9).run(True, scale=scale).check(True, scale=scale)


@pytest.mark.gpu
def test_packed_attention_sequences_do_not_see_each_other():
    cu = [0, 50, 130, 300]
    clean = Packed(cu, 300, 4, 4, 64, seed=5).run(True)
    dirty = Packed(cu, 300, 4, 4, 64, seed=5)
    dirty.qkv[50:130] = float("nan")
    dirty.run(True)
    for a, b in ((clean.o, dirty.o), (clean.dqkv, dirty.dqkv)):
        assert torch.equal(a[:50], b[:50]) and torch.equal(a[130:], b[130:])
    assert bool(dirty.o[50:130].isnan().all())


@pytest.mark.gpu
def test_packed_attention_of_separate_tensors_and_many_short_sequences():
    N = native()
    g = torch.Generator().manual_seed(9)
    lens = torch.randint(0, 6, (3000,), generator=g)
    cu = [0] + lens.cumsum(0).tolist()
    T, H, D = cu[-1], 2, 64
    q, k, v, do = ((torch.randn(T, H, D, generator=g)).to(torch.bfloat16) for _ in range(4))
    qd, kd, vd, dod = (t.to(DEV) for t in (q, k, v, do))
    o, dq, dk, dv = (torch.empty_like(qd) for _ in range(4))
    lse, delta = torch.empty(H, T, device=DEV), torch.empty(H, T, device=DEV)
    plan = N.attn_packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), T)
    N.attn_packed_fwd(qd, kd, vd, o, lse, plan)
    N.attn_packed_bwd(qd, kd, vd, o, lse, dod, dq, dk, dv, delta, plan)
    # sequences of at most 5 rows: one block-diagonal product instead of 3000 small ones
    q, k, v, do = (t.double().transpose(0, 1) for t in (q, k, v, do))
    seq = torch.repeat_interleave(torch.arange(3000), lens)
    pos = torch.arange(T)
    near = torch.stack([pos - i for i in range(5)], -1)          # a row sees itself and up to 4 before it
    seen = (near >= 0) & (seq[near.clamp(min=0)] == seq[:, None])
    near = near.clamp(min=0)
    S = (q[:, :, None] * k[:, near]).sum(-1) * D ** -0.5
    P = torch.softmax(S.masked_fill(~seen, float("-inf")), -1)
    want = (P[..., None] * v[:, near]).sum(2)
    bound = (P[..., None] * v[:, near].abs()).sum(2) * (U + 2.0 ** -12) + (U + 2.0 ** -12) * want.abs()
    within(o.transpose(0, 1), want, bound, "o")
    dP = (do[:, :, None] * v[:, near]).sum(-1)
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    want = torch.zeros_like(q).index_add(1, near.flatten(), (P[..., None] * do[:, :, None]).flatten(1, 2))
    bound = torch.zeros_like(q).index_add(1, near.flatten(), (P[..., None] * do[:, :, None].abs()).flatten(1, 2))
    within(dv.transpose(0, 1), want, bound * (U + 2.0 ** -12) + (U + 2.0 ** -12) * want.abs(), "dv")
    d_err = (do.abs() * (U + 2.0 ** -12) * ((P[..., None] * v[:, near].abs()).sum(2) * 2)).sum(-1)[..., None]
    want = (dS[..., None] * k[:, near]).sum(2) * D ** -0.5
    bound = ((U * dS.abs() + P * (d_err + 2.0 ** -12 * dP.abs()))[..., None] * k[:, near].abs()).sum(2) * D ** -0.5 * 1.01
    within(dq.transpose(0, 1), want, bound + (U + 2.0 ** -12) * want.abs(), "dq")


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[1, 2], [2, 1, 3, 2], [8, 33, 64]])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_attention_query_gradient_of_few_keys(lens, causal, D):
    """With one block of keys the row sums in dS are those of P dP: the rounding of the output does not reach dQ.
    What is left: dS rounded to bf16 (2^-8 of each term of the sum over the keys), dQ rounded to bf16, and 2^-16 of every
    term of dS for the fp32 exponentials and sums (scores up to 2^5: P is off by 2^5 2^-22, the sums over D by D 2^-24)."""
    N = native()
    H, T = 5, sum(lens)
    g = torch.Generator().manual_seed(T + D)
    q, k, v, do = (torch.randn(T, H, D, generator=g).to(torch.bfloat16) for _ in range(4))
    cu = torch.tensor([0] + lens).cumsum(0).int()
    qd, kd, vd, dod = (t.to(DEV) for t in (q, k, v, do))
    o, dq, dk, dv = (torch.empty_like(qd) for _ in range(4))
    lse, delta = (torch.empty(H, T, device=DEV) for _ in range(2))
    plan = N.attn_packed_plan(cu.to(DEV), T)
    N.attn_packed_fwd(qd, kd, vd, o, lse, plan, causal=causal)
    N.attn_packed_bwd(qd, kd, vd, o, lse, dod, dq, dk, dv, delta, plan, causal=causal)
    scale = D ** -0.5
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        Q, K, V, dO = (t[a:b].double().transpose(0, 1) for t in (q, k, v, do))
        S = Q @ K.transpose(1, 2) * scale
        if causal:
            S = S.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), float("-inf"))
        P = torch.softmax(S, -1)
        dP = dO @ V.transpose(1, 2)
        row = (P * dP).sum(-1, keepdim=True)
        dS = P * (dP - row)
        want = dS @ K * scale
        noise = P * (dP.abs() + (P * dP.abs()).sum(-1, keepdim=True))
        bound = scale * (U * dS.abs() + 2.0 ** -16 * noise) @ K.abs() + U * want.abs()
        within(dq[a:b].transpose(0, 1), want, 1.01 * bound + 1e-30, "dq")


@pytest.mark.gpu
def test_packed_attention_gradients_agree_with_differences():
    """The directional derivative of <o, do> from the kernel's gradients against central differences of the
    definition in 64 bits."""
    cu, causal = [0, 40, 41, 150], True
    b = Packed(cu, 150, 4, 2, 64, seed=11).run(causal)
    q, k, v = (t.cpu().double() for t in b.sections(b.qkv))
    do = b.do.cpu().double()
    _, tol = attention_reference(q, k, v, do, cu, causal)
    loss = lambda q, k, v: float((O.attention_packed(q, k, v, cu, causal)[0] * do).sum())  # noqa: E731
    g = torch.Generator().manual_seed(1)
    for i, (name, got) in enumerate(zip(("dq", "dk", "dv"), b.sections(b.dqkv))):
        u = torch.randn(got.shape, generator=g, dtype=torch.float64)
        eps = 1e-5
        plus, minus = [[t + s * eps * u if j == i else t for j, t in enumerate((q, k, v))] for s in (1, -1)]
        slope = (loss(*plus) - loss(*minus)) / (2 * eps)
        bound = float((tol[name] * u.abs()).sum()) + 1e-6 * (1 + abs(slope))
        # the rounding errors of thousands of elements do not line up: a tenth of the worst case is still generous
        assert abs(float((got.cpu().double() * u).sum()) - slope) <= 0.1 * bound, name


@pytest.mark.gpu
def test_packed_attention_is_the_same_on_every_run_and_under_another_plan_order():
    cu = [0, 300, 301, 700, 1000]
    a, b = (Packed(cu, 1000, 8, 2, 128, seed=2).run(True) for _ in range(2))
    first = [t.clone() for t in (b.o, b.lse, b.dqkv)]
    b.plan = native().attn_packed_plan(b.cu_dev, 1000)
    b.run(True)
    for x, y, z in zip(first, (a.o, a.lse, a.dqkv), (b.o, b.lse, b.dqkv)):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.gpu
def test_packed_attention_ignores_bounds_that_are_out_of_order_or_range():
    N = native()
    b = Packed([0, 64, 100], 100, 2, 2, 64, seed=4)
    good = b.run(True).o.clone()
    for cu in ([0, 64, 30], [0, 64, 500], [0, 64, -5]):       # the second sequence counts as empty
        b.outputs()
        b.plan = N.attn_packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), 100)
        b.run(True)
        assert torch.equal(b.o[:64], good[:64]) and bool((b.o[64:] == SENTINEL).all())


@pytest.mark.gpu
def test_packed_attention_captured_with_its_plan():
    """A captured step that rebuilds its plan follows new sequence bounds on replay."""
    N = native()
    b = Packed([0, 100, 200, 300], 300, 4, 2, 64, seed=6)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        N.attn_packed_plan(b.cu_dev, b.rows, out=b.plan)
        b.run(True)

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for cu in ([0, 100, 200, 300], [0, 10, 290, 295], [0, 0, 1, 300], [0, 150, 150, 200]):
        eager = Packed(cu, 300, 4, 2, 64, seed=6).run(True)
        b.cu_dev.copy_(torch.tensor(cu, dtype=torch.int32))
        for t in (b.o, b.lse, b.dqkv):
            t.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        for x, y in ((b.o, eager.o), (b.lse, eager.lse), (b.dqkv, eager.dqkv)):
            assert torch.equal(x, y)


@pytest.mark.gpu
def test_packed_attention_far_into_a_large_buffer():
    """Rows whose byte offsets pass 2^32 (elements past 2^31), in one long sequence and in a short one behind it."""
    N = native()
    H, D, stride, T = 1, 64, 16384, 140000
    buf = torch.empty(T, stride, dtype=torch.bfloat16, device=DEV)
    q, k, v, o, do, dq, dk, dv = (buf[:, 64 * i:64 * i + 64].unflatten(-1, (1, 64)) for i in range(8))
    g = torch.Generator().manual_seed(8)
    for t in (q, k, v, do):
        t.copy_(torch.randn(T, 1, D, generator=g).to(torch.bfloat16))
    lse, delta = torch.empty(H, T, device=DEV), torch.empty(H, T, device=DEV)
    cu = [0, 139900, T]
    plan = N.attn_packed_plan(torch.tensor(cu, dtype=torch.int32, device=DEV), T)
    N.attn_packed_fwd(q, k, v, o, lse, plan)
    last = [t[139900:].cpu() for t in (q, k, v, do)]
    want, tol = attention_reference(*last, [0, 100], True)
    within(o[139900:], want["o"], tol["o"], "o of the last sequence")
    # a late query of the long sequence against all its keys
    i = 139899
    s = k[:i + 1, 0].double() @ q[i, 0].double() * D ** -0.5
    p = torch.softmax(s, 0)
    want_o = (p @ v[:i + 1, 0].double()).cpu()
    bound = (p @ v[:i + 1, 0].double().abs()).cpu() * (U + 2.0 ** -10) + U * want_o.abs()
    within(o[i, 0], want_o, bound, "o of a late query")
    # backward of the short sequence alone, under a plan that leaves the long one out
    plan = N.attn_packed_plan(torch.tensor([139900, T], dtype=torch.int32, device=DEV), T)
    N.attn_packed_bwd(q, k, v, o, lse, do, dq, dk, dv, delta, plan)
    for name, t in (("dq", dq), ("dk", dk), ("dv", dv)):
        within(t[139900:], want[name], tol[name], name)


@pytest.mark.gpu
def test_packed_attention_refuses():
    N = native()
    b = Packed([0, 10], 10, 4, 2, 64)
    q, k, v = b.sections(b.qkv)
    for bad, match in ((lambda: N.attn_packed_fwd(q.float(), k, v, b.o, b.lse, b.plan), "bf16"),
                       (lambda: N.attn_packed_fwd(q, k, v[:, :1], b.o, b.lse, b.plan), "v must"),
                       (lambda: N.attn_packed_fwd(q[:9], k[:9], v[:9], b.o[:9], b.lse[:, :9].contiguous(), b.plan), "plan of 10 rows"),
                       (lambda: N.attn_packed_fwd(q, k, v, b.o, b.lse.t().contiguous(), b.plan), "lse"),
                       (lambda: N.attn_packed_fwd(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, b.o, b.lse, b.plan), "heads of a row"),
                       (lambda: N.attn_packed_plan(b.cu_dev.long(), 10), "int32"),
                       (lambda: N.attn_packed_plan(b.cu_dev, 11, out=b.plan), "other sizes")):
        with pytest.raises(ValueError, match=match):
            bad()
    with pytest.raises(RuntimeError, match="head_dim"):
        t = torch.zeros(10, 4, 32, dtype=torch.bfloat16, device=DEV)
        N.attn_packed_fwd(t, t, t, t.clone(), b.lse, b.plan)


# ---- routing ----------------------------------------------------------------------------------------
ROUTES = [
    # T, E, k, scoring, bias, groups, kept, group score, renorm, fp32
    (1, 2, 1, "softmax", False, 1, 1, "max", True, False),
    (37, 8, 2, "softmax", False, 1, 1, "max", True, False),
    (65, 8, 8, "sigmoid", True, 1, 1, "max", False, True),
    (50, 61, 6, "softmax", False, 1, 1, "max", False, False),
    (33, 64, 16, "sigmoid", True, 8, 3, "top2", True, True),
    (40, 72, 5, "softmax", True, 3, 1, "max", True, False),
    (29, 160, 6, "softmax", False, 8, 3, "max", False, True),
    (31, 256, 8, "sigmoid", True, 8, 4, "top2", True, True),
    (17, 257, 4, "softmax", False, 1, 1, "max", True, False),
    (20, 500, 10, "sigmoid", False, 4, 2, "top2", True, False),
    (19, 512, 16, "softmax", True, 64, 7, "top2", True, True),
]


@functools.lru_cache(maxsize=None)
def route_case(i):
    T, E, k, scoring, bias, groups, kept, group_score, renorm, fp32 = ROUTES[i]
    g = torch.Generator().manual_seed(100 + i)
    x = torch.randn(T, E, generator=g)
    if not fp32:
        x = x.to(torch.bfloat16)
    x[T // 2] = 0.5                             # a row of ties
    b = torch.randn(E, generator=g) * 0.05 if bias else None
    if b is not None:
        b[E // 2] = b[0]
    how = dict(scoring=scoring, n_group=groups, topk_group=kept, group_score=group_score, renorm=renorm, scale=1.7)
    return x, b, k, how


def route_sums(E):
    return (E / 8 + 64) * 2.0 ** -24            # fp32 sums over a lane's experts and the lanes, exp, divisions


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(ROUTES)))
def test_routing_matches_its_definition(i):
    N = native()
    x, b, k, how = route_case(i)
    T, E = x.shape
    xd = torch.full((T, E + 5), 9.0, dtype=x.dtype, device=DEV)     # rows with padding columns behind them
    xd[:, :E] = x.to(DEV)
    idx = torch.full((T, k), -7, dtype=torch.int32, device=DEV)
    gate = torch.full((T, k), -7.0, device=DEV)
    N.moe_route(xd, idx, gate, bias=None if b is None else b.to(DEV), E=E, **how)
    ref_idx, ref_gate = O.moe_route(x.double(), k, bias=None if b is None else b.double(), **how)
    assert torch.equal(idx.cpu().long(), ref_idx)
    within(gate, ref_gate, 2 * route_sums(E) * ref_gate.abs(), "gate")


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(ROUTES)))
@pytest.mark.parametrize("given", [True, False])
def test_routing_gradient_matches_the_formula_and_differences(i, given):
    N = native()
    x, b, k, how = route_case(i)
    T, E = x.shape
    g = torch.Generator().manual_seed(i)
    xr = x.double().requires_grad_(True)
    idx, _ = O.moe_route(x.double(), k, bias=None if b is None else b.double(), **how)
    _, gate = O.moe_route(xr, k, idx=idx, **how)
    C = 72
    pos = torch.randperm(T * k, generator=g)
    y = torch.randn(T * k, C, generator=g).to(torch.bfloat16)
    dout = torch.randn(T, C, generator=g).to(torch.bfloat16)
    rows = y.double()[pos].view(T, k, C)
    dgate = (rows * dout.double()[:, None]).sum(-1)
    dg_err = torch.zeros_like(dgate)
    if given:
        dgate = dgate.float().double()
    else:
        dg_err = (C + 8) * 2.0 ** -24 * (rows.abs() * dout.double()[:, None].abs()).sum(-1)
    want, = torch.autograd.grad((gate * dgate).sum(), xr)
    # differences of the definition along one direction, the selection held
    u = torch.randn(T, E, generator=g, dtype=torch.float64)
    f = lambda z: float((O.moe_route(z, k, idx=idx, **how)[1] * dgate).sum())  # noqa: E731
    slope = (f(x.double() + 1e-5 * u) - f(x.double() - 1e-5 * u)) / 2e-5
    assert abs(float((want * u).sum()) - slope) <= 1e-6 * (1 + float((want * u).abs().sum()))
    # |d| of every slot and what an error of the score sums and of dgate does to it
    score = torch.softmax(x.double(), -1) if how["scoring"] == "softmax" else torch.sigmoid(x.double())
    s = score.gather(-1, idx)
    if how["renorm"]:
        S = s.sum(-1, keepdim=True)
        size = how["scale"] * (dgate.abs() + (s / S * dgate.abs()).sum(-1, keepdim=True)) / S
        extra = how["scale"] * (dg_err + (s / S * dg_err).sum(-1, keepdim=True)) / S
    else:
        size, extra = how["scale"] * dgate.abs(), how["scale"] * dg_err
    err = 4 * route_sums(E) * size + extra
    spread = torch.zeros_like(score).scatter(1, idx, err)
    if how["scoring"] == "softmax":
        bound = score * (spread + (s * (err + 4 * route_sums(E) * size)).sum(-1, keepdim=True))
    else:
        bound = spread * score * (1 - score + 2.0 ** -22)
    bound = bound + (2.0 ** -22 if x.dtype == torch.float32 else U) * want.abs() + 1e-30
    bound = bound * 1.01
    cols = (E + 7) // 8 * 8 if E < 505 else 512
    dl = torch.full((T, cols + 3), 9.0, dtype=x.dtype, device=DEV)[:, :cols]
    src = dict(dgate=dgate.float().to(DEV)) if given else dict(dout=dout.to(DEV), y=y.to(DEV), pos=pos.int().to(DEV))
    N.moe_route_bwd(x.to(DEV), idx.int().to(DEV), dl, scoring=how["scoring"], renorm=how["renorm"], scale=how["scale"], **src)
    within(dl[:, :E], want, bound, "dlogits")
    assert bool((dl[:, E:] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_routing_with_experts_taken_out(scoring, groups):
    N = native()
    T, E, k = 12, 16, 4
    x = torch.randn(T, E, generator=torch.Generator().manual_seed(0))
    x[0] = float("-inf")                        # a padding token: nothing is left
    x[1, 1:] = float("-inf")
    x[2, :13] = float("-inf")
    x[3, ::2] = float("-inf")
    x[4, 5] = -1e30                             # tiny, but there
    how = dict(scoring=scoring, n_group=groups, topk_group=1 if groups == 1 else 2, group_score="top2")
    idx = torch.empty(T, k, dtype=torch.int32, device=DEV)
    gate = torch.empty(T, k, device=DEV)
    bias = torch.linspace(-0.2, 0.2, E)
    N.moe_route(x.to(DEV), idx, gate, bias=bias.to(DEV), **how)
    ref_idx, ref_gate = O.moe_route(x.double(), k, bias=bias.double(), **how)
    assert torch.equal(idx.cpu().long(), ref_idx)
    assert idx[0].tolist() == [-1] * 4 and idx[1].tolist() == [0, -1, -1, -1]
    within(gate, ref_gate, 2 * route_sums(E) * ref_gate, "gate")
    dl = torch.empty(T, E, device=DEV)
    N.moe_route_bwd(x.to(DEV), idx, dl, dgate=torch.ones(T, k, device=DEV), scoring=scoring, renorm=False)
    assert bool(dl.isfinite().all()) and bool((dl[0] == 0).all()) and bool((dl[3, ::2] == 0).all())


@pytest.mark.gpu
def test_routing_of_nan_logits_stays_in_range():
    N = native()
    x = torch.randn(6, 24, device=DEV)
    x[1, 3] = float("nan")
    x[2] = float("nan")
    x[3, 7] = float("inf")
    idx = torch.empty(6, 4, dtype=torch.int32, device=DEV)
    gate = torch.empty(6, 4, device=DEV)
    for scoring in ("softmax", "sigmoid"):
        N.moe_route(x, idx, gate, scoring=scoring)
        assert bool(((idx >= 0) & (idx < 24)).all())
        assert all(len(set(row)) == 4 for row in idx.tolist())
        assert 3 not in idx[1].tolist() and idx[2].tolist() == [0, 1, 2, 3] and int(idx[3, 0]) == 7
        assert bool(gate[2].isnan().all()) and bool(gate[[0, 4, 5]].isfinite().all())


@pytest.mark.gpu
def test_routing_tells_choices_apart_that_differ_by_less_than_a_rounding():
    """Scores plus bias that are equal in fp32 and not in 64 bits."""
    N = native()
    E, k = 64, 8
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(512, E, generator=g) * 1e-4).float()
    bias = torch.full((E,), 0.25)
    for scoring in ("softmax", "sigmoid"):
        idx = torch.empty(512, k, dtype=torch.int32, device=DEV)
        gate = torch.empty(512, k, device=DEV)
        N.moe_route(x.to(DEV), idx, gate, bias=bias.to(DEV), scoring=scoring)
        choice = (torch.softmax(x.double(), -1) if scoring == "softmax" else torch.sigmoid(x.double())) + 0.25
        want = torch.sort(choice, dim=-1, descending=True, stable=True).indices[:, :k]
        assert torch.equal(idx.cpu().long(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("E,k", [(16, 3), (16, 16), (64, 8), (100, 16), (256, 3), (256, 8), (512, 16)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [True, False])
def test_routing_of_rows_with_an_order(E, k, scoring, biased):
    """Rows whose largest experts are neighbours, whose experts are equal, or whose scores round to the same in fp32."""
    N = native()
    g = torch.Generator().manual_seed(E + k)
    up = torch.linspace(-2, 2, E)
    rows = [up, -up, torch.zeros(E), torch.full((E,), 3.0), (up * 4).round(), 20 + up, 20 + up[torch.randperm(E, generator=g)],
            torch.where(torch.arange(E) % 7 == 3, 1.5, -1.5)]
    for first in range(0, E, max(k, E // 5)):       # the largest ones side by side, over every border of lanes
        rows.append(torch.randn(E, generator=g) * 0.1)
        rows[-1][first:first + k] += 5
    few = torch.full((E,), float("-inf"))
    few[E // 2] = few[-1] = few[0] = 0.25
    x = torch.stack(rows + [few] + [torch.randn(E, generator=g) for _ in range(9)])
    bias = torch.where(torch.arange(E) % 2 == 0, 0.25, 0.5) if biased else None
    T = x.shape[0]
    idx = torch.full((T, k), -7, dtype=torch.int32, device=DEV)
    gate = torch.full((T, k), -7.0, device=DEV)
    N.moe_route(x.to(DEV), idx, gate, bias=None if bias is None else bias.to(DEV), scoring=scoring)
    want, want_gate = O.moe_route(x.double(), k, bias=None if bias is None else bias.double(), scoring=scoring)
    assert torch.equal(idx.cpu().long(), want)
    within(gate, want_gate, 2 * route_sums(E) * want_gate, "gate")


# ---- permutation ------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n,E", [(0, 4), (1, 1), (10, 64), (96, 64), (2048, 8), (2049, 3), (5001, 256), (40000, 1024),
                                 (70001, 129), (262145, 17), (1048577, 300)])
def test_permutation_of_many_slots_bit_exact(n, E):
    N = native()
    g = torch.Generator().manual_seed(n)
    slots = torch.randint(0, E, (n,), generator=g, dtype=torch.int32)
    if n > 2000:
        slots[slots == 1] = 0                                  # an expert without tokens
    seg = torch.full((E + 1,), -7, dtype=torch.int32, device=DEV)
    row_src, pos = (torch.full((n,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    ws = torch.full((N.moe_permute_workspace(n, E),), -9, dtype=torch.int32, device=DEV)
    N.moe_permute_ws(slots.to(DEV), E, seg, row_src, pos, ws)
    ref_seg, ref_rows, ref_pos = O.moe_permutation(slots, E)
    assert torch.equal(seg.cpu().long(), ref_seg)
    assert torch.equal(row_src.cpu().long(), ref_rows) and torch.equal(pos.cpu().long(), ref_pos)
    if 0 < n and E <= 64:                                      # the one-work-group form leaves the same
        seg1, rows1, pos1 = (torch.empty_like(t) for t in (seg, row_src, pos))
        N.moe_permute(slots.to(DEV), E, seg1, rows1, pos1)
        assert torch.equal(seg, seg1) and torch.equal(row_src, rows1) and torch.equal(pos, pos1)


@pytest.mark.gpu
def test_permutation_drops_slots_without_an_expert():
    N = native()
    g = torch.Generator().manual_seed(4)
    n, E = 9000, 100
    slots = torch.randint(-3, E + 5, (n,), generator=g, dtype=torch.int32)
    kept = (slots >= 0) & (slots < E)
    seg = torch.empty(E + 1, dtype=torch.int32, device=DEV)
    row_src, pos = (torch.full((n,), -7, dtype=torch.int32, device=DEV) for _ in range(2))
    ws = torch.empty(N.moe_permute_workspace(n, E), dtype=torch.int32, device=DEV)
    N.moe_permute_ws(slots.to(DEV), E, seg, row_src, pos, ws)
    order = torch.sort(torch.where(kept, slots, torch.full_like(slots, E)), stable=True).indices
    m = int(kept.sum())
    assert int(seg[-1]) == m and torch.equal(row_src[:m].cpu().long(), order[:m])
    assert bool((row_src[m:] == -7).all()) and bool((pos.cpu()[~kept] == -1).all())
    assert torch.equal(pos.cpu()[order[:m]].long(), torch.arange(m))
    slots[:] = -1
    N.moe_permute_ws(slots.to(DEV), E, seg, row_src, pos, ws)
    assert bool((seg == 0).all()) and bool((pos == -1).all())


# ---- dropout ----------------------------------------------------------------------------------------
def rng_state(seed=0x1234567890ABCDEF, offset=0x300000005):
    return torch.tensor([seed, offset], dtype=torch.int64, device=DEV), seed, offset


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (1000,), (5, 13), (33, 64), (3, 2, 24)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.99999, 1.0])
def test_dropout_forward_and_backward(dtype, shape, p):
    N = native()
    g = torch.Generator().manual_seed(sum(shape))
    x, r, dy = (torch.randn(shape, generator=g).to(dtype) for _ in range(3))
    rng, seed, offset = rng_state()
    f = O.dropout_factors(x.numel(), p, seed, offset, 9).view(shape)
    half = U if dtype == torch.bfloat16 else 2.0 ** -24
    xd, rd, dyd = (t.to(DEV) for t in (x, r, dy))
    y, dx = torch.empty_like(xd), torch.empty_like(xd)
    N.dropout_add(xd, y, rng, p, resid=rd, site=9)
    want = r.double() + f * x.double()
    # scale and sum in fp32 (two roundings at most), then the stored one
    size = r.double().abs() + (f * x.double()).abs()
    within(y, want, 2.0 ** -23 * size + half * (1 + 2.0 ** -20) * want.abs(), "y")
    N.dropout_add(xd, y, rng, p, site=9)
    within(y, f * x.double(), (half + 2.0 ** -23) * (f * x.double()).abs(), "y without a residual")
    assert torch.equal(y.cpu() == 0, (f == 0) | (x == 0))
    N.dropout_bwd(dyd, dx, rng, p, site=9)
    within(dx, f * dy.double(), (half + 2.0 ** -23) * (f * dy.double()).abs(), "dx")


@pytest.mark.gpu
def test_dropout_of_rows_in_place_and_of_values_that_are_not_finite():
    N = native()
    rng, seed, offset = rng_state(offset=1)
    R, C, p = 37, 72, 0.3
    buf = torch.randn(R, 3 * C, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    x, r, y = buf[:, :C], buf[:, C:2 * C], torch.full((R, C + 8), SENTINEL, dtype=torch.bfloat16, device=DEV)
    f = O.dropout_factors(R * C, p, seed, offset, 0).view(R, C)
    want = r.double().cpu() + f * x.double().cpu()
    N.dropout_add(x, y[:, :C], rng, p, resid=r)
    within(y[:, :C], want, 2.0 ** -22 * (1 + want.abs()) + U * want.abs(), "rows")
    assert bool((y[:, C:] == SENTINEL).all())
    out = y[:, :C].clone()
    N.dropout_add(x, x, rng, p, resid=r)        # into its own input
    assert torch.equal(x, out)
    bad = torch.full((64,), float("inf"), dtype=torch.bfloat16, device=DEV)
    bad[::3] = float("nan")
    kept = O.dropout_factors(64, p, seed, offset, 0) != 0
    N.dropout_add(bad, bad, rng, p)
    assert bool((bad.cpu()[~kept] == 0).all()) and not bool(bad.cpu()[kept].isfinite().any())


@pytest.mark.gpu
def test_dropout_captured_follows_its_state():
    """A captured step with its own advance masks anew on every replay, forward and backward alike."""
    N = native()
    rng, seed, offset = rng_state(seed=5, offset=(1 << 32) - 2)     # the low half of the offset overflows
    x = torch.ones(4096, dtype=torch.bfloat16, device=DEV)
    y, dx = torch.empty_like(x), torch.empty_like(x)

    def step():
        N.rng_advance(rng)
        N.dropout_add(x, y, rng, 0.25, site=2)
        N.dropout_bwd(x, dx, rng, 0.25, site=2)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert rng.tolist() == [seed, offset + 2 + i]
        f = O.dropout_factors(4096, 0.25, seed, offset + 2 + i, 2).to(torch.bfloat16)
        assert torch.equal(y.cpu(), f) and torch.equal(dx, y)


@pytest.mark.gpu
def test_dropout_masks_are_independent_of_the_layout_and_of_the_type():
    N = native()
    rng, _, _ = rng_state()
    wide = torch.ones(20, 96, device=DEV)
    flat, rows = torch.empty(20, 96, device=DEV), torch.empty(20, 128, device=DEV)[:, :96]
    low = torch.empty(20, 96, dtype=torch.bfloat16, device=DEV)
    N.dropout_add(wide, flat, rng, 0.5)
    N.dropout_add(wide, rows, rng, 0.5)
    N.dropout_add(wide.bfloat16(), low, rng, 0.5)
    assert torch.equal(flat, rows) and torch.equal(flat, low.float())


@pytest.mark.gpu
def test_operators_refuse_tensors_that_do_not_fit():
    N = native()
    x = torch.zeros(4, 64, dtype=torch.bfloat16, device=DEV)
    rng, _, _ = rng_state()
    idx, gate = torch.zeros(4, 2, dtype=torch.int32, device=DEV), torch.zeros(4, 2, device=DEV)
    for call, match in ((lambda: N.dropout_add(x, x.float(), rng, 0.1), "one shape and type"),
                        (lambda: N.dropout_add(x, x, rng.int(), 0.1), "rng must"),
                        (lambda: N.dropout_add(x.t(), x.t(), rng, 0.1), "contiguous rows"),
                        (lambda: N.moe_route(x, idx.long(), gate), "topk_idx"),
                        (lambda: N.moe_route(x, idx, gate.bfloat16()), "gate"),
                        (lambda: N.moe_route(x, idx, gate, scoring="tanh"), "scoring"),
                        (lambda: N.moe_route(x, idx, gate, group_score="mean"), "group_score"),
                        (lambda: N.moe_route(x, idx, gate, bias=torch.zeros(63, device=DEV)), "bias"),
                        (lambda: N.moe_route(x, idx, gate, E=65), "65 experts"),
                        (lambda: N.moe_route_bwd(x, idx, x.clone()), "needs dgate"),
                        (lambda: N.moe_route_bwd(x, idx, x.float(), dgate=gate), "dlogits"),
                        (lambda: N.moe_permute_workspace(10, 2000), "out of range"),
                        (lambda: N.moe_permute_ws(idx, 8, idx, idx, idx, idx), "seg_start")):
        with pytest.raises(ValueError, match=match):
            call()


@pytest.mark.gpu
def test_launch_lists_hold_the_operators():
    """Route, permute, gather, dropout and the router's gradient as launch-list ops, with tokens that go to no expert."""
    from pippy_amd import _program as P
    N = native()
    g = torch.Generator().manual_seed(2)
    T, E, K, C = 60, 20, 3, 64
    logits = torch.randn(T, 24, generator=g).to(torch.bfloat16)
    logits[7:20, :E] = float("-inf")
    logits[20:25, 2:E] = float("-inf")
    ld = logits.to(DEV)
    x = torch.randn(T, C, generator=g).to(torch.bfloat16).to(DEV)
    rng, seed, offset = rng_state(seed=3, offset=10)
    idx, gate = torch.empty(T, K, dtype=torch.int32, device=DEV), torch.empty(T, K, device=DEV)
    seg = torch.empty(E + 1, dtype=torch.int32, device=DEV)
    row_src = torch.full((T * K,), 2 ** 30, dtype=torch.int32, device=DEV)      # never read past the placed rows
    pos = torch.empty(T * K, dtype=torch.int32, device=DEV)
    ws = torch.empty(N.moe_permute_workspace(T * K, E), dtype=torch.int32, device=DEV)
    rows = torch.full((T * K, C), SENTINEL, dtype=torch.bfloat16, device=DEV)
    y, dx, wide = torch.empty_like(x), torch.empty_like(x), torch.empty(T, 2 * C, dtype=torch.bfloat16, device=DEV)
    dl = torch.full_like(ld, 9.0)
    how = dict(scoring="sigmoid", n_group=4, topk_group=2, group_score="top2")
    ops = P.OpList()
    ops.append(P.op_rng_advance(rng))
    ops.append(P.op_moe_route(ld, idx, gate, E, **how))
    ops.append(P.op_moe_permute_ws(idx.view(-1), E, seg, row_src, pos, ws))
    ops.append(P.op_moe_gather(x, row_src, K, rows, n_rows=seg[E:]))
    ops.append(P.op_moe_combine(rows, pos, K, y, gate=gate.view(-1)))
    ops.append(P.op_dropout(y, wide[:, C:], rng, 0.4, 5, resid=x))
    ops.append(P.op_dropout(x, dx, rng, 0.4, 5))
    ops.append(P.op_moe_route_bwd(ld, idx, dl, E, x, rows, pos, scoring="sigmoid"))
    ops.run()
    torch.cuda.synchronize()
    assert rng.tolist() == [seed, offset + 1]
    ref_idx, ref_gate = O.moe_route(logits[:, :E].double(), K, **how)
    assert torch.equal(idx.cpu().long(), ref_idx)
    placed = int((ref_idx >= 0).sum())
    assert int(seg[E]) == placed < T * K and bool((rows[placed:] == SENTINEL).all())
    # every placed row is its token's, so the weighted sum is the token times the sum of its weights
    total = gate.cpu().double().sum(-1, keepdim=True)
    want = x.cpu().double() * total
    within(y, want, (U + 2.0 ** -20) * want.abs(), "combine")
    f = O.dropout_factors(T * C, 0.4, seed, offset + 1, 5).view(T, C)
    want = x.cpu().double() + f * y.cpu().double()
    within(wide[:, C:], want, 2.0 ** -22 * (1 + want.abs()) + U * want.abs(), "dropout")
    within(dx, f * x.cpu().double(), (U + 2.0 ** -22) * (f * x.cpu().double()).abs(), "dx")
    # the rows of a token are all alike: the gradient of renormalised weights is zero but for roundings of |x|^2
    size = x.cpu().double().pow(2).sum(-1, keepdim=True)
    assert bool((dl.cpu().double().abs() <= 2.0 ** -16 * size * (ref_idx >= 0).any(-1, keepdim=True)).all())


# ---- together ---------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_a_step_of_all_of_them_as_a_layer_uses_them():
    """Packed attention, dropout onto the residual stream, routing, permutation, expert products, the weighted sum
    and a second dropout; then the gradients back to the router and through the first dropout.  Stage by stage
    against 64 bits, each from the kernels' own inputs of that stage."""
    N = native()
    g = torch.Generator().manual_seed(21)
    cu, T, H, D, E, K = [0, 90, 91, 250], 256, 2, 64, 72, 4
    C = H * D
    rng, seed, offset = rng_state(seed=77, offset=4)
    b = Packed(cu, T, H, H, D, seed=21)
    b.o.zero_()
    b.lse.zero_()
    x = torch.randn(T, C, generator=g).to(torch.bfloat16).to(DEV)
    b.run(True, backward=False)
    h = torch.empty_like(x)
    N.dropout_add(b.o.view(T, C), h, rng, 0.2, resid=x, site=0)
    f0 = O.dropout_factors(T * C, 0.2, seed, offset, 0).view(T, C)
    want = x.cpu().double() + f0 * b.o.view(T, C).cpu().double()
    within(h, want, 2.0 ** -22 * (1 + want.abs()) + U * want.abs(), "residual stream")

    wr = (torch.randn(E, C, generator=g) * 0.2).to(torch.bfloat16).to(DEV)
    logits = torch.empty(T, E, dtype=torch.bfloat16, device=DEV)
    N.gemm_bf16(h, wr, logits)
    logits[cu[-1]:] = float("-inf")             # rows of no sequence go to no expert
    idx, gate = torch.empty(T, K, dtype=torch.int32, device=DEV), torch.empty(T, K, device=DEV)
    how = dict(scoring="softmax", n_group=6, topk_group=3)
    N.moe_route(logits, idx, gate, **how)
    ref_idx, ref_gate = O.moe_route(logits.cpu().double(), K, **how)
    assert torch.equal(idx.cpu().long(), ref_idx) and bool((idx[cu[-1]:] == -1).all())
    within(gate, ref_gate, 2 * route_sums(E) * ref_gate, "gate")

    n = T * K
    seg = torch.empty(E + 1, dtype=torch.int32, device=DEV)
    row_src, pos = torch.zeros(n, dtype=torch.int32, device=DEV), torch.empty(n, dtype=torch.int32, device=DEV)
    ws = torch.empty(N.moe_permute_workspace(n, E), dtype=torch.int32, device=DEV)
    N.moe_permute_ws(idx.view(-1), E, seg, row_src, pos, ws)
    placed = int(seg[-1])
    assert placed == cu[-1] * K
    xp, yp = torch.zeros(n, C, dtype=torch.bfloat16, device=DEV), torch.zeros(n, C, dtype=torch.bfloat16, device=DEV)
    N.moe_gather(h, row_src, K, xp, n_rows=seg[-1:])
    w = (torch.randn(E, C, C, generator=g) * C ** -0.5).to(torch.bfloat16).to(DEV)
    ptrs = torch.tensor([w[e].data_ptr() for e in range(E)], dtype=torch.int64, device=DEV)
    N.gemm_bf16_segmented(xp, ptrs, yp, seg, N.SEG_ROWS)
    y, out = torch.empty_like(x), torch.empty_like(x)
    N.moe_combine(yp, pos, K, y, gate=gate.view(-1))
    N.dropout_add(y, out, rng, 0.2, resid=h, site=1)
    hd, wd = h.cpu().double(), w.cpu().double()
    gd, ix = gate.cpu().double(), idx.cpu().long()
    ref, size = torch.zeros(T, C, dtype=torch.float64), torch.zeros(T, C, dtype=torch.float64)
    for t in range(cu[-1]):
        for j in range(K):
            row = wd[ix[t, j]] @ hd[t]
            ref[t] += gd[t, j] * row
            size[t] += gd[t, j] * (row.abs() * U + (wd[ix[t, j]].abs() @ hd[t].abs()) * (C + 8) * 2.0 ** -24)
    f1 = O.dropout_factors(n // K * C, 0.2, seed, offset, 1).view(T, C)
    want = hd + f1 * ref
    within(out, want, f1 * (size + U * ref.abs()) * 1.01 + U * want.abs() + 2.0 ** -20, "layer output")

    dout = torch.randn(T, C, generator=g).to(torch.bfloat16).to(DEV)
    dy, dl = torch.empty_like(dout), torch.empty_like(logits)
    N.dropout_bwd(dout, dy, rng, 0.2, site=1)
    assert torch.equal(dy.cpu() == 0, (f1 == 0) | (dout.cpu() == 0))
    N.moe_route_bwd(logits, idx, dl, dout=dy, y=yp, pos=pos, scoring="softmax")
    xr = logits[:cu[-1]].cpu().double().requires_grad_(True)
    _, gate_r = O.moe_route(xr, K, idx=ix[:cu[-1]], scoring="softmax")
    rows = yp.cpu().double()[pos[:cu[-1] * K].cpu().long()].view(-1, K, C)
    dg = (rows * dy[:cu[-1]].cpu().double()[:, None]).sum(-1)
    want, = torch.autograd.grad((gate_r * dg).sum(), xr)
    slack = 2.0 ** -14 * (rows.abs() * dy[:cu[-1]].cpu().double().abs()[:, None]).sum(-1).amax(-1, keepdim=True)
    within(dl[:cu[-1]], want, U * want.abs() + slack, "dlogits")
    assert bool((dl[cu[-1]:] == 0).all())
