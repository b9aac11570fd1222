"""Stages whose blocks use the routing, permutation and dropout kernels, end to end against the fp32 oracle."""
import copy
import statistics

import pytest
import torch
import torch.nn as nn

from _util import BF16_TOL, assert_close_rel, check_gradients, max_rel
from oracle import ops as O
from oracle import pipeline as OP

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ce(o, t):
    return nn.functional.cross_entropy(o.reshape(-1, o.shape[-1]), t.reshape(-1))


def _reference_stages(ref, n_stages):
    per = len(ref.h) // n_stages
    parts = [list(ref.h[s * per:(s + 1) * per]) for s in range(n_stages)]
    parts[0].insert(0, ref.embed)
    parts[-1].append(ref.head)
    return [nn.Sequential(*p) for p in parts]


ROUTERS = [
    (12, dict(top_k=3, scoring="sigmoid", routed_scale=2.5, balance_bias=True)),
    (16, dict(top_k=4, scoring="sigmoid", n_group=4, topk_group=2, group_score="top2", balance_bias=True)),
    (72, dict(top_k=6, norm_topk=False)),
    (9, dict(top_k=1, n_group=3, topk_group=1)),
]


@pytest.mark.parametrize("E,routing", ROUTERS)
def test_a_mixture_of_experts_pipeline_with_any_router_matches_the_oracle(E, routing):
    """Two native stages under interleaved 1F1B; the oracle gets the run's own selection, which is compared with the
    definition on the run's own router logits."""
    import pippy_amd as pp
    from pippy_amd.configs import MoEDecoderLM, equal_split_spec
    torch.manual_seed(E)
    M, S, vocab, L, K = 4, 96, 256, 4, routing["top_k"]
    model = MoEDecoderLM(vocab=vocab, dim=128, n_layers=L, n_heads=2, ffn=128, n_experts=E, **routing)
    with torch.no_grad():
        for layer in model.h:
            layer.block_sparse_moe.gate.weight.mul_(10)     # decisive routing
            if routing.get("balance_bias"):
                layer.block_sparse_moe.balance_bias.normal_(std=0.1)
    ref, ref16 = copy.deepcopy(model).float(), copy.deepcopy(model)
    ids = torch.randint(0, vocab, (2 * M, S))
    target = torch.randint(0, vocab, (2 * M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    stages = [pp.PipelineStage(pipe, i, DEV, group=1) for i in range(2)]
    assert all(st.is_native for st in stages), [st.eager_reason for st in stages]
    losses = []
    out = pp.ScheduleInterleaved1F1B(stages, M, loss_fn=pp.CrossEntropyLoss()).step(
        ids.to(DEV), target=target.to(DEV), losses=losses)
    torch.cuda.synchronize()
    routed = [[] for _ in range(L)]
    for s, st in enumerate(stages):
        for m in range(M):
            acts = st.saved_activations(m)
            idx, logits, seg = ([v for k, v in acts.items() if k.endswith(name)]
                                for name in ("topk_idx", "router_logits", "seg_start"))
            for j in range(L // 2):
                layer = ref.h[s * (L // 2) + j]
                bias = layer.block_sparse_moe.balance_bias.double() if routing.get("balance_bias") else None
                how = {k: v for k, v in layer.routing.items() if k in ("scoring", "n_group", "topk_group", "group_score")}
                want, _ = O.moe_route(logits[j][:, :E].double().cpu(), K, bias=bias, **how)
                assert torch.equal(idx[j].cpu().long(), want)
                assert int(seg[j][-1]) == 2 * S * K
                routed[s * (L // 2) + j].append(idx[j].cpu().long())
    for l in range(L):
        ref.h[l].forced_routing = list(routed[l])
    ref_out, ref_losses = OP.step(_reference_stages(ref, 2), ids, target, M, _ce)
    assert_close_rel(out, ref_out, BF16_TOL, "merged logits")
    for a, b in zip(losses, ref_losses):
        assert_close_rel(a.reshape(1), b.reshape(1), BF16_TOL, "loss")
    named, ref_named = dict(model.named_parameters()), dict(ref.named_parameters())
    for name in [n for n, rp in ref_named.items() if rp.grad is None]:      # an expert without tokens
        assert float(named[name].main_grad.abs().max()) == 0.0, name
        del ref_named[name]
    if K == 1:      # the weight of a single expert is 1 whatever its logit: no gradient
        for name in [n for n in ref_named if n.endswith("gate.weight")]:
            assert float(named[name].main_grad.abs().max()) <= 1e-7, name
            del ref_named[name]

    def run_in_bf16():
        again = copy.deepcopy(ref16)
        for l in range(L):
            again.h[l].forced_routing = list(routed[l])
        OP.step(_reference_stages(again, 2), ids, target, M, _ce)
        return dict(again.named_parameters())

    # An expert sees about 2 S K / E tokens of a microbatch (16 with 72 experts), so little averages out in its
    # weights' gradients.  Between the loss and those of the first layer lie 16 roundings to bf16 on the shortest way: of
    # the logits' gradient, the head's input gradient and its norm's; two residual sums in each of three layers; the
    # weighted rows, dh and du; and on the other factor the embedding, the residual sum, the norm and the gate.  Each
    # is off by at most 2^-8 of its value: 16 x 2^-8 = 6.3e-2.  That nothing but rounding is at work shows in the
    # median over the experts, which is that of torch's own bf16 autograd (the same noise drawn again).
    experts = [n for n in ref_named if ".experts." in n]
    mine = [max_rel(named[n].main_grad, ref_named[n].grad) for n in experts]
    assert max(mine) <= 16 * 2.0 ** -8, max(mine)
    if max(mine) > BF16_TOL:
        theirs = run_in_bf16()
        theirs = [max_rel(theirs[n].grad.float(), ref_named[n].grad) for n in experts]
        assert statistics.median(mine) <= 1.5 * statistics.median(theirs)
    rest = {n: rp for n, rp in ref_named.items() if ".experts." not in n}
    check_gradients(named, rest, run_in_bf16, f"{E} experts")


def test_the_torch_statement_of_the_selection_is_the_definition():
    from pippy_amd.stage_modules import MoELayer
    torch.manual_seed(3)
    for E, routing in ROUTERS:
        layer = MoELayer(64, 1, 64, E, dtype=torch.float32, **routing)
        if routing.get("balance_bias"):
            layer.block_sparse_moe.balance_bias.normal_(std=0.1)
        logits = torch.randn(40, E, dtype=torch.float64)
        score = torch.softmax(logits, -1) if layer.routing["scoring"] == "softmax" else torch.sigmoid(logits)
        how = {k: v for k, v in layer.routing.items() if k not in ("renorm", "scale")}
        bias = layer._balance_bias()
        want, _ = O.moe_route(logits, routing["top_k"], bias=None if bias is None else bias.double(), **how)
        assert torch.equal(layer._select(logits, score), want)


def _masks(stage, n_layers, M, shape, p):
    """Per layer and branch, the factor of every microbatch's last forward, from the states the kernels used."""
    sp = stage._stage_program()
    per_layer = [([], []) for _ in range(n_layers)]
    for m in range(M):
        seed, offset = sp.rng_state(m).tolist()
        for l in range(n_layers):
            for which in range(2):
                f = O.dropout_factors(shape.numel(), p, seed, offset, 2 * l + which).view(shape)
                per_layer[l][which].append(f.float())
    return per_layer


@pytest.mark.parametrize("schedule", ["Schedule1F1B", "ScheduleZeroBubble"])
@pytest.mark.parametrize("pre_ln", [True, False])
def test_a_pipeline_with_dropout_matches_the_oracle_under_the_same_masks(schedule, pre_ln):
    import pippy_amd as pp
    from pippy_amd.configs import DecoderLM, equal_split_spec
    torch.manual_seed(5)
    M, S, vocab, L, dim, p = 3, 64, 128, 4, 64, 0.2
    model = DecoderLM(vocab=vocab, max_seq=S, dim=dim, n_layers=L, n_heads=1, ffn=128, pre_ln=pre_ln, dropout=p)
    ref = copy.deepcopy(model).float()
    ids = torch.randint(0, vocab, (M, S))
    target = torch.randint(0, vocab, (M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    stages = [pp.PipelineStage(pipe, i, DEV) for i in range(2)]
    assert all(st.is_native for st in stages), [st.eager_reason for st in stages]
    sched = getattr(pp, schedule)(stages, M, loss_fn=pp.CrossEntropyLoss())
    outs = []
    for _ in range(2):                                       # the second step draws other masks
        sched.zero_grad()
        losses = []
        outs.append(sched.step(ids.to(DEV), target=target.to(DEV), losses=losses).clone())
    torch.cuda.synchronize()
    assert not torch.equal(outs[0], outs[1])
    for s, st in enumerate(stages):
        masks = _masks(st, L // 2, M, torch.Size((1, S, dim)), p)
        assert st._stage_program().rng_state(1).tolist()[1] == (1 << 32) + 2
        for l in range(L // 2):
            layer = ref.h[s * (L // 2) + l]
            layer._drop = lambda branch, which, own=masks[l]: branch * own[which].pop(0)
    ref_out, ref_losses = OP.step(_reference_stages(ref, 2), ids, target, M, _ce)
    assert_close_rel(outs[1], ref_out, BF16_TOL, "merged logits")
    for a, b in zip(losses, ref_losses):
        assert_close_rel(a.reshape(1), b.reshape(1), BF16_TOL, "loss")
    named = dict(model.named_parameters())
    for name, rp in ref.named_parameters():
        err = max_rel(named[name].main_grad, rp.grad)
        assert err <= BF16_TOL, f"grad of {name}: max relative error {err:.3e}"


def test_dropout_follows_the_mode_of_the_model():
    """Eval mode runs without masks and repeats itself; back in training mode the masks go on where they were."""
    import pippy_amd as pp
    from pippy_amd.configs import DecoderLM, equal_split_spec
    torch.manual_seed(6)
    M, S, vocab = 2, 64, 128
    model = DecoderLM(vocab=vocab, max_seq=S, dim=64, n_layers=2, n_heads=1, ffn=128, dropout=0.3)
    plain = copy.deepcopy(model)
    for layer in plain.h:
        layer.dropout = 0.0
    ids = torch.randint(0, vocab, (M, S)).to(DEV)

    def run(m):
        pipe = pp.pipeline(m, M, (ids.cpu(),), split_spec=equal_split_spec(2, 2))
        stages = [pp.PipelineStage(pipe, i, DEV) for i in range(2)]
        assert all(st.is_native for st in stages)
        return pp.ScheduleGPipe(stages, M), stages

    sched, stages = run(model)
    without = run(plain)[0].step(ids).clone()
    first = sched.step(ids).clone()
    for st in stages:
        st.submod.eval()
    quiet = [sched.step(ids).clone() for _ in range(2)]
    assert torch.equal(quiet[0], quiet[1]) and torch.equal(quiet[0], without)
    for st in stages:
        st.submod.train()
    second = sched.step(ids).clone()
    assert not torch.equal(first, without) and not torch.equal(first, second)
    assert stages[0]._stage_program().rng_state(0).tolist()[1] == 2


def test_blocks_refuse_options_that_do_not_fit():
    from pippy_amd.stage_modules import MoELayer, TransformerLayer
    for bad in (dict(dropout=1.0), dict(dropout=-0.1)):
        with pytest.raises(ValueError, match="dropout"):
            TransformerLayer(64, 1, 64, **bad)
    for bad in (dict(top_k=17, n_experts=64), dict(n_group=5), dict(n_group=4, topk_group=1, top_k=3),
                dict(scoring="tanh"), dict(top_k=3, group_score="mean"), dict(n_experts=513), dict(top_k=0)):
        with pytest.raises(ValueError):
            MoELayer(64, 1, 64, **dict(dict(n_experts=8), **bad))
