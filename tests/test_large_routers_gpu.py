"""Stages whose mixture-of-experts layers have as many experts, and as many of them per token, as the router takes."""
import copy

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


@pytest.mark.parametrize("E,routing", [
    (512, dict(top_k=16, scoring="sigmoid", n_group=8, topk_group=4, group_score="top2", routed_scale=2.5, balance_bias=True)),
    (500, dict(top_k=10, n_group=4, topk_group=2)),
    (257, dict(top_k=8, scoring="sigmoid", norm_topk=False)),
    (256, dict(top_k=2)),
])
def test_a_pipeline_of_layers_with_many_experts_matches_the_oracle(E, routing):
    """Two native stages, a layer each; the oracle gets the run's own selection, which is compared with the definition on the
    run's own router logits."""
    import pippy_amd as pp
    from pippy_amd.configs import MoEDecoderLM, equal_split_spec
    torch.manual_seed(E)
    M, S, vocab, L, K = 2, 80, 128, 2, routing["top_k"]
    model = MoEDecoderLM(vocab=vocab, dim=64, n_layers=L, n_heads=1, ffn=64, n_experts=E, **routing)
    with torch.no_grad():
        for layer in model.h:
            layer.block_sparse_moe.gate.weight.mul_(10)     # decisive routing
            if routing.get("balance_bias"):
                layer.block_sparse_moe.balance_bias.normal_(std=0.1)
    ref, ref16 = copy.deepcopy(model).float(), copy.deepcopy(model)
    ids = torch.randint(0, vocab, (2 * M, S))
    target = torch.randint(0, vocab, (2 * M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    stages = [pp.PipelineStage(pipe, i, DEV) for i in range(2)]
    assert all(st.is_native for st in stages), [st.eager_reason for st in stages]
    losses = []
    out = pp.Schedule1F1B(stages, M, loss_fn=pp.CrossEntropyLoss()).step(ids.to(DEV), target=target.to(DEV), losses=losses)
    torch.cuda.synchronize()
    routed = [[] for _ in range(L)]
    for l, st in enumerate(stages):
        layer = ref.h[l]
        bias = layer.block_sparse_moe.balance_bias.double() if routing.get("balance_bias") else None
        how = {k: v for k, v in layer.routing.items() if k in ("scoring", "n_group", "topk_group", "group_score")}
        for m in range(M):
            acts = st.saved_activations(m)
            (idx,), (logits,), (seg,) = ([v for k, v in acts.items() if k.endswith(name)]
                                         for name in ("topk_idx", "router_logits", "seg_start"))
            want, _ = O.moe_route(logits[:, :E].double().cpu(), K, bias=bias, **how)
            assert torch.equal(idx.cpu().long(), want) and int(seg[-1]) == 2 * S * K
            routed[l].append(want)

    def oracle(of):
        for l in range(L):
            of.h[l].forced_routing = list(routed[l])
        stages_of = [nn.Sequential(of.embed, of.h[0]), nn.Sequential(of.h[1], of.head)]
        return OP.step(stages_of, ids, target, M, _ce)

    ref_out, ref_losses = oracle(ref)
    assert_close_rel(out, ref_out, BF16_TOL, "merged logits")
    for a, b in zip(losses, ref_losses):
        assert_close_rel(a.reshape(1), b.reshape(1), BF16_TOL, "loss")
    named, ref_named = dict(model.named_parameters()), dict(ref.named_parameters())
    # the experts of a layer as one tensor each: a few tokens of every expert average little out, so the roundings between
    # the loss and the first layer's experts count one by one.  On the shortest way they are those of the logits' gradient,
    # the head's input gradient, its norm's, two residual sums in one layer, the weighted rows, dh and du, and on the other
    # factor the embedding, the residual sum, the norm and the gate: 12, each by at most 2^-8 of its value
    for l in range(L):
        for w in ("w1", "w2", "w3"):
            names = [f"h.{l}.block_sparse_moe.experts.{e}.{w}.weight" for e in range(E)]
            zero = torch.zeros_like(ref_named[names[0]])
            want = torch.stack([zero if ref_named[n].grad is None else ref_named[n].grad for n in names])
            got = torch.stack([named[n].main_grad.cpu() for n in names])
            assert max_rel(got, want) <= 12 * 2.0 ** -8, f"{w} of layer {l}"
            assert bool((got[[ref_named[n].grad is None for n in names]] == 0).all())   # an expert without tokens

    def run_in_bf16():
        oracle(ref16)
        return dict(ref16.named_parameters())

    rest = {n: rp for n, rp in ref_named.items() if ".experts." not in n}
    check_gradients(named, rest, run_in_bf16, f"{E} experts")
