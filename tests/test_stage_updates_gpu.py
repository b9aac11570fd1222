"""What a native stage reads of its blocks beside parameters (a router's balancing bias, a layer's dropout rate) is what the
module holds when a step runs, whatever was done to it between two steps."""
import pytest
import torch

from oracle import ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
K, E, L, M, S, VOCAB = 2, 12, 2, 2, 64, 128


# ---- the balancing bias of a router ----------------------------------------------------------------------------
def moe_model():
    from pippy_amd.configs import MoEDecoderLM
    torch.manual_seed(3)
    return MoEDecoderLM(vocab=VOCAB, dim=64, n_layers=L, n_heads=1, ffn=64, n_experts=E, top_k=K, scoring="sigmoid",
                        balance_bias=True)


def moe_pipeline(model):
    import pippy_amd as pp
    from pippy_amd.configs import equal_split_spec
    ids = torch.randint(0, VOCAB, (M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    stages = [pp.PipelineStage(pipe, i, DEV, group=1) for i in range(2)]
    assert all(st.is_native for st in stages), [st.eager_reason for st in stages]
    sched = pp.ScheduleGPipe(stages, M, loss_fn=pp.CrossEntropyLoss())
    target = torch.randint(0, VOCAB, (M, S)).to(DEV)
    ids = ids.to(DEV)

    def step():
        sched.zero_grad()
        sched.step(ids, target=target, losses=[])
        torch.cuda.synchronize()

    return stages, step


def selected_under(stages, biases):
    """Every layer's selection is the definition's on the run's own logits under the bias given for it."""
    for s, st in enumerate(stages):
        for m in range(M):
            acts = st.saved_activations(m)
            idx, = (v for k, v in acts.items() if k.endswith("topk_idx"))
            logits, = (v for k, v in acts.items() if k.endswith("router_logits"))
            want, _ = O.moe_route(logits[:, :E].double().cpu(), K, scoring="sigmoid", bias=biases[s].double().cpu())
            assert torch.equal(idx.cpu().long(), want), f"stage {s}, microbatch {m}"


def pushing(expert):
    bias = torch.zeros(E)
    bias[expert] = 5.0
    return bias


def test_the_balancing_bias_is_followed_in_place_through_a_reference_taken_before_the_first_step():
    model = moe_model()
    held = [layer.block_sparse_moe.balance_bias for layer in model.h]
    stages, step = moe_pipeline(model)
    step()
    selected_under(stages, [torch.zeros(E)] * L)
    for first in (1, 7):
        for l, bias in enumerate(held):
            bias.zero_()
            bias[first + l] += 5.0
        step()
        selected_under(stages, [pushing(first), pushing(first + 1)])
        for layer, bias in zip(model.h, held):
            assert torch.equal(layer.block_sparse_moe.balance_bias.cpu(), bias.cpu())


def test_the_balancing_bias_is_followed_when_it_is_replaced():
    model = moe_model()
    stages, step = moe_pipeline(model)
    step()
    moe = [layer.block_sparse_moe for layer in model.h]
    for e, place in enumerate((lambda b: b, lambda b: b.to(DEV), lambda b: b.to(DEV).bfloat16(), lambda b: b.double(),
                               lambda b: torch.stack([b, b], -1)[:, 0])):
        for l, m in enumerate(moe):
            m.balance_bias = place(pushing(e + l))
        # what the old storage would be reused for
        junk = [torch.full((E,), -9.0, device=DEV) for _ in range(64)]
        step()
        selected_under(stages, [pushing(e), pushing(e + 1)])
        for l, m in enumerate(moe):                     # and in place from there on
            m.balance_bias.copy_(pushing(e + l + 3))
        step()
        selected_under(stages, [pushing(e + 3), pushing(e + 4)])
        del junk
    for l, m in enumerate(moe):
        m.load_state_dict({**m.state_dict(), "balance_bias": pushing(9 + l).to(DEV)}, assign=True)
    step()
    selected_under(stages, [pushing(9), pushing(10)])
    for l, m in enumerate(moe):
        m.load_state_dict({**m.state_dict(), "balance_bias": pushing(2 + l)})
    step()
    selected_under(stages, [pushing(2), pushing(3)])


def test_two_pipelines_over_one_model_read_the_same_balancing_bias():
    import pippy_amd as pp
    from pippy_amd.configs import equal_split_spec
    model = moe_model()
    stages, step = moe_pipeline(model)
    step()
    ids = torch.randint(0, VOCAB, (M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    others = [pp.PipelineStage(pipe, i, DEV, group=1) for i in range(2)]
    sched = pp.ScheduleGPipe(others, M)
    for e in (4, 8):
        for l, layer in enumerate(model.h):
            layer.block_sparse_moe.balance_bias = pushing(e + l)
        sched.step(ids.to(DEV))
        torch.cuda.synchronize()
        selected_under(others, [pushing(e), pushing(e + 1)])
        step()
        selected_under(stages, [pushing(e), pushing(e + 1)])


def test_a_balancing_bias_that_does_not_fit_is_refused():
    model = moe_model()
    stages, step = moe_pipeline(model)
    step()
    for bad in (torch.zeros(E + 1), None):
        model.h[0].block_sparse_moe.balance_bias = bad
        with pytest.raises(RuntimeError, match="balance_bias"):
            step()
        model.h[0].block_sparse_moe.balance_bias = pushing(3)
        for st in stages:
            st.clear_runtime_states()
    step()
    selected_under(stages, [pushing(3), torch.zeros(E)])


def test_a_tensor_assigned_as_balancing_bias_stays_where_it_is_and_is_read_anew_every_step():
    model = moe_model()
    stages, step = moe_pipeline(model)
    own = [pushing(1), pushing(2)]
    for layer, bias in zip(model.h, own):
        layer.block_sparse_moe.balance_bias = bias
    for e in (1, 6):
        for l, bias in enumerate(own):
            bias.copy_(pushing(e + l))
        step()
        selected_under(stages, [pushing(e), pushing(e + 1)])
        assert all(layer.block_sparse_moe.balance_bias is bias and bias.device.type == "cpu"
                   for layer, bias in zip(model.h, own))

def test_a_balancing_bias_that_was_put_aside_keeps_its_values():
    model = moe_model()
    stages, step = moe_pipeline(model)
    first = [layer.block_sparse_moe.balance_bias for layer in model.h]
    step()
    for l, layer in enumerate(model.h):
        layer.block_sparse_moe.balance_bias = first[l] + pushing(4 + l).to(first[l].device)
    step()
    selected_under(stages, [pushing(4), pushing(5)])
    for layer, bias in zip(model.h, first):
        assert bool((bias == 0).all())
        layer.block_sparse_moe.balance_bias = bias
    step()
    selected_under(stages, [torch.zeros(E)] * L)


# ---- the dropout rate of a layer ------------------------------------------------------------------------------
def dropout_pipeline(**options):
    import pippy_amd as pp
    from pippy_amd.configs import DecoderLM, equal_split_spec
    torch.manual_seed(6)
    model = DecoderLM(vocab=VOCAB, max_seq=S, dim=64, n_layers=L, n_heads=1, ffn=128, **options)
    ids = torch.randint(0, VOCAB, (M, S))
    pipe = pp.pipeline(model, M, (ids,), split_spec=equal_split_spec(L, 2))
    stages = [pp.PipelineStage(pipe, i, DEV) for i in range(2)]
    assert all(st.is_native for st in stages), [st.eager_reason for st in stages]
    sched = pp.ScheduleGPipe(stages, M, loss_fn=pp.CrossEntropyLoss())
    target = torch.randint(0, VOCAB, (M, S)).to(DEV)
    ids = ids.to(DEV)

    def step():
        sched.zero_grad()
        out = sched.step(ids, target=target, losses=[]).clone()
        torch.cuda.synchronize()
        return out, {n: p.main_grad.clone() for n, p in model.named_parameters()}

    return model, stages, step


def same(a, b):
    return torch.equal(a[0], b[0]) and all(torch.equal(v, b[1][n]) for n, v in a[1].items())


def test_a_dropout_rate_changed_between_steps_is_followed():
    """A pipeline built at one rate and set to another gives what one built at that rate gives from the same state."""
    def at(rate, offset):
        model, stages, step = dropout_pipeline(dropout=rate)
        if rate:
            for st in stages:
                for m in range(M):
                    st._stage_program().rng_state(m)[1] += offset
        return step()

    model, stages, step = dropout_pipeline(dropout=0.0)
    assert same(step(), at(0.0, 0))
    for n, rate in enumerate((0.2, 0.5, 0.0, 0.1)):         # (a step without dropout does not move the state)
        for layer in model.h:
            layer.dropout = rate
        assert same(step(), at(rate, n if rate != 0.1 else n - 1)), rate
    for layer in model.h:
        layer.dropout = 0                                   # an integer is a rate, too
    assert same(step(), at(0.0, 0))


@pytest.mark.parametrize("rate", [1.0, -0.1, float("nan")])
def test_a_dropout_rate_out_of_range_is_refused(rate):
    model, stages, step = dropout_pipeline(dropout=0.1)
    step()
    model.h[1].dropout = rate
    with pytest.raises(RuntimeError, match="dropout"):
        step()
    model.h[1].dropout = 0.1
    for st in stages:
        st.clear_runtime_states()
    step()


@pytest.mark.parametrize("pre_ln", [True, False])
def test_dropout_keeps_no_activation_of_its_own(pre_ln):
    """What a microbatch keeps for its backward is the same with dropout and without: the mask is formed again, and nothing
    reads the branches in front of it."""
    kept = []
    for rate in (0.0, 0.2):
        _, stages, step = dropout_pipeline(dropout=rate, pre_ln=pre_ln)
        step()
        kept.append([sorted((tuple(t.shape), t.dtype) for t in st.saved_activations(0).values()) for st in stages])
    assert kept[0] == kept[1]
