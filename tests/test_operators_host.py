"""Packed attention, routing, permutation and dropout without a GPU: the oracle's statements pinned to something
outside of them, and what the C entry points refuse (they check on the host, before anything is launched)."""
import ctypes as C

import pytest
import torch

from oracle import ops as O
from pippy_amd import _native as N
from pippy_amd.stage_modules import MoELayer


# ---- the oracle -----------------------------------------------------------------------------------
def test_packed_attention_is_attention_of_every_sequence():
    torch.manual_seed(0)
    cu = [0, 3, 3, 10, 11]
    q = torch.randn(12, 4, 8, dtype=torch.float64)
    k, v = torch.randn(2, 12, 2, 8, dtype=torch.float64).unbind(0)
    for causal in (True, False):
        o, lse = O.attention_packed(q, k, v, cu, causal)
        assert bool((o[11] == 0).all()) and bool((lse[:, 11] == 0).all())
        for a, b in zip(cu[:-1], cu[1:]):
            if a == b:
                continue
            qs, ks, vs = (t[a:b].transpose(0, 1)[None] for t in (q, k.repeat_interleave(2, 1), v.repeat_interleave(2, 1)))
            want = torch.nn.functional.scaled_dot_product_attention(qs, ks, vs, is_causal=causal)[0].transpose(0, 1)
            assert torch.allclose(o[a:b], want, rtol=1e-12, atol=1e-12)
    # the log-sum-exp of one visible key is its score
    assert torch.allclose(O.attention_packed(q, k, v, cu, True)[1][3, 10], (q[10, 3] * k[10, 1]).sum() * 8 ** -0.5)


def test_routing_agrees_with_topk_and_with_the_top2_router():
    torch.manual_seed(1)
    x = torch.randn(50, 12, dtype=torch.float64)
    idx, gate = O.moe_route(x, 3)
    assert torch.equal(idx, torch.topk(x, 3, -1).indices)
    assert torch.allclose(gate, torch.softmax(torch.topk(x, 3, -1).values, -1))
    i2, g2 = O.moe_route_top2(x)
    idx, gate = O.moe_route(x, 2)
    assert torch.equal(idx, i2) and torch.allclose(gate, g2.double(), atol=1e-6)
    # a bias moves the selection, not the weights; groups keep the experts of the best groups only
    bias = torch.zeros(12, dtype=torch.float64)
    bias[7] = 10.0
    idx, gate = O.moe_route(x, 2, "sigmoid", bias=bias, renorm=False)
    assert bool((idx[:, 0] == 7).all()) and torch.allclose(gate[:, 0], torch.sigmoid(x[:, 7]))
    idx, _ = O.moe_route(x, 2, n_group=4, topk_group=1)
    assert torch.equal(idx[:, 0], x.argmax(-1)) and bool((idx[:, 0] // 3 == idx[:, 1] // 3).all())
    # experts taken out
    x[0] = float("-inf")
    x[1, 1:] = float("-inf")
    idx, gate = O.moe_route(x, 2)
    assert idx[:2].tolist() == [[-1, -1], [0, -1]] and gate[:2].tolist() == [[0, 0], [1, 0]]


def test_dropout_refuses_rows_that_overlap():
    """Expanded and overlapping rows have no leading dimension that the kernels could take."""
    x = torch.zeros(4, 16)
    for bad in (torch.zeros(1, 16).expand(4, 16), torch.zeros(64).as_strided((4, 16), (8, 1))):
        with pytest.raises(ValueError, match="overlap"):
            N._dropout_rows(bad, x, None)
        with pytest.raises(ValueError, match="overlap"):
            N._dropout_rows(x, x, bad)
    assert N._dropout_rows(torch.zeros(4, 24)[:, :16], x, None) == (4, 16, 24, 0, 16)
    assert N._dropout_rows(torch.zeros(4, 24)[:1, :16], x[:1], None) == (1, 16, 16, 16, 16)


def test_moe_layer_refuses_groups_that_do_not_exist():
    for bad in (dict(topk_group=3), dict(group_score="mean"), dict(n_group=3), dict(n_group=4, topk_group=5), dict(top_k=9)):
        with pytest.raises(ValueError):
            MoELayer(128, 2, 16, 8, **bad)


def test_philox_known_answers():
    """The vectors that the generator's authors publish with it."""
    assert O.philox4x32_10([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert O.philox4x32_10([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert O.philox4x32_10([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_dropout_factors_have_the_right_rate_and_mean():
    f = O.dropout_factors(20000, 0.1, seed=7, offset=3, site=1)
    # 20000 draws of rate 0.1: a standard deviation of 0.0021, five of them
    assert abs(float((f == 0).double().mean()) - 0.1) < 0.0106 and abs(float(f.mean()) - 1.0) < 0.012
    assert not torch.equal(f, O.dropout_factors(20000, 0.1, seed=7, offset=4, site=1))
    assert not torch.equal(f, O.dropout_factors(20000, 0.1, seed=7, offset=3, site=2))
    assert bool((O.dropout_factors(64, 0.0, 1, 1, 1) == 1).all()) and bool((O.dropout_factors(64, 1.0, 1, 1, 1) == 0).all())


# ---- what the entry points refuse -------------------------------------------------------------------
A, B = 0x10000, 0x20000     # stand-ins for 16-byte aligned device addresses; nothing is launched


def refused(rc, match):
    assert rc in (N.PP_ERR_INVALID, N.PP_ERR_UNSUPPORTED)
    assert match in N.lib().pp_last_error().decode()


def packed(**change):
    d = N.AttnPackedDesc()
    for name in ("q", "k", "v", "o", "lse", "d_o", "dq", "dk", "dv", "delta", "plan"):
        setattr(d, name, A)
    d.n_seq, d.T, d.H, d.Hkv, d.D = 2, 100, 8, 2, 64
    for name in ("q", "o", "do", "dq"):
        setattr(d, "stride_" + name, 512)
    for name in ("k", "v", "dk", "dv"):
        setattr(d, "stride_" + name, 128)
    d.scale, d.causal = 0.125, 1
    for name, value in change.items():
        setattr(d, name, value)
    return C.byref(d)


@pytest.mark.parametrize("change,match", [
    (dict(T=-1), "bad shape"), (dict(T=2 ** 31), "bad shape"), (dict(n_seq=-1), "bad shape"), (dict(H=0), "bad shape"),
    (dict(Hkv=3), "bad shape"), (dict(Hkv=0), "bad shape"), (dict(D=96), "head_dim"), (dict(scale=0.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=None), "q must"),
    (dict(k=A + 8), "k must"), (dict(o=A + 2), "o must"), (dict(stride_q=504), "stride"), (dict(stride_k=132), "stride"),
    (dict(stride_v=2 ** 23 + 8), "stride"), (dict(lse=None), "null"), (dict(plan=None), "null"),
    (dict(plan=A + 4), "null"), (dict(T=2 ** 31 - 64, H=1024, Hkv=8, stride_q=65536, stride_o=65536, stride_k=512,
                                      stride_v=512), "grid"),
])
def test_packed_attention_refuses(change, match):
    refused(N.lib().pp_attn_packed_fwd(packed(**change), None), match)


@pytest.mark.parametrize("change,match", [(dict(scale=1e-30), "scale"), (dict(scale=1e30), "scale"), (dict(H=2 ** 18), "shape")])
def test_packed_attention_refuses_sizes_beyond_its_arithmetic(change, match):
    refused(N.lib().pp_attn_packed_fwd(packed(**change), None), match)


@pytest.mark.parametrize("change,match", [
    (dict(d_o=None), "d_o must"), (dict(dq=A + 4), "dq must"), (dict(stride_dk=120), "stride"), (dict(delta=None), "null"),
])
def test_packed_attention_backward_refuses(change, match):
    refused(N.lib().pp_attn_packed_bwd(packed(**change), None), match)


def test_packed_plan_refuses():
    L = N.lib()
    assert L.pp_attn_packed_plan_ints(-1, 5) == L.pp_attn_packed_plan_ints(5, -1) == L.pp_attn_packed_plan_ints(1, 2 ** 31) == -1
    assert L.pp_attn_packed_plan_ints(0, 0) > 0
    refused(L.pp_attn_packed_plan(A, -1, 5, A, None), "bad shape")
    refused(L.pp_attn_packed_plan(None, 1, 5, A, None), "null")
    refused(L.pp_attn_packed_plan(A, 1, 5, None, None), "null")
    refused(L.pp_attn_packed_plan(A, 1, 5, A + 4, None), "16-byte")


def route(**change):
    d = N.MoeRouteDesc()
    for name in ("logits", "topk_idx", "gate", "dgate", "dlogits"):
        setattr(d, name, A)
    d.ld, d.T, d.E, d.topk, d.scale = 64, 10, 64, 6, 1.0
    d.cols_dl = d.ld_dl = 64
    for name, value in change.items():
        setattr(d, name, value)
    return C.byref(d)


@pytest.mark.parametrize("change,match", [
    (dict(T=-1), "bad shape"), (dict(E=1), "bad shape"), (dict(E=513, ld=513), "bad shape"), (dict(topk=0), "bad shape"),
    (dict(topk=17), "bad shape"), (dict(E=4, topk=5), "bad shape"), (dict(ld=63), "bad shape"),
    (dict(scoring=2), "scoring"), (dict(dtype=2), "dtype"), (dict(logits=None), "null"), (dict(topk_idx=None), "null"),
    (dict(gate=None), "null"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(n_group=3, topk_group=1), "groups"), (dict(n_group=8, topk_group=0), "groups"),
    (dict(n_group=8, topk_group=9), "groups"), (dict(n_group=32, topk_group=2), "groups"),
    (dict(n_group=8, topk_group=2, group_score=2), "groups"), (dict(E=130, ld=130, n_group=65, topk_group=9), "groups"),
])
def test_routing_refuses(change, match):
    refused(N.lib().pp_moe_route(route(**change), None), match)


@pytest.mark.parametrize("change,match", [
    (dict(dlogits=None), "dlogits"), (dict(cols_dl=63), "dlogits"), (dict(cols_dl=72), "dlogits"), (dict(ld_dl=60), "dlogits"),
    (dict(dgate=None), "needs dgate"), (dict(dgate=None, dout=A, y=A, pos=A, C=60, ld_dout=64, ld_y=64), "needs dgate"),
    (dict(dgate=None, dout=A, y=A + 8, pos=A, C=64, ld_dout=64, ld_y=64), "needs dgate"),
    (dict(dgate=None, dout=A, y=A, pos=A, C=64, ld_dout=56, ld_y=64), "needs dgate"),
])
def test_routing_backward_refuses(change, match):
    refused(N.lib().pp_moe_route_bwd(route(**change), None), match)


def test_permutation_refuses():
    L = N.lib()
    assert L.pp_moe_permute_workspace_ints(10, 1025) == L.pp_moe_permute_workspace_ints(-1, 8) == \
        L.pp_moe_permute_workspace_ints(10, 0) == L.pp_moe_permute_workspace_ints(2 ** 24 + 1, 8) == -1
    need = L.pp_moe_permute_workspace_ints(5000, 100)
    assert need >= 100
    refused(L.pp_moe_permute_ws(A, 5000, 1025, A, A, A, A, 1 << 20, None), "at most 1024 experts")
    refused(L.pp_moe_permute_ws(None, 5000, 100, A, A, A, A, need, None), "bad arguments")
    refused(L.pp_moe_permute_ws(A, 5000, 100, A, A, A, A, need - 1, None), "needs")
    refused(L.pp_moe_permute_ws(A, 5000, 100, A, A, A, None, need, None), "needs")


@pytest.mark.parametrize("change,match", [
    (dict(dtype=3), "dtype"), (dict(p=-0.1), "p must"), (dict(p=1.5), "p must"), (dict(p=float("nan")), "p must"),
    (dict(rows=-1), "bad shape"), (dict(x=None), "null"), (dict(x=A + 8), "aligned"), (dict(y=A + 2), "aligned"),
    (dict(resid=A + 4), "aligned"), (dict(rng=None), "null"), (dict(rng=A + 4), "aligned"), (dict(C=60), "multiples of 8"),
    (dict(ld_x=60), "multiples of 8"), (dict(ld_x=56), "multiples of 8"), (dict(resid=A, ld_r=68), "multiples of 8"),
    (dict(rows=1, C=2 ** 36), "2^35"), (dict(rows=2 ** 33, C=64), "2^35"),
])
def test_dropout_refuses(change, match):
    a = dict(x=A, ld_x=64, resid=None, ld_r=0, y=B, ld_y=64, rows=4, C=64, dtype=0, p=0.1, rng=A)
    a.update(change)
    refused(N.lib().pp_dropout_add(a["x"], a["ld_x"], a["resid"], a["ld_r"], a["y"], a["ld_y"], a["rows"], a["C"],
                                   a["dtype"], a["p"], a["rng"], 0, None), match)
    if "resid" not in change:
        refused(N.lib().pp_dropout_bwd(a["x"], a["ld_x"], a["y"], a["ld_y"], a["rows"], a["C"], a["dtype"], a["p"],
                                       a["rng"], 0, None), match)


def test_empty_calls_launch_nothing():
    L = N.lib()
    assert L.pp_attn_packed_fwd(packed(T=0), None) == L.pp_attn_packed_bwd(packed(n_seq=0), None) == N.PP_OK
    assert L.pp_moe_route(route(T=0), None) == L.pp_moe_route_bwd(route(T=0), None) == N.PP_OK
    assert L.pp_dropout_add(None, 0, None, 0, None, 0, 0, 64, 0, 0.1, None, 0, None) == N.PP_OK


def test_the_bindings_refuse_tensors_that_are_not_on_the_gpu():
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    rng = torch.zeros(2, dtype=torch.int64)
    idx, gate = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    for call in (lambda: N.dropout_add(x, x, rng, 0.1), lambda: N.dropout_bwd(x, x, rng, 0.1),
                 lambda: N.moe_route(x, idx, gate), lambda: N.moe_route_bwd(x, idx, x, dgate=gate),
                 lambda: N.moe_permute_ws(idx, 8, idx, idx, idx, idx), lambda: N.rng_advance(rng),
                 lambda: N.attn_packed_plan(idx.view(-1), 4)):
        with pytest.raises(RuntimeError, match="device tensors"):
            call()


def test_descriptor_layouts_match_the_header(tmp_path):
    import subprocess
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pippy_amd.h"\n'
                   'int main(void){printf("%zu %zu %zu %zu\\n", sizeof(pp_attn_packed_desc), offsetof(pp_attn_packed_desc, '
                   'scale), sizeof(pp_moe_route_desc), offsetof(pp_moe_route_desc, dgate));return 0;}\n')
    exe = tmp_path / "sizes"
    import pathlib
    inc = pathlib.Path(N.__file__).resolve().parent.parent / "include"
    subprocess.run(["gcc", "-I", str(inc), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(N.AttnPackedDesc), N.AttnPackedDesc.scale.offset, C.sizeof(N.MoeRouteDesc),
                   N.MoeRouteDesc.dgate.offset]
