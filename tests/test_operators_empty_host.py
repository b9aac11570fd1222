"""Empty batches: tensors without elements have no address, and the entry points take them."""
import ctypes as C

from pippy_amd import _native as N

A = 0x10000     # stands for a 16-byte aligned device address; nothing is launched


def test_the_entry_points_take_empty_tensors():
    L = N.lib()
    d = N.AttnPackedDesc()
    d.plan, d.n_seq, d.T, d.H, d.Hkv, d.D, d.scale = A, 2, 0, 8, 2, 64, 0.125
    for name in ("q", "o", "do", "dq"):
        setattr(d, "stride_" + name, 512)
    for name in ("k", "v", "dk", "dv"):
        setattr(d, "stride_" + name, 128)
    assert L.pp_attn_packed_fwd(C.byref(d), None) == L.pp_attn_packed_bwd(C.byref(d), None) == N.PP_OK
    r = N.MoeRouteDesc()
    r.ld, r.T, r.E, r.topk, r.scale, r.cols_dl, r.ld_dl = 64, 0, 64, 6, 1.0, 64, 64
    assert L.pp_moe_route(C.byref(r), None) == L.pp_moe_route_bwd(C.byref(r), None) == N.PP_OK
    r.E = 600           # a shape out of range is refused all the same
    assert L.pp_moe_route(C.byref(r), None) == N.PP_ERR_INVALID
    d.D = 96
    assert L.pp_attn_packed_fwd(C.byref(d), None) == N.PP_ERR_UNSUPPORTED
