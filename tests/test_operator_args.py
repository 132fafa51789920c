"""CPU tests of the routing and adapter operators' boundary: size queries, the C
entry points' checks (before any device call) and the Python refusals that need no
device."""

import pytest
import torch


def _lib():
    from kernels import _lib
    return _lib, _lib.load()


def test_size_queries():
    L, lib = _lib()
    assert lib.mxgg_plan_rows(8, 4, 32) == (8 + 4 * 31) // 32 * 32 == 128
    assert lib.mxgg_plan_rows(2, 8, 32) == 64                    # two entries use two groups at most
    assert lib.mxgg_plan_rows(33280, 8, 32) == 33280 + 7 * 32    # 8 * 31 rows more, in whole steps
    assert lib.mxgg_plan_rows(100, 7, 1) == 100 and lib.mxgg_plan_rows(0, 7, 32) == 0
    assert lib.mxgg_token_plan_workspace_size(512, 8) == 0 and lib.mxgg_token_plan_workspace_size(0, 8) == 0
    assert lib.mxgg_token_plan_workspace_size(100000, 8) > 0
    assert lib.mxgg_moe_route_workspace_size(1, 32) == 0 and lib.mxgg_moe_route_workspace_size(16640, 8) > 0
    assert lib.mxgg_lora_hidden_floats(10, 17) == 10 * 32 and lib.mxgg_lora_hidden_floats(10, 513) == 0
    assert lib.mxgg_lora_workspace_floats(0, 4, 16, 512) == 0
    assert lib.mxgg_lora_workspace_floats(64, 64, 16, 8192) >= 64 * 16
    assert lib.mxgg_lora_grad_workspace_floats(8320, 4, 16, 2048, 8192) >= 8320 * 16


P = 1 << 20     # never dereferenced: every call below stops before the device


def _route(lib, **kw):
    a = dict(logits=P, dtype=2, T=64, E=8, ld=8, k=2, normalize=1, multiple=32, M=lib.mxgg_plan_rows(128, 8, 32), z=P)
    a.update(kw)
    return lib.mxgg_moe_route(a["logits"], a["dtype"], a["T"], a["E"], a["ld"], a["k"], a["normalize"], a["multiple"], P, P,
                              P, P, a["M"], P, P, P, a["z"], P, None, 0, None)


def _lora(lib, **kw):
    a = dict(x=P, dtype=0, T=64, K=128, ldx=128, ldd=128, N=256, ldu=256, r=16, ldb=256, out=P, ldo=256, L=4, M=64, ws=P,
             floats=1 << 30)
    a.update(kw)
    return lib.mxgg_lora_grouped_mm(a["x"], a["dtype"], a["T"], a["K"], a["ldx"], P, a["ldd"], a["ldd"] * a["r"], P, a["N"],
                                    a["ldu"], a["ldu"] * a["r"], a["r"], None, P, a["ldb"], a["out"], a["ldo"], P, P, P,
                                    a["L"], a["M"], None, a["ws"], a["floats"], None)


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=7), "element type"), (dict(E=0), "experts"), (dict(E=513, ld=513), "experts"), (dict(k=9), "top_k"),
    (dict(k=0), "top_k"), (dict(E=64, ld=64, k=33), "top_k"), (dict(ld=7), "row stride"), (dict(logits=None), "null"),
    (dict(multiple=0), "multiple"), (dict(M=1), "rows, expected"), (dict(z=None), "null"), (dict(T=-1), "T=-1"),
])
def test_route_refusals_without_gpu(kw, needle):
    L, lib = _lib()
    assert _route(lib, **kw) == L.ERR_INVALID_ARG
    assert needle in lib.mxgg_last_error_string().decode()


@pytest.mark.parametrize("kw,needle", [
    (dict(dtype=2), "neither bf16 nor f16"), (dict(r=0), "rank 0"), (dict(r=513), "rank 513"), (dict(L=0), "adapters"),
    (dict(L=1025), "adapters"), (dict(K=0), "out of range"), (dict(ldx=127), "row stride"), (dict(ldo=255), "row stride"),
    (dict(ldb=255), "row stride"), (dict(ldd=127), "row stride"), (dict(ldu=255), "row stride"), (dict(x=None), "null"),
    (dict(out=None), "null"), (dict(T=65), "tokens in a plan"),
])
def test_lora_refusals_without_gpu(kw, needle):
    L, lib = _lib()
    assert _lora(lib, **kw) == L.ERR_INVALID_ARG
    assert needle in lib.mxgg_last_error_string().decode()


def test_valid_calls_stop_at_the_device():
    """Valid arguments pass every check; too little workspace does not."""
    L, lib = _lib()
    assert _route(lib) == L.ERR_NO_DEVICE
    assert _lora(lib) == L.ERR_NO_DEVICE and _lora(lib, ws=None) == L.ERR_WORKSPACE and _lora(lib, floats=8) == L.ERR_WORKSPACE
    big = 16640
    assert _route(lib, T=big, M=lib.mxgg_plan_rows(2 * big, 8, 32)) == L.ERR_WORKSPACE
    assert lib.mxgg_lora_grouped_mm(None, 0, 0, 128, 128, None, 128, 128, None, 256, 256, 256, 1, None, None, 0, None, 256,
                                    None, None, None, 4, 0, None, None, 0, None) == L.OK          # no tokens
    plan = lambda **kw: lib.mxgg_token_plan(P, kw.get("n", 64), kw.get("E", 8), kw.get("m", 1), P, P, kw.get("M", 64),
                                            P, kw.get("offs", P), None, 0, None)
    assert plan() == L.ERR_NO_DEVICE
    for bad in (dict(E=0), dict(E=1025), dict(m=0), dict(M=63), dict(n=-1), dict(offs=None)):
        assert plan(**bad) == L.ERR_INVALID_ARG
    assert plan(n=100000, M=100000) == L.ERR_WORKSPACE
    move = lambda **kw: lib.mxgg_moe_dispatch(P, kw.get("dtype", 0), kw.get("T", 4), kw.get("H", 64), kw.get("ldx", 64), P,
                                              kw.get("k", 2), P, P, kw.get("E", 8), kw.get("M", 32), P, kw.get("ldo", 64), None)
    assert move() == L.ERR_NO_DEVICE and move(M=0) == L.OK and move(H=0) == L.OK
    for bad in (dict(dtype=3), dict(T=-1), dict(ldx=63), dict(ldo=63), dict(k=0), dict(E=0)):
        assert move(**bad) == L.ERR_INVALID_ARG
    back = lambda **kw: lib.mxgg_moe_combine(kw.get("y", P), 0, 4, 64, kw.get("ldy", 64), P, 2, None, P, kw.get("ldo", 64), None)
    assert back() == L.ERR_NO_DEVICE
    for bad in (dict(y=None), dict(ldy=63), dict(ldo=63)):
        assert back(**bad) == L.ERR_INVALID_ARG


def test_host_tensors_are_refused():
    import kernels
    x = torch.zeros((4, 8))
    with pytest.raises(TypeError):
        kernels.moe_route(x, 2)
    with pytest.raises(TypeError):
        kernels.token_plan(torch.zeros((4,), dtype=torch.int32), 2)
    plan = kernels.TokenPlan(*(torch.zeros(s, dtype=torch.int32) for s in ((4, 1), (4,), (2,), (2,))))
    with pytest.raises(TypeError):
        kernels.moe_dispatch(x, plan)
    with pytest.raises(TypeError):
        kernels.moe_combine(x, x, plan)
    with pytest.raises(TypeError):
        kernels.lora_grouped_mm(x.to(torch.bfloat16), torch.zeros((2, 1, 8)), torch.zeros((2, 1, 8)), plan)
