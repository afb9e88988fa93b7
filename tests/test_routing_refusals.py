"""What the sparse-routing entry points refuse, without a GPU: every check comes before the first launch."""
import ctypes

import pytest
import torch

P = 1 << 20  # an aligned address that is never read


@pytest.fixture
def L(pkg):
    return pkg._cabi.lib()


def options(pkg, k=2, score=0, groups=1, top_groups=1, group_score=0, renormalise=0, scale=1.0):
    return ctypes.byref(pkg._cabi.RouteOptions(k, score, groups, top_groups, group_score, renormalise, scale))


def route(pkg, L, T=4, E=16, dtype=0, scores=P, expert=P, weight=P, ptr=P, slot=P, pos=P, ws=P, size=1 << 30, **o):
    return L.mps_route(scores, dtype, None, T, E, options(pkg, **o), expert, weight, ptr, slot, pos, ws, size, None)


INVALID, UNSUPPORTED, WORKSPACE, ALIGNMENT = 1, 2, 3, 4


@pytest.mark.parametrize("args,status", [
    (dict(T=-1), INVALID), (dict(E=0), INVALID), (dict(k=0), INVALID), (dict(k=17), INVALID), (dict(dtype=3), INVALID),
    (dict(score=2), INVALID), (dict(scores=None), INVALID), (dict(expert=None), INVALID), (dict(weight=None), INVALID),
    (dict(slot=None), INVALID), (dict(pos=None), INVALID), (dict(ptr=None), INVALID),
    (dict(E=1025), UNSUPPORTED), (dict(E=64, k=33), UNSUPPORTED), (dict(T=2 ** 30, k=2), UNSUPPORTED),
    (dict(groups=3), INVALID), (dict(groups=4, top_groups=0), INVALID), (dict(groups=4, top_groups=5), INVALID),
    (dict(groups=16, top_groups=4, group_score=1), INVALID), (dict(groups=4, group_score=2), INVALID),
    (dict(groups=8, top_groups=1, k=3), INVALID), (dict(E=256, groups=128, top_groups=8), UNSUPPORTED),
    (dict(scores=P + 2), ALIGNMENT), (dict(weight=P + 1), ALIGNMENT), (dict(pos=P + 2), ALIGNMENT),
    (dict(T=100000, ws=None), WORKSPACE), (dict(T=100000, size=16), WORKSPACE), (dict(T=100000, ws=P + 4), ALIGNMENT),
])
def test_route(pkg, L, args, status):
    assert route(pkg, L, **args) == status


def test_route_without_options(pkg, L):
    assert L.mps_route(P, 0, None, 4, 16, None, P, P, P, P, P, None, 0, None) == INVALID
    assert L.mps_route_backward(P, 0, P, P, 4, 16, None, P, None) == INVALID


def test_route_backward(pkg, L):
    for args, status in (((P, 5, P, P, 4, 16), INVALID), ((P, 0, None, P, 4, 16), INVALID), ((P, 0, P, None, 4, 16), INVALID),
                         ((P, 0, P, P, 4, 1), INVALID), ((P, 0, P, P, 4, 2000), UNSUPPORTED), ((P + 1, 1, P, P, 4, 16), ALIGNMENT)):
        assert L.mps_route_backward(*args, options(pkg), P, None) == status
    assert L.mps_route_backward(P, 0, P, P, 4, 16, options(pkg), None, None) == INVALID
    assert L.mps_route_backward(None, 0, None, None, 0, 16, options(pkg), None, None) == 0


def test_workspace_sizes(pkg, L):
    n = ctypes.c_size_t()
    assert L.mps_route_workspace_bytes(1, 8, 2, ctypes.byref(n)) == 0 and n.value == 0
    assert L.mps_route_workspace_bytes(16384, 256, 8, ctypes.byref(n)) == 0 and n.value > 0
    assert L.mps_route_workspace_bytes(16384, 256, 8, None) == INVALID
    assert L.mps_route_workspace_bytes(2 ** 30, 256, 8, ctypes.byref(n)) == UNSUPPORTED
    assert L.mps_adapters_workspace_bytes(8, 2, 16, 64, ctypes.byref(n)) == 0 and n.value >= 8 * 16 * 4
    assert L.mps_adapters_workspace_bytes(8, 2, 257, 64, ctypes.byref(n)) == UNSUPPORTED
    assert L.mps_adapters_workspace_bytes(8, 0, 16, 64, ctypes.byref(n)) == INVALID
    assert L.mps_adapters_workspace_bytes(8, 2, 16, 64, None) == INVALID


def test_columns(L):
    assert L.mps_route_columns(P, 4, 1025, 1, P, P, P, None, 0, None) == UNSUPPORTED
    assert L.mps_route_columns(None, 4, 8, 1, P, P, P, None, 0, None) == INVALID
    assert L.mps_route_columns(P, 4, 8, 1, P, None, P, None, 0, None) == INVALID
    assert L.mps_route_columns(P, 100000, 8, 1, P, P, P, None, 0, None) == WORKSPACE
    assert L.mps_route_columns(P, 4, 8, 0, P, P, P, None, 0, None) == INVALID


@pytest.mark.parametrize("args,status", [
    (dict(M=-1), INVALID), (dict(E=0), INVALID), (dict(N=0), INVALID), (dict(K=0), INVALID), (dict(dtype=-1), INVALID),
    (dict(k=0), INVALID), (dict(M=7, k=2), INVALID), (dict(ptr=None), INVALID), (dict(A=None), INVALID),
    (dict(B=None), INVALID), (dict(out=None), INVALID), (dict(A=P + 1), ALIGNMENT), (dict(slot=P + 2), ALIGNMENT),
    (dict(N=2 ** 30), UNSUPPORTED), (dict(M=2 ** 31 - 1), UNSUPPORTED),
])
def test_experts(L, args, status):
    a = dict(A=P, B=P, out=P, dtype=1, ptr=P, slot=P, k=1, M=8, E=4, N=16, K=16)
    a.update(args)
    for fn in (L.mps_experts_mm, L.mps_experts_mm_dw):
        assert fn(a["A"], a["B"], a["out"], a["dtype"], a["ptr"], a["slot"], a["k"], a["M"], a["E"], a["N"], a["K"], None) == status
    if "k" not in args and "slot" not in args:
        assert L.mps_experts_mm_dx(a["A"], a["B"], a["out"], a["dtype"], a["ptr"], a["M"], a["E"], a["N"], a["K"], None) == status
    assert L.mps_experts_mm(None, P, None, 1, P, None, 1, 0, 4, 16, 16, None) == 0  # no rows, nothing to do


def test_combine(L):
    assert L.mps_combine(P, P, P, None, P, 0, 4, 0, 8, 16, None) == INVALID
    assert L.mps_combine(P, P, P, None, P, 3, 4, 2, 8, 16, None) == INVALID
    assert L.mps_combine(None, P, P, None, P, 0, 4, 2, 8, 16, None) == INVALID
    assert L.mps_combine(P, None, P, None, P, 0, 4, 2, 8, 16, None) == INVALID
    assert L.mps_combine(P, P, P, P + 2, P, 0, 4, 2, 8, 16, None) == ALIGNMENT
    assert L.mps_combine(P, P, P, None, P, 0, 2 ** 30, 4, 8, 16, None) == UNSUPPORTED
    assert L.mps_combine(None, None, None, None, None, 0, 0, 2, 0, 16, None) == 0
    assert L.mps_combine_backward(P, None, P, P, 4, P, P, P, 0, 4, 2, 16, None) == INVALID
    assert L.mps_combine_backward(P, P, P, None, 4, P, P, P, 0, 4, 2, 16, None) == INVALID
    assert L.mps_combine_backward(P, P, P, P, 4, P, P, P + 2, 0, 4, 2, 16, None) == ALIGNMENT
    assert L.mps_combine_backward(P, P, P, P, 4, P, P, P, 0, 2 ** 30, 4, 16, None) == UNSUPPORTED


@pytest.mark.parametrize("args,status", [
    (dict(T=-1), INVALID), (dict(E=0), INVALID), (dict(R=0), INVALID), (dict(K=0), INVALID), (dict(N=0), INVALID),
    (dict(dtype=9), INVALID), (dict(R=257), UNSUPPORTED), (dict(E=1025), UNSUPPORTED), (dict(T=2 ** 20), UNSUPPORTED),
    (dict(X=None), INVALID), (dict(A=None), INVALID), (dict(B=None), INVALID), (dict(Y=None), INVALID),
    (dict(ptr=None), INVALID), (dict(row=None), INVALID), (dict(X=P + 1), ALIGNMENT), (dict(ws=P + 8), ALIGNMENT),
    (dict(ws=None), WORKSPACE), (dict(size=8), WORKSPACE), (dict(T=0), 0),
])
def test_adapters(L, args, status):
    a = dict(X=P, A=P, B=P, Y=P, dtype=2, ptr=P, row=P, T=8, E=4, R=16, K=64, N=64, ws=P, size=1 << 30)
    a.update(args)
    assert L.mps_adapters_mm(a["X"], a["A"], a["B"], None, None, a["Y"], a["dtype"], a["ptr"], a["row"], a["T"], a["E"], a["R"],
                             a["K"], a["N"], a["ws"], a["size"], None) == status


def test_tensors_on_the_host_are_refused(pkg):
    r = pkg.routing
    with pytest.raises(TypeError):
        r.route(torch.zeros(2, 4), 1)
    with pytest.raises(TypeError):
        r.experts_mm(torch.zeros(2, 4), torch.zeros(1, 3, 4), torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError):
        r.columns(torch.zeros(2, 1, dtype=torch.int32), 3)
    with pytest.raises(TypeError):
        r.combine(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32))


def test_route_options_are_values(pkg):
    """A scale that is a tensor counts with the value that it has at the call, also after it was changed in place."""
    def of(**o):
        a = dict(k=8, score="softmax", groups=1, top_groups=1, group_score="max", renormalise=False, scale=1.0)
        a.update(o)
        return pkg.routing._options(**a)._obj

    scale = torch.nn.Parameter(torch.tensor(2.5))
    assert of(scale=scale).scale == 2.5
    with torch.no_grad():
        scale.fill_(4.0)
    assert of(scale=scale).scale == 4.0
    flag = torch.tensor(False)
    assert of(renormalise=flag).renormalise == 0
    flag.fill_(True)
    assert of(renormalise=flag).renormalise == 1
    k = torch.tensor(3)
    assert of(k=k).k == 3
    k.fill_(4)
    assert of(k=k).k == 4
    assert of(k=1, groups=1, scale=1).k == 1 and of(k=True, groups=1, scale=1.0).scale == 1.0
    for bad in (dict(k=2.5), dict(groups="2"), dict(scale="x"), dict(scale=None)):
        with pytest.raises((TypeError, ValueError)):
            of(**bad)


def test_experts_of_more_tiles_than_a_launch_holds(L):
    for fn in (L.mps_experts_mm, L.mps_experts_mm_dw):
        assert fn(P, P, P, 1, P, None, 1, 64, 1 << 24, 1, 1, None) == UNSUPPORTED
        assert fn(P, P, P, 0, P, None, 1, 1 << 20, 1 << 22, 1000, 8, None) == UNSUPPORTED
    assert L.mps_experts_mm(P, P, P, 2, P, None, 1, 1 << 30, 1 << 10, 1 << 20, 8, None) == UNSUPPORTED
    assert L.mps_experts_mm_dx(P, P, P, 1, P, 64, 1 << 24, 1, 1, None) == UNSUPPORTED
    assert L.mps_experts_mm(P, P, P, 1, P, None, 1, 64, 2 ** 31 - 1, 1, 1, None) == UNSUPPORTED
    # 2^66 tiles of 64 x 64, less 2^44
    n = (1 << 29) - 64
    assert L.mps_experts_mm_dw(P, P, P, 0, P, None, 1, 64, 1 << 20, n, n, None) == UNSUPPORTED
