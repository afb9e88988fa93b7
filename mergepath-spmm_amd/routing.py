"""Sparse routing on torch tensors: routing to experts, the experts' products, their combination, and low-rank adapters
of many requests.

A routing matrix is a sparse matrix of T tokens by E experts with k nonzeros in a row, held by its rows (`expert`,
`weight`) and by its columns (`expert_ptr`, `slot`, `pos`); include/mpspmm.h says what each array holds.  As in
spmm.py, torch gives device memory and the stream only, every computation is a call through the C ABI, and tensors
must be contiguous.  Data may be float32, float16 or bfloat16; sums are held in fp32.  Every function takes its result
tensors as `out` arguments where the caller wants to own them.  Calls run on the current stream of the tensors' device,
which need not be the current device.  No counterpart in the reference.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _cabi
from ._cabi import check

_DTYPES = {torch.float32: _cabi.MPS_F32, torch.float16: _cabi.MPS_F16, torch.bfloat16: _cabi.MPS_BF16}
_SCORES = {"softmax": _cabi.MPS_SCORE_SOFTMAX, "sigmoid": _cabi.MPS_SCORE_SIGMOID}
_GROUP_SCORES = {"max": _cabi.MPS_GROUP_MAX, "top2": _cabi.MPS_GROUP_TOP2}


class Routing(NamedTuple):
    """A routing matrix: expert int32[T, k], weight float32[T, k]; expert_ptr int32[E + 1], slot int32[T * k],
    pos int32[T, k]."""
    expert: torch.Tensor
    weight: torch.Tensor
    expert_ptr: torch.Tensor
    slot: torch.Tensor
    pos: torch.Tensor


def _data(t, name, dims, like=None):
    """A contiguous matrix of a type that the kernels take; on the device (and of the type) of `like`."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA/HIP torch tensor" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    if like is not None and t.dtype != like.dtype:
        raise TypeError("%s must have dtype %s, got %s" % (name, like.dtype, t.dtype))
    return _shaped(t, name, dims, like)


def _array(t, name, dtype, dims, like):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA/HIP torch tensor" % name)
    if t.dtype != dtype:
        raise TypeError("%s must have dtype %s, got %s" % (name, dtype, t.dtype))
    return _shaped(t, name, dims, like)


def _shaped(t, name, dims, like):
    if t.dim() != len(dims) or any(d is not None and d != s for d, s in zip(dims, t.shape)):
        raise ValueError("%s must have the shape [%s], got %s"
                         % (name, ", ".join("any" if d is None else str(d) for d in dims), list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    if like is not None and t.device != like.device:
        raise ValueError("%s is on %s, the other tensors on %s" % (name, t.device, like.device))
    return t


def _fits(*sizes):
    """Sizes travel as 32-bit ints; a larger one must not come out as another number."""
    if any(not 0 <= n <= 0x7FFFFFFF for n in sizes):
        check(_cabi.MPS_ERR_UNSUPPORTED, "sizes beyond 32 bits")


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _call(name, like, *args):
    """mps_<name>(args, stream) on the device of `like`."""
    fn = getattr(_cabi.lib(), name)
    index = like.device.index
    if index == torch.cuda.current_device():
        check(fn(*args, torch.cuda.current_stream(index).cuda_stream), name)
    else:
        with torch.cuda.device(index):
            check(fn(*args, torch.cuda.current_stream(index).cuda_stream), name)


def _options(k, score, groups, top_groups, group_score, renormalise, scale):
    if score not in _SCORES:
        raise ValueError("score must be one of %s" % sorted(_SCORES))
    if group_score not in _GROUP_SCORES:
        raise ValueError("group_score must be one of %s" % sorted(_GROUP_SCORES))
    return _cabi.RouteOptions(int(k), _SCORES[score], int(groups), int(top_groups), _GROUP_SCORES[group_score],
                              int(bool(renormalise)), float(scale))


def _workspace(T, E, k, like):
    """Device memory for the columns of a long routing matrix; None where none is needed."""
    need = ctypes.c_size_t()
    check(_cabi.lib().mps_route_workspace_bytes(T, E, k, ctypes.byref(need)), "mps_route_workspace_bytes")
    ws = torch.empty(need.value, dtype=torch.uint8, device=like.device) if need.value else None
    return ws, need.value


def route(scores, k, *, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalise=False,
          scale=1.0, out=None):
    """Routing to experts (mps_route): scores [T, E] -> Routing.

    s = softmax or sigmoid of the scores; the k experts with the largest s + bias (float32[E]) are chosen, where
    `groups` is given only among the `top_groups` best groups of E / groups experts each (a group counts as its largest
    member, or with "top2" as the sum of its two largest); ties go to the lower index, the choice is that of 64 bits.
    Weights are scale * s, with `renormalise` divided by the sum of the chosen s.  A score of -inf is never chosen: a
    slot that finds no expert holds -1, weight 0 and pos -1."""
    _data(scores, "scores", (None, None))
    T, E = scores.shape
    opt = _options(k, score, groups, top_groups, group_score, renormalise, scale)
    if bias is not None:
        _array(bias, "bias", torch.float32, (E,), scores)
    if k < 1:
        raise ValueError("k must be positive")
    _fits(T * k, E)
    if out is None:
        ints = torch.empty(3 * T * k + E + 1, dtype=torch.int32, device=scores.device)
        n = T * k
        out = Routing(ints[:n].view(T, k), torch.empty((T, k), dtype=torch.float32, device=scores.device), ints[3 * n:],
                      ints[n:2 * n], ints[2 * n:3 * n].view(T, k))
    else:
        _check_routing(out, T, E, k, scores)
    ws, size = _workspace(T, E, k, scores)
    _call("mps_route", scores, _ptr(scores), _DTYPES[scores.dtype], _ptr(bias), T, E, ctypes.byref(opt),
          _ptr(out.expert), _ptr(out.weight), _ptr(out.expert_ptr), _ptr(out.slot), _ptr(out.pos), _ptr(ws), size)
    return out


def _check_routing(r, T, E, k, like):
    _array(r.expert, "expert", torch.int32, (T, k), like)
    _array(r.weight, "weight", torch.float32, (T, k), like)
    _array(r.expert_ptr, "expert_ptr", torch.int32, (E + 1,), like)
    _array(r.slot, "slot", torch.int32, (T * k,), like)
    _array(r.pos, "pos", torch.int32, (T, k), like)


def columns(expert, n_experts):
    """(expert_ptr, slot, pos) of a routing matrix whose rows expert int32[T, k] are given (mps_route_columns): a stable
    counting sort.  Ids outside [0, n_experts) count as -1.  With k = 1 and the adapters of the tokens, expert_ptr and
    slot are what adapters_mm takes."""
    if not isinstance(expert, torch.Tensor) or expert.dim() != 2:
        raise ValueError("expert must be a matrix [T, k]")
    T, k = expert.shape
    _array(expert, "expert", torch.int32, (T, k), expert)
    _fits(T * k, n_experts)
    ptr = torch.empty(n_experts + 1, dtype=torch.int32, device=expert.device)
    slot = torch.empty(T * k, dtype=torch.int32, device=expert.device)
    pos = torch.empty((T, k), dtype=torch.int32, device=expert.device)
    ws, size = _workspace(T, n_experts, k, expert)
    _call("mps_route_columns", expert, _ptr(expert), T, n_experts, k, _ptr(ptr), _ptr(slot), _ptr(pos), _ptr(ws), size)
    return ptr, slot, pos


def route_backward(scores, expert, dweight, *, score="softmax", renormalise=False, scale=1.0, out=None):
    """Gradient of the scores from that of the weights (mps_route_backward)."""
    _data(scores, "scores", (None, None))
    T, E = scores.shape
    if not isinstance(expert, torch.Tensor) or expert.dim() != 2:
        raise ValueError("expert must be a matrix [T, k]")
    k = expert.shape[1]
    _array(expert, "expert", torch.int32, (T, k), scores)
    _array(dweight, "dweight", torch.float32, (T, k), scores)
    _fits(T * k, E)
    opt = _options(k, score, 1, 1, "max", renormalise, scale)
    out = torch.empty_like(scores) if out is None else _data(out, "out", (T, E), scores)
    _call("mps_route_backward", scores, _ptr(scores), _DTYPES[scores.dtype], _ptr(expert), _ptr(dweight), T, E,
          ctypes.byref(opt), _ptr(out))
    return out


def _places(slot, k, rows, like, name):
    """Number of places of rows that are gathered through `slot`, or that stand in order."""
    _fits(rows * max(k, 1))
    if slot is None:
        return rows
    if k < 1:
        raise ValueError("k must be positive")
    _array(slot, "slot", torch.int32, (rows * k,), like)
    return rows * k


def experts_mm(X, W, expert_ptr, *, slot=None, k=1, out=None):
    """Products of the experts (mps_experts_mm): Y[p] = X[row(p)] @ W[e].T for every place p of expert e; W [E, N, K].

    Without `slot` X is [M, K] in the order of the places; with it X holds the tokens, [M / k, K], and row(p) =
    slot[p] // k.  Rows of Y behind expert_ptr[E] are left as they were (undefined in a new tensor)."""
    _data(X, "X", (None, None))
    _data(W, "W", (None, None, X.shape[1]), X)
    E, N, K = W.shape
    _fits(E, N, K)
    _array(expert_ptr, "expert_ptr", torch.int32, (E + 1,), X)
    M = _places(slot, k, X.shape[0], X, "X")
    out = torch.empty((M, N), dtype=X.dtype, device=X.device) if out is None else _data(out, "out", (M, N), X)
    _call("mps_experts_mm", X, _ptr(X), _ptr(W), _ptr(out), _DTYPES[X.dtype], _ptr(expert_ptr), _ptr(slot),
          k if slot is not None else 1, M, E, N, K)
    return out


def experts_mm_dx(dY, W, expert_ptr, *, out=None):
    """Gradient of the rows (mps_experts_mm_dx): dX[p] = dY[p] @ W[e], in the order of the places; that of gathered
    tokens is combine(dX, pos).  Rows behind expert_ptr[E] are left as they were."""
    _data(dY, "dY", (None, None))
    _data(W, "W", (None, dY.shape[1], None), dY)
    E, N, K = W.shape
    _fits(E, N, K)
    _array(expert_ptr, "expert_ptr", torch.int32, (E + 1,), dY)
    M = dY.shape[0]
    _fits(M)
    out = torch.empty((M, K), dtype=dY.dtype, device=dY.device) if out is None else _data(out, "out", (M, K), dY)
    _call("mps_experts_mm_dx", dY, _ptr(dY), _ptr(W), _ptr(out), _DTYPES[dY.dtype], _ptr(expert_ptr), M, E, N, K)
    return out


def experts_mm_dw(dY, X, expert_ptr, *, slot=None, k=1, out=None):
    """Gradient of the weights (mps_experts_mm_dw): dW[e] = dY[places of e].T @ X[row(places)], zero for an expert
    without places.  `slot` and `k` as in experts_mm."""
    _data(X, "X", (None, None))
    M = _places(slot, k, X.shape[0], X, "X")
    _data(dY, "dY", (M, None), X)
    E, N, K = _experts_of(expert_ptr), dY.shape[1], X.shape[1]
    _fits(E, N, K)
    _array(expert_ptr, "expert_ptr", torch.int32, (E + 1,), X)
    out = torch.empty((E, N, K), dtype=X.dtype, device=X.device) if out is None else _data(out, "out", (E, N, K), X)
    _call("mps_experts_mm_dw", X, _ptr(dY), _ptr(X), _ptr(out), _DTYPES[X.dtype], _ptr(expert_ptr), _ptr(slot),
          k if slot is not None else 1, M, E, N, K)
    return out


def _experts_of(expert_ptr):
    if not isinstance(expert_ptr, torch.Tensor) or expert_ptr.dim() != 1 or expert_ptr.numel() < 2:
        raise ValueError("expert_ptr must be an array of E + 1 places")
    return expert_ptr.numel() - 1


def combine(Z, pos, weight=None, *, base=None, out=None):
    """Product of the routing matrix with the experts' rows (mps_combine): Y[t] = base[t] + sum_j weight[t, j] *
    Z[pos[t, j]] over the slots that have a place; weight None = 1."""
    _data(Z, "Z", (None, None))
    M, N = Z.shape
    if not isinstance(pos, torch.Tensor) or pos.dim() != 2:
        raise ValueError("pos must be a matrix [T, k]")
    T, k = pos.shape
    _fits(T * k, M, N)
    _array(pos, "pos", torch.int32, (T, k), Z)
    if weight is not None:
        _array(weight, "weight", torch.float32, (T, k), Z)
    if base is not None:
        _data(base, "base", (T, N), Z)
    out = torch.empty((T, N), dtype=Z.dtype, device=Z.device) if out is None else _data(out, "out", (T, N), Z)
    _call("mps_combine", Z, _ptr(Z), _ptr(pos), _ptr(weight), _ptr(base), _ptr(out), _DTYPES[Z.dtype], T, k, M, N)
    return out


def combine_backward(dY, Z, weight, expert_ptr, slot):
    """Gradients of combine (mps_combine_backward): {"dZ": [M, N], "dweight": float32[T, k]}; zero where there is no
    expert."""
    _data(dY, "dY", (None, None))
    T, N = dY.shape
    _array(weight, "weight", torch.float32, (T, None), dY)
    k = weight.shape[1]
    _fits(T * k, N)
    _data(Z, "Z", (T * k, N), dY)
    E = _experts_of(expert_ptr)
    _array(expert_ptr, "expert_ptr", torch.int32, (E + 1,), dY)
    _array(slot, "slot", torch.int32, (T * k,), dY)
    dZ, dweight = torch.empty_like(Z), torch.empty_like(weight)
    _call("mps_combine_backward", dY, _ptr(dY), _ptr(Z), _ptr(weight), _ptr(expert_ptr), E, _ptr(slot), _ptr(dZ),
          _ptr(dweight), _DTYPES[dY.dtype], T, k, N)
    return {"dZ": dZ, "dweight": dweight}


def adapters_mm(X, A, B, scale, adapter_ptr, row, *, base=None, out=None):
    """Low-rank adapters of many requests (mps_adapters_mm): Y[t] = base[t] + scale[a] * (X[t] @ A[a].T) @ B[a].T for the
    tokens row[adapter_ptr[a]:adapter_ptr[a + 1]] of adapter a, Y[t] = base[t] for those behind adapter_ptr[E]; A [E, R, K],
    B [E, N, R], scale float32[E] or None.  `row` names every token once (columns() of the tokens' adapters).  `out` may
    be `base`."""
    _data(X, "X", (None, None))
    T, K = X.shape
    _data(A, "A", (None, None, K), X)
    E, R = A.shape[0], A.shape[1]
    _data(B, "B", (E, None, R), X)
    N = B.shape[1]
    _fits(T, E, R, K, N)
    if scale is not None:
        _array(scale, "scale", torch.float32, (E,), X)
    _array(adapter_ptr, "adapter_ptr", torch.int32, (E + 1,), X)
    _array(row, "row", torch.int32, (T,), X)
    if base is not None:
        _data(base, "base", (T, N), X)
    out = torch.empty((T, N), dtype=X.dtype, device=X.device) if out is None else _data(out, "out", (T, N), X)
    need = ctypes.c_size_t()
    check(_cabi.lib().mps_adapters_workspace_bytes(T, E, R, K, ctypes.byref(need)), "mps_adapters_workspace_bytes")
    ws = torch.empty(max(need.value, 16), dtype=torch.uint8, device=X.device)
    _call("mps_adapters_mm", X, _ptr(X), _ptr(A), _ptr(B), _ptr(scale), _ptr(base), _ptr(out), _DTYPES[X.dtype],
          _ptr(adapter_ptr), _ptr(row), T, E, R, K, N, _ptr(ws), need.value)
    return out
