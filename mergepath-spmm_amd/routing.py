"""Sparse routing on torch tensors: routing to experts, the experts' products, their combination, and low-rank adapters
of many requests.

A routing matrix is a sparse matrix of T tokens by E experts with k nonzeros in a row, held by its rows (`expert`,
`weight`) and by its columns (`expert_ptr`, `slot`, `pos`); include/mpspmm.h says what each array holds.  As in
spmm.py, torch gives device memory and the stream only, every computation is a call through the C ABI, and tensors
must be contiguous.  Data may be float32, float16 or bfloat16; sums are held in fp32.  Every function takes its result
tensors as `out` arguments where the caller wants to own them.  Calls run on the current stream of the tensors' device,
which need not be the current device.  They build no autograd graph: gradients are functions of their own
(route_backward, experts_mm_dx, experts_mm_dw, combine_backward), to be called in a caller's autograd.Function or
training step.  No counterpart in the reference.
"""
import ctypes
import functools
import operator
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


def _first(t, name, dims):
    """The operand that says of which type and on which device the others are: (type, device)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA/HIP torch tensor" % name)
    if t.dtype not in _DTYPES:
        raise TypeError("%s must be float32, float16 or bfloat16, got %s" % (name, t.dtype))
    if t.dim() != dims:
        raise ValueError("%s must have %d dimensions, got the shape %s" % (name, dims, list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    return t.dtype, t.get_device()


def _need(t, name, dtype, shape, device):
    if (isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.get_device() == device
            and device >= 0 and t.is_contiguous()):
        return t
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("%s must be a CUDA/HIP torch tensor" % name)
    if t.dtype != dtype:
        raise TypeError("%s must have dtype %s, got %s" % (name, dtype, t.dtype))
    if t.shape != shape:
        raise ValueError("%s must have the shape %s, got %s" % (name, list(shape), list(t.shape)))
    if not t.is_contiguous():
        raise ValueError("%s must be contiguous" % name)
    raise ValueError("%s is on %s, the other tensors on cuda:%d" % (name, t.device, device))


def _shape_of(t, name, dims):
    """The shape of a tensor that _need will look at more closely."""
    if not isinstance(t, torch.Tensor) or t.dim() != dims:
        raise ValueError("%s must be a tensor of %d dimensions" % (name, dims))
    return t.shape


def _fits(*sizes):
    """Sizes travel as 32-bit ints; a larger one must not come out as another number."""
    for n in sizes:
        if not 0 <= n <= 0x7FFFFFFF:
            check(_cabi.MPS_ERR_UNSUPPORTED, "sizes beyond 32 bits")


def _ptr(t):
    return t.data_ptr() if t is not None else None


@functools.lru_cache(maxsize=None)
def _entry(name):
    return getattr(_cabi.lib(), name)


def _call(name, device, *args):
    """mps_<name>(args, stream) on GPU number `device`, on the stream that is current there."""
    if device == torch._C._cuda_getDevice():
        status = _entry(name)(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = _entry(name)(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        check(status, name)


def _options(k, score, groups, top_groups, group_score, renormalise, scale):
    """mps_route_options, as an argument of a call.  Kept by the numbers that it holds: what the caller gives may be a
    tensor, whose value changes in place."""
    if score not in _SCORES:
        raise ValueError("score must be one of %s" % sorted(_SCORES))
    if group_score not in _GROUP_SCORES:
        raise ValueError("group_score must be one of %s" % sorted(_GROUP_SCORES))
    return _options_of(operator.index(k), _SCORES[score], operator.index(groups), operator.index(top_groups),
                       _GROUP_SCORES[group_score], bool(renormalise), ctypes.c_float(scale).value)


@functools.lru_cache(maxsize=64)
def _options_of(*numbers):
    """The structure is only read."""
    return ctypes.byref(_cabi.RouteOptions(*numbers))


@functools.lru_cache(maxsize=256)
def _workspace_bytes(name, *sizes):
    """mps_<name>(sizes, &bytes)."""
    need = ctypes.c_size_t()
    check(getattr(_cabi.lib(), name)(*sizes, ctypes.byref(need)), name)
    return need.value


def _workspace(T, E, k, device):
    """Device memory for the columns of a long routing matrix; None where none is needed."""
    size = _workspace_bytes("mps_route_workspace_bytes", T, E, k)
    return torch.empty(size, dtype=torch.uint8, device="cuda:%d" % device) if size else None, size


def route(scores, k, *, score="softmax", bias=None, groups=1, top_groups=1, group_score="max", renormalise=False,
          scale=1.0, out=None):
    """Routing to experts (mps_route): scores [T, E] -> Routing.

    s = softmax or sigmoid of the scores; the k experts with the largest s + bias (float32[E]) are chosen, where
    `groups` is given only among the `top_groups` best groups of E / groups experts each (a group counts as its largest
    member, or with "top2" as the sum of its two largest); ties go to the lower index, the choice is that of 64 bits.
    Weights are scale * s, with `renormalise` divided by the sum of the chosen s.  An expert whose score or bias is -inf
    is never chosen: a slot that finds none holds -1, weight 0 and pos -1."""
    t, device = _first(scores, "scores", 2)
    T, E = scores.shape
    k = operator.index(k)
    opt = _options(k, score, groups, top_groups, group_score, renormalise, scale)
    if bias is not None:
        _need(bias, "bias", torch.float32, (E,), device)
    if k < 1:
        raise ValueError("k must be positive")
    n = T * k
    _fits(n, E)
    ws, size = _workspace(T, E, k, device) if n > 2048 else (None, 0)  # short ones are known to need none
    if out is None:
        # One allocation for all that is as long as there are slots, the weights' bits among them.  `.data`: a version
        # counter for each, so that an in-place change of the weights is none of the indices that autograd has kept.
        ints = scores.new_empty((4, T, k), dtype=torch.int32)
        expert, weight, slot, pos = ints.unbind()
        out = Routing(expert.data, weight.view(torch.float32).data, scores.new_empty((E + 1,), dtype=torch.int32),
                      slot.view(n).data, pos.data)
        at = ints.data_ptr()
        at = at, at + 4 * n, out.expert_ptr.data_ptr(), at + 8 * n, at + 12 * n
    else:
        _need(out.expert, "expert", torch.int32, (T, k), device)
        _need(out.weight, "weight", torch.float32, (T, k), device)
        _need(out.expert_ptr, "expert_ptr", torch.int32, (E + 1,), device)
        _need(out.slot, "slot", torch.int32, (n,), device)
        _need(out.pos, "pos", torch.int32, (T, k), device)
        at = tuple(x.data_ptr() for x in out)
    _call("mps_route", device, scores.data_ptr(), _DTYPES[t], _ptr(bias), T, E, opt, *at, _ptr(ws), size)
    return out


def columns(expert, n_experts):
    """(expert_ptr, slot, pos) of a routing matrix whose rows expert int32[T, k] are given (mps_route_columns): a stable
    counting sort.  Ids outside [0, n_experts) count as -1.  With k = 1 and the adapters of the tokens, expert_ptr and
    slot are what adapters_mm takes."""
    T, k = _shape_of(expert, "expert", 2)
    device = expert.get_device()
    _need(expert, "expert", torch.int32, (T, k), device)
    _fits(T * k, n_experts)
    ptr = torch.empty(n_experts + 1, dtype=torch.int32, device=expert.device)
    slot = torch.empty(T * k, dtype=torch.int32, device=expert.device)
    pos = torch.empty((T, k), dtype=torch.int32, device=expert.device)
    ws, size = _workspace(T, n_experts, k, device)
    _call("mps_route_columns", device, expert.data_ptr(), T, n_experts, k, ptr.data_ptr(), slot.data_ptr(),
          pos.data_ptr(), _ptr(ws), size)
    return ptr, slot, pos


def route_backward(scores, expert, dweight, *, score="softmax", renormalise=False, scale=1.0, out=None):
    """Gradient of the scores from that of the weights (mps_route_backward)."""
    t, device = _first(scores, "scores", 2)
    T, E = scores.shape
    k = _shape_of(expert, "expert", 2)[1]
    _need(expert, "expert", torch.int32, (T, k), device)
    _need(dweight, "dweight", torch.float32, (T, k), device)
    _fits(T * k, E)
    opt = _options(k, score, 1, 1, "max", renormalise, scale)
    out = torch.empty_like(scores) if out is None else _need(out, "out", t, (T, E), device)
    _call("mps_route_backward", device, scores.data_ptr(), _DTYPES[t], expert.data_ptr(), dweight.data_ptr(), T, E,
          opt, out.data_ptr())
    return out


def _places(slot, k, rows, device):
    """Number of places of rows that are gathered through `slot`, or that stand in order."""
    if slot is None:
        _fits(rows)
        return rows
    if k < 1:
        raise ValueError("k must be positive")
    _fits(rows * k)
    _need(slot, "slot", torch.int32, (rows * k,), device)
    return rows * k


def experts_mm(X, W, expert_ptr, *, slot=None, k=1, out=None):
    """Products of the experts (mps_experts_mm): Y[p] = X[row(p)] @ W[e].T for every place p of expert e; W [E, N, K].

    Without `slot` X is [M, K] in the order of the places; with it X holds the tokens, [M / k, K], and row(p) =
    slot[p] // k.  Rows of Y behind expert_ptr[E] are left as they were (undefined in a new tensor)."""
    t, device = _first(X, "X", 2)
    rows, K = X.shape
    E, N, _ = _shape_of(W, "W", 3)
    _need(W, "W", t, (E, N, K), device)
    _need(expert_ptr, "expert_ptr", torch.int32, (E + 1,), device)
    M = _places(slot, k, rows, device)
    _fits(E, N, K)
    out = X.new_empty((M, N)) if out is None else _need(out, "out", t, (M, N), device)
    _call("mps_experts_mm", device, X.data_ptr(), W.data_ptr(), out.data_ptr(), _DTYPES[t], expert_ptr.data_ptr(),
          _ptr(slot), k if slot is not None else 1, M, E, N, K)
    return out


def experts_mm_dx(dY, W, expert_ptr, *, out=None):
    """Gradient of the rows (mps_experts_mm_dx): dX[p] = dY[p] @ W[e], in the order of the places; that of gathered
    tokens is combine(dX, pos).  Rows behind expert_ptr[E] are left as they were."""
    t, device = _first(dY, "dY", 2)
    M, N = dY.shape
    E, _, K = _shape_of(W, "W", 3)
    _need(W, "W", t, (E, N, K), device)
    _need(expert_ptr, "expert_ptr", torch.int32, (E + 1,), device)
    _fits(M, E, N, K)
    out = dY.new_empty((M, K)) if out is None else _need(out, "out", t, (M, K), device)
    _call("mps_experts_mm_dx", device, dY.data_ptr(), W.data_ptr(), out.data_ptr(), _DTYPES[t], expert_ptr.data_ptr(), M,
          E, N, K)
    return out


def _experts_of(expert_ptr):
    E = _shape_of(expert_ptr, "expert_ptr", 1)[0] - 1
    if E < 1:
        raise ValueError("expert_ptr must be an array of E + 1 places")
    return E


def experts_mm_dw(dY, X, expert_ptr, *, slot=None, k=1, out=None):
    """Gradient of the weights (mps_experts_mm_dw): dW[e] = dY[places of e].T @ X[row(places)], zero for an expert
    without places.  `slot` and `k` as in experts_mm."""
    t, device = _first(X, "X", 2)
    rows, K = X.shape
    M = _places(slot, k, rows, device)
    N = _shape_of(dY, "dY", 2)[1]
    _need(dY, "dY", t, (M, N), device)
    E = _experts_of(expert_ptr)
    _need(expert_ptr, "expert_ptr", torch.int32, (E + 1,), device)
    _fits(E, N, K)
    out = X.new_empty((E, N, K)) if out is None else _need(out, "out", t, (E, N, K), device)
    _call("mps_experts_mm_dw", device, dY.data_ptr(), X.data_ptr(), out.data_ptr(), _DTYPES[t], expert_ptr.data_ptr(),
          _ptr(slot), k if slot is not None else 1, M, E, N, K)
    return out


def combine(Z, pos, weight=None, *, base=None, out=None):
    """Product of the routing matrix with the experts' rows (mps_combine): Y[t] = base[t] + sum_j weight[t, j] *
    Z[pos[t, j]] over the slots that have a place; weight None = 1.  `out` may be `base`."""
    t, device = _first(Z, "Z", 2)
    M, N = Z.shape
    T, k = _shape_of(pos, "pos", 2)
    _need(pos, "pos", torch.int32, (T, k), device)
    if weight is not None:
        _need(weight, "weight", torch.float32, (T, k), device)
    if base is not None:
        _need(base, "base", t, (T, N), device)
    _fits(T * k, M, N)
    out = Z.new_empty((T, N)) if out is None else _need(out, "out", t, (T, N), device)
    _call("mps_combine", device, Z.data_ptr(), pos.data_ptr(), _ptr(weight), _ptr(base), out.data_ptr(), _DTYPES[t], T, k,
          M, N)
    return out


def combine_backward(dY, Z, weight, expert_ptr, slot):
    """Gradients of combine (mps_combine_backward): {"dZ": [M, N], "dweight": float32[T, k]}; zero where there is no
    expert."""
    t, device = _first(dY, "dY", 2)
    T, N = dY.shape
    k = _shape_of(weight, "weight", 2)[1]
    _need(weight, "weight", torch.float32, (T, k), device)
    _need(Z, "Z", t, (T * k, N), device)
    E = _experts_of(expert_ptr)
    _need(expert_ptr, "expert_ptr", torch.int32, (E + 1,), device)
    _need(slot, "slot", torch.int32, (T * k,), device)
    _fits(T * k, E, N)
    dZ, dweight = torch.empty_like(Z), torch.empty_like(weight)
    _call("mps_combine_backward", device, dY.data_ptr(), Z.data_ptr(), weight.data_ptr(), expert_ptr.data_ptr(), E,
          slot.data_ptr(), dZ.data_ptr(), dweight.data_ptr(), _DTYPES[t], T, k, N)
    return {"dZ": dZ, "dweight": dweight}


def adapters_mm(X, A, B, scale, adapter_ptr, row, *, base=None, out=None):
    """Low-rank adapters of many requests (mps_adapters_mm): Y[t] = base[t] + scale[a] * (X[t] @ A[a].T) @ B[a].T for the
    tokens row[adapter_ptr[a]:adapter_ptr[a + 1]] of adapter a, Y[t] = base[t] for those behind adapter_ptr[E]; A [E, R, K],
    B [E, N, R], scale float32[E] or None.  `row` names every token once (columns() of the tokens' adapters).  `out` may
    be `base`."""
    t, device = _first(X, "X", 2)
    T, K = X.shape
    E, R, _ = _shape_of(A, "A", 3)
    N = _shape_of(B, "B", 3)[1]
    _need(A, "A", t, (E, R, K), device)
    _need(B, "B", t, (E, N, R), device)
    if scale is not None:
        _need(scale, "scale", torch.float32, (E,), device)
    _need(adapter_ptr, "adapter_ptr", torch.int32, (E + 1,), device)
    _need(row, "row", torch.int32, (T,), device)
    if base is not None:
        _need(base, "base", t, (T, N), device)
    _fits(T, E, R, K, N)
    out = X.new_empty((T, N)) if out is None else _need(out, "out", t, (T, N), device)
    size = _workspace_bytes("mps_adapters_workspace_bytes", T, E, R, K)
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=X.device)
    _call("mps_adapters_mm", device, X.data_ptr(), A.data_ptr(), B.data_ptr(), _ptr(scale), _ptr(base), out.data_ptr(),
          _DTYPES[t], adapter_ptr.data_ptr(), row.data_ptr(), T, E, R, K, N, ws.data_ptr(), size)
    return out
