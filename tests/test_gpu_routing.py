"""Sparse routing on the GPU against the definitions in 64 bits.

Tolerances, fixed from the arithmetic.  u = 2^-24 is half a step of fp32, `half(t)` half a step of the result's type.
 - Weights and gradients of the scores: exp within 2 u of itself, a sigmoid or a quotient 4 u more, sums of positive
   numbers (at most 16 in a lane, then 6 levels) 22 u: below 32 u = 2^-19, relative to the sum of the terms' magnitudes.
 - Products: a sum of n terms in any order is off by at most n u times the sum of the magnitudes; a product of two fp32
   numbers adds u.  Twice that for a matrix instruction's own steps: (2 n + 2) u * sum |x| |w|.
 - The result's rounding: half(t) of the value, or half of the smallest subnormal step.
"""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24
SUBNORMAL = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def half(t):
    return torch.finfo(t).eps / 2


@pytest.fixture
def r(pkg, dev):
    return pkg.routing


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(seed, *shape, t=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen(seed), dtype=torch.float64) * scale).to(t)


def close(got, ref, magnitude, n, t):
    """|got - ref| <= half(t) |ref| + (2 n + 2) u (1 + half) * magnitude, all in 64 bits on the CPU."""
    got = got.detach().cpu().double()
    bound = half(t) * ref.abs() + (2 * n + 2) * U * 1.01 * magnitude + SUBNORMAL[t]
    bad = (got - ref).abs() > bound
    assert torch.isfinite(got).all()
    assert not bad.any(), "off by %.3g, allowed %.3g" % (float((got - ref).abs()[bad].max()), float(bound[bad].max()))


# ---------------------------------------------------------------------------------------------------------------------
# The definition of the routing
# ---------------------------------------------------------------------------------------------------------------------

def exact_route(l, bias, k, score="softmax", groups=1, top_groups=1, group_score="max", renormalise=False, scale=1.0):
    """expert, weight from the scores l (64 bits, numpy), one token after the other."""
    T, E = l.shape
    expert, weight = np.full((T, k), -1, np.int32), np.zeros((T, k))
    for t in range(T):
        x = l[t]
        can = x > -np.inf
        if not can.any():
            continue
        if score == "softmax":
            p = np.where(can, np.exp(x - x.max()), 0.0)
            s = p / p.sum()
        else:
            s = 1.0 / (1.0 + np.exp(-x))
        c = x.copy() if bias is None and (groups == 1 or group_score == "max") else s + (0.0 if bias is None else bias)
        c = np.where(can, c, -np.inf)
        if groups > 1:
            g = np.sort(c.reshape(groups, -1), axis=1)
            of = g[:, -1] if group_score == "max" else g[:, -1] + g[:, -2]
            kept = np.argsort(-of, kind="stable")[:top_groups]
            c = np.where(np.isin(np.arange(E) // (E // groups), kept), c, -np.inf)
        order = [e for e in np.argsort(-c, kind="stable")[:k] if c[e] > -np.inf]
        expert[t, :len(order)] = order
        if renormalise:
            # relative to the largest, so that nothing vanishes: log s = -log1p(exp(-x)) for the sigmoid
            logs = x[order] if score == "softmax" else -np.logaddexp(0.0, -x[order])
            w = np.exp(logs - logs.max()) if order else np.zeros(0)
            w = w / w.sum() if order else w
        else:
            w = s[order]
        weight[t, :len(order)] = scale * w
    return expert, weight


def exact_columns(expert, E):
    flat = expert.reshape(-1)
    key = np.where((flat < 0) | (flat >= E), E, flat)
    slot = np.argsort(key, kind="stable").astype(np.int32)
    ptr = np.concatenate([[0], np.cumsum(np.bincount(key, minlength=E + 1)[:E])]).astype(np.int32)
    pos = np.empty(flat.size, np.int32)
    pos[slot] = np.arange(flat.size, dtype=np.int32)
    pos[key == E] = -1
    return ptr, slot, pos.reshape(expert.shape)


def check_routing(m, expert, weight, E):
    assert np.array_equal(m.expert.cpu().numpy(), expert)
    got = m.weight.cpu().double().numpy()
    assert (np.abs(got - weight) <= 2.0 ** -19 * np.abs(weight) + 1e-37).all()
    for got, ref in zip((m.expert_ptr, m.slot, m.pos), exact_columns(expert, E)):
        assert np.array_equal(got.cpu().numpy(), ref)


GROUPED = dict(score="sigmoid", groups=8, top_groups=4, group_score="top2", renormalise=True, scale=2.5)


@pytest.mark.parametrize("T,E,k,t,biased,options", [
    (1, 1, 1, "f32", False, {}),
    (1, 8, 2, "bf16", True, dict(score="sigmoid")),
    (3, 7, 7, "f16", False, dict(renormalise=True)),
    (4, 256, 8, "f32", True, GROUPED),
    (65, 64, 6, "bf16", False, dict(scale=16.0)),
    (129, 65, 5, "f32", True, dict(renormalise=True)),
    (200, 72, 6, "f16", True, dict(groups=6, top_groups=2, group_score="max")),
    (257, 128, 32, "bf16", False, dict(score="sigmoid", renormalise=True)),
    (50, 160, 6, "bf16", False, dict(groups=8, top_groups=3, group_score="max", renormalise=True)),
    (300, 256, 8, "bf16", True, GROUPED),
    (33, 320, 9, "f16", True, dict(score="sigmoid", groups=64, top_groups=5, group_score="top2")),
    (41, 512, 10, "f32", False, dict(score="softmax", groups=4, top_groups=1, group_score="top2")),
    (21, 1024, 16, "f32", True, dict(score="softmax", groups=2, top_groups=2, renormalise=True)),
    (19, 999, 1, "bf16", True, dict(score="sigmoid")),
])
def test_route(r, dev, T, E, k, t, biased, options):
    l = normal(T + E, T, E, t=TYPES[t], scale=2.0)
    bias = normal(E, E, scale=0.1) if biased else None
    m = r.route(l.to(dev), k, bias=None if bias is None else bias.to(dev), **options)
    expert, weight = exact_route(l.double().numpy(), None if bias is None else bias.double().numpy(), k, **options)
    check_routing(m, expert, weight, E)


@pytest.mark.parametrize("options", [dict(), dict(renormalise=True), dict(score="sigmoid"),
                                     dict(score="sigmoid", renormalise=True), GROUPED,
                                     dict(GROUPED, group_score="max"), dict(GROUPED, score="softmax")])
@pytest.mark.parametrize("bias", [None, "zero", "steps"])
@pytest.mark.parametrize("E,k", [(16, 4), (64, 8), (256, 8)])
def test_route_ties_and_masks(r, dev, options, bias, E, k):
    """Scores on a coarse grid (ties everywhere), rows masked to a few experts, to one, to none, rows of the type's
    lowest value, and rows whose sigmoids vanish in 32 bits."""
    T = 96
    g = gen(E + k)
    l = torch.randint(-4, 5, (T, E), generator=g).float() * 0.5
    l[8:24] = torch.where(torch.rand(16, E, generator=g) < 0.8, torch.tensor(-np.inf), l[8:24])
    l[24] = -np.inf
    l[25] = -np.inf
    l[25, E // 2] = 1.0
    l[26] = torch.finfo(torch.float32).min
    l[27] = torch.finfo(torch.float32).min
    l[27, 3] = 0.0
    l[28] -= 150.0
    l[29] = torch.linspace(-200.0, -100.0, E)
    l[30] = 30.0
    b = None if bias is None else torch.zeros(E) if bias == "zero" else (torch.arange(E) % 3).float() * 2.0 ** -26
    m = r.route(l.to(dev), k, bias=None if b is None else b.to(dev), **options)
    with np.errstate(over="ignore"):
        expert, weight = exact_route(l.double().numpy(), None if b is None else b.double().numpy(), k, **options)
    if options.get("renormalise") and options.get("score") == "sigmoid":
        low = expert[26] >= 0  # all equal, further down than 64 bits reach: equal shares
        weight[26] = np.where(low, options.get("scale", 1.0) / max(1, low.sum()), 0.0)
    check_routing(m, expert, weight, E)


def test_route_next_to_a_border(r, dev):
    """Choice scores that differ by less than 32 bits can tell are told apart in 64: pairs of experts with the same
    score whose bias differs in its last bit, in both orders."""
    T, E = 64, 32
    l = normal(1, T, 1, scale=1.0).expand(T, E).contiguous()
    b = torch.full((E,), 2.0 ** -27)
    b[1::2] = torch.nextafter(b[1::2], torch.ones(()))
    m = r.route(l.to(dev), 16, bias=b.to(dev), score="sigmoid")
    expert, weight = exact_route(l.double().numpy(), b.double().numpy(), 16, score="sigmoid")
    assert np.array_equal(expert, np.tile(np.arange(1, 32, 2, dtype=np.int32), (T, 1)))
    check_routing(m, expert, weight, E)


def test_route_groups_next_to_a_border(r, dev):
    """Groups whose scores differ by 2^-44 or not at all: told apart, and ties to the lower group."""
    T, E, groups = 20, 64, 8
    l = torch.zeros(T, E)
    rank = torch.tensor([3, 1, 3, 0, 2, 1, 0, 3])
    b = (rank.repeat_interleave(E // groups) * 2.0 ** -45).float()
    options = dict(score="sigmoid", groups=groups, top_groups=4, group_score="top2")
    for few in (T, 3):
        m = r.route(l[:few].to(dev), 28, bias=b.to(dev), **options)
        expert, weight = exact_route(l[:few].double().numpy(), b.double().numpy(), 28, **options)
        assert sorted(set(expert[0] // 8)) == [0, 2, 4, 7]
        check_routing(m, expert, weight, E)


@pytest.mark.parametrize("T", [1, 2, 4, 5, 15, 16, 17, 33])
@pytest.mark.parametrize("E,k,options", [(8, 2, {}), (64, 6, dict(renormalise=True)), (200, 20, dict(score="sigmoid")), (256, 31, {}),
                                         (256, 8, GROUPED), (300, 32, dict(renormalise=True)), (512, 16, GROUPED), (1024, 9, {})])
def test_route_few_tokens(r, dev, T, E, k, options):
    """Around the number of tokens that one launch takes, for every number of experts in a lane."""
    l = normal(T + k, T, E, t=torch.bfloat16, scale=2.0)
    l[T // 2] = -np.inf
    m = r.route(l.to(dev), k, bias=torch.zeros(E, device=dev) if E == 256 else None, **options)
    expert, weight = exact_route(l.double().numpy(), np.zeros(E) if E == 256 else None, k, **options)
    check_routing(m, expert, weight, E)


def test_no_tokens(r, dev):
    m = r.route(torch.zeros(0, 16, device=dev), 4)
    assert m.expert.shape == (0, 4) and m.expert_ptr.cpu().tolist() == [0] * 17
    W = torch.ones(16, 8, 24, device=dev)
    assert r.experts_mm(torch.zeros(0, 24, device=dev), W, m.expert_ptr, slot=m.slot, k=4).shape == (0, 8)
    assert r.experts_mm_dx(torch.zeros(0, 8, device=dev), W, m.expert_ptr).shape == (0, 24)
    out = torch.full((16, 8, 24), 7.0, device=dev)
    r.experts_mm_dw(torch.zeros(0, 8, device=dev), torch.zeros(0, 24, device=dev), m.expert_ptr, slot=m.slot, k=4, out=out)
    assert (out == 0).all()
    assert r.combine(torch.zeros(0, 24, device=dev), m.pos, m.weight).shape == (0, 24)
    back = r.combine_backward(torch.zeros(0, 24, device=dev), torch.zeros(0, 24, device=dev), m.weight, m.expert_ptr, m.slot)
    assert back["dZ"].shape == (0, 24) and back["dweight"].shape == (0, 4)
    assert r.route_backward(torch.zeros(0, 16, device=dev), m.expert, m.weight).shape == (0, 16)
    A, B = torch.zeros(3, 8, 24, device=dev), torch.zeros(3, 8, 8, device=dev)
    ptr, row, _ = r.columns(torch.zeros(0, 1, dtype=torch.int32, device=dev), 3)
    assert r.adapters_mm(torch.zeros(0, 24, device=dev), A, B, None, ptr, row).shape == (0, 8)


def test_results_in_the_callers_tensors(r, dev):
    l = normal(1, 30, 24).to(dev)
    ref = r.route(l, 3)
    out = r.Routing(*(torch.full_like(x, 77) for x in ref))
    assert r.route(l, 3, out=out) is out
    for a, b in zip(out, ref):
        assert torch.equal(a, b)
    with pytest.raises(ValueError):
        r.route(l, 4, out=out)


def test_tables_that_do_not_fit_reach_nothing_outside(r, dev):
    """expert_ptr beyond the places, falling, or negative: clamped.  The results mean nothing, but what lies behind them
    is not touched."""
    M, N, K = 40, 24, 32
    X, W, dY = normal(1, M, K).to(dev), normal(2, 3, N, K).to(dev), normal(3, M, N).to(dev)
    for ptr in ([0, 10, 1000, 2000], [-5, 20, 10, 40], [30, 20, 10, 0], [0, 0, 0, 2 ** 31 - 1], [50, 60, 70, 80]):
        p = torch.tensor(ptr, dtype=torch.int32, device=dev)
        buf = torch.full((M + 8, N), 7.0, device=dev)
        r.experts_mm(X, W, p, out=buf[:M])
        assert (buf[M:] == 7.0).all()
        buf = torch.full((M + 8, K), 7.0, device=dev)
        r.experts_mm_dx(dY, W, p, out=buf[:M])
        assert (buf[M:] == 7.0).all()
        assert r.experts_mm_dw(dY, X, p).shape == (3, N, K)


def test_route_nan_shows(r, dev):
    l = normal(3, 6, 40)
    l[1, 7] = np.nan
    for options in (dict(), dict(renormalise=True), dict(score="sigmoid", renormalise=True)):
        m = r.route(l.to(dev), 4, bias=torch.zeros(40, device=dev), **options)
        w = m.weight.cpu()
        assert torch.isnan(w[1]).any() and torch.isfinite(w[[0, 2, 3, 4, 5]]).all()
        assert (m.expert.cpu()[1] >= 0).all()


@pytest.mark.parametrize("n,E,k", [(0, 3, 1), (1, 1, 1), (63, 5, 3), (64, 2, 1), (65, 511, 1), (2047, 512, 1), (2048, 64, 8),
                                   (4100, 1023, 4), (5000, 1024, 1), (6000, 256, 8), (70001, 300, 7), (262144, 48, 2)])
def test_columns(r, dev, n, E, k):
    g = np.random.default_rng(n + E)
    expert = g.integers(-2, E + 2, size=(n // k if k > 1 else n, k)).astype(np.int32)
    expert[g.random(expert.shape) < 0.3] = E // 2
    got = r.columns(torch.from_numpy(expert).to(dev), E)
    for x, y in zip(got, exact_columns(expert, E)):
        assert np.array_equal(x.cpu().numpy(), y)


# ---------------------------------------------------------------------------------------------------------------------
# Gradient of the scores
# ---------------------------------------------------------------------------------------------------------------------

def weights_of(l, expert, score, renormalise, scale):
    """The weights as a differentiable function of the scores, in 64 bits."""
    has = expert >= 0
    at = expert.clamp(min=0).long()
    if renormalise:
        logs = (l if score == "softmax" else torch.nn.functional.logsigmoid(l)).gather(1, at)
        logs = logs.masked_fill(~has, -np.inf)
        some = has.any(1)
        out = torch.zeros_like(logs)
        out[some] = torch.softmax(logs[some], 1)
        return out * scale
    s = torch.softmax(l, 1) if score == "softmax" else torch.sigmoid(l)
    return torch.where(has, s.gather(1, at), torch.zeros((), dtype=l.dtype)) * scale


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("T,E,k,t", [(1, 1, 1, "f32"), (5, 72, 6, "f16"), (67, 64, 8, "bf16"), (9, 300, 32, "f32"),
                                     (130, 5, 3, "f32"), (3, 1024, 7, "bf16")])
def test_route_backward(r, dev, score, renormalise, T, E, k, t):
    l = normal(T + E, T, E, t=TYPES[t], scale=1.5)
    expert, _ = exact_route(l.double().numpy(), None, k)
    expert[0, -1] = -1  # a slot without an expert
    expert = torch.from_numpy(expert)
    dw = normal(k, T, k)
    x = l.double().requires_grad_()
    w = weights_of(x, expert, score, renormalise, 2.5)
    w.backward(dw.double())
    got = r.route_backward(l.to(dev), expert.to(dev), dw.to(dev), score=score, renormalise=renormalise, scale=2.5)
    assert got.dtype == l.dtype
    # the terms of dl_e are at most 2.5 max |dw|, once for the choice and once in the row's mean
    magnitude = 2 * 2.5 * dw.double().abs().amax(1, keepdim=True).expand(T, E)
    close(got, x.grad, magnitude, 16, TYPES[t])


def test_route_backward_against_differences(r, dev):
    """The gradient of sum(dw * weight) along a direction, against the difference of the forward weights of fp32 scores
    one step of 2^-7 to each side: the third derivative leaves 2^-14 / 6 times a few, the weights' own 2^-19 / 2^-6 a sum
    of k terms."""
    T, E, k = 20, 48, 6
    for score in ("softmax", "sigmoid"):
        for renormalise in (False, True):
            l = normal(5, T, E, scale=1.0)
            m = r.route(l.to(dev), k, score=score, renormalise=renormalise)
            dw = normal(6, T, k)
            grad = r.route_backward(l.to(dev), m.expert, dw.to(dev), score=score, renormalise=renormalise).cpu().double()
            v = normal(7, T, E, scale=1.0).clamp(-2, 2)
            h = 2.0 ** -7
            up, down = ((weights_of((l + d * v).double(), m.expert.cpu(), score, renormalise, 1.0) * dw.double()).sum(1)
                        for d in (h, -h))
            slope = (up - down) / (2 * h)
            assert ((grad * v.double()).sum(1) - slope).abs().max() < 8 * 6 * h * h + 1e-4


def test_route_backward_repeated_and_foreign_experts(r, dev):
    l = normal(8, 2, 10)
    dw = torch.tensor([[1.0, 2.0, -1.0], [0.5, 1.0, 3.0]])
    e = torch.tensor([[4, 4, 9], [2, 77, -5]], dtype=torch.int32)
    got = r.route_backward(l.to(dev), e.to(dev), dw.to(dev), score="sigmoid").cpu().double()
    s = torch.sigmoid(l.double())
    ds = s * (1 - s)
    ref = torch.zeros(2, 10, dtype=torch.float64)
    ref[0, 4], ref[0, 9], ref[1, 2] = 3.0 * ds[0, 4], -ds[0, 9], 0.5 * ds[1, 2]
    close(got, ref, ref.abs(), 16, torch.float32)


# ---------------------------------------------------------------------------------------------------------------------
# Products of the experts
# ---------------------------------------------------------------------------------------------------------------------

def segments(counts, tail=0):
    """expert_ptr of the given rows per expert, and the number of places with `tail` unrouted ones behind."""
    ptr = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    return torch.from_numpy(ptr), int(ptr[-1]) + tail


def shuffled_slots(M, seed):
    return torch.randperm(M, generator=gen(seed)).int()


CASES = [  # rows of the experts, unrouted places, k, N, K
    ([1], 0, 1, 1, 1),
    ([0, 3, 0, 0, 2, 1], 2, 2, 40, 64),
    ([5, 1, 17, 16, 15], 0, 3, 64, 128),
    ([0, 0, 0], 3, 3, 16, 32),
    ([1] * 70, 2, 6, 136, 96),
    ([130, 0, 127, 128, 1], 14, 4, 144, 72),
    ([300, 261], 3, 4, 257, 130),
    ([33, 31], 0, 8, 129, 333),
    ([700], 0, 1, 200, 264),
    ([64, 65, 63], 0, 2, 512, 1040),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_experts_mm(r, dev, t, gather, case):
    counts, tail, k, N, K = CASES[case]
    ptr, M = segments(counts, tail)
    t = TYPES[t]
    slot = shuffled_slots(M, 1)
    X = normal(2, M // k if gather else M, K, t=t)
    W = normal(3, len(counts), N, K, t=t, scale=K ** -0.5)
    Y = torch.full((M, N), 7.0, dtype=t)
    out = Y.to(dev)
    r.experts_mm(X.to(dev), W.to(dev), ptr.to(dev), slot=slot.to(dev) if gather else None, k=k if gather else 1, out=out)
    rows = X.double()[slot.long() // k] if gather else X.double()
    ref, magnitude = Y.double(), torch.zeros(M, N, dtype=torch.float64)
    for e in range(len(counts)):
        a, b = int(ptr[e]), int(ptr[e + 1])
        ref[a:b] = rows[a:b] @ W[e].double().t()
        magnitude[a:b] = rows[a:b].abs() @ W[e].double().abs().t()
    close(out, ref, magnitude, K, t)
    assert (out[int(ptr[-1]):].cpu() == 7.0).all()  # rows behind the last expert


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("case", range(len(CASES)))
def test_experts_mm_dx(r, dev, t, case):
    counts, tail, _, N, K = CASES[case]
    ptr, M = segments(counts, tail)
    t = TYPES[t]
    dY = normal(4, M, N, t=t)
    W = normal(5, len(counts), N, K, t=t, scale=N ** -0.5)
    out = torch.full((M, K), 7.0, dtype=t, device=dev)
    r.experts_mm_dx(dY.to(dev), W.to(dev), ptr.to(dev), out=out)
    ref, magnitude = torch.full((M, K), 7.0, dtype=torch.float64), torch.zeros(M, K, dtype=torch.float64)
    for e in range(len(counts)):
        a, b = int(ptr[e]), int(ptr[e + 1])
        ref[a:b] = dY[a:b].double() @ W[e].double()
        magnitude[a:b] = dY[a:b].double().abs() @ W[e].double().abs()
    close(out, ref, magnitude, N, t)
    assert (out[int(ptr[-1]):].cpu() == 7.0).all()


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_experts_mm_dw(r, dev, t, gather, case):
    counts, tail, k, N, K = CASES[case]
    ptr, M = segments(counts, tail)
    t = TYPES[t]
    slot = shuffled_slots(M, 6)
    X = normal(7, M // k if gather else M, K, t=t)
    dY = normal(8, M, N, t=t)
    out = torch.full((len(counts), N, K), 7.0, dtype=t, device=dev)
    r.experts_mm_dw(dY.to(dev), X.to(dev), ptr.to(dev), slot=slot.to(dev) if gather else None, k=k if gather else 1, out=out)
    rows = X.double()[slot.long() // k] if gather else X.double()
    ref, magnitude = (torch.zeros(len(counts), N, K, dtype=torch.float64) for _ in range(2))
    for e in range(len(counts)):
        a, b = int(ptr[e]), int(ptr[e + 1])
        ref[e] = dY[a:b].double().t() @ rows[a:b]
        magnitude[e] = dY[a:b].double().abs().t() @ rows[a:b].abs()
    close(out, ref, magnitude, max(counts), t)


@pytest.mark.parametrize("t", list(TYPES))
def test_experts_unaligned(r, dev, t):
    """Contiguous matrices that begin one element behind an aligned address."""
    t = TYPES[t]
    ptr, M = segments([9, 0, 30])
    N, K = 48, 64

    def shifted(x):
        buf = torch.empty(x.numel() + 1, dtype=t, device=dev)
        buf[1:] = x.reshape(-1).to(dev)
        return buf[1:].view(x.shape)

    X, W, dY = normal(1, M, K, t=t), normal(2, 3, N, K, t=t, scale=0.125), normal(3, M, N, t=t)
    out = shifted(torch.zeros(M, N, dtype=t))
    r.experts_mm(shifted(X), shifted(W), ptr.to(dev), out=out)
    assert torch.equal(out, r.experts_mm(X.to(dev), W.to(dev), ptr.to(dev)))
    assert torch.equal(r.experts_mm_dx(shifted(dY), shifted(W), ptr.to(dev)), r.experts_mm_dx(dY.to(dev), W.to(dev), ptr.to(dev)))
    assert torch.equal(r.experts_mm_dw(shifted(dY), shifted(X), ptr.to(dev)), r.experts_mm_dw(dY.to(dev), X.to(dev), ptr.to(dev)))


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("counts,N,K", [([30 + e % 7 for e in range(130)], 520, 72), ([30 + e % 7 for e in range(130)], 515, 67),
                                        ([500, 0, 390, 640], 304, 136), ([500, 0, 390, 640], 301, 131)])
def test_experts_many_tiles(r, dev, t, counts, N, K):
    """Enough tiles, and long enough segments, for the larger tile shapes, with rows of whole 16 bytes and others."""
    t = TYPES[t]
    ptr, M = segments(counts)
    X, W, dY = normal(1, M, K, t=t), normal(2, len(counts), N, K, t=t, scale=K ** -0.5), normal(3, M, N, t=t)
    x, w, dy, p = X.to(dev), W.to(dev), dY.to(dev), ptr.to(dev)
    Y, dX, dW = r.experts_mm(x, w, p), r.experts_mm_dx(dy, w, p), r.experts_mm_dw(dy, x, p)
    X, W, dY = X.double(), W.double(), dY.double()
    for e in range(len(counts)):
        a = slice(int(ptr[e]), int(ptr[e + 1]))
        if counts[e]:
            close(Y[a], X[a] @ W[e].t(), X[a].abs() @ W[e].abs().t(), K, t)
            close(dX[a], dY[a] @ W[e], dY[a].abs() @ W[e].abs(), N, t)
        close(dW[e], dY[a].t() @ X[a], dY[a].abs().t() @ X[a].abs(), counts[e], t)


def test_experts_offsets_beyond_32_bits(r, dev):
    """Rows and weights that lie further than 2^32 bytes from where their matrices begin."""
    t = torch.bfloat16
    K, N, M = 4096, 16, (1 << 19) + 40  # X: 4.3 GB
    ptr = torch.tensor([0, M - 30, M], dtype=torch.int32)
    X = torch.zeros(M, K, dtype=t, device=dev)
    tail = normal(1, 64, K, t=t)
    X[-64:] = tail.to(dev)
    W = normal(2, 2, N, K, t=t, scale=K ** -0.5)
    Y = r.experts_mm(X, W.to(dev), ptr.to(dev))[-64:]
    for rows, e in ((slice(0, 34), 0), (slice(34, 64), 1)):
        x, w = tail[rows].double(), W[e].double()
        close(Y[rows], x @ w.t(), x.abs() @ w.abs().t(), K, t)
    dY = torch.zeros(M, N, dtype=t, device=dev)
    dY[-64:] = normal(3, 64, N, t=t).to(dev)
    d = dY[-64:].cpu().double()
    dW = r.experts_mm_dw(dY, X, ptr.to(dev))
    close(dW[1], d[34:].t() @ tail[34:].double(), d[34:].abs().t() @ tail[34:].double().abs(), 30, t)
    # the matrix [M, K] as dX, written to its end
    dX = r.experts_mm_dx(dY, W.to(dev), ptr.to(dev), out=X)[-64:]
    close(dX[34:], d[34:] @ W[1].double(), d[34:].abs() @ W[1].double().abs(), N, t)
    del X, dX
    N = K = 16384
    W = torch.zeros(9, N, K, dtype=t, device=dev)  # 4.8 GB
    W[8, -32:] = normal(4, 32, K, t=t, scale=K ** -0.5).to(dev)
    x = normal(5, 40, K, t=t)
    for counts in ([0] * 8 + [40], [4] * 8 + [8]):
        ptr, M = segments(counts)
        Y = r.experts_mm(x.to(dev), W, ptr.to(dev))
        a, w = x[-counts[8]:].double(), W[8, -32:].cpu().double()
        close(Y[-counts[8]:, -32:], a @ w.t(), a.abs() @ w.abs().t(), K, t)


def test_experts_infinities_stay_in_their_rows(r, dev):
    """Infinities and NaN in one row, or in rows that no expert has, reach no other row."""
    ptr, M = segments([3, 2], 3)
    X = normal(1, M, 40)
    X[1, 5] = np.inf
    X[5:] = np.nan
    W = normal(2, 2, 24, 40)
    dY = normal(3, M, 24)
    dY[5:] = np.nan
    out = torch.zeros(M, 24, device=dev)
    r.experts_mm(X.to(dev), W.to(dev), ptr.to(dev), out=out)
    fine = torch.isfinite(out.cpu()).all(1)
    assert fine.tolist() == [True, False, True, True, True, True, True, True]
    dW = r.experts_mm_dw(dY.to(dev), X.to(dev), ptr.to(dev)).cpu()
    assert torch.isfinite(dW[1]).all() and torch.isfinite(dW[0][:, :5]).all()


def test_experts_foreign_slots(r, dev):
    """Slots out of range count as rows of zeros."""
    ptr, M = segments([4, 4])
    X, W, dY = normal(1, 4, 32), normal(2, 2, 16, 32), normal(3, 8, 16)
    slot = torch.tensor([0, -3, 2, 1000, 4, 5, 6, 2 ** 31 - 1], dtype=torch.int32)
    rows = X.double()[(slot.long() // 2).clamp(0, 3)]
    rows[[1, 3, 7]] = 0.0
    Y = r.experts_mm(X.to(dev), W.to(dev), ptr.to(dev), slot=slot.to(dev), k=2)
    dW = r.experts_mm_dw(dY.to(dev), X.to(dev), ptr.to(dev), slot=slot.to(dev), k=2)
    for e in range(2):
        a = slice(4 * e, 4 * e + 4)
        close(Y[a], rows[a] @ W[e].double().t(), rows[a].abs() @ W[e].double().abs().t(), 32, torch.float32)
        close(dW[e], dY[a].double().t() @ rows[a], dY[a].double().abs().t() @ rows[a].abs(), 4, torch.float32)


# ---------------------------------------------------------------------------------------------------------------------
# Combination
# ---------------------------------------------------------------------------------------------------------------------

def routing_of(T, E, k, none, seed):
    g = np.random.default_rng(seed)
    expert = np.stack([g.choice(E, size=k, replace=False) for _ in range(T)]).astype(np.int32) if T else np.zeros((0, k), np.int32)
    expert[g.random(expert.shape) < none] = -1
    ptr, slot, pos = exact_columns(expert, E)
    return torch.from_numpy(ptr), torch.from_numpy(slot), torch.from_numpy(pos)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("T,E,k,N,none", [(1, 2, 1, 1, 0.0), (3, 4, 4, 8, 0.3), (70, 16, 6, 1030, 0.1), (129, 9, 5, 264, 0.0),
                                          (17, 8, 8, 4097, 0.5), (5, 3, 2, 16, 1.0), (67, 5, 3, 39, 0.2), (40, 6, 4, 64, 0.1),
                                          (33, 4, 2, 121, 0.1), (21, 7, 5, 250, 0.3), (9, 2, 1, 512, 0.0)])
def test_combine(r, dev, t, T, E, k, N, none):
    t = TYPES[t]
    ptr, slot, pos = routing_of(T, E, k, none, T + N)
    M = T * k
    Z, dY, base = normal(1, M, N, t=t), normal(2, T, N, t=t), normal(3, T, N, t=t)
    Z[int(ptr[-1]):] = np.nan  # rows that nobody has
    w = torch.rand(T, k, generator=gen(4))
    has = pos >= 0
    rows = torch.where(has[:, :, None], Z.double()[pos.clamp(min=0).long()], torch.zeros((), dtype=torch.float64))
    ref = (rows * w.double()[:, :, None]).sum(1)
    size = (rows.abs() * w.double()[:, :, None]).sum(1)
    close(r.combine(Z.to(dev), pos.to(dev), w.to(dev)), ref, size, k, t)
    close(r.combine(Z.to(dev), pos.to(dev), w.to(dev), base=base.to(dev)), ref + base.double(), size + base.double().abs(), k + 1, t)
    y = base.to(dev)
    r.combine(Z.to(dev), pos.to(dev), base=y, out=y)
    close(y, rows.sum(1) + base.double(), rows.abs().sum(1) + base.double().abs(), k + 1, t)

    got = r.combine_backward(dY.to(dev), Z.to(dev), w.to(dev), ptr.to(dev), slot.to(dev))
    dZ = torch.zeros(M, N, dtype=torch.float64)
    token = torch.arange(T)[:, None].expand(T, k)
    dZ[pos[has].long()] = w.double()[has][:, None] * dY.double()[token[has]]
    close(got["dZ"], dZ, dZ.abs(), 0, t)
    close(got["dweight"], (rows * dY.double()[:, None, :]).sum(2), (rows.abs() * dY.double().abs()[:, None, :]).sum(2), N,
          torch.float32)


def test_combine_is_the_product_with_the_routing_matrix(r, pkg, dev):
    """The same sum through the merge-path SpMM, whose sums have another order: both within k + 1 roundings of the
    definition."""
    T, E, k, N = 150, 10, 4, 64
    ptr, slot, pos = routing_of(T, E, k, 0.0, 5)
    Z, w = normal(6, T * k, N), torch.rand(T, k, generator=gen(7))
    mine = r.combine(Z.to(dev), pos.to(dev), w.to(dev)).cpu().double()
    # a square matrix of T * k rows of which the first T have nonzeros
    row_ptr = torch.clamp(torch.arange(T * k + 1) * k, max=T * k).int()
    sp = pkg.spmm
    csr = sp.CsrDevice(row_ptr.to(dev), pos.reshape(-1).to(dev), w.reshape(-1).to(dev))
    other = sp.spmm_merge_path(csr, Z.to(dev), sp.generate_mp_sched(csr.row_ptr, T * k)).cpu().double()[:T]
    size = (Z.double()[pos.long()].abs() * w.double()[:, :, None]).sum(1)
    assert ((mine - other).abs() <= 2 * (k + 1) * U * size).all()


# ---------------------------------------------------------------------------------------------------------------------
# Adapters
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("T,E,R,K,N,none", [(1, 1, 1, 1, 1, 0.0), (1, 4, 16, 512, 320, 0.0), (2, 3, 8, 64, 40, 1.0),
                                            (40, 64, 16, 1024, 72, 0.1), (33, 2, 24, 130, 131, 0.2), (200, 5, 64, 2048, 300, 0.1),
                                            (17, 1, 100, 96, 64, 0.0), (50, 3, 256, 320, 129, 0.3), (700, 6, 33, 257, 65, 0.1)])
@pytest.mark.parametrize("with_base", [False, True])
def test_adapters(r, dev, t, T, E, R, K, N, none, with_base):
    t = TYPES[t]
    g = gen(T + K)
    adapter = torch.randint(0, E, (T, 1), generator=g)
    adapter[torch.rand(T, 1, generator=g) < none] = -1
    X, A, B = normal(1, T, K, t=t), normal(2, E, R, K, t=t, scale=K ** -0.5), normal(3, E, N, R, t=t, scale=R ** -0.5)
    scale = torch.rand(E, generator=g) + 0.5
    base = normal(4, T, N, t=t) if with_base else None
    ptr, row, _ = r.columns(adapter.int().to(dev), E)
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), scale.to(dev), ptr, row, base=base.to(dev) if with_base else None)
    ref = base.double() if with_base else torch.zeros(T, N, dtype=torch.float64)
    size, split = ref.abs(), torch.zeros(T, N, dtype=torch.float64)
    for e in range(E):
        at = (adapter[:, 0] == e)
        v = X[at].double() @ A[e].double().t()
        v_size = X[at].double().abs() @ A[e].double().abs().t()
        ref[at] += scale[e].double() * v @ B[e].double().t()
        size[at] += scale[e].double() * v_size @ B[e].double().abs().t()
        split[at] = scale[e].double() * v.abs() @ B[e].double().abs().t()
    # V stands as the sum of two numbers of the type: off by at most half(t)^2 of it, or for fp16 by half of its
    # smallest subnormal step, 2^-25, times |B|
    n = K + R + 4
    extra = 0.0 if t == torch.float32 else half(t) ** 2 * split
    if t == torch.float16:
        extra = extra + 2.0 ** -25 * torch.stack([B[a].double().abs().sum(1) if a >= 0 else torch.zeros(N, dtype=torch.float64)
                                                  for a in adapter[:, 0].tolist()])
    close(out, ref, size + extra / ((2 * n + 2) * U), n, t)
    if with_base:
        y = base.to(dev)
        assert torch.equal(r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), scale.to(dev), ptr, row, base=y, out=y), out)
        assert y.data_ptr() != 0 and torch.equal(y, out)


def test_adapters_beyond_the_range_of_fp16(r, dev):
    """V over 65504 in fp16, taken down again by B: the result is finite.  And infinite inputs stay in their rows."""
    T, K, N = 20, 256, 32
    X, A = torch.full((T, K), 64.0, dtype=torch.float16), torch.full((1, 8, K), 8.0, dtype=torch.float16)
    B = torch.full((1, N, 8), 2.0 ** -10, dtype=torch.float16)
    ptr, row, _ = r.columns(torch.zeros(T, 1, dtype=torch.int32, device=dev), 1)
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), None, ptr, row)
    assert (out.cpu() == 64 * 8 * 256 * 8 / 1024).all()
    # one token's large values take no bits from its neighbours'
    X = normal(1, T, K, t=torch.float16, scale=0.01)
    B2 = normal(2, 1, N, 8, t=torch.float16)
    alone = r.adapters_mm(X.to(dev), A.to(dev), B2.to(dev), None, ptr, row).cpu()
    X[3] = 64.0
    beside = r.adapters_mm(X.to(dev), A.to(dev), B2.to(dev), None, ptr, row).cpu()
    others = torch.arange(T) != 3
    assert torch.equal(alone[others], beside[others])
    X = torch.full((T, K), 64.0, dtype=torch.float16)
    X[3, 9] = np.inf
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), None, ptr, row).cpu()
    assert torch.isinf(out[3]).all() and (out[[0, 1, 2, 4, 19]] == 1024.0).all()


# ---------------------------------------------------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------------------------------------------------

def test_layer_forward_and_backward(r, dev):
    """A layer of experts as it is used: route, gathered first product, activation, second product, combination; and its
    whole backward pass, against autograd in 64 bits.  bf16 data: every tensor between is rounded to 2^-9 of itself, and
    the sums that follow average that, so 2^-5 of the largest value of a row of results leaves room for 16 of them."""
    T, E, k, D, H = 96, 12, 3, 128, 160
    t = torch.bfloat16
    X, G = normal(1, T, D, t=t), normal(2, E, D, t=t, scale=D ** -0.5)
    W1, W2 = normal(3, E, H, D, t=t, scale=D ** -0.5), normal(4, E, D, H, t=t, scale=H ** -0.5)
    dOut = normal(5, T, D, t=t)
    x, w1, w2 = (v.to(dev) for v in (X, W1, W2))
    scores = (X.float() @ G.float().t())
    m = r.route(scores.to(dev), k, renormalise=True)
    h = r.experts_mm(x, w1, m.expert_ptr, slot=m.slot, k=k)
    a = torch.relu(h)
    z = r.experts_mm(a, w2, m.expert_ptr)
    y = r.combine(z, m.pos, m.weight)
    back = r.combine_backward(dOut.to(dev), z, m.weight, m.expert_ptr, m.slot)
    dw2 = r.experts_mm_dw(back["dZ"], a, m.expert_ptr)
    dh = r.experts_mm_dx(back["dZ"], w2, m.expert_ptr) * (h > 0)
    dw1 = r.experts_mm_dw(dh, x, m.expert_ptr, slot=m.slot, k=k)
    dx = r.combine(r.experts_mm_dx(dh, w1, m.expert_ptr), m.pos)
    dscores = r.route_backward(scores.to(dev), m.expert, back["dweight"], renormalise=True)

    X6, W16, W26, S6 = (v.double().requires_grad_() for v in (X, W1, W2, scores))
    w = weights_of(S6, m.expert.cpu(), "softmax", True, 1.0)
    e = m.expert.cpu().long()
    keep = (h.cpu() > 0)[m.pos.cpu().long()].double()  # the kernel's own signs: relu is not smooth
    hid = torch.einsum("td,tkhd->tkh", X6, W16[e]) * keep
    Y6 = (torch.einsum("tkh,tkdh->tkd", hid, W26[e]) * w[:, :, None]).sum(1)
    Y6.backward(dOut.double())
    for got, ref in ((y, Y6), (dx, X6.grad), (dw1, W16.grad), (dw2, W26.grad), (dscores, S6.grad)):
        ref = ref.detach().reshape(-1, ref.shape[-1])
        got = got.cpu().double().reshape(ref.shape)
        assert ((got - ref).abs() <= 2.0 ** -5 * ref.abs().amax(1, keepdim=True) + 1e-6).all()


def test_captured_layer(r, dev):
    """Route, products, combination and adapters in one captured graph: every replay with new inputs gives what the eager
    calls give, bit for bit, with eager work between the replays."""
    T, E, k, D = 40, 16, 2, 64
    t = torch.bfloat16
    W = normal(1, E, D, D, t=t, scale=0.125).to(dev)
    A, B = normal(2, 3, 8, D, t=t, scale=0.125).to(dev), normal(3, 3, D, 8, t=t, scale=0.3).to(dev)
    x, scores = torch.zeros(T, D, dtype=t, device=dev), torch.zeros(T, E, device=dev)
    adapter = (torch.arange(T, dtype=torch.int32, device=dev) % 4).view(T, 1)

    def layer():
        m = r.route(scores, k, score="sigmoid", renormalise=True)
        z = r.experts_mm(x, W, m.expert_ptr, slot=m.slot, k=k)
        y = r.combine(z, m.pos, m.weight)
        ptr, row, _ = r.columns(adapter, 3)
        dw = r.experts_mm_dw(z, x, m.expert_ptr, slot=m.slot, k=k)
        return r.adapters_mm(x, A, B, None, ptr, row, base=y), dw, m.expert

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()
    for n in range(4):
        x.copy_(normal(10 + n, T, D, t=t))
        scores.copy_(normal(20 + n, T, E))
        graph.replay()
        torch.cuda.synchronize()
        for got, ref in zip(captured, layer()):
            assert torch.equal(got, ref)


def test_on_another_stream(r, dev):
    """Calls run on the stream that is current, in its order."""
    scores = normal(1, 5000, 64).to(dev)
    ref = r.route(scores, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(scores)
        for _ in range(20):
            late.add_(0.0)
        late.copy_(scores)
        got = r.route(late, 4)
    side.synchronize()
    for a, b in zip(got, ref):
        assert torch.equal(a, b)


def test_results_repeat(r, dev):
    """The same bits from call to call."""
    l = normal(1, 9000, 96, t=torch.bfloat16).to(dev)
    a, b = r.route(l, 6), r.route(l, 6)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    X, W = normal(2, 9000, 64, t=torch.bfloat16).to(dev), normal(3, 96, 48, 64, t=torch.bfloat16).to(dev)
    Y = [r.experts_mm(X, W, a.expert_ptr, slot=a.slot, k=6) for _ in range(2)]
    assert torch.equal(*Y)
    assert torch.equal(*(r.experts_mm_dw(Y[0], X, a.expert_ptr, slot=a.slot, k=6) for _ in range(2)))


def test_python_refusals(r, dev):
    """Arguments that the Python face refuses before any kernel runs."""
    x, w = torch.zeros(8, 32, device=dev), torch.zeros(2, 16, 32, device=dev)
    ptr = torch.tensor([0, 4, 8], dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        r.experts_mm(x.t(), w, ptr)
    with pytest.raises(ValueError):
        r.experts_mm(x[:, ::2], torch.zeros(2, 16, 16, device=dev), ptr)
    with pytest.raises(TypeError):
        r.experts_mm(x, w.half(), ptr)
    with pytest.raises(TypeError):
        r.experts_mm(x, w, ptr.long())
    with pytest.raises(ValueError):
        r.experts_mm(x, w, ptr[:2])
    with pytest.raises(ValueError):
        r.experts_mm(x, w, ptr, slot=ptr, k=2)
    with pytest.raises(TypeError):
        r.experts_mm(x.double(), w.double(), ptr)
    with pytest.raises(ValueError):
        r.experts_mm(x, w, ptr, out=torch.zeros(8, 15, device=dev))
    with pytest.raises(ValueError):
        r.route(x, 2, score="tanh")
    for k, options in ((33, {}), (0, {}), (2, dict(groups=5)), (2, dict(groups=4, top_groups=5)),
                       (20, dict(groups=4, top_groups=2))):
        with pytest.raises((ValueError, r._cabi.MpsError)):
            r.route(x, k, **options)
    with pytest.raises(r._cabi.MpsError):
        r.route(torch.zeros(2, 1025, device=dev), 2)
    with pytest.raises(TypeError):
        r.combine(x, ptr.view(1, 3), weight=torch.zeros(1, 3, device=dev).half())
    with pytest.raises(ValueError):
        r.adapters_mm(x, torch.zeros(2, 4, 32, device=dev), torch.zeros(2, 16, 8, device=dev), None, ptr, ptr)
