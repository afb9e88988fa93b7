"""Sparse routing at its edges: masked groups, NaN and infinities in the choice, small and large values between the two
products of an adapter, sizes beyond one launch's threads, and the kernels' shapes one by one."""
import numpy as np
import pytest
import torch

from test_gpu_routing import GROUPED, TYPES, check_routing, close, exact_columns, gen, half, normal, routing_of, segments
from test_gpu_routing import shuffled_slots, weights_of

pytestmark = pytest.mark.gpu


@pytest.fixture
def r(pkg, dev):
    return pkg.routing


# ---------------------------------------------------------------------------------------------------------------------
# The choice among groups that a mask leaves with one expert or with none, NaN, infinities
# ---------------------------------------------------------------------------------------------------------------------

def rank(c):
    """Order of choice scores: NaN above everything."""
    return (1, 0.0) if np.isnan(c) else (0, c)


def exact_choice(l, bias, k, score, groups, top_groups, group_score):
    """Experts of one token, from the definition: c = s + bias, -inf where the score or the bias is; a group counts as the
    largest of its c or as the sum of the two largest, by the arithmetic of infinities; ties to the lower index."""
    can = ~((l == -np.inf) | (bias == -np.inf))
    with np.errstate(all="ignore"):
        if score == "sigmoid":
            s = 1.0 / (1.0 + np.exp(-l))
        elif np.isnan(l).any() or l.max() == np.inf:
            s = np.full(l.shape, np.nan)
        else:
            s = np.where(l > -np.inf, np.exp(l - l.max()), 0.0) if l.max() > -np.inf else np.zeros(l.shape)
            s = s / s.sum() if s.sum() else s
        c = np.where(can, s + bias, -np.inf)
        of = []
        for g in c.reshape(groups, -1):
            best = sorted(g, key=rank, reverse=True)
            of.append(best[0] if group_score == "max" else best[0] + best[1])
    kept = sorted(range(groups), key=lambda g: rank(of[g]), reverse=True)[:top_groups]
    at = [e for e in range(len(l)) if e * groups // len(l) in kept and c[e] != -np.inf]
    at = sorted(at, key=lambda e: rank(c[e]), reverse=True)[:k]
    return at + [-1] * (k - len(at))


LAYOUTS = [(8, 2, 1, 2), (64, 8, 4, 6), (256, 8, 4, 8), (72, 6, 3, 9), (90, 18, 5, 7), (320, 64, 9, 5), (512, 4, 2, 31),
           (1024, 16, 3, 32)]  # experts, groups, kept ones, k: groups in whole lanes and others


def masked_groups(seed, T, E, groups):
    """Scores of which the mask leaves every group none, one, two or all of its experts."""
    g = np.random.default_rng(seed)
    l = g.normal(size=(T, groups, E // groups)).astype(np.float32)
    for t in range(T):
        for h in range(groups):
            left = g.choice([0, 1, 1, 2, E // groups], p=[0.3, 0.2, 0.2, 0.2, 0.1])
            l[t, h, g.permutation(E // groups)[left:]] = -np.inf
    return l.reshape(T, E)


def check_choice(m, l, bias, k, score, groups, top_groups, group_score="top2"):
    bias = np.zeros(l.shape[1]) if bias is None else bias.astype(np.float64)
    ref = np.array([exact_choice(x, bias, k, score, groups, top_groups, group_score) for x in l.astype(np.float64)], np.int32)
    assert np.array_equal(m.expert.cpu().numpy(), ref)
    for got, x in zip((m.expert_ptr, m.slot, m.pos), exact_columns(ref, l.shape[1])):
        assert np.array_equal(got.cpu().numpy(), x)
    return ref


@pytest.mark.parametrize("T", [1, 4, 33])
@pytest.mark.parametrize("E,groups,top_groups,k", LAYOUTS)
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_that_a_mask_leaves_with_few_experts(r, dev, T, E, groups, top_groups, k, score, biased):
    """With the sum of the two largest a group with one expert left counts as one with none: -inf, and the lower group
    comes first.  No token has a tie of finite sums."""
    l = masked_groups(E + T, T, E, groups)
    bias = np.random.default_rng(E).normal(size=E).astype(np.float32) * 0.1 if biased else None
    for group_score in ("top2", "max"):
        m = r.route(torch.from_numpy(l).to(dev), k, score=score, bias=torch.from_numpy(bias).to(dev) if biased else None,
                    groups=groups, top_groups=top_groups, group_score=group_score)
        if group_score == "max" and not biased:  # l itself is compared, which is the same where nothing saturates
            check_choice(m, l, None, k, "sigmoid", groups, top_groups, "max")
        else:
            check_choice(m, l, bias, k, score, groups, top_groups, group_score)


@pytest.mark.parametrize("T", [1, 4, 33])
@pytest.mark.parametrize("E,groups,top_groups,k", LAYOUTS)
@pytest.mark.parametrize("group_score", ["top2", "max"])
def test_groups_with_nan_and_infinities(r, dev, T, E, groups, top_groups, k, group_score):
    """NaN scores (one or two of a group, beside masked ones too) and infinite biases: classes of their own, the larger
    first, ties to the lower group and expert."""
    g = np.random.default_rng(E + 7 * T)
    l = masked_groups(E + 1, T, E, groups)
    for t in range(T):
        l[t, g.integers(0, E, size=g.integers(0, 4))] = np.nan
    bias = g.normal(size=E).astype(np.float32) * 0.1
    bias[g.integers(0, E, size=3)] = np.inf
    m = r.route(torch.from_numpy(l).to(dev), k, score="sigmoid", bias=torch.from_numpy(bias).to(dev), groups=groups,
                top_groups=top_groups, group_score=group_score)
    check_choice(m, l, bias, k, "sigmoid", groups, top_groups, group_score)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("E,groups,top_groups,k", LAYOUTS)
def test_a_token_does_not_depend_on_its_neighbours(r, dev, score, biased, E, groups, top_groups, k):
    """Rows with masks beside a few with ties, which are chosen with every bit of a double: in another order every row has
    the same experts and the same weights, bit for bit."""
    T = 256
    l = torch.from_numpy(masked_groups(E, T, E, groups))
    l[::16] = 0.5
    bias = torch.zeros(E, device=dev) if biased else None
    options = dict(score=score, bias=bias, groups=groups, top_groups=top_groups, group_score="top2")
    m = r.route(l.to(dev), k, **options)
    for seed in range(3):
        order = torch.randperm(T, generator=gen(seed))
        other = r.route(l[order].to(dev), k, **options)
        assert torch.equal(other.expert, m.expert[order.to(dev)])
        assert torch.equal(other.weight, m.weight[order.to(dev)])


@pytest.mark.parametrize("T", [1, 5, 40])
@pytest.mark.parametrize("E,groups,top_groups,k", [(16, 1, 1, 3), (200, 1, 1, 12), (700, 1, 1, 32)] + LAYOUTS[1:5])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_a_bias_of_minus_infinity_masks_nan(r, dev, T, E, groups, top_groups, k, score):
    """An expert that its bias masks is never chosen, also where its score, or what the softmax makes of its row, is NaN
    or infinite."""
    g = np.random.default_rng(E + T)
    l = g.normal(size=(T, E)).astype(np.float32)
    bias = g.normal(size=E).astype(np.float32) * 0.1
    masked = g.permutation(E)[:E // 3]
    bias[masked] = -np.inf
    l[:, masked[0]] = np.nan
    l[::2, masked[1]] = np.inf
    m = r.route(torch.from_numpy(l).to(dev), k, score=score, bias=torch.from_numpy(bias).to(dev), groups=groups,
                top_groups=top_groups, group_score="top2" if groups > 1 else "max")
    ref = check_choice(m, l, bias, k, score, groups, top_groups, "top2" if groups > 1 else "max")
    assert not np.isin(ref, masked).any()
    w = m.weight.cpu().numpy()
    assert (np.isnan(w[ref >= 0]) if score == "softmax" else np.isfinite(w)).all()


# ---------------------------------------------------------------------------------------------------------------------
# What stands between the two products of an adapter
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("T", [3, 300])
@pytest.mark.parametrize("R", [4, 16, 40, 130])
@pytest.mark.parametrize("x,a,b", [(2.0 ** -14, 2.0 ** -6, 2.0 ** 10), (2.0 ** -10, 2.0 ** -14, 2.0 ** 12), (2.0 ** -20, 2.0 ** -12, 2.0 ** 13),
                                   (1.0, 1.0, 1.0), (2.0 ** 11, 2.0 ** 8, 2.0 ** -10), (2.0 ** 14, 2.0 ** 14, 2.0 ** -14)])
def test_adapters_fp16_of_any_size(r, dev, T, R, x, a, b):
    """V = X A^T from far below fp16's smallest numbers to far above its largest, with B that brings it back.  The largest
    of a token's V is taken to 2^14 or more, so that with two halves each V is off by at most 2^-22 of itself (twice half a
    step) or by 2^-25 of where the largest is 2^14 (half of the smallest step): 2^-39 of the largest."""
    t, K, N, E = torch.float16, 64, 48, 2
    X, A, B = normal(T, T, K, t=t, scale=x / 8), normal(2, E, R, K, t=t, scale=a / 8), normal(3, E, N, R, t=t, scale=b / 4)
    down = 2.0 ** -8 if x * a * b > 2.0 ** 10 else 1.0  # the results are numbers of fp16
    B = (B.double() * down).to(t)
    adapter = torch.arange(T) % E
    ptr, row, _ = r.columns(adapter.int().view(T, 1).to(dev), E)
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), None, ptr, row)
    V = torch.stack([X[i].double() @ A[adapter[i]].double().t() for i in range(T)])
    V_size = torch.stack([X[i].double().abs() @ A[adapter[i]].double().abs().t() for i in range(T)])
    ref, size, split, all_b = (torch.stack([v[i] @ B[adapter[i]].double().abs().t() if v is not V else
                                            V[i] @ B[adapter[i]].double().t() for i in range(T)])
                               for v in (V, V_size, V.abs(), torch.ones_like(V)))
    n = K + R + 4
    extra = 2.0 ** -22 * split + 2.0 ** -39 * V.abs().amax(1, keepdim=True) * all_b
    assert ref.abs().max() < 60000
    close(out, ref, size + extra / ((2 * n + 2) * 2.0 ** -24), n, t)


def test_adapters_fp16_large_values_leave_the_others_their_bits(r, dev):
    """One value of V above fp16's largest, which B multiplies by zero, beside ordinary ones; and values above 2^32 that
    cancel: the result is finite and exact to 32 bits' sums."""
    t, K = torch.float16, 32
    X = torch.zeros(2, K, dtype=t)
    X[:, 0] = 1.0
    X[1, 1] = 32768.0
    A = torch.zeros(1, 4, K, dtype=t)
    A[0, :, 0] = torch.tensor([0.0, 0.02, 0.3, 0.5])
    A[0, 0, 1] = 2.125
    B = torch.tensor([[[0.0, 1.0, 1.0, 1.0]] * 8], dtype=t)
    ptr, row, _ = r.columns(torch.zeros(2, 1, dtype=torch.int32, device=dev), 1)
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), None, ptr, row).cpu()
    ref = A[0, 1:, 0].double().sum()
    # V to 2^-39 of 69632 < 2^-22, three of them; then the result's half step of 2^-11
    assert ((out.double() - ref).abs() <= 2.0 ** -11 * ref + 3 * 2.0 ** -22 + 2.0 ** -22).all()
    assert torch.equal(out[0], out[1])
    A[0, 0, 1] = A[0, 1, 1] = 32768.0 * 1.5
    A[0, :2, 2:] = A[0, 0, 1]
    X[1, 2:] = 32768.0  # V = 5e10, twice
    B = torch.tensor([[[1.0, -1.0, 0.0, 0.0]] * 8], dtype=t)
    A[0, :, 0] = 0.0
    out = r.adapters_mm(X.to(dev), A.to(dev), B.to(dev), None, ptr, row).cpu()
    assert (out == 0).all()


def test_adapters_fp16_infinite_and_far_values_keep_their_signs(r, dev):
    """A value that the scale makes infinite beside a finite one of the other sign, far beyond fp16: infinite, not NaN."""
    t, K = torch.float16, 16
    X, A = torch.zeros(1, K, dtype=t), torch.zeros(1, 2, K, dtype=t)
    X[0, 0], X[0, 1] = 32768.0, -2.0 ** -10
    A[0, 0, 0], A[0, 1, 1] = 1.0, 2.0 ** -10
    scale = torch.full((1,), 3.0e38)
    ptr, row, _ = r.columns(torch.zeros(1, 1, dtype=torch.int32, device=dev), 1)
    out = r.adapters_mm(X.to(dev), A.to(dev), torch.ones(1, 8, 2, dtype=t).to(dev), scale.to(dev), ptr, row).cpu()
    assert (out == np.inf).all()


def test_parts_of_a_routing_matrix_change_apart(r, dev):
    """An in-place change of the weights is none of the indices, which autograd may hold for a backward pass."""
    class Chosen(torch.autograd.Function):
        @staticmethod
        def forward(ctx, w, expert):
            ctx.save_for_backward(expert)
            return w * 2

        @staticmethod
        def backward(ctx, d):
            return d * (ctx.saved_tensors[0] >= 0), None

    m = r.route(normal(1, 20, 16).to(dev), 2)
    before = [x._version for x in m]
    leaf = torch.ones(20, 2, device=dev, requires_grad=True)
    out = Chosen.apply(leaf, m.expert)
    m.weight.mul_(0.5)
    assert [x._version for x in m] == [before[0], before[1] + 1] + before[2:]
    out.sum().backward()
    assert torch.equal(leaf.grad, torch.ones_like(leaf))


# ---------------------------------------------------------------------------------------------------------------------
# More rows than one dimension of a launch has threads
# ---------------------------------------------------------------------------------------------------------------------

def test_route_backward_of_many_tokens(r, dev):
    """2^26 tokens and some, a wavefront each: 2^32 threads."""
    T, E = (1 << 26) + 77, 2
    scores = torch.zeros(T, E, dtype=torch.float16, device=dev)
    expert = torch.zeros(T, 1, dtype=torch.int32, device=dev)
    dweight = torch.zeros(T, 1, device=dev)
    for first in (0, 1 << 25, T - 1000):
        scores[first:first + 900] = normal(first, 900, E, t=torch.float16).to(dev)
        expert[first:first + 900:2] = 1
        dweight[first:first + 900] = normal(first + 1, 900, 1).to(dev)
    out = r.route_backward(scores, expert, dweight)
    for at in (slice(0, 1000), slice(1 << 25, (1 << 25) + 1000), slice(T - 1000, T)):
        x = scores[at].cpu().double().requires_grad_()
        dw = dweight[at].cpu().double()
        weights_of(x, expert[at].cpu(), "softmax", False, 1.0).backward(dw)
        close(out[at], x.grad, 2 * dw.abs().expand(-1, E), 16, torch.float16)


def test_route_of_many_tokens(r, dev):
    """2^28 tokens and some, 16 lanes each."""
    T, E = (1 << 28) + 77, 3
    scores = torch.zeros(T, E, dtype=torch.bfloat16, device=dev)
    scores[:, 2] = 1.0
    scores[-77:, 1] = 2.0
    scores[:50, 0] = 3.0
    m = r.route(scores, 1, score="sigmoid")
    assert m.expert_ptr.cpu().tolist() == [0, 50, 127, T]
    assert (m.expert[:50] == 0).all() and (m.expert[50:-77] == 2).all() and (m.expert[-77:] == 1).all()
    assert torch.equal(m.slot[:50].cpu(), torch.arange(50, dtype=torch.int32))
    assert torch.equal(m.slot[50:127].cpu(), torch.arange(T - 77, T, dtype=torch.int32))
    assert torch.equal(m.pos[-77:, 0].cpu(), torch.arange(50, 127, dtype=torch.int32))
    assert int(m.pos[T - 78, 0]) == T - 1
    one = (1.0 / (1.0 + np.exp(-1.0)))
    assert (m.weight[50:-77] - one).abs().max() <= 2.0 ** -19


def test_combine_backward_of_many_places(r, dev):
    """2^29 places and some, 8 lanes each."""
    k = 32
    T = (1 << 24) + 3
    M, t = T * k, torch.bfloat16
    g = torch.Generator(device=dev).manual_seed(1)
    dY = torch.randint(-8, 9, (T, 1), generator=g, device=dev).to(t)
    Z = torch.randint(-8, 9, (M, 1), generator=g, device=dev, dtype=torch.int8).to(t)
    weight = torch.full((T, k), 0.5, device=dev)
    ptr = torch.tensor([0, M - 5], dtype=torch.int32, device=dev)
    slot = torch.arange(M, dtype=torch.int32, device=dev).flip(0)
    got = r.combine_backward(dY, Z, weight, ptr, slot)
    del weight, slot
    rows = dY.view(T, 1).expand(T, k).reshape(M)  # of every slot
    want = (rows * Z.view(M).flip(0)).float()     # whole numbers below 2^7
    want[:5] = 0.0
    assert torch.equal(got["dweight"].view(M), want)
    want = (rows * 0.5).flip(0)
    want[-5:] = 0.0
    assert torch.equal(got["dZ"].view(M), want)


def test_combine_of_many_rows(r, dev):
    """More than 2^32 chunks of 16 bytes in the result."""
    N, t = 1024, torch.float16
    T = (1 << 25) + 9
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(dev)[0] < 80 << 30:
        pytest.skip("the result takes 64 GB")
    Z = normal(1, 40, N, t=t).to(dev)
    pos = (torch.arange(T, device=dev) % 41).int().view(T, 1)
    pos[pos == 40] = -1
    out = r.combine(Z, pos)
    for at in (slice(0, 300), slice(T // 2, T // 2 + 300), slice(T - 300, T)):
        p = pos[at, 0].long()
        assert torch.equal(out[at], torch.where((p < 0)[:, None], torch.zeros((), dtype=t, device=dev), Z[p.clamp(min=0)]))
    del out
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------------------------------
# The shapes of the experts' products
# ---------------------------------------------------------------------------------------------------------------------

def ragged(mean, E, seed):
    """Rows of E experts with the given mean exactly, uneven, one expert without rows where there are more than two."""
    g = np.random.default_rng(seed)
    share = g.random(E) + 0.1
    if E > 2:
        share[E // 2] = 0.0
    counts = np.floor(share / share.sum() * mean * E).astype(int)
    counts[0] += mean * E - counts.sum()
    return counts.tolist()


# Every shape of the three products by the rows of an expert, the number of tiles and the rows' alignment (whole 16 bytes
# or not): few rows, 64 and 128 wide through registers and straight into LDS, 256 x 256.
SHAPES = [  # mean rows, experts, k, N, K
    (8, 5, 4, 96, 200),          # 16 rows a tile
    (24, 5, 3, 80, 136),         # 32 rows a tile
    (25, 6, 5, 200, 264),        # 64 wide
    (150, 4, 2, 333, 203),       # 64 wide, odd rows
    (40, 64, 4, 640, 1032),      # 128 wide, all three products: 512 tiles and more
    (40, 64, 4, 645, 1031),      # the same, odd rows
    (384, 3, 3, 320, 568),       # 256 x 256 for 16 bits: several experts, several tiles of columns
    (500, 4, 5, 264, 1032),
    (500, 4, 5, 261, 1027),
]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_experts_shapes(r, dev, t, gather, shape):
    mean, E, k, N, K = SHAPES[shape]
    counts = ragged(mean, E, shape)
    ptr, M = segments(counts, 0)
    assert M == mean * E and M % k == 0
    t = TYPES[t]
    slot = shuffled_slots(M, 9)
    X = normal(1, M // k if gather else M, K, t=t)
    W, dY = normal(2, E, N, K, t=t, scale=K ** -0.5), normal(3, M, N, t=t)
    x, w, dy, p = X.to(dev), W.to(dev), dY.to(dev), ptr.to(dev)
    how = dict(slot=slot.to(dev), k=k) if gather else {}
    Y, dW = r.experts_mm(x, w, p, **how), r.experts_mm_dw(dy, x, p, **how)
    dX = None if gather else r.experts_mm_dx(dy, w, p)
    rows = X.double()[slot.long() // k] if gather else X.double()
    W, dY = W.double(), dY.double()
    for e in range(E):
        a = slice(int(ptr[e]), int(ptr[e + 1]))
        if counts[e]:
            close(Y[a], rows[a] @ W[e].t(), rows[a].abs() @ W[e].abs().t(), K, t)
            if not gather:
                close(dX[a], dY[a] @ W[e], dY[a].abs() @ W[e].abs(), N, t)
        close(dW[e], dY[a].t() @ rows[a], dY[a].abs().t() @ rows[a].abs(), counts[e], t)


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("counts", [[0, 0, 1000, 0, 0, 0, 0, 0, 0, 0] * 12, [700] + [0] * 99, [1] * 99 + [301]])
def test_experts_of_uneven_length(r, dev, t, counts):
    """One expert with nearly all rows, at means that choose the kernels for few rows."""
    t = TYPES[t]
    E, N, K = len(counts), 72, 96
    ptr, M = segments(counts)
    X, W, dY = normal(1, M, K, t=t), normal(2, E, N, K, t=t, scale=0.1), normal(3, M, N, t=t)
    x, w, dy, p = X.to(dev), W.to(dev), dY.to(dev), ptr.to(dev)
    Y, dX, dW = r.experts_mm(x, w, p), r.experts_mm_dx(dy, w, p), r.experts_mm_dw(dy, x, p).cpu()
    X, W, dY = X.double(), W.double(), dY.double()
    for e in range(E):
        a = slice(int(ptr[e]), int(ptr[e + 1]))
        if counts[e]:
            close(Y[a], X[a] @ W[e].t(), X[a].abs() @ W[e].abs().t(), K, t)
            close(dX[a], dY[a] @ W[e], dY[a].abs() @ W[e].abs(), N, t)
            close(dW[e], dY[a].t() @ X[a], dY[a].abs().t() @ X[a].abs(), counts[e], t)
        else:
            assert (dW[e] == 0).all()


# ---------------------------------------------------------------------------------------------------------------------
# The gradient of the scores
# ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("E,k", [(8, 3), (72, 6), (300, 32)])
def test_route_backward_of_masked_scores(r, dev, score, renormalise, E, k):
    """Rows with some scores, all but one and all of them -inf: their gradient is zero, and nothing is NaN."""
    T = 40
    l = normal(1, T, E, scale=1.5)
    l[torch.rand(T, E, generator=gen(2)) < 0.6] = -np.inf
    l[3], l[4] = -np.inf, -np.inf
    l[4, E // 2] = 0.25
    m = r.route(l.to(dev), k, score=score, renormalise=renormalise, scale=2.5)
    expert, dw = m.expert.cpu(), normal(3, T, k)
    assert (expert[3] == -1).all() and expert[4].tolist() == [E // 2] + [-1] * (k - 1)
    got = r.route_backward(l.to(dev), m.expert, dw.to(dev), score=score, renormalise=renormalise, scale=2.5)
    x = l.double().clamp(min=-1e4).requires_grad_()  # exp(-1e4) is zero in 64 bits too, and its derivative
    weights_of(x, expert, score, renormalise, 2.5).backward(dw.double())
    ref = x.grad
    ref[l == -np.inf] = 0.0
    close(got, ref, 2 * 2.5 * dw.double().abs().amax(1, keepdim=True).expand(T, E), 16, torch.float32)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [False, True])
def test_route_backward_against_differences_of_the_kernel(r, dev, score, renormalise):
    """The gradient along a direction against the difference of the weights that the forward kernel itself gives a step
    of h = 2^-7 to each side, where it makes the same choice.  With |v| <= 2 the third derivative of a share w of one is
    below 170 w (powers and moments of numbers that differ by at most 4: 64 + 48 + 8, and 50 for the curvature of the
    sigmoid's logarithm), and that of a sigmoid below 1; with |dw| <= 4 and shares that add up to one: 4 * 170 h^2 / 6 <
    0.007.  The weights' own 2^-19: 6 * 4 * 2^-19 / h < 0.006; the scores' rounding to 2^-22 less than 0.001."""
    T, E, k = 40, 48, 6
    l = normal(5, T, E)
    dw = normal(6, T, k).clamp(-4, 4)
    v = normal(7, T, E).clamp(-2, 2)
    h = 2.0 ** -7
    m, up, down = (r.route((l + d * v).to(dev), k, score=score, renormalise=renormalise) for d in (0.0, h, -h))
    grad = r.route_backward(l.to(dev), m.expert, dw.to(dev), score=score, renormalise=renormalise).cpu().double()
    same = ((up.expert == m.expert) & (down.expert == m.expert)).all(1).cpu()
    assert same.sum() >= T // 4
    slope = ((up.weight.cpu().double() - down.weight.cpu().double()) * dw.double()).sum(1) / (2 * h)
    assert ((grad * v.double()).sum(1) - slope)[same].abs().max() < 0.014


# ---------------------------------------------------------------------------------------------------------------------
# Captured
# ---------------------------------------------------------------------------------------------------------------------

def test_two_captured_graphs_with_workspaces(r, dev):
    """Long routings, their gradients and adapters, whose calls take workspaces, in two graphs: replayed in turn, with
    eager calls between, each gives what the eager calls give, bit for bit."""
    T, E, k, D = 3000, 40, 4, 64
    t = torch.float16
    A, B = normal(2, 3, 24, D, t=t, scale=0.125).to(dev), normal(3, 3, D, 24, t=t, scale=0.3).to(dev)
    bias = normal(4, E, scale=0.1).to(dev)
    adapter = (torch.arange(T, dtype=torch.int32, device=dev) % 4).view(T, 1)
    options = dict(score="sigmoid", renormalise=True)

    def layer(x, scores):
        m = r.route(scores, k, bias=bias, groups=4, top_groups=2, group_score="top2", **options)
        z = x[m.slot.long() // k]
        g = r.combine_backward(x, z, m.weight, m.expert_ptr, m.slot)
        ds = r.route_backward(scores, m.expert, g["dweight"], **options)
        ptr, row, _ = r.columns(adapter, 3)
        return r.adapters_mm(x, A, B, None, ptr, row, base=r.combine(z, m.pos, m.weight)), ds, g["dZ"], *m

    def masked(seed):
        return torch.from_numpy(masked_groups(seed, T, E, 4))

    inputs = [(torch.zeros(T, D, dtype=t, device=dev), torch.zeros(T, E, device=dev)) for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in inputs:
            layer(*a)
    torch.cuda.current_stream().wait_stream(side)
    graphs, captured = [torch.cuda.CUDAGraph() for _ in inputs], []
    for graph, a in zip(graphs, inputs):
        with torch.cuda.graph(graph):
            captured.append(layer(*a))
    for n in range(3):
        for i, a in enumerate(inputs):
            a[0].copy_(normal(10 * n + i, T, D, t=t))
            a[1].copy_(masked(10 * n + i))
        for graph in graphs:
            graph.replay()
        for graph, got, a in zip(graphs, captured, inputs):
            ref = layer(*a)
            torch.cuda.synchronize()
            for x, y in zip(got, ref):
                assert torch.equal(x, y)
