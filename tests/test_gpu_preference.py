"""Log-probabilities of item lists and the preference loss against 64 bits.

Tolerances, u = 2^-24: a row's maximum is exact; exp(x - max) has the rounding of the difference and of the factor
log2 e (2 u |x - max| relative, weighted by exp(x - max) itself: at most 0.74 u in the sum) and 4 u of the
instruction; a thread adds k = V / 256 + 32 terms one after the other and 8 pairs are merged, each with another
exponential: the sum is off by (k + 64) u relative.  So
  row = (k + 64) u + 2 u (|x_y - max| + |log sum|),      list = sum of its rows + u |logp|
  dx  = |dx| (2 u |log p| + 2 row + 16 u + h) + p |dc|,  |dc| <= beta^2 list / P + 16 u |c|  (sigmoid and squared:
        2 list / P; hinge: 0 away from its corner), h = eps / 2 of the tensors' type."""
import pytest
import torch

from recommend_amd.loss import list_logps, preference_loss

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else U


def plain(scores, items, average):
    """(logps, their tolerance, d logps[s] / d scores as a function of upstream weights) in 64 bits."""
    x = scores.detach().cpu().double()
    used = items.cpu() != -100
    y = torch.where(used, items.cpu(), torch.zeros_like(items.cpu())).long().unsqueeze(-1)
    lse = torch.logsumexp(x, -1, keepdim=True)
    logp = (x.gather(-1, y) - lse).squeeze(-1)
    top = x.amax(-1)
    k = x.shape[-1] / 256 + 32
    row = (k + 64) * U + 2 * U * ((x.gather(-1, y).squeeze(-1) - top).abs() + (lse.squeeze(-1) - top).abs())
    zero = torch.zeros_like(logp)
    n = used.sum(-1).clamp_min(1) if average else torch.ones(x.shape[0])
    logps = torch.where(used, logp, zero).sum(-1) / n
    tol = torch.where(used, row, zero).sum(-1) / n + U * logps.abs() * 2
    p = torch.exp(x - lse)

    def grad(c, dc):
        c, dc = (c / n).view(-1, 1, 1), (dc / n).view(-1, 1, 1)
        one = torch.zeros_like(x).scatter_(-1, y, 1.0)
        on = used.unsqueeze(-1)
        d = torch.where(on, c * (one - p), torch.zeros_like(x))
        # at the item itself c and c p are rounded before they are subtracted
        size = c.abs() * (one + p)
        slack = size * (2 * U * torch.where(p > 0, -torch.log(p), torch.zeros_like(p)) + 2 * row.unsqueeze(-1) + 16 * U)
        slack = slack + d.abs() * half(scores.dtype) + (one + p) * dc.abs()
        if scores.dtype == torch.float16:
            slack = slack + 2.0 ** -25
        return d, torch.where(on, slack, torch.zeros_like(x)) * 1.01 + 1e-37

    return logps, tol * 1.01, grad


def pair_loss(logps, ref, beta, eps, kind):
    P = logps.shape[0] // 2
    d = (logps - ref)[:P] - (logps - ref)[P:]
    if kind == "sigmoid":
        f = torch.nn.functional.logsigmoid
        return -((1 - eps) * f(beta * d) + eps * f(-beta * d)).mean()
    if kind == "hinge":
        return (1 - beta * d).clamp_min(0).mean()
    return ((d - 1 / (2 * beta)) ** 2).mean()


def make(S, T, V, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    scores = (spread * torch.randn(S, T, V, generator=g)).to(dtype).to(DEV)
    items = torch.randint(V, (S, T), generator=g)
    items[torch.rand(S, T, generator=g) < 0.3] = -100
    if S > 1:
        items[1] = -100                                  # a list without any place in use
    ref = -4.0 * T + torch.randn(S, generator=g)
    return scores.requires_grad_(True), items.to(DEV), ref.to(DEV)


SHAPES = [(2, 1, 1), (2, 1, 2), (4, 3, 7), (6, 2, 63), (2, 70, 65), (4, 5, 1000), (2, 2, 4097), (8, 3, 7050), (2, 1, 63001),
          (2, 300, 129), (34, 1, 515), (6, 3, 1024), (6, 3, 1025), (6, 3, 2047), (6, 3, 2049)]


@pytest.mark.parametrize("S,T,V", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("average", [False, True])
def test_list_logps_vs_float64(S, T, V, dtype, average):
    scores, items, _ = make(S, T, V, dtype, S + T + V)
    logps = list_logps(scores, items, average=average)
    want, tol, grad = plain(scores, items, average)
    assert bool(((logps.detach().cpu().double() - want).abs() <= tol).all())
    assert float(logps.detach()[1]) == 0.0
    g = torch.randn(S, generator=torch.Generator().manual_seed(1))
    dx, = torch.autograd.grad(logps, scores, g.to(DEV))
    wd, slack = grad(g.double(), torch.zeros(S).double())
    err = (dx.cpu().double() - wd).abs()
    assert bool((err <= slack).all()), float((err - slack).max())
    assert torch.equal(logps, list_logps(scores, items, average=average))


@pytest.mark.parametrize("kind,eps", [("sigmoid", 0.0), ("sigmoid", 0.2), ("sigmoid", 1.0), ("hinge", 0.0), ("squared", 0.0)])
@pytest.mark.parametrize("S,T,V,dtype", [(2, 1, 33, torch.float32), (6, 4, 1001, torch.float32), (6, 4, 1001, torch.bfloat16),
                                         (40, 2, 300, torch.float16), (4, 3, 18357, torch.bfloat16)])
def test_preference_loss_vs_float64(kind, eps, S, T, V, dtype):
    scores, items, ref = make(S, T, V, dtype, S * T)
    beta = 0.3
    loss, logps = preference_loss(scores, items, ref, beta=beta, label_smoothing=eps, kind=kind)
    want, tol, grad = plain(scores, items, False)
    leaf = want.clone().requires_grad_(True)
    wl = pair_loss(leaf, ref.cpu().double(), beta, eps, kind)
    c, = torch.autograd.grad(wl, leaf)
    P = S // 2
    sum_tol = tol + 4 * U * (want.abs() + ref.cpu().double().abs())
    pair_tol = sum_tol[:P] + sum_tol[P:]
    assert bool(((logps.detach().cpu().double() - want).abs() <= tol).all())
    steep = {"sigmoid": beta, "hinge": beta}.get(kind)
    d = (want - ref.cpu().double())[:P] - (want - ref.cpu().double())[P:]
    slope = torch.full_like(d, steep) if steep else 2 * (d - 0.5 / beta).abs()
    loss_tol = float((slope * pair_tol).mean().detach()) + 32 * U * (abs(float(wl.detach())) + 1)
    assert abs(float(loss.detach()) - float(wl.detach())) <= loss_tol
    bend = {"sigmoid": beta ** 2, "hinge": 0.0, "squared": 2.0}[kind]
    dc = (bend * pair_tol / P).repeat(2) + 16 * U * c.abs()
    dx, = torch.autograd.grad(loss, scores)
    wd, slack = grad(c, dc)
    err = (dx.cpu().double() - wd).abs()
    assert bool((err <= slack).all()), float((err - slack).max())


# more rows than one workgroup joins, up to and above the pairs that one adds up
@pytest.mark.parametrize("kind,eps", [("sigmoid", 0.1), ("squared", 0.0)])
@pytest.mark.parametrize("S,T,V,dtype", [(8192, 1, 5, torch.float32), (8194, 1, 5, torch.float16), (10002, 1, 41, torch.float32),
                                         (16500, 3, 18, torch.bfloat16), (1000, 5, 30, torch.float32),
                                         (66, 70, 33, torch.float32), (4, 1500, 20, torch.float32),
                                         (10, 513, 9, torch.bfloat16), (2, 1, 70001, torch.bfloat16),
                                         (130, 1, 40000, torch.float32), (260, 4, 9001, torch.float32)])
def test_many_lists_vs_float64(kind, eps, S, T, V, dtype):
    test_preference_loss_vs_float64(kind, eps, S, T, V, dtype)


def test_both_results_are_differentiable():
    """loss + a term on the preferred lists' own log-probabilities: the gradients add."""
    scores, items, ref = make(4, 3, 200, torch.float32, 9)
    loss, logps = preference_loss(scores, items, ref)
    both, = torch.autograd.grad(loss - 0.5 * logps[:2].sum(), scores, retain_graph=True)
    one, = torch.autograd.grad(loss, scores, retain_graph=True)
    two, = torch.autograd.grad(-0.5 * logps[:2].sum(), scores)
    # c = c1 + c2 in one pass against two passes added: a few roundings of each
    assert bool(((both - one - two).abs() <= 8 * U * (one.abs() + two.abs() + both.abs()) + 1e-30).all())


def test_gradient_against_differences():
    scores, items, ref = make(4, 2, 50, torch.float32, 5)
    dx, = torch.autograd.grad(preference_loss(scores, items, ref, beta=0.5, label_smoothing=0.1)[0], scores)
    g = torch.Generator().manual_seed(6)
    step = torch.randn(scores.shape, generator=g).double()
    f = lambda e: pair_loss(plain(scores.detach().cpu().double() + e * step, items, False)[0], ref.cpu().double(), 0.5, 0.1, "sigmoid")  # noqa: E731,E501
    # central difference of the formula in 64 bits (error e^2 / 6 times a third derivative of order |step|^3) against the
    # kernel's gradient along the same direction
    change = float(f(1e-4) - f(-1e-4)) / 2e-4
    slope = float((dx.cpu().double() * step).sum())
    assert abs(change - slope) <= 1e-8 * float(step.abs().sum()) + float((dx.cpu().double() * step).abs().sum()) * 200 * U


def test_masked_scores_and_places():
    """-inf and the type's lowest value among the scores, NaN in places that are not in use, a row of -inf only."""
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        x = torch.zeros(4, 2, 6, dtype=dtype, device=DEV)
        x[:, :, 3] = float("-inf")
        x[:, :, 4] = low
        items = torch.tensor([[0, -100], [3, 0], [4, 0], [-100, 1]], device=DEV)
        x[0, 1] = float("nan")
        x[3, 0] = float("-inf")
        x.requires_grad_(True)
        logps = list_logps(x, items)
        got = logps.detach().cpu().double()
        want = -torch.log(torch.tensor(4.0, dtype=torch.float64))     # four scores of zero count
        assert abs(got[0] - want) <= 100 * U and abs(got[3] - want) <= 100 * U
        assert got[1] == float("-inf") and abs(got[2] - (low + 2 * want)) <= abs(low) * U
        dx, = torch.autograd.grad(logps.sum(), x)
        assert bool((dx[0, 1] == 0).all()) and bool((dx[3, 0] == 0).all())
        assert bool(torch.isfinite(dx).all()) and bool((dx[:, :, 3][items != 3] == 0).all())
        assert float(dx[1, 0, 3]) == 1.0                              # the item itself has no probability: 1 - 0
        bad = x.detach().clone()
        bad[0, 0] = float("-inf")                                     # no score left: no distribution
        assert bool(torch.isnan(list_logps(bad, items)[0]))
        bad[0, 0, 0] = float("inf")
        assert bool(torch.isnan(list_logps(bad, items)[0]))
        bad[0, 0], bad[0, 0, 2] = 0, float("nan")
        assert torch.isnan(list_logps(bad, items)).tolist() == [True, False, False, False]
        all_low = torch.full((2, 1, 500), low, dtype=dtype, device=DEV)
        got = list_logps(all_low, torch.tensor([[3], [499]], device=DEV))
        assert bool(((got.cpu().double() + torch.log(torch.tensor(500.0).double())).abs() <= 200 * U).all())


def test_items_outside_the_catalogue_make_their_list_nan():
    x = torch.zeros(4, 2, 10, device=DEV, requires_grad=True)
    items = torch.tensor([[0, 10], [1, 2], [-1, 3], [1 << 40, 2]], device=DEV)
    logps = list_logps(x, items)
    assert torch.isnan(logps).tolist() == [True, False, True, True]
    dx, = torch.autograd.grad(logps[1], x)
    assert bool(torch.isfinite(dx[1]).all())
    assert bool(torch.isnan(preference_loss(x, items, torch.zeros(4, device=DEV))[0]))


def test_extreme_ratios():
    """Ratios far from zero: the loss grows linearly on one side and vanishes on the other, without overflow."""
    x = torch.zeros(4, 1, 2, device=DEV)
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 1], x[3, 0, 0] = 8e4, 8e4, 8e4, 8e4
    x.requires_grad_(True)
    items = torch.zeros(4, 1, dtype=torch.int64, device=DEV)
    loss, logps = preference_loss(x, items, torch.zeros(4, device=DEV), beta=1.0)
    assert logps.tolist() == [0.0, -8e4, -8e4, 0.0]
    assert float(loss.detach()) == 4e4                                         # pairs (0, 2): 0, (1, 3): 8e4
    dx, = torch.autograd.grad(loss, x)
    assert bool(torch.isfinite(dx).all()) and float(dx[1, 0, 0]) == -0.5 and float(dx[0].abs().max()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_scores(dtype):
    """All places but the last of a longer tensor, every second list, rows that begin at odd addresses, scores whose
    rows are not contiguous, one row expanded over the lists: the values of a contiguous copy."""
    g = torch.Generator().manual_seed(8)
    big = (2 * torch.randn(8, 6, 301, generator=g)).to(dtype).to(DEV)
    items = torch.randint(300, (4, 5), generator=g).to(DEV)
    ref = torch.zeros(4, device=DEV)
    for view in (big[:4, :-1], big[::2, 1:], big[4:, 1:, 1:], big[:4, :5, ::2], big[:1, :5].expand(4, 5, 301)):
        it = items.clamp_max(view.shape[2] - 1)
        a, b = view.detach().requires_grad_(True), view.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        la, pa = preference_loss(a, it, ref)
        lb, pb = preference_loss(b, it, ref)
        assert torch.equal(la, lb) and torch.equal(pa, pb)
        assert torch.equal(*(torch.autograd.grad(l, s)[0].contiguous() for l, s in ((la, a), (lb, b))))
    wide = items.repeat(1, 2)[:, ::2]                                  # strided and 32-bit items
    assert torch.equal(list_logps(big[:4, :5], wide), list_logps(big[:4, :5], wide.to(torch.int32)))


def test_saved_tensors_that_were_kept_on_the_host():
    """They come back with other strides than they had."""
    g = torch.Generator().manual_seed(18)
    big = torch.randn(8, 6, 301, generator=g).to(DEV)
    items, ref = torch.randint(300, (4, 5), generator=g).to(DEV), torch.zeros(4, device=DEV)
    for view in (big[::2, 1:, 1:], big[:1, :5].expand(4, 5, 301), big[:4, :5, ::2]):
        it = items.clamp_max(view.shape[2] - 1)
        a = view.detach().requires_grad_(True)
        want, = torch.autograd.grad(preference_loss(a, it, ref)[0], a)
        with torch.autograd.graph.save_on_cpu():
            loss, _ = preference_loss(a, it, ref)
        got, = torch.autograd.grad(loss, a)
        assert torch.equal(got, want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:2]):
        loss, _ = preference_loss(a, it, ref)
    with pytest.raises(RuntimeError, match="not those of the forward pass"):
        loss.backward()


def test_lists_of_one_item_without_a_place_axis():
    g = torch.Generator().manual_seed(10)
    x = torch.randn(6, 40, generator=g).to(DEV).requires_grad_(True)
    items, ref = torch.randint(40, (6,), generator=g).to(DEV), torch.zeros(6, device=DEV)
    loss, logps = preference_loss(x, items, ref)
    same, _ = preference_loss(x.unsqueeze(1), items.unsqueeze(1), ref)
    assert torch.equal(loss, same)
    dx, = torch.autograd.grad(loss, x)
    assert dx.shape == x.shape and bool((dx != 0).any())
    assert list_logps(x[:0], items[:0]).shape == (0,)


def test_against_bpr_on_single_scores():
    """One place and the same scores for both lists of a pair: the normaliser cancels and the loss is BPR's."""
    g = torch.Generator().manual_seed(11)
    row = torch.randn(5, 100, generator=g).to(DEV)
    pos, neg = torch.randint(100, (2, 5), generator=g).to(DEV)
    loss, _ = preference_loss(torch.cat([row, row]), torch.cat([pos, neg]), torch.zeros(10, device=DEV), beta=1.0)
    from recommend_amd.loss import bpr_loss
    want = bpr_loss(row.gather(1, pos.view(-1, 1)).squeeze(1), row.gather(1, neg.view(-1, 1)))
    assert abs(float(loss) - float(want)) <= 200 * U * (1 + abs(float(want)))


def test_recorded_in_a_graph_and_replayed_beside_eager_work():
    g = torch.Generator().manual_seed(12)
    scores = torch.zeros(8, 3, 5000, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    items, ref = torch.zeros(8, 3, dtype=torch.int64, device=DEV), torch.zeros(8, device=DEV)

    def step():
        loss, logps = preference_loss(scores, items, ref)
        dx, = torch.autograd.grad(loss, scores)
        return loss.detach(), logps.detach(), dx

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        recorded = step()
    for _ in range(4):
        with torch.no_grad():
            scores.copy_(torch.randn(8, 3, 5000, generator=g))
        items.copy_(torch.randint(5000, (8, 3), generator=g))
        items[2, 1] = -100
        ref.copy_(torch.randn(8, generator=g))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(recorded, eager))
