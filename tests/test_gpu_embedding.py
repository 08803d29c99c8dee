"""Embedding lookup with scaling and its sorted gradient against 64-bit indexing.

Tolerances, u = 2^-24 (half a step of fp32) and h = eps / 2 of the tensors' type:
  lookup    the factor and the product round in fp32, the result once more: |ref| (2 u + h)
  gradient  k terms summed in fp32 in any order: at most k u times the sum of their magnitudes; the factor, the
            product and the last rounding as above.
Second-order terms are covered by a factor of 1.01."""
import math

import pytest
import torch

from recommend_amd import _ffi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
TYPES = (torch.float32, torch.bfloat16, torch.float16)


def half(t):
    return torch.finfo(t).eps / 2 if t != torch.float32 else 0.0


def ids_of(kind, rows, n, g):
    if kind == "uniform":
        return torch.randint(rows, (n,), generator=g)
    if kind == "same":
        return torch.full((n,), rows - 1)
    if kind == "runs":                                   # runs of all lengths, in the order of their ids
        return (torch.arange(n) // 37).clamp_max(rows - 1)
    return (rows * torch.rand(n, generator=g) ** 4).long().clamp_max(rows - 1)   # skewed


def reference(weight, ids, grad, scale, pad):
    w, g = weight.double(), grad.double()
    valid = (ids >= 0) & (ids < w.shape[0])
    safe = torch.where(valid, ids, torch.zeros_like(ids))
    out = w[safe] * scale
    keep = valid & (ids != pad) if pad is not None else valid
    g = torch.where(keep.unsqueeze(1), g, torch.zeros_like(g))
    dw = torch.zeros_like(w).index_add_(0, safe, g) * scale
    mag = torch.zeros_like(w).index_add_(0, safe, g.abs()) * abs(scale)
    count = torch.zeros(w.shape[0], dtype=torch.float64).index_add_(0, safe, keep.double())
    return out, valid, dw, mag, count


def check(weight, ids, grad, scale, pad, out, dw):
    t = weight.dtype
    want, valid, wd, mag, count = reference(weight.cpu(), ids.cpu().long(), grad.cpu(), scale, pad)
    got = out.cpu().double()
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps if t == torch.float16 else 0.0
    assert bool(torch.isnan(got[~valid]).all())
    assert bool(((got - want).abs() <= (want.abs() * (2 * U + half(t)) * 1.01 + tiny))[valid].all())
    err = (dw.cpu().double() - wd).abs()
    tol = (mag * U * count.unsqueeze(1) + wd.abs() * (2 * U + half(t))) * 1.01 + tiny
    assert bool((err <= tol).all()), float((err - tol).max())
    assert bool((dw.cpu()[count == 0] == 0).all())


def run(weight, ids, grad, scale, pad):
    w = weight.detach().requires_grad_(True)
    out = ops.embedding_lookup(w, ids, scale=scale, padding_idx=pad)
    return out, torch.autograd.grad(out, w, grad)[0]


CASES = [
    # rows, D, n, ids
    (1, 1, 1, "same"), (5, 3, 1, "uniform"), (3, 8, 7, "uniform"), (9, 7, 200, "skewed"), (300, 64, 0, "uniform"),
    (7, 1, 3000, "uniform"), (1000, 64, 512, "uniform"), (1000, 64, 4096, "skewed"), (1000, 64, 4097, "skewed"),
    (400, 100, 6000, "runs"), (500, 33, 20000, "same"), (26495, 128, 3200, "skewed"), (300, 256, 9000, "skewed"),
    (70000, 16, 50000, "skewed"), (300000, 10, 30000, "uniform"), (200, 2056, 700, "skewed"), (2, 1030, 5000, "uniform"),
    (511, 65, 10000, "uniform"), (40, 64, 512, "same"), (40, 64, 511, "runs"), (7050, 33, 513, "skewed"), (3, 300, 400, "uniform"), (9000000, 3, 300, "uniform"), (512, 64, 100000, "runs"), (4, 64, 200000, "uniform"),
    (40, 1025, 9000, "runs"), (3, 1029, 4000, "same"), (2500001, 2, 9000, "uniform"),
    (2100000, 5, 700, "skewed"),
]


@pytest.mark.parametrize("rows,D,n,kind", CASES)
@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_and_gradient_vs_float64(rows, D, n, kind, dtype):
    g = torch.Generator().manual_seed(rows + D + n)
    ids = ids_of(kind, rows, n, g).to(torch.int32 if (rows + n) % 2 else torch.int64).to(DEV)
    weight = torch.randn(rows, D, generator=g).to(dtype).to(DEV)
    grad = torch.randn(n, D, generator=g).to(dtype).to(DEV)
    scale, pad = math.sqrt(D), (rows - 1 if n % 3 == 2 else None)
    out, dw = run(weight, ids, grad, scale, pad)
    check(weight, ids, grad, scale, pad, out, dw)
    out2, dw2 = run(weight, ids, grad, scale, pad)
    assert torch.equal(dw, dw2)                          # the same bits on every run
    if pad is not None:
        assert bool((dw[pad] == 0).all())


def test_ids_of_any_shape_and_padding_from_the_end():
    g = torch.Generator().manual_seed(1)
    weight = torch.randn(50, 24, generator=g).to(DEV).requires_grad_(True)
    ids = torch.randint(50, (4, 3, 5), generator=g).to(DEV)
    ids[0] = 49
    out = ops.embedding_lookup(weight, ids, padding_idx=-1)
    assert out.shape == (4, 3, 5, 24) and torch.equal(out, weight.detach()[ids])
    out.backward(torch.ones_like(out))
    count = torch.bincount(ids.flatten(), minlength=50).float()
    count[49] = 0
    assert torch.equal(weight.grad, count.unsqueeze(1).expand(50, 24))
    assert ops.embedding_lookup(weight.detach(), ids[0, 0, 0]).shape == (24,)     # a single id


def test_ids_outside_the_table_read_nothing_and_add_nothing():
    weight = torch.ones(10, 16, device=DEV, requires_grad=True)
    for dtype, bad in ((torch.int64, [-1, 10, 1 << 31, (1 << 32) + 3, -(1 << 40)]), (torch.int32, [-1, 10, 2 ** 31 - 1, -2 ** 31])):
        ids = torch.tensor([3] + bad + [3], dtype=dtype, device=DEV)
        out, dw = run(weight, ids, torch.ones(len(ids), 16, device=DEV), 2.0, None)
        assert bool((out[[0, -1]] == 2).all()) and bool(torch.isnan(out[1:-1]).all())
        want = torch.zeros(10, 16, device=DEV)
        want[3] = 4
        assert torch.equal(dw, want)


def test_gradients_of_padded_places_do_not_leak():
    ids = torch.tensor([0, 1, 0, 2], device=DEV)
    grad = torch.ones(4, 64, device=DEV)
    grad[0], grad[2] = float("nan"), float("inf")
    _, dw = run(torch.ones(3, 64, device=DEV), ids, grad, 1.0, 0)
    assert bool((dw[0] == 0).all()) and bool((dw[1:] == 1).all())
    _, dw = run(torch.ones(3, 64, device=DEV), ids, grad, 1.0, None)              # not padded: they count
    assert bool(torch.isnan(dw[0]).all()) and bool((dw[1:] == 1).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_views_of_tables_and_gradients(dtype):
    """Rows with other rows' data between them, a base that is aligned to one element only, expanded and
    transposed gradients."""
    g = torch.Generator().manual_seed(2)
    big = torch.randn(40, 101, generator=g).to(dtype).to(DEV)
    ids = torch.randint(40, (300,), generator=g).to(DEV)
    for view in (big[:, 3:36], big[:, 1:65], big.t()[:40, :20], big[:1].expand(40, 101)):
        D = view.shape[1]
        grads = [torch.randn(1, D, generator=g).to(dtype).to(DEV).expand(300, D),
                 torch.randn(D, 300, generator=g).to(dtype).to(DEV).t(), torch.randn(601, D, generator=g).to(dtype).to(DEV)[1::2]]
        for grad in grads:
            w = view.detach().requires_grad_(True)
            out = ops.embedding_lookup(w, ids, scale=0.5)
            dw, = torch.autograd.grad(out, w, grad)
            check(view, ids, grad, 0.5, None, out, dw)


def test_saved_ids_that_were_kept_on_the_host():
    w = torch.randn(50, 8, device=DEV, requires_grad=True)
    ids = torch.randint(50, (6, 7), device=DEV)
    want, = torch.autograd.grad(ops.embedding_lookup(w, ids).square().sum(), w)
    with torch.autograd.graph.save_on_cpu():
        loss = ops.embedding_lookup(w, ids).square().sum()
    assert torch.equal(torch.autograd.grad(loss, w)[0], want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:2]):
        out = ops.embedding_lookup(w, ids)
    with pytest.raises(RuntimeError, match="not those of the forward pass"):
        out.sum().backward()


def test_a_table_of_one_row_with_any_stride():
    w = torch.randn(8, device=DEV)
    one = torch.as_strided(w, (1, 8), (0, 1))
    assert torch.equal(ops.embedding_lookup(one, torch.zeros(3, dtype=torch.long, device=DEV)), w.expand(3, 8))


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(3)
    weight = torch.randn(30, 20, generator=g).to(DEV)
    ids, probe = torch.randint(30, (90,), generator=g).to(DEV), torch.randn(90, 20, generator=g).to(DEV)
    step = torch.randn(30, 20, generator=g).to(DEV)
    _, dw = run(weight, ids, probe, 3.0, None)
    f = lambda w: (ops.embedding_lookup(w, ids, scale=3.0).double() * probe.double()).sum()  # noqa: E731
    # linear in the table: the difference is exact up to the rounding of the 1800 looked-up values (3 u of
    # values up to 15 times probes up to 4) and of the gradient's 600 products
    change = float(f(weight + step) - f(weight - step)) / 2
    slope = float((dw.double() * step.double()).sum())
    assert abs(change - slope) <= 1800 * 3 * U * 15 * 4 + 600 * 90 * U * 12


def test_two_lookups_share_a_table_and_no_grad_needs_no_graph():
    weight = torch.randn(20, 64, device=DEV, requires_grad=True)
    a, b = torch.tensor([1, 2, 2], device=DEV), torch.tensor([2, 3], device=DEV)
    (ops.embedding_lookup(weight, a).sum() + 2 * ops.embedding_lookup(weight, b).sum()).backward()
    want = torch.zeros(20, device=DEV)
    want[[1, 2, 3]] = torch.tensor([1.0, 4.0, 2.0], device=DEV)
    assert torch.equal(weight.grad, want.unsqueeze(1).expand(20, 64))
    with torch.no_grad():
        assert ops.embedding_lookup(weight, a).grad_fn is None
    assert ops.embedding_lookup(torch.empty(0, 4, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV)).shape == (0, 4)
    with pytest.raises(ValueError, match="several devices|HIP device") if torch.cuda.device_count() > 1 else pytest.raises(_ffi.RkError):
        ops.embedding_lookup(weight, a.cpu())


@pytest.mark.parametrize("n", [700, 9000])
def test_recorded_in_a_graph_and_replayed(n):
    g = torch.Generator().manual_seed(4)
    weight = torch.randn(3000, 64, generator=g).to(DEV).requires_grad_(True)
    ids, grad = torch.zeros(n, dtype=torch.int64, device=DEV), torch.zeros(n, 64, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run(weight, ids, grad, 1.5, 0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, dw = run(weight, ids, grad, 1.5, 0)
    for _ in range(4):
        ids.copy_(torch.randint(3000, (n,), generator=g))
        grad.copy_(torch.randn(n, 64, generator=g))
        graph.replay()
        eager = run(weight, ids.clone(), grad.clone(), 1.5, 0)
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(dw, eager[1])
