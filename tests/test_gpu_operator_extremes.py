"""The embedding, list and AdamW operators at the far ends of what they accept, and in the calls that programs make
around them: other streams and threads, repeated backward passes, transforms of torch.func."""
import threading

import pytest
import torch

from recommend_amd import _ffi, ops
from recommend_amd.loss import list_logps, preference_loss
from recommend_amd.optim import FusedAdamW, FusedClipAdam
from recommend_amd.train_step import GraphedTrainStep

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype,D", [(torch.float32, (1 << 27) + 5), (torch.bfloat16, (1 << 28) + 9)])
@pytest.mark.parametrize("n", [0, 1])
def test_rows_whose_vectors_pass_32_bits(dtype, D, n):
    """64 rows of more than 2^25 vectors of 16 bytes have more than 2^31 of them.  Rows without an id are zeros, in memory
    that held something else; factors of two round nothing."""
    ids = torch.ones(n, dtype=torch.int64, device=DEV)
    table = torch.empty(3, D, dtype=dtype, device=DEV)
    table[0], table[1], table[2] = 3.0, 1.5, 5.0
    table[1, 7::11] = -0.25
    table.requires_grad_(True)
    out = ops.embedding_lookup(table, ids, scale=2.0)
    grad = torch.full((n, D), 0.5, dtype=dtype, device=DEV)
    grad[:, ::13] = -4.0
    for i in range(n):
        assert torch.equal(out[i], 2 * table.detach()[1])
    torch.full((3, D), float("nan"), dtype=dtype, device=DEV)          # (the next tensor of this size gets its memory)
    dw, = torch.autograd.grad(out, table, grad)
    assert bool((dw[0] == 0).all()) and bool((dw[2] == 0).all())
    assert torch.equal(dw[1], 2 * grad[0] if n else torch.zeros_like(dw[1]))


@pytest.mark.parametrize("make", [lambda p: FusedAdamW(p, lr=1e-2, max_grad_norm=1.0, state_bits=8),
                                  lambda p: FusedAdamW(p, lr=1e-2, max_grad_norm=1.0),
                                  lambda p: FusedClipAdam(p, lr=1e-2, max_grad_norm=1.0)], ids=["8", "32", "clip"])
def test_recorded_step_goes_on_after_a_checkpoint_without_its_moments(make):
    """A step is recorded, then the checkpoint from before the first step is loaded: replays do what a new optimizer
    does, and touch nothing that was allocated since."""
    g = torch.Generator().manual_seed(5)
    start = [torch.randn(s, generator=g).to(DEV) for s in ((100, 64), (64,))]
    ours = [torch.nn.Parameter(w.clone()) for w in start]
    opt = make(ours)
    saved = opt.state_dict()
    for p in ours:
        p.grad = torch.randn(p.shape, generator=g).to(DEV)
    for _ in range(2):
        opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    opt.load_state_dict(saved)
    with torch.no_grad():
        for p, w in zip(ours, start):
            p.copy_(w)
    # every size that a moment or a workspace has had: freed ones would be given out here
    others = [torch.full((n,), 7, dtype=torch.uint8, device=DEV) for n in (6400, 25600, 400, 256, 32) for _ in range(20)]
    fresh = [torch.nn.Parameter(w.clone()) for w in start]
    same = make(fresh)
    for k in range(4):
        for p, q in zip(ours, fresh):
            p.grad.copy_(torch.randn(p.shape, generator=g))
            q.grad = p.grad.clone()
        if k < 3:
            graph.replay()
        else:
            opt.step()
        same.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ours, fresh)) and int(opt.step_count) == int(same.step_count) == k + 1
    assert all(bool((o == 7).all()) for o in others)
    for p, q in zip(ours, fresh):
        assert all(torch.equal(v.view(torch.uint8), same.state[q][k].view(torch.uint8)) for k, v in opt.state[p].items())


def test_recorded_training_step_clips_to_the_norm_that_the_optimizer_was_given():
    g = torch.Generator().manual_seed(6)
    model = torch.nn.Linear(8, 1, bias=False).to(DEV)
    batch = {"x": torch.randn(32, 8, generator=g).to(DEV)}
    twin = torch.nn.Parameter(model.weight.detach().clone())
    opt, same = FusedAdamW(model.parameters(), lr=0.1, max_grad_norm=0.25), FusedAdamW([twin], lr=0.1, max_grad_norm=0.25)
    net = torch.nn.Module()
    net.weight = model.weight
    net.forward = lambda b: b["x"] * net.weight
    step = GraphedTrainStep(net, opt, lambda out, b: 50 * out.square().mean(), batch, warmup_steps=1)
    step(batch)
    for _ in range(2):
        twin.grad, = torch.autograd.grad(50 * (batch["x"] * twin).square().mean(), twin)
        same.step()
    torch.cuda.synchronize()
    assert opt.max_grad_norm == 0.25 and float(opt.grad_norm) > 0.25
    assert torch.equal(model.weight, twin) and torch.equal(opt.state[model.weight]["exp_avg"], same.state[twin]["exp_avg"])


def test_a_late_parameter_is_corrected_with_the_common_count():
    """20 steps without it, then its first gradient: m = 0.1 g, v = 0.001 g^2, corrected with count 21.  The update rounds
    a dozen times (16 u) and the parameter once."""
    a, late = (torch.nn.Parameter(torch.ones(70, device=DEV)) for _ in range(2))
    opt = FusedAdamW([a, late], lr=1e-2, weight_decay=0.0, eps=0.0)
    for _ in range(20):
        a.grad = torch.ones_like(a)
        opt.step()
    late.grad = torch.full_like(late, 3.0)
    opt.step()
    move = 1e-2 / (1 - 0.9 ** 21) * 0.1 / (0.001 / (1 - 0.999 ** 21)) ** 0.5
    assert int(opt.step_count) == 21
    assert float((late.detach().double() - (1 - move)).abs().max()) <= (16 * move + 1) * 2.0 ** -24


def inputs(seed, n=700, rows=900):
    """Of a lookup with gradient (counting sort) and of a preference step."""
    g = torch.Generator().manual_seed(seed)
    table, grad = torch.randn(rows, 64, generator=g).to(DEV), torch.randn(n, 64, generator=g).to(DEV)
    scores = torch.randn(8, 3, 5000, generator=g).to(DEV)
    items, ref = torch.randint(5000, (8, 3), generator=g).to(DEV), torch.randn(8, generator=g).to(DEV)
    return table, torch.randint(rows, (n,), generator=g).to(DEV), grad, scores, items, ref


def both(table, ids, grad, scores, items, ref):
    table, scores = table.requires_grad_(True), scores.requires_grad_(True)
    out = ops.embedding_lookup(table, ids, scale=1.5, padding_idx=0)
    loss, logps = preference_loss(scores, items, ref)
    return [out.detach(), torch.autograd.grad(out, table, grad)[0], loss.detach(), logps.detach(), torch.autograd.grad(loss, scores)[0]]


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_second_backward_pass_with_the_graph_retained():
    table, ids, grad, scores, items, ref = inputs(1)
    want = both(table, ids, grad, scores, items, ref)
    out, (loss, _) = ops.embedding_lookup(table, ids, scale=1.5, padding_idx=0), preference_loss(scores, items, ref)
    for _ in range(2):
        assert torch.equal(torch.autograd.grad(out, table, grad, retain_graph=True)[0], want[1])
        assert torch.equal(torch.autograd.grad(loss, scores, retain_graph=True)[0], want[4])
    for y, x, g in ((out, table, grad), (loss, scores, None)):
        torch.autograd.grad(y, x, g)
        with pytest.raises(RuntimeError, match="second time|freed"):
            torch.autograd.grad(y, x, g)


def test_inputs_changed_between_the_passes_are_refused():
    table, ids, grad, scores, items, ref = inputs(2)
    out, (loss, _) = (ops.embedding_lookup(table.requires_grad_(True), ids),
                      preference_loss(scores.requires_grad_(True), items, ref))
    ids.add_(0)
    items.add_(0)
    for y, x, g in ((out, table, grad), (loss, scores, None)):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, x, g)


def test_on_another_stream_than_the_default_one():
    """Forward and backward on a side stream behind slow work, without a wait by the host."""
    args = inputs(3)
    want = both(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        slow = torch.randn(4096, 4096, device=DEV)
        late = [torch.zeros_like(a) for a in args]
        for _ in range(20):
            slow = slow @ slow / 64
        for a, b in zip(late, args):
            with torch.no_grad():
                a.copy_(b)
        got = both(*[a.detach() for a in late])
        p, q = (torch.nn.Parameter(args[0].detach().clone()) for _ in range(2))
        p.grad = late[2][:1].expand(900, 64).contiguous()
        FusedAdamW([p], lr=0.1, max_grad_norm=1.0).step()
    torch.cuda.current_stream().wait_stream(side)
    q.grad = args[2][:1].expand(900, 64).contiguous()
    FusedAdamW([q], lr=0.1, max_grad_norm=1.0).step()
    assert same(got, want) and torch.equal(p, q)


def test_from_several_threads_at_once():
    cases = [inputs(10 + k, n=300 + 400 * k) for k in range(4)]
    want = [both(*c) for c in cases]
    params = [torch.nn.Parameter(c[0].detach().clone()) for c in cases]
    twins = [torch.nn.Parameter(c[0].detach().clone()) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                opt = FusedAdamW([params[k]], lr=1e-2, max_grad_norm=1.0, state_bits=8 if k % 2 else 32)
                for _ in range(20):
                    got = both(*cases[k])
                    params[k].grad = got[1]
                    opt.step()
                    torch.cuda.current_stream().synchronize()
                    if not same(got, want[k]):
                        wrong.append(k)
        except Exception as e:                            # (seen by the test, not only by the thread)
            wrong.append(e)

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    for k, (p, q) in enumerate(zip(params, twins)):
        opt = FusedAdamW([q], lr=1e-2, max_grad_norm=1.0, state_bits=8 if k % 2 else 32)
        for _ in range(20):
            q.grad = want[k][1]
            opt.step()
        assert torch.equal(p, q)


def test_transforms_and_tensors_without_memory_raise():
    """grad, vmap and jvp of torch.func, and fake tensors, hand over tensors whose memory cannot be read."""
    table, ids, grad, scores, items, ref = inputs(4)
    calls = (lambda t, i, s, y: ops.embedding_lookup(t, i).sum(), lambda t, i, s, y: list_logps(s, y).sum(),
             lambda t, i, s, y: preference_loss(s, y, ref)[0])
    args = (table, ids, scores, items)
    for f, over in zip(calls, (0, 2, 2)):
        with pytest.raises((RuntimeError, NotImplementedError, _ffi.RkError)):
            torch.func.grad(f, argnums=over)(*args)
        with pytest.raises((RuntimeError, NotImplementedError, _ffi.RkError)):
            torch.func.jvp(lambda x: f(*args[:over], x, *args[over + 1:]), (args[over],), (args[over],))
        for which in (over, over + 1):
            dims = tuple(0 if k == which else None for k in range(4))
            batched = [torch.stack([a, a]) if k == which else a for k, a in enumerate(args)]
            with pytest.raises((RuntimeError, NotImplementedError, _ffi.RkError)):
                torch.func.vmap(f, in_dims=dims)(*batched)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode() as mode:
        fake = [mode.from_tensor(a) for a in args]
        for f in calls[:2]:
            with pytest.raises((RuntimeError, NotImplementedError, _ffi.RkError)):
                f(*fake)


@pytest.mark.parametrize("make", [FusedAdamW, FusedClipAdam])
def test_recorded_training_step_follows_a_scheduler(make):
    g = torch.Generator().manual_seed(8)
    net = torch.nn.Module()
    net.weight = torch.nn.Parameter(torch.randn(64, generator=g).to(DEV))
    net.forward = lambda b: b["x"] * net.weight
    batches = [{"x": torch.randn(32, 64, generator=g).to(DEV)} for _ in range(6)]
    twin = torch.nn.Parameter(net.weight.detach().clone())
    opt, same = make([net.weight], lr=0.1, max_grad_norm=1.0), make([twin], lr=0.1, max_grad_norm=1.0)
    step = GraphedTrainStep(net, opt, lambda out, b: out.square().mean(), batches[0], warmup_steps=1)
    rates = [torch.optim.lr_scheduler.StepLR(o, 2, gamma=0.3) for o in (opt, same)]
    for k, b in enumerate([batches[0]] + batches):
        if k > 0:
            step(b)
        twin.grad, = torch.autograd.grad((b["x"] * twin).square().mean(), twin)
        same.step()
        for r in rates:
            r.step()
        torch.cuda.synchronize()
        assert torch.equal(net.weight, twin), k
    assert opt.param_groups[0]["lr"] < 0.01


def test_a_step_over_leaves_of_a_living_graph_is_not_captured():
    """Refused before anything is recorded; once the outputs are gone the same step is captured and replayed."""
    g = torch.Generator().manual_seed(9)
    net = torch.nn.Module()
    net.weight = torch.nn.Parameter(torch.randn(64, 8, generator=g).to(DEV))
    net.forward = lambda b: ops.embedding_lookup(net.weight, b["ids"], padding_idx=0)
    batch = {"ids": torch.randint(64, (30,), generator=g).to(DEV)}
    make = lambda: GraphedTrainStep(net, FusedAdamW([net.weight], lr=1e-2), lambda out, b: out.square().mean(), batch)  # noqa: E731
    out = net(batch)
    with pytest.raises(RuntimeError, match="delete its outputs"):
        make()
    with torch.no_grad():
        net(batch)
    del out
    step, before = make(), net.weight.detach().clone()
    step(batch)
    torch.cuda.synchronize()
    assert not torch.equal(net.weight, before)


def test_a_backward_pass_over_a_leaf_of_a_living_graph_is_not_recorded():
    table, ids, grad, scores, items, ref = inputs(5)
    table, scores = table.requires_grad_(True), scores.requires_grad_(True)
    alive = ops.embedding_lookup(table, ids), list_logps(scores, items)
    side = torch.cuda.Stream()
    for y, x, up, name in ((lambda: ops.embedding_lookup(table, ids), table, grad, "embedding_lookup"),
                           (lambda: list_logps(scores, items), scores, torch.ones(8, device=DEV), "list_logps"),
                           (lambda: preference_loss(scores, items, ref)[0], scores, None, "preference_loss")):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                    # eagerly it is fine
            want, = torch.autograd.grad(y(), x, up)
        torch.cuda.current_stream().wait_stream(side)
        with pytest.raises(RuntimeError, match=name + ": a backward pass over this leaf cannot be recorded"):
            with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
                torch.autograd.grad(y(), x, up)
        torch.cuda.synchronize()
        assert torch.equal(torch.autograd.grad(y(), x, up)[0], want)
    del alive
    with torch.cuda.stream(side):
        torch.autograd.grad(ops.embedding_lookup(table, ids), table, grad)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        dw, = torch.autograd.grad(ops.embedding_lookup(table, ids), table, grad)
    want, = torch.autograd.grad(ops.embedding_lookup(table, ids), table, grad)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, want)
