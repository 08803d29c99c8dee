"""FusedAdamW against torch.optim.AdamW in 64 bits (32-bit moments) and against the same steps written in torch
(8-bit moments: the same codes).

Tolerances, u = 2^-24, over n steps with gradients up to G, parameters up to W and rate r (updates up to about 4 r):
  moments   every step rounds three times: n 3 u of their largest value (and n 2 u G of the factors' rounding)
  p         n roundings of p (two a step) and of the update (16 u 4 r, plus the moments' own error, relative)."""
import copy

import pytest
import torch

from recommend_amd import _ffi
from recommend_amd.optim import FusedAdamW, FusedClipAdam, decode_moment, encode_moment

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
SHAPES = [(64, 64), (64,), (1,), (64, 4096), (5000, 7), (128, 128), (3,), (4097,), (0, 5)]


def params_of(shapes, g, dtype=torch.float32):
    return [torch.nn.Parameter((torch.randn(s, generator=g) * 0.1).to(dtype).to(DEV)) for s in shapes]


@pytest.mark.parametrize("wd,max_norm", [(0.0, 1.0), (0.1, 0.3), (0.01, None)])
def test_matches_torch_adamw_over_ten_steps(wd, max_norm):
    g = torch.Generator().manual_seed(3)
    ours = params_of(SHAPES, g)
    ref = [torch.nn.Parameter(p.detach().cpu().double()) for p in ours]
    unused = torch.nn.Parameter(torch.ones(10, device=DEV))
    half = len(SHAPES) // 2
    opt = FusedAdamW([{"params": ours[:half] + [unused]}, {"params": ours[half:], "weight_decay": 0.0, "lr": 2e-3, "betas": (0.8, 0.99)}],
                     lr=1e-3, weight_decay=wd, max_grad_norm=max_norm)
    topt = torch.optim.AdamW([{"params": ref[:half]}, {"params": ref[half:], "weight_decay": 0.0, "lr": 2e-3, "betas": (0.8, 0.99)}],
                             lr=1e-3, weight_decay=wd)
    for step in range(10):
        scale = 10.0 if step % 3 == 0 else 0.05
        for p, q in zip(ours, ref):
            gr = torch.randn(p.shape, generator=g) * scale
            p.grad, q.grad = gr.to(DEV), gr.double()
        if max_norm is not None:
            want = torch.nn.utils.clip_grad_norm_(ref, max_norm)
        topt.step()
        opt.step()
        if max_norm is not None:
            assert abs(float(opt.grad_norm) - float(want)) <= 2 * U * float(want)
        if step == 4:
            for o in (opt, topt):
                o.param_groups[0]["lr"] = 5e-4
    big = 60.0 if max_norm is None else max_norm
    for p, q in zip(ours, ref):
        if not p.numel():
            continue
        st, tst = opt.state[p], topt.state[q]
        for k, top in (("exp_avg", big), ("exp_avg_sq", big * big)):
            tol = 50 * U * max(float(tst[k].abs().max()), top * 0.2)
            assert float((st[k].cpu().double() - tst[k]).abs().max()) <= tol, (k, p.shape)
        # an element's update is m / sqrt(v): where v is small against the moments' rounding above nothing is left of it, so
        # the error of the updates is taken relative, 10 steps of up to 4 r each with 64 u
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) <= 10 * (2 * U * float(q.detach().abs().max()) + 64 * U * 4 * 2e-3)
    assert bool((unused == 1).all()) and not opt.state[unused]
    assert int(opt.step_count) == 10


def plain_step(p, g, m, v, t, lr, b1, b2, eps, wd, coef=None):
    """One step in fp32 torch operations in the kernel's order; m and v are updated, the new p is returned."""
    g = g.float()
    if coef is not None:
        g = g * coef
    m.copy_(m * b1 + g * (1 - b1))
    v.copy_(v * b2 + (g * g) * (1 - b2))
    x = p.float()
    x = x - x * (lr * wd)
    return (x - (lr / (1 - b1 ** t)) * (m / (v.sqrt() / (1 - b2 ** t) ** 0.5 + eps))).to(p.dtype)


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("pd,gd", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                   (torch.bfloat16, torch.float32), (torch.float16, torch.float16), (torch.float16, torch.float32)])
@pytest.mark.parametrize("bits", [8, 32])
def test_states_are_those_of_the_same_steps_in_torch(bits, pd, gd, max_norm):
    """Moments and codes bit for bit over five steps; parameters to one rounding of their type and the update's own
    error (16 u of it)."""
    g = torch.Generator().manual_seed(7)
    shapes = [(100, 65), (64, 64), (5000,), (17,), (4096,), (4095,), (129, 33)]
    ours = params_of(shapes, g, pd)
    for p in ours:
        p.grad_dtype = gd
    ref = [p.detach().clone() for p in ours]
    m = [torch.zeros(s, device=DEV) for s in shapes]
    v = [torch.zeros(s, device=DEV) for s in shapes]
    opt = FusedAdamW(ours, lr=1e-2, weight_decay=0.1, max_grad_norm=max_norm, state_bits=bits)
    for t in range(1, 6):
        for i, p in enumerate(ours):
            rough = torch.randn(p.shape, generator=g) * torch.exp(2 * torch.randn(p.shape, generator=g))
            rough[torch.rand(p.shape, generator=g) < 0.2] = 0
            p.grad = rough.to(gd).to(DEV)
        coef = None
        if max_norm is not None:
            norm = sum((p.grad.double() ** 2).sum() for p in ours).sqrt()
            coef = (max_norm / (norm + 1e-6)).clamp_max(1.0).float()
        opt.step()
        for i, p in enumerate(ours):
            before = ref[i]
            ref[i] = plain_step(before, p.grad, m[i], v[i], t, 1e-2, 0.9, 0.999, 1e-8, 0.1, coef)
            st = opt.state[p]
            if bits == 8 and p.numel() >= 4096:
                for key, x, keep in (("exp_avg8", m[i], False), ("exp_avg_sq8", v[i].sqrt(), True)):
                    code, scale = encode_moment(x, keep)
                    assert torch.equal(st[key].view(torch.uint8), code.view(torch.uint8)), (key, t, p.shape)
                    assert torch.equal(st[key + "_scale"], scale)
                    back = decode_moment(code, scale, p)
                    (m if key == "exp_avg8" else v)[i].copy_(back if key == "exp_avg8" else back * back)
            else:
                assert torch.equal(st["exp_avg"], m[i]) and torch.equal(st["exp_avg_sq"], v[i]), (t, p.shape)
            # one rounding of p in its type, and u of the two subtractions, 16 u of the update
            moved = (ref[i].double() - before.double()).abs()
            tol = ref[i].double().abs() * (torch.finfo(pd).eps if pd != torch.float32 else 4 * U) + 16 * U * (moved + 0.1) + 1e-7 * (pd == torch.float16)
            assert bool(((p.detach().double() - ref[i].double()).abs() <= tol).all()), (t, p.shape)
            ref[i] = p.detach().clone()
    assert int(opt.step_count) == 5


def test_moments_that_are_not_zero_keep_their_update_bounded():
    """A row beside one whose gradients are 1e6 times larger: its root moment stays above zero when its gradient stops,
    and the update with it below the rate times 1 / (1 - beta2)^(1/2)."""
    p = torch.nn.Parameter(torch.zeros(4096, device=DEV))
    opt = FusedAdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    grad = torch.full((4096,), 1e-6, device=DEV)
    grad[::64] = 1.0
    for k in range(6):
        before = p.detach().clone()
        p.grad = grad if k < 3 else torch.zeros_like(grad)
        opt.step()
        assert float((p.detach() - before).abs().max()) <= 1e-3 * 33
    assert bool((opt.state[p]["exp_avg_sq8"].float() > 0).all())


def test_non_finite_gradients_are_seen():
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.zeros(5000, device=DEV))
        opt = FusedAdamW([p], state_bits=bits, max_grad_norm=1.0)
        p.grad = torch.ones(5000, device=DEV)
        p.grad[77] = float("nan")
        opt.step()
        assert bool(torch.isnan(opt.grad_norm)) and bool(torch.isnan(p).all())   # clip_grad_norm_ spreads it too
        q = torch.nn.Parameter(torch.zeros(5000, device=DEV))
        opt = FusedAdamW([q], state_bits=bits)
        q.grad = torch.ones(5000, device=DEV)
        q.grad[77] = float("nan")
        opt.step()
        opt.step()
        assert bool(torch.isnan(q[77])) and bool(torch.isfinite(q[128:]).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_unaligned_parameters_and_gradients(bits):
    """Parameters that begin at odd addresses inside a larger buffer: neighbours are left as they were."""
    for dtype in (torch.float32, torch.bfloat16):
        buf, gbuf = torch.full((9003,), 7.0, device=DEV, dtype=dtype), torch.ones(9007, device=DEV, dtype=dtype)
        p = torch.nn.Parameter(buf[1:8998])
        p.grad = gbuf[3:9000]
        same = torch.nn.Parameter(torch.full((8997,), 7.0, device=DEV, dtype=dtype))
        same.grad = torch.ones(8997, device=DEV, dtype=dtype)
        for q in (p, same):
            FusedAdamW([q], lr=0.1, state_bits=bits).step()
        assert torch.equal(p.detach(), same.detach()) and float((p.detach() - 7).abs().max()) > 0.01
        assert buf[0] == 7 and bool((buf[8998:] == 7).all())


def test_many_tensors_take_several_launches():
    g = torch.Generator().manual_seed(5)
    ours = params_of([(50 + i,) for i in range(110)] + [(300, 300)], g)
    one = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    opt = FusedAdamW(ours, lr=1e-2, max_grad_norm=1.0)
    parts = FusedAdamW(one, lr=1e-2)
    for _ in range(3):
        grads = [torch.randn(p.shape, generator=g).to(DEV) for p in ours]
        norm = sum((x.double() ** 2).sum() for x in grads).sqrt()
        coef = (1.0 / (norm + 1e-6)).float()
        for p, q, x in zip(ours, one, grads):
            p.grad, q.grad = x, x * coef
        opt.step()
        parts.step()
        assert abs(float(opt.grad_norm) - float(norm)) <= 2 * U * float(norm)
    assert all(torch.equal(p, q) for p, q in zip(ours, one))


@pytest.mark.parametrize("bits", [8, 32])
def test_checkpoints_continue(bits):
    g = torch.Generator().manual_seed(9)
    shapes = [(100, 64), (64,)]
    ours = params_of(shapes, g, torch.bfloat16)
    opt = FusedAdamW(ours, lr=1e-2, state_bits=bits)
    grads = [[torch.randn(s, generator=g).to(torch.bfloat16).to(DEV) for s in shapes] for _ in range(6)]

    def steps(o, ps, k0, k1):
        for k in range(k0, k1):
            for p, x in zip(ps, grads[k]):
                p.grad = x
            o.step()

    steps(opt, ours, 0, 3)
    saved, weights = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in ours]
    steps(opt, ours, 3, 6)
    fresh = [torch.nn.Parameter(w.clone()) for w in weights]
    again = FusedAdamW(fresh, lr=1e-2, state_bits=bits)
    again.load_state_dict(saved)
    assert all(v.dtype == saved["state"][0][k].dtype for k, v in again.state[fresh[0]].items() if k != "step")
    steps(again, fresh, 3, 6)
    assert all(torch.equal(a, b) for a, b in zip(ours, fresh)) and int(again.step_count) == 6
    # into an optimizer that has stepped: its buffers keep their memory
    held = {k: v.data_ptr() for k, v in again.state[fresh[0]].items() if k != "step"}
    with torch.no_grad():
        for p, w in zip(fresh, weights):
            p.copy_(w)
    again.load_state_dict(saved)
    assert held == {k: v.data_ptr() for k, v in again.state[fresh[0]].items() if k != "step"}
    steps(again, fresh, 3, 6)
    assert all(torch.equal(a, b) for a, b in zip(ours, fresh))


def test_checkpoints_of_other_forms_load():
    g = torch.Generator().manual_seed(10)
    ref = [torch.nn.Parameter(torch.randn(90, 64, generator=g).to(DEV))]
    topt = torch.optim.AdamW(ref, lr=1e-3)
    ref[0].grad = torch.randn(90, 64, generator=g).to(DEV)
    topt.step()
    p = [torch.nn.Parameter(ref[0].detach().clone())]
    o32, o8 = FusedAdamW(p, lr=1e-3), FusedAdamW(p, lr=1e-3, state_bits=8)
    o32.load_state_dict(topt.state_dict())
    assert torch.equal(o32.state[p[0]]["exp_avg"], topt.state[ref[0]]["exp_avg"]) and int(o32.state[p[0]]["step"]) == 1
    o8.load_state_dict(o32.state_dict())
    st, want = o8.state[p[0]], topt.state[ref[0]]
    for key, x in (("exp_avg8", want["exp_avg"]), ("exp_avg_sq8", want["exp_avg_sq"].sqrt())):
        got = decode_moment(st[key], st[key + "_scale"], x)
        # half a step of e4m3, or of the smallest code (2^-9 of 448 of the block's largest)
        assert bool(((got - x).abs() <= torch.maximum(x.abs() * 2.0 ** -4, x.abs().max() * 2.0 ** -10 / 448) * 1.001).all())
    back = FusedAdamW(p, lr=1e-3)
    back.load_state_dict(o8.state_dict())
    assert torch.equal(back.state[p[0]]["exp_avg"], decode_moment(st["exp_avg8"], st["exp_avg8_scale"], p[0]))


@pytest.mark.parametrize("bits", [8, 32])
def test_copies_continue(bits):
    g = torch.Generator().manual_seed(12)
    p = params_of([(100, 64)], g)[0]
    opt = FusedAdamW([p], lr=1e-2, max_grad_norm=1.0, state_bits=bits)
    grads = [torch.randn(100, 64, generator=g).to(DEV) for _ in range(3)]
    p.grad = grads[0]
    opt.step()
    q, other = copy.deepcopy((p, opt))
    assert other.param_groups[0]["params"][0] is q
    for x in grads[1:]:
        p.grad, q.grad = x, x.clone()
        opt.step()
        other.step()
    assert torch.equal(p, q) and int(other.step_count) == 3


@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_in_a_graph_and_replayed(bits):
    g = torch.Generator().manual_seed(13)
    ours = params_of([(100, 64), (64,)], g)
    eager = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a, b = (FusedAdamW(x, lr=1e-2, max_grad_norm=1.0, state_bits=bits) for x in (ours, eager))
    for p, q in zip(ours, eager):
        p.grad, q.grad = torch.ones_like(p), torch.ones_like(q)
    a.step()
    b.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.step()
    for k in range(4):
        for p, q in zip(ours, eager):
            x = torch.randn(p.shape, generator=g)
            p.grad.copy_(x)
            q.grad.copy_(x)
        if k == 2:
            for o in (a, b):
                o.param_groups[0]["lr"] = 3e-3
            a.sync_lr()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ours, eager)) and int(a.step_count) == int(b.step_count) == k + 2


def test_recorded_step_outlives_a_larger_workspace():
    """A step over one tensor is recorded; later steps over more tensors need a larger workspace.  The recorded step
    goes on with its own, which nothing else has been given meanwhile."""
    first, more = params_of([(300, 64)], torch.Generator().manual_seed(16))[0], [torch.nn.Parameter(torch.zeros(8, device=DEV))
                                                                               for _ in range(60)]
    opt = FusedAdamW([first], lr=1e-2, max_grad_norm=1.0)
    first.grad = torch.ones_like(first)
    opt.step()
    size = opt._ws.numel()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.add_param_group({"params": more})
    for p in more:
        p.grad = torch.ones_like(p)
    opt.step()
    assert opt._ws.numel() > size
    others = [torch.full((size,), 7.0, dtype=torch.float64, device=DEV) for _ in range(20)]
    twin = torch.nn.Parameter(first.detach().clone())
    same = FusedAdamW([twin], lr=1e-2, max_grad_norm=1.0)
    twin.grad = first.grad
    same.load_state_dict({"state": {0: {k: v.clone() for k, v in opt.state[first].items()} | {"step": 2}},
                          "param_groups": same.state_dict()["param_groups"]})
    for _ in range(3):
        graph.replay()
        same.step()
        torch.cuda.synchronize()
        assert torch.equal(first, twin)
    assert all(bool((o == 7.0).all()) for o in others)


def test_a_first_step_is_not_recorded():
    a, b = params_of([(300, 64), (64,)], torch.Generator().manual_seed(17))
    opt = FusedAdamW([a, b], lr=1e-2)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    for missing in (2, 1):                               # both parameters' moments, then one's
        before = [p.detach().clone() for p in (a, b)]
        with pytest.raises(RuntimeError, match="before capturing"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                opt.step()
        assert torch.equal(a, before[0]) and torch.equal(b, before[1])
        if missing == 2:
            b.grad = None
            opt.step()
            b.grad = torch.ones_like(b)
    opt.step()
    assert int(opt.step_count) == 2


def test_refuses_what_it_cannot_update():
    opt = FusedAdamW([torch.nn.Parameter(torch.zeros(8, 8, device=DEV).t()[1:])])
    p = opt.param_groups[0]["params"][0]
    for bad in (torch.zeros_like(p), ):
        p.grad = bad
        with pytest.raises(_ffi.RkError, match="contiguous"):
            opt.step()
    q = torch.nn.Parameter(torch.zeros(8, device=DEV, dtype=torch.float64))
    q.grad = torch.zeros_like(q)
    with pytest.raises(_ffi.RkError, match="fp32, bfloat16 or fp16"):
        FusedAdamW([q]).step()
    r = torch.nn.Parameter(torch.zeros(8, 4, device=DEV))
    r.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 4), (8, 4)).to(DEV)
    with pytest.raises(_ffi.RkError, match="dense"):
        FusedAdamW([r]).step()


def test_state_of_other_sizes_is_refused():
    for bits in (8, 32):
        p = torch.nn.Parameter(torch.zeros(5000, device=DEV))
        p.grad = torch.ones_like(p)
        opt = FusedAdamW([p], state_bits=bits)
        opt.step()
        key = "exp_avg8" if bits == 8 else "exp_avg"
        for bad in (opt.state[p][key][:-64], opt.state[p][key].float().half(), opt.state[p][key].cpu()):
            keep, opt.state[p][key] = opt.state[p][key], bad
            with pytest.raises(ValueError, match="not what this optimizer made"):
                opt.step()
            opt.state[p][key] = keep
        opt.step()


def test_the_same_step_as_clip_adam_without_decay():
    """Without weight decay AdamW and Adam are the same update: FusedClipAdam's result to the rounding of three steps."""
    g = torch.Generator().manual_seed(15)
    ours = params_of([(64, 64), (300,)], g)
    ref = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a, b = FusedAdamW(ours, lr=1e-3, weight_decay=0.0, max_grad_norm=1.0), FusedClipAdam(ref, lr=1e-3, max_grad_norm=1.0)
    for _ in range(3):
        for p, q in zip(ours, ref):
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
            q.grad = p.grad.clone()
        a.step()
        b.step()
    # FusedClipAdam takes 1 - beta2^t in fp32: off by up to 2^-14 relative in the first steps, half of that in its root
    for p, q in zip(ours, ref):
        assert float((p - q).abs().max()) <= 3 * (1e-3 * 4 * 2.0 ** -14)
