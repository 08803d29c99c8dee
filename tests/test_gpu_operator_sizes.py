"""The embedding, list and AdamW operators where element offsets pass 32 bits, and where launches are cut."""
import pytest
import torch

from recommend_amd import ops
from recommend_amd.loss import preference_loss
from recommend_amd.optim import FusedAdamW

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def test_lookup_and_gradient_beyond_2_31_elements():
    rows, D, n = 5000, 136, (1 << 24) + 3                 # 2.28e9 elements of rows and of gradients
    g = torch.Generator(device=DEV).manual_seed(1)
    ids = torch.randint(rows, (n,), generator=g, device=DEV)
    ids[: n // 8] = 17                                    # one run through thousands of workgroups
    table = torch.arange(rows, device=DEV, dtype=torch.float32).unsqueeze(1).expand(rows, D).contiguous().requires_grad_(True)
    out = ops.embedding_lookup(table, ids, scale=2.0)
    for a in (0, n // 2, n - 4096):
        assert torch.equal(out[a:a + 4096], 2 * table.detach()[ids[a:a + 4096]])
    grad = torch.ones(1, D, device=DEV).expand(n, D).contiguous()
    dw, = torch.autograd.grad(out, table, grad)
    count = torch.bincount(ids, minlength=rows).float()   # below 2^24: sums of ones are exact in any order
    assert torch.equal(dw, 2 * count.unsqueeze(1).expand(rows, D))


def test_lists_beyond_2_31_scores():
    S, T, V = 2, 20000, 63001                             # 2.52e9 scores; more rows than one workgroup joins
    g = torch.Generator(device=DEV).manual_seed(2)
    scores = torch.empty(S, T, V, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    items = torch.randint(V, (S, T), generator=g, device=DEV)
    items[:, 1::2] = -100
    scores.requires_grad_(True)
    loss, logps = preference_loss(scores, items, torch.zeros(S, device=DEV), beta=1e-4)
    want = torch.zeros(S, dtype=torch.float64, device=DEV)
    x = scores.detach()
    for s in range(S):
        for t in range(0, T, 500):
            at = torch.arange(t, t + 500, 2, device=DEV)
            rows = x[s, at].double()
            want[s] += (rows.gather(1, items[s, at].unsqueeze(1)).squeeze(1) - torch.logsumexp(rows, 1)).sum()
    # a row is off by (V / 256 / 16 + 96) u at most (its parts' threads add that many terms) and the rounding of a value
    # of about 11; the sum of 10000 rows rounds in 64 bits and once more at the end
    tol = 10000 * (130 + 3 * 12) * U + U * want.abs()
    assert bool(((logps.detach().double() - want).abs() <= tol).all())
    dx, = torch.autograd.grad(loss, scores)
    assert bool((dx[:, 1::2] == 0).all())
    d = 1e-4 * (want[0] - want[1])
    c = 1e-4 / (1 + torch.exp(d))
    for s, sign in ((0, -1.0), (1, 1.0)):
        row = x[s, T - 2].double()
        p = torch.softmax(row, 0)
        e = -sign * c * p
        e[items[s, T - 2]] += sign * c
        # half a step of bfloat16, the exponential's 32 u and what d's error moves c by
        slack = e.abs() * (2.0 ** -8 + 64 * U + 1e-4 * float(2 * tol.max())) + c * 64 * U * (p + (e.abs() > c / 2))
        assert bool(((dx[s, T - 2].double() - e).abs() <= slack).all())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_beyond_2_31_elements(bits):
    n = (1 << 31) + 5000 if bits == 8 else (1 << 30) + 5000      # (32 bits: the moments pass 2^32 bytes)
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device=DEV))
    p.grad = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    opt = FusedAdamW([p], lr=0.5, weight_decay=0.0, state_bits=bits, max_grad_norm=1e6)
    opt.step()
    # the first step moves every element by lr: -0.5 up to a rounding of the update, the same one in all elements
    assert float(p.detach().min()) == float(p.detach().max()) == -0.5
    assert abs(float(opt.grad_norm) - n ** 0.5) <= 2 * U * n ** 0.5
    st = opt.state[p]
    last = st["exp_avg8"][-64:].float() * st["exp_avg8_scale"][-1] if bits == 8 else st["exp_avg"][-64:]
    assert bool(((last[:5] - 0.1).abs() <= 0.1 * 4 * U).all())
