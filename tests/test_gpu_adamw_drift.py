"""8-bit moments against 32-bit ones over long runs: how well roots and updates follow, and where they do not.

Bounds.  A stored root is a code times its block's scale, and a step moves a root by a factor between sqrt(beta2) and
whatever its gradient makes of it.  With beta2 = 0.999 the decay is 0.05 %, below half a code (2^-5 of the value at least),
so a code falls against its block's largest only where that one grows, and rises where a gradient lifts the root by half a
code: g^2 > 60 to 120 v.  In steady state a root then stays anywhere up to a few codes (each 2^-3 of the value at most) from
the 32-bit one: four of them either way, (1 + 1/8)^4 = 1.6, and the 32-bit root itself moves by 5 % under
1000 averaged squares: 0.55 to 1.8.  A cosine under relative errors e of the roots, spread evenly up to that, is
1 / sqrt(1 + var e) >= 0.97 for a spread of 25 %.  Where every second element's gradients fall tenfold, their roots stay where
they were: up to 10 x 1.8 too large, and the others' can lose what their block's scale loses: not below 1 / 10 / 1.8."""
import pytest
import torch

from recommend_amd.optim import FusedAdamW, decode_moment

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
STEPS, AT, N = 2500, 500, 64 * 512


def run(factor, second=True, beta2=0.999):
    """(cosine of the update, 8-bit roots over 32-bit roots of the changed elements, of the others) after STEPS steps in
    which the gradients of all or of every second element change by `factor` after step AT."""
    g = torch.Generator(device=DEV).manual_seed(21)
    p, q = (torch.nn.Parameter(torch.zeros(N, device=DEV)) for _ in range(2))
    eight, full = (FusedAdamW([x], lr=1e-3, weight_decay=0.0, betas=(0.9, beta2), state_bits=b) for x, b in ((p, 8), (q, 32)))
    size = torch.exp(torch.randn(N, generator=g, device=DEV))
    changed = torch.arange(N, device=DEV) % 2 == 0 if second else torch.ones(N, dtype=torch.bool, device=DEV)
    for t in range(STEPS):
        if t == AT:
            size = torch.where(changed, size * factor, size)
        p.grad = size * torch.randn(N, generator=g, device=DEV)
        q.grad = p.grad
        if t == STEPS - 1:
            before = p.detach().double(), q.detach().double()
        eight.step()
        full.step()
    moved = [x.detach().double() - b for x, b in zip((p, q), before)]
    st = eight.state[p]
    root = decode_moment(st["exp_avg_sq8"], st["exp_avg_sq8_scale"], p) / full.state[q]["exp_avg_sq"].sqrt()
    cosine = float(torch.nn.functional.cosine_similarity(*moved, dim=0))
    return cosine, root[changed].sort().values, root[~changed].sort().values


def within(x, lo, hi):
    """But for one element of 500 at either end (the largest of a block moves it alone)."""
    cut = len(x) // 500
    return lo <= float(x[cut]) and float(x[-1 - cut]) <= hi


def test_steady_gradients_and_changes_of_whole_blocks_are_followed():
    for factor in (1.0, 0.1):
        cosine, root, _ = run(factor, second=False)
        assert cosine >= 0.97 and within(root, 0.55, 1.8) and abs(float(root.median()) - 1) <= 0.1, (factor, cosine)


def test_a_short_average_is_followed_everywhere():
    """beta2 = 0.95: a step takes 2.5 % off a root, and 20 averaged squares move the true one by 16 %."""
    cosine, changed, others = run(0.1, beta2=0.95)
    assert cosine >= 0.97 and within(changed, 0.55, 1.8) and within(others, 0.55, 1.8)


def test_elements_that_shrink_against_their_block_are_bounded_only():
    cosine, changed, others = run(0.1)
    assert cosine >= 0.5 and within(changed, 0.55, 18.0) and within(others, 0.055, 1.8)
