"""Rows of the filtered token choice where float arithmetic is at its limits, on a real MI355X.  Tokens have to equal the
definition, with its weights rounded to 2^-45 of the largest (which u = 1, taken as 1 - 2^-53, tells from unrounded ones)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = math.inf
ONE = 1 - 2.0 ** -24      # the largest number torch.rand gives
UNIT = 2 ** 45            # (V <= 131072)


def choose(z, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """The definition, row by row, with whole numbers as weights; temperature > 0, no infinite logit."""
    out = []
    for row, ur in zip(z.double().cpu(), u.double().cpu()):
        V = row.numel()
        row = torch.where(torch.isnan(row), torch.full_like(row, -INF), row)
        w = torch.round(torch.exp((row - row.max()) / temperature) * UNIT).to(torch.int64)
        order = torch.argsort(row, descending=True, stable=True)
        ws = w[order]
        keep = torch.arange(V) < (top_k or V)
        cum = torch.cumsum(torch.where(keep, ws, 0), 0)
        if top_p < 1.0:
            keep &= cum - torch.where(keep, ws, 0) < math.ceil(top_p * int(cum[-1]))
        keep &= ws >= math.ceil(min_p * UNIT)
        c = torch.cumsum(torch.zeros_like(w).scatter_(0, order, torch.where(keep, ws, 0)), 0)
        target = int(min(max(float(ur), 0.0), 1 - 2.0 ** -53) * int(c[-1]))
        out.append(int((c <= target).sum()))
    return torch.tensor(out)


@pytest.mark.parametrize("row,temperature", [([20.0, 0, 0, 0, 0], 7e-8), ([20.0, 0, 0, 0, 0], 8.4e-8), ([2e8, -INF, -INF], 0.712),
                                             ([-50.0, -INF, math.nan, -50.5], 2.1e-7)])
@pytest.mark.parametrize("u", [0.0, 0.5, ONE, 1.0])
def test_dead_places_weigh_nothing(dev, row, temperature, u):
    """Temperatures of a few steps of the largest logit: the masked places and the columns behind the last one are never taken."""
    from src import ops
    z = torch.tensor([row])
    assert choose(z, torch.tensor([u]), temperature=temperature).tolist() == [0]
    got = ops.sample_tokens(z.to(dev), torch.tensor([u], device=dev), temperature=temperature)
    assert got.tolist() == [0]


@pytest.mark.parametrize("V", [5, 1025, 8200, 30522])
@pytest.mark.parametrize("mx", [20.0, 30.0, 100.0, 300.0, -77.0, 2e8])
def test_temperatures_of_a_few_steps_of_the_largest_logit(dev, V, mx):
    from src import ops
    at = V // 3
    z = torch.full((4, V), -INF)
    z[:, at] = mx
    z[1, ::2] = math.nan
    z[1, at] = mx
    step = float(torch.nextafter(torch.tensor(mx), torch.tensor(INF)) - torch.tensor(mx))
    z[2, V - 1] = mx - step                 # one step below the largest, and two
    z[3, [0, V - 1]] = torch.tensor([mx - 2 * step, mx - step])
    for steps in (0.011, 0.02, 0.0225, 0.029, 0.031, 0.045, 0.09, 0.11, 0.31, 1.0, 3.0):
        T = steps * step
        for u in (0.25, ONE, 1.0):
            ur = torch.full((4,), u)
            for f in (dict(), dict(top_p=0.999), dict(top_k=V - 1), dict(top_k=3, top_p=0.9), dict(min_p=1e-9)):
                got = ops.sample_tokens(z.to(dev), ur.to(dev), temperature=T, **f).cpu()
                assert int(got.max()) < V, (steps, u, f, got)
                assert torch.equal(got, choose(z, ur, temperature=T, **f)), (steps, u, f)


def agree(dev, z, u, copies=1, **f):
    """The rows' tokens, with every row `copies` times (the number of rows decides which kernel runs)."""
    from src import ops
    got = ops.sample_tokens(z.to(dev).repeat(copies, 1), u.to(dev).repeat(copies), **f).cpu().view(copies, -1)
    want = choose(z, u, **f)
    assert bool((got == want).all()), (f, got[0], want)
    return want


@pytest.mark.parametrize("V,copies", [(1000, 1), (5000, 1), (9000, 1), (9000, 130), (9000, 260), (30522, 1)])
def test_thousands_of_different_logits_in_one_bin(dev, V, copies):
    """Nearly flat rows and one far lower finite logit: the bins span that distance, the second histogram's too."""
    g = torch.Generator().manual_seed(V)
    z = 1e-6 * torch.randn(4, V, generator=g)
    z[:, 7] = -40.0
    z[1, ::3] = z[1, 5]                           # a third of them equal, at an ordinary place
    z[2] = torch.round(z[2] * 3e7) / 3e7          # every value many times
    z[2, 7] = -1e5
    z[3, : V // 2] = torch.sort(z[3, : V // 2]).values
    z[3, 7] = -40.0
    u = torch.rand(4, generator=g)
    cluster = V - 1
    for f in (dict(top_k=V // 2), dict(top_k=V // 3 + 1, temperature=0.5), dict(top_p=0.5), dict(top_p=0.3, temperature=1.7),
              dict(top_k=2 * V // 3, top_p=0.5), dict(top_k=cluster, top_p=0.999), dict(top_p=0.7, min_p=0.5)):
        for uu in (u, torch.full((4,), ONE), torch.zeros(4)):
            agree(dev, z, uu, copies, **f)


@pytest.mark.parametrize("V,copies", [(8192, 1), (9000, 1), (65000, 1), (65000, 260), (126464, 1), (126464, 130)])
def test_mass_that_the_estimate_does_not_see(dev, V, copies):
    """A tail of tokens that an estimate in units of 2^-32 rounds to nothing, and a top_p whose border lies in it."""
    g = torch.Generator().manual_seed(V)
    z = torch.empty(4, V)
    low = 33.03 * math.log(2.0)                   # weight 2^-33.03 of the largest
    z[0] = -low
    z[1] = -low * (1 + 0.01 * torch.rand(V, generator=g))
    z[2] = -low * (1 + 1e-6 * torch.rand(V, generator=g))
    z[3] = -low * (1 + 0.2 * torch.rand(V, generator=g))
    z[:, V // 5] = 0.0
    tail = 2.0 ** -33.03 * V
    moved = 0
    for share in (0.3, 0.8):
        # kept mass of the tail: about `share` of it (less where its weights differ)
        top_p = (1 + share * tail) / (1 + tail)
        for f in (dict(), dict(min_p=2.0 ** -33.5), dict(top_k=V - 3)):
            for u in (1 - 2.0 ** -22, ONE, 0.5):
                moved += int((agree(dev, z, torch.full((4,), u), copies, top_p=top_p, **f) != V // 5).sum())
    assert moved > 0                              # (the tail was drawn from)
