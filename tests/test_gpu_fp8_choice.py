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
