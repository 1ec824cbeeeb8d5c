"""The ragged operators where an argument or a neighbour is extreme: large caps, rows beside the live ones, windows whose
old pages are gone, far distances, long item lists. Tolerances are ragged_ref's unless a test derives its own."""
import math

import pytest
import torch

from ragged_ref import attend64, attend_check

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
ROWS = [1, 1000]  # rows per KV head that max_q announces: one for each kernel


def starts(dev, *counts):
    return torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32, device=dev)


def randn(dev, shape, seed, dtype, gain=1.0):
    return (torch.randn(shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev) * gain).to(dtype)


# ---------------------------------------------------------------- capped scores
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("cap", [0.25, 50.0, 1e3, 1e4, 1e6, 1e12, 1e30, 1.9e38])
def test_caps_of_any_size(pkg, dev, dtype, rows, slope, cap):
    """cap tanh(s / cap) is s itself where the cap is large: a fixed cap must not cost the score its digits. fp32 forms it
    with a relative error below 2^-20, so scores below 32 in the base-2 exponent keep to the 1e-4 of attend_check."""
    n, m, D = 5, 300, 128
    q, k, v = randn(dev, (n, 2, D), 1, dtype), randn(dev, (m, 1, D), 2, dtype), randn(dev, (m, 1, D), 3, dtype)
    slopes = torch.tensor([0.05, 0.01], device=dev) if slope else None
    lse = torch.empty((n, 2), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(dev, n), starts(dev, m), softcap=cap, slopes=slopes, lse=lse,
                              max_q=rows)
    want, l64, mass = attend64(q, k, v, softcap=cap, slopes=slopes)
    attend_check(out, want, mass, dtype, m, v.abs().max().item())
    assert ((lse.double() - l64).abs() < 2e-4).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("slope", [False, True])
@pytest.mark.parametrize("cap", [1e3, 1e5])
def test_large_cap_beside_scores_beyond_it(pkg, dev, dtype, rows, slope, cap):
    """Some keys score far below -cap (a padded key of the type's lowest values): the others keep their digits."""
    n, m, D = 3, 200, 128
    q, k, v = randn(dev, (n, 2, D), 4, dtype), randn(dev, (m, 1, D), 5, dtype), randn(dev, (m, 1, D), 6, dtype)
    q[..., 0], k[..., 0] = 40.0, 0.0
    k[::17, 0] = 0.0
    k[::17, 0, 0] = -60000.0  # the score -212000
    slopes = torch.tensor([0.05, 0.01], device=dev) if slope else None
    lse = torch.empty((n, 2), device=dev)
    out = pkg.ops.attn_packed(q, k, v, starts(dev, n), starts(dev, m), softcap=cap, slopes=slopes, lse=lse,
                              max_q=rows)
    want, l64, mass = attend64(q, k, v, softcap=cap, slopes=slopes)
    attend_check(out, want, mass, dtype, m, v.abs().max().item())
    assert ((lse.double() - l64).abs() < 2e-4).all()
