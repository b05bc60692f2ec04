"""Probabilities far below a row's maximum: the exponent's factor log2(e) / T is needed to more than 24 bits there."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0.0, 5.0, -700.0, 1900.0])
@pytest.mark.parametrize("v", [33, 1000, 16385, 40000, 128256, 140000])
def test_far_probabilities(v, shift):
    """One logit carries the row, the others lie 30 to 80 T below it, so the sum is that one weight and every error
    left is the element's own. p = 2^E / S, in units of a relative error: the fraction of each exponent in two
    roundings below one half (2 x 2^-25, times ln 2) and 2^x of it (2^-22), for the element and for the sum's one
    term; the scale between two slices' maxima, the element's slice's own and the sum's slice's own, 2^x each in two
    units of the last place (2 x 2^-23), whose arguments are rounded below 2^-24, times ln 2; the sum's scaling, its
    other terms (140,000 e^-30 in all), 1 / S and three products, 2^-24 each: 1.8e-6. With a factor of 24 bits alone
    the weights at 80 T would be off by up to 3.9e-6 at these temperatures."""
    from laicompute_b200.serving import logits_probs
    temp = [1.0, 0.7, 0.3, 1.3, 7.5, 2.9, 0.11, 0.93]
    rng = np.random.default_rng(v)
    x = np.zeros((len(temp), v), np.float32)
    for r, t in enumerate(temp):
        x[r] = (shift - rng.uniform(30, 80, size=v)) * t
        x[r, rng.integers(v)] = shift * t
    x = torch.from_numpy(x)
    t = torch.tensor(temp, dtype=torch.float32)
    dev, td, out = x.cuda(), t.cuda(), torch.zeros(len(temp), v, device="cuda")
    logits_probs(len(temp), v, dev.data_ptr(), td.data_ptr(), out.data_ptr())
    want = torch.softmax(x.double() / t.double()[:, None], dim=1)
    rel = 2 * (2 * 2.0 ** -25 * 0.6932 + 2.0 ** -22) + 3 * (2 * 2.0 ** -23 + 2.0 ** -24 * 0.6932) + 6 * 2.0 ** -24
    err = ((out.cpu().double() - want).abs() / want).max(dim=1).values
    print(v, shift, (err / rel).numpy().round(2))
    assert bool((err <= rel).all()), (err / rel)
