"""The softmax weights of attention over shared pages keep more bits than the output where that is asked for, in bfloat16 too.

Tolerance. The terms in float32 are those at the head of test_gpu_share.py, twice, as a sum of products on the tensor cores may be cut where a
float32 sum is rounded: 4 ((d + 8) S + n + 8) u of the weighted mean of |v|. Weights go into the product with the values as two bfloat16
parts: the first is off by 2^-8 of the weight at most, the second by 2^-8 of what that left, so 2^-16 of the mean. The output is rounded
to bfloat16 (2^-8 of itself). Weights of one part would be off by up to 2^-8 of the mean, sixteen times what is left for them here where
keys are few.
"""
import pytest
import torch

from test_gpu_share import B16, BATCHES, Case, path

pytestmark = pytest.mark.gpu

FEW = {"single-few-keys": [(path(), i, 1) for i in range(1, 20)],
       "runs-few-keys": [(path(), 0, 40), (path(("a", 1)), 64, 33), (path(("a", 1)), 65, 20), (path(), 3, 90)]}


def slack(c, want, mean, S, n):
    u = 2.0 ** -24
    return (4 * u * ((c.hd + 8) * S[..., None] + n[:, None, None] + 8) + 2.0 ** -16) * mean + 2.0 ** -8 * want.abs() + 1e-30


@pytest.mark.parametrize("layout", [(16, 4, 64, 64), (32, 32, 64, 64), (32, 8, 128, 128), (16, 4, 64, 128), (8, 1, 128, 64), (10, 2, 48, 40)], ids=str)
@pytest.mark.parametrize("batch", [*FEW, "nested", "runs", "long-runs", "many"])
def test_weights_keep_more_bits_than_the_output(batch, layout):
    c = Case(FEW.get(batch) or BATCHES[batch], layout, B16, seed=11)
    want, mean, S, n = c.formula()
    off = (c.run(exact_weights=True).double().view_as(want) - want).abs()
    over = off / slack(c, want, mean, S, n)
    assert bool((over <= 1).all()), float(over.max())


@pytest.mark.parametrize("layout", [(16, 4, 64, 64), (32, 8, 128, 128)], ids=str)
def test_capped_scores_and_sinks_keep_them_too(layout):
    """A cap of c takes a score to c tanh(s / c): tanh by an exponential and a reciprocal is off by a few 1e-7 (4e-7 here), times the cap."""
    for batch in ("runs-few-keys", "nested"):
        c = Case(FEW.get(batch) or BATCHES[batch], layout, B16, seed=12)
        sink = torch.linspace(-3, 3, layout[0]).cuda()
        want, mean, S, n = c.formula(softcap=4.0, sink=sink)
        off = (c.run(softcap=4.0, sink=sink, exact_weights=True).double().view_as(want) - want).abs()
        over = off / (slack(c, want, mean, S, n) + 2 * 4.0 * 4e-7 * mean)
        assert bool((over <= 1).all()), float(over.max())


def test_the_same_numbers_again():
    c = Case("runs", (16, 4, 64, 64), B16, seed=13)
    plan = c.plan()
    a, b = c.run(plan, exact_weights=True), c.run(plan, exact_weights=True)
    assert torch.equal(a, b) and not torch.equal(a, c.run(plan))
