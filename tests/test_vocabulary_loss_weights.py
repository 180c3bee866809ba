"""A weight that all tokens have in common is not rounded into every term of the loss's
bfloat16 gradients."""

import pytest
import torch

from test_sequence import F64, lib  # noqa: F401
from test_vocabulary_loss import Want, inputs
from test_vocabulary_loss_rows import gradients

# d's rounding, beside the results' own.  A result's own rounding to 8 bits has a norm
# of at most 2^-8 / sqrt(3) of its own, and of about 0.68 of that where mantissas are
# spread (1 / sqrt(E[m^2]) over a factor of two): 0.0015.  Against a weight of exactly
# itself a token's own term is -(1 - p), which 8 bits hold to 2^-9 at most: sqrt(0.0015^2
# + 0.00195^2) = 0.0025.  A weight halfway between two of 8 bits is off by 2^-8 =
# 0.0039 in every term alike, which adds to the norm: sqrt(0.0015^2 + 0.0039^2) = 0.0042.
ALIKE = 0.64 * 2.0 ** -8
HALFWAY = (1 + 2.0 ** -8 - 2.0 ** -20) * 2.0 ** -9


def alike(case, rounded):
    """The gradients' relative errors in norm with d rounded to 8 bits, relative to the
    weight or absolutely; x, table, target, scale."""
    n, rows, width, _ = case
    t, code, gen, x, table, target, scale = inputs(case, "bf16")
    scale = 0.25
    want = Want(x, table, target, scale, torch.full((n,), HALFWAY / scale))
    z = x.to(F64) @ table.to(F64).T * scale
    p = torch.exp(z - want.lse[:, None])
    one = torch.zeros_like(p)
    one.scatter_(1, torch.where(want.counts, target, 0).long()[:, None], 1.0)
    d = torch.where(want.counts[:, None], p - one, 0.0)
    d = d.bfloat16().to(F64) * HALFWAY if rounded == "relative" else (d * HALFWAY).bfloat16().to(F64)
    x0 = torch.where(want.counts[:, None], x.to(F64), 0.0)
    got = (d @ table.to(F64)).bfloat16().to(F64), (d.T @ x0).bfloat16().to(F64)
    return [((g - w).norm() / w.norm()).item() for g, w in zip(got, (want.dx, want.dtable))]


ALIKE_CASES = [(300, 700, 64, 0), (1100, 2500, 128, 0)]


@pytest.mark.parametrize("case", ALIKE_CASES)
def test_the_bound_tells_relative_from_absolute_weights(case):
    """By the oracle: d relative to the weight is within the bound, d rounded with its
    weight is not."""
    assert max(alike(case, "relative")) <= ALIKE
    assert min(alike(case, "absolute")) > 1.4 * ALIKE


@pytest.mark.gpu
@pytest.mark.parametrize("case", ALIKE_CASES)
def test_a_common_weight_is_not_rounded(lib, case):  # noqa: F811
    n, rows, width, _ = case
    t, code, gen, x, table, target, _ = inputs(case, "bf16")
    scale = 0.25
    dloss = torch.full((n,), HALFWAY / scale)
    got, want = gradients(lib, case, x, table, target, scale, dloss, 0)
    for g, w in zip(got, (want.dx, want.dtable)):
        assert (g.to(F64) - w).norm() <= ALIKE * w.norm()
