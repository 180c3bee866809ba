"""Dropout's gradients in a ragged batch.  By x it is the same call on dy; by the
residual it is dy inside the sequences and 0 past their ends, whose rows are zeros
whatever the residual holds: the same call on dy with p = 0."""

import pytest
import torch

from test_dropout import call, keep_of
from test_sequence import DTYPES, F64, laid_out, lib, rnd, stream  # noqa: F401
from ns_fps_amd import capi


def plain(x, r, keep, lens, p):
    """The definition in 64 bits."""
    inside = torch.arange(x.shape[1])[None, :, None] < torch.tensor(lens)[:, None, None]
    factor = 65536 / (65536 - round(p * 65536))
    return torch.where(inside, r + torch.where(keep, x * factor, 0.0), 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("channels,how", [(64, "plain"), (321, "odd")])
def test_gradients_of_a_ragged_batch(lib, channels, how, dtype):  # noqa: F811
    t, code = DTYPES[dtype]
    case, lens, p = (4, 40, channels, how), [40, 0, 13, 39], 0.25
    gen = torch.Generator().manual_seed(channels)
    x, r, dy = (rnd(gen, 4, 40, channels, dtype=t) for _ in range(3))
    seed = torch.tensor([5, 6], dtype=torch.int64)
    leaves = [v.to(F64).requires_grad_() for v in (x, r)]
    y = plain(*leaves, keep_of(4, 40, channels, p, seed.tolist()), lens, p)
    want = torch.autograd.grad((y * dy.to(F64)).sum(), leaves)
    sd, ld = seed.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    got = []
    for q in (p, 0.0):
        out = laid_out(torch.full_like(dy, float("nan")).cuda(), how)
        call(lib, case, code, laid_out(dy.cuda(), how), None, out, q, sd, ld)
        got.append(out.cpu().to(F64))
    assert torch.equal(got[1], want[1])
    assert want[1][1].eq(0).all() and not torch.equal(want[1], dy.to(F64))  # it is not dy itself
    tol = 2.0 ** -23 + (2.0 ** -8 if t == torch.bfloat16 else 0.0)
    assert ((got[0] - want[0]).abs() <= tol * want[0].abs()).all()


def test_the_definition_against_differences():
    """By the residual, row by row: what the formula gives inside, nothing past the end."""
    gen = torch.Generator().manual_seed(1)
    x, r, dy = (torch.randn(2, 5, 9, generator=gen, dtype=F64) for _ in range(3))
    keep, lens = keep_of(2, 5, 9, 0.5, [1, 2]), [5, 2]
    for b in range(2):
        for row in range(5):
            step = torch.zeros_like(r)
            step[b, row] = torch.randn(9, generator=gen, dtype=F64)
            diff = ((plain(x, r + step, keep, lens, 0.5) - plain(x, r - step, keep, lens, 0.5))
                    * dy).sum() / 2
            want = (step * dy).sum() if row < lens[b] else 0.0
            assert abs(diff - want) < 1e-12
