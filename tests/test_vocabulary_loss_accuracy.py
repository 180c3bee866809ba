"""Losses that are far smaller than their logits."""

import math

import pytest
import torch

from ns_fps_amd import capi
from test_sequence import DTYPES, F64, lib, stream  # noqa: F401
from test_vocabulary_loss import args_of, give


def run_loss(lib, x, table, target, scale):  # noqa: F811
    loss, lse = (torch.full((len(x),), float("nan"), device="cuda") for _ in range(2))
    code = capi.F32 if x.dtype == torch.float32 else capi.BF16
    xd, td, tg = x.cuda(), table.cuda(), target.cuda()
    args = args_of((len(x), len(table), x.shape[1], 0), code, xd, td, tg, scale, loss, lse)
    ws = give(args, lib.loss_workspace_bytes(args))
    lib.loss_device(args, stream())
    torch.cuda.synchronize()
    del ws
    return loss.cpu().to(F64), lse.cpu().to(F64)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("width,scale,rows", [(16, 1.0, 1), (64, 1.0, 2), (64, 0.7, 1), (80, -1.3, 2),
                                              (320, 3.0, 1)])
def test_losses_keep_what_is_below_their_logits(lib, width, scale, rows, dtype):  # noqa: F811
    """Rows alike, whole numbers, so that every product's sum is exact: lse is the
    logit and log(rows), the loss log(rows) however large the logit is.  The sum of
    exponentials and its logarithm are off by 2^-21 at most (the running maximum's
    rounding goes into both and drops out, as do the roundings of scale * log2(e));
    z itself, scale times a whole number, is taken in float64.  A sum of two
    exponentials of 2^-24 relative error each, its logarithm's and the loss's own
    rounding: 2^-21; lse is rounded once more, by 2^-24 of itself."""
    t, _ = DTYPES[dtype]
    gen = torch.Generator().manual_seed(width)
    table = torch.randint(-2, 3, (1, width), generator=gen).repeat(rows, 1).to(t)
    n = 40
    x = torch.randint(-8, 9, (n, width), generator=gen).to(t)
    x[0] = 0
    target = torch.randint(0, rows, (n,), generator=gen, dtype=torch.int32)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    z = scale * (x.to(F64) @ table[0].to(F64))
    assert z.abs().max() > 40
    loss, lse = run_loss(lib, x, table, target, scale)
    want = math.log(rows)
    assert (loss - want).abs().max() <= 2.0 ** -21, (loss - want).abs().max().item()
    assert ((lse - z - want).abs() <= 2.0 ** -21 + 2.0 ** -24 * (z.abs() + 1)).all()
