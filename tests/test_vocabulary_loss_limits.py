"""What the vocabulary loss's documentation says of accuracy, of what lies beside rows,
of its workspace and of its numbers' ends."""

import math

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import within
from test_sequence import A, DTYPES, EINVAL, F64, lib, ptr, rnd, stream  # noqa: F401
from test_vocabulary_loss import Want, args_of, give, good, good_grads, inputs

# ------------------------------------------------------------------- accuracy


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
    assert z.abs().max() > 60
    loss, lse = run_loss(lib, x, table, target, scale)
    want = math.log(rows)
    assert (loss - want).abs().max() <= 2.0 ** -21, (loss - want).abs().max().item()
    assert ((lse - z - want).abs() <= 2.0 ** -21 + 2.0 ** -24 * (z.abs() + 1)).all()


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


# --------------------------------------------------------- what lies beside rows

def gradients(lib, case, x, table, target, scale, dloss, pad, grad="bf16"):  # noqa: F811
    """Gradients with NaN beside every row read, and beside every row written, where
    they have to stay."""
    n, rows, width, _ = case
    t = x.dtype
    gt, gcode = DTYPES[grad]
    xd, td = (torch.full((len(v), width + pad), float("nan"), dtype=t) for v in (x, table))
    xd[:, :width], td[:, :width] = x, table
    xd, td, tg, dl = xd.cuda(), td.cuda(), target.cuda(), dloss.cuda()
    loss, lse = (torch.full((n,), float("nan"), device="cuda") for _ in range(2))
    code = capi.F32 if t == torch.float32 else capi.BF16
    args = args_of(case, code, xd, td, tg, scale, loss, lse)
    dx = torch.full((n, width + pad), float("nan"), dtype=t, device="cuda")
    dtable = torch.full((rows, width + pad), float("nan"), dtype=gt, device="cuda")
    grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width + pad, dtable_stride=width + pad,
                           grad_dtype=gcode, d_dx=ptr(dx), d_dtable=ptr(dtable))
    ws = give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, stream())
    lib.loss_grad_device(args, grads, stream())
    torch.cuda.synchronize()
    del ws
    want = Want(xd[:, :width], td[:, :width], tg, scale, dl)
    within(lse, want.lse.cpu(), want.E.cpu(), "lse")
    within(loss, want.loss.cpu(), 2 * want.E.cpu(), "loss")
    assert dx[:, width:].isnan().all() and dtable[:, width:].isnan().all()
    return (dx[:, :width], dtable[:, :width]), want


@pytest.mark.gpu
@pytest.mark.parametrize("case,dtype,grad", [
    # straight to LDS, both results straight from the products, or from their sums
    ((2000, 1100, 320, 8), "bf16", "bf16"), ((1000, 2300, 512, 8), "bf16", "bf16"),
    ((4100, 2500, 64, 16), "bf16", "bf16"), ((300, 700, 64, 8), "bf16", "bf16"),
    # copied first for the gradient, for the loss too, in pieces
    ((3000, 3000, 72, 3), "bf16", "bf16"), ((6000, 4300, 83, 5), "bf16", "bf16"),
    ((6000, 4300, 83, 45), "bf16", "bf16"), ((513, 4300, 840, 56), "bf16", "bf16"),
    ((600, 66000, 700, 1), "bf16", "bf16"), ((2100, 2500, 128, 1), "bf16", "bf16"),
    # through registers, tiles of 128 and 64, one and more terms
    ((2000, 3000, 40, 24), "f32", "f32"), ((1500, 2500, 7, 1), "bf16", "f32"),
    ((2100, 1200, 95, 33), "bf16", "f32"), ((130, 90, 129, 7), "f32", "bf16"),
    ((30, 3000, 71, 9), "bf16", "bf16")])
def test_nothing_beside_rows_is_read_or_written(lib, case, dtype, grad):  # noqa: F811
    n, rows, width, pad = case
    t, code, gen, x, table, target, scale = inputs(case, dtype)
    got, want = gradients(lib, case, x, table, target, scale, rnd(gen, n), pad, grad)
    own = want.off(22 if dtype == "f32" else 8)[0]
    by_table = want.off(22 if dtype == "f32" else 16 if grad == "f32" else 8)[1]
    within(got[0], want.dx.cpu(), own.cpu(), "dx")
    within(got[1], want.dtable.cpu(), by_table.cpu(), "dtable")


# ------------------------------------------------------------ sizes and refusals

@pytest.mark.parametrize("width", [64, 65, 256, 320])
@pytest.mark.parametrize("dtype", [capi.F32, capi.BF16])
def test_workspaces_go_by_sizes_and_types_alone(width, dtype):
    L = capi.Lib()
    for tokens in (1, 64, 65, 300, 511, 512, 3000, 16384):
        for rows in (1, 255, 5003, 70000, 262144):
            sizes = {(L.loss_workspace_bytes(a), L.loss_grad_workspace_bytes(a, good_grads()))
                     for a in (good(tokens=tokens, rows=rows, width=width, dtype=dtype, x_stride=xs,
                                    table_stride=ts, d_x=p)
                               for xs, ts, p in ((0, 0, None), (width, width, A), (width + 1, width, A),
                                                 (width, width + 3, A + 4), (1 << 24, 1 << 24, A)))}
            assert len(sizes) == 1, (tokens, rows)


@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_scales_whose_logits_have_no_number_are_refused(scale):
    """Logits are found in powers of two: scale * log2(e) has to be a number."""
    L = capi.Lib()
    for call in (lambda a: L.loss_device(a), lambda a: L.loss_grad_device(a, good_grads())):
        with pytest.raises(capi.NsfpsError) as e:
            call(good(scale=scale))
        assert e.value.status == EINVAL and "scale" in str(e.value)
