"""What lies beside the vocabulary loss's rows is neither read nor written, whichever
way the sizes choose; and its workspace goes by sizes and types."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import within
from test_sequence import A, DTYPES, lib, ptr, rnd, stream  # noqa: F401
from test_vocabulary_loss import Want, args_of, give, good, good_grads, inputs


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
