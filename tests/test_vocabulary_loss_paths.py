"""The vocabulary loss along the paths that its sizes choose: tiles straight to
LDS with the tokens in registers or not, through registers in two sizes, rows
of fewer than eight values, several pieces, products with and without splits;
scales of either sign; offsets beyond 32 bits; graphs and streams.  References
in 64 bits on the device; the tolerances are those of test_vocabulary_loss.py."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import within
from test_sequence import DTYPES, F64, lib, ptr, rnd, stream  # noqa: F401
from test_vocabulary_loss import Want, args_of, give, inputs


def both(lib, case, dtype, grad, scale=None, dloss=None):  # noqa: F811
    """Loss and gradient: (got, want)."""
    n, rows, width, pad = case
    t, code, gen, x, table, target, ordinary = inputs(case, dtype)
    scale = ordinary if scale is None else scale
    dloss = rnd(gen, n) if dloss is None else dloss
    gt, gcode = DTYPES[grad]
    xd, td = torch.zeros(n, width + pad, dtype=t), torch.zeros(rows, width + pad, dtype=t)
    xd[:, :width], td[:, :width] = x, table
    xd, td, tg, dl = xd.cuda(), td.cuda(), target.cuda(), dloss.cuda()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    args = args_of(case, code, xd, td, tg, scale, loss, lse)
    dx = torch.full((n, width), float("nan"), dtype=t, device="cuda")
    dtable = torch.full((rows, width), float("nan"), dtype=gt, device="cuda")
    grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width, dtable_stride=width, grad_dtype=gcode,
                           d_dx=ptr(dx), d_dtable=ptr(dtable))
    ws = give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, stream())
    lib.loss_grad_device(args, grads, stream())
    torch.cuda.synchronize()
    del ws
    return (loss, lse, dx, dtable), Want(xd[:, :width], td[:, :width], tg, scale, dl)


def check(got, want, dtype, grad):
    own = want.off(22 if dtype == "f32" else 8)[0]
    by_table = want.off(22 if dtype == "f32" else 16 if grad == "f32" else 8)[1]
    within(got[1], want.lse.cpu(), want.E.cpu(), "lse")
    within(got[0], want.loss.cpu(), 2 * want.E.cpu(), "loss")
    within(got[2], want.dx.cpu(), own.cpu(), "dx")
    within(got[3], want.dtable.cpu(), by_table.cpu(), "dtable")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("case", [
    # whole 64s: one to four stages in registers, then both from LDS
    (300, 700, 64, 0), (513, 300, 128, 0), (700, 129, 192, 0), (256, 1500, 256, 0),
    (257, 600, 320, 0), (300, 257, 512, 8), (1000, 130, 384, 0),
    # the same with fewer tokens than whole tiles are worth
    (3, 900, 256, 0), (130, 64, 320, 0),
    # through registers: large tiles, narrow rows, widths around a stage's ends
    (2000, 3000, 40, 0), (3000, 2000, 72, 3), (300, 500, 1, 0), (129, 300, 3, 0), (1500, 2500, 7, 1),
    (200, 300, 8, 0), (200, 300, 9, 0), (64, 65, 65, 0), (70, 70, 127, 0), (2100, 1200, 95, 0),
    # the gradient straight to LDS too: every width of a product's tiles
    (2000, 1100, 320, 0), (1000, 2300, 512, 8), (900, 3100, 256, 0), (4100, 2500, 64, 0),
    (2100, 2500, 128, 0), (257, 6000, 384, 0),
    # few rows, few tokens
    (1000, 1, 64, 0), (1000, 5, 33, 0), (1, 3000, 100, 0), (2, 2, 2, 0)])
def test_every_path(lib, case, dtype, grad):  # noqa: F811
    got, want = both(lib, case, dtype, grad)
    check(got, want, dtype, grad)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [256, 128, 64])
def test_pieces_straight_to_lds(lib, width):  # noqa: F811
    """More tokens than one piece of d holds rows for, the last piece short."""
    case = (66000, 2300, width, 0)
    got, want = both(lib, case, "bf16", "bf16")
    check(got, want, "bf16", "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("width", [64, 128, 192, 256])
def test_long_sweeps(lib, width):  # noqa: F811
    """Tokens and rows of 129 and 33 tiles, the last ones short: a workgroup's tokens stay in
    registers over eight tiles and more."""
    got, want = both(lib, (16500, 4100, width, 0), "bf16", "bf16")
    check(got, want, "bf16", "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("case", [
    # rows copied for the gradient; for the loss too; several pieces of the table in
    # the loss, the last one short; several in the gradient
    (3000, 3000, 72, 3), (6000, 4300, 83, 5), (513, 4300, 840, 0), (600, 66000, 700, 1),
    (66000, 2300, 33, 0)])
def test_rows_copied_first(lib, case):  # noqa: F811
    """Many tokens with rows that cannot go straight to LDS; NaN beside the rows."""
    got, want = both(lib, case, "bf16", "bf16")
    check(got, want, "bf16", "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("width", [128, 320])
def test_addresses_do_not_matter(lib, width):  # noqa: F811
    """Rows of whole 64s at odd addresses, copied first, give the bits of aligned ones,
    in a workspace of the same size; rows that count for nothing hold NaN."""
    n, rows = 4000, 4100
    case = (n, rows, width, 0)
    t, code, gen, x, table, target, scale = inputs(case, "bf16")
    dloss = rnd(gen, n).cuda()
    x[(target < 0) | (target >= rows)] = float("nan")
    results = []
    for shift in (0, 1):
        xd, td = (torch.empty(v.numel() + 8, dtype=t, device="cuda")[shift:shift + v.numel()]
                  .view(v.shape).copy_(v) for v in (x, table))
        tg = target.cuda()
        loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
        args = args_of(case, code, xd, td, tg, scale, loss, lse)
        dx, dtable = torch.empty_like(xd), torch.empty_like(td)
        grads = capi.LossGrads(d_dloss=ptr(dloss), dx_stride=width, dtable_stride=width,
                               grad_dtype=code, d_dx=ptr(dx), d_dtable=ptr(dtable))
        sizes = lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)
        ws = give(args, max(sizes))
        lib.loss_device(args, stream())
        lib.loss_grad_device(args, grads, stream())
        torch.cuda.synchronize()
        results.append((sizes, loss, dx, dtable))
        del ws
    assert results[0][0] == results[1][0]
    for a, b in zip(results[0][1:], results[1][1:]):
        assert torch.equal(a, b) and not a.isnan().any()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.7, 0.0, 3.0])
@pytest.mark.parametrize("case,dtype", [((300, 700, 64, 0), "bf16"), ((300, 333, 320, 0), "bf16"),
                                        ((2100, 2500, 128, 0), "bf16"),
                                        ((90, 200, 50, 0), "f32"), ((90, 200, 50, 0), "bf16")])
def test_scales(lib, case, dtype, scale):  # noqa: F811
    got, want = both(lib, case, dtype, dtype, scale=scale)
    check(got, want, dtype, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(300, 700, 64, 0), (2100, 2500, 128, 0)])
@pytest.mark.parametrize("weights", ["alike", "first is zero", "tiny", "huge", "none"])
def test_weights_of_the_tokens(lib, case, weights):  # noqa: F811
    """d is held relative to one token's weight, whichever that is."""
    n = case[0]
    dloss = torch.full((n,), 1.0 / 300)
    if weights == "first is zero":
        dloss[:100] = 0
    elif weights == "tiny":
        dloss *= 1e-12
        dloss[7] = 1e-3
    elif weights == "huge":
        dloss[1::2] *= 1e12
    elif weights == "none":
        dloss[:] = 0
    got, want = both(lib, case, "bf16", "bf16", dloss=dloss)
    check(got, want, "bf16", "bf16")
    if weights == "alike":
        # a rounding of 8 bits each of the results, with d's own below it: the norm of
        # the difference is at most 2^-8 of the result's
        for g, w in ((got[2], want.dx), (got[3], want.dtable)):
            assert (g.to(F64) - w).norm() <= 2.0 ** -8 * w.norm()


@pytest.mark.gpu
def test_beyond_32_bit_offsets(lib):  # noqa: F811
    """A table above 2^32 elements: its last rows are read and their gradient
    written where they are."""
    rows, width, n = (1 << 31) // 4096 + 9, 8192, 3
    table = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    table[-1], table[3] = 2.0 ** -6, -(2.0 ** -6)
    x = torch.ones(n, width, dtype=torch.bfloat16, device="cuda") * 2.0 ** -4
    target = torch.tensor([rows - 1, 3, -1], dtype=torch.int32, device="cuda")
    loss, lse, one = (torch.ones(n, device="cuda") for _ in range(3))
    args = args_of((n, rows, width, 0), capi.BF16, x, table, target, 1.0, loss, lse)
    dx, dtable = torch.empty_like(x), torch.empty_like(table)
    grads = capi.LossGrads(d_dloss=ptr(one), dx_stride=width, dtable_stride=width,
                           grad_dtype=capi.BF16, d_dx=ptr(dx), d_dtable=ptr(dtable))
    ws = give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, stream())
    lib.loss_grad_device(args, grads, stream())
    # logits: 8 and -8 at the two rows, 0 elsewhere
    z = torch.zeros(rows, dtype=F64)
    z[-1], z[3] = 8.0, -8.0
    want = torch.logsumexp(z, 0)
    E = 2.0 ** -19 * (8 + want + 1)
    assert (lse.cpu().to(F64) - want).abs().max() <= E
    assert abs(loss[0].item() - (want - 8).item()) <= 2 * E and loss[2] == 0
    assert abs(loss[1].item() - (want + 8).item()) <= 2 * E
    p = torch.exp(z - want)
    for v in (rows - 1, 3, 0, rows - 2):
        d = 2 * p[v] - float(v in (rows - 1, 3))
        got = dtable[v].cpu().to(F64)
        size = (2 * p[v] + 1.0 * (v in (rows - 1, 3))) * 2.0 ** -4
        assert (got - d * 2.0 ** -4).abs().max() <= (2.0 ** -7 + 4 * E) * size
    del ws


def calls(lib, gen, cases):  # noqa: F811
    """One loss and gradient of each case on new inputs: (call, outputs)."""
    held, outs, todo = [], [], []
    for case, dtype in cases:
        n, rows, width, _ = case
        t, code = DTYPES[dtype]
        x, table = rnd(gen, n, width, dtype=t).cuda(), rnd(gen, rows, width, dtype=t).cuda()
        target = torch.randint(-1, rows, (n,), generator=gen, dtype=torch.int32).cuda()
        dl = rnd(gen, n).cuda()
        loss, lse = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        dx, dtable = torch.zeros_like(x), torch.zeros_like(table)
        args = args_of(case, code, x, table, target, 0.3, loss, lse)
        grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width, dtable_stride=width,
                               grad_dtype=code, d_dx=ptr(dx), d_dtable=ptr(dtable))
        ws = give(args, max(lib.loss_workspace_bytes(args),
                            lib.loss_grad_workspace_bytes(args, grads)))
        held.append((x, table, target, dl, ws))
        outs += [loss, lse, dx, dtable]
        todo.append((args, grads))

    def call():
        for args, grads in todo:
            lib.loss_device(args, stream())
            lib.loss_grad_device(args, grads, stream())
        return held
    return call, outs


MANY = [((300, 700, 256, 0), "bf16"), ((2000, 2200, 256, 0), "bf16"), ((2000, 2200, 65, 0), "bf16"),
        ((300, 500, 50, 0), "bf16"), ((150, 400, 33, 0), "f32"),
        ((66000, 1100, 64, 0), "bf16")]


@pytest.mark.gpu
@pytest.mark.parametrize("stride", [(1 << 23) - 8, 1 << 23])
def test_rows_far_apart(lib, stride):  # noqa: F811
    """Rows of x and of the table as far apart as tiles straight to LDS take them, and
    one step farther: a tile's rows span 2 GB and more."""
    case = (130, 150, 128, 0)
    n, rows, width, _ = case
    _, code, gen, x, table, target, scale = inputs(case, "bf16")
    wide = torch.empty(rows, stride, dtype=torch.bfloat16, device="cuda")
    far = torch.empty(n, stride, dtype=torch.bfloat16, device="cuda")
    wide[:, :width], far[:, :width] = table.cuda(), x.cuda()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    tg = target.cuda()
    args = args_of(case, code, far, wide, tg, scale, loss, lse)
    ws = give(args, lib.loss_workspace_bytes(args))
    lib.loss_device(args, stream())
    torch.cuda.synchronize()
    want = Want(x, table, target, scale)
    within(lse, want.lse, want.E, "lse")
    within(loss, want.loss, 2 * want.E, "loss")
    del ws


@pytest.mark.gpu
def test_graph_replays_equal_eager_calls(lib):  # noqa: F811
    call, outs = calls(lib, torch.Generator().manual_seed(2), MANY)
    call()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        for o in outs:
            o.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
        call()  # the program's own eager work between replays
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.gpu
def test_calls_on_other_streams(lib):  # noqa: F811
    gen = torch.Generator().manual_seed(3)
    sets = [calls(lib, gen, MANY) for _ in range(2)]
    wants = []
    for call, outs in sets:
        call()
        torch.cuda.synchronize()
        wants.append([o.clone() for o in outs])
        for o in outs:
            o.fill_(3.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for (call, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                call()
    torch.cuda.synchronize()
    for (_, outs), want in zip(sets, wants):
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("case,copied", [((6000, 4300, 83, 5), True), ((513, 4300, 840, 0), True),
                                         ((600, 66000, 700, 1), True), ((500, 4300, 840, 0), False),
                                         ((3000, 3000, 72, 3), False)])
def test_sizes_reach_the_copies(case, copied):
    """What test_rows_copied_first is for: the loss's workspace holds the tokens' copy
    and a piece's of the table, or does not."""
    n, rows, width, pad = case
    args = capi.LossArgs(tokens=n, rows=rows, width=width, dtype=capi.BF16, x_stride=width + pad,
                         table_stride=width + pad)
    copies = 2 * (n + min(rows, 65536)) * ((width + 63) // 64 * 64)
    assert (capi.Lib().loss_workspace_bytes(args) >= copies) == copied
