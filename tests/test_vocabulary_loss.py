"""The vocabulary loss and its gradient against 64 bits; and the refusals.

Tolerances.  With S the largest sum of a token's |x| |table| over the
vocabulary, times |scale|: a logit's sum is off by 2^-19 S (a few dozen
additions of 32 products each, at 2^-23 of the sum so far, and what three
bfloat16 terms of a float32 value leave out, 2^-22).  The exponents' roundings
(2^-23 of a logit) and those of the logarithm's sum come on top: lse is off by
E = 2^-19 (S + |lse| + 1), a loss by 2 E.  An exponential is off by 2 E + 2^-18
of itself, and enters the products rounded to 8, 16 or 24 bits: 2^-8, 2^-16,
2^-22 of a term; the sums of the products add 2^-18 of their terms' sizes, and a
bfloat16 result is rounded once more, by 2^-8 of itself at most."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import within
from test_sequence import A, DTYPES, EINVAL, EUNSUPPORTED, F64, lib, ptr, rnd, stream, \
    workspace  # noqa: F401

# tokens, rows, width, padding of rows
CASES = [(1, 1, 1, 0), (1, 64, 16, 0), (7, 300, 33, 0), (130, 129, 64, 0), (257, 1000, 100, 4),
         (64, 5000, 256, 0), (300, 70, 383, 3), (1000, 4096, 64, 8), (129, 257, 640, 0),
         (5, 2000, 1024, 0), (128, 128, 128, 0), (2, 40000, 20, 4), (900, 3, 24, 0)]


def padded(t, pad):
    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype)
    wide[:, :t.shape[1]] = t
    return wide.cuda()


def inputs(case, dtype):
    n, rows, width, pad = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(n + 7 * rows + 31 * width)
    x, table = rnd(gen, n, width, dtype=t), rnd(gen, rows, width, dtype=t)
    target = torch.randint(0, rows, (n,), generator=gen, dtype=torch.int32)
    target[-1] = rows - 1
    out = torch.rand(n, generator=gen) < 0.2
    if n > 5:
        out[:5] = torch.tensor([False, True, True, True, True])
        target[1:5] = torch.tensor([-1, rows, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)
    target = torch.where(out & (target >= 0) & (target < rows), -1, target)
    return t, code, gen, x, table, target, 2.0 / width ** 0.5


def args_of(case, code, x, table, target, scale, loss, lse):
    n, rows, width, _ = case
    return capi.LossArgs(tokens=n, rows=rows, width=width, dtype=code, scale=scale,
                         x_stride=x.stride(0), table_stride=table.stride(0), d_x=ptr(x),
                         d_table=ptr(table), d_targets=ptr(target), d_loss=ptr(loss), d_lse=ptr(lse))


def give(args, nbytes):
    ws = workspace(nbytes)
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    return ws


class Want:
    """In 64 bits, and the sizes that the tolerances go by."""

    def __init__(self, x, table, target, scale, dloss=None):
        x, table = x.to(F64), table.to(F64)
        rows = table.shape[0]
        scale = float(torch.tensor(scale, dtype=torch.float32))
        self.counts = (target >= 0) & (target < rows)
        z = x @ table.T * scale
        self.lse = torch.logsumexp(z, 1)
        at = torch.where(self.counts, target, 0).long()[:, None]
        self.loss = torch.where(self.counts, self.lse - z.gather(1, at)[:, 0], 0.0)
        S = (x.abs() @ table.abs().T).amax(1) * abs(scale)
        self.E = 2.0 ** -19 * (S + self.lse.abs() + 1)
        if dloss is not None:
            p = torch.exp(z - self.lse[:, None])
            weight = torch.where(self.counts, dloss.to(F64) * scale, 0.0)[:, None]
            d = p * weight
            sizes = d.abs() * (2 * self.E[:, None] + 2.0 ** -18)
            d.scatter_add_(1, at, -weight)
            sizes += d.abs() * 2.0 ** -18
            x = torch.where(self.counts[:, None], x, 0.0)
            self.dx, self.dtable = d @ table, d.T @ x
            self.off = lambda bits: ((sizes + d.abs() * 2.0 ** -bits) @ table.abs(),
                                     (sizes + d.abs() * 2.0 ** -bits).T @ x.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_loss(lib, case, dtype):  # noqa: F811
    n, rows, width, pad = case
    t, code, gen, x, table, target, scale = inputs(case, dtype)
    xd, td, tg = padded(x, pad), padded(table, pad), target.cuda()
    loss, lse = (torch.full((n,), float("nan"), device="cuda") for _ in range(2))
    args = args_of(case, code, xd, td, tg, scale, loss, lse)
    runs = []
    for _ in range(2):
        ws = give(args, lib.loss_workspace_bytes(args))
        lib.loss_device(args, stream())
        runs.append((loss.clone(), lse.clone()))
        del ws
    want = Want(x, table, target, scale)
    within(runs[0][1], want.lse, want.E, "lse")
    within(runs[0][0], want.loss, 2 * want.E, "loss")
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert runs[0][0].cpu()[~want.counts].eq(0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                        ("f32", "bf16")])
@pytest.mark.parametrize("case", CASES)
def test_loss_gradient(lib, case, dtype, grad):  # noqa: F811
    n, rows, width, pad = case
    t, code, gen, x, table, target, scale = inputs(case, dtype)
    gt, gcode = DTYPES[grad]
    dloss = rnd(gen, n)
    want = Want(x, table, target, scale, dloss)
    held = x.clone()
    held[~want.counts] = float("nan")  # a row that counts for nothing may hold anything
    xd, td, tg, dl = padded(held, pad), padded(table, pad), target.cuda(), dloss.cuda()
    lse = want.lse.float().cuda()
    lse[~want.counts.cuda()] = float("nan")
    args = args_of(case, code, xd, td, tg, scale, None, lse)
    dx = torch.full((n, width + pad), float("nan"), dtype=t, device="cuda")
    dtable = torch.full((rows, width + pad), float("nan"), dtype=gt, device="cuda")
    grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width + pad, dtable_stride=width + pad,
                           grad_dtype=gcode, d_dx=ptr(dx), d_dtable=ptr(dtable))
    runs = []
    for _ in range(2):
        ws = give(args, lib.loss_grad_workspace_bytes(args, grads))
        lib.loss_grad_device(args, grads, stream())
        runs.append((dx[:, :width].clone(), dtable[:, :width].clone()))
        del ws
    own = want.off(22 if dtype == "f32" else 8)[0]
    by_table = want.off(22 if dtype == "f32" else 16 if grad == "f32" else 8)[1]
    within(runs[0][0], want.dx, own, "dx")
    within(runs[0][1], want.dtable, by_table, "dtable")
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    assert torch.isnan(dx[:, width:]).all() and torch.isnan(dtable[:, width:]).all()


@pytest.mark.gpu
def test_loss_gradient_against_differences(lib):  # noqa: F811
    """One direction through x and table: differences of the 64-bit loss."""
    case = (70, 150, 40, 0)
    n, rows, width, _ = case
    t, code, gen, x, table, target, scale = inputs(case, "f32")
    dloss = rnd(gen, n)
    xd, td, tg, dl = x.cuda(), table.cuda(), target.cuda(), dloss.cuda()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    args = args_of(case, code, xd, td, tg, scale, loss, lse)
    dx, dtable = torch.empty_like(xd), torch.empty_like(td)
    grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width, dtable_stride=width, d_dx=ptr(dx),
                           d_dtable=ptr(dtable))
    ws = give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, stream())
    lib.loss_grad_device(args, grads, stream())
    dirs = [torch.randn(v.shape, generator=gen, dtype=F64) for v in (x, table)]
    terms = torch.cat([(g.cpu().to(F64) * d).flatten() for g, d in zip((dx, dtable), dirs)])

    def total(e):
        return (Want(x.to(F64) + e * dirs[0], table.to(F64) + e * dirs[1], target, scale).loss
                * dloss.to(F64)).sum()
    diff = (total(1e-6) - total(-1e-6)) / 2e-6
    assert abs(terms.sum() - diff) <= 2.0 ** -14 * terms.norm() + 1e-5
    del ws


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,rows", [(0, 5), (4, 0), (3, 9)])
def test_empty_vocabularies_and_targets(lib, tokens, rows):  # noqa: F811
    """No vocabulary: lse of -infinity, no loss.  No target: no gradient."""
    width = 12
    x, table = torch.randn(max(tokens, 1), width).cuda(), torch.randn(max(rows, 1), width).cuda()
    target = torch.full((max(tokens, 1),), -1, dtype=torch.int32, device="cuda")
    loss, lse = (torch.full((max(tokens, 1),), 7.0, device="cuda") for _ in range(2))
    args = args_of((tokens, rows, width, 0), capi.F32, x, table, target, 1.0, loss, lse)
    dx, dtable = torch.full_like(x, 7.0), torch.full_like(table, 7.0)
    grads = capi.LossGrads(d_dloss=ptr(loss), dx_stride=width, dtable_stride=width, d_dx=ptr(dx),
                           d_dtable=ptr(dtable))
    ws = give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, stream())
    if tokens:
        assert loss.eq(0).all()
        if not rows:
            assert torch.isneginf(lse).all()
    lib.loss_grad_device(args, grads, stream())
    assert dx[:tokens].eq(0).all() and dtable[:rows].eq(0).all()
    assert dx[tokens:].eq(7).all() and dtable[rows:].eq(7).all()
    del ws


@pytest.mark.gpu
def test_far_logits_and_values_that_are_not_finite(lib):  # noqa: F811
    """Logits of +-2^13 neither overflow nor lose the sum; an infinite or NaN
    row of x spoils its own token's loss only."""
    n, rows, width = 6, 500, 8
    gen = torch.Generator().manual_seed(4)
    x, table = rnd(gen, n, width), rnd(gen, rows, width)
    x[0] *= 2048
    x[1] = 0
    target = torch.arange(n, dtype=torch.int32)
    case = (n, rows, width, 0)
    xd, td, tg = x.cuda(), table.cuda(), target.cuda()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    args = args_of(case, capi.F32, xd, td, tg, 1.0, loss, lse)
    ws = give(args, lib.loss_workspace_bytes(args))
    lib.loss_device(args, stream())
    want = Want(x, table, target, 1.0)
    within(lse, want.lse, want.E, "lse")
    within(loss, want.loss, 2 * want.E, "loss")
    xd[3, 2], xd[4, 0] = float("nan"), float("inf")
    again = loss.clone()
    lib.loss_device(args, stream())
    fine = torch.tensor([0, 1, 2, 5]).cuda()
    assert torch.equal(loss[fine], again[fine])
    assert not torch.isfinite(loss[3:5]).any()
    del ws


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_several_pieces(lib, dtype):  # noqa: F811
    """Sizes whose vocabulary is taken in pieces, the last of them short:
    references in 64 bits on the device."""
    case = (66000, 2500, 24, 0)
    n, rows, width, _ = case
    t, code, gen, x, table, target, scale = inputs(case, dtype)
    dloss = rnd(gen, n)
    xd, td, tg, dl = x.cuda(), table.cuda(), target.cuda(), dloss.cuda()
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    args = args_of(case, code, xd, td, tg, scale, loss, lse)
    dx, dtable = torch.empty_like(xd), torch.empty_like(td)
    grads = capi.LossGrads(d_dloss=ptr(dl), dx_stride=width, dtable_stride=width, grad_dtype=code,
                           d_dx=ptr(dx), d_dtable=ptr(dtable))
    need = lib.loss_grad_workspace_bytes(args, grads)
    more = capi.LossArgs(tokens=n, rows=100000, width=width, dtype=code)
    assert lib.loss_grad_workspace_bytes(more, grads) == need  # pieces, whatever the rows
    ws = give(args, max(lib.loss_workspace_bytes(args), need))
    lib.loss_device(args, stream())
    lib.loss_grad_device(args, grads, stream())
    want = Want(xd, td, tg, scale, dl)
    own, by_table = want.off(22 if dtype == "f32" else 8)
    within(lse, want.lse.cpu(), want.E.cpu(), "lse")
    within(loss, want.loss.cpu(), 2 * want.E.cpu(), "loss")
    within(dx, want.dx.cpu(), own.cpu(), "dx")
    within(dtable, want.dtable.cpu(), by_table.cpu(), "dtable")
    del ws


# -------------------------------------------------------------------- refusals

def good(**kw):
    return capi.LossArgs(**{**dict(tokens=4, rows=4, width=8, scale=1.0, x_stride=8, table_stride=8,
                                   d_x=A, d_table=A, d_targets=A, d_loss=A, d_lse=A, workspace=A,
                                   workspace_bytes=1 << 40), **kw})


def good_grads(**kw):
    return capi.LossGrads(**{**dict(d_dloss=A, dx_stride=8, dtable_stride=8, d_dx=A, d_dtable=A),
                             **kw})


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("change,status", [
    (dict(width=0), EINVAL), (dict(dtype=2), EINVAL), (dict(x_stride=7), EINVAL),
    (dict(table_stride=7), EINVAL), (dict(table_stride=1 << 62), EINVAL), (dict(d_x=None), EINVAL),
    (dict(d_x=A + 2), EINVAL), (dict(d_table=None), EINVAL), (dict(d_targets=A + 2), EINVAL),
    (dict(d_lse=None), EINVAL), (dict(scale=float("inf")), EINVAL),
    (dict(scale=float("nan")), EINVAL), (dict(tokens=1 << 31), EUNSUPPORTED),
    (dict(rows=1 << 31), EUNSUPPORTED),
    (dict(width=65537, x_stride=65537, table_stride=65537), EUNSUPPORTED),
    (dict(workspace=None), EINVAL), (dict(workspace=A + 16), EINVAL),
    (dict(workspace_bytes=16), EINVAL)])
def test_refusals(change, status, grad):
    L = capi.Lib()
    with pytest.raises(capi.NsfpsError) as e:
        if grad:
            L.loss_grad_device(good(**change), good_grads())
        else:
            L.loss_device(good(**change))
    assert e.value.status == status


@pytest.mark.parametrize("change", [
    dict(d_dloss=None), dict(d_dx=None), dict(d_dx=A + 2), dict(d_dtable=None), dict(dx_stride=7),
    dict(dtable_stride=7), dict(dx_stride=1 << 62), dict(grad_dtype=2), dict(d_dtable=A + 2)])
def test_gradients_are_checked(change):
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().loss_grad_device(good(), good_grads(**change))
    assert e.value.status == EINVAL


def test_null_structs_and_empty_calls():
    L = capi.Lib()
    assert L.lib.nsfps_loss_device(None, None) == EINVAL
    assert L.lib.nsfps_loss_grad_device(good(), None, None) == EINVAL
    assert L.lib.nsfps_loss_grad_workspace_bytes(good(), None, None) == EINVAL
    with pytest.raises(capi.NsfpsError):
        L.loss_device(good(d_loss=None))
    L.loss_device(good(tokens=0, d_x=None))
    L.loss_grad_device(good(tokens=0, rows=0, d_x=None, d_table=None), good_grads(d_dx=None))


def test_the_workspace_stays_small():
    """A training batch over a large vocabulary: far below its logits."""
    L = capi.Lib()
    args = capi.LossArgs(tokens=16384, rows=262144, width=256, dtype=capi.BF16)
    logits = 2 * 16384 * 262144
    assert L.loss_workspace_bytes(args) < logits // 16
    assert L.loss_grad_workspace_bytes(args, capi.LossGrads(grad_dtype=capi.BF16)) < logits // 16
