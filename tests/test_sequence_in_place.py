"""Norms, dropout and the vocabulary loss with an output over an input.  Norms and
dropout take every value before they write its place, so an output may be an input's
very rows; anything else that the strides show to overlap is refused, as is all of it
for the loss, whose products read rows again after others are written."""

import random

import pytest
import torch

import test_dropout
import test_head_norm
import test_vocabulary_loss
from ns_fps_amd import capi
from test_head_norm import EPS
from test_sequence import A, DTYPES, EINVAL, laid_out, lib, ptr, rnd, rows, stream, \
    workspace  # noqa: F401

FAR = [A + (k << 30) for k in range(1, 9)]


def refused(call, *args):
    with pytest.raises(capi.NsfpsError) as e:
        call(*args)
    assert e.value.status == EINVAL and "overlap" in str(e.value)


def taken(call, *args):
    """Every check passed: the next one is for a device (a taken call would run)."""
    if capi.Lib().device_count():
        pytest.skip("a taken call would run")
    with pytest.raises(capi.NsfpsError) as e:
        call(*args)
    assert "no HIP device" in str(e.value)


# ----------------------------------------------------------------------- norms

def norm(**kw):
    """Rows of 2 + 1 heads of 8, float32, each tensor on its own."""
    return test_head_norm.good(**{**dict(q=(FAR[0], 128, 16), k=(FAR[1], 64, 8),
                                         q_out=(FAR[2], 128, 16), k_out=(FAR[3], 64, 8)), **kw})


def norm_grads(**kw):
    return test_head_norm.good_grads(**{**dict(dq_out=(FAR[4], 128, 16), dk_out=(FAR[5], 64, 8),
                                               dq=(FAR[6], 128, 16), dk=(FAR[7], 64, 8)), **kw})


SHARED = (FAR[0], 24 * 8, 24)        # q ahead of k in rows of 24
BEHIND = (FAR[0] + 16 * 4, 24 * 8, 24)


@pytest.mark.parametrize("change", [
    {}, dict(q_out=(FAR[0], 128, 16)), dict(k_out=(FAR[1], 64, 8)),
    dict(q=SHARED, k=BEHIND), dict(q=SHARED, k=BEHIND, q_out=SHARED, k_out=BEHIND),
    dict(q_out=SHARED, k_out=BEHIND, q=(FAR[2], 128, 16)),
    # one sequence, whose batch stride says nothing; one token, whose row stride says nothing
    dict(batch=1, q_out=(FAR[0], 999, 16)), dict(length=1, q_out=(FAR[0], 128, 77))])
def test_norms_in_place_are_taken(change):
    taken(capi.Lib().norm_device, norm(**change))


@pytest.mark.parametrize("change", [
    dict(q_out=(FAR[0] + 4, 128, 16)), dict(q_out=(FAR[0] - 4, 128, 16)),
    dict(q_out=(FAR[0] + 16 * 4, 128, 16)),                   # a token later
    dict(q_out=(FAR[0] + 15 * 4, 128, 16)), dict(q_out=(FAR[0], 16 * 9, 18)),
    dict(q=(FAR[0], 0, 0), q_out=(FAR[0], 128, 16)),          # one row for all tokens
    dict(q_out=(FAR[1], 128, 16)), dict(k_out=(FAR[0], 64, 8)),
    dict(q=SHARED, k=BEHIND, q_out=BEHIND, k_out=SHARED),     # exchanged
    dict(q_out=SHARED, k_out=(FAR[0] + 15 * 4, 24 * 8, 24)),  # the outputs over each other
    dict(k_out=(FAR[2], 64, 8))])
def test_norms_over_something_else_are_refused(change):
    refused(capi.Lib().norm_device, norm(**change))


@pytest.mark.parametrize("change", [
    {}, dict(dq=(FAR[0], 128, 16)), dict(dq=(FAR[4], 128, 16)), dict(dk=(FAR[1], 64, 8)),
    dict(dk=(FAR[5], 64, 8)), dict(dq=(FAR[0], 128, 16), dk=(FAR[5], 64, 8)),
    dict(dq=SHARED[:1] + (24 * 8, 24), dk=BEHIND)])
def test_norm_gradients_in_place_are_taken(change):
    args = dict(q=SHARED, k=BEHIND) if change.get("dk") == BEHIND else {}
    taken(capi.Lib().norm_grad_device, norm(**args), norm_grads(**change))


@pytest.mark.parametrize("change", [
    dict(dq=(FAR[0] + 4, 128, 16)), dict(dq=(FAR[4] + 64, 128, 16)), dict(dq=(FAR[1], 128, 16)),
    dict(dq=(FAR[5], 128, 16)), dict(dk=(FAR[0], 64, 8)), dict(dk=(FAR[4], 64, 8)),
    dict(dk=(FAR[6], 64, 8)), dict(dk=(FAR[6] + 60, 64, 8))])
def test_norm_gradients_over_something_else_are_refused(change):
    refused(capi.Lib().norm_grad_device, norm(), norm_grads(**change))


# batch, length, q_heads, k_heads, head_dim, rotary_dim, neighbours, layout
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", [(2, 65, 3, 3, 33, 32, 1, "odd"), (3, 70, 1, 2, 64, 32, 1, "padded"),
                                  (2, 9000, 5, 3, 64, 64, 0, "plain"), (1, 33, 2, 1, 255, 100, 0, "odd"),
                                  (1, 130, 4, 4, 128, 128, 1, "swapped")])
def test_norms_in_place(lib, case, dtype):  # noqa: F811
    """The same bits as into memory of its own; the gradient over x and over g."""
    t, code, gen, x, w, freq, lens, pos = test_head_norm.inputs(case, dtype)
    how = case[-1]
    args, keep = test_head_norm.on_device(case, code, x, w, freq, lens, pos)
    out = {k: laid_out(torch.full_like(v, 7.0).cuda(), how) for k, v in x.items()}
    args.q_out, args.k_out = rows(out["q"]), rows(out["k"])
    lib.norm_device(args, stream())
    want = {k: v.clone() for k, v in out.items()}
    over = {k: laid_out(v.cuda(), how) for k, v in x.items()}
    args.q, args.k = args.q_out, args.k_out = rows(over["q"]), rows(over["k"])
    lib.norm_device(args, stream())
    assert all(torch.equal(over[k], want[k]) for k in "qk")

    dy = {k: rnd(gen, *v.shape, dtype=t) for k, v in x.items()}
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    results = []
    for place in ("apart", "x", "g"):
        X, G, O = ({k: laid_out(v.cuda(), how) for k, v in s.items()} for s in (x, dy, x))
        to = {"apart": O, "x": X, "g": G}[place]
        dw = {k: torch.full((case[4],), 9.0, device="cuda") for k in "qk"}
        args.q, args.k = rows(X["q"]), rows(X["k"])
        lib.norm_grad_device(args, capi.NormGrads(
            dq_out=rows(G["q"]), dk_out=rows(G["k"]), dq=rows(to["q"]), dk=rows(to["k"]),
            d_dq_weight=ptr(dw["q"]), d_dk_weight=ptr(dw["k"])), stream())
        results.append([to["q"], to["k"], dw["q"], dw["k"]])
    for got in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got, results[0]))
    del ws, keep


# --------------------------------------------------------------------- dropout

def dropout(**kw):
    return test_dropout.good(**{**dict(x=(FAR[0], 64, 8), residual=(FAR[1], 64, 8),
                                       y=(FAR[2], 64, 8)), **kw})


@pytest.mark.parametrize("change", [{}, dict(y=(FAR[0], 64, 8)), dict(y=(FAR[1], 64, 8)),
                                    dict(x=(FAR[1], 64, 8), y=(FAR[1], 64, 8)),
                                    dict(x=(FAR[0], 128, 16), y=(FAR[0] + 32, 128, 16))])
def test_dropout_in_place_is_taken(change):
    taken(capi.Lib().dropout_device, dropout(**change))


@pytest.mark.parametrize("change", [
    dict(y=(FAR[0] + 4, 64, 8)), dict(y=(FAR[0] + 32, 64, 8)), dict(y=(FAR[1] - 28, 64, 8)),
    dict(residual=(FAR[1], 0, 0), y=(FAR[1], 64, 8)), dict(x=(FAR[0], 0, 8), y=(FAR[0], 64, 8))])
def test_dropout_over_something_else_is_refused(change):
    refused(capi.Lib().dropout_device, dropout(**change))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("channels,how", [(640, "plain"), (321, "odd"), (64, "padded")])
def test_dropout_in_place(lib, channels, how, dtype):  # noqa: F811
    t, code = DTYPES[dtype]
    case, lens = (3, 130, channels, how), torch.tensor([130, 0, 77], dtype=torch.int32).cuda()
    gen = torch.Generator().manual_seed(channels)
    x, r = (rnd(gen, 3, 130, channels, dtype=t) for _ in range(2))
    seed = torch.tensor([11, 12], dtype=torch.int64).cuda()
    results = []
    for place in ("apart", "x", "residual"):
        X, R, Y = (laid_out(v.cuda(), how) for v in (x, r, x))
        to = {"apart": Y, "x": X, "residual": R}[place]
        test_dropout.call(lib, case, code, X, R, to, 0.3, seed, lens)
        results.append(to)
    assert torch.equal(results[1], results[0]) and torch.equal(results[2], results[0])


# ------------------------------------------------------------------------ loss

def loss(**kw):
    """4 tokens, 4 rows of 8, float32."""
    return test_vocabulary_loss.good(**{**dict(d_x=FAR[0], d_table=FAR[1], d_targets=FAR[2],
                                               d_loss=FAR[3], d_lse=FAR[4]), **kw})


def loss_grads(**kw):
    return test_vocabulary_loss.good_grads(**{**dict(d_dloss=FAR[5], d_dx=FAR[6], d_dtable=FAR[7]),
                                              **kw})


def test_losses_apart_are_taken():
    taken(capi.Lib().loss_device, loss())


def test_loss_gradients_apart_are_taken():
    L = capi.Lib()
    taken(L.loss_grad_device, loss(), loss_grads())
    # dx beside x in rows of 16, the table's gradient of another type behind the table
    taken(L.loss_grad_device, loss(x_stride=16), loss_grads(d_dx=FAR[0] + 32, dx_stride=16))
    taken(L.loss_grad_device, loss(), loss_grads(d_dtable=FAR[1] + 4 * 4 * 8, grad_dtype=capi.BF16))


@pytest.mark.parametrize("change", [
    dict(d_loss=FAR[4]), dict(d_loss=FAR[4] + 12), dict(d_lse=FAR[3] + 4), dict(d_loss=FAR[2]),
    dict(d_lse=FAR[2] + 8), dict(d_loss=FAR[0]), dict(d_lse=FAR[1] + 124)])
def test_losses_over_something_else_are_refused(change):
    refused(capi.Lib().loss_device, loss(**change))


@pytest.mark.parametrize("change", [
    dict(d_dx=FAR[0]), dict(d_dx=FAR[0] + 4), dict(d_dx=FAR[1] + 96), dict(d_dx=FAR[7]),
    dict(d_dtable=FAR[1]), dict(d_dtable=FAR[0] - 124), dict(d_dtable=FAR[6] + 64),
    dict(d_dtable=FAR[1], grad_dtype=capi.BF16), dict(d_dtable=FAR[1] + 126, grad_dtype=capi.BF16),
    dict(d_dx=FAR[2]), dict(d_dx=FAR[4]), dict(d_dtable=FAR[5])])
def test_loss_gradients_over_something_else_are_refused(change):
    refused(capi.Lib().loss_grad_device, loss(), loss_grads(**change))


def bytes_of(p, rows, stride, width):
    return {p + r * stride + c for r in range(rows) for c in range(width)}


def test_every_pair_of_spans_is_told():
    """Random small matrices against their bytes: all overlaps are refused where one
    side has no gaps or the strides are alike, and none is refused that is not there."""
    rng, L, told = random.Random(11), capi.Lib(), []
    for _ in range(2000):
        tokens, rows_, width = rng.randint(1, 4), rng.randint(1, 4), rng.randint(1, 4)
        xs, ts = width + rng.choice([0, 0, 1, 3]), width + rng.choice([0, 0, 2, 5])
        dxs = rng.choice([width, xs, width + 2])
        at = FAR[0] + 4 * rng.randint(-20, 20)
        args = loss(tokens=tokens, rows=rows_, width=width, x_stride=xs, table_stride=ts)
        grads = loss_grads(d_dx=at, dx_stride=dxs, dtable_stride=width)
        met = bool(bytes_of(at, tokens, 4 * dxs, 4 * width) & bytes_of(FAR[0], tokens, 4 * xs, 4 * width))
        sure = dxs == width or xs in (width, dxs) or tokens == 1
        told.append(met)
        if met and sure:
            refused(L.loss_grad_device, args, grads)
        elif not met and L.device_count() == 0:
            with pytest.raises(capi.NsfpsError) as e:
                L.loss_grad_device(args, grads)
            assert "no HIP device" in str(e.value)
    assert 300 < sum(told) < 1700


def test_every_pair_of_rows_of_two_widths_is_told():
    """q's rows are wider than k's: k_out against q, element by element."""
    rng, L, told = random.Random(12), capi.Lib(), []
    for _ in range(2000):
        batch, length, d = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 3)
        hq, hk = rng.randint(1, 3), rng.randint(1, 3)
        near = max(hq, hk) * d + rng.randint(0, 6)
        far = (length - 1) * near + max(hq, hk) * d + rng.randint(0, 6)
        shift = rng.randint(-50, 50)
        q, k_out = (FAR[0], far, near), (FAR[0] + 4 * shift, far, near)

        def elements(p, width):
            return {p // 4 + b * far + t * near + c for b in range(batch) for t in range(length)
                    for c in range(width)}
        args = test_head_norm.good(batch=batch, length=length, q_heads=hq, k_heads=hk, head_dim=d,
                                   rotary_dim=0, q=q, k=(FAR[1], far, near), q_out=(FAR[2], far, near),
                                   k_out=k_out)
        told.append(bool(elements(q[0], hq * d) & elements(k_out[0], hk * d)))
        if told[-1]:
            refused(L.norm_device, args)
        elif L.device_count() == 0:
            with pytest.raises(capi.NsfpsError) as e:
                L.norm_device(args)
            assert "no HIP device" in str(e.value)
    assert 300 < sum(told) < 1700
