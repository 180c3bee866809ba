"""Rows past a sequence's end: zeros in every gradient, whatever the sequence
holds, and nothing of them in the gradients before the end."""

import pytest
import torch

import test_sequence as base
from ns_fps_amd import capi
from test_sequence import DTYPES, F64, close, lib, ptr, rnd, rows, stream, workspace  # noqa: F401
from test_sequence_decays import INF, NAN, finite_scan_inputs, run_scan_grad


def same(got, want):
    """The same bits, NaN where NaN is."""
    return torch.equal(torch.isnan(got), torch.isnan(want)) and \
        torch.equal(torch.nan_to_num(got, nan=-7.0), torch.nan_to_num(want, nan=-7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [INF, -INF, NAN])
@pytest.mark.parametrize("channels", [3, 64])
def test_convolution_gradient_past_the_end_is_zero(lib, dtype, bad, channels):  # noqa: F811
    """A sequence whose last inputs are not finite has zeros after its end, and
    the sequence beside it keeps its bits."""
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(7)
    batch, length, width, n = 2, 70, 4, 37
    x = rnd(gen, batch, length, channels, dtype=t)
    dy, weight = rnd(gen, batch, length, channels, dtype=t), rnd(gen, channels, width, dtype=t)
    lens = torch.tensor([n, length], dtype=torch.int32, device="cuda")
    outs = []
    for last in (0.5, bad):
        x[0, n - 1] = last
        xd, gd, wd = x.cuda(), dy.cuda(), weight.cuda()
        dx = torch.full_like(xd, NAN)
        dw = torch.empty(channels, width, device="cuda")
        args = capi.ConvArgs(batch=batch, length=length, channels=channels, width=width, dtype=code,
                             x=rows(xd), d_weight=ptr(wd), d_lengths=ptr(lens))
        ws = workspace(lib.conv_grad_workspace_bytes(args))
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.conv_grad_device(args, capi.ConvGrads(dy=rows(gd), dx=rows(dx), d_dweight=ptr(dw)),
                             stream())
        outs.append(dx.cpu())
    assert outs[1][0, n:].eq(0).all()
    assert torch.equal(outs[1][1], outs[0][1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("channels", [3, 64])
def test_convolution_gradient_reads_no_slope_past_the_end(lib, dtype, channels):  # noqa: F811
    """The convolution would overflow only after the last token: the gradients
    are those of the tokens there are."""
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(8)
    length, width, n = 40, 2, 21
    x, dy = rnd(gen, 1, length, channels, dtype=t), rnd(gen, 1, length, channels, dtype=t)
    weight = torch.ones(channels, width, dtype=t)
    weight[:, 0] = 1e20
    x[:, :n - 1] = 0.0
    x[:, n - 1] = 1e30  # times 1e20 is beyond float32
    xd, gd, wd = x.cuda(), dy.cuda(), weight.cuda()
    dx = torch.full_like(xd, NAN)
    dw, db = torch.empty(channels, width, device="cuda"), torch.empty(channels, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    args = capi.ConvArgs(batch=1, length=length, channels=channels, width=width, dtype=code,
                         x=rows(xd), d_weight=ptr(wd), d_lengths=ptr(lens))
    ws = workspace(lib.conv_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.conv_grad_device(args, capi.ConvGrads(dy=rows(gd), dx=rows(dx), d_dweight=ptr(dw),
                                              d_dbias=ptr(db)), stream())
    x64, w64 = x.to(F64)[0, :n], weight.to(F64)
    pre = x64 * w64[:, 1]
    pre[1:] += x64[:-1] * w64[:, 0]
    sig = torch.sigmoid(pre)
    g = dy.to(F64)[0, :n] * sig * (1 + pre * (1 - sig))
    want = torch.zeros(length, channels, dtype=F64)
    want[:n] = g * w64[:, 1]
    want[:n - 1] += g[1:] * w64[:, 0]
    close(dx[0], want, "dx")
    close(dw, torch.stack([(g[1:] * x64[:-1]).sum(0), (g * x64).sum(0)], 1), "dweight")
    close(db, g.sum(0), "dbias")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("what", ["x", "dt", "b", "c", "dy"])
@pytest.mark.parametrize("case", [(3, 100, 4, 2, 16, 24, "plain"), (2, 100, 5, 1, 100, 64, "plain")])
def test_scan_gradient_past_the_end_is_zero(lib, case, dtype, what):  # noqa: F811
    """A sequence spoiled by one NaN has zeros after its end in every output,
    and the sequences beside it keep their bits."""
    t, code, gen, x, dt, a, bm, cm, d, bias, _ = finite_scan_inputs(case, dtype)
    batch, length, heads, groups, p, n, _ = case
    dy = rnd(gen, batch, length, heads, p, dtype=t)
    lens = [70] * batch
    outs = []
    for spoil in (False, True):
        if spoil:
            {"x": x, "dt": dt, "b": bm, "c": cm, "dy": dy}[what][0, 66] = NAN
        D = base.on_device(case, x, dt, a, bm, cm, d, bias, lens)
        outs.append(run_scan_grad(lib, case, code, D, dy.flatten(2).cuda())[:4])
    for clean, got in zip(*outs):
        assert got[0, 70:].eq(0).all()
        assert same(got[1:], clean[1:])
