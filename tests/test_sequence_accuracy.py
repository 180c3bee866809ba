"""The exponentials of the sequence operators keep their relative accuracy where
their argument is large."""

import pytest
import torch

from ns_fps_amd import capi
from test_sequence import F64, lib, ptr, rows, stream, workspace  # noqa: F401


@pytest.mark.gpu
@pytest.mark.parametrize("channels", [1, 4])
def test_silu_keeps_its_relative_accuracy(lib, channels):  # noqa: F811
    """One tap of weight 1, so the convolution's sum is its input.  The
    exponential (one ulp, 2^-23, and a correction's rounding, 2^-24), 1 + it
    (2^-24), its reciprocal (2^-23) and two products (2^-24 each): 2^-21 of the
    value, however large the argument."""
    v = torch.cat([torch.linspace(-80, 80, 20001), torch.linspace(-3, 3, 20001)]).float()
    v = v[:v.numel() // channels * channels]
    x = v.reshape(1, -1, channels).cuda()
    length = x.shape[1]
    weight = torch.tensor([[0.0, 1.0]] * channels).cuda()
    y, dx = torch.empty_like(x), torch.empty_like(x)
    args = capi.ConvArgs(batch=1, length=length, channels=channels, width=2, x=rows(x), y=rows(y),
                         d_weight=ptr(weight))
    ws = workspace(lib.conv_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.conv_device(args, stream())
    dw = torch.empty(channels, 2, device="cuda")
    dy = torch.ones_like(x)
    lib.conv_grad_device(args, capi.ConvGrads(dy=rows(dy), dx=rows(dx), d_dweight=ptr(dw)), stream())
    w = v.to(F64)
    sig = torch.sigmoid(w)
    off = (y.cpu().flatten().to(F64) - w * sig).abs()
    worst = (off / (w * sig).abs().clamp(min=1e-300)).max()
    assert (off <= 2.0 ** -21 * (w * sig).abs()).all(), f"{worst:.3g}"
    # the slope's two terms cancel near -1.28: relative to their sizes, twice the roundings
    off = (dx.cpu().flatten().to(F64) - sig * (1 + w * (1 - sig))).abs()
    assert (off <= 2.0 ** -20 * sig * (1 + w.abs() * (1 - sig))).all()


@pytest.mark.gpu
def test_softplus_keeps_its_relative_accuracy(lib):  # noqa: F811
    """One token of states of one number with x = b = c = 1: y is the step.
    The exponential as above (2^-22) and the logarithm's two ulps (2^-22), the
    sum's rounding among them: 2^-21 of the value."""
    heads = 4096
    raw = torch.linspace(-20, 20, heads).float()
    ones = torch.ones(1, 1, heads, device="cuda")
    one = torch.ones(1, 1, 1, device="cuda")
    dt, a = raw[None, None].cuda(), torch.full((heads,), -1.0, device="cuda")
    y = torch.empty(1, 1, heads, device="cuda")
    args = capi.ScanArgs(batch=1, length=1, heads=heads, groups=1, head_dim=1, state_dim=1,
                         x=rows(ones), b=rows(one), c=rows(one), dt=rows(dt), y=rows(y), d_a=ptr(a))
    ws = workspace(lib.scan_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.scan_device(args, stream())
    want = torch.nn.functional.softplus(raw.to(F64), threshold=100.0)
    off = (y.cpu().flatten().to(F64) - want).abs() / want
    assert off.max() <= 2.0 ** -21, f"{off.max():.3g}"


@pytest.mark.gpu
def test_step_decay_keeps_its_relative_accuracy(lib):  # noqa: F811
    """A state of 1 without input after one token: y is the decay.  Steps of
    30 are exact, so exp(30 a) has the exponential's own error (2^-22), whose
    argument's last bits a float32 product would lose."""
    heads = 4096
    a = -torch.linspace(0.01, 2.5, heads)
    raw = torch.full((1, heads), 30.0, device="cuda")
    xbc = torch.zeros(1, heads + 2, device="cuda")
    xbc[0, -1] = 40.0  # SiLU of 40 is 40
    weight = torch.tensor([[0.0, 1.0]] * (heads + 2)).cuda()
    ring, state = torch.zeros(1, 2, heads + 2, device="cuda"), torch.ones(1, heads, 1, 1).cuda()
    pos = torch.ones(1, dtype=torch.int32, device="cuda")
    y, ad = torch.empty(1, heads, device="cuda"), a.cuda()
    lib.scan_step_device(capi.StepArgs(
        batch=1, heads=heads, groups=1, head_dim=1, state_dim=1, width=2, xbc_stride=heads + 2,
        dt_stride=heads, y_stride=heads, d_xbc=ptr(xbc), d_weight=ptr(weight), d_dt=ptr(raw),
        d_a=ptr(ad), d_positions=ptr(pos), d_cache=ptr(ring), d_state=ptr(state), d_y=ptr(y)),
        stream())
    want = torch.exp(30.0 * a.to(F64))
    off = (state.cpu().flatten().to(F64) - want).abs() / want
    assert off.max() <= 2.0 ** -21, f"{off.max():.3g}"
