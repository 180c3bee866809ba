"""Norms at the ends of their numbers: heads whose squares pass float32, and an eps
below the ordinary numbers."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import EPS
from test_sequence import DTYPES, F64, lib, ptr, rows, stream, workspace  # noqa: F401


def both(lib, x, g, w, eps=EPS):  # noqa: F811
    """Norms of [B, L, D] as one head and the gradient: y, dx, dw."""
    code = capi.F32 if x.dtype == torch.float32 else capi.BF16
    b, length, d = x.shape
    y, dx = torch.full_like(g, float("nan")), torch.full_like(g, float("nan"))
    dw = torch.full((d,), 9.0, device="cuda")
    args = capi.NormArgs(batch=b, length=length, q_heads=1, head_dim=d, dtype=code, eps=eps,
                         q=rows(x), q_out=rows(y), d_q_weight=ptr(w))
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_device(args, stream())
    lib.norm_grad_device(args, capi.NormGrads(dq_out=rows(g), dq=rows(dx), d_dq_weight=ptr(dw)),
                         stream())
    torch.cuda.synchronize()
    del ws
    return y, dx, dw


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e19, 1e25, 3e38])
def test_heads_whose_squares_pass_float32(lib, dtype, size):  # noqa: F811
    """Such a head is zeros, and so are its gradient and its part of the weights'."""
    t, _ = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(3)
    d = 64
    x = torch.randn(1, 4, d, generator=gen, device="cuda")
    x[0, 1] = size * torch.where(x[0, 1] < 0, -1.0, 1.0)
    g = 30 * torch.randn(1, 4, d, generator=gen, device="cuda")
    g[0, 1] = 30 * torch.where(x[0, 1] < 0, -1.0, 1.0)  # the sum of their products passes, too
    x, g, w = x.to(t), g.to(t), torch.ones(d, device="cuda").to(t)
    y, dx, dw = both(lib, x, g, w)
    assert y[0, 1].eq(0).all() and dx[0, 1].eq(0).all()
    x2 = x.clone()
    x2[0, 1] = 0
    y2, dx2, dw2 = both(lib, x2, g, w)
    others = torch.tensor([0, 2, 3]).cuda()
    assert torch.equal(y[0, others], y2[0, others]) and torch.equal(dx[0, others], dx2[0, others])
    assert torch.equal(dw, dw2)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-45, 1e-40, 1.1e-38, 1e-37])
def test_heads_of_zeros_with_the_smallest_eps(lib, eps):  # noqa: F811
    """0 * root(1 / eps) is 0; the gradient by x is g * root(1 / eps), finite."""
    x = torch.zeros(1, 2, 32, device="cuda")
    x[0, 1] = 1.0
    g = torch.full_like(x, 1e-20)
    y, dx, dw = both(lib, x, g, torch.ones(32, device="cuda"), eps)
    assert y[0, 0].eq(0).all() and (y[0, 1] - 1).abs().max() <= 2.0 ** -20
    exact = float(torch.tensor(eps, dtype=torch.float32))
    want = 1e-20 / exact ** 0.5
    assert (dx[0, 0].cpu().to(F64) - want).abs().max() <= 2.0 ** -20 * want
    # the other head lies along its g: nothing is left of it but roundings
    assert dx[0, 1].abs().max() <= 2.0 ** -20 * 1e-20
    assert (dw.cpu().to(F64) - 1e-20).abs().max() <= 2.0 ** -20 * 1e-20
