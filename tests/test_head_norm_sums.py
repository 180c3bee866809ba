"""A weight's gradient over very many tokens."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import EPS, good
from test_sequence import F64, lib, ptr, stream, workspace  # noqa: F401


@pytest.mark.gpu
def test_weights_gradient_over_very_many_tokens(lib):  # noqa: F811
    """67 million tokens, all alike (rows may repeat), so that every term has one
    sign: a lane adds at most 256 of them in a row (2^-16 of the sum of the terms'
    sizes), what follows is added in float64, and a term itself is off by 2^-20."""
    tokens, d = 1 << 26, 33
    gen = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(1, 1, d, generator=gen, device="cuda").bfloat16()
    g = torch.randn(1, 1, d, generator=gen, device="cuda").bfloat16()
    w = torch.ones(d, device="cuda").bfloat16()
    dx = torch.empty(tokens, d, dtype=torch.bfloat16, device="cuda")
    dw = torch.empty(d, device="cuda")
    args = capi.NormArgs(batch=1, length=tokens, q_heads=1, head_dim=d, dtype=capi.BF16, eps=EPS,
                         q=(x.data_ptr(), 0, 0), d_q_weight=ptr(w))
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_grad_device(args, capi.NormGrads(dq_out=(g.data_ptr(), 0, 0),
                                              dq=(dx.data_ptr(), 0, d), d_dq_weight=ptr(dw)),
                         stream())
    v = x[0, 0].cpu().to(F64)
    want = g[0, 0].cpu().to(F64) * v / torch.sqrt(v.square().mean() + EPS) * tokens
    off = ((dw.cpu().to(F64) - want) / want).abs()
    assert (off <= 2.0 ** -16 + 2.0 ** -20).all(), off.max().item()
    assert torch.equal(dx[0], dx[-1])
    del ws


def test_workspace_follows_the_tokens():
    """Few tokens need no more than 1,024 workgroups' sums; the room grows with the
    tokens where lanes would add more than 256 heads."""
    L = capi.Lib()

    def need(tokens, heads, d):
        return L.norm_grad_workspace_bytes(good(batch=1, length=tokens, q_heads=heads, k_heads=0,
                                                head_dim=d, rotary_dim=0))
    assert need(1, 1, 64) == need(1 << 18, 8, 64) == 4 * 1024 * 2 * 64
    # 8 groups of 32 lanes a workgroup for single values
    assert need(1 << 26, 1, 33) == 4 * 2 * 33 * ((1 << 26) // (8 * 256))
