"""Angles of the rotation at the farthest positions and at frequencies above 1.

The reference reduces position * frequency in rational numbers.  Tolerance: the
angle 2^-22; cosine and sine two units of float32 (2^-22), the normed pair three
roundings and the root's two units (2^-21.4), the rotation's products and sum three
more (2^-22.4): below 2^-20 of the pair's length."""

import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import EPS
from test_sequence import F64, lib, ptr, rows, stream, workspace  # noqa: F401

PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862089986,
              10 ** 82)


def reduced(position, freq):
    """The angle's distance from the nearest whole turn, in radians."""
    angle = Fraction(position) * Fraction(float(freq))
    return float(angle - 2 * PI * round(angle / (2 * PI)))


def test_the_reference_reduces():
    assert abs(reduced(1, 1.0) - 1.0) < 1e-15 and abs(reduced(-7, 0.5) - (2 * math.pi - 3.5)) < 1e-15
    # 355 radians are 56.5 turns and 3e-5
    assert abs(abs(reduced(355, 1.0)) - math.pi) < 1e-4


FREQS = np.float32([1.0, 0.99999994, 0.7390851, 1e-4, 3.0, 1000.0, 1234567.0, 2.0 ** 39 * 1.1, -5.5,
                    0.0])
STARTS = [0, 1, 65535, 2 ** 24 + 1, 2 ** 31 - 1]


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [False, True])
def test_far_positions_and_fast_rotations(lib, grad):  # noqa: F811
    """Heads of (1, 0) pairs: the outputs are cosines and sines.  The gradient turns
    back by the same angles: with the normed head's part of g taken out it is
    root * g turned, and a g across every head leaves it whole."""
    half, length = len(FREQS), 3
    batch, d = len(STARTS), 2 * half
    x = torch.zeros(batch, length, d, device="cuda")
    x[..., :half] = 1.0
    freq = torch.from_numpy(FREQS).cuda()
    pos = torch.tensor(STARTS, dtype=torch.int32, device="cuda")
    turn = torch.tensor([[[reduced(p + t, f) for f in FREQS] for t in range(length)]
                         for p in STARTS], dtype=F64)
    c, s = torch.cos(turn), torch.sin(turn)
    root = 1 / math.sqrt(0.5 + EPS)
    args = capi.NormArgs(batch=batch, length=length, q_heads=1, head_dim=d, rotary_dim=d, eps=EPS,
                         q=rows(x), d_freq=ptr(freq), d_positions=ptr(pos))
    out = torch.full_like(x, float("nan"))
    if grad:
        g = torch.zeros_like(x)  # (0, 1) turned by the angle: back to (0, 1)
        g[..., :half], g[..., half:] = (-s).float().cuda(), c.float().cuda()
        ws = workspace(lib.norm_grad_workspace_bytes(args))
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.norm_grad_device(args, capi.NormGrads(dq_out=rows(g), dq=rows(out)), stream())
        want = torch.cat([torch.zeros_like(c), torch.ones_like(c)], -1) * root
    else:
        args.q_out = rows(out)
        lib.norm_device(args, stream())
        want = torch.cat([c, s], -1) * root
    off = (out.cpu().to(F64) - want).abs().amax((0, 1))
    assert (off <= 2.0 ** -20 * root).all(), off.tolist()
