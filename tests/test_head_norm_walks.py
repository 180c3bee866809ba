"""Norms and their gradient where a group of lanes takes several heads of a token and
several tokens, as training batches do: the walk over an item's heads from q's to k's,
the grid's next items, and the weights' sums across both.  References in 64 bits on
the device; the tolerances are those of test_head_norm.py."""

import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import EPS, lengths_of_pairs, turned, within
from test_sequence import DTYPES, F64, lib, ptr, rows, stream, workspace  # noqa: F401

# batch, length, q_heads, k_heads, head_dim, rotary_dim, neighbours: every set of them
# at both types, so that one or the other has the walk that is meant
CASES = [
    # items of three heads, of two and three sides: 5 + 3 heads as 3 + 3 + 2
    (3, 3500, 5, 3, 64, 64, 0), (3, 7000, 5, 3, 64, 32, 1),
    # all heads an item, more tokens than the gradient's workgroups hold at once
    (3, 25001, 5, 3, 64, 64, 0),
    # the same with single values a lane: one vector of them a lane, and two
    (3, 6001, 2, 1, 33, 32, 1), (2, 3001, 1, 2, 255, 100, 0),
    # one side alone
    (2, 50001, 0, 3, 32, 16, 0)]


def split(case, dtype):
    """How a call is laid out: heads of an item, items of a token, items that 1,024
    workgroups take at once, for rows at 16-byte boundaries."""
    batch, length, hq, hk, d, r, _ = case
    half, behind = r // 2, d - r
    v = 4 if dtype == "f32" else 8
    while v > 1 and (half % v or behind % (2 * v) or d % v):
        v //= 2
    lanes = 1
    while lanes < 64 and lanes * v < half + (behind + 1) // 2:
        lanes *= 2
    heads = hq + hk
    chunks = min(heads, max(1, 2 ** 18 // (batch * length * lanes)))
    per = -(-heads // chunks)
    return per, -(-heads // per), 1024 * (256 // lanes)


def test_sizes_reach_the_walks():
    """What the cases are for, by the rule that the launch goes by."""
    seen = {(c, t): split(c, t) for c in CASES for t in DTYPES}
    assert all(per > 1 for per, _, _ in seen.values())
    uneven = [k for k, (per, chunks, _) in seen.items() if chunks > 1 and sum(k[0][2:4]) % per]
    crossing = [k for k, (per, chunks, _) in seen.items() if chunks > 1 and k[0][2] % per]
    assert {t for _, t in uneven} == {t for _, t in crossing} == set(DTYPES)
    again = [k for k, (_, chunks, room) in seen.items() if k[0][0] * k[0][1] * chunks > room]
    assert {t for _, t in again} == set(DTYPES)
    assert all((c, t) in again for c in CASES[2:5] for t in DTYPES if c != CASES[4] or t == "f32")


def on_device(case, dtype):
    batch, length, hq, hk, d, r, neighbours = case
    t, code = DTYPES[dtype]
    gen = torch.Generator(device="cuda").manual_seed(d + length)

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=gen, device="cuda") * scale

    x = {k: normal(batch, length, h * d).to(t) for k, h in (("q", hq), ("k", hk))}
    dy = {k: normal(*v.shape).to(t) for k, v in x.items()}
    w = {k: (1 + normal(d, scale=0.3)).to(t) for k in "qk"}
    freq = (10000.0 ** (-torch.arange(r // 2, device="cuda", dtype=F64) * 2 / r)).float()
    lens = [length, 2 * length // 3, 1][:batch]
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    pos = torch.arange(batch, dtype=torch.int32, device="cuda") * 1001
    inside = torch.arange(length, device="cuda")[None] < ld[:, None]
    for s in (x, dy):
        for k, v in s.items():
            s[k] = torch.where(inside[..., None], v, torch.full_like(v, float("nan")))
    args = capi.NormArgs(batch=batch, length=length, q_heads=hq, k_heads=hk, head_dim=d,
                         rotary_dim=r, neighbours=neighbours, dtype=code, eps=EPS,
                         d_q_weight=ptr(w["q"]), d_k_weight=ptr(w["k"]), d_freq=ptr(freq),
                         d_lengths=ptr(ld), d_positions=ptr(pos))
    for k in "qk":
        if x[k].numel():
            setattr(args, k, rows(x[k]))
    at = pos.to(F64)[:, None] + torch.arange(length, device="cuda", dtype=F64)
    angle = (at[..., None] * freq.to(F64))[:, :, None]
    return args, x, dy, w, angle, inside[..., None, None], (freq, ld, pos)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_walks(lib, case, dtype):  # noqa: F811
    batch, length, hq, hk, d, r, neighbours = case
    args, x, dy, w, angle, inside, held = on_device(case, dtype)
    out = {k: torch.full_like(v, float("nan")) for k, v in x.items()}
    dx = {k: torch.full_like(v, float("nan")) for k, v in x.items()}
    dw = {k: torch.full((d,), 9.0, device="cuda") for k in "qk"}
    grads = capi.NormGrads(d_dq_weight=ptr(dw["q"]), d_dk_weight=ptr(dw["k"]))
    for k in "qk":
        if x[k].numel():
            setattr(args, f"{k}_out", rows(out[k]))
            setattr(grads, f"d{k}_out", rows(dy[k]))
            setattr(grads, f"d{k}", rows(dx[k]))
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_device(args, stream())
    lib.norm_grad_device(args, grads, stream())
    for k, heads in (("q", hq), ("k", hk)):
        if not heads:
            assert dw[k].eq(0).all()
            continue
        v, g = (torch.where(inside, s[k].to(F64).reshape(batch, length, heads, d), 0.0)
                for s in (x, dy))
        wk = w[k].to(F64)
        root = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
        n = v * root
        want = turned(n * wk, angle, neighbours) * inside
        tol = 2.0 ** -18 * lengths_of_pairs(want, r, neighbours)
        within(out[k], want.flatten(2).cpu(), tol.flatten(2).cpu(), k)
        size = lengths_of_pairs(g, r, neighbours)
        g = turned(g, -angle, neighbours)
        terms = (size * n).abs().sum((0, 1, 2))
        within(dw[k], (g * n).sum((0, 1, 2)).cpu(), (2.0 ** -17 * terms).cpu(), f"d{k}_weight")
        g = g * wk
        tol = 2.0 ** -17 * root * (size * wk.abs()
                                   + n.abs() * (size * wk * n).abs().mean(-1, keepdim=True))
        want = root * (g - n * (g * n).mean(-1, keepdim=True))
        within(dx[k], want.flatten(2).cpu(), tol.flatten(2).cpu(), f"d{k}")
    del held, ws
