"""Decays of the selective scan at their edges: a parameter that is not finite,
and tokens that wipe the state."""

import pytest
import torch

import test_sequence as base
from ns_fps_amd import capi
from test_sequence import F64, close, lib, ptr, rnd, rows, stream, workspace  # noqa: F401

INF, NAN = float("inf"), float("nan")


def run_scan(lib, case, code, D, cache, lens=None):  # noqa: F811
    """y [B, L, H, P] and the cache after the call."""
    batch, length, heads, _, p, _, _ = case
    args = base.scan_args(case, code, *D)
    y = torch.full((batch, length, heads * p), NAN, dtype=D[0].dtype, device="cuda")
    state = cache.cuda()
    pos = torch.ones(batch, dtype=torch.int32, device="cuda")
    args.y, args.d_state, args.d_positions = rows(y), ptr(state), ptr(pos)
    ws = workspace(lib.scan_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.scan_device(args, stream())
    return y.unflatten(2, (heads, p)).cpu(), state.cpu()


def run_scan_grad(lib, case, code, D, dy):  # noqa: F811
    """dx, ddt, db, dc, da, dd, ddt_bias."""
    batch, length, heads, groups, p, n, _ = case
    args = base.scan_args(case, code, *D)
    outs = [torch.full((batch, length, k), NAN, dtype=D[0].dtype, device="cuda")
            for k in (heads * p, heads, groups * n, groups * n)]
    small = [torch.full((heads,), 9.0, device="cuda") for _ in range(3)]
    ws = workspace(lib.scan_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.scan_grad_device(args, capi.ScanGrads(
        dy=rows(dy), dx=rows(outs[0]), db=rows(outs[2]), dc=rows(outs[3]), ddt=rows(outs[1]),
        d_da=ptr(small[0]), d_dd=ptr(small[1]), d_ddt_bias=ptr(small[2])), stream())
    return [outs[0].unflatten(2, (heads, p)).cpu(), outs[1].cpu(),
            *(v.unflatten(2, (groups, n)).cpu() for v in outs[2:]), *(v.cpu() for v in small)]


def finite_scan_inputs(case, dtype):
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = base.scan_inputs(case, dtype)
    dt = torch.nan_to_num(dt, neginf=-3.0)
    return t, code, gen, x, dt, a, bm, cm, d, bias, [case[1]] * case[0]


# one and several chunks; a prompt of one token, as the step reads it
DECAYS = [(1, 1, 4, 2, 16, 24, "plain"), (2, 40, 4, 2, 16, 24, "plain"),
          (1, 200, 4, 2, 64, 64, "plain"), (64, 200, 8, 2, 8, 16, "plain")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [NAN, -INF])
@pytest.mark.parametrize("case", DECAYS)
def test_a_decay_that_is_not_finite(lib, case, dtype, bad):  # noqa: F811
    """a = NaN spoils its head's outputs, state and gradients; a = -infinity
    forgets the state at every token; other heads keep their bits."""
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = finite_scan_inputs(case, dtype)
    batch, length, heads, groups, p, n, _ = case
    cache = rnd(gen, batch, heads, p, n)
    dy = rnd(gen, batch, length, heads * p, dtype=t).cuda()
    one = 1  # the head, of the first group
    spoiled = a.clone()
    spoiled[one] = bad
    others = [h for h in range(heads) if h != one]
    D, S = (base.on_device(case, x, dt, v, bm, cm, d, bias, lens) for v in (a, spoiled))
    y0, s0 = run_scan(lib, case, code, D, cache)
    y1, s1 = run_scan(lib, case, code, S, cache)
    assert torch.equal(y1[:, :, others], y0[:, :, others])
    assert torch.equal(s1[:, others], s0[:, others])
    g0, g1 = run_scan_grad(lib, case, code, D, dy), run_scan_grad(lib, case, code, S, dy)
    for k in (0, 1):  # dx, ddt
        assert torch.equal(g1[k][:, :, others], g0[k][:, :, others])
    for k in (2, 3):  # db, dc: the other groups'
        assert torch.equal(g1[k][:, :, 1:], g0[k][:, :, 1:])
    for k in (4, 5, 6):
        assert torch.equal(g1[k][others], g0[k][others])
    if bad != bad:
        assert torch.isnan(y1[:, :, one]).all() and torch.isnan(s1[:, one]).all()
        for g in (g1[0][:, :, one], g1[1][:, :, one], g1[2][:, :, 0], g1[3][:, :, 0]):
            assert torch.isnan(g).all()
        assert torch.isnan(g1[4][one]) and torch.isnan(g1[6][one])
        return
    wide = [v.to(F64) for v in (x, dt, spoiled, bm, cm, d, bias)]
    wide[2][one] = -1e30  # exp(step * a) is 0 here too, and 0 * a is not NaN
    leaves = [v.requires_grad_() for v in wide]
    y, ends = base.scan_plain(*leaves, lens, cache.to(F64))
    close(y1, y.detach(), "y")
    close(s1, ends.detach(), "state")
    fresh, _ = base.scan_plain(*leaves, lens, torch.zeros(batch, heads, p, n, dtype=F64))
    want = torch.autograd.grad((fresh * dy.cpu().to(F64).unflatten(2, (heads, p))).sum(), leaves)
    for k, w in ((0, want[0]), (2, want[3]), (3, want[4]), (5, want[5])):
        close(g1[k], w, "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [NAN, -INF])
def test_prompt_and_step_agree_on_decays_that_are_not_finite(lib, dtype, bad):  # noqa: F811
    """The prompt of one token over the step's own channels (its convolution
    the identity's SiLU) and the step: NaN in the same places, else close."""
    case = (3, 1, 4, 2, 16, 24, "plain")
    batch, _, heads, groups, p, n, _ = case
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = finite_scan_inputs(case, dtype)
    a[2] = bad
    channels, width = heads * p + 2 * groups * n, 2
    xbc = torch.cat([x.flatten(1), bm.flatten(1), cm.flatten(1)], 1)
    act = base.silu(xbc.to(F64))
    weight = torch.zeros(channels, width, dtype=t)
    weight[:, 1] = 1.0
    cache = rnd(gen, batch, heads, p, n)
    D = [v.cuda() for v in (xbc, weight, dt[:, 0], a, d, bias)]
    ring, state = torch.zeros(batch, width, channels, dtype=t, device="cuda"), cache.cuda()
    pos = torch.ones(batch, dtype=torch.int32, device="cuda")
    y = torch.empty(batch, heads * p, dtype=t, device="cuda")
    lib.scan_step_device(capi.StepArgs(
        batch=batch, heads=heads, groups=groups, head_dim=p, state_dim=n, width=width, dtype=code,
        xbc_stride=channels, dt_stride=heads, y_stride=heads * p, d_xbc=ptr(D[0]),
        d_weight=ptr(D[1]), d_dt=ptr(D[2]), d_a=ptr(D[3]), d_d=ptr(D[4]), d_dt_bias=ptr(D[5]),
        d_positions=ptr(pos), d_cache=ptr(ring), d_state=ptr(state), d_y=ptr(y)), stream())
    parts = [v.unflatten(2, (k, -1)) for v, k in zip(
        torch.split(act[:, None].float(), [heads * p, groups * n, groups * n], 2),
        (heads, groups, groups))]
    E = base.on_device(case, parts[0], dt.float(), a, parts[1], parts[2], d, bias, lens)
    y1, s1 = run_scan(lib, case, capi.F32, E, cache)
    ok = [h for h in range(heads) if h != 2] if bad != bad else list(range(heads))
    y = y.unflatten(1, (heads, p))
    close(y[:, ok], y1[:, 0, ok].to(F64), "y")
    close(state[:, ok], s1[:, ok].to(F64), "state")
    for v in (y[:, 2], y1[:, 0, 2], state[:, 2], s1[:, 2]):
        assert torch.isnan(v).all() == (bad != bad)


@pytest.mark.gpu
@pytest.mark.parametrize("case", DECAYS[1:])
def test_tokens_that_wipe_the_state_keep_later_decays(lib, case):  # noqa: F811
    """A step of 10^9 at a token without input: what comes before is gone, and
    the decays after it are as exact as without it."""
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = finite_scan_inputs(case, "f32")
    dt[:, 3::50] = 1e9
    x[:, 3::50] = 0.0
    cache = rnd(gen, case[0], case[2], case[4], case[5])
    y1, s1 = run_scan(lib, case, code, base.on_device(case, x, dt, a, bm, cm, d, bias, lens), cache)
    y, ends = base.scan_plain(*(v.to(F64) for v in (x, dt, a, bm, cm, d, bias)), lens,
                              cache.to(F64))
    close(y1, y, "y")
    close(s1, ends, "state")
