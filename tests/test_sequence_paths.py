"""The paths that large calls of the sequence operators take: the scan's walk
over several chunks of a segment and over many segments, groups of more than
four heads, the step of a full batch, whole bfloat16 tiles of the convolution,
and the lookup gradient's longest sorts.  Against 64 bits, with the tolerances
of test_sequence.py: their derivation (sums of float32 products for float32
outputs, one rounding for bfloat16 ones) does not hang on the length, since a
state's terms decay and the sums over tokens are in float64."""

import pytest
import torch

import test_sequence as base
from ns_fps_amd import capi
from test_sequence import (DTYPES, F64, close, embed_args, lib, ptr, rnd, rows, stream,  # noqa: F401
                           workspace)

# ------------------------------------------------------------------------ scan

# batch, length, heads, groups, head_dim, state_dim, layout; chunks a segment, segments
WALKS = [((64, 400, 8, 1, 16, 24, "plain"), 7, 1), ((16, 610, 16, 2, 8, 8, "swapped"), 5, 2),
         ((5, 1600, 8, 1, 16, 16, "padded"), 3, 9), ((32, 200, 8, 2, 72, 16, "odd"), 4, 1),
         ((16, 130, 32, 4, 64, 128, "plain"), 3, 1), ((8, 576, 18, 2, 16, 100, "odd"), 3, 3)]


def reference(x, dt, a, bm, cm, d, bias, lens, state):
    """The recurrence in float64, all sequences at once."""
    each = x.shape[2] // bm.shape[2]
    inside = torch.arange(x.shape[1], device=x.device)[None] < lens[:, None]
    delta = torch.where(inside[..., None],
                        torch.nn.functional.softplus(dt + bias, threshold=700.0), 0.0)
    decay, xd = torch.exp(delta * a), delta[..., None] * x
    bm, cm = bm.repeat_interleave(each, 2), cm.repeat_interleave(each, 2)
    ys = []
    for t in range(x.shape[1]):
        state = decay[:, t, :, None, None] * state + xd[:, t, :, :, None] * bm[:, t, :, None, :]
        ys.append((state * cm[:, t, :, None, :]).sum(-1))
    y = torch.stack(ys, 1) + d[:, None] * x
    return torch.where(inside[..., None, None], y, 0.0), state


def inputs(case, dtype, strong):
    """Inputs of test_sequence.py with every token past its end spoiled, the
    call's tensors, and 64-bit copies on the device."""
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = base.scan_inputs(case, dtype, strong)
    base.spoil(lens, x, dt, bm, cm)
    wide = [torch.nan_to_num(v.to(F64), neginf=float("-inf")).cuda()
            for v in (x, dt, a, bm, cm, d, bias)]
    D = base.on_device(case, x, dt, a, bm, cm, d, bias, lens)
    return t, code, gen, lens, wide, D, base.scan_args(case, code, *D)


@pytest.mark.parametrize("case,seg,segs", WALKS)
def test_walks_have_several_chunks(case, seg, segs):
    """What the cases below are for: the workspace holds a state and a total
    of every segment, and a segment has several chunks."""
    batch, length, heads, groups, p, n, _ = case
    args = capi.ScanArgs(batch=batch, length=length, heads=heads, groups=groups, head_dim=p,
                         state_dim=n)
    each = [4 * batch * heads * segs * k for k in (p * n, 1)]
    want = 256 if segs == 1 else sum((v + 255) // 256 * 256 for v in each)
    assert capi.Lib().scan_workspace_bytes(args) == want
    assert seg >= 2 and -(-(-(-length // 64)) // seg) == segs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strong", [False, True])
@pytest.mark.parametrize("case", [w[0] for w in WALKS])
def test_scan_over_several_chunks(lib, case, dtype, strong):  # noqa: F811
    batch, length, heads, groups, p, n, how = case
    t, code, gen, lens, wide, D, args = inputs(case, dtype, strong)
    pos = torch.randint(0, 3, (batch,), generator=gen).tolist()
    slots = torch.randperm(batch + 2, generator=gen)[:batch].tolist()
    slots[2] = -1
    cache = rnd(gen, batch + 2, heads, p, n)
    keeps = [s >= 0 and q > 0 for s, q in zip(slots, pos)]
    for s, k in zip(slots, keeps):
        if s >= 0 and not k:
            cache[s] = float("nan")
    y = base.laid_out(torch.full((batch, length, heads * p), float("nan"), dtype=t, device="cuda"),
                      how)
    state = cache.cuda()
    pd, sd = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (pos, slots))
    args.y, args.d_state, args.d_positions, args.d_slots = rows(y), ptr(state), ptr(pd), ptr(sd)
    ws = workspace(lib.scan_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.scan_device(args, stream())
    first = torch.stack([cache[s].to(F64) if k else torch.zeros(heads, p, n, dtype=F64)
                         for s, k in zip(slots, keeps)]).cuda()
    want, ends = reference(*wide, torch.tensor(lens, device="cuda"), first)
    close(y, want.flatten(2).cpu(), "y")
    used = [(b, s) for b, s in enumerate(slots) if s >= 0 and lens[b]]
    close(state[[s for _, s in used]], ends[[b for b, _ in used]].cpu(), "state")
    left = [s for s in range(batch + 2) if s not in [q for _, q in used]]
    assert torch.equal(torch.nan_to_num(state[left].cpu(), nan=-7.0),
                       torch.nan_to_num(cache[left], nan=-7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strong", [False, True])
@pytest.mark.parametrize("case", [w[0] for w in WALKS] + [(2, 150, 9, 1, 24, 40, "plain"),
                                                          (1, 70, 5, 1, 100, 64, "padded")])
def test_scan_gradient_over_several_chunks(lib, case, dtype, strong):  # noqa: F811
    """Also more heads a group than the four whose steps are found together."""
    batch, length, heads, groups, p, n, how = case
    assert heads // groups > 4 or p > 64
    t, code, gen, lens, wide, D, args = inputs(case, dtype, strong)
    dy = rnd(gen, batch, length, heads, p, dtype=t)
    base.spoil(lens, dy)
    outs = [base.laid_out(torch.full((batch, length, k), float("nan"), dtype=t, device="cuda"), how)
            for k in (heads * p, groups * n, groups * n, heads)]
    gd = base.laid_out(dy.flatten(2).cuda(), how)
    small = [torch.full((heads,), 9.0, device="cuda") for _ in range(3)]
    ws = workspace(lib.scan_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    grads = capi.ScanGrads(dy=rows(gd), dx=rows(outs[0]), db=rows(outs[1]), dc=rows(outs[2]),
                           ddt=rows(outs[3]), d_da=ptr(small[0]), d_dd=ptr(small[1]),
                           d_ddt_bias=ptr(small[2]))
    lib.scan_grad_device(args, grads, stream())
    leaves = [v.requires_grad_() for v in wide]
    zero = torch.zeros(batch, heads, p, n, dtype=F64, device="cuda")
    y, _ = reference(*leaves, torch.tensor(lens, device="cuda"), zero)
    want = torch.autograd.grad(y, leaves, torch.nan_to_num(dy.to(F64)).cuda())
    names = ("dx", "ddt", "da", "db", "dc", "dd", "ddt_bias")
    got = (outs[0], outs[3], small[0], outs[1], outs[2], small[1], small[2])
    for g, w, name in zip(got, want, names):
        close(g, (w.flatten(2) if w.ndim == 4 else w).cpu(), name)


# ---------------------------------------------------------------- convolution

TILES = [(3, 130, 64, 4, "plain"), (2, 100, 264, 2, "swapped"), (5, 257, 40, 3, "padded")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", TILES)
@pytest.mark.parametrize("cached", [False, True])
def test_convolution_of_whole_tiles(lib, case, dtype, cached):  # noqa: F811
    """Channels of whole vectors, tiles of tokens inside the sequence, and
    tiles that read the inputs of the one before."""
    base.test_convolution(lib, case, dtype, cached)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", TILES)
def test_convolution_gradient_of_whole_tiles(lib, case, dtype):  # noqa: F811
    base.test_convolution_gradient(lib, case, dtype)


# -------------------------------------------------------------- one-token step

FULL = [(1024, 1, 1, 17, 33, 2), (130, 8, 2, 64, 128, 4), (256, 2, 1, 100, 7, 3),
        (70, 16, 4, 64, 64, 4), (32, 8, 2, 64, 128, 4), (43, 3, 1, 128, 33, 2), (85, 3, 3, 17, 64, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", FULL)
@pytest.mark.parametrize("pad", [0, 3])
def test_step_of_full_batches(lib, case, dtype, pad):  # noqa: F811
    """From 256 workgroups of 64 rows on, a workgroup holds 64 rows; the last
    case has one less."""
    batch, heads, _, p, _, _ = case
    assert (batch * heads * -(-p // 64) >= 256) == (case != FULL[-1])
    base.test_step(lib, case, dtype, pad)


# ------------------------------------------------------------- lookup gradient

def lookup_gradient(lib, table_rows, tokens, width):  # noqa: F811
    """Two runs' tables, the tokens and the rows' gradients (on the device)."""
    gen = torch.Generator().manual_seed(table_rows % 1000 + tokens)
    tok = torch.randint(-2, min(table_rows + 2, 2 ** 31 - 1), (tokens,), generator=gen,
                        dtype=torch.int64).to(torch.int32)
    tok[:2] = torch.tensor([table_rows - 1, 0])
    dout = torch.randn(tokens, width, generator=gen)
    td, dd = tok.cuda(), dout.cuda()
    outs = []
    for _ in range(2):
        table = torch.full((table_rows, width), float("nan"), device="cuda")
        args = embed_args(table_rows, width, td, table, dd, 0)
        ws = workspace(lib.embed_grad_workspace_bytes(args))
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.embed_grad_device(args, stream())
        outs.append(table)
    return outs, td, dd


@pytest.mark.gpu
@pytest.mark.parametrize("table_rows,tokens", [
    (1, 262144), (3, 262144), (1, 262145), (3, 262145), (1023, 300000), (1 << 20, 3000),
    ((1 << 20) + 5, 70000), ((1 << 24) + 3, 1025),
    (40000, 511), (40000, 512), (40000, 513), ((1 << 20) + 5, 512), ((1 << 20) + 5, 513)])
def test_lookup_gradient_sorts(lib, table_rows, tokens):  # noqa: F811
    """One pass over whole keys, one, two and three passes over digits, one
    launch for few tokens, up to its last and beyond; rows of 10^5 terms (added in float64, so the tolerance stays)."""
    outs, td, dd = lookup_gradient(lib, table_rows, tokens, 3)
    hit = (td >= 0) & (td < table_rows)
    want = torch.zeros(table_rows + 1, 3, dtype=F64)
    want.index_add_(0, torch.where(hit, td, table_rows).long().cpu(), dd.cpu().to(F64))
    close(outs[0], want[:table_rows], "table gradient")
    assert torch.equal(outs[0], outs[1])


@pytest.mark.gpu
def test_lookup_gradient_of_four_passes(lib):  # noqa: F811
    """2^30 rows and more: the rows with a token, and how many are not zero."""
    table_rows = (1 << 30) + 1
    outs, td, dd = lookup_gradient(lib, table_rows, 2000, 1)
    used, at = torch.unique(td[(td >= 0) & (td < table_rows)].long().cpu(), return_inverse=True)
    inside = ((td >= 0) & (td < table_rows)).cpu()
    want = torch.zeros(len(used), 1, dtype=F64).index_add_(0, at, dd.cpu()[inside].to(F64))
    close(outs[0][used.cuda()], want, "rows with a token")
    assert torch.count_nonzero(outs[0]) == torch.count_nonzero(want)
    assert torch.equal(outs[0], outs[1])
