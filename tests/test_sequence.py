"""The sequence operators (embedding lookup and its gradient, causal
convolution, selective scan, their gradients, the one-token step) against
plain implementations in 64 bits on the CPU, at the sizes, masks, strides and
caches where they can go wrong; and their refusals.

Tolerances.  A float32 output is a float32 sum of at most a few hundred
products with at most two roundings a term (2^-24 each): 2^-16 of the value
plus 2^-16 of the output's root mean square, which leaves a factor of 256 for
the terms that cancel.  A bfloat16 output is rounded once (2^-9 of the value)
from sums whose factors hold 16 bits: 2^-8 of the value plus 2^-10 of the root
mean square."""

import ctypes

import numpy as np
import pytest
import torch

from ns_fps_amd import capi

F64 = torch.float64
DTYPES = {"f32": (torch.float32, capi.F32), "bf16": (torch.bfloat16, capi.BF16)}


@pytest.fixture(scope="module")
def lib():
    L = capi.Lib()
    if L.device_count() < 1:
        pytest.fail("no HIP device visible: GPU tests need an MI355X")
    return L


def close(got, want, what=""):
    """got (device) against want (float64, CPU)."""
    g, w = got.detach().cpu().to(F64), want
    assert g.shape == w.shape, what
    assert torch.isfinite(g).all(), what
    rms = w.square().mean().sqrt() if w.numel() else torch.zeros((), dtype=F64)
    tol = (2.0 ** -8 * w.abs() + 2.0 ** -10 * rms) if got.dtype == torch.bfloat16 else \
        (2.0 ** -16 * w.abs() + 2.0 ** -16 * rms)
    off = (g - w).abs() - tol
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} beyond, rms {rms.item():.3g}"


def rnd(gen, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=gen, dtype=F64) * scale).to(dtype)


def dev(t):
    return None if t is None else t.cuda()


def ptr(t):
    return None if t is None else t.data_ptr()


def rows(t, offset=0):
    return (t.data_ptr() + offset * t.element_size(), t.stride(0), t.stride(1))


def stream():
    return torch.cuda.current_stream().cuda_stream


def workspace(nbytes):
    # filled with NaN bits: nothing may depend on what it held
    return torch.full((max(nbytes, 1),), 0xFF, dtype=torch.uint8, device="cuda")


# ------------------------------------------------------------------- embedding

def embed_args(table_rows, width, tokens, table, out, dtype, grad_dtype=0, scale=1.0):
    return capi.EmbedArgs(tokens=len(tokens), rows=table_rows, width=width, dtype=dtype,
                          grad_dtype=grad_dtype, scale=scale, table_stride=table.stride(0),
                          out_stride=out.stride(0) if len(tokens) else width,
                          d_table=table.data_ptr(), d_tokens=ptr(tokens), d_out=out.data_ptr())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,table_rows,width,pad", [
    (1, 1, 1, 0), (1, 7, 64, 0), (65, 4096, 384, 0), (1000, 512, 383, 0), (300, 33, 640, 8),
    (257, 100, 12, 4), (129, 9, 2049, 3), (5, 3, 65536, 0)])
def test_lookup(lib, dtype, tokens, table_rows, width, pad):
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(tokens * width)
    table = rnd(gen, table_rows, width + pad, dtype=t).cuda()
    tok = torch.randint(-1, table_rows + 1, (tokens,), generator=gen, dtype=torch.int32)
    tok[0] = table_rows - 1
    if tokens > 3:
        tok[1:4] = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0], dtype=torch.int32)
    out = torch.full((tokens, width + pad), float("nan"), dtype=t, device="cuda")
    lib.embed_device(embed_args(table_rows, width, tok.cuda(), table, out, code, scale=1.5),
                     stream())
    ok = (tok >= 0) & (tok < table_rows)
    want = table.cpu().to(F64)[tok.long().clamp(0, table_rows - 1), :width] * 1.5
    close(out[:, :width], want * ok[:, None], "lookup")
    assert torch.isnan(out[:, width:]).all()  # nothing beside the rows is written


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,grad", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"),
                                        ("f32", "bf16")])
@pytest.mark.parametrize("tokens,table_rows,width,pad,kind", [
    (0, 5, 16, 0, "any"), (1, 1, 1, 0, "any"), (1, 1000, 64, 0, "any"), (64, 3, 8, 0, "any"),
    (4096, 300, 384, 0, "any"), (1000, 70000, 20, 4, "any"), (1500, 17, 383, 1, "any"),
    (5000, 40, 64, 0, "one"), (70000, 1 << 18, 32, 0, "crowded"), (3000, 9, 130, 2, "none"),
    (20000, 256, 12, 0, "crowded")])
def test_lookup_gradient(lib, dtype, grad, tokens, table_rows, width, pad, kind):
    t, code = DTYPES[dtype]
    gt, gcode = DTYPES[grad]
    gen = torch.Generator().manual_seed(tokens + width)
    tok = torch.randint(-1, table_rows + 1, (tokens,), generator=gen, dtype=torch.int32)
    if kind == "one":
        tok[:] = table_rows - 1
    elif kind == "none":
        tok[::2], tok[1::2] = -1, table_rows
    elif kind == "crowded":
        tok[torch.rand(tokens, generator=gen) < 0.7] = 3
    dout = rnd(gen, max(tokens, 1), width + pad, dtype=t).cuda()
    table = torch.full((table_rows, width + pad), float("nan"), dtype=gt, device="cuda")
    tk = tok.cuda()
    args = embed_args(table_rows, width, tk, table, dout, code, gcode, 0.25)
    runs = []
    for _ in range(2):
        ws = workspace(lib.embed_grad_workspace_bytes(args))
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.embed_grad_device(args, stream())
        runs.append(table[:, :width].clone())
    ok = (tok >= 0) & (tok < table_rows)
    want = torch.zeros(table_rows + 1, width, dtype=F64)
    want.index_add_(0, torch.where(ok, tok, table_rows).long(),
                    dout.cpu().to(F64)[:tokens, :width])
    close(runs[0], want[:table_rows] * 0.25, "table gradient")
    assert torch.equal(runs[0], runs[1])  # the same bits every time
    assert torch.isnan(table[:, width:]).all()


@pytest.mark.gpu
def test_lookup_beyond_32_bit_offsets(lib):
    table_rows, width = (1 << 31) // 4096 + 9, 8192  # the last rows lie above 2^32 elements
    table = torch.zeros(table_rows, width, dtype=torch.bfloat16, device="cuda")
    table[-1], table[3] = 2.0, 1.0
    tok = torch.tensor([table_rows - 1, 3, -1], dtype=torch.int32, device="cuda")
    out = torch.empty(3, width, dtype=torch.bfloat16, device="cuda")
    lib.embed_device(embed_args(table_rows, width, tok, table, out, capi.BF16), stream())
    assert out[0].eq(2).all() and out[1].eq(1).all() and out[2].eq(0).all()
    args = embed_args(table_rows, width, tok, table, out, capi.BF16, capi.BF16)
    ws = workspace(lib.embed_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    out.copy_(torch.tensor([5.0, 7.0, 9.0]).cuda()[:, None])
    lib.embed_grad_device(args, stream())
    assert table[-1].eq(5).all() and table[3].eq(7).all()
    assert table[-2].eq(0).all() and table[0].eq(0).all()


# ----------------------------------------------------------------- convolution

def silu(v):
    return v * torch.sigmoid(v)


def conv_plain(x, weight, bias, lens, pos=None, ring=None):
    """float64, sequence by sequence; the ring is updated in place."""
    y = torch.zeros_like(x)
    width = weight.shape[1]
    for b in range(x.shape[0]):
        n, p = lens[b], 0 if pos is None else max(pos[b], 0)
        before = [ring[b, (p - k) % width].clone() if ring is not None and p >= k
                  else torch.zeros_like(x[b, 0]) for k in range(width - 1, 0, -1)]
        seen = torch.stack(before + [x[b, t] for t in range(n)])
        for t in range(n):
            y[b, t] = silu((seen[t:t + width].T * weight).sum(1) + bias)
        if ring is not None:
            for t in range(max(0, n - width), n):
                ring[b, (p + t) % width] = x[b, t]
    return y


def laid_out(t, how):
    """The same values with other strides: rows padded by 16 or by 3
    elements, or tokens ahead of sequences."""
    if how == "plain":
        return t
    if how == "swapped":
        return t.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((*t.shape[:-1], t.shape[-1] + (16 if how == "padded" else 3)), float("nan"),
                      dtype=t.dtype, device=t.device)
    wide[..., :t.shape[-1]] = t
    return wide[..., :t.shape[-1]]


CONV = [(1, 1, 1, 2, "plain"), (2, 3, 5, 4, "plain"), (3, 17, 64, 3, "padded"),
        (1, 130, 321, 4, "odd"), (2, 64, 260, 2, "swapped"), (4, 33, 36, 4, "plain"),
        (2, 100, 1028, 3, "plain")]


def conv_inputs(case, dtype):
    batch, length, channels, width, how = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(length * channels)
    x = rnd(gen, batch, length, channels, dtype=t)
    weight, bias = rnd(gen, channels, width, dtype=t), rnd(gen, channels, dtype=t)
    lens = torch.randint(0, length + 1, (batch,), generator=gen).tolist()
    lens[0] = length
    if batch > 1:
        lens[-1] = 0
    for b in range(batch):
        x[b, lens[b]:] = float("nan")  # past the end: never read
    return t, code, gen, x, weight, bias, lens


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CONV)
@pytest.mark.parametrize("cached", [False, True])
def test_convolution(lib, case, dtype, cached):
    batch, length, channels, width, how = case
    t, code, gen, x, weight, bias, lens = conv_inputs(case, dtype)
    pos = torch.randint(0, 9, (batch,), generator=gen).tolist()
    pos[0] = 2 ** 31 - 1 - length if length > 64 else pos[0]
    slots = torch.randperm(batch + 2, generator=gen)[:batch].tolist()
    if cached and batch > 2:
        slots[1] = -1
    ring = rnd(gen, batch + 2, width, channels, dtype=t)
    for b in range(batch):
        if slots[b] >= 0 and pos[b] < width:  # entries that no token has filled
            for e in range(pos[b], width):
                ring[slots[b], e] = float("nan")
    xd, yd = laid_out(x.cuda(), how), laid_out(torch.full_like(x, float("nan")).cuda(), how)
    wd, bd, rd = weight.cuda(), bias.cuda(), ring.cuda()
    ld, pd, sd = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (lens, pos, slots))
    args = capi.ConvArgs(batch=batch, length=length, channels=channels, width=width, dtype=code,
                         x=rows(xd), y=rows(yd), d_weight=ptr(wd), d_bias=ptr(bd), d_lengths=ptr(ld))
    if cached:
        args.d_positions, args.d_slots, args.d_cache = ptr(pd), ptr(sd), ptr(rd)
    lib.conv_device(args, stream())
    x64 = torch.nan_to_num(x.to(F64))
    if cached:
        mine = ring.to(F64)[[s if s >= 0 else 0 for s in slots]]
        y = conv_plain(x64, weight.to(F64), bias.to(F64), lens,
                       [p if s >= 0 else 0 for p, s in zip(pos, slots)], mine)
        want = ring.clone()
        for b, s in enumerate(slots):
            if s >= 0:
                want[s] = mine[b].to(t)
        assert torch.equal(torch.nan_to_num(rd.cpu().float(), nan=-77.0),
                           torch.nan_to_num(want.float(), nan=-77.0))
    else:
        y = conv_plain(x64, weight.to(F64), bias.to(F64), lens)
    close(yd, y, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CONV)
def test_convolution_gradient(lib, case, dtype):
    batch, length, channels, width, how = case
    t, code, gen, x, weight, bias, lens = conv_inputs(case, dtype)
    dy = rnd(gen, batch, length, channels, dtype=t)
    for b in range(batch):
        dy[b, lens[b]:] = float("nan")
    xd, gd = laid_out(x.cuda(), how), laid_out(dy.cuda(), how)
    dx = laid_out(torch.full_like(x, float("nan")).cuda(), how)
    wd, bd = weight.cuda(), bias.cuda()
    ld = torch.tensor(lens, dtype=torch.int32, device="cuda")
    dw, db = torch.full((channels, width), 9.0).cuda(), torch.full((channels,), 9.0).cuda()
    args = capi.ConvArgs(batch=batch, length=length, channels=channels, width=width, dtype=code,
                         x=rows(xd), d_weight=ptr(wd), d_bias=ptr(bd), d_lengths=ptr(ld))
    ws = workspace(lib.conv_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.conv_grad_device(args, capi.ConvGrads(dy=rows(gd), dx=rows(dx), d_dweight=ptr(dw),
                                              d_dbias=ptr(db)), stream())
    leaves = [torch.nan_to_num(v.to(F64)).requires_grad_() for v in (x, weight, bias)]
    g64 = torch.nan_to_num(dy.to(F64))

    def loss(xv, wv, bv):
        total = torch.zeros((), dtype=F64)
        for b, n in enumerate(lens):
            if n:
                seen = torch.cat([torch.zeros(width - 1, channels, dtype=F64), xv[b, :n]])
                pre = sum(wv[:, k] * seen[k:k + n] for k in range(width)) + bv
                total = total + (silu(pre) * g64[b, :n]).sum()
        return total

    want = torch.autograd.grad(loss(*leaves), leaves)
    for got, w, name in zip((dx, dw, db), want, ("dx", "dweight", "dbias")):
        close(got, w, name)
    # and along one direction, by differences of the loss itself
    with torch.no_grad():
        dirs = [torch.randn(v.shape, generator=gen, dtype=F64) for v in leaves]
        eps = 1e-6
        diff = (loss(*[v + eps * d for v, d in zip(leaves, dirs)])
                - loss(*[v - eps * d for v, d in zip(leaves, dirs)])) / (2 * eps)
        terms = [(g.cpu().to(F64) * d) for g, d in zip((dx, dw, db), dirs)]
        norm = torch.cat([v.flatten() for v in terms]).norm()
        assert abs(sum(v.sum() for v in terms) - diff) <= (2.0 ** -6 if dtype == "bf16"
                                                          else 2.0 ** -14) * norm + 1e-5


# ------------------------------------------------------------------------ scan

def scan_plain(x, dt, a, bm, cm, d, bias, lens, states):
    """float64 recurrence; x [B, L, H, P], b and c [B, L, G, N], states
    [B, H, P, N].  Returns y and the last states."""
    each = x.shape[2] // bm.shape[2]
    ys, ends = [], []
    for b in range(x.shape[0]):
        h, out = states[b], []
        for t in range(x.shape[1]):
            if t >= lens[b]:
                out.append(torch.zeros_like(x[b, 0]))
                continue
            delta = torch.nn.functional.softplus(dt[b, t] + bias, threshold=700.0)
            bt, ct = bm[b, t].repeat_interleave(each, 0), cm[b, t].repeat_interleave(each, 0)
            h = torch.exp(delta * a)[:, None, None] * h \
                + (delta[:, None] * x[b, t])[:, :, None] * bt[:, None, :]
            out.append((h * ct[:, None, :]).sum(-1) + d[:, None] * x[b, t])
        ys.append(torch.stack(out))
        ends.append(h)
    return torch.stack(ys), torch.stack(ends)


# batch, length, heads, groups, head_dim, state_dim, layout
SCAN = [(1, 1, 1, 1, 1, 1, "plain"), (2, 2, 2, 1, 64, 64, "plain"), (1, 63, 2, 2, 32, 16, "plain"),
        (3, 64, 4, 2, 64, 128, "padded"), (2, 65, 3, 3, 5, 33, "odd"),
        (1, 200, 4, 1, 48, 100, "swapped"), (2, 130, 2, 1, 128, 64, "plain"),
        (1, 129, 2, 1, 65, 128, "padded"), (1, 300, 1, 1, 16, 32, "plain"),
        (5, 70, 6, 3, 24, 40, "plain"), (1, 150, 1, 1, 100, 7, "odd")]


def scan_inputs(case, dtype, strong=False):
    batch, length, heads, groups, p, n, how = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(length * 131 + p)
    x = rnd(gen, batch, length, heads, p, dtype=t)
    bm, cm = (rnd(gen, batch, length, groups, n, dtype=t) for _ in range(2))
    dt = rnd(gen, batch, length, heads, dtype=t)
    a = -torch.exp(rnd(gen, heads))
    d, bias = rnd(gen, heads), rnd(gen, heads) - 2
    if strong:  # a few tokens that wipe the state between others that keep it
        dt[:, ::7] = 60.0
        a = a * 100
        bias = bias - 4
    lens = torch.randint(0, length + 1, (batch,), generator=gen).tolist()
    lens[0] = length
    if batch > 2:
        lens[1] = 0
    dt[0, length // 2] = float("-inf")  # a token that leaves the state as it is
    return t, code, gen, x, dt, a, bm, cm, d, bias, lens


def spoil(lens, *tensors):
    for v in tensors:
        for b, n in enumerate(lens):
            v[b, n:] = float("nan")


def scan_args(case, code, x, dt, a, bm, cm, d, bias, lens):
    batch, length, heads, groups, p, n, _ = case
    return capi.ScanArgs(batch=batch, length=length, heads=heads, groups=groups, head_dim=p,
                         state_dim=n, dtype=code, x=rows(x), b=rows(bm), c=rows(cm), dt=rows(dt),
                         d_a=ptr(a), d_d=ptr(d), d_dt_bias=ptr(bias), d_lengths=ptr(lens))


def on_device(case, x, dt, a, bm, cm, d, bias, lens):
    """Rows flattened and laid out as the case says."""
    how = case[-1]
    flat = [laid_out(v.flatten(2).cuda(), how) for v in (x, dt, bm, cm)]
    return [flat[0], flat[1], a.cuda(), flat[2], flat[3], dev(d), dev(bias),
            torch.tensor(lens, dtype=torch.int32, device="cuda")]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strong", [False, True])
@pytest.mark.parametrize("case", SCAN)
def test_scan(lib, case, dtype, strong):
    batch, length, heads, groups, p, n, how = case
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = scan_inputs(case, dtype, strong)
    spoil(lens, x, dt, bm, cm)
    pos = torch.randint(0, 3, (batch,), generator=gen).tolist()
    slots = torch.randperm(batch + 2, generator=gen)[:batch].tolist()
    if batch > 2:
        slots[2] = -1
    cache = rnd(gen, batch + 2, heads, p, n)
    keeps = [s >= 0 and q > 0 for s, q in zip(slots, pos)]
    for s, k in zip(slots, keeps):
        if s >= 0 and not k:
            cache[s] = float("nan")  # a sequence that starts anew never reads it
    D = on_device(case, x, dt, a, bm, cm, d, bias, lens)
    args = scan_args(case, code, *D)
    y = laid_out(torch.full((batch, length, heads * p), float("nan"), dtype=t, device="cuda"), how)
    state = cache.cuda()
    pd, sd = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (pos, slots))
    args.y, args.d_state, args.d_positions, args.d_slots = rows(y), ptr(state), ptr(pd), ptr(sd)
    ws = workspace(lib.scan_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.scan_device(args, stream())
    first = torch.stack([cache[s].to(F64) if k else torch.zeros(heads, p, n, dtype=F64)
                         for s, k in zip(slots, keeps)])
    want, ends = scan_plain(*(v.to(F64) for v in (x, dt, a, bm, cm, d, bias)), lens, first)
    close(y, want.flatten(2), "y")
    for b, s in enumerate(slots):
        if s >= 0 and lens[b]:
            close(state[s], ends[b], "state")
    left = [s for s in range(batch + 2)
            if s not in [q for q, m in zip(slots, lens) if m]]  # no token: left as it was
    assert torch.equal(torch.nan_to_num(state[left].cpu(), nan=-7.0),
                       torch.nan_to_num(cache[left], nan=-7.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("strong", [False, True])
@pytest.mark.parametrize("case", SCAN)
def test_scan_gradient(lib, case, dtype, strong):
    batch, length, heads, groups, p, n, how = case
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = scan_inputs(case, dtype, strong)
    dy = rnd(gen, batch, length, heads, p, dtype=t)
    spoil(lens, x, dt, bm, cm, dy)
    D = on_device(case, x, dt, a, bm, cm, d, bias, lens)
    args = scan_args(case, code, *D)
    outs = [laid_out(torch.full((batch, length, k), float("nan"), dtype=t, device="cuda"), how)
            for k in (heads * p, groups * n, groups * n, heads)]
    gd = laid_out(dy.flatten(2).cuda(), how)
    small = [torch.full((heads,), 9.0, device="cuda") for _ in range(3)]
    ws = workspace(lib.scan_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    grads = capi.ScanGrads(dy=rows(gd), dx=rows(outs[0]), db=rows(outs[1]), dc=rows(outs[2]),
                           ddt=rows(outs[3]), d_da=ptr(small[0]), d_dd=ptr(small[1]),
                           d_ddt_bias=ptr(small[2]))
    lib.scan_grad_device(args, grads, stream())
    leaves = [torch.nan_to_num(v.to(F64), neginf=float("-inf")).requires_grad_()
              for v in (x, dt, a, bm, cm, d, bias)]
    g64 = torch.nan_to_num(dy.to(F64))
    zero = torch.zeros(batch, heads, p, n, dtype=F64)
    y, _ = scan_plain(*leaves, lens, zero)
    want = torch.autograd.grad((y * g64).sum(), leaves)
    names = ("dx", "ddt", "da", "db", "dc", "dd", "ddt_bias")
    got = (outs[0], outs[3], small[0], outs[1], outs[2], small[1], small[2])
    for g, w, name in zip(got, want, names):
        w = torch.nan_to_num(w)  # the derivative of softplus at -infinity is 0
        close(g, w.flatten(2) if w.ndim == 4 else w, name)


@pytest.mark.gpu
def test_scan_gradient_against_differences(lib):
    """One direction through all inputs: differences of the 64-bit loss."""
    case = (2, 90, 4, 2, 20, 24, "plain")
    t, code, gen, x, dt, a, bm, cm, d, bias, lens = scan_inputs(case, "f32")
    dt = torch.nan_to_num(dt, neginf=-3.0)
    dy = rnd(gen, *x.shape)
    D = on_device(case, x, dt, a, bm, cm, d, bias, lens)
    args = scan_args(case, code, *D)
    outs = [torch.empty_like(D[k]) for k in (0, 3, 4, 1)]
    gd = dy.flatten(2).cuda()
    small = [torch.empty(4, device="cuda") for _ in range(3)]
    ws = workspace(lib.scan_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    grads = capi.ScanGrads(dy=rows(gd), dx=rows(outs[0]), db=rows(outs[1]), dc=rows(outs[2]),
                           ddt=rows(outs[3]), d_da=ptr(small[0]), d_dd=ptr(small[1]),
                           d_ddt_bias=ptr(small[2]))
    lib.scan_grad_device(args, grads, stream())
    at = [v.to(F64) for v in (x, dt, a, bm, cm, d, bias)]
    dirs = [torch.randn(v.shape, generator=gen, dtype=F64) for v in at]
    zero = torch.zeros(2, 4, 20, 24, dtype=F64)

    def loss(e):
        y, _ = scan_plain(*[v + e * q for v, q in zip(at, dirs)], lens, zero)
        return (y * dy.to(F64)).sum()

    eps = 1e-6
    diff = (loss(eps) - loss(-eps)) / (2 * eps)
    got = (outs[0], outs[3], small[0], outs[1], outs[2], small[1], small[2])
    terms = [(g.cpu().to(F64).reshape(q.shape) * q).flatten() for g, q in zip(got, dirs)]
    norm = torch.cat(terms).norm()
    assert abs(torch.cat(terms).sum() - diff) <= 2.0 ** -14 * norm + 1e-5


# ------------------------------------------------------------- one-token step

STEP = [(1, 1, 1, 1, 1, 2), (1, 8, 1, 64, 128, 4), (5, 6, 3, 24, 40, 3), (3, 4, 2, 128, 64, 4),
        (70, 2, 2, 17, 33, 2), (2, 1, 1, 100, 7, 4)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", STEP)
@pytest.mark.parametrize("pad", [0, 3, 16])
def test_step(lib, case, dtype, pad):
    batch, heads, groups, p, n, width = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(p * n)
    channels = heads * p + 2 * groups * n
    xbc, dt = rnd(gen, batch, channels, dtype=t), rnd(gen, batch, heads, dtype=t)
    weight, wbias = rnd(gen, channels, width, dtype=t), rnd(gen, channels, dtype=t)
    a, d, bias = -torch.exp(rnd(gen, heads)), rnd(gen, heads), rnd(gen, heads) - 2
    pos = torch.randint(0, 7, (batch,), generator=gen)
    slots = torch.randperm(batch + 3, generator=gen)[:batch]
    if batch > 2:
        slots[1] = -1
    ring, state = rnd(gen, batch + 3, width, channels, dtype=t), rnd(gen, batch + 3, heads, p, n)
    for b in range(batch):
        if slots[b] >= 0 and pos[b] == 0:
            ring[slots[b]], state[slots[b]] = float("nan"), float("nan")
    wide = [laid_out(v[None].cuda(), {0: "plain", 3: "odd", 16: "padded"}[pad])[0]
            for v in (xbc, dt, torch.full((batch, heads * p), float("nan"), dtype=t))]
    D = [v.cuda() for v in (weight, wbias, a, d, bias)]
    rd, sd = ring.cuda(), state.cuda()
    pd, td = pos.to(torch.int32).cuda(), slots.to(torch.int32).cuda()
    args = capi.StepArgs(batch=batch, heads=heads, groups=groups, head_dim=p, state_dim=n,
                         width=width, dtype=code, xbc_stride=wide[0].stride(0),
                         dt_stride=wide[1].stride(0), y_stride=wide[2].stride(0),
                         d_xbc=ptr(wide[0]), d_weight=ptr(D[0]), d_bias=ptr(D[1]), d_dt=ptr(wide[1]),
                         d_a=ptr(D[2]), d_d=ptr(D[3]), d_dt_bias=ptr(D[4]), d_positions=ptr(pd),
                         d_slots=ptr(td), d_cache=ptr(rd), d_state=ptr(sd), d_y=ptr(wide[2]))
    lib.scan_step_device(args, stream())
    want_y = torch.zeros(batch, heads * p, dtype=F64)
    want_ring = ring.clone()
    for b in range(batch):
        s, q = int(slots[b]), int(pos[b])
        if s < 0:
            continue
        mine = ring[s].to(F64)[None].clone()
        act = conv_plain(xbc[b].to(F64)[None, None], weight.to(F64), wbias.to(F64), [1], [q], mine)
        want_ring[s, q % width] = xbc[b]
        xs, bs, cs = torch.split(act[0, 0], [heads * p, groups * n, groups * n])
        first = state[s].to(F64) if q else torch.zeros(heads, p, n, dtype=F64)
        y, end = scan_plain(xs.view(1, 1, heads, p), dt[b].to(F64).view(1, 1, heads), a.to(F64),
                            bs.view(1, 1, groups, n), cs.view(1, 1, groups, n), d.to(F64),
                            bias.to(F64), [1], first[None])
        want_y[b] = y.flatten()
        close(sd[s], end[0], "state")
    close(wide[2], want_y, "y")
    assert torch.equal(torch.nan_to_num(rd.cpu().float(), nan=-7.0),
                       torch.nan_to_num(want_ring.float(), nan=-7.0))


@pytest.mark.gpu
def test_step_beyond_32_bit_offsets(lib):
    """A state cache above 2^32 bytes: the last place's offset passes 32 bits."""
    heads, p, n, width = 8, 64, 128, 4
    slots = (1 << 32) // (heads * p * n * 4) + 3
    channels = heads * p + 2 * n
    state = torch.zeros(slots, heads, p, n, device="cuda")
    ring = torch.zeros(slots, width, channels, device="cuda")
    gen = torch.Generator().manual_seed(5)
    xbc, weight = rnd(gen, 2, channels).cuda(), rnd(gen, channels, width).cuda()
    dt, a = rnd(gen, 2, heads).cuda(), -torch.ones(heads, device="cuda")
    xbc[1], dt[1] = xbc[0], dt[0]
    pos = torch.tensor([5, 5], dtype=torch.int32, device="cuda")
    at = torch.tensor([0, slots - 1], dtype=torch.int32, device="cuda")
    y = torch.empty(2, heads * p, device="cuda")
    args = capi.StepArgs(batch=2, heads=heads, groups=1, head_dim=p, state_dim=n, width=width,
                         dtype=capi.F32, xbc_stride=channels, dt_stride=heads, y_stride=heads * p,
                         d_xbc=ptr(xbc), d_weight=ptr(weight), d_dt=ptr(dt), d_a=ptr(a),
                         d_positions=ptr(pos), d_slots=ptr(at), d_cache=ptr(ring),
                         d_state=ptr(state), d_y=ptr(y))
    lib.scan_step_device(args, stream())
    assert y[0].abs().sum() > 0 and torch.equal(y[0], y[1])
    assert torch.equal(state[0], state[-1]) and state[1].eq(0).all()
    assert torch.equal(ring[0, 1], xbc[0]) and torch.equal(ring[-1, 1], xbc[0])


# -------------------------------------------------------------------- together

@pytest.mark.gpu
def test_steps_continue_a_prompt_and_prompts_continue_each_other(lib):
    """A sequence read at once, in two prompts, and as a prompt and steps,
    through the same caches: the same outputs and states."""
    heads, groups, p, n, width, length = 4, 2, 32, 48, 4, 150
    gen = torch.Generator().manual_seed(3)
    channels = heads * p + 2 * groups * n
    xbc, dt = rnd(gen, 1, length, channels).cuda(), rnd(gen, 1, length, heads).cuda()
    weight, wbias = rnd(gen, channels, width).cuda(), rnd(gen, channels).cuda()
    a, d, bias = (-torch.exp(rnd(gen, heads))).cuda(), rnd(gen, heads).cuda(), rnd(gen, heads).cuda()

    def caches():
        return torch.zeros(1, width, channels, device="cuda"), \
            torch.zeros(1, heads, p, n, device="cuda")

    def prompt(first, last, ring, state):
        k = last - first
        pos = torch.tensor([first], dtype=torch.int32, device="cuda")
        xs, ds = xbc[:, first:last], dt[:, first:last]
        u, y = torch.empty(1, k, channels, device="cuda"), torch.empty(1, k, heads * p, device="cuda")
        lib.conv_device(capi.ConvArgs(batch=1, length=k, channels=channels, width=width, x=rows(xs),
                                      y=rows(u), d_weight=ptr(weight), d_bias=ptr(wbias),
                                      d_positions=ptr(pos), d_cache=ptr(ring)), stream())
        args = capi.ScanArgs(batch=1, length=k, heads=heads, groups=groups, head_dim=p,
                             state_dim=n, x=rows(u), b=rows(u, heads * p),
                             c=rows(u, heads * p + groups * n), dt=rows(ds), y=rows(y), d_a=ptr(a),
                             d_d=ptr(d), d_dt_bias=ptr(bias), d_positions=ptr(pos),
                             d_state=ptr(state))
        ws = workspace(lib.scan_workspace_bytes(args))
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.scan_device(args, stream())
        torch.cuda.synchronize()
        return y[0]

    def steps(first, last, ring, state):
        out = torch.empty(last - first, heads * p, device="cuda")
        for t in range(first, last):
            pos = torch.tensor([t], dtype=torch.int32, device="cuda")
            lib.scan_step_device(capi.StepArgs(
                batch=1, heads=heads, groups=groups, head_dim=p, state_dim=n, width=width,
                xbc_stride=channels, dt_stride=heads, y_stride=heads * p,
                d_xbc=ptr(xbc[0, t]), d_weight=ptr(weight), d_bias=ptr(wbias), d_dt=ptr(dt[0, t]),
                d_a=ptr(a), d_d=ptr(d), d_dt_bias=ptr(bias), d_positions=ptr(pos), d_cache=ptr(ring),
                d_state=ptr(state), d_y=ptr(out[t - first])), stream())
            torch.cuda.synchronize()
        return out

    whole, two, then = caches(), caches(), caches()
    y0 = prompt(0, length, *whole)
    y1 = torch.cat([prompt(0, 71, *two), prompt(71, length, *two)])
    y2 = torch.cat([prompt(0, 130, *then), steps(130, length, *then)])
    for y, c in ((y1, two), (y2, then)):
        close(y, y0.cpu().to(F64), "y")
        close(c[1], whole[1].cpu().to(F64), "state")
        assert torch.equal(c[0], whole[0])


def everything(lib, gen, dtype="bf16"):
    """One call of each operator on new inputs: (call, outputs)."""
    t, code = DTYPES[dtype]
    case = (2, 100, 4, 2, 64, 64, "plain")
    _, _, g2, x, dt, a, bm, cm, d, bias, lens = scan_inputs(case, dtype)
    D = on_device(case, x, dt, a, bm, cm, d, bias, lens)
    args = scan_args(case, code, *D)
    y = torch.zeros(2, 100, 256, dtype=t, device="cuda")
    args.y = rows(y)
    dy = rnd(g2, 2, 100, 256, dtype=t).cuda()
    outs = [torch.zeros_like(D[k]) for k in (0, 3, 4, 1)]
    small = [torch.zeros(4, device="cuda") for _ in range(3)]
    grads = capi.ScanGrads(dy=rows(dy), dx=rows(outs[0]), db=rows(outs[1]), dc=rows(outs[2]),
                           ddt=rows(outs[3]), d_da=ptr(small[0]), d_dd=ptr(small[1]),
                           d_ddt_bias=ptr(small[2]))
    ws = workspace(max(lib.scan_workspace_bytes(args), lib.scan_grad_workspace_bytes(args)))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    tok = torch.randint(0, 50, (3000,), generator=gen, dtype=torch.int32).cuda()
    table, rowsd = torch.zeros(50, 96, dtype=t, device="cuda"), rnd(gen, 3000, 96, dtype=t).cuda()
    emb = embed_args(50, 96, tok, table, rowsd, code, code)
    ws2 = workspace(lib.embed_grad_workspace_bytes(emb))
    emb.workspace, emb.workspace_bytes = ws2.data_ptr(), ws2.numel()
    xc, yc, w = rnd(gen, 2, 90, 64, dtype=t).cuda(), torch.zeros(2, 90, 64, dtype=t, device="cuda"), \
        rnd(gen, 64, 4, dtype=t).cuda()
    dxc, dw = torch.zeros_like(yc), torch.zeros(64, 4, device="cuda")
    conv = capi.ConvArgs(batch=2, length=90, channels=64, width=4, dtype=code, x=rows(xc), y=rows(yc),
                         d_weight=ptr(w))
    ws3 = workspace(lib.conv_grad_workspace_bytes(conv))
    conv.workspace, conv.workspace_bytes = ws3.data_ptr(), ws3.numel()
    keep = (D, dy, ws, tok, rowsd, ws2, xc, w, ws3)

    def call():
        s = stream()
        lib.scan_device(args, s)
        lib.scan_grad_device(args, grads, s)
        lib.embed_grad_device(emb, s)
        lib.conv_device(conv, s)
        lib.conv_grad_device(conv, capi.ConvGrads(dy=rows(yc), dx=rows(dxc), d_dweight=ptr(dw)), s)
        return keep

    return call, [y, *outs, *small, table, yc, dxc, dw]


@pytest.mark.gpu
def test_graph_replays_equal_eager_calls(lib):
    gen = torch.Generator().manual_seed(11)
    call, outs = everything(lib, gen)
    call()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for _ in range(4):
        for o in outs:
            o.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
        call()  # the program's own eager work between replays
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


@pytest.mark.gpu
def test_calls_on_other_streams(lib):
    gen = torch.Generator().manual_seed(12)
    sets = [everything(lib, gen) for _ in range(2)]
    wants = []
    for call, outs in sets:
        call()
        torch.cuda.synchronize()
        wants.append([o.clone() for o in outs])
        for o in outs:
            o.fill_(3.0)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        for (call, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                call()
    torch.cuda.synchronize()
    for (_, outs), want in zip(sets, wants):
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


# -------------------------------------------------------------------- refusals

A = 0x10000  # a device pointer that no refused call reads


def good_embed(**kw):
    return capi.EmbedArgs(**{**dict(tokens=4, rows=4, width=8, table_stride=8, out_stride=8,
                                    d_table=A, d_tokens=A, d_out=A, workspace=A,
                                    workspace_bytes=1 << 30), **kw})


def good_conv(**kw):
    return capi.ConvArgs(**{**dict(batch=2, length=8, channels=8, width=4, x=(A, 64, 8),
                                   y=(A, 64, 8), d_weight=A, workspace=A,
                                   workspace_bytes=1 << 30), **kw})


def good_scan(**kw):
    return capi.ScanArgs(**{**dict(batch=2, length=8, heads=4, groups=2, head_dim=8, state_dim=8,
                                   x=(A, 256, 32), b=(A, 128, 16), c=(A, 128, 16), dt=(A, 32, 4),
                                   y=(A, 256, 32), d_a=A, workspace=A,
                                   workspace_bytes=1 << 30), **kw})


def good_grads(**kw):
    return capi.ScanGrads(**{**dict(dy=(A, 256, 32), dx=(A, 256, 32), db=(A, 128, 16),
                                    dc=(A, 128, 16), ddt=(A, 32, 4), d_da=A), **kw})


def good_step(**kw):
    return capi.StepArgs(**{**dict(batch=2, heads=4, groups=2, head_dim=8, state_dim=8, width=4,
                                   xbc_stride=64, dt_stride=4, y_stride=32, d_xbc=A, d_weight=A,
                                   d_dt=A, d_a=A, d_positions=A, d_cache=A, d_state=A, d_y=A), **kw})


EINVAL, EUNSUPPORTED = capi.NSFPS_EINVAL, capi.NSFPS_EUNSUPPORTED
REFUSED = [
    ("embed", good_embed, dict(width=0), EINVAL), ("embed", good_embed, dict(dtype=2), EINVAL),
    ("embed", good_embed, dict(out_stride=7), EINVAL),
    ("embed", good_embed, dict(d_tokens=None), EINVAL),
    ("embed", good_embed, dict(d_table=A + 2), EINVAL),
    ("embed", good_embed, dict(table_stride=1 << 62), EINVAL),
    ("embed", good_embed, dict(tokens=1 << 31), EUNSUPPORTED),
    ("embed", good_embed, dict(width=65537, table_stride=65537, out_stride=65537), EUNSUPPORTED),
    ("embed_grad", good_embed, dict(grad_dtype=9), EINVAL),
    ("embed_grad", good_embed, dict(workspace_bytes=16), EINVAL),
    ("embed_grad", good_embed, dict(workspace=None), EINVAL),
    ("embed_grad", good_embed, dict(workspace=A + 16), EINVAL),
    ("conv", good_conv, dict(width=1), EUNSUPPORTED), ("conv", good_conv, dict(width=5), EUNSUPPORTED),
    ("conv", good_conv, dict(channels=0), EINVAL), ("conv", good_conv, dict(y=(A, 64, 7)), EINVAL),
    ("conv", good_conv, dict(y=(A, 63, 8)), EINVAL), ("conv", good_conv, dict(x=(None, 64, 8)), EINVAL),
    ("conv", good_conv, dict(d_weight=None), EINVAL),
    ("conv", good_conv, dict(d_positions=A), EINVAL),  # no cache to continue from
    ("conv", good_conv, dict(d_lengths=A + 2), EINVAL),
    ("conv", good_conv, dict(length=1 << 31), EUNSUPPORTED),
    ("conv_grad", good_conv, dict(d_cache=A), EINVAL), ("conv_grad", good_conv, dict(d_slots=A), EINVAL),
    ("conv_grad", good_conv, dict(workspace_bytes=8), EINVAL),
    ("scan", good_scan, dict(groups=3), EINVAL), ("scan", good_scan, dict(heads=0), EINVAL),
    ("scan", good_scan, dict(head_dim=129), EUNSUPPORTED),
    ("scan", good_scan, dict(state_dim=129), EUNSUPPORTED),
    ("scan", good_scan, dict(dtype=7), EINVAL), ("scan", good_scan, dict(d_a=None), EINVAL),
    ("scan", good_scan, dict(y=(A, 255, 32)), EINVAL), ("scan", good_scan, dict(d_positions=A), EINVAL),
    ("scan", good_scan, dict(batch=1 << 20), EUNSUPPORTED),
    ("scan", good_scan, dict(workspace_bytes=8), EINVAL),
    ("scan_grad", good_scan, dict(d_state=A), EINVAL),
    ("scan_grad", good_scan, dict(workspace=None), EINVAL),
    ("scan_step", good_step, dict(width=5), EUNSUPPORTED),
    ("scan_step", good_step, dict(d_positions=None), EINVAL),
    ("scan_step", good_step, dict(y_stride=31), EINVAL), ("scan_step", good_step, dict(d_state=None), EINVAL),
    ("scan_step", good_step, dict(groups=0), EINVAL),
]


def call_by_name(L, name, args):
    if name == "conv_grad":
        return L.conv_grad_device(args, capi.ConvGrads(dy=(A, 64, 8), dx=(A, 64, 8), d_dweight=A))
    if name == "scan_grad":
        return L.scan_grad_device(args, good_grads())
    return getattr(L, f"{name}_device")(args)


@pytest.mark.parametrize("name,make,change,status", REFUSED)
def test_refusals(name, make, change, status):
    """Every refused call names its reason and enqueues nothing (no pointer
    here is one, and no device is needed)."""
    L = capi.Lib()
    with pytest.raises(capi.NsfpsError) as e:
        call_by_name(L, name, make(**change))
    assert e.value.status == status
    assert len(str(e.value)) > len("nsfps status 1: ")


def test_null_structs_are_refused():
    L = capi.Lib()
    for name in ("embed", "embed_grad", "conv", "scan", "scan_step"):
        fn = getattr(L.lib, f"nsfps_{name}_device")
        assert fn(None, None) == EINVAL
    assert L.lib.nsfps_scan_grad_device(good_scan(), None, None) == EINVAL
    assert L.lib.nsfps_scan_workspace_bytes(None, ctypes.c_uint64()) == EINVAL
    assert L.lib.nsfps_scan_workspace_bytes(good_scan(), None) == EINVAL


@pytest.mark.parametrize("args,call", [
    (good_embed(tokens=0, d_tokens=None, d_out=None), "embed"),
    (good_conv(length=0, x=(None, 0, 0), y=(None, 0, 0)), "conv"),
    (good_scan(batch=0, x=(None, 0, 0)), "scan"), (good_step(batch=0, d_xbc=None), "scan_step")])
def test_empty_calls_do_nothing(args, call):
    getattr(capi.Lib(), f"{call}_device")(args)


def test_overlapping_strides_that_repeat_inputs_are_taken():
    """A broadcast input (a stride of 0) is fine to read, not to write."""
    L = capi.Lib()
    n = L.scan_workspace_bytes(good_scan(b=(A, 0, 16)))
    assert n > 0
    with pytest.raises(capi.NsfpsError):
        L.scan_device(good_scan(y=(A, 0, 32)))


@pytest.mark.parametrize("name,struct", [
    ("nsfps_rows", capi.Rows), ("nsfps_embed_args", capi.EmbedArgs), ("nsfps_conv_args", capi.ConvArgs),
    ("nsfps_conv_grads", capi.ConvGrads), ("nsfps_scan_args", capi.ScanArgs),
    ("nsfps_scan_grads", capi.ScanGrads), ("nsfps_step_args", capi.StepArgs)])
def test_bindings_mirror_the_header(name, struct, tmp_path):
    """Sizes and offsets of every field as the C compiler lays them out."""
    import os
    import subprocess
    from conftest import ROOT
    fields = [f for f, _ in struct._fields_]
    prints = "".join(f'printf("%zu ", offsetof({name}, {f}));' for f in fields)
    src = tmp_path / "layout.c"
    src.write_text('#include "nsfps.h"\n#include <stddef.h>\n#include <stdio.h>\n'
                   f'int main(void) {{ {prints} printf("%zu", sizeof({name})); return 0; }}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    want = [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]
    assert np.array_equal([int(v) for v in out], want)
