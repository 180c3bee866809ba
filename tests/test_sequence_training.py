"""The operators of a training step together: lookup, convolution, norms with
rotation, scan, dropout onto the residual and the vocabulary loss, forward and
back, against one 64-bit model with automatic derivatives; and a prompt followed
by single tokens through convolution, norms and scan.

Tolerance.  Every operator keeps about 2^-18 of its terms' sizes in float32 (their
own tests); six of them follow each other, forward and back, which leaves 2^-13
of a gradient's norm for what adds up."""

import pytest
import torch

from ns_fps_amd import capi
from test_dropout import keep_of
from test_sequence import F64, lib, ptr, rnd, rows, scan_plain, silu, stream, \
    workspace  # noqa: F401
from test_head_norm import EPS, angles, norm_plain

B, L, HEADS, GROUPS, P, N, WIDTH, MODEL, VOCAB, DROP = 2, 75, 4, 2, 16, 24, 4, 40, 90, 0.2
INNER, CHANNELS = HEADS * P, HEADS * P + 2 * GROUPS * N
LENS, SEED = [75, 50], [123456789, 5]


def parameters(gen):
    return {"table": rnd(gen, VOCAB, MODEL), "w_in": rnd(gen, MODEL, CHANNELS + HEADS, scale=0.2),
            "conv_w": rnd(gen, CHANNELS, WIDTH, scale=0.5), "conv_b": rnd(gen, CHANNELS, scale=0.1),
            "b_weight": 1 + rnd(gen, N, scale=0.1), "c_weight": 1 + rnd(gen, N, scale=0.1),
            "a": -torch.exp(rnd(gen, HEADS)), "d": rnd(gen, HEADS), "dt_bias": rnd(gen, HEADS) - 2,
            "w_out": rnd(gen, INNER, MODEL, scale=0.2)}


FREQ = 100.0 ** (-torch.arange(N // 2, dtype=F64) / (N // 2))


def step(lib, p, tokens, target, dloss, lens, seed, freq):  # noqa: F811
    """Losses and gradients on the device, and what has to be kept meanwhile."""
    def new(*shape):
        return torch.full(shape, float("nan"), device="cuda")

    def embed(table, out):
        return capi.EmbedArgs(tokens=B * L, rows=VOCAB, width=MODEL, scale=2.0, table_stride=MODEL,
                              out_stride=MODEL, d_table=ptr(table), d_tokens=ptr(tokens),
                              d_out=ptr(out))
    s, held = stream(), []

    def give(args, nbytes):
        held.append(workspace(nbytes))
        args.workspace, args.workspace_bytes = held[-1].data_ptr(), held[-1].numel()

    e = new(B, L, MODEL)
    lib.embed_device(embed(p["table"], e), s)
    u = e @ p["w_in"]
    v, bc, y = new(B, L, CHANNELS), new(B, L, 2 * GROUPS * N), new(B, L, INNER)
    conv = capi.ConvArgs(batch=B, length=L, channels=CHANNELS, width=WIDTH, x=rows(u), y=rows(v),
                         d_weight=ptr(p["conv_w"]), d_bias=ptr(p["conv_b"]), d_lengths=ptr(lens))
    lib.conv_device(conv, s)
    norm = capi.NormArgs(batch=B, length=L, q_heads=GROUPS, k_heads=GROUPS, head_dim=N, rotary_dim=N,
                         eps=EPS, k=rows(v, INNER), q=rows(v, INNER + GROUPS * N), k_out=rows(bc),
                         q_out=rows(bc, GROUPS * N), d_k_weight=ptr(p["b_weight"]),
                         d_q_weight=ptr(p["c_weight"]), d_freq=ptr(freq), d_lengths=ptr(lens))
    lib.norm_device(norm, s)
    scan = capi.ScanArgs(batch=B, length=L, heads=HEADS, groups=GROUPS, head_dim=P, state_dim=N,
                         x=rows(v), b=rows(bc), c=rows(bc, GROUPS * N), dt=rows(u, CHANNELS),
                         y=rows(y), d_a=ptr(p["a"]), d_d=ptr(p["d"]), d_dt_bias=ptr(p["dt_bias"]),
                         d_lengths=ptr(lens))
    give(scan, max(lib.scan_workspace_bytes(scan), lib.scan_grad_workspace_bytes(scan)))
    lib.scan_device(scan, s)
    o = y @ p["w_out"]
    h = new(B, L, MODEL)
    drop = capi.DropoutArgs(batch=B, length=L, channels=MODEL, p=DROP, x=rows(o), residual=rows(e),
                            y=rows(h), d_seed=ptr(seed), d_lengths=ptr(lens))
    lib.dropout_device(drop, s)
    loss, lse = new(B * L), new(B * L)
    args = capi.LossArgs(tokens=B * L, rows=VOCAB, width=MODEL, scale=0.25, x_stride=MODEL,
                         table_stride=MODEL, d_x=ptr(h), d_table=ptr(p["table"]),
                         d_targets=ptr(target), d_loss=ptr(loss), d_lse=ptr(lse))
    g = {k: torch.full_like(t, float("nan")) for k, t in p.items()}
    dh, tied = new(B, L, MODEL), new(VOCAB, MODEL)
    grads = capi.LossGrads(d_dloss=ptr(dloss), dx_stride=MODEL, dtable_stride=MODEL, d_dx=ptr(dh),
                           d_dtable=ptr(tied))
    give(args, max(lib.loss_workspace_bytes(args), lib.loss_grad_workspace_bytes(args, grads)))
    lib.loss_device(args, s)
    lib.loss_grad_device(args, grads, s)
    do = new(B, L, MODEL)
    lib.dropout_device(capi.DropoutArgs(batch=B, length=L, channels=MODEL, p=DROP, x=rows(dh),
                                        y=rows(do), d_seed=ptr(seed), d_lengths=ptr(lens)), s)
    g["w_out"] = y.flatten(0, 1).T @ do.flatten(0, 1)
    dy, dv, dbc, du = do @ p["w_out"].T, new(B, L, CHANNELS), new(B, L, 2 * GROUPS * N), \
        new(B, L, CHANNELS + HEADS)
    lib.scan_grad_device(scan, capi.ScanGrads(
        dy=rows(dy), dx=rows(dv), db=rows(dbc), dc=rows(dbc, GROUPS * N), ddt=rows(du, CHANNELS),
        d_da=ptr(g["a"]), d_dd=ptr(g["d"]), d_ddt_bias=ptr(g["dt_bias"])), s)
    give(norm, lib.norm_grad_workspace_bytes(norm))
    lib.norm_grad_device(norm, capi.NormGrads(
        dk_out=rows(dbc), dq_out=rows(dbc, GROUPS * N), dk=rows(dv, INNER),
        dq=rows(dv, INNER + GROUPS * N), d_dk_weight=ptr(g["b_weight"]),
        d_dq_weight=ptr(g["c_weight"])), s)
    give(conv, lib.conv_grad_workspace_bytes(conv))
    lib.conv_grad_device(conv, capi.ConvGrads(dy=rows(dv), dx=rows(du), d_dweight=ptr(g["conv_w"]),
                                              d_dbias=ptr(g["conv_b"])), s)
    g["w_in"] = e.flatten(0, 1).T @ du.flatten(0, 1)
    de = (du @ p["w_in"].T + dh).contiguous()
    back = embed(g["table"], de)
    give(back, lib.embed_grad_workspace_bytes(back))
    lib.embed_grad_device(back, s)
    g["table"] += tied
    return loss, g, (held, u, v, bc, y, o, h, dh, do, dy, dv, dbc, du, de, e)


def model(p, tokens, target, dloss):
    """The same in float64."""
    keep = keep_of(B, L, MODEL, DROP, SEED)
    inside = torch.tensor([[t < n for t in range(L)] for n in LENS])[..., None]
    e = 2.0 * p["table"][tokens.long().clamp(0)] * (tokens >= 0)[..., None]
    u = e @ p["w_in"]
    seen = torch.cat([torch.zeros(B, WIDTH - 1, CHANNELS, dtype=F64), u[..., :CHANNELS]], 1)
    v = silu(sum(p["conv_w"][:, k] * seen[:, k:k + L] for k in range(WIDTH)) + p["conv_b"]) * inside
    x, bm, cm = torch.split(v, [INNER, GROUPS * N, GROUPS * N], -1)
    turn = angles([0] * B, L, FREQ)
    bm, cm = (norm_plain(t.reshape(B, L, GROUPS, N), w, turn, 0)
              for t, w in ((bm, p["b_weight"]), (cm, p["c_weight"])))
    y, _ = scan_plain(x.reshape(B, L, HEADS, P), u[..., CHANNELS:], p["a"], bm, cm, p["d"],
                      p["dt_bias"], LENS, torch.zeros(B, HEADS, P, N, dtype=F64))
    o = y.flatten(2) @ p["w_out"]
    kept = 65536 / (65536 - round(DROP * 65536))
    h = (e + torch.where(keep, o * kept, 0.0)) * inside
    z = 0.25 * h.flatten(0, 1) @ p["table"].T
    at = target.flatten().long()
    losses = torch.logsumexp(z, 1) - z.gather(1, at.clamp(0)[:, None])[:, 0]
    losses = torch.where(at >= 0, losses, 0.0)
    return losses, (losses * dloss.to(F64)).sum()


@pytest.mark.gpu
def test_a_training_step(lib):  # noqa: F811
    gen = torch.Generator().manual_seed(17)
    p = parameters(gen)
    tokens = torch.randint(0, VOCAB, (B, L), generator=gen, dtype=torch.int32)
    target = torch.randint(0, VOCAB, (B, L), generator=gen, dtype=torch.int32)
    for b, n in enumerate(LENS):
        tokens[b, n:], target[b, n - 1:] = -1, -1
    dloss = rnd(gen, B * L)
    on = {k: t.cuda() for k, t in p.items()}
    loss, grads, held = step(lib, on, tokens.cuda(), target.cuda(), dloss.cuda(),
                             torch.tensor(LENS, dtype=torch.int32).cuda(),
                             torch.tensor(SEED, dtype=torch.int64).cuda(), FREQ.float().cuda())
    torch.cuda.synchronize()
    leaves = {k: t.to(F64).requires_grad_() for k, t in p.items()}
    losses, total = model(leaves, tokens, target, dloss)
    want = dict(zip(leaves, torch.autograd.grad(total, list(leaves.values()))))
    off = (loss.cpu().to(F64) - losses.detach()).norm() / losses.detach().norm()
    assert off <= 2.0 ** -13, off
    for k, g in grads.items():
        off = (g.cpu().to(F64) - want[k]).norm() / want[k].norm()
        assert off <= 2.0 ** -13, (k, off.item())
    del held


@pytest.mark.gpu
def test_single_tokens_continue_a_prompt(lib):  # noqa: F811
    """Convolution, norms and scan over a whole sequence, and over a prompt and
    then one token a call (length 1, positions, caches): the same outputs."""
    gen = torch.Generator().manual_seed(4)
    p = {k: t.cuda() for k, t in parameters(gen).items()}
    u = rnd(gen, 1, L, CHANNELS + HEADS).cuda()
    freq = FREQ.float().cuda()

    def run(first, last, ring, state):
        k = last - first
        x = u[:, first:last]
        pos = torch.tensor([first], dtype=torch.int32, device="cuda")
        v, bc = torch.empty(1, k, CHANNELS, device="cuda"), torch.empty(1, k, 2 * GROUPS * N,
                                                                        device="cuda")
        y = torch.empty(1, k, INNER, device="cuda")
        lib.conv_device(capi.ConvArgs(batch=1, length=k, channels=CHANNELS, width=WIDTH, x=rows(x),
                                      y=rows(v), d_weight=ptr(p["conv_w"]), d_bias=ptr(p["conv_b"]),
                                      d_positions=ptr(pos), d_cache=ptr(ring)), stream())
        lib.norm_device(capi.NormArgs(
            batch=1, length=k, q_heads=GROUPS, k_heads=GROUPS, head_dim=N, rotary_dim=N, eps=EPS,
            k=rows(v, INNER), q=rows(v, INNER + GROUPS * N), k_out=rows(bc),
            q_out=rows(bc, GROUPS * N), d_k_weight=ptr(p["b_weight"]),
            d_q_weight=ptr(p["c_weight"]), d_freq=ptr(freq), d_positions=ptr(pos)), stream())
        scan = capi.ScanArgs(batch=1, length=k, heads=HEADS, groups=GROUPS, head_dim=P, state_dim=N,
                             x=rows(v), b=rows(bc), c=rows(bc, GROUPS * N), dt=rows(x, CHANNELS),
                             y=rows(y), d_a=ptr(p["a"]), d_d=ptr(p["d"]), d_dt_bias=ptr(p["dt_bias"]),
                             d_positions=ptr(pos), d_state=ptr(state))
        ws = workspace(lib.scan_workspace_bytes(scan))
        scan.workspace, scan.workspace_bytes = ws.data_ptr(), ws.numel()
        lib.scan_device(scan, stream())
        torch.cuda.synchronize()
        return y[0], bc[0]

    def caches():
        return torch.zeros(1, WIDTH, CHANNELS, device="cuda"), torch.zeros(1, HEADS, P, N,
                                                                           device="cuda")
    whole, bc = run(0, L, *caches())
    c = caches()
    parts = [run(0, 40, *c)] + [run(t, t + 1, *c) for t in range(40, L)]
    assert torch.equal(torch.cat([q[1] for q in parts]), bc)  # each token's norms on their own
    y = torch.cat([q[0] for q in parts])
    assert (y - whole).norm() <= 2.0 ** -14 * whole.norm()


@pytest.mark.gpu
def test_steps_in_a_graph_and_on_streams(lib):  # noqa: F811
    """The calls of a training step captured once and replayed equal the eager
    calls; two steps on two streams do not disturb each other."""
    gen = torch.Generator().manual_seed(8)
    lens = torch.tensor(LENS, dtype=torch.int32).cuda()
    seed, freq = torch.tensor(SEED, dtype=torch.int64).cuda(), FREQ.float().cuda()
    x = rnd(gen, B, L, CHANNELS).cuda()
    g = rnd(gen, B, L, 2 * GROUPS * N).cuda()
    w = (1 + rnd(gen, N, scale=0.1)).cuda()

    def make():
        outs = [torch.zeros(B, L, 2 * GROUPS * N, device="cuda") for _ in range(3)]
        outs += [torch.zeros(N, device="cuda") for _ in range(2)]
        norm = capi.NormArgs(batch=B, length=L, q_heads=GROUPS, k_heads=GROUPS, head_dim=N,
                             rotary_dim=N, eps=EPS, k=rows(x, INNER), q=rows(x, INNER + GROUPS * N),
                             k_out=rows(outs[0]), q_out=rows(outs[0], GROUPS * N), d_k_weight=ptr(w),
                             d_q_weight=ptr(w), d_freq=ptr(freq), d_lengths=ptr(lens))
        ws = workspace(lib.norm_grad_workspace_bytes(norm))
        norm.workspace, norm.workspace_bytes = ws.data_ptr(), ws.numel()
        grads = capi.NormGrads(dk_out=rows(g), dq_out=rows(g, GROUPS * N), dk=rows(outs[1]),
                               dq=rows(outs[1], GROUPS * N), d_dk_weight=ptr(outs[3]),
                               d_dq_weight=ptr(outs[4]))
        drop = capi.DropoutArgs(batch=B, length=L, channels=2 * GROUPS * N, p=DROP, x=rows(outs[0]),
                                residual=rows(g), y=rows(outs[2]), d_seed=ptr(seed),
                                d_lengths=ptr(lens))

        def call():
            lib.norm_device(norm, stream())
            lib.norm_grad_device(norm, grads, stream())
            lib.dropout_device(drop, stream())
            return ws
        return call, outs

    call, outs = make()
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
        assert all(torch.equal(o, q) for o, q in zip(outs, want))
        call()
        torch.cuda.synchronize()
        assert all(torch.equal(o, q) for o, q in zip(outs, want))
    sets, streams = [make() for _ in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for (one, _), st in zip(sets, streams):
            with torch.cuda.stream(st):
                one()
    torch.cuda.synchronize()
    for _, got in sets:
        assert all(torch.equal(o, q) for o, q in zip(got, want))


@pytest.mark.gpu
def test_rows_beyond_32_bit_offsets(lib):  # noqa: F811
    """Sequences more than 2^32 elements apart, in norms and dropout."""
    far = (1 << 31) + 64
    x = torch.zeros(2 * far, dtype=torch.bfloat16, device="cuda")
    row = torch.randn(64, device="cuda").bfloat16()
    x[:64], x[far:far + 64] = row, row
    y = torch.zeros_like(x)
    at = (x.data_ptr(), far, 64)
    lib.norm_device(capi.NormArgs(batch=2, length=1, q_heads=1, head_dim=64, dtype=capi.BF16,
                                  eps=EPS, q=at, q_out=(y.data_ptr(), far, 64)), stream())
    assert y[:64].ne(0).any() and torch.equal(y[:64], y[far:far + 64]) and y[64:far].eq(0).all()
    seed = torch.tensor(SEED, dtype=torch.int64).cuda()
    lib.dropout_device(capi.DropoutArgs(batch=2, length=1, channels=64, dtype=capi.BF16, p=0.0, x=at,
                                        y=(y.data_ptr(), far, 64), d_seed=ptr(seed)), stream())
    assert torch.equal(y[:64], row) and torch.equal(y[far:far + 64], row)
