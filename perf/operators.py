"""The operators of a sequence model over sampled points, as a program uses them.

Samples of a cloud, put in the order of their grid cells, are the tokens of a
sequence model: the cell is the token (a vocabulary of ``total_blocks`` rows),
and a selective state space scan with its short causal convolution mixes the
sequence.  Operators (``op``):

* ``lookup``       rows of an embedding table by token, times a scale
* ``lookup_grad``  the table's gradient from the rows' gradients
* ``conv``         short causal convolution and SiLU; with ``train`` its gradient too
* ``scan``         selective scan over prompts; with ``train`` its gradient too
* ``step``         one token of every request: convolution and scan over the caches

``own`` false computes them from elementary torch operations in 32 bits;
``own`` true calls ns_fps_amd.  Types: ``bf16`` or ``f32``; A, D, the step
bias, states and parameter gradients are float32 with both.
"""

import math

import torch
import torch.nn.functional as F

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
_CHUNK = 64  # tokens a chunk of the plain scan


# ------------------------------------------------------------------ the cases

def _lookup(op, tokens, rows, width, dtype):
    return {"op": op, "tokens": tokens, "rows": rows, "width": width, "dtype": dtype}


def _conv(batch, length, channels, width, dtype, train=False, ragged=False, resume=False):
    return {"op": "conv", "batch": batch, "length": length, "channels": channels,
            "width": width, "dtype": dtype, "train": train, "ragged": ragged, "resume": resume}


def _scan(batch, length, heads, groups, head_dim, state_dim, dtype, train=False, ragged=False,
          resume=False):
    return {"op": "scan", "batch": batch, "length": length, "heads": heads, "groups": groups,
            "head_dim": head_dim, "state_dim": state_dim, "dtype": dtype, "train": train,
            "ragged": ragged, "resume": resume}


def _step(batch, slots, heads, groups, head_dim, state_dim, width, dtype):
    return {"op": "step", "batch": batch, "slots": slots, "heads": heads, "groups": groups,
            "head_dim": head_dim, "state_dim": state_dim, "width": width, "dtype": dtype}


def listed():
    return [
        # the quickstart call's 1,000 samples over its 16^3 grid: latency counts
        dict(_lookup("lookup", 1000, 4096, 384, "bf16"), name="lookup_quickstart"),
        # every sample of the 8M-point cloud, a 64^3 vocabulary
        dict(_lookup("lookup", 524288, 262144, 256, "bf16"), name="lookup_clustered"),
        # a LiDAR scan's samples over its 32 x 32 x 8 grid, an odd width, full precision
        dict(_lookup("lookup_grad", 16384, 8192, 383, "f32"), name="lookup_grad_lidar"),
        # the largest training batch of tokens
        dict(_lookup("lookup_grad", 524288, 262144, 256, "bf16"), name="lookup_grad_clustered"),
        # one scan's samples appended to a sequence, odd channels, full precision
        dict(_conv(1, 16384, 323, 3, "f32", resume=True), name="conv_lidar_f32"),
        # a training batch: 64 clouds of up to 4,096 samples, fewer where a cloud ended early
        dict(_conv(64, 4096, 640, 4, "bf16", train=True, ragged=True), name="conv_train_batched"),
        # one quickstart cloud as a prompt
        dict(_scan(1, 1000, 8, 1, 64, 64, "bf16"), name="scan_quickstart"),
        # one long prompt, 65,536 samples of the 1M-point cube: the split over the long axis
        dict(_scan(1, 65536, 8, 1, 64, 128, "bf16"), name="scan_long"),
        # a training batch of ragged clouds, heads sharing one group
        dict(_scan(64, 4096, 8, 1, 64, 64, "bf16", train=True, ragged=True),
             name="scan_train_batched"),
        # a small model in full precision, odd sizes, several groups
        dict(_scan(3, 1001, 6, 3, 48, 33, "f32", train=True), name="scan_train_odd_f32"),
        # one request served alone
        dict(_step(1, 16, 8, 1, 64, 128, 4, "bf16"), name="step_one"),
        # a full serving batch
        dict(_step(512, 1024, 16, 2, 64, 128, 4, "bf16"), name="step_512"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng, most):
    groups = rng.choice([1, 1, 2, 4])
    return groups * rng.randint(1, max(1, most // groups)), groups


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "conv", "conv", "scan", "scan", "scan", "step"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    room = 1 if dtype == "bf16" else 2  # full precision costs more a value
    if op in ("lookup", "lookup_grad"):
        width = _log_int(rng, 16, 1024)
        most = 524288 * 256 // room // width
        return _lookup(op, _log_int(rng, 1, min(524288, most)), _log_int(rng, 64, min(262144, most)),
                       width, dtype)
    if op == "step":
        heads, groups = _heads(rng, 16)
        batch = _log_int(rng, 1, 512)
        return _step(batch, batch + rng.randint(0, 512), heads, groups, rng.randint(16, 64),
                     rng.randint(16, 128), rng.choice([2, 3, 4]), dtype)
    train, ragged = rng.random() < 0.5, rng.random() < 0.5
    resume = not train and rng.random() < 0.5
    batch = _log_int(rng, 1, 64)
    length = _log_int(rng, 1, min(65536, 262144 // room // batch))
    if op == "conv":
        channels = _log_int(rng, 32, min(2048, 167772160 // room // (batch * length)))
        return _conv(batch, length, channels, rng.choice([2, 3, 4]), dtype, train, ragged, resume)
    heads, groups = _heads(rng, 8)
    head_dim = rng.choice([32, 64, rng.randint(16, 64)])
    state_dim = rng.choice([16, 64, 128, rng.randint(16, 128)])
    if train or dtype == "f32":  # at most the training batch's work
        length = min(length, max(1, 262144 * 8 * 64 * 64 // 2 //
                                 (batch * heads * head_dim * state_dim)))
    return _scan(batch, length, heads, groups, head_dim, state_dim, dtype, train, ragged, resume)


# ------------------------------------------------------------------ the inputs

def _tokens(gen, count, rows):
    """Cells of samples: crowded cells near the objects, and 1 in 64 the -1
    that pads the row of a cloud that ended early."""
    u = torch.rand(count, generator=gen, device="cuda")
    cell = torch.clamp((u * u * rows).to(torch.int64), max=rows - 1)
    cell = (cell * 40503) % rows if rows % 40503 else cell  # crowded cells lie anywhere
    pad = torch.rand(count, generator=gen, device="cuda") < 1 / 64
    return torch.where(pad, -1, cell).to(torch.int32)


def _lengths(gen, case):
    b, length = case["batch"], case["length"]
    if not case["ragged"]:
        return None
    f = 0.5 + 0.5 * torch.rand(b, generator=gen, device="cuda")
    return (f * length).ceil().to(torch.int32)


def _step_bias(gen, heads):
    """Inverse softplus of step sizes spread over 0.001 to 0.1."""
    step = torch.exp(torch.rand(heads, generator=gen, device="cuda") * math.log(100.0)
                     + math.log(0.001))
    return step + torch.log(-torch.expm1(-step))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = {"case": case, "dtype": dtype}
    if op in ("lookup", "lookup_grad"):
        s["tokens"] = _tokens(gen, case["tokens"], case["rows"])
        s["scale"] = math.sqrt(case["width"])
        if op == "lookup":
            s["table"] = normal(case["rows"], case["width"], scale=0.02)
        else:
            s["dout"] = normal(case["tokens"], case["width"], scale=0.01)
        return s

    b = case["batch"]
    if op == "step":
        h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
        channels = h * p + 2 * g * n
        s["xbc"] = normal(b, channels)
        s["weight"] = normal(channels, case["width"], scale=0.5)
        s["bias"] = normal(channels, scale=0.1)
        s["dt"] = normal(b, h, scale=0.5)
        s["a"] = -1.0 - 15.0 * torch.rand(h, generator=gen, device="cuda")
        s["d"] = 1.0 + 0.1 * torch.randn(h, generator=gen, device="cuda")
        s["dt_bias"] = _step_bias(gen, h)
        s["slots"] = torch.randperm(case["slots"], generator=gen, device="cuda")[:b].to(torch.int32)
        s["positions"] = torch.randint(0, 5000, (b,), generator=gen, device="cuda",
                                       dtype=torch.int32)
        s["ring"] = normal(case["slots"], case["width"], channels)
        s["state"] = normal(case["slots"], h, p, n, scale=0.1, dtype=torch.float32)
        return s

    length = case["length"]
    s["lengths"] = _lengths(gen, case)
    s["positions"] = torch.randint(1, 5000, (b,), generator=gen, device="cuda",
                                   dtype=torch.int32) if case["resume"] else None
    if op == "conv":
        c, w = case["channels"], case["width"]
        s["x"] = normal(b, length, c)
        s["weight"] = normal(c, w, scale=0.5)
        s["bias"] = normal(c, scale=0.1)
        if case["train"]:
            s["dy"] = normal(b, length, c, scale=0.1)
        else:
            s["ring"] = normal(b, w, c)
        return s
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    s["xbc"] = F.silu(normal(b, length, h * p + 2 * g * n, dtype=torch.float32)).to(dtype)
    s["dt"] = normal(b, length, h, scale=0.5)
    s["a"] = -1.0 - 15.0 * torch.rand(h, generator=gen, device="cuda")
    s["d"] = 1.0 + 0.1 * torch.randn(h, generator=gen, device="cuda")
    s["dt_bias"] = _step_bias(gen, h)
    if case["train"]:
        s["dy"] = normal(b, length, h, p, scale=0.1)
    else:
        s["state"] = normal(b, h, p, n, scale=0.1, dtype=torch.float32)
    return s


# ------------------------------------------------------------- the plain forms

def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _silu(v):
    return v / (1 + torch.exp(-v))


def _split(xbc, case):
    """x [.., H, P], B and C [.., G, N] of a row [.., H P + 2 G N]."""
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    x, bm, cm = torch.split(xbc, [h * p, g * n, g * n], dim=-1)
    return x.unflatten(-1, (h, p)), bm.unflatten(-1, (g, n)), cm.unflatten(-1, (g, n))


def _plain_lookup(s):
    tok = s["tokens"].long()
    hit = (tok >= 0) & (tok < s["table"].shape[0])
    rows = s["table"][torch.where(hit, tok, 0)].float() * s["scale"]
    return torch.where(hit[:, None], rows, 0.0).to(s["dtype"])


def _plain_lookup_grad(s):
    rows = s["case"]["rows"]
    tok = s["tokens"].long()
    hit = (tok >= 0) & (tok < rows)
    grad = torch.zeros(rows + 1, s["dout"].shape[1], device="cuda")
    grad.index_add_(0, torch.where(hit, tok, rows), s["dout"].float())
    return (grad[:rows] * s["scale"]).to(s["dtype"])


def _inside(s):
    """[B, L]: which tokens are inside their row's length."""
    case = s["case"]
    t = torch.arange(case["length"], device="cuda")
    if s["lengths"] is None:
        return torch.ones(case["batch"], case["length"], dtype=torch.bool, device="cuda")
    return t[None] < s["lengths"][:, None]


def _plain_conv(x, weight, bias, before, inside):
    """SiLU of the convolution; ``before``: the width - 1 tokens ahead of x."""
    seen = torch.cat([before, torch.where(inside[..., None], x, 0.0)], dim=1)
    pre = (seen.unfold(1, weight.shape[1], 1) * weight).sum(-1) + bias
    return torch.where(inside[..., None], _silu(pre), 0.0)


def _plain_conv_prompt(s):
    case, width = s["case"], s["case"]["width"]
    x, ring, inside = s["x"].float(), s["ring"], _inside(s)
    pos = torch.zeros(case["batch"], dtype=torch.long, device="cuda") \
        if s["positions"] is None else s["positions"].long()
    back = pos[:, None] - torch.arange(width - 1, 0, -1, device="cuda")  # tokens ahead of x
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    before = torch.where(back[..., None] >= 0, ring[rows, back % width].float(), 0.0)
    y = _plain_conv(x, s["weight"].float(), s["bias"].float(), before, inside).to(s["dtype"])
    # entry e of the ring holds the last token whose position is e modulo width
    last = pos[:, None] + inside.sum(1)[:, None] - 1
    t = last - (last - torch.arange(width, device="cuda")) % width - pos[:, None]
    new = torch.where(t[..., None] >= 0, s["x"][rows, torch.clamp(t, min=0)], ring)
    ring.copy_(new)
    return {"y": y, "ring": ring}


def _plain_conv_train(s):
    inside = _inside(s)
    x, w, b = (s[k].float().requires_grad_() for k in ("x", "weight", "bias"))
    before = x.new_zeros(x.shape[0], w.shape[1] - 1, x.shape[2])
    y = _plain_conv(x, w, b, before, inside)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].float())
    return {"y": y.detach().to(s["dtype"]), "dx": dx.to(s["dtype"]), "dweight": dw, "dbias": db}


def _decays(a):
    """exp of the sums of a over j < k <= i, [.., i, j]; zero where i < j."""
    n = a.shape[-1]
    low = torch.ones(n, n, dtype=torch.bool, device=a.device).tril()
    sums = torch.cumsum(torch.where(low.tril(-1), a[..., :, None], 0.0), dim=-2)
    return torch.exp(torch.where(low, sums, -math.inf))


def _plain_scan(x, dt, a, bm, cm, d, dt_bias, inside, state):
    """The scan in chunks of products: y and the last state."""
    batch, length, heads, _ = x.shape
    q = _CHUNK
    pad = -length % q
    delta = torch.where(inside[..., None], _softplus(dt + dt_bias), 0.0)
    keep = inside[..., None, None]
    x, bm, cm = (F.pad(torch.where(keep, v, 0.0), (0, 0, 0, 0, 0, pad)) for v in (x, bm, cm))
    delta = F.pad(delta, (0, 0, 0, pad))
    nc = (length + pad) // q
    x, bm, cm = (v.unflatten(1, (nc, q)).transpose(2, 3) for v in (x, bm, cm))  # [B, c, H, q, .]
    bm, cm = (v.repeat_interleave(heads // v.shape[2], dim=2) for v in (bm, cm))
    delta = delta.unflatten(1, (nc, q)).transpose(2, 3)                          # [B, c, H, q]
    s = torch.cumsum(delta * a[:, None], dim=-1)
    decay = _decays(delta * a[:, None])
    xd = x * delta[..., None]
    y = (cm @ bm.transpose(-1, -2) * decay) @ xd
    add = (xd * decay[..., -1, :, None]).transpose(-1, -2) @ bm                  # [B, c, H, P, N]
    # states at the chunks' starts and at the end: decays over whole chunks
    whole = _decays(F.pad(s[..., -1], (0, 0, 1, 0)).transpose(1, 2))              # [B, H, c + 1, ..]
    parts = torch.cat([state[:, None], add], dim=1).transpose(1, 2)               # [B, H, c + 1, ..]
    states = (whole @ parts.flatten(3)).unflatten(3, state.shape[2:])
    y = y + torch.exp(s)[..., None] * (cm @ states[:, :, :-1].transpose(1, 2).transpose(-1, -2))
    y = (y + d[:, None, None] * x).transpose(2, 3).flatten(1, 2)[:, :length]
    return torch.where(inside[..., None, None], y, 0.0), states[:, :, -1]


def _plain_scan_prompt(s):
    x, bm, cm = _split(s["xbc"].float(), s["case"])
    start = s["state"] if s["positions"] is not None else torch.zeros_like(s["state"])
    y, last = _plain_scan(x, s["dt"].float(), s["a"], bm, cm, s["d"], s["dt_bias"], _inside(s),
                          start)
    s["state"].copy_(last)
    return {"y": y.to(s["dtype"]), "state": s["state"]}


def _plain_scan_train(s):
    case = s["case"]
    x, bm, cm = (v.clone().requires_grad_() for v in _split(s["xbc"].float(), case))
    dt, a, d, dt_bias = (s[k].float().clone().requires_grad_() for k in ("dt", "a", "d", "dt_bias"))
    zero = x.new_zeros(case["batch"], case["heads"], case["head_dim"], case["state_dim"])
    y, _ = _plain_scan(x, dt, a, bm, cm, d, dt_bias, _inside(s), zero)
    g = torch.autograd.grad(y, (x, bm, cm, dt, a, d, dt_bias), s["dy"].float())
    t = s["dtype"]
    return {"y": y.detach().to(t), "dx": g[0].to(t), "db": g[1].to(t), "dc": g[2].to(t),
            "ddt": g[3].to(t), "da": g[4], "dd": g[5], "ddt_bias": g[6]}


def _plain_step(s):
    case, width = s["case"], s["case"]["width"]
    slots, pos = s["slots"].long(), s["positions"].long()
    back = pos[:, None] - torch.arange(width - 1, 0, -1, device="cuda")
    before = torch.where(back[..., None] >= 0, s["ring"][slots[:, None], back % width].float(), 0.0)
    seen = torch.cat([before, s["xbc"].float()[:, None]], dim=1)                 # [B, W, C]
    act = _silu((seen * s["weight"].float().t()).sum(1) + s["bias"].float())
    x, bm, cm = _split(act, case)
    bm, cm = (v.repeat_interleave(case["heads"] // case["groups"], dim=1) for v in (bm, cm))
    delta = _softplus(s["dt"].float() + s["dt_bias"])
    state = torch.where(pos[:, None, None, None] > 0, s["state"][slots], 0.0)
    state = torch.exp(delta * s["a"])[..., None, None] * state \
        + (delta[..., None] * x)[..., None] * bm[:, :, None, :]
    y = (state * cm[:, :, None, :]).sum(-1) + s["d"][:, None] * x
    s["state"][slots] = state
    s["ring"][slots, pos % width] = s["xbc"]
    return {"y": y.to(s["dtype"]), "state": s["state"], "ring": s["ring"]}


# ------------------------------------------------------- the framework's calls

_library = None


def _lib():
    global _library
    if _library is None:
        from ns_fps_amd import capi
        _library = capi.Lib()
    return _library


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _dt(s):
    from ns_fps_amd import capi
    return capi.BF16 if s["dtype"] == torch.bfloat16 else capi.F32


def _ptr(v):
    return None if v is None else v.data_ptr()


def _rows(v, offset=0):
    """(pointer, batch stride, row stride) of [B, L, ...], from ``offset`` on."""
    return (v.data_ptr() + offset * v.element_size(), v.stride(0), v.stride(1))


def _workspace(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


def _own_lookup(s):
    from ns_fps_amd import capi
    case = s["case"]
    out = torch.empty(case["tokens"], case["width"], dtype=s["dtype"], device="cuda")
    if "args" not in s:
        s["args"] = capi.EmbedArgs(tokens=case["tokens"], rows=case["rows"], width=case["width"],
                                   dtype=_dt(s), scale=s["scale"], table_stride=case["width"],
                                   out_stride=case["width"], d_table=s["table"].data_ptr(),
                                   d_tokens=s["tokens"].data_ptr())
    s["args"].d_out = out.data_ptr()
    _lib().embed_device(s["args"], _stream())
    return out


def _own_lookup_grad(s):
    from ns_fps_amd import capi
    case = s["case"]
    grad = torch.empty(case["rows"], case["width"], dtype=s["dtype"], device="cuda")
    if "args" not in s:
        s["args"] = args = capi.EmbedArgs(
            tokens=case["tokens"], rows=case["rows"], width=case["width"], dtype=_dt(s),
            grad_dtype=_dt(s), scale=s["scale"], table_stride=case["width"],
            out_stride=case["width"], d_tokens=s["tokens"].data_ptr(), d_out=s["dout"].data_ptr())
        s["workspace"] = _workspace(_lib().embed_grad_workspace_bytes(args))
        args.workspace, args.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    s["args"].d_table = grad.data_ptr()
    _lib().embed_grad_device(s["args"], _stream())
    return grad


def _own_conv(s):
    from ns_fps_amd import capi
    case = s["case"]
    y = torch.empty_like(s["x"])
    if "args" not in s:
        s["args"] = args = capi.ConvArgs(
            batch=case["batch"], length=case["length"], channels=case["channels"],
            width=case["width"], dtype=_dt(s), x=_rows(s["x"]), d_weight=s["weight"].data_ptr(),
            d_bias=s["bias"].data_ptr(), d_lengths=_ptr(s["lengths"]),
            d_positions=_ptr(s["positions"]))
        if case["train"]:
            s["workspace"] = _workspace(_lib().conv_grad_workspace_bytes(args))
            args.workspace = s["workspace"].data_ptr()
            args.workspace_bytes = s["workspace"].numel()
        else:
            args.d_cache = s["ring"].data_ptr()
    args = s["args"]
    args.y = _rows(y)
    _lib().conv_device(args, _stream())
    if not case["train"]:
        return {"y": y, "ring": s["ring"]}
    dx = torch.empty_like(y)
    dw = torch.empty(case["channels"], case["width"], device="cuda")
    db = torch.empty(case["channels"], device="cuda")
    grads = capi.ConvGrads(dy=_rows(s["dy"]), dx=_rows(dx), d_dweight=dw.data_ptr(),
                           d_dbias=db.data_ptr())
    _lib().conv_grad_device(args, grads, _stream())
    return {"y": y, "dx": dx, "dweight": dw, "dbias": db}


def _own_scan(s):
    from ns_fps_amd import capi
    case, xbc = s["case"], s["xbc"]
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    y = torch.empty(*xbc.shape[:2], h, p, dtype=s["dtype"], device="cuda")
    if "args" not in s:
        s["args"] = args = capi.ScanArgs(
            batch=case["batch"], length=case["length"], heads=h, groups=g, head_dim=p,
            state_dim=n, dtype=_dt(s), x=_rows(xbc), b=_rows(xbc, h * p),
            c=_rows(xbc, h * p + g * n), dt=_rows(s["dt"]), d_a=s["a"].data_ptr(),
            d_d=s["d"].data_ptr(), d_dt_bias=s["dt_bias"].data_ptr(),
            d_lengths=_ptr(s["lengths"]), d_positions=_ptr(s["positions"]))
        need = _lib().scan_workspace_bytes(args)
        if case["train"]:
            need = max(need, _lib().scan_grad_workspace_bytes(args))
        else:
            args.d_state = s["state"].data_ptr()
        s["workspace"] = _workspace(need)
        args.workspace, args.workspace_bytes = s["workspace"].data_ptr(), s["workspace"].numel()
    args = s["args"]
    args.y = _rows(y)
    _lib().scan_device(args, _stream())
    if not case["train"]:
        return {"y": y, "state": s["state"]}
    dxbc, ddt = torch.empty_like(xbc), torch.empty_like(s["dt"])
    da, dd, dbias = (torch.empty(h, device="cuda") for _ in range(3))
    grads = capi.ScanGrads(dy=_rows(s["dy"]), dx=_rows(dxbc), db=_rows(dxbc, h * p),
                           dc=_rows(dxbc, h * p + g * n), ddt=_rows(ddt), d_da=da.data_ptr(),
                           d_dd=dd.data_ptr(), d_ddt_bias=dbias.data_ptr())
    _lib().scan_grad_device(args, grads, _stream())
    dx, db, dc = _split(dxbc, case)
    return {"y": y, "dx": dx, "db": db, "dc": dc, "ddt": ddt, "da": da, "dd": dd,
            "ddt_bias": dbias}


def _own_step(s):
    from ns_fps_amd import capi
    case = s["case"]
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    y = torch.empty(case["batch"], h, p, dtype=s["dtype"], device="cuda")
    if "args" not in s:
        s["args"] = capi.StepArgs(
            batch=case["batch"], heads=h, groups=g, head_dim=p, state_dim=n, width=case["width"],
            dtype=_dt(s), xbc_stride=s["xbc"].stride(0), dt_stride=s["dt"].stride(0),
            y_stride=h * p, d_xbc=s["xbc"].data_ptr(), d_weight=s["weight"].data_ptr(),
            d_bias=s["bias"].data_ptr(), d_dt=s["dt"].data_ptr(), d_a=s["a"].data_ptr(),
            d_d=s["d"].data_ptr(), d_dt_bias=s["dt_bias"].data_ptr(),
            d_positions=s["positions"].data_ptr(), d_slots=s["slots"].data_ptr(),
            d_cache=s["ring"].data_ptr(), d_state=s["state"].data_ptr())
    s["args"].d_y = y.data_ptr()
    _lib().scan_step_device(s["args"], _stream())
    return {"y": y, "state": s["state"], "ring": s["ring"]}


_PLAIN = {"lookup": _plain_lookup, "lookup_grad": _plain_lookup_grad, "step": _plain_step}
_OWN = {"lookup": _own_lookup, "lookup_grad": _own_lookup_grad, "step": _own_step,
        "conv": _own_conv, "scan": _own_scan}


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    if op == "conv":
        return (_plain_conv_train if state["case"]["train"] else _plain_conv_prompt)(state)
    if op == "scan":
        return (_plain_scan_train if state["case"]["train"] else _plain_scan_prompt)(state)
    return _PLAIN[op](state)


# -------------------------------------------------------------------- the work

def work(case):
    """Bytes and operations that one pass cannot do without."""
    op, z = case["op"], _SIZE[case["dtype"]]
    if op in ("lookup", "lookup_grad"):
        used = min(case["tokens"], case["rows"]) if op == "lookup" else case["rows"]
        cells = (case["tokens"] + used) * case["width"]
        return {"bytes": cells * z + 4 * case["tokens"], "flops": case["tokens"] * case["width"]}
    if op == "step":
        h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
        channels = h * p + 2 * g * n
        row = 8 * h * p * n + z * (channels * (case["width"] + 1) + h * p + h) + 8
        return {"bytes": case["batch"] * row + z * channels * (case["width"] + 1),
                "flops": case["batch"] * (5 * h * p * n + 2 * channels * case["width"])}
    tokens = case["batch"] * case["length"] * (0.75 if case["ragged"] else 1.0)
    if op == "conv":
        cells = tokens * case["channels"]
        if case["train"]:  # x, dy; y, dx
            return {"bytes": 4 * cells * z, "flops": cells * (6 * case["width"] + 12)}
        return {"bytes": 2 * cells * z, "flops": cells * (2 * case["width"] + 4)}
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    row = z * (2 * h * p + 2 * g * n + h)  # x, B, C, dt; y
    state = case["batch"] * h * p * n * 4
    flops = tokens * h * p * n * 5
    if case["train"]:  # and dy; dx, dB, dC, ddt
        row += z * (2 * h * p + 2 * g * n + h)
        return {"bytes": tokens * row, "flops": 4 * flops}
    return {"bytes": tokens * row + (2 if case["resume"] else 1) * state, "flops": flops}


# ------------------------------------------------------- from the definition

def _pad_exact(x, inside, before):
    return torch.cat([before, x * inside[..., None]], dim=1)


def _conv_exact(s, want_ring):
    """The convolution's sums tap by tap, and their derivatives written out."""
    case, w = s["case"], s["case"]["width"]
    length, inside = case["length"], _inside(s).double()
    x, weight, bias = s["x"].double(), s["weight"].double(), s["bias"].double()
    before = x.new_zeros(case["batch"], w - 1, case["channels"])
    ring = s["ring"].double() if want_ring else None
    if s["positions"] is not None:
        for b, pos in enumerate(s["positions"].tolist()):
            for k in range(1, w):
                if pos >= k:
                    before[b, w - 1 - k] = ring[b, (pos - k) % w]
    seen = _pad_exact(x, inside, before)
    pre = bias + sum(weight[:, k] * seen[:, k:k + length] for k in range(w))
    sig = torch.sigmoid(pre)
    y = pre * sig * inside[..., None]
    if want_ring:
        lens = inside.sum(1).long().tolist()
        pos = [0] * case["batch"] if s["positions"] is None else s["positions"].tolist()
        for b in range(case["batch"]):
            for t in range(max(0, lens[b] - w), lens[b]):
                ring[b, (pos[b] + t) % w] = x[b, t]
        return {"y": y, "ring": ring}
    g = s["dy"].double() * inside[..., None] * sig * (1 + pre * (1 - sig))
    dx = torch.zeros_like(x)
    dw = torch.empty_like(weight)
    for k in range(w):
        ahead = w - 1 - k  # x[t] meets tap k in the output `ahead` tokens later
        dx[:, :max(0, length - ahead)] += weight[:, k] * g[:, ahead:]
        dw[:, k] = (g * seen[:, k:k + length]).sum((0, 1))
    return {"y": y, "dx": dx * inside[..., None], "dweight": dw, "dbias": g.sum((0, 1))}


def _scan_terms(s):
    """Per token, in 64 bits: x, B and C per head, step and decay."""
    case = s["case"]
    each = case["heads"] // case["groups"]
    inside = _inside(s).double()
    x, bm, cm = (v * inside[..., None, None] for v in _split(s["xbc"].double(), case))
    head = torch.arange(case["heads"], device="cuda") // each
    raw = s["dt"].double() + s["dt_bias"].double()
    delta = F.softplus(raw, threshold=1000.0) * inside[..., None]
    return x, bm[:, :, head], cm[:, :, head], raw, delta, torch.exp(delta * s["a"].double()), inside


def _scan_exact(s):
    """The recurrence, token by token."""
    x, bm, cm, _, delta, decay, inside = _scan_terms(s)
    state = s["state"].double()
    state = state.clone() if s["positions"] is not None else torch.zeros_like(state)
    y = torch.empty_like(x)
    xd = delta[..., None] * x
    for t in range(x.shape[1]):
        state = decay[:, t, :, None, None] * state
        state += xd[:, t, :, :, None] * bm[:, t, :, None, :]
        torch.sum(state * cm[:, t, :, None, :], -1, out=y[:, t])
    y += s["d"].double()[:, None] * x
    return {"y": y * inside[..., None, None], "state": state}


def _scan_train_exact(s):
    """The recurrence and its adjoint, token by token; states are kept for
    every 64th token and found again between."""
    x, bm, cm, raw, delta, decay, inside = _scan_terms(s)
    case, length, d = s["case"], s["case"]["length"], s["d"].double()
    dy = s["dy"].double() * inside[..., None, None]

    def on(state, t):
        return decay[:, t, :, None, None] * state \
            + (delta[:, t, :, None] * x[:, t])[..., None] * bm[:, t, :, None, :]

    state = x.new_zeros(case["batch"], case["heads"], case["head_dim"], case["state_dim"])
    kept, y = [], torch.empty_like(x)
    for t in range(length):
        if t % 64 == 0:
            kept.append(state)
        state = on(state, t)
        y[:, t] = (state * cm[:, t, :, None, :]).sum(-1)
    y += d[:, None] * x
    dx, db, dc, ddelta = (torch.empty_like(v) for v in (x, bm, cm, delta))
    dlog = torch.empty_like(delta)  # of the exponent delta * A
    grad = torch.zeros_like(state)
    for first in range((length - 1) // 64 * 64, -1, -64):
        states = [kept.pop()]
        for t in range(first, min(first + 64, length)):
            states.append(on(states[-1], t))
        for t in range(min(first + 64, length) - 1, first - 1, -1):
            after = states.pop()
            grad += dy[:, t, :, :, None] * cm[:, t, :, None, :]
            dc[:, t] = (after * dy[:, t, :, :, None]).sum(2)
            gb = (grad * bm[:, t, :, None, :]).sum(-1)
            dx[:, t] = delta[:, t, :, None] * gb
            db[:, t] = delta[:, t, :, None] * (grad * x[:, t, :, :, None]).sum(2)
            grad *= decay[:, t, :, None, None]
            dlog[:, t] = (grad * states[-1]).sum((2, 3))
            ddelta[:, t] = (gb * x[:, t]).sum(-1)
    ddt = (ddelta + s["a"].double() * dlog) * torch.sigmoid(raw) * inside[..., None]
    shape = (case["batch"], length, case["groups"], -1, case["state_dim"])
    return {"y": y * inside[..., None, None],
            "dx": (dx + d[:, None] * dy) * inside[..., None, None],
            "db": db.reshape(shape).sum(3) * inside[..., None, None],
            "dc": dc.reshape(shape).sum(3) * inside[..., None, None],
            "ddt": ddt, "da": (dlog * delta).sum((0, 1)), "dd": (dy * x).sum((0, 1, 3)),
            "ddt_bias": ddt.sum((0, 1))}


def _step_exact(s):
    case, w = s["case"], s["case"]["width"]
    h, p, n, g = case["heads"], case["head_dim"], case["state_dim"], case["groups"]
    xbc, weight = s["xbc"].double(), s["weight"].double()
    ring, state = s["ring"].double(), s["state"].double()
    slot, pos = s["slots"].long(), s["positions"].long()
    pre = s["bias"].double() + weight[:, w - 1] * xbc
    for k in range(1, w):
        old = ring[slot, (pos - k) % w] * (pos >= k).double()[:, None]
        pre = pre + weight[:, w - 1 - k] * old
    act = pre * torch.sigmoid(pre)
    head = torch.arange(h, device="cuda") // (h // g)
    x = act[:, :h * p].reshape(-1, h, p)
    bm = act[:, h * p:h * p + g * n].reshape(-1, g, n)[:, head]
    cm = act[:, h * p + g * n:].reshape(-1, g, n)[:, head]
    delta = F.softplus(s["dt"].double() + s["dt_bias"].double(), threshold=1000.0)
    old = state[slot] * (pos > 0).double()[:, None, None, None]
    new = torch.exp(delta * s["a"].double())[..., None, None] * old \
        + (delta[..., None] * x)[..., None] * bm[:, :, None, :]
    state[slot] = new
    ring[slot, pos % w] = xbc
    return {"y": (new * cm[:, :, None, :]).sum(-1) + s["d"].double()[:, None] * x,
            "state": state, "ring": ring}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("lookup", "lookup_grad"):
        rows = case["rows"]
        tok = s["tokens"].long()
        hit = ((tok >= 0) & (tok < rows)).double()[:, None]
        if op == "lookup":
            return s["scale"] * s["table"].double()[tok.clamp(0, rows - 1)] * hit
        order = torch.argsort(tok, stable=True)
        sums = F.pad(torch.cumsum((s["dout"].double() * hit)[order], 0), (0, 0, 1, 0))
        ends = torch.searchsorted(tok[order], torch.arange(-1, rows, device="cuda"), right=True)
        return s["scale"] * (sums[ends[1:]] - sums[ends[:-1]])
    if op == "conv":
        return _conv_exact(s, not case["train"])
    if op == "scan":
        return _scan_train_exact(s) if case["train"] else _scan_exact(s)
    return _step_exact(s)
