"""What a sequence model over sampled points needs beside lookup, convolution
and scan, as a program uses it.

Samples in the order of their grid cells are tokens, a sample's cell being its
token.  Between convolution and scan the scan's keys (b) and queries (c) are
normed head by head and rotated by their position; dropout thins what a layer
adds to the residual; and the loss is a cross entropy over all cells.
Operators (``op``):

* ``norm``     norms of queries and keys and their rotation; with ``train`` the gradient too
* ``dropout``  dropout from a counter-based generator, onto a residual; with ``train`` the gradient too
* ``loss``     softmax cross entropy over the vocabulary; with ``train`` the gradient too

``own`` false computes them from elementary torch operations in 32 bits
(angles in 64, the generator in whole numbers); ``own`` true calls ns_fps_amd.
Types: ``bf16`` or ``f32``; losses and the norm weights' gradients are float32
with both, the table's gradient has the table's type.
"""

import math

import numpy as np
import torch
import torch.nn.functional as F

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
_EPS = 1e-6
_DROP = 0.1


# ------------------------------------------------------------------ the cases

def _norm(batch, length, q_heads, k_heads, head_dim, rotary_dim, dtype, train=False, ragged=False,
          resume=False, neighbours=False):
    return {"op": "norm", "batch": batch, "length": length, "q_heads": q_heads, "k_heads": k_heads,
            "head_dim": head_dim, "rotary_dim": rotary_dim, "dtype": dtype, "train": train,
            "ragged": ragged, "resume": resume, "neighbours": neighbours}


def _dropout(batch, length, channels, dtype, residual=True, train=False, ragged=False):
    return {"op": "dropout", "batch": batch, "length": length, "channels": channels,
            "dtype": dtype, "residual": residual, "train": train, "ragged": ragged}


def _loss(tokens, rows, width, dtype, train=False):
    return {"op": "loss", "tokens": tokens, "rows": rows, "width": width, "dtype": dtype,
            "train": train}


def listed():
    return [
        # one quickstart cloud as a prompt, one group of 64: latency counts
        dict(_norm(1, 1000, 1, 1, 64, 64, "bf16"), name="norm_quickstart"),
        # one token of a full serving batch, at each request's own position
        dict(_norm(512, 1, 2, 2, 128, 128, "bf16", resume=True), name="norm_step_512"),
        # a training batch: 64 clouds of up to 4,096 samples, eight groups
        dict(_norm(64, 4096, 8, 8, 64, 64, "bf16", train=True, ragged=True),
             name="norm_train_batched"),
        # a small model in full precision: odd heads, one value unrotated, pairs of neighbours
        dict(_norm(3, 1001, 3, 3, 33, 32, "f32", train=True, neighbours=True),
             name="norm_train_odd_f32"),
        # one quickstart cloud's rows onto the residual
        dict(_dropout(1, 1000, 384, "bf16"), name="dropout_quickstart"),
        # a training batch of ragged clouds
        dict(_dropout(64, 4096, 640, "bf16", train=True, ragged=True),
             name="dropout_train_batched"),
        # one LiDAR scan's rows, odd channels, full precision, no residual
        dict(_dropout(1, 16384, 323, "f32", residual=False, train=True), name="dropout_lidar_f32"),
        # the quickstart samples scored over their 16^3 grid
        dict(_loss(1000, 4096, 384, "bf16"), name="loss_quickstart"),
        # a few tokens of requests scored over the 64^3 grid: the table is all the traffic
        dict(_loss(7, 262144, 256, "bf16"), name="loss_few"),
        # a training step of the smallest model, full precision
        dict(_loss(1000, 4096, 64, "f32", train=True), name="loss_train_small_f32"),
        # one LiDAR scan's samples over the 32 x 32 x 8 grid, an odd width, full precision
        dict(_loss(16384, 8192, 383, "f32", train=True), name="loss_train_lidar_f32"),
        # a training batch over the 64^3 grid: the largest vocabulary
        dict(_loss(16384, 262144, 256, "bf16", train=True), name="loss_train_clustered"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "dropout", "loss", "loss", "loss"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    train = rng.random() < 0.6
    if op == "loss":
        width = _log_int(rng, 16, 1024)
        room = 16384 * 262144 * 256 // (1 if dtype == "bf16" else 8) // width
        tokens = _log_int(rng, 1, 16384)
        return _loss(tokens, _log_int(rng, 64, max(64, min(262144, room // tokens))), width, dtype,
                     train)
    ragged = rng.random() < 0.5
    batch = _log_int(rng, 1, 512)
    room = (1 if dtype == "bf16" else 2) * batch  # full precision costs more a value
    if op == "dropout":
        length = _log_int(rng, 1, min(65536, 262144 // room))
        channels = _log_int(rng, 16, min(2048, 167772160 // room // length))
        return _dropout(batch, length, channels, dtype, rng.random() < 0.5, train, ragged)
    head_dim = rng.choice([64, 128, rng.randint(16, 128)])
    rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, 0]) // 2 * 2
    heads = rng.choice([1, 1, 2, 4, 8])
    most = 262144 * 8 * 64 // (room * heads * head_dim)
    return _norm(batch, _log_int(rng, 1, max(1, min(65536, most))), heads,
                 heads if rng.random() < 0.5 else rng.randint(1, heads), head_dim, rotary_dim,
                 dtype, train, ragged, rng.random() < 0.5, rng.random() < 0.3)


# ------------------------------------------------------------------ the inputs

def _lengths(gen, case):
    if not case["ragged"]:
        return None
    f = 0.5 + 0.5 * torch.rand(case["batch"], generator=gen, device="cuda")
    return (f * case["length"]).ceil().to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    s = {"case": case, "dtype": dtype}
    if op == "loss":
        n, rows, width = case["tokens"], case["rows"], case["width"]
        s["x"] = normal(n, width)
        s["table"] = normal(rows, width, scale=0.02)
        s["scale"] = 100.0 / math.sqrt(width)  # logits of a deviation of 2
        u = torch.rand(n, generator=gen, device="cuda")
        cell = torch.clamp((u * u * rows).to(torch.int64), max=rows - 1)  # crowded cells
        pad = torch.rand(n, generator=gen, device="cuda") < 1 / 64        # ended early: -1
        s["targets"] = torch.where(pad, -1, cell).to(torch.int32)
        if case["train"]:  # the mean over the tokens that count
            s["dloss"] = torch.where(pad, 0.0, 1.0 / n).to(torch.float32)
        return s
    b, length = case["batch"], case["length"]
    s["lengths"] = _lengths(gen, case)
    if op == "dropout":
        s["x"] = normal(b, length, case["channels"])
        if case["residual"]:
            s["residual"] = normal(b, length, case["channels"], scale=2.0)
        if case["train"]:
            s["dy"] = normal(b, length, case["channels"], scale=0.1)
        # the generator's key and the call's number
        s["seed"] = torch.tensor([seed * 0x9E3779B1 + 12345, 7 + seed % 100], dtype=torch.int64,
                                 device="cuda")
        return s
    hq, hk, d, r = case["q_heads"], case["k_heads"], case["head_dim"], case["rotary_dim"]
    inner = 64 * hq  # the rows hold the scan's x as well, ahead of keys and queries
    s["rows"] = normal(b, length, inner + (hk + hq) * d)
    s["k"], s["q"] = s["rows"][..., inner:inner + hk * d], s["rows"][..., inner + hk * d:]
    s["q_weight"] = (1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
    s["k_weight"] = (1.0 + 0.1 * torch.randn(d, generator=gen, device="cuda")).to(dtype)
    pair = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    s["freq"] = (10000.0 ** (-2 * pair / max(r, 1))).float()
    s["positions"] = torch.randint(1, 500000, (b,), generator=gen, device="cuda",
                                   dtype=torch.int32) if case["resume"] else None
    if case["train"]:
        s["dq_out"] = normal(b, length, hq * d, scale=0.1)
        s["dk_out"] = normal(b, length, hk * d, scale=0.1)
    return s


# ------------------------------------------------------------- the plain forms

def _inside(s):
    """[B, L]: which tokens are inside their row's length."""
    case = s["case"]
    t = torch.arange(case["length"], device="cuda")
    if s["lengths"] is None:
        return torch.ones(case["batch"], case["length"], dtype=torch.bool, device="cuda")
    return t[None] < s["lengths"][:, None]


def _turn(s):
    """Cosines and sines of every token, [B, L, 1, R / 2]: angles in 64 bits."""
    pos = torch.arange(s["case"]["length"], device="cuda", dtype=torch.float64)[None]
    if s["positions"] is not None:
        pos = pos + s["positions"][:, None]
    angle = (pos[..., None] * s["freq"].double())[:, :, None]
    return torch.cos(angle).float(), torch.sin(angle).float()


def _rotate(v, cos, sin, neighbours):
    """Pairs (first, second) turned by their angle; what is behind them stays."""
    r = 2 * cos.shape[-1]
    a, b = (v[..., 0:r:2], v[..., 1:r:2]) if neighbours else (v[..., :r // 2], v[..., r // 2:r])
    a, b = a * cos - b * sin, a * sin + b * cos
    both = torch.stack([a, b], -1).flatten(-2) if neighbours else torch.cat([a, b], -1)
    return torch.cat([both, v[..., r:]], -1)


def _plain_norm(s):
    case, keep = s["case"], _inside(s)[..., None, None]
    cos, sin = _turn(s)
    out = {}

    def one(name, heads):
        x = s[name].float().unflatten(-1, (heads, case["head_dim"]))
        x = torch.where(keep, x, 0.0)
        w = s[name + "_weight"].float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        y = _rotate(x * r * w, cos, sin, case["neighbours"])
        out[name] = torch.where(keep, y, 0.0).flatten(2).to(s["dtype"])
        if not case["train"]:
            return
        g = s[f"d{name}_out"].float().unflatten(-1, (heads, case["head_dim"]))
        g = _rotate(torch.where(keep, g, 0.0), cos, -sin, case["neighbours"])
        n = x * r
        out[f"d{name}_weight"] = (g * n).sum((0, 1, 2))
        g = g * w
        out[f"d{name}"] = (r * (g - n * (g * n).mean(-1, keepdim=True))).flatten(2).to(s["dtype"])

    one("q", case["q_heads"])
    one("k", case["k_heads"])
    return out


_LOW = 0xFFFFFFFF


def _mul(a, m):
    """High and low words of the product of 32-bit a (in 64) and constant m."""
    low, high = (a & 0xFFFF) * m, (a >> 16) * m
    return (high + (low >> 16)) >> 16, (low + (high << 16)) & _LOW


def _plain_keep(s):
    """Which values stay: 16 random bits each, eight values a block of the
    generator (Philox 4x32-10: counter = block of the row, row, call's number;
    key = seed), against the drop probability in 65536ths."""
    case = s["case"]
    blocks = -(-case["channels"] // 8)
    row = torch.arange(case["batch"] * case["length"], device="cuda")[:, None]
    c0 = torch.arange(blocks, device="cuda")[None].expand(row.shape[0], blocks)
    c1 = row.expand_as(c0)
    key, call = s["seed"][0], s["seed"][1]
    c2, c3 = (call & _LOW).expand_as(c0), ((call >> 32) & _LOW).expand_as(c0)
    k0, k1 = key & _LOW, (key >> 32) & _LOW
    for _ in range(10):
        (h0, l0), (h1, l1) = _mul(c0, 0xD2511F53), _mul(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).flatten(1)[:, :case["channels"]]
    keep = bits >= round(_DROP * 65536)
    return keep.reshape(case["batch"], case["length"], case["channels"])


def _plain_dropout(s):
    case, inside = s["case"], _inside(s)[..., None]
    factor = 65536.0 / (65536 - round(_DROP * 65536))
    keep = _plain_keep(s) & inside
    y = torch.where(keep, s["x"].float() * factor, 0.0)
    if case["residual"]:
        y = y + torch.where(inside, s["residual"].float(), 0.0)
    out = {"y": y.to(s["dtype"])}
    if case["train"]:
        out["dx"] = torch.where(keep, s["dy"].float() * factor, 0.0).to(s["dtype"])
    return out


def _plain_loss(s):
    case = s["case"]
    x, table, target = s["x"].float(), s["table"].float(), s["targets"].long()
    counts = target >= 0
    z = (x @ table.t()) * s["scale"]
    top = z.amax(1, keepdim=True)
    lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))
    at = torch.where(counts, target, 0)[:, None]
    out = {"loss": torch.where(counts, (lse - z.gather(1, at))[:, 0], 0.0), "lse": lse[:, 0]}
    if case["train"]:
        weight = torch.where(counts, s["dloss"] * s["scale"], 0.0)[:, None]
        dz = torch.exp(z.sub_(lse)).mul_(weight)
        dz.scatter_add_(1, at, -weight)
        out["dx"] = (dz @ table).to(s["dtype"])
        out["dtable"] = (dz.t() @ x).to(s["dtype"])
    return out


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


def _rows(v):
    """(pointer, batch stride, row stride) of [B, L, ...]."""
    return (v.data_ptr(), v.stride(0), v.stride(1))


def _with_workspace(s, args, *sizes):
    need = max(size(args) for size in sizes)
    s["workspace"] = torch.empty(need, dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = s["workspace"].data_ptr(), need


def _own_norm(s):
    from ns_fps_amd import capi
    case, (b, length) = s["case"], s["rows"].shape[:2]
    hq, hk, d = case["q_heads"], case["k_heads"], case["head_dim"]
    q = torch.empty(b, length, hq * d, dtype=s["dtype"], device="cuda")
    k = torch.empty(b, length, hk * d, dtype=s["dtype"], device="cuda")
    if "args" not in s:
        s["args"] = args = capi.NormArgs(
            batch=b, length=length, q_heads=hq, k_heads=hk, head_dim=d,
            rotary_dim=case["rotary_dim"], neighbours=int(case["neighbours"]), dtype=_dt(s),
            eps=_EPS, q=_rows(s["q"]), k=_rows(s["k"]), d_q_weight=s["q_weight"].data_ptr(),
            d_k_weight=s["k_weight"].data_ptr(),
            d_freq=s["freq"].data_ptr() if case["rotary_dim"] else None,
            d_lengths=_ptr(s["lengths"]), d_positions=_ptr(s["positions"]))
        if case["train"]:
            _with_workspace(s, args, _lib().norm_grad_workspace_bytes)
    args = s["args"]
    args.q_out, args.k_out = _rows(q), _rows(k)
    _lib().norm_device(args, _stream())
    out = {"q": q, "k": k}
    if case["train"]:
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        dqw, dkw = (torch.empty(d, device="cuda") for _ in range(2))
        grads = capi.NormGrads(dq_out=_rows(s["dq_out"]), dk_out=_rows(s["dk_out"]), dq=_rows(dq),
                               dk=_rows(dk), d_dq_weight=dqw.data_ptr(),
                               d_dk_weight=dkw.data_ptr())
        _lib().norm_grad_device(args, grads, _stream())
        out.update(dq=dq, dk=dk, dq_weight=dqw, dk_weight=dkw)
    return out


def _own_dropout(s):
    from ns_fps_amd import capi
    case = s["case"]

    def args(x, residual=None):
        a = capi.DropoutArgs(batch=case["batch"], length=case["length"],
                             channels=case["channels"], dtype=_dt(s), p=_DROP, x=_rows(x),
                             d_seed=s["seed"].data_ptr(), d_lengths=_ptr(s["lengths"]))
        if residual is not None:
            a.residual = _rows(residual)
        return a

    if "args" not in s:
        s["args"] = args(s["x"], s.get("residual"))
        s["back"] = args(s["dy"]) if case["train"] else None
    y = torch.empty_like(s["x"])
    s["args"].y = _rows(y)
    _lib().dropout_device(s["args"], _stream())
    out = {"y": y}
    if case["train"]:
        dx = torch.empty_like(y)
        s["back"].y = _rows(dx)
        _lib().dropout_device(s["back"], _stream())
        out["dx"] = dx
    return out


def _own_loss(s):
    from ns_fps_amd import capi
    case = s["case"]
    n, width = case["tokens"], case["width"]
    loss, lse = (torch.empty(n, device="cuda") for _ in range(2))
    if "args" not in s:
        s["args"] = args = capi.LossArgs(
            tokens=n, rows=case["rows"], width=width, dtype=_dt(s), scale=s["scale"],
            x_stride=width, table_stride=width, d_x=s["x"].data_ptr(),
            d_table=s["table"].data_ptr(), d_targets=s["targets"].data_ptr())
        if case["train"]:
            s["grads"] = capi.LossGrads(d_dloss=s["dloss"].data_ptr(), dx_stride=width,
                                        dtable_stride=width, grad_dtype=_dt(s))
            _with_workspace(s, args, _lib().loss_workspace_bytes,
                            lambda a: _lib().loss_grad_workspace_bytes(a, s["grads"]))
        else:
            _with_workspace(s, args, _lib().loss_workspace_bytes)
    args = s["args"]
    args.d_loss, args.d_lse = loss.data_ptr(), lse.data_ptr()
    _lib().loss_device(args, _stream())
    out = {"loss": loss, "lse": lse}
    if case["train"]:
        dx, dtable = torch.empty_like(s["x"]), torch.empty_like(s["table"])
        s["grads"].d_dx, s["grads"].d_dtable = dx.data_ptr(), dtable.data_ptr()
        _lib().loss_grad_device(args, s["grads"], _stream())
        out.update(dx=dx, dtable=dtable)
    return out


_PLAIN = {"norm": _plain_norm, "dropout": _plain_dropout, "loss": _plain_loss}
_OWN = {"norm": _own_norm, "dropout": _own_dropout, "loss": _own_loss}


def run(state):
    op = state["case"]["op"]
    return _OWN[op](state) if own else _PLAIN[op](state)


# -------------------------------------------------------------------- the work

def work(case):
    """Bytes and operations that one pass cannot do without."""
    op, z, train = case["op"], _SIZE[case["dtype"]], case["train"]
    if op == "loss":
        # the logits are not kept, so a gradient finds them again
        cells, pairs = (case["tokens"] + case["rows"]) * case["width"], case["tokens"] * case["rows"]
        return {"bytes": (2 if train else 1) * cells * z + 12 * case["tokens"],
                "flops": (8 if train else 2) * pairs * case["width"]}
    tokens = case["batch"] * case["length"] * (0.75 if case["ragged"] else 1.0)
    if op == "dropout":  # x, residual; y; dy; dx
        cells = tokens * case["channels"]
        return {"bytes": cells * z * (2 + case["residual"] + 2 * train),
                "flops": cells * (2 + train)}
    cells = tokens * (case["q_heads"] + case["k_heads"]) * case["head_dim"]
    return {"bytes": cells * z * (5 if train else 2), "flops": cells * (24 if train else 8)}


# ------------------------------------------------------- from the definition

def _norm_exact(s):
    """The rotation as a complex product, the norm's gradient by its Jacobian's
    two terms."""
    case, d, r = s["case"], s["case"]["head_dim"], s["case"]["rotary_dim"]
    keep = _inside(s).double()[..., None, None]
    pos = torch.arange(case["length"], device="cuda", dtype=torch.float64).expand(case["batch"], -1)
    if s["positions"] is not None:
        pos = pos + s["positions"].double()[:, None]
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       (pos[..., None] * s["freq"].double())[:, :, None])
    first = torch.arange(0, r, 2, device="cuda") if case["neighbours"] \
        else torch.arange(r // 2, device="cuda")
    second = first + (1 if case["neighbours"] else r // 2)

    def turned(v, by):
        w = torch.complex(v[..., first], v[..., second]) * by
        v = v.clone()
        v[..., first], v[..., second] = w.real, w.imag
        return v

    out = {}
    for name, heads in (("q", case["q_heads"]), ("k", case["k_heads"])):
        x = s[name].double().unflatten(-1, (heads, d)) * keep
        w = s[name + "_weight"].double()
        size = torch.sqrt((x * x).sum(-1, keepdim=True) / d + _EPS)
        out[name] = (turned(x / size * w, turn) * keep).flatten(2)
        if case["train"]:
            g = turned(s[f"d{name}_out"].double().unflatten(-1, (heads, d)) * keep, turn.conj())
            out[f"d{name}_weight"] = (g * x / size).sum((0, 1, 2))
            g = g * w
            along = (g * x).sum(-1, keepdim=True) / d
            out[f"d{name}"] = (g / size - x * along / size ** 3).flatten(2)
    return out


def _dropout_exact(s):
    """The generator in numpy, on 64-bit words."""
    case = s["case"]
    blocks = -(-case["channels"] // 8)
    tokens = case["batch"] * case["length"]
    key, call = (int(v) & (2 ** 64 - 1) for v in s["seed"].tolist())
    word, low = np.uint64(32), np.uint64(2 ** 32 - 1)
    c = [np.tile(np.arange(blocks, dtype=np.uint64), tokens),
         np.repeat(np.arange(tokens, dtype=np.uint64), blocks),
         np.full(tokens * blocks, call % 2 ** 32, np.uint64),
         np.full(tokens * blocks, call >> 32, np.uint64)]
    k0, k1 = key % 2 ** 32, key >> 32
    for i in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> word) ^ c[1] ^ np.uint64((k0 + i * 0x9E3779B9) % 2 ** 32), b & low,
             (a >> word) ^ c[3] ^ np.uint64((k1 + i * 0xBB67AE85) % 2 ** 32), a & low]
    bits = np.stack(c, 1).astype("<u4").view("<u2").reshape(tokens, -1)[:, :case["channels"]]
    dropped = round(_DROP * 65536)
    keep = torch.from_numpy(bits >= dropped).cuda().reshape(s["x"].shape)
    inside = _inside(s).double()[..., None]
    factor = keep.double() * inside / (1 - dropped / 65536)
    y = s["x"].double() * factor
    if case["residual"]:
        y += s["residual"].double() * inside
    return {"y": y, "dx": s["dy"].double() * factor} if case["train"] else {"y": y}


def _loss_exact(s):
    x, table = s["x"].double(), s["table"].double()
    logp = torch.matmul(x, table.t()).mul_(float(np.float32(s["scale"])))
    lse = torch.logsumexp(logp, 1)
    logp -= lse[:, None]
    tokens = torch.nonzero(s["targets"] >= 0)[:, 0]
    target = s["targets"].long()[tokens]
    loss = torch.zeros_like(lse)
    loss[tokens] = -logp[tokens, target]
    out = {"loss": loss, "lse": lse}
    if s["case"]["train"]:
        p = logp.exp_()
        p[tokens, target] -= 1
        weight = torch.zeros_like(lse)
        weight[tokens] = s["dloss"].double()[tokens] * float(np.float32(s["scale"]))
        p *= weight[:, None]
        out.update(dx=p @ table, dtable=p.t() @ x)
    return out


def exact(case, seed):
    return {"norm": _norm_exact, "dropout": _dropout_exact,
            "loss": _loss_exact}[case["op"]](prepare(case, seed))
