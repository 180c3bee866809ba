"""Samples of a cloud as the tokens of a small sequence model: trained by a few
steps, then fed sample by sample.

    python examples/sequence_model.py [--samples M] [--steps K]

Farthest point sampling picks the samples; in the order of their grid cells
they are a sequence, a sample's cell being its token.  The model is

    e = scale * table[token]            nsfps_embed
    u = e @ w_in  ->  x, b, c, dt       (the caller's product)
    v = silu(conv(x, b, c))             nsfps_conv
    y = scan(v, dt)                     nsfps_scan
    z = y @ w_out                       (the caller's product)

and learns to give a token's embedding from the tokens before it.  The
gradients come from nsfps_scan_grad, nsfps_conv_grad and nsfps_embed_grad.
Afterwards the first half of the sequence is read as a prompt and the other
half one token a call (nsfps_scan_step), over the same caches.

torch holds the device memory and does the two products.
"""

import argparse
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from ns_fps_amd import capi  # noqa: E402
from ns_fps_amd.workloads import make_workload  # noqa: E402

HEADS, GROUPS, HEAD_DIM, STATE_DIM, WIDTH, MODEL = 4, 1, 32, 32, 4, 64
INNER = HEADS * HEAD_DIM
CHANNELS = INNER + 2 * GROUPS * STATE_DIM  # x, b, c: what the convolution mixes


def rows(t, offset=0):
    """nsfps_rows of [B, L, C], from channel ``offset`` on."""
    return (t.data_ptr() + offset * t.element_size(), t.stride(0), t.stride(1))


def stream():
    return torch.cuda.current_stream().cuda_stream


def cell_tokens(points, bounds, blocks):
    """A point's cell of the grid, as a token."""
    lo, hi = np.array(bounds[0::2]), np.array(bounds[1::2])
    cell = ((points - lo) / (hi - lo) * blocks).astype(np.int64).clip(0, np.array(blocks) - 1)
    return (cell[:, 0] * blocks[1] + cell[:, 1]) * blocks[2] + cell[:, 2]


class Model:
    def __init__(self, lib, vocabulary, gen):
        def normal(*shape, scale):
            return torch.randn(*shape, generator=gen, device="cuda") * scale
        self.lib, self.vocabulary = lib, vocabulary
        self.p = {"table": normal(vocabulary, MODEL, scale=1 / math.sqrt(MODEL)),
                  "w_in": normal(MODEL, CHANNELS + HEADS, scale=1 / math.sqrt(MODEL)),
                  "conv_w": normal(CHANNELS, WIDTH, scale=0.5),
                  "conv_b": torch.zeros(CHANNELS, device="cuda"),
                  "a": -1 - torch.arange(HEADS, device="cuda").float(),
                  "d": torch.ones(HEADS, device="cuda"),
                  "dt_bias": torch.full((HEADS,), -2.0, device="cuda"),
                  "w_out": normal(INNER, MODEL, scale=1 / math.sqrt(INNER))}
        self.scale = math.sqrt(MODEL)

    def with_workspace(self, args, *sizes):
        ws = torch.empty(max(size(args) for size in sizes), dtype=torch.uint8, device="cuda")
        args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
        return ws  # the caller keeps it while calls with these args may run

    def embed_args(self, tokens, table, out):
        return capi.EmbedArgs(tokens=tokens.numel(), rows=self.vocabulary, width=MODEL,
                              scale=self.scale, table_stride=MODEL, out_stride=MODEL,
                              d_table=table.data_ptr(), d_tokens=tokens.data_ptr(),
                              d_out=out.data_ptr())

    def embed(self, tokens):
        out = torch.empty(1, tokens.numel(), MODEL, device="cuda")
        self.lib.embed_device(self.embed_args(tokens, self.p["table"], out), stream())
        return out

    def conv_args(self, u, v):
        p = self.p
        return capi.ConvArgs(batch=1, length=u.shape[1], channels=CHANNELS, width=WIDTH, x=rows(u),
                             y=rows(v), d_weight=p["conv_w"].data_ptr(),
                             d_bias=p["conv_b"].data_ptr())

    def scan_args(self, u, v, y):
        p = self.p
        return capi.ScanArgs(batch=1, length=u.shape[1], heads=HEADS, groups=GROUPS,
                             head_dim=HEAD_DIM, state_dim=STATE_DIM, x=rows(v), b=rows(v, INNER),
                             c=rows(v, INNER + GROUPS * STATE_DIM), dt=rows(u, CHANNELS), y=rows(y),
                             d_a=p["a"].data_ptr(), d_d=p["d"].data_ptr(),
                             d_dt_bias=p["dt_bias"].data_ptr())

    def caches(self):
        """Of one sequence: the convolution's last inputs, and the state."""
        return (torch.zeros(1, WIDTH, CHANNELS, device="cuda"),
                torch.zeros(1, HEADS, HEAD_DIM, STATE_DIM, device="cuda"))

    def forward(self, tokens, caches=None):
        """A whole prompt; with ``caches`` it leaves them for the tokens after it."""
        e = self.embed(tokens)
        u = e @ self.p["w_in"]
        v = torch.empty(1, tokens.numel(), CHANNELS, device="cuda")
        y = torch.empty(1, tokens.numel(), INNER, device="cuda")
        conv, scan = self.conv_args(u, v), self.scan_args(u, v, y)
        if caches:
            conv.d_cache, scan.d_state = (c.data_ptr() for c in caches)
        ws = self.with_workspace(scan, self.lib.scan_workspace_bytes)
        self.lib.conv_device(conv, stream())
        self.lib.scan_device(scan, stream())
        return y @ self.p["w_out"], (e, u, v, y, ws)

    def backward(self, tokens, kept, dz):
        """Gradients of all parameters from the output's."""
        p, lib, n = self.p, self.lib, tokens.numel()
        e, u, v, y, _ = kept
        g = {k: torch.empty_like(t) for k, t in p.items()}
        g["w_out"] = y[0].T @ dz[0]
        dy = dz @ p["w_out"].T
        dv, du = torch.empty_like(v), torch.empty_like(u)
        scan = self.scan_args(u, v, y)
        ws1 = self.with_workspace(scan, lib.scan_grad_workspace_bytes)
        lib.scan_grad_device(scan, capi.ScanGrads(
            dy=rows(dy), dx=rows(dv), db=rows(dv, INNER),
            dc=rows(dv, INNER + GROUPS * STATE_DIM), ddt=rows(du, CHANNELS),
            d_da=g["a"].data_ptr(), d_dd=g["d"].data_ptr(),
            d_ddt_bias=g["dt_bias"].data_ptr()), stream())
        conv = self.conv_args(u, v)
        ws2 = self.with_workspace(conv, lib.conv_grad_workspace_bytes)
        lib.conv_grad_device(conv, capi.ConvGrads(
            dy=rows(dv), dx=rows(du), d_dweight=g["conv_w"].data_ptr(),
            d_dbias=g["conv_b"].data_ptr()), stream())
        g["w_in"] = e[0].T @ du[0]
        de = (du @ p["w_in"].T).reshape(n, MODEL)
        embed = self.embed_args(tokens, g["table"], de)
        ws3 = self.with_workspace(embed, lib.embed_grad_workspace_bytes)
        lib.embed_grad_device(embed, stream())
        del ws1, ws2, ws3  # torch reuses them on this stream only, after these calls
        return g

    def step(self, token, position, caches):
        """One token over the caches; position is a device int32 [1]."""
        p = self.p
        u = (self.embed(token) @ p["w_in"])[0]
        y = torch.empty(1, INNER, device="cuda")
        self.lib.scan_step_device(capi.StepArgs(
            batch=1, heads=HEADS, groups=GROUPS, head_dim=HEAD_DIM, state_dim=STATE_DIM,
            width=WIDTH, xbc_stride=u.stride(0), dt_stride=u.stride(0), y_stride=INNER,
            d_xbc=u.data_ptr(), d_weight=p["conv_w"].data_ptr(), d_bias=p["conv_b"].data_ptr(),
            d_dt=u.data_ptr() + 4 * CHANNELS, d_a=p["a"].data_ptr(), d_d=p["d"].data_ptr(),
            d_dt_bias=p["dt_bias"].data_ptr(), d_positions=position.data_ptr(),
            d_cache=caches[0].data_ptr(), d_state=caches[1].data_ptr(), d_y=y.data_ptr()),
            stream())
        return y @ p["w_out"]


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--samples", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=20)
    opt = ap.parse_args(argv)
    if opt.samples < 2 or opt.steps < 1:
        ap.error("at least 2 samples and 1 step")
    lib = capi.Lib()
    work = make_workload("quickstart")
    cloud, bounds, blocks = work["clouds"][0], work["range"][:6], work["range"][6:]
    picked = cloud[lib.fps(cloud, opt.samples, work["range"])]
    cells = cell_tokens(picked, bounds, blocks)
    tokens = torch.from_numpy(np.sort(cells).astype(np.int32)).cuda()
    gen = torch.Generator(device="cuda").manual_seed(0)
    model = Model(lib, int(np.prod(blocks)), gen)

    losses = []
    target = model.embed(tokens)[:, 1:].clone()  # fixed: the first table's rows
    speed = {k: torch.zeros_like(v) for k, v in model.p.items()}
    for _ in range(opt.steps):
        z, kept = model.forward(tokens)
        miss = torch.zeros_like(z)
        miss[:, :-1] = z[:, :-1] - target
        losses.append(miss.square().mean().item())
        grads = model.backward(tokens, kept, miss * (2 / miss.numel()))
        for k, v in model.p.items():
            # steps of the gradient's direction, with momentum
            speed[k] = 0.8 * speed[k] + grads[k] / (grads[k].norm() + 1e-12)
            v -= 0.02 * v.norm().clamp(min=0.1) * speed[k]
        model.p["a"].clamp_(max=-1e-3)
    print(f"{len(tokens)} samples, loss {losses[0]:.4f} -> {losses[-1]:.4f}")

    whole, _ = model.forward(tokens)
    half = len(tokens) // 2
    caches = model.caches()
    out = [model.forward(tokens[:half], caches)[0][0]]
    for t in range(half, len(tokens)):
        position = torch.tensor([t], dtype=torch.int32, device="cuda")
        out.append(model.step(tokens[t:t + 1], position, caches))
    off = ((torch.cat(out) - whole[0]).norm() / whole.norm()).item()
    print(f"prompt of {half} and {len(tokens) - half} single tokens: relative difference {off:.1e}")
    return losses, off


if __name__ == "__main__":
    main()
