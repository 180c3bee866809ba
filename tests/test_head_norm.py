"""Norms of queries and keys by head with their rotation, and the gradient,
against plain implementations in 64 bits; and the refusals.

Tolerances.  A head's sum of squares adds up to 22 roundings (16 values a lane,
six steps across lanes), half of which the root passes on, and the root's own
two units: 2^-20.  Two products (2^-23), cosine and sine with their angle
(2^-21) and the rotation's sum follow: 2^-18 of the pair's length, which the
rotation keeps, is twice the whole.  A bfloat16 output is rounded once more, by
2^-8 of itself at most.  The gradient goes through as many again: 2^-17 of its
terms' sizes.  The weights' sums have up to 64 terms in a row: 2^-17 of the sum
of the terms' sizes."""

import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT
from ns_fps_amd import capi
from test_sequence import A, DTYPES, EINVAL, EUNSUPPORTED, F64, laid_out, lib, ptr, rnd, rows, \
    stream, workspace  # noqa: F401

EPS = 1e-5


def inside_of(lens, length):
    return torch.arange(length)[None] < torch.tensor(lens)[:, None]


def pairs(r, neighbours):
    i = torch.arange(r // 2)
    return (2 * i, 2 * i + 1) if neighbours else (i, i + r // 2)


def angles(pos, length, freq):
    """[B, L, 1, R / 2], float64."""
    t = torch.tensor([max(p, 0) for p in pos], dtype=F64)[:, None] + torch.arange(length, dtype=F64)
    return (t[..., None] * freq.to(F64))[:, :, None]


def turned(v, angle, neighbours):
    r = 2 * angle.shape[-1]
    first, second = pairs(r, neighbours)
    a, b = v[..., first], v[..., second]
    out = v.clone()
    out[..., first] = a * torch.cos(angle) - b * torch.sin(angle)
    out[..., second] = a * torch.sin(angle) + b * torch.cos(angle)
    return out


def lengths_of_pairs(v, r, neighbours):
    """Every value's pair's length (behind the rotation its own size)."""
    first, second = pairs(r, neighbours)
    out = v.abs().clone()
    both = torch.hypot(v[..., first], v[..., second])
    out[..., first], out[..., second] = both, both
    return out


def norm_plain(x, w, angle, neighbours):
    """x [B, L, H, D] in float64."""
    n = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
    return turned(n * w, angle, neighbours)


# batch, length, q_heads, k_heads, head_dim, rotary_dim, neighbours, layout
CASES = [(1, 1, 1, 1, 1, 0, 0, "plain"), (1, 1, 1, 0, 2, 2, 1, "plain"),
         (2, 3, 2, 1, 64, 64, 0, "plain"), (3, 70, 1, 2, 64, 32, 1, "padded"),
         (1, 130, 4, 4, 128, 128, 1, "swapped"), (2, 65, 3, 3, 33, 32, 1, "odd"),
         (2, 17, 0, 2, 96, 48, 0, "plain"), (5, 9, 1, 1, 256, 256, 0, "padded"),
         (1, 33, 2, 1, 255, 100, 0, "odd"), (4, 20, 2, 2, 20, 4, 0, "plain"),
         (1, 5, 9, 3, 6, 6, 0, "plain"), (2, 64, 1, 1, 127, 126, 1, "plain"),
         (3, 12, 2, 2, 48, 0, 0, "plain"), (1, 1, 40, 40, 64, 64, 0, "plain")]


def inputs(case, dtype):
    batch, length, hq, hk, d, r, neighbours, how = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(1000 * d + length)
    x = {"q": rnd(gen, batch, length, hq * d, dtype=t), "k": rnd(gen, batch, length, hk * d, dtype=t)}
    x["q"][:, ::3] *= 1e-4  # heads at the size of eps
    w = {k: (1 + rnd(gen, d, scale=0.3)).to(t) for k in "qk"}
    freq = (10000.0 ** (-torch.arange(r // 2, dtype=F64) * 2 / max(r, 1))).float()
    lens = torch.randint(0, length + 1, (batch,), generator=gen).tolist()
    lens[0] = length
    if batch > 2:
        lens[1] = 0
    pos = torch.randint(0, 9, (batch,), generator=gen).tolist()
    pos[-1] = 2 ** 31 - 1 - length
    if batch > 1:
        pos[0] = -5
    return t, code, gen, x, w, freq, lens, pos


def on_device(case, code, x, w, freq, lens, pos):
    batch, length, hq, hk, d, r, neighbours, how = case
    D = {k: laid_out(v.cuda(), how) for k, v in x.items()}
    keep = [D, w["q"].cuda(), w["k"].cuda(), freq.cuda(),
            torch.tensor(lens, dtype=torch.int32).cuda(), torch.tensor(pos, dtype=torch.int32).cuda()]
    args = capi.NormArgs(batch=batch, length=length, q_heads=hq, k_heads=hk, head_dim=d,
                         rotary_dim=r, neighbours=neighbours, dtype=code, eps=EPS, q=rows(D["q"]),
                         k=rows(D["k"]), d_q_weight=ptr(keep[1]), d_k_weight=ptr(keep[2]),
                         d_freq=ptr(keep[3]) if r else None, d_lengths=ptr(keep[4]),
                         d_positions=ptr(keep[5]))
    return args, keep


def within(got, want, tol, what):
    g = got.detach().cpu().to(F64)
    assert g.shape == want.shape and torch.isfinite(g).all(), what
    tol = tol + (2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else 0) + 1e-35
    off = (g - want).abs() - tol
    assert (off <= 0).all(), f"{what}: {off.max().item():.3g} beyond"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_norm(lib, case, dtype):  # noqa: F811
    batch, length, hq, hk, d, r, neighbours, how = case
    t, code, gen, x, w, freq, lens, pos = inputs(case, dtype)
    clean = {k: v.clone() for k, v in x.items()}
    for v in x.values():
        for b, n in enumerate(lens):
            v[b, n:] = float("nan")  # past the end: never read
    args, keep = on_device(case, code, x, w, freq, lens, pos)
    out = {k: laid_out(torch.full_like(v, float("nan")).cuda(), how) for k, v in x.items()}
    args.q_out, args.k_out = rows(out["q"]), rows(out["k"])
    lib.norm_device(args, stream())
    angle, inside = angles(pos, length, freq), inside_of(lens, length)[..., None, None]
    for k, heads in (("q", hq), ("k", hk)):
        v = clean[k].to(F64).reshape(batch, length, heads, d)
        want = norm_plain(v, w[k].to(F64), angle, neighbours) * inside
        tol = 2.0 ** -18 * lengths_of_pairs(want, r, neighbours)
        within(out[k], want.reshape(batch, length, -1), tol.reshape(batch, length, -1), k)
        if how in ("padded", "odd") and heads:  # nothing beside the rows is written
            whole = out[k]._base
            assert torch.isnan(whole[..., heads * d:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES)
def test_norm_gradient(lib, case, dtype):  # noqa: F811
    batch, length, hq, hk, d, r, neighbours, how = case
    t, code, gen, x, w, freq, lens, pos = inputs(case, dtype)
    dy = {k: rnd(gen, *v.shape, dtype=t) for k, v in x.items()}
    clean = [{k: v.clone() for k, v in s.items()} for s in (x, dy)]
    for s in (x, dy):
        for v in s.values():
            for b, n in enumerate(lens):
                v[b, n:] = float("nan")
    args, keep = on_device(case, code, x, w, freq, lens, pos)
    G = {k: laid_out(v.cuda(), how) for k, v in dy.items()}
    out = {k: laid_out(torch.full_like(v, float("nan")).cuda(), how) for k, v in x.items()}
    dw = {k: torch.full((d,), 9.0, device="cuda") for k in "qk"}
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_grad_device(args, capi.NormGrads(
        dq_out=rows(G["q"]), dk_out=rows(G["k"]), dq=rows(out["q"]), dk=rows(out["k"]),
        d_dq_weight=ptr(dw["q"]), d_dk_weight=ptr(dw["k"])), stream())
    angle, inside = angles(pos, length, freq), inside_of(lens, length)[..., None, None].to(F64)
    for k, heads in (("q", hq), ("k", hk)):
        v = clean[0][k].to(F64).reshape(batch, length, heads, d).requires_grad_()
        wk = w[k].to(F64).requires_grad_()
        g = clean[1][k].to(F64).reshape(batch, length, heads, d) * inside
        want = torch.autograd.grad((norm_plain(v, wk, angle, neighbours) * g).sum(), (v, wk))
        with torch.no_grad():
            size = lengths_of_pairs(g, r, neighbours)
            root = 1 / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)
            n = v * root
            tol = 2.0 ** -17 * root * (size * wk.abs()
                                       + n.abs() * (size * wk * n).abs().mean(-1, keepdim=True))
            terms = (size * n).abs().sum((0, 1, 2))
        within(out[k], want[0].reshape(batch, length, -1), tol.reshape(batch, length, -1), f"d{k}")
        within(dw[k], want[1], 2.0 ** -17 * terms, f"d{k}_weight")


@pytest.mark.gpu
def test_norm_gradient_against_differences(lib):  # noqa: F811
    """One direction through all inputs: differences of the 64-bit loss."""
    case = (2, 40, 3, 2, 24, 16, 1, "plain")
    batch, length, hq, hk, d, r, neighbours, how = case
    t, code, gen, x, w, freq, lens, pos = inputs(case, "f32")
    dy = {k: rnd(gen, *v.shape) for k, v in x.items()}
    args, keep = on_device(case, code, x, w, freq, lens, pos)
    G = {k: v.cuda() for k, v in dy.items()}
    out = {k: torch.empty_like(v) for k, v in G.items()}
    dw = {k: torch.empty(d, device="cuda") for k in "qk"}
    ws = workspace(lib.norm_grad_workspace_bytes(args))
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_grad_device(args, capi.NormGrads(
        dq_out=rows(G["q"]), dk_out=rows(G["k"]), dq=rows(out["q"]), dk=rows(out["k"]),
        d_dq_weight=ptr(dw["q"]), d_dk_weight=ptr(dw["k"])), stream())
    angle, inside = angles(pos, length, freq), inside_of(lens, length)[..., None, None].to(F64)
    dirs = {k: torch.randn(x[k].shape, generator=gen, dtype=F64) for k in "qk"}
    wdirs = {k: torch.randn(d, generator=gen, dtype=F64) for k in "qk"}

    def loss(e):
        total = 0
        for k, heads in (("q", hq), ("k", hk)):
            v = (x[k].to(F64) + e * dirs[k] * x[k].to(F64).abs()).reshape(batch, length, heads, d)
            y = norm_plain(v, w[k].to(F64) + e * wdirs[k], angle, neighbours) * inside
            total = total + (y.reshape(batch, length, -1) * dy[k].to(F64)).sum()
        return total

    eps = 1e-6
    diff = (loss(eps) - loss(-eps)) / (2 * eps)
    terms = [(out[k].cpu().to(F64) * dirs[k] * x[k].to(F64).abs()).flatten() for k in "qk"]
    terms += [dw[k].cpu().to(F64) * wdirs[k] for k in "qk"]
    terms = torch.cat(terms)
    assert abs(terms.sum() - diff) <= 2.0 ** -14 * terms.norm() + 1e-5


@pytest.mark.gpu
def test_ones_for_weights_and_empty_calls(lib):  # noqa: F811
    """No weights are ones; a gradient of no tokens has weights' gradients of 0."""
    x = torch.randn(1, 4, 32, device="cuda")
    y, z = torch.empty_like(x), torch.empty_like(x)
    one = torch.ones(32, device="cuda")
    args = capi.NormArgs(batch=1, length=4, q_heads=1, head_dim=32, eps=EPS, q=rows(x), q_out=rows(y))
    lib.norm_device(args, stream())
    args.d_q_weight, args.q_out = ptr(one), rows(z)
    lib.norm_device(args, stream())
    assert torch.equal(y, z)
    dw = torch.full((32,), 7.0, device="cuda")
    empty = capi.NormArgs(batch=0, length=4, q_heads=1, head_dim=32, eps=EPS)
    ws = workspace(lib.norm_grad_workspace_bytes(empty))
    empty.workspace, empty.workspace_bytes = ws.data_ptr(), ws.numel()
    lib.norm_grad_device(empty, capi.NormGrads(d_dq_weight=ptr(dw)), stream())
    assert dw.eq(0).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_head(lib):  # noqa: F811
    x = torch.randn(1, 3, 4 * 16, device="cuda")
    want = torch.empty_like(x)
    freq = torch.ones(8, device="cuda")

    def call(src, dst):
        lib.norm_device(capi.NormArgs(batch=1, length=3, q_heads=4, head_dim=16, rotary_dim=16,
                                      eps=EPS, q=rows(src), q_out=rows(dst), d_freq=ptr(freq)),
                        stream())
    call(x, want)
    bad = x.clone()
    bad[0, 1, 16], bad[0, 1, 40] = float("nan"), float("inf")
    got = torch.empty_like(x)
    call(bad, got)
    clean = torch.ones(1, 3, 64, dtype=torch.bool, device="cuda")
    clean[0, 1, 16:48] = False
    assert torch.equal(got[clean], want[clean])
    assert torch.isnan(got[0, 1, 16:32]).all()


# -------------------------------------------------------------------- refusals

def good(**kw):
    return capi.NormArgs(**{**dict(batch=2, length=8, q_heads=2, k_heads=1, head_dim=8, rotary_dim=8,
                                   eps=1e-5, q=(A, 128, 16), k=(A, 64, 8), q_out=(A, 128, 16),
                                   k_out=(A, 64, 8), d_freq=A, workspace=A,
                                   workspace_bytes=1 << 30), **kw})


def good_grads(**kw):
    return capi.NormGrads(**{**dict(dq_out=(A, 128, 16), dk_out=(A, 64, 8), dq=(A, 128, 16),
                                    dk=(A, 64, 8)), **kw})


REFUSED = [
    (dict(head_dim=0, rotary_dim=0), EINVAL), (dict(q_heads=0, k_heads=0), EINVAL),
    (dict(head_dim=257), EUNSUPPORTED), (dict(rotary_dim=7), EINVAL), (dict(rotary_dim=10), EINVAL),
    (dict(eps=0.0), EINVAL), (dict(eps=-1.0), EINVAL), (dict(eps=float("nan")), EINVAL),
    (dict(eps=float("inf")), EINVAL), (dict(dtype=2), EINVAL), (dict(q=(None, 128, 16)), EINVAL),
    (dict(q=(A + 2, 128, 16)), EINVAL), (dict(q_heads=1 << 22), EUNSUPPORTED),
    (dict(d_freq=None), EINVAL), (dict(d_freq=A + 2), EINVAL), (dict(d_lengths=A + 1), EINVAL),
    (dict(d_positions=A + 2), EINVAL), (dict(d_q_weight=A + 1), EINVAL),
    (dict(batch=1 << 20, length=1 << 12), EUNSUPPORTED), (dict(q=(A, 1 << 62, 16)), EINVAL)]


@pytest.mark.parametrize("change,status", REFUSED)
@pytest.mark.parametrize("grad", [False, True])
def test_refusals(change, status, grad):
    L = capi.Lib()
    with pytest.raises(capi.NsfpsError) as e:
        if grad:
            L.norm_grad_device(good(**change), good_grads())
        else:
            L.norm_device(good(**change))
    assert e.value.status == status


@pytest.mark.parametrize("change", [dict(q_out=(A, 128, 15)), dict(q_out=(A, 127, 16)),
                                    dict(k_out=(None, 64, 8)), dict(k_out=(A, 0, 8))])
def test_outputs_are_checked(change):
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().norm_device(good(**change))
    assert e.value.status == EINVAL


@pytest.mark.parametrize("args,grads", [
    (dict(workspace=None), {}), (dict(workspace=A + 16), {}), (dict(workspace_bytes=16), {}),
    ({}, dict(dq=(A, 128, 15))), ({}, dict(dk_out=(None, 64, 8))), ({}, dict(d_dq_weight=A + 2))])
def test_gradients_are_checked(args, grads):
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().norm_grad_device(good(**args), good_grads(**grads))
    assert e.value.status == EINVAL


def test_null_structs_and_empty_calls():
    L = capi.Lib()
    assert L.lib.nsfps_norm_device(None, None) == EINVAL
    assert L.lib.nsfps_norm_grad_device(None, good_grads(), None) == EINVAL
    assert L.lib.nsfps_norm_grad_device(good(), None, None) == EINVAL
    assert L.lib.nsfps_norm_grad_workspace_bytes(good(), None) == EINVAL
    L.norm_device(good(batch=0, q=(None, 0, 0)))
    L.norm_device(good(length=0, q=(None, 0, 0)))


def layout_of(name, struct, tmp_path):
    """Sizes and offsets of every field, as the C compiler lays them out and as
    the binding does."""
    fields = [f for f, _ in struct._fields_]
    prints = "".join(f'printf("%zu ", offsetof({name}, {f}));' for f in fields)
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include "nsfps.h"\n#include <stddef.h>\n#include <stdio.h>\n'
                   f'int main(void) {{ {prints} printf("%zu", sizeof({name})); return 0; }}\n')
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, stdout=subprocess.PIPE, text=True).stdout.split()
    return [int(v) for v in out], [getattr(struct, f).offset for f in fields] + [ctypes.sizeof(struct)]


@pytest.mark.parametrize("name,struct", [
    ("nsfps_norm_args", capi.NormArgs), ("nsfps_norm_grads", capi.NormGrads),
    ("nsfps_dropout_args", capi.DropoutArgs), ("nsfps_loss_args", capi.LossArgs),
    ("nsfps_loss_grads", capi.LossGrads)])
def test_bindings_mirror_the_header(name, struct, tmp_path):
    got, want = layout_of(name, struct, tmp_path)
    assert np.array_equal(got, want)
