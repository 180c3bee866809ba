"""Dropout: its mask against the generator written out in numpy, its values in
64 bits; and the refusals.

Tolerances.  A value is one fused product and sum (2^-24 of it) with a factor
that is rounded itself (2^-24 of the product): 2^-23 of the two terms' sizes in
float32; a bfloat16 output is rounded once more, by 2^-8 of
itself at most."""

import numpy as np
import pytest
import torch

from ns_fps_amd import capi
from test_head_norm import inside_of, within
from test_sequence import A, DTYPES, EINVAL, EUNSUPPORTED, F64, laid_out, lib, ptr, rnd, rows, \
    stream  # noqa: F401


def philox(counter, key):
    """Ten rounds of Philox 4x32 on 64-bit words; counter [4, n], key (2)."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k, low, half = [int(v) for v in key], np.uint64(2 ** 32 - 1), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]),
             a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c)


@pytest.mark.parametrize("counter,key,want", [
    ([0] * 4, [0] * 2, [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]),
    ([0xffffffff] * 4, [0xffffffff] * 2, [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]),
    ([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0],
     [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1])])
def test_the_generator_gives_its_published_answers(counter, key, want):
    got = philox([[v] for v in counter], key)[:, 0]
    assert [int(v) for v in got] == want


def keep_of(batch, length, channels, p, seed):
    blocks, rows_n = -(-channels // 8), batch * length
    key, call = (int(v) % 2 ** 64 for v in seed)
    c = [np.tile(np.arange(blocks), rows_n), np.repeat(np.arange(rows_n), blocks),
         np.full(rows_n * blocks, call % 2 ** 32), np.full(rows_n * blocks, call >> 32)]
    words = philox(c, [key % 2 ** 32, key >> 32])
    bits = np.ascontiguousarray(words.T).astype("<u4").view("<u2").reshape(rows_n, -1)
    keep = bits[:, :channels] >= round(p * 65536)
    return torch.from_numpy(keep).reshape(batch, length, channels)


# batch, length, channels, layout
CASES = [(1, 1, 1, "plain"), (1, 1, 8, "plain"), (2, 3, 7, "plain"), (1, 130, 640, "plain"),
         (3, 17, 64, "padded"), (2, 33, 321, "odd"), (2, 9, 1000, "swapped"), (4, 5, 513, "plain"),
         (1, 2, 4096, "plain"), (2, 40, 24, "odd")]


def call(lib, case, code, x, residual, y, p, seed, lens):  # noqa: F811
    batch, length, channels, _ = case
    args = capi.DropoutArgs(batch=batch, length=length, channels=channels, dtype=code, p=p,
                            x=rows(x), y=rows(y), d_seed=ptr(seed), d_lengths=ptr(lens))
    if residual is not None:
        args.residual = rows(residual)
    lib.dropout_device(args, stream())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("p,with_residual", [(0.1, True), (0.5, False), (0.0, True), (1.0, True)])
def test_dropout(lib, case, dtype, p, with_residual):  # noqa: F811
    batch, length, channels, how = case
    t, code = DTYPES[dtype]
    gen = torch.Generator().manual_seed(channels)
    x, r = rnd(gen, batch, length, channels, dtype=t), rnd(gen, batch, length, channels, dtype=t)
    lens = torch.randint(0, length + 1, (batch,), generator=gen).tolist()
    lens[0] = length
    seed = torch.tensor([-3 - channels, (5 << 40) + length], dtype=torch.int64)
    keep = keep_of(batch, length, channels, p, seed.tolist())
    inside = inside_of(lens, length)[..., None]
    kept = 65536 / (65536 - round(p * 65536)) if p < 1 else 0.0
    a = torch.where(keep & inside, x.to(F64) * kept, 0.0)
    b = torch.where(inside, r.to(F64), 0.0) if with_residual else torch.zeros_like(a)
    xd, rd = x.clone(), r.clone()
    xd[~keep] = float("nan")  # what is dropped may hold anything
    for v in (xd, rd):
        for i, n in enumerate(lens):
            v[i, n:] = float("inf")
    xd, rd = laid_out(xd.cuda(), how), laid_out(rd.cuda(), how)
    y = laid_out(torch.full((batch, length, channels), float("nan"), dtype=t, device="cuda"), how)
    sd, ld = seed.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    call(lib, case, code, xd, rd if with_residual else None, y, p, sd, ld)
    within(y, a + b, 2.0 ** -23 * (a.abs() + b.abs()), "y")
    dropped = ~keep & inside
    assert torch.equal(y.cpu()[dropped].to(F64), b[dropped])  # the residual as it was
    if how in ("padded", "odd"):
        assert torch.isnan(y._base[..., channels:]).all()


@pytest.mark.gpu
def test_masks_hang_on_sizes_and_seed_alone(lib):  # noqa: F811
    """Types, strides, the residual and lengths leave the mask; the key and the
    call's number make another; replays of a graph read the seed they find."""
    case = (2, 50, 264, "plain")
    ones = torch.ones(2, 50, 264, device="cuda")
    seed = torch.tensor([1, 2], dtype=torch.int64, device="cuda")

    def mask(x, code=capi.F32, seed=seed):
        y = torch.empty_like(x)
        call(lib, case, code, x, None, y, 0.3, seed, None)
        return y != 0
    want = mask(ones)
    assert torch.equal(mask(ones.bfloat16(), capi.BF16), want)
    assert torch.equal(mask(laid_out(ones, "odd")), want)
    for other in ([2, 2], [1, 3], [1 + (1 << 32), 2], [1, 2 + (1 << 32)]):
        m = mask(ones, seed=torch.tensor(other, dtype=torch.int64, device="cuda"))
        # two independent masks differ in 2 * 0.3 * 0.7 = 0.42 of 26,400 values: a
        # deviation of 0.003
        assert abs((m != want).float().mean().item() - 0.42) < 0.02
    # 26,400 values dropped with 0.3: a deviation of 0.0028
    assert abs((~want).float().mean().item() - 0.3) < 0.015
    y = torch.empty_like(ones)
    graph = torch.cuda.CUDAGraph()
    call(lib, case, capi.F32, ones, None, y, 0.3, seed, None)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call(lib, case, capi.F32, ones, None, y, 0.3, seed, None)
    for n in (2, 9, 2, 40):
        seed[1] = n
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y != 0, mask(ones))
    assert not torch.equal(y != 0, want)


# -------------------------------------------------------------------- refusals

def good(**kw):
    return capi.DropoutArgs(**{**dict(batch=2, length=8, channels=8, p=0.1, x=(A, 64, 8),
                                      residual=(A, 64, 8), y=(A, 64, 8), d_seed=A), **kw})


@pytest.mark.parametrize("change,status", [
    (dict(p=-0.1), EINVAL), (dict(p=1.5), EINVAL), (dict(p=float("nan")), EINVAL),
    (dict(dtype=3), EINVAL), (dict(channels=0), EINVAL), (dict(channels=(1 << 24) + 1), EUNSUPPORTED),
    (dict(batch=1 << 16, length=1 << 16), EUNSUPPORTED), (dict(x=(None, 64, 8)), EINVAL),
    (dict(residual=(A + 1, 64, 8)), EINVAL), (dict(y=(A, 64, 7)), EINVAL), (dict(y=(A, 63, 8)), EINVAL),
    (dict(d_seed=None), EINVAL), (dict(d_seed=A + 4), EINVAL), (dict(d_lengths=A + 2), EINVAL),
    (dict(x=(A, 1 << 60, 8)), EINVAL)])
def test_refusals(change, status):
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().dropout_device(good(**change))
    assert e.value.status == status


def test_null_and_empty_calls():
    L = capi.Lib()
    assert L.lib.nsfps_dropout_device(None, None) == EINVAL
    L.dropout_device(good(batch=0, x=(None, 0, 0)))
    L.dropout_device(good(length=0, y=(None, 0, 0)))
