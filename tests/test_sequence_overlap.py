"""The convolution and its gradient read tokens beside the ones they write: an
output over an input is refused where the strides show it, and interleaved
tensors that share no element are taken.  No call here reaches a device: calls
that would be taken are made only where there is none."""

import itertools
import random

import pytest

from ns_fps_amd import capi
from test_sequence import A, good_conv

Z = 4  # bytes of an element


FAR = A + (1 << 30)


@pytest.mark.parametrize("x,dy,dx", [
    ((A, 64, 8), (FAR, 64, 8), (A, 64, 8)), ((FAR, 64, 8), (A, 64, 8), (A, 64, 8)),  # in place
    ((FAR, 64, 8), (A, 0, 0), (A, 64, 8)),                   # a broadcast dy that starts there
    ((FAR, 64, 8), (A + 8 * Z, 64, 8), (A, 64, 8)),          # a token later
    ((FAR, 64, 8), (A - 8 * Z, 64, 8), (A, 64, 8)),          # a token before
    ((FAR, 64, 8), (A + 64 * Z, 64, 8), (A, 64, 8)),         # a sequence later
    ((FAR, 64, 8), (A + Z, 64, 8), (A, 64, 8)),              # a channel later
    ((A + 16 * Z, 8, 16), (FAR, 8, 16), (A, 8, 16)),         # tokens ahead of sequences
])
def test_gradient_over_its_inputs_is_refused(x, dy, dx):
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().conv_grad_device(good_conv(x=x), capi.ConvGrads(dy=dy, dx=dx, d_dweight=A))
    assert e.value.status == capi.NSFPS_EINVAL and "overlap" in str(e.value)


def test_forward_in_place_is_refused():
    with pytest.raises(capi.NsfpsError) as e:
        capi.Lib().conv_device(good_conv(y=(A + 8 * Z, 64, 8)))
    assert e.value.status == capi.NSFPS_EINVAL and "overlap" in str(e.value)


def meet(out, inp, batch, length, width):
    """Element by element."""
    def elements(p, bs, rs):
        return {p // Z + b * bs + t * rs + c for b in range(batch) for t in range(length)
                for c in range(width)}
    return bool(elements(*out) & elements(*inp))


def test_every_pair_of_equal_strides_is_told():
    """Random small layouts, both orders of the strides, against the elements
    themselves."""
    rng = random.Random(5)
    lib = capi.Lib()
    told = []
    for _ in range(3000):
        batch, length, width = rng.randint(1, 3), rng.randint(1, 4), rng.randint(1, 4)
        near = width + rng.randint(0, 6)
        many = [(length, "t"), (batch, "b")]
        if rng.random() < 0.5:
            many.reverse()
        far = (many[0][0] - 1) * near + width + rng.randint(0, 9)
        rs, bs = (near, far) if many[0][1] == "t" else (far, near)
        shift = rng.randint(-60, 60)
        dx, dy = (A + 4096, bs, rs), (A + 4096 + shift * Z, bs, rs)
        args = good_conv(batch=batch, length=length, channels=width, x=(FAR, bs, rs))
        grads = capi.ConvGrads(dy=dy, dx=dx, d_dweight=A)
        if meet(dx, dy, batch, length, width):
            with pytest.raises(capi.NsfpsError) as e:
                lib.conv_grad_device(args, grads)
            assert "overlap" in str(e.value)
            told.append(True)
        else:
            told.append(False)
            if lib.device_count() == 0:  # taken: the next check is for a device
                with pytest.raises(capi.NsfpsError) as e:
                    lib.conv_grad_device(args, grads)
                assert "no HIP device" in str(e.value)
    assert 300 < sum(told) < 2700


@pytest.mark.parametrize("order", list(itertools.permutations(range(3))))
def test_interleaved_tensors_are_taken(order):
    """x, dy and dx as thirds of one row."""
    lib = capi.Lib()
    if lib.device_count():
        pytest.skip("a taken call would run")
    x, dy, dx = ((A + 8 * Z * k, 24 * 8, 24) for k in order)
    with pytest.raises(capi.NsfpsError) as e:
        lib.conv_grad_device(good_conv(x=x), capi.ConvGrads(dy=dy, dx=dx, d_dweight=A))
    assert "no HIP device" in str(e.value)
