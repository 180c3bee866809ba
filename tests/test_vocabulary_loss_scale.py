"""Scales at the end of their numbers."""

import pytest

from ns_fps_amd import capi
from test_sequence import EINVAL
from test_vocabulary_loss import good, good_grads


@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_scales_whose_logits_have_no_number_are_refused(scale):
    """Logits are found in powers of two: scale * log2(e) has to be a number."""
    L = capi.Lib()
    for call in (lambda a: L.loss_device(a), lambda a: L.loss_grad_device(a, good_grads())):
        with pytest.raises(capi.NsfpsError) as e:
            call(good(scale=scale))
        assert e.value.status == EINVAL and "scale" in str(e.value)
