"""The example that runs sampling and the sequence operators as one model."""

import importlib.util
import os

import pytest

from conftest import ROOT


def load():
    spec = importlib.util.spec_from_file_location(
        "sequence_model", os.path.join(ROOT, "examples", "sequence_model.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.gpu
@pytest.mark.parametrize("samples", [2, 65, 1000])
def test_model_learns_and_continues_a_prompt(samples):
    """The loss falls, and prompt + single tokens give the whole sequence's
    outputs: both are float32, so 2^-14 of the outputs' norm."""
    losses, off = load().main(["--samples", str(samples), "--steps", "12"])
    assert losses[-1] < losses[0]
    assert off <= 2.0 ** -14


def test_bad_arguments_are_refused():
    with pytest.raises(SystemExit):
        load().main(["--samples", "1"])
