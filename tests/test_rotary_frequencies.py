"""Rotary options whose numbers pass what a float holds are refused like any others that are none."""
import pytest
import torch

from rns_llm_amd import HipRNSBackend


def create(**options):
    return object.__new__(HipRNSBackend).create_rotary(device=torch.device("cpu"), **{"rotary_dim": 128, **options})


@pytest.mark.parametrize("options", [
    {"base": 5e-324}, {"scaling": "base", "factor": 1e308}, {"scaling": "linear", "factor": 1e-320},
    {"scaling": "bands", "factor": 1e-320, "original_length": 1}, {"magnitude": 1e39}, {"magnitude": -1e39},
    {"scaling": "base", "factor": 1e-5, "base": 1e-322},
])
def test_numbers_past_a_float(options):
    with pytest.raises(ValueError):
        create(**options)


def test_large_numbers_that_are_some():
    assert create(base=1e300).frequencies[-1] > 0 and create(magnitude=3e38).magnitude == 3e38
    assert create(frequencies=[1e300] * 64).steps.shape == (64,)
