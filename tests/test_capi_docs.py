"""Docstrings of the Python binding say what their function does, in sentences, and hold no code that a replacement put there."""
import inspect
import re

import pytest

from sddmm_gpu_amd import capi

DOCUMENTED = [(name, f) for owner in (capi, capi.Plan, capi.Coo, capi.AttentionDesc, capi.RotaryDesc)
              for name, f in vars(owner).items() if inspect.isfunction(getattr(f, "__func__", f)) and getattr(f, "__doc__", None)]


@pytest.mark.parametrize("name,f", DOCUMENTED, ids=[n for n, _ in DOCUMENTED])
def test_no_assignments(name, f):
    assert not re.search(r"^\s*[A-Z_0-9, ]+ = ", f.__doc__, re.M), f.__doc__


def test_spmm_form():
    assert capi.Plan.spmm_form.__doc__.startswith("SPMM_CSR, SPMM_TILES, SPMM_WALK or SPMM_BLOCKS: ")
