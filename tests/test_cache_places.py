"""Scales of a cache in each other's place, or in that of other arrays, which sddmm_cache_append refuses (no GPU needed: nothing is launched)."""
import pytest

from sddmm_gpu_amd import capi
from tests.test_cache_refusals import A, append, cache, desc, refuses

SIZE = 50 * 2 * 1 * 4  # bytes of a scale array of the cache there


@pytest.mark.parametrize("kw", [dict(k_scale=11 * A), dict(k_scale=11 * A + 4), dict(k_scale=11 * A + SIZE - 4), dict(k_scale=11 * A - SIZE + 4), dict(k_scale=11 * A - 8)])
def test_one_array_for_both(kw):
    refuses(lambda: append(desc(), cache(**kw)), "place")
    refuses(lambda: append(desc(), cache(type=capi.TYPE_E4M3, **kw)), "place")


@pytest.mark.parametrize("name", ["k_scale", "v_scale"])
def test_in_the_place_of_other_arrays(name):
    for kw in (dict(q=5 * A), dict(q_out=5 * A), dict(k=5 * A), dict(v=5 * A)):
        refuses(lambda: append(desc(), cache(**{name: 5 * A}), **kw), "place")
    for at in (8 * A, 9 * A):  # the cache's keys and values
        refuses(lambda: append(desc(), cache(**{name: at})), "place")
