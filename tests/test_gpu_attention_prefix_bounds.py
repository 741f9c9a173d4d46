"""Prefixes far outside a sequence: below 0 none, above its keys all of them, behind shared keys too."""
import pytest

from test_gpu_attention import BF16, F32, Case

pytestmark = pytest.mark.gpu

FAR = [-2 ** 31, -1, 2 ** 31 - 1, 2 ** 30, -2 ** 31 + 5]
LENS = [(3, 40), (1, 7), (5, 90), (2, 2), (4, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shared", [0, 1, 300])
def test_far_prefixes(dtype, shared):
    c = Case(dtype, LENS, 4, 2, 64, -1, 0, prefix=FAR, packed=False, shared=shared)
    c.run()
    c.prefix = [min(max(p, 0), 10 ** 6) for p in FAR]  # (the same prefixes: a sequence has fewer keys)
    c.check()
