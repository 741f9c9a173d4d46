"""sddmm_attention_* on sequences with more rows than keys under bounded right windows: rows whose position lies before the first key see the
keys that their window reaches, forwards and backwards, whichever kernel takes them."""
import pytest

from test_gpu_attention import BF16, F16, F32, Case
from test_gpu_attention_backward import backward, check

pytestmark = pytest.mark.gpu

# windows to the right of 1, of fewer and of more than the keys; to the left too; rows before the first that sees a key among them
WINDOWS = [(-1, 1), (-1, 5), (20, 33), (-1, 200), (7, 1000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("left,right", WINDOWS)
def test_few_keys(dtype, packed, left, right):
    lens = [(10, 8), (40, 20), (300, 130), (129, 1), (5, 0), (33, 33)]
    check(backward(Case(dtype, lens, 4, 2, 64, left, right, packed=packed)).check())
    check(backward(Case(dtype, lens, 2, 2, 96, left, right, packed=packed, prefix=[0, 3, 50, 1, 2, 40], cap=4.0, bias=True)).check())


# (the lengths of head take these to tiles of 64 and of 128 keys)
@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 104), (F32, 32)])
@pytest.mark.parametrize("left,right", WINDOWS[1:4])
def test_whole_tiles_of_keys(dtype, dim, left, right):
    # of four sequences, and cut into pieces of the rows that see them
    check(backward(Case(dtype, [(1100, 700), (1000, 750), (1100, 690), (900, 640)], 8, 8, dim, left, right)).check())
    check(backward(Case(dtype, [(1500, 900)], 16, 1, dim, left, right)).check())
