"""sddmm_attention_paged over rows that are wider than their heads: what follows a head's elements in a row of the cache does not reach the results."""
import pytest
import torch

import tests.test_gpu_cache as base
from tests.test_gpu_cache import BF16, F16, F32, check_attend

pytestmark = pytest.mark.gpu


class Padded(base.Pages):
    """Rows end in elements that are no numbers (8-bit integers: the largest code)."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        for g in self.gpu.values():
            g.view(torch.uint8)[..., self.dim * g.element_size():] = 127 if self.held == "i8" else 255


@pytest.fixture(autouse=True)
def padded(monkeypatch):
    monkeypatch.setattr(base, "Pages", Padded)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 80, 88, 104, 112, 120])
def test_head_sizes(dtype, held, dim):
    """Few rows, many rows, and both in one batch."""
    check_attend(dtype, held, [1, 4], [70, 100], 4, 2, dim, 16, 8, by_token=dim % 16 == 8, pad=1)
    check_attend(dtype, held, [70, 3], [100, 47], 4, 2, dim, 32, 8, by_token=dim % 16 == 0, pad=1)
    check_attend(dtype, held, [90, 1, 1, 2, 1, 1, 1], [130, 70, 1, 33, 300, 64, 17], 4, 2, dim, 32, 16, pad=1)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dim", [72, 80, 88, 104, 112, 120])
def test_many_sequences(held, dim):
    """So many rows that a workgroup takes 256."""
    check_attend(BF16, held, [120] * 16, [120 + 9 * i for i in range(16)], 8, 8, dim, 16, 4, pad=1)
