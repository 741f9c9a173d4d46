"""sddmm_attention_backward where keys that a row does not see hold infinities and NaNs: they reach no row of another tile and no other key's
gradients, and keys that no row sees get 0, whatever kernel takes them."""
import math

import pytest
import torch

import attention_reference as ref
from test_gpu_attention import BF16, F16, F32, Case
from test_gpu_attention_backward import backward

pytestmark = pytest.mark.gpu

NOT_FINITE = [math.nan, math.inf, -math.inf]
# few rows, tiles of 64 and of 128 rows: (sequences, heads)
BATCHES = [(1, 2), (16, 16), (60, 16)]


def spoil(c, begin, end):
    """Keys begin .. end - 1 of every sequence: one element of each, or all of them, is no number."""
    for _, rk in c.where:
        k = c.k[rk]
        for i in range(begin, end):
            if i % 2:
                k[i] = NOT_FINITE[i % 3]
            else:
                k[i, :, (7 * i) % c.dim] = NOT_FINITE[i % 3]


@pytest.mark.parametrize("dtype,dim", [(F32, 32), (F32, 56), (F32, 104), (BF16, 56), (BF16, 104), (F16, 64)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, True)])
@pytest.mark.parametrize("n,heads", BATCHES)
def test_rows_before_such_keys(dtype, dim, cap, bias, n, heads):
    """Causal: rows before the first such key give what they give without it, those of its tile of rows but for dq.  (32 rows raise their running maximum
    together, so those of a tile with NaNs are held to the bounds of attention in 64 bits instead of to the same bits.)"""
    good, c = (Case(dtype, [(200, 200)] * n, heads, heads, dim, -1, 0, cap=cap, bias=bias) for _ in range(2))
    spoil(c, 141, 160)
    backward(good)
    backward(c)
    for rq, _ in c.where:
        for a, b in ((c.out, good.out), (c.lse, good.lse), (c.dq, good.dq)):
            assert torch.equal(a[rq][:128], b[rq][:128])
        assert torch.isfinite(c.out[rq][:141]).all() and torch.isfinite(c.lse[rq][:141]).all()
        assert torch.isnan(c.dq[rq][141:]).any()
    for s in (0, n - 1):
        q, k, v = (x[:141] for x in c.operands(s, heads - 1))
        r = ref.head(q, k, v, -1, 0, 0, c.scale, cap, float(c.slopes[heads - 1]))
        assert ((c.out[c.where[s][0]][:141, heads - 1].cpu().double() - r["out"]).abs() <= r["out_tol"]).all()
        assert ((c.lse[c.where[s][0]][:141, heads - 1].cpu().double() - r["lse"]).abs() <= r["lse_tol"]).all()


@pytest.mark.parametrize("dtype,dim", [(F32, 32), (F32, 104), (BF16, 56), (BF16, 104), (F16, 64)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (5.0, True)])
@pytest.mark.parametrize("n,heads", BATCHES)
def test_keys_that_no_row_sees(dtype, dim, cap, bias, n, heads):
    """A window whose first row begins at key 155, in the middle of a tile: such keys before it change nothing and get gradients of 0."""
    good, c = (Case(dtype, [(100, 300)] * n, heads, heads, dim, 45, 0, cap=cap, bias=bias) for _ in range(2))
    spoil(c, 120, 155)
    backward(good)
    backward(c)
    for a, b in ((c.out, good.out), (c.dq, good.dq), (c.dk, good.dk), (c.dv, good.dv)) + (((c.ds, good.ds),) if bias else ()):
        assert torch.equal(a, b)
    for _, rk in c.where:
        assert (c.dk[rk][:155] == 0).all() and (c.dv[rk][:155] == 0).all()
