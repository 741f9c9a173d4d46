"""sddmm_attention_*: bounds of max_q and max_k far above what the packed arrays hold are as good as exact ones."""
import pytest
import torch

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read
MOST = (1 << 30) - 1


def packed(max_q, max_k, rows, keys, n_seq, heads, kv, **more):
    return capi.AttentionDesc.packed(capi.TYPE_BF16, n_seq, heads, kv, 64, max_q=max_q, max_k=max_k, q_ptr=A, k_ptr=A, q_rows=rows, k_rows=keys, window_right=0, **more)


@pytest.mark.parametrize("rows,keys,n_seq,heads,kv", [(4, 2000, 1, 8, 1), (64, 64, 3, 128, 1), (1, 5000, 1, 256, 2), (3000, 3000, 4, 16, 16), (10, 0, 2, 4, 4), (0, 7, 2, 4, 4)])
def test_workspace_of_wide_bounds(rows, keys, n_seq, heads, kv):
    for max_q, max_k in ((MOST, MOST), (MOST, keys), (rows, MOST), (rows + 1, keys + 1)):
        assert capi.attention_workspace_bytes(packed(max_q, max_k, rows, keys, n_seq, heads, kv)) == capi.attention_workspace_bytes(packed(rows, keys, rows, keys, n_seq, heads, kv))


@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,kv", [([(1, 1), (30, 40), (33, 3)], 128, 1), ([(4, 2000)], 8, 1), ([(70, 90)] * 70, 8, 2), ([(300, 200), (0, 5), (9, 0)], 4, 4)])
def test_wide_bounds(lens, heads, kv):
    from test_gpu_attention import BF16, Case
    from test_gpu_attention_backward import backward, check
    c = Case(BF16, lens, heads, kv, 64, -1, 0)
    c.desc.max_q, c.desc.max_k = c.desc.q_rows, c.desc.k_rows
    want = [x.clone() for x in (backward(c).out, c.lse, c.dq, c.dk, c.dv)]
    c.desc.max_q = c.desc.max_k = MOST
    check(backward(c).check())
    for a, b in zip(want, (c.out, c.lse, c.dq, c.dk, c.dv)):
        assert torch.equal(a, b)
