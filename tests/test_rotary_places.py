"""Results of sddmm_rotary in the place of operands: their own with the same strides, and nothing else."""
import pytest
import torch

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read


def desc(**kw):
    d = dict(type=capi.TYPE_BF16, n_rows=10, n_heads=4, n_kv_heads=4, head_dim=64, rot_dim=64, layout=capi.ROTARY_HALF)
    d.update(kw)
    return capi.RotaryDesc.packed(**d)


OTHER = dict(q_out_row=64, q_out_head=640)  # [head, row] instead of [row, head]
OTHER_K = dict(k_out_row=64, k_out_head=640)


@pytest.mark.parametrize("kw,places", [
    (OTHER, (A, A, 2 * A, 3 * A)), (OTHER_K, (A, 2 * A, 3 * A, 3 * A)), (dict(q_out_row=512), (A, A, 2 * A, 3 * A)), (dict(n_rows=1, q_out_head=128), (A, A, 2 * A, 3 * A)),
    (dict(n_kv_heads=0, **OTHER), (A, A, 0, 0)),
    ({}, (A, 2 * A, 2 * A, 3 * A)), ({}, (A, 2 * A, 3 * A, A)), ({}, (A, 2 * A, 3 * A, 2 * A)), ({}, (A, A, 2 * A, A)), ({}, (A, A, A, 2 * A))])
def test_refusals(kw, places):
    with pytest.raises(capi.SddmmError, match="place") as e:
        capi.rotary(desc(**kw), A, A, *places)
    assert e.value.code == capi.ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("layout", [capi.ROTARY_HALF, capi.ROTARY_INTERLEAVED])
def test_in_place(layout):
    """In place of one operand and not of the other, and with strides that no second row or head makes use of."""
    dev = "cuda:0"
    freq = torch.from_numpy(capi.rotary_frequencies(48)[0]).to(dev)
    for rows, heads, more in ((10, 4, {}), (1, 4, dict(q_out_row=999936)), (10, 1, dict(q_out_head=7))):
        q, k = (torch.randn(rows, heads, 64, device=dev).bfloat16() for _ in range(2))
        want, wk, other = torch.empty_like(q), torch.empty_like(k), torch.empty_like(k)
        capi.rotary(desc(n_rows=rows, n_heads=heads, n_kv_heads=heads, rot_dim=48, layout=layout, first_position=5), 0, freq.data_ptr(), q.data_ptr(), want.data_ptr(), k.data_ptr(), wk.data_ptr())
        d = desc(n_rows=rows, n_heads=heads, n_kv_heads=heads, rot_dim=48, layout=layout, first_position=5, **more)
        capi.rotary(d, 0, freq.data_ptr(), q.data_ptr(), q.data_ptr(), k.data_ptr(), other.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(q, want) and torch.equal(other, wk)
