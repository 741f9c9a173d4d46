"""Strides of sddmm_attention_* that no memory has are refused, also those whose bytes pass 64 bits (no GPU needed: nothing is launched)."""
import pytest

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read


@pytest.mark.parametrize("code,size", [(capi.TYPE_BF16, 2), (capi.TYPE_F16, 2), (capi.TYPE_F32, 4)])
@pytest.mark.parametrize("name", ["q_row", "k_row", "v_row", "o_row"])
def test_long_rows(code, size, name):
    for stride in ((1 << 23) // size, 1 << 40, 1 << 61, 1 << 62, (1 << 63) - 64):
        d = capi.AttentionDesc.packed(code, n_seq=2, n_heads=4, n_kv_heads=2, head_dim=64, max_q=100, max_k=100, **{name: stride})
        for call in (capi.attention_workspace_bytes, lambda d: capi.attention_forward(d, A, A, A, 2 * A, 0, A, 1 << 40)):
            with pytest.raises(capi.SddmmError, match="strides") as e:
                call(d)
            assert e.value.code == capi.ERR_ARG
    d = capi.AttentionDesc.packed(code, n_seq=2, n_heads=4, n_kv_heads=2, head_dim=64, max_q=100, max_k=100, **{name: (1 << 23) // size - 64})
    capi.attention_workspace_bytes(d)
