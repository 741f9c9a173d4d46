"""How large a workspace sddmm_attention_paged asks for (no GPU needed: nothing is launched)."""
import pytest

from sddmm_gpu_amd import capi


def workspace(type, held, n_seq, heads, kv, dim, max_q, rows, max_k, packed=True):
    more = dict(q_ptr=1 << 20, q_rows=rows) if packed else {}
    d = capi.AttentionDesc.packed(type, n_seq, heads, kv, dim, max_q=max_q, max_k=max_k, k_seq=0, v_seq=0, **more)
    c = capi.CacheDesc.packed(held, 1 << 20, 64, kv, dim, block_len=16, k=1 << 21, v=1 << 22, k_scale=1 << 23, v_scale=1 << 24, table=1 << 25, table_row=(max_k + 63) // 64)
    return capi.attention_paged_workspace_bytes(d, c)


@pytest.mark.parametrize("type,held", [(capi.TYPE_BF16, capi.TYPE_I8), (capi.TYPE_F16, capi.TYPE_F16), (capi.TYPE_F32, capi.TYPE_E4M3)])
@pytest.mark.parametrize("heads,kv", [(32, 1), (32, 8), (40, 2), (8, 8), (96, 2)])
@pytest.mark.parametrize("n_seq,max_q,rows", [(4, 16384, 16384), (32, 2048, 2079), (32, 8192, 8223), (256, 512, 2048), (1000, 100, 2000), (5000, 7, 5000), (1, 4096, 4096), (64, 1, 64), (3, 20, 25)])
def test_parts_stay_small(type, held, heads, kv, n_seq, max_q, rows):
    """A call keeps parts of rows for as many workgroups as fill the card some times over, whatever the lengths: 4096 of at most 32 rows, 512 of at most 256, each row of
    a head's elements and two statistics in fp32, besides parts of as many rows as there are."""
    dim = 128
    for max_k in (1000, 16384, 131072, 1 << 20, 1 << 29):
        row = 4 * (dim + 2)
        assert workspace(type, held, n_seq, heads, kv, dim, max_q, rows, max_k) <= row * (2 * rows * heads + 4096 * 32 + 2 * 512 * 256 + 256), max_k


def test_mixed_batches():
    """Packed batches of long and short sequences: no more for longer caches than short sequences' own rows need."""
    for n_seq, heads, kv, max_q, rows in ((32, 32, 8, 2048, 2079), (32, 32, 8, 8192, 8223), (4, 32, 1, 16384, 16384), (4, 32, 8, 16384, 16384)):
        short = workspace(capi.TYPE_BF16, capi.TYPE_I8, n_seq, heads, kv, 128, max_q, rows, 4096)
        for max_k in (32768, 131072, 1 << 20):
            assert workspace(capi.TYPE_BF16, capi.TYPE_I8, n_seq, heads, kv, 128, max_q, rows, max_k) - short <= 4096 * 32 * 4 * 130 + 1024


def test_few_rows_of_many_heads():
    """Packed batches of fewer rows than a tile holds, whose longest sequence is bounded by nothing but their sum."""
    for n_seq, heads, kv in ((42, 96, 32), (19, 160, 32), (54, 96, 3), (382, 64, 2), (30, 128, 64)):
        for max_k in (4096, 131072, 1 << 24):
            rows, row = n_seq, 4 * (128 + 2)
            assert workspace(capi.TYPE_BF16, capi.TYPE_I8, n_seq, heads, kv, 128, rows, rows, max_k) <= row * (2 * rows * heads + 4096 * 32 + 512 * 256 + 256), (n_seq, heads, kv, max_k)
