"""sddmm_cache_append and sddmm_attention_paged on rows of one array of queries, keys and values, results in rows of another's, and batches of more sequences than a wave has lanes."""
import pytest
import torch

from sddmm_gpu_amd import capi
from tests import cache_reference as cref
from tests.test_gpu_cache import BF16, CODE, DEV, F16, F32, Pages, check_attend, normal, stream, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (F16, "own"), (F32, "e4m3")])
@pytest.mark.parametrize("heads,kv,dim,rot,layout", [(4, 2, 64, 64, 0), (6, 1, 128, 40, 0), (8, 8, 40, 40, 1), (4, 2, 72, 72, 0)])
@pytest.mark.parametrize("n_new,after", [([3, 1, 2], [20, 1, 47]), ([70, 5, 33], [70, 90, 40])])
def test_rows_of_one_array(packed, dtype, held, heads, kv, dim, rot, layout, n_new, after):
    """The same bits as contiguous arrays give, and everything beside the rows stays."""
    page, block = 16, 8
    table, n_pages = tables(after, page, 3)
    total, most, wide = sum(n_new), max(n_new), (heads + 2 * kv) * dim + 16
    n_rows = total if packed else len(n_new) * most
    q, k, v = (normal(5 + i, n_rows, h, dim).to(dtype).to(DEV) for i, h in enumerate((heads, kv, kv)))
    one = torch.full((n_rows, wide), 9.0, dtype=dtype, device=DEV)
    views, at = {}, 0
    for name, x, h in (("q", q, heads), ("k", k, kv), ("v", v, kv)):
        views[name] = one.as_strided((n_rows, h, dim), (wide, dim, 1), at)
        views[name].copy_(x)
        at += h * dim
    before = one.clone()
    t, length = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, after))
    more = dict(max_q=most, max_k=max(after), k_len=length.data_ptr(), window_right=0)
    if packed:
        ptr = torch.tensor([0] + n_new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
        more.update(q_ptr=ptr.data_ptr(), q_rows=total)
    else:
        new = torch.tensor(n_new, dtype=torch.int32, device=DEV)
        more.update(q_len=new.data_ptr(), k_seq=most * kv * dim, v_seq=most * kv * dim)
    freq = torch.tensor([10000.0 ** (-2 * e / rot) for e in range(rot // 2)], dtype=torch.float64, device=DEV)
    results = []
    for strided in (False, True):
        pages = Pages(dtype, held, n_pages, page, block, kv, dim, False, 8)
        desc = capi.AttentionDesc.packed(CODE[dtype], len(n_new), heads, kv, dim, **more)
        wide_out = heads * dim + 32
        out = torch.full((n_rows, wide_out), 7.0, dtype=dtype, device=DEV)
        if strided:
            desc.q_row = desc.k_row = desc.v_row = wide
            desc.q_seq = desc.k_seq = desc.v_seq = most * wide
            desc.q_head = desc.k_head = desc.v_head = dim
            desc.o_row, desc.o_seq, desc.o_head = wide_out, most * wide_out, dim
            pq, pk, pv = (views[n].data_ptr() for n in "qkv")
            result = out.as_strided((n_rows, heads, dim), (wide_out, dim, 1), 0)
        else:
            turned = q.clone()
            pq, pk, pv = turned.data_ptr(), k.data_ptr(), v.data_ptr()
            result = torch.full((n_rows, heads, dim), 7.0, dtype=dtype, device=DEV)
        cache = pages.desc(t, rot_dim=rot, rot_layout=layout, rot_freq=freq.data_ptr())
        capi.cache_append(desc, cache, pq, pq, pk, pv, stream())
        size = capi.attention_paged_workspace_bytes(desc, cache)
        ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=DEV)
        capi.attention_paged(desc, cache, pq, result.data_ptr() if not strided else out.data_ptr(), 0, ws.data_ptr(), size, stream())
        torch.cuda.synchronize()
        got = views["q"] if strided else turned
        results.append([got.cpu().clone(), result.cpu().clone()] + [x.cpu().clone() for n in "kv" for x in (pages.gpu[n].view(torch.uint8), pages.scales[n]) if x is not None])
        if strided:
            assert torch.equal(one[:, heads * dim:], before[:, heads * dim:])  # keys, values and what follows them
            assert (out[:, heads * dim:] == 7.0).all()
    for x, y in zip(*results):
        assert torch.equal(x.nan_to_num(5.5) if x.is_floating_point() else x, y.nan_to_num(5.5) if y.is_floating_point() else y)


@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (F16, "e4m3"), (BF16, "own"), (F32, "i8")])
def test_more_sequences_than_lanes(dtype, held):
    """Packed: few rows in more than one tile of rows, a mixed batch, many rows."""
    check_attend(dtype, held, [9, 1, 0, 5] * 25, [9 + 3 * (i % 40) for i in range(100)], 8, 2, 64, 16, 8)
    check_attend(dtype, held, [1] * 40 + [90, 2, 0] + [1] * 40, [90 + i for i in range(83)], 4, 2, 64, 32, 16)
    check_attend(dtype, held, [17, 40] * 35, [40 + i for i in range(70)], 4, 1, 64, 32, 16)
