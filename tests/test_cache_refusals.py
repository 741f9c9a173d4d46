"""What sddmm_cache_append and sddmm_attention_paged refuse, and what they say (no GPU needed: nothing is launched)."""
import pytest

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read


def desc(**kw):
    d = dict(type=capi.TYPE_BF16, n_seq=2, n_heads=4, n_kv_heads=2, head_dim=64, max_q=3, max_k=100)
    d.update(kw)
    kv = d["n_kv_heads"] * d["head_dim"]
    d.setdefault("k_seq", d["max_q"] * kv)
    d.setdefault("v_seq", d["max_q"] * kv)
    return capi.AttentionDesc.packed(**d)


def cache(dim=64, **kw):
    d = dict(type=capi.TYPE_I8, n_pages=50, page_len=16, n_kv_heads=2, head_dim=dim, block_len=16, k=8 * A, v=9 * A, k_scale=10 * A, v_scale=11 * A, table=12 * A, table_row=7,
             rot_dim=dim, rot_freq=13 * A)
    d.update(kw)
    return capi.CacheDesc.packed(**d)


def append(d, c, q=A, q_out=2 * A, k=3 * A, v=4 * A):
    capi.cache_append(d, c, q, q_out, k, v)


def attend(d, c, q=A, out=2 * A, lse=0, ws=A, n=1 << 40):
    capi.attention_paged(d, c, q, out, lse, ws, n)


def refuses(call, says, code=capi.ERR_ARG):
    with pytest.raises(capi.SddmmError, match=says) as e:
        call()
    assert e.value.code == code


CACHES = [
    (dict(type=capi.TYPE_F16), "type"), (dict(type=capi.TYPE_F32), "type"), (dict(type=5), "type"), (dict(type=-1), "type"),
    (dict(page_len=0), "page_len"), (dict(page_len=8), "page_len"), (dict(page_len=24), "page_len"), (dict(page_len=1 << 17), "page_len"), (dict(page_len=-16), "page_len"),
    (dict(block_len=0), "block_len"), (dict(block_len=3), "block_len"), (dict(block_len=32), "block_len"), (dict(block_len=128, page_len=256), "block_len"), (dict(block_len=-1), "block_len"),
    (dict(k_row=60), "rows of the cache"), (dict(v_row=72), "rows of the cache"), (dict(k_row=1 << 23), "rows of the cache"),
    (dict(k_page=8), "strides of pages"), (dict(v_head=-16), "strides of pages"), (dict(k_head=1 << 41), "strides of pages"),
    (dict(table_row=6), "table_row"), (dict(table_row=-1), "table_row"),
    (dict(k=8 * A + 8), "16-byte"), (dict(v=9 * A + 4), "16-byte"), (dict(k_scale=A + 2), "aligned"), (dict(table=A + 1), "aligned"),
    (dict(k=0), "NULL device"), (dict(v=0), "NULL device"), (dict(table=0), "NULL device"), (dict(k_scale=0), "NULL device"), (dict(v_scale=0), "NULL device"),
]


@pytest.mark.parametrize("kw,says", CACHES)
def test_caches(kw, says):
    refuses(lambda: append(desc(), cache(**kw)), says)
    refuses(lambda: attend(desc(), cache(**kw)), says)
    if "NULL" not in says:
        refuses(lambda: capi.attention_paged_workspace_bytes(desc(), cache(**kw)), says)


def test_ranges():
    for call in (append, attend):
        for kw in (dict(n_pages=-1), dict(n_pages=1 << 31), dict(k_page=1 << 32), dict(page_len=65536, v_row=65536, table_row=1)):
            refuses(lambda: call(desc(), cache(**kw)), "n_pages|2\\^32 bytes", capi.ERR_RANGE)


def test_descriptions():
    for call in (append, attend):
        for kw, says in ((dict(head_dim=68), "head_dim"), (dict(n_heads=3), "key heads"), (dict(shared_len=4), "shared_len"), (dict(k_ptr=A, k_rows=100), "shared_len"),
                         (dict(q_ptr=A, q_rows=6, q_len=A), "lengths beside"), (dict(k_len=A + 2), "aligned"), (dict(q_row=60), "strides"), (dict(max_k=-1), "negative")):
            refuses(lambda: call(desc(**kw), cache()), says)
    refuses(lambda: append(desc(k_row=12), cache()), "strides")
    refuses(lambda: append(desc(v_seq=-8), cache()), "strides")
    for fn, args in ((capi.lib().sddmm_cache_append, (A, A, A, A, None)), (capi.lib().sddmm_attention_paged, (A, A, None, None, 0, None))):
        with pytest.raises(capi.SddmmError, match="NULL description"):
            capi.check(fn(None, cache(), *args))
        with pytest.raises(capi.SddmmError, match="NULL description of the cache"):
            capi.check(fn(desc(), None, *args))


def test_rotations():
    for kw, says in ((dict(rot_layout=2), "layout"), (dict(rot_dim=3), "rot_dim"), (dict(rot_dim=-2), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(rot_amplitude=float("inf")), "amplitude"),
                     (dict(rot_freq=0), "NULL device"), (dict(rot_freq=A + 4), "aligned")):
        refuses(lambda: append(desc(), cache(**kw)), says)


def test_pointers():
    for kw in (dict(k=0), dict(v=0), dict(q_out=0)):
        refuses(lambda: append(desc(), cache(), **kw), "NULL device")
    for kw in (dict(q=A + 8), dict(k=A + 2), dict(v=A + 4), dict(q_out=A + 8)):
        refuses(lambda: append(desc(), cache(), **kw), "16-byte")
    for kw in (dict(q=0), dict(out=0)):
        refuses(lambda: attend(desc(), cache(), **kw), "NULL device")
    for kw in (dict(q=A + 8), dict(out=A + 2)):
        refuses(lambda: attend(desc(), cache(), **kw), "16-byte")
    refuses(lambda: attend(desc(), cache(), lse=A + 2), "lse")


def test_results_in_each_others_place():
    for kw in (dict(k=8 * A), dict(v=9 * A), dict(q_out=8 * A), dict(q=9 * A), dict(q_out=3 * A), dict(q_out=4 * A)):
        refuses(lambda: append(desc(), cache(), **kw), "place")
    refuses(lambda: append(desc(), cache(v=8 * A)), "place")
    for kw in (dict(out=A), dict(out=8 * A), dict(out=9 * A), dict(lse=2 * A), dict(out=10 * A), dict(lse=11 * A)):
        refuses(lambda: attend(desc(), cache(), **kw), "place")
    refuses(lambda: append(desc(q_head=0), cache()), "queries overlap")
    refuses(lambda: attend(desc(o_head=0), cache()), "result overlap")
    for kw in (dict(k_page=64), dict(v_head=0), dict(k_row=128, k_head=64, k_page=1024)):
        refuses(lambda: append(desc(), cache(**kw)), "rows of the cache overlap")


def test_workspace():
    d, c = desc(n_seq=1, max_q=1, max_k=2000), cache(table_row=125)
    need = capi.attention_paged_workspace_bytes(d, c)
    assert need > 0
    for kw in (dict(ws=0), dict(n=need - 1), dict(ws=A + 16)):
        refuses(lambda: attend(d, c, **kw), "workspace")
    # the same with other lengths on the device, other pages and pointers
    assert capi.attention_paged_workspace_bytes(desc(n_seq=1, max_q=1, max_k=2000, k_len=A), cache(table_row=125, n_pages=9, k=5 * A)) == need
    assert capi.attention_paged_workspace_bytes(desc(n_seq=1, max_q=1, max_k=100), cache()) == 0 or need > 0


def test_nothing_to_do():
    for d in (desc(n_seq=0), desc(max_q=0, q_seq=0, o_seq=0, k_seq=0, v_seq=0)):
        append(d, cache(), 0, 0, 0, 0)
        attend(d, cache(), 0, 0, 0, 0, 0)


def test_more_than_a_launch_holds():
    for kw in (dict(n_seq=1 << 24, max_q=1, k_seq=128, v_seq=128), dict(n_seq=1 << 22, max_q=64, q_seq=1 << 14, o_seq=1 << 14, k_seq=1 << 13, v_seq=1 << 13)):
        refuses(lambda: append(desc(**kw), cache()), "one launch", capi.ERR_RANGE)
        refuses(lambda: attend(desc(**kw), cache()), "one launch", capi.ERR_RANGE)
