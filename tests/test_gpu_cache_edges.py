"""sddmm_cache_append and sddmm_attention_paged at the ends of their ranges: more sequences than a grid's second and third dimension hold, positions near 2^30,
keys that are no numbers behind a row, blocks of 64 tokens in a graph, the rows' own precision."""
import math

import pytest
import torch

from sddmm_gpu_amd import capi
from tests import attention_reference as ref
from tests import cache_reference as cref
from tests.test_gpu_cache import BF16, CODE, DEV, F16, F32, Pages, attend, lost, normal, stream, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("held", ["i8", "own"])
@pytest.mark.parametrize("n_new", [1, 30])
def test_many_sequences(held, n_new):
    """70,000 sequences of one page each, of one or of 30 new tokens: brought in, then attended to; a sample of them against 64 bits."""
    n, page, heads, dim = 70000, 32, 4, 16
    pages = Pages(BF16, held, n, page, 16, 1, dim, False, 3, filled=False)
    g = torch.Generator().manual_seed(1)
    table = torch.randperm(n, generator=g).int().view(n, 1)
    t = table.to(DEV)
    q, k, v = (normal(4 + i, n * n_new, h, dim).to(BF16).to(DEV) for i, h in enumerate((heads, 1, 1)))
    ptr = (torch.arange(n + 1) * n_new).int().to(DEV)
    length = torch.full((n,), n_new, dtype=torch.int32, device=DEV)
    desc = capi.AttentionDesc.packed(capi.TYPE_BF16, n, heads, 1, dim, max_q=n_new, max_k=n_new, k_len=length.data_ptr(), q_ptr=ptr.data_ptr(), q_rows=n * n_new)
    cache = pages.desc(t)
    capi.cache_append(desc, cache, 0, 0, k.data_ptr(), v.data_ptr(), stream())
    out = torch.full_like(q, 7.0)
    size = capi.attention_paged_workspace_bytes(desc, cache)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=DEV)
    capi.attention_paged(desc, cache, q.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), size, stream())
    torch.cuda.synchronize()
    q, k, v, out = (x.view(n, n_new, -1, dim).cpu() for x in (q, k, v, out))
    read = {name: pages.read(name) for name in "kv"}
    for s in [0, 1, 65534, 65535, 65536, n - 1] + torch.randint(n, (20,), generator=g).tolist():
        rows = [table[s].tolist()]
        keys = {name: cref.gathered(read[name], 0, n_new, rows, page, 16, held) for name in "kv"}
        for name, x in (("k", k), ("v", v)):
            want = (torch.zeros(n, page, 1, dim, dtype=torch.float64)[:1], torch.zeros(1, 1, page // 16) if held == "i8" else None)
            cref.append(want, x[s].float(), [n_new], [n_new], [[0]], page, 16, held, BF16)
            assert torch.equal(keys[name], cref.gathered(want, 0, n_new, [[0]], page, 16, held))
        for h in range(heads):
            r = ref.head(q[s, :, h], keys["k"][:, 0], keys["v"][:, 0], -1, -1, 0, dim ** -0.5, 0.0, 0.0)  # (no bounds: the description's defaults)
            assert ((out[s, :, h].double() - r["out"]).abs() <= r["out_tol"] + lost(BF16, held, n_new, keys["v"])).all(), (s, h)


@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (F32, "e4m3"), (F16, "own")])
@pytest.mark.parametrize("n_new", [3, 200])
def test_far_positions(dtype, held, n_new):
    """The last tokens before position 2^30, of a table with 16,384 entries; a window of 100 keys."""
    page, block, heads, kv, dim, end, back = 65536, 16, 4, 2, 32, (1 << 30) - 5, 512
    pages = Pages(dtype, held, 3, page, block, kv, dim, False, 5)
    table = [[0] * 16382 + [1, 2]]
    t = torch.tensor(table, dtype=torch.int32, device=DEV)
    q, k, v = (normal(9 + i, n_new, h, dim).to(dtype) for i, h in enumerate((heads, kv, kv)))
    freq = torch.tensor([10000.0 ** (-2 * e / dim) for e in range(dim // 2)], dtype=torch.float64)
    pos = torch.arange(end - n_new, end)
    turned = {name: cref.turned(x, pos, freq, dim, cref.HALF, 1.0) for name, x in (("q", q), ("k", k))}
    cref.append(pages.cpu["k"], turned["k"].float(), [n_new], [end], table, page, block, held, dtype)
    cref.append(pages.cpu["v"], v.float(), [n_new], [end], table, page, block, held, dtype)
    dq, dk, dv, d_freq = (x.to(DEV) for x in (q, k, v, freq))
    length = torch.tensor([end], dtype=torch.int32, device=DEV)
    desc = capi.AttentionDesc.packed(CODE[dtype], 1, heads, kv, dim, max_q=n_new, max_k=(1 << 30) - 1, k_len=length.data_ptr(), window_left=100, window_right=0)
    cache = pages.desc(t, rot_dim=dim, rot_layout=cref.HALF, rot_freq=d_freq.data_ptr())
    turned_q, out = torch.full_like(dq, 7.0), torch.full_like(dq, 7.0)
    capi.cache_append(desc, cache, dq.data_ptr(), turned_q.data_ptr(), dk.data_ptr(), dv.data_ptr(), stream())
    size = capi.attention_paged_workspace_bytes(desc, cache)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device=DEV)
    capi.attention_paged(desc, cache, turned_q.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), size, stream())
    torch.cuda.synchronize()
    # (bounds of turned rows as in the other tests of them: cosine, sine, a product and the sum rounded to fp32, of at most the pair's size, then the type)
    coarse = 0.0 if dtype == F32 else 4 * 2.0 ** -24
    small = 2.0 ** -24 if dtype == F16 else 1e-37
    near = (ref.HALF[dtype] + 2.0 ** -23) * turned["q"].abs() + small + 1e-12 * q.double().abs().amax(-1, keepdim=True) + coarse * cref.pair_sizes(q, dim, cref.HALF, 1.0)
    assert ((turned_q.cpu().double() - turned["q"]).abs() <= near).all()
    keys = {}
    for name in "kv":
        (got, scale), (want, want_scale) = pages.read(name), pages.cpu[name]
        if held == "own":
            bound = 2 * (ref.HALF[dtype] + 2.0 ** -23) * want.abs() + small + (coarse * 1.01 * 8 if name == "k" else 0.0)  # (pairs are below 8)
            assert ((got - want).abs() <= bound).all()
        else:
            assert torch.equal(got, want) and torch.equal(scale, want_scale)
        at = torch.arange(end - back, end)
        p = torch.tensor(table[0])[at // page]
        x = got[p, at % page]
        keys[name] = x if held == "own" else x * scale[p][torch.arange(back), :, (at % page) // block][..., None].double()
    for h in range(heads):
        r = ref.head(turned_q[:, h].cpu(), keys["k"][:, h // 2], keys["v"][:, h // 2], 100, 0, 0, dim ** -0.5, 0.0, 0.0)
        assert ((out[:, h].cpu().double() - r["out"]).abs() <= r["out_tol"] + lost(dtype, held, back, keys["v"])).all()


@pytest.mark.parametrize("dtype,held", [(BF16, "own"), (F16, "own"), (F32, "own"), (BF16, "e4m3"), (F16, "e4m3"), (F32, "e4m3")])
@pytest.mark.parametrize("n_new,heads,kv,dim", [([12], 4, 2, 64), ([300, 150], 2, 2, 64), ([2100], 16, 16, 72), ([200, 1, 1, 2, 1, 1], 4, 2, 128)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_keys_that_are_no_numbers(dtype, held, n_new, heads, kv, dim, cap):
    """Causal: rows before the first such key give what they give without it; the rows that see it are not a number.  (Rows that raise their maximum together with such rows
    are held to the bounds of attention in 64 bits.)"""
    after = [n + 40 for n in n_new]
    spoiled = n_new[0] - 6 + 40  # the key of the sixth row from the end of the first sequence
    table, n_pages = tables(after, 32, 7)
    pages = Pages(dtype, held, n_pages, 32, 16, kv, dim, False, 8)
    q = normal(11, sum(n_new), heads, dim).to(dtype)
    p, i = table[0][spoiled // 32], spoiled % 32
    at = pages._view(pages.gpu["k"])[p, i]
    row = at.float().cpu()
    row[:, 3] = math.nan
    at.copy_(row.to(pages.store))
    out, stat = attend(dtype, pages, table, n_new, after, heads, q, True, cap=cap)
    good = n_new[0] - 6
    assert out[good: n_new[0]].isnan().all()
    assert not out[:good].isnan().any() and not stat[:good].isnan().any() and not out[n_new[0]:].isnan().any()
    k, v = (cref.gathered(pages.cpu[name], 0, good + 40, table, 32, 16, held) for name in "kv")
    for h in (0, heads - 1):
        r = ref.head(q[:good, h], k[:, h * kv // heads], v[:, h * kv // heads], -1, 0, 0, dim ** -0.5, cap, 0.0)
        assert ((out[:good, h].double() - r["out"]).abs() <= r["out_tol"] + lost(dtype, held, good + 40, v)).all()
        assert ((stat[:good, h].double() - r["lse"]).abs() <= r["lse_tol"]).all()


def test_long_blocks_in_a_graph():
    """fp32 rows of 128 elements in blocks of 64 tokens: the angles' table takes more LDS than a launch gets by itself, under a capture too."""
    dim, page, block, n = 128, 64, 64, 100
    freq = torch.tensor([10000.0 ** (-2 * e / dim) for e in range(dim // 2)], dtype=torch.float64, device=DEV)
    q, k, v = (normal(2 + i, n, h, dim).to(DEV) for i, h in enumerate((4, 2, 2)))
    t = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    length = torch.tensor([130], dtype=torch.int32, device=DEV)
    desc = capi.AttentionDesc.packed(capi.TYPE_F32, 1, 4, 2, dim, max_q=n, max_k=192, k_len=length.data_ptr())
    results = []
    for captured in (True, False):
        pages = Pages(F32, "i8", 4, page, block, 2, dim, False, 6)
        before = {name: (pages.gpu[name].clone(), pages.scales[name].clone()) for name in "kv"}
        cache = pages.desc(t, rot_dim=dim, rot_layout=cref.HALF, rot_freq=freq.data_ptr())
        out = torch.zeros_like(q)
        if captured:
            graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=side):
                capi.cache_append(desc, cache, q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr(), torch.cuda.current_stream().cuda_stream)
        for replay in range(3):
            for name in "kv":
                pages.gpu[name].copy_(before[name][0]), pages.scales[name].copy_(before[name][1])
            out.fill_(9.0)
            torch.cuda.synchronize()
            if captured:
                graph.replay()
            else:
                capi.cache_append(desc, cache, q.data_ptr(), out.data_ptr(), k.data_ptr(), v.data_ptr(), stream())
            torch.cuda.synchronize()
            results.append([x.cpu() for x in (out, pages.gpu["k"], pages.gpu["v"], pages.scales["k"], pages.scales["v"])])
    for r in results[:-1]:
        assert all(torch.equal(x, y) for x, y in zip(r, results[-1]))


def test_bf16_weights_keep_their_bits():
    """Few rows of bf16: weights are multiplied as two operands, so that results are off by their own rounding (half a step) and what fp32 makes of scores, sums and the
    weights' 16 bits (2^-16 each, half a step of the rest): no more than 2^-8 |out| + 2^-16 sum p |v|."""
    for held in ("own", "i8", "e4m3"):
        after, n_new = [700, 33, 5, 64], [1, 2, 1, 3]
        table, n_pages = tables(after, 32, 7)
        pages = Pages(BF16, held, n_pages, 32, 16, 2, 128, False, 8)
        q = normal(11, sum(n_new), 8, 128).to(BF16)
        out, _ = attend(BF16, pages, table, n_new, after, 8, q, True)
        at = 0
        for s, (n, m) in enumerate(zip(n_new, after)):
            k, v = (cref.gathered(pages.cpu[name], s, m, table, 32, 16, held) for name in "kv")
            for h in range(8):
                r = ref.head(q[at: at + n, h].float(), k[:, h // 4], v[:, h // 4], -1, 0, 0, 128 ** -0.5, 0.0, 0.0)  # (fp32: bounds without the type's rounding)
                pv = ref.head(q[at: at + n, h].float(), k[:, h // 4], v[:, h // 4].abs(), -1, 0, 0, 128 ** -0.5, 0.0, 0.0)["out"]
                bound = 2.0 ** -8 * (r["out"].abs() + r["out_tol"]) + 2.0 ** -16 * 1.02 * pv + r["out_tol"]
                assert ((out[at: at + n, h].double() - r["out"]).abs() <= bound).all(), (held, s, h)
            at += n


@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (BF16, "own"), (F32, "e4m3")])
@pytest.mark.parametrize("n_new", [[2, 1], [70, 40], [90, 1, 1, 1, 1, 1, 1]])
def test_places_beyond_32_bits(dtype, held, n_new):
    """Keys in pages 2^32 - 16 bytes apart, heads within them 2^31, and values in rows of nearly 2^23: the same bits as a compact cache gives."""
    page, block, kv, heads, dim = 16, 8, 2, 4, 64
    after = [n + 9 for n in n_new]
    table, n_pages = tables(after, page, 3)
    small = Pages(dtype, held, n_pages, page, block, kv, dim, False, 4)
    size = small.gpu["k"].element_size()
    strides = {"k": ((2 ** 32 - 16) // size, 2 ** 31 // size, 256 // size), "v": (2 ** 28 // size, (2 ** 27 + 2 ** 23 - 4096) // size, (2 ** 23 - 16) // size)}  # page, head, row
    t = torch.tensor(table, dtype=torch.int32, device=DEV)
    total, most = sum(n_new), max(n_new)
    length = torch.tensor(after, dtype=torch.int32, device=DEV)
    ptr = torch.tensor([0] + n_new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    q, k, v = (normal(6 + i, total, h, dim).to(dtype).to(DEV) for i, h in enumerate((heads, kv, kv)))
    desc = capi.AttentionDesc.packed(CODE[dtype], len(n_new), heads, kv, dim, max_q=most, max_k=max(after), k_len=length.data_ptr(), q_ptr=ptr.data_ptr(), q_rows=total, window_right=0)
    far, views, scales = {}, {}, {}
    for name in "kv":
        p, h, r = strides[name]
        far[name] = torch.empty((n_pages - 1) * p + (kv - 1) * h + page * r, dtype=small.store, device=DEV)
        views[name] = far[name].as_strided((n_pages, kv, page, dim), (p, h, r, 1))
        views[name].copy_(small.gpu[name])
        scales[name] = small.scales[name].clone() if held != "own" else None
    more = dict(k=far["k"].data_ptr(), v=far["v"].data_ptr())
    for name in "kv":
        more[name + "_page"], more[name + "_head"], more[name + "_row"] = strides[name]
        if held != "own":
            more[name + "_scale"] = scales[name].data_ptr()
    outs = []
    for cache in (small.desc(t), small.desc(t, **more)):
        capi.cache_append(desc, cache, 0, 0, k.data_ptr(), v.data_ptr(), stream())
        out = torch.full_like(q, 7.0)
        n = capi.attention_paged_workspace_bytes(desc, cache)
        ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=DEV)
        capi.attention_paged(desc, cache, q.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), n, stream())
        torch.cuda.synchronize()
        outs.append(out)
    assert torch.equal(*outs) and not outs[0].isnan().any()
    for name in "kv":
        assert torch.equal(views[name].contiguous().view(torch.uint8), small.gpu[name].view(torch.uint8))
        assert held == "own" or torch.equal(scales[name], small.scales[name])
    del far, views
    torch.cuda.empty_cache()
