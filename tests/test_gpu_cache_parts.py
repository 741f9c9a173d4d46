"""sddmm_attention_paged over mixed batches whose long rows, short rows, both or none have parts: results against 64 bits, and nothing behind the workspace is touched."""
import pytest
import torch

from sddmm_gpu_amd import capi
from tests import attention_reference as ref
from tests import cache_reference as cref
from tests.test_gpu_cache import BF16, CODE, DEV, F16, Pages, lost, normal, stream, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (F16, "e4m3"), (BF16, "own")])
@pytest.mark.parametrize("heads,kv", [(8, 2), (20, 1), (8, 8)])
@pytest.mark.parametrize("n_new,after,max_k", [
    ([90, 1, 1, 0, 1, 1, 1, 2], [130, 70, 1, 33, 300, 64, 17, 5], 300),           # short caches
    ([90, 1, 1, 0, 1, 1, 1, 2], [130, 70, 1, 33, 300, 64, 17, 5], 100000),        # the same under a long bound
    ([200, 1, 3, 1, 70], [3000, 5000, 3, 4999, 70], 5000),                        # long caches: parts of both
    ([1, 1, 1, 1, 1, 1, 900, 1, 1, 1], [900] * 10, 1000),
    ([0, 0, 0, 90, 0, 0, 1], [0, 9, 700, 90, 1, 0, 2000], 2000),
])
def test_parts_of_both(dtype, held, heads, kv, n_new, after, max_k):
    page, block, dim, guard = 32, 8, 64, 4096
    table, n_pages = tables(after, page, 3)
    pages = Pages(dtype, held, n_pages, page, block, kv, dim, False, 5)
    q = normal(8, sum(n_new), heads, dim).to(dtype)
    width = -(-max_k // page)
    t = torch.tensor([row + [-1] * (width - len(row)) for row in table], dtype=torch.int32, device=DEV)
    length = torch.tensor(after, dtype=torch.int32, device=DEV)
    ptr = torch.tensor([0] + n_new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
    rows = sum(n_new) + 5  # (rows behind the last sequence stay as they are)
    dq = torch.cat([q, torch.full((5, heads, dim), 3.0, dtype=dtype)]).to(DEV)
    desc = capi.AttentionDesc.packed(CODE[dtype], len(n_new), heads, kv, dim, max_q=max(n_new), max_k=max_k, k_len=length.data_ptr(), q_ptr=ptr.data_ptr(), q_rows=rows, window_right=0)
    cache = pages.desc(t)
    size = capi.attention_paged_workspace_bytes(desc, cache)
    ws = torch.full((size + guard,), 255, dtype=torch.uint8, device=DEV)
    for again in range(2):  # (the second call finds the first one's parts)
        out, lse = torch.full_like(dq, 7.0), torch.full((rows, heads), 7.0, device=DEV)
        capi.attention_paged(desc, cache, dq.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), size, stream())
        torch.cuda.synchronize()
        assert (ws[size:] == 255).all() and (out[-5:] == 7.0).all() and (lse[-5:] == 7.0).all()
        got, stat = out.cpu(), lse.cpu()
        at = 0
        for s, (n, m) in enumerate(zip(n_new, after)):
            k, v = (cref.gathered(pages.cpu[name], s, m, table, page, block, held) for name in "kv")
            for h in range(heads) if n < 100 else (0, heads - 1):
                c = h // (heads // kv)
                r = ref.head(q[at: at + n, h], k[:, c], v[:, c], -1, 0, 0, dim ** -0.5, 0.0, 0.0)
                assert ((got[at: at + n, h].double() - r["out"]).abs() <= r["out_tol"] + lost(dtype, held, m, v[:, c])).all(), (s, h)
                x, y = stat[at: at + n, h].double(), r["lse"]
                assert ((x == y) | ((x - y).abs() <= r["lse_tol"])).all(), (s, h)
            at += n


def test_mixed_batches_in_a_graph():
    """A captured append and attention over a packed batch, replayed with other sequences long, others without rows and other lengths, with eager work between."""
    n_seq, heads, kv, dim, page, block, most, rows = 9, 8, 2, 64, 32, 8, 120, 160
    longest = 3000
    width = -(-longest // page)
    table = torch.arange(n_seq * width, dtype=torch.int32).view(n_seq, width).flip(1).contiguous().to(DEV)
    freq = torch.from_numpy(capi.rotary_frequencies(dim)[0]).to(DEV)
    sides = []
    for _ in range(2):
        pages = Pages(BF16, "e4m3", n_seq * width, page, block, kv, dim, False, 5)
        s = dict(pages=pages, ptr=torch.zeros(n_seq + 1, dtype=torch.int32, device=DEV), len=torch.zeros(n_seq, dtype=torch.int32, device=DEV))
        s.update({n: torch.zeros(rows, h, dim, dtype=BF16, device=DEV) for n, h in (("q", heads), ("k", kv), ("v", kv), ("out", heads))})
        s["desc"] = capi.AttentionDesc.packed(capi.TYPE_BF16, n_seq, heads, kv, dim, max_q=most, max_k=longest, k_len=s["len"].data_ptr(), q_ptr=s["ptr"].data_ptr(), q_rows=rows, window_right=0)
        s["cache"] = pages.desc(table, rot_dim=dim, rot_layout=0, rot_freq=freq.data_ptr())
        s["size"] = capi.attention_paged_workspace_bytes(s["desc"], s["cache"])
        s["ws"] = torch.full((s["size"],), 255, dtype=torch.uint8, device=DEV)
        sides.append(s)

    def calls(s, st):
        capi.cache_append(s["desc"], s["cache"], s["q"].data_ptr(), s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), st)
        capi.attention_paged(s["desc"], s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), 0, s["ws"].data_ptr(), s["size"], st)

    assert sides[0]["size"] > 0
    for s in sides:
        calls(s, stream())  # (code is loaded outside the capture; no rows)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        calls(sides[0], torch.cuda.current_stream().cuda_stream)
    for step, (new, after) in enumerate([([100, 1, 1, 0, 1, 1, 3, 1, 1], [100, 2000, 30, 0, 1, 2999, 90, 64, 700]), ([1, 1, 1, 120, 0, 1, 1, 30, 1], [101, 2001, 31, 1200, 1, 3000, 91, 94, 701]),
                                         ([1] * 9, [102, 2002, 32, 1201, 2, 2500, 92, 95, 702]), ([0, 0, 0, 0, 0, 0, 0, 0, 120], [102, 2002, 32, 1201, 2, 2500, 92, 95, 822])]):
        q, k, v = (normal(30 * step + i, rows, h, dim).to(BF16) for i, h in enumerate((heads, kv, kv)))
        for s in sides:
            s["ptr"].copy_(torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32)), s["len"].copy_(torch.tensor(after, dtype=torch.int32))
            s["q"].copy_(q), s["k"].copy_(k), s["v"].copy_(v), s["out"].fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        calls(sides[1], stream())
        junk = torch.ones(1000, device=DEV).sum()
        torch.cuda.synchronize()
        assert float(junk) == 1000.0
        x, y = sides
        assert torch.equal(x["out"], y["out"]) and torch.equal(x["q"], y["q"]) and not x["out"].isnan().any() and (x["out"][sum(new):] == 5.0).all()
        for name in "kv":
            assert torch.equal(x["pages"].gpu[name].view(torch.uint8), y["pages"].gpu[name].view(torch.uint8)) and torch.equal(x["pages"].scales[name], y["pages"].scales[name])
