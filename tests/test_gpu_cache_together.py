"""sddmm_cache_append and sddmm_attention_paged as a serving program runs them: a prompt in pieces, then token by token, in and out of graphs, on
other streams, with caches that calls share; and against the calls for contiguous caches."""
import math

import pytest
import torch

from sddmm_gpu_amd import capi
from tests import attention_reference as ref
from tests import cache_reference as cref
from tests.test_gpu_cache import BF16, CODE, DEV, F16, F32, Pages, normal, stream, tables

pytestmark = pytest.mark.gpu


class Layer:
    """One layer's cache and calls; new tokens are packed, or max_q for each sequence where `padded`."""

    def __init__(self, dtype, held, n_seq, longest, heads, kv, dim, page, block, rot, max_new, padded=False, seed=0, rows=None):
        self.dtype, self.heads, self.kv, self.dim, self.n_seq = dtype, heads, kv, dim, n_seq
        self.table_rows, n_pages = tables([longest] * n_seq, page, seed)
        self.pages = Pages(dtype, held, n_pages, page, block, kv, dim, False, seed, filled=False)
        self.table = torch.tensor(self.table_rows, dtype=torch.int32, device=DEV)
        self.len = torch.zeros(n_seq, dtype=torch.int32, device=DEV)
        self.ptr = torch.zeros(n_seq + 1, dtype=torch.int32, device=DEV)
        freq, _ = capi.rotary_frequencies(rot)
        self.freq = torch.from_numpy(freq).to(DEV)
        self.cache = self.pages.desc(self.table, rot_dim=rot, rot_layout=capi.ROTARY_HALF, rot_freq=self.freq.data_ptr())
        self.rows = rows if rows is not None else n_seq * max_new
        more = dict(max_q=max_new, max_k=longest, k_len=self.len.data_ptr(), window_right=0)
        if padded:
            more.update(k_seq=max_new * kv * dim, v_seq=max_new * kv * dim)
        else:
            more.update(q_ptr=self.ptr.data_ptr(), q_rows=self.rows)
        self.desc = capi.AttentionDesc.packed(CODE[dtype], n_seq, heads, kv, dim, **more)
        self.q, self.out = (torch.zeros(self.rows, heads, dim, dtype=dtype, device=DEV) for _ in range(2))
        self.k, self.v = (torch.zeros(self.rows, kv, dim, dtype=dtype, device=DEV) for _ in range(2))
        n = capi.attention_paged_workspace_bytes(self.desc, self.cache)
        self.ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=DEV)

    def calls(self, s=None):
        s = stream() if s is None else s
        capi.cache_append(self.desc, self.cache, self.q.data_ptr(), self.q.data_ptr(), self.k.data_ptr(), self.v.data_ptr(), s)
        capi.attention_paged(self.desc, self.cache, self.q.data_ptr(), self.out.data_ptr(), 0, self.ws.data_ptr(), self.ws.numel(), s)


def inputs(seed, n, heads, kv, dim, dtype):
    return tuple(normal(seed + i, n, h, dim).to(dtype) for i, h in enumerate((heads, kv, kv)))


@pytest.mark.parametrize("dtype,held", [(BF16, "i8"), (F16, "e4m3"), (BF16, "own"), (F32, "i8")])
def test_pieces_then_tokens(dtype, held):
    """Two sequences: pieces of 37 and 20 tokens and more, then single tokens.  The cache that the calls leave is what the definition leaves, step by step, and every step's
    result the attention over it."""
    heads, kv, dim, page, block, rot = 4, 2, 64, 16, 16, 64
    steps = [(37, 20), (90, 1), (1, 33), (1, 1), (1, 1), (0, 1), (2, 3)]
    layer = Layer(dtype, held, 2, 160, heads, kv, dim, page, block, rot, 100, rows=130)
    after = [0, 0]
    freq = torch.from_numpy(capi.rotary_frequencies(rot)[0])
    for step, new in enumerate(steps):
        n = sum(new)
        q, k, v = inputs(100 * step, n, heads, kv, dim, dtype)
        after = [a + b for a, b in zip(after, new)]
        layer.q[:n], layer.k[:n], layer.v[:n] = q.to(DEV), k.to(DEV), v.to(DEV)
        layer.out.fill_(7.0)
        layer.len.copy_(torch.tensor(after, dtype=torch.int32))
        layer.ptr.copy_(torch.tensor([0, new[0], n], dtype=torch.int32))
        layer.calls()
        torch.cuda.synchronize()
        assert (layer.out[n:] == 7.0).all()
        pos = torch.cat([torch.arange(a - m, a) for m, a in zip(new, after)])
        if held != "own":
            for name, x in (("k", cref.turned(k, pos, freq, rot, 0, 1.0).float()), ("v", v.float())):
                cref.append(layer.pages.cpu[name], x, list(new), after, layer.table_rows, page, block, held, dtype)
                got, scale = layer.pages.read(name)
                assert torch.equal(scale, layer.pages.cpu[name][1]) and torch.equal(got, layer.pages.cpu[name][0])
        turned = layer.q[:n].cpu()
        at = 0
        for s in range(2):
            keys, values = (cref.gathered((layer.pages.read(name)[0], layer.pages.read(name)[1]), s, after[s], layer.table_rows, page, block, held) for name in "kv")
            for h in range(heads):
                r = ref.head(turned[at: at + new[s], h], keys[:, h // 2], values[:, h // 2], -1, 0, 0, dim ** -0.5, 0.0, 0.0)
                tol = r["out_tol"] + (after[s] * 2.0 ** -21 * values.abs().max() + 2.0 ** -25 if dtype == F16 else 2.0 ** -25 * values.abs().max())
                assert ((layer.out[at: at + new[s], h].cpu().double() - r["out"]).abs() <= tol).all(), (step, s, h)
            at += new[s]


def test_same_as_contiguous():
    """A cache of the operands' type against sddmm_rotary and sddmm_attention_forward over a contiguous one: the same keys to the last step but one, and results alike."""
    heads, kv, dim, n_seq, longest = 8, 2, 128, 5, 300
    layer = Layer(BF16, "own", n_seq, longest, heads, kv, dim, 64, 1, 128, longest, padded=True)
    lengths = torch.tensor([300, 1, 77, 256, 129], dtype=torch.int32)
    new = layer.n_seq * longest
    q, k, v = inputs(3, new, heads, kv, dim, BF16)
    layer.q.copy_(q), layer.k.copy_(k), layer.v.copy_(v)
    layer.desc.q_len = layer.len.data_ptr()
    layer.len.copy_(lengths)
    layer.calls()
    d = capi.RotaryDesc.packed(capi.TYPE_BF16, new, heads, kv, dim, 128, capi.ROTARY_HALF)
    pos = (torch.arange(new, dtype=torch.int32) % longest).to(DEV)
    dq, dk, dv = q.to(DEV), k.to(DEV), v.to(DEV)
    capi.rotary(d, pos.data_ptr(), layer.freq.data_ptr(), dq.data_ptr(), dq.data_ptr(), dk.data_ptr(), dk.data_ptr(), stream())
    a = capi.AttentionDesc.packed(capi.TYPE_BF16, n_seq, heads, kv, dim, max_q=longest, max_k=longest, q_len=layer.len.data_ptr(), k_len=layer.len.data_ptr(), window_right=0)
    out = torch.zeros_like(dq)
    ws = torch.empty(max(16, capi.attention_workspace_bytes(a)[0]), dtype=torch.uint8, device=DEV)
    capi.attention_forward(a, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), ws.numel(), stream())
    torch.cuda.synchronize()
    # both calls round cosines and sines to fp32 somewhere: keys and queries are the same or neighbours, 2^-7 of their size apart at most (two halves of a step of 2^-7)
    paged = layer.pages.read("k")[0]
    for s, n in enumerate(lengths.tolist()):
        got = cref.gathered((paged, None), s, n, layer.table_rows, 64, 1, "own")
        want = dk[s * longest: s * longest + n].cpu().double()
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 1e-6).all()
        # scores off by less than 2^-7 of sums of |q k| would allow far more than what differs here: neighbours are rare, results differ by roundings
        x, y = layer.out[s * longest: s * longest + n].double().cpu(), out[s * longest: s * longest + n].double().cpu()
        assert float((x - y).norm() / y.norm()) < 2.0 ** -7
        assert not layer.out[s * longest + n: (s + 1) * longest].any()


@pytest.mark.parametrize("held,max_new", [("i8", 1), ("e4m3", 4), ("own", 1)])
def test_graph_of_steps(held, max_new):
    """A captured decoding step, replayed with longer caches, other tokens and other pages, with eager work between; each replay against the same calls outside."""
    args = (BF16, held, 6, 700, 8, 2, 64, 16, 16, 64, max_new)
    captured, eager = (Layer(*args, padded=True, seed=4) for _ in range(2))
    lengths = torch.tensor([1, 640, 33, 0, 300, 15], dtype=torch.int32)
    for x in (captured, eager):
        x.calls()  # (code is loaded outside the capture)
    torch.cuda.synchronize()
    for name in "kv":
        for x in (captured, eager):
            x.pages.gpu[name].zero_()
            if held != "own":
                x.pages.scales[name].fill_(0.0)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        captured.calls(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    for step in range(6):
        lengths = lengths + torch.tensor([1, max_new, 2, step % 2, 3, 4], dtype=torch.int32)
        q, k, v = inputs(50 * step, 6 * max_new, 8, 2, 64, BF16)
        if step == 3:  # the sequences' pages change places
            for x in (captured, eager):
                x.table.copy_(x.table.flip(0))
        for x in (captured, eager):
            x.len.copy_(lengths)
            x.q.copy_(q), x.k.copy_(k), x.v.copy_(v)
            x.out.fill_(5.0)
        torch.cuda.synchronize()
        graph.replay()
        eager.calls()
        junk = torch.ones(1000, device=DEV).sum()
        torch.cuda.synchronize()
        assert float(junk) == 1000.0
        assert torch.equal(captured.out, eager.out) and torch.equal(captured.q, eager.q)
        for name in "kv":
            assert torch.equal(captured.pages.gpu[name].view(torch.uint8), eager.pages.gpu[name].view(torch.uint8))
            if held != "own":
                assert torch.equal(captured.pages.scales[name], eager.pages.scales[name])
        assert not captured.out.isnan().any()


def test_streams():
    """Calls of two layers under way together on two streams, each with a workspace of its own, against the same one after the other."""
    args = (BF16, "i8", 40, 2000, 8, 2, 128, 64, 16, 128, 1)
    layers = [Layer(*args, padded=True, seed=s) for s in (1, 2)]
    again = [Layer(*args, padded=True, seed=s) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    lengths = torch.randint(1, 2001, (40,), generator=torch.Generator().manual_seed(5)).to(torch.int32)
    for group in (layers, again):
        for s, x in enumerate(group):
            q, k, v = inputs(9 + s, 40, 8, 2, 128, BF16)
            x.len.copy_(lengths), x.q.copy_(q), x.k.copy_(k), x.v.copy_(v)
    torch.cuda.synchronize()
    for step in range(5):
        for x, st in zip(layers, streams):
            x.calls(st.cuda_stream)
        for x in again:
            x.calls()
        torch.cuda.synchronize()
        for x, y in zip(layers, again):
            assert torch.equal(x.out, y.out) and torch.equal(x.q, y.q) and torch.equal(x.pages.gpu["k"], y.pages.gpu["k"])


def test_shared_pages():
    """Sequences whose first pages are the same pages: as if each had a copy."""
    heads, kv, dim, page = 4, 2, 64, 32
    x = Layer(BF16, "e4m3", 3, 200, heads, kv, dim, page, 8, 64, 2, padded=True, seed=7)
    y = Layer(BF16, "e4m3", 3, 200, heads, kv, dim, page, 8, 64, 2, padded=True, seed=7)
    for name in "kv":
        codes = (normal(3, *y.pages.gpu[name].shape) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)
        scale = torch.rand(y.pages.scales[name].shape, generator=torch.Generator().manual_seed(4)) * 0.01
        for z in (x, y):
            z.pages.gpu[name].copy_(codes.to(DEV))
            z.pages.scales[name].copy_(scale)
        for s in (1, 2):  # y: copies of the first three pages of sequence 0
            for i in range(3):
                y.pages.gpu[name][y.table_rows[s][i]] = y.pages.gpu[name][y.table_rows[0][i]]
                y.pages.scales[name][y.table_rows[s][i]] = y.pages.scales[name][y.table_rows[0][i]]
    x.table[1:, :3] = x.table[0, :3]
    q, k, v = inputs(11, 6, heads, kv, dim, BF16)
    for z in (x, y):
        z.len.copy_(torch.tensor([150, 98, 200], dtype=torch.int32))
        z.q.copy_(q), z.k.copy_(k), z.v.copy_(v)
        z.calls()
    torch.cuda.synchronize()
    assert torch.equal(x.out, y.out)


def test_wrong_tables_stay_inside():
    """Page numbers outside the cache, lengths beyond max_k and below 0, pointers that do not rise: whatever comes out, the bytes around the arrays stay as they were."""
    heads, kv, dim, page, n_pages = 4, 2, 64, 16, 9
    guard = 1 << 16
    size = n_pages * page * kv * dim
    for held, block in (("i8", 16), ("own", 1)):
        e = 1 if held == "i8" else 2
        bufs = {n: torch.full((guard + size * e + guard,), 17, dtype=torch.uint8, device=DEV) for n in ("k", "v")}
        scales = {n: torch.full((64 + n_pages * kv * page // block + 64,), 0.5, device=DEV) for n in ("k", "v")}
        for table in ([[-5, 100, 1 << 30, 3], [-(1 << 31), 8, 9, 2]],):
            for lengths in ([1 << 30, -7], [64, 63], [3, 1 << 20]):
                for ptr in ([0, 5, 9], [9, 4, 0], [0, 1 << 30, 9], [-3, 2, 9]):
                    t = torch.tensor(table, dtype=torch.int32, device=DEV)
                    length, p = torch.tensor(lengths, dtype=torch.int32, device=DEV), torch.tensor(ptr, dtype=torch.int32, device=DEV)
                    q, k, v = (x.to(DEV) for x in inputs(1, 9, heads, kv, dim, BF16))
                    out = torch.full((guard // 128 + 9 + guard // 128, heads, dim), 3.0, dtype=BF16, device=DEV)
                    mid = out[guard // 128: guard // 128 + 9]
                    freq = torch.ones(32, dtype=torch.float64, device=DEV)
                    d = capi.AttentionDesc.packed(capi.TYPE_BF16, 2, heads, kv, dim, max_q=9, max_k=64, q_ptr=p.data_ptr(), q_rows=9, k_len=length.data_ptr(), window_right=0)
                    c = capi.CacheDesc.packed(capi.TYPE_I8 if held == "i8" else capi.TYPE_BF16, n_pages, page, kv, dim, block_len=block, table=t.data_ptr(), table_row=4, k=bufs["k"].data_ptr() + guard,
                                              v=bufs["v"].data_ptr() + guard, rot_dim=64, rot_freq=freq.data_ptr(),
                                              **(dict(k_scale=scales["k"].data_ptr() + 256, v_scale=scales["v"].data_ptr() + 256) if held == "i8" else {}))
                    capi.cache_append(d, c, q.data_ptr(), mid.data_ptr(), k.data_ptr(), v.data_ptr(), stream())
                    n = capi.attention_paged_workspace_bytes(d, c)
                    ws = torch.empty(max(n, 16), dtype=torch.uint8, device=DEV)
                    capi.attention_paged(d, c, q.data_ptr(), mid.data_ptr(), 0, ws.data_ptr(), n, stream())
                    torch.cuda.synchronize()
                    for name in "kv":
                        assert (bufs[name][:guard] == 17).all() and (bufs[name][-guard:] == 17).all()
                        assert (scales[name][:64] == 0.5).all() and (scales[name][-64:] == 0.5).all()
                    assert (out[: guard // 128] == 3.0).all() and (out[guard // 128 + 9:] == 3.0).all()
