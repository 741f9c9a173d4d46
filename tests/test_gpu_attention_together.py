"""Rotary positions, attention, its gradients and the way back through the rotation, as a program runs them; the same against the sparse path of
the library; and recorded into a graph."""
import math

import numpy as np
import pytest
import torch

import attention_reference as ref
from sddmm_gpu_amd import capi
from test_gpu_attention import BF16, CODE, DEV, F32, normal
from test_gpu_rotary import turned

pytestmark = pytest.mark.gpu


class Layer:
    """Rotation of q and k, attention forward and backward over packed sequences, rotation back: every buffer and workspace made once."""

    def __init__(self, dtype, lens, heads, kv, dim, rot, layout, **more):
        self.lens, self.heads, self.kv, self.dim, self.rot, self.layout, self.dtype = lens, heads, kv, dim, rot, layout, dtype
        rows = sum(lens)
        self.x = {n: torch.empty(rows, h, dim, dtype=dtype, device=DEV) for n, h in (("q", heads), ("k", kv), ("v", kv), ("qr", heads), ("kr", kv), ("out", heads), ("dout", heads),
                                                                                     ("dqr", heads), ("dkr", kv), ("dv", kv), ("dq", heads), ("dk", kv))}
        self.lse = torch.empty(rows, heads, device=DEV)
        self.pos = torch.cat([torch.arange(n) for n in lens]).int().to(DEV)
        self.ptr = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=DEV)
        freq, _ = capi.rotary_frequencies(rot)
        self.freq = torch.from_numpy(freq).to(DEV)
        self.turn = [capi.RotaryDesc.packed(CODE[dtype], rows, heads, kv, dim, rot, layout, inverse=i) for i in (0, 1)]
        self.desc = capi.AttentionDesc.packed(CODE[dtype], len(lens), heads, kv, dim, max_q=max(lens), max_k=max(lens), q_rows=rows, k_rows=rows, q_ptr=self.ptr.data_ptr(),
                                              k_ptr=self.ptr.data_ptr(), window_right=0, **more)
        self.n = max(capi.attention_workspace_bytes(self.desc))
        self.ws = torch.empty(self.n + 256, dtype=torch.uint8, device=DEV)

    def fill(self, seed):
        for i, n in enumerate(("q", "k", "v", "dout")):
            self.x[n].copy_(normal(seed + i, *self.x[n].shape, dtype=self.dtype))

    def run(self):
        st = torch.cuda.current_stream().cuda_stream
        p = {n: t.data_ptr() for n, t in self.x.items()}
        pos, freq, lse, ws = self.pos.data_ptr(), self.freq.data_ptr(), self.lse.data_ptr(), self.ws.data_ptr()
        capi.rotary(self.turn[0], pos, freq, p["q"], p["qr"], p["k"], p["kr"], st)
        capi.attention_forward(self.desc, p["qr"], p["kr"], p["v"], p["out"], lse, ws, self.n, st)
        capi.attention_backward(self.desc, p["qr"], p["kr"], p["v"], p["out"], lse, p["dout"], p["dqr"], p["dkr"], p["dv"], 0, ws, self.n, st)
        capi.rotary(self.turn[1], pos, freq, p["dqr"], p["dq"], p["dkr"], p["dk"], st)

    def results(self):
        torch.cuda.synchronize()
        return {n: self.x[n].clone() for n in ("out", "dq", "dk", "dv")}


def reference(layer):
    """The same in 64 bits from the operands, by automatic differentiation."""
    q, k, v = (layer.x[n].cpu().double().requires_grad_() for n in ("q", "k", "v"))
    half = layer.rot // 2
    first = torch.arange(half) * (1 if layer.layout == capi.ROTARY_HALF else 2)
    second = first + (half if layer.layout == capi.ROTARY_HALF else 1)
    angle = layer.pos.cpu().double()[:, None, None] * layer.freq.cpu()

    def turn(x):
        a, b = x[..., first], x[..., second]
        y = x.clone()
        y[..., first], y[..., second] = a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()
        return y

    qr, kr, outs, begin = turn(q), turn(k), [], 0
    for n in layer.lens:
        at = slice(begin, begin + n)
        hidden = torch.ones(n, n, dtype=torch.bool).triu(1)
        group = layer.heads // layer.kv
        outs.append(torch.stack([torch.softmax((qr[at, h] @ kr[at, h // group].T * layer.dim ** -0.5).masked_fill(hidden, -math.inf), 1) @ v[at, h // group]
                                 for h in range(layer.heads)], 1))
        begin += n
    out = torch.cat(outs)
    (out * layer.x["dout"].cpu().double()).sum().backward()
    return dict(out=out.detach(), dq=q.grad, dk=k.grad, dv=v.grad)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("layout", [capi.ROTARY_HALF, capi.ROTARY_INTERLEAVED])
def test_layer(dtype, layout):
    """Relative to a result's norm.  fp32: sums of up to 300 terms of 2^-24 each and a handful of roundings, below 40 e.  bf16: the rotated
    operands are off by 2^-9 rms at most (a score by that times the root of its 64 terms, some 2^-9 of a score of size 1, and so a probability), then
    probabilities, gradients of scores, results and rotated gradients by as much each: six independent ones, 2.5 of 2^-9, doubled."""
    layer = Layer(dtype, [130, 1, 70, 200], 4, 2, 64, 48, layout)
    layer.fill(7)
    layer.run()
    got, want = layer.results(), reference(layer)
    bound = 40 * 2.0 ** -24 if dtype == F32 else 5 * 2.0 ** -9
    for n in want:
        off = float((got[n].cpu().double() - want[n]).norm() / want[n].norm())
        assert off <= bound, (n, off)


def test_graph():
    """Recorded once, replayed with new operands and the program's own work between: the bits of the calls themselves."""
    layer = Layer(BF16, [300, 77], 8, 2, 128, 128, capi.ROTARY_HALF)
    layer.fill(1)
    layer.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            layer.run()
    torch.cuda.synchronize()
    for seed in (20, 30, 40, 50):
        layer.fill(seed)
        layer.run()
        want = layer.results()
        for n in ("out", "dq", "dk", "dv", "qr", "kr", "dqr", "dkr"):
            layer.x[n].fill_(3.0)
        layer.ws.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        got = layer.results()
        for n in want:
            assert torch.equal(got[n], want[n]), (seed, n)


def test_decoding_graph():
    """A decoding step (rotation into the cache, attention over it, in pieces) recorded once; lengths and positions change between the replays."""
    n, heads, kv, dim, cap = 3, 8, 2, 64, 900
    q, k = (torch.empty(n, h, dim, dtype=BF16, device=DEV) for h in (heads, kv))
    cache_k, cache_v = normal(1, n, cap, kv, dim, dtype=BF16).to(DEV), normal(2, n, cap, kv, dim, dtype=BF16).to(DEV)
    qr, out = torch.empty_like(q), torch.empty_like(q)
    lens, pos = torch.empty(n, dtype=torch.int32, device=DEV), torch.empty(n, dtype=torch.int32, device=DEV)
    freq = torch.from_numpy(capi.rotary_frequencies(dim)[0]).to(DEV)
    new = torch.empty_like(k)
    turn = capi.RotaryDesc.packed(capi.TYPE_BF16, n, heads, kv, dim, dim, capi.ROTARY_HALF)
    d = capi.AttentionDesc.packed(capi.TYPE_BF16, n, heads, kv, dim, max_q=1, max_k=cap, window_right=0, k_len=lens.data_ptr())
    size = capi.attention_workspace_bytes(d)[0]
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)

    def step():
        st = torch.cuda.current_stream().cuda_stream
        capi.rotary(turn, pos.data_ptr(), freq.data_ptr(), q.data_ptr(), qr.data_ptr(), k.data_ptr(), new.data_ptr(), st)
        cache_k.view(-1, kv, dim).index_copy_(0, pos.long() + torch.arange(n, device=DEV) * cap, new)
        capi.attention_forward(d, qr.data_ptr(), cache_k.data_ptr(), cache_v.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), size, st)

    def fill(i):
        at = torch.tensor([5, 400, 800]) + 7 * i
        pos.copy_(at.int())
        lens.copy_(at.int() + 1)
        q.copy_(normal(10 + i, n, heads, dim, dtype=BF16))
        k.copy_(normal(20 + i, n, kv, dim, dtype=BF16))
        return at

    fill(0)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step()
    for i in range(1, 6):
        at = fill(i)
        out.fill_(9.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for s in range(n):
            want, tol = turned(q[s:s + 1].cpu(), at[s:s + 1], freq.cpu(), dim, capi.ROTARY_HALF)
            assert ((qr[s].cpu().double() - want[0]).abs() <= tol[0]).all()
            m = int(at[s]) + 1
            for h in range(heads):
                r = ref.head(qr[s, h:h + 1].cpu(), cache_k[s, :m, h // 4].cpu(), cache_v[s, :m, h // 4].cpu(), -1, 0, 0, dim ** -0.5, 0.0, 0.0)
                assert ((out[s, h:h + 1].cpu().double() - r["out"]).abs() <= r["out_tol"]).all(), (i, s, h)


def test_against_the_sparse_path():
    """A window as a CSR pattern through sddmm_execute_softmax and sddmm_plan_spmm, and as a mask: fp32, both within what 64 terms in a score and 121 in
    a row may differ by."""
    n, half, K = 700, 60, 64
    q, k, v = normal(1, n, K, dtype=F32), normal(2, n, K, dtype=F32), normal(3, n, K, dtype=F32)
    rows = np.repeat(np.arange(n), 2 * half + 1)
    cols = rows + np.tile(np.arange(-half, half + 1), n)
    keep = (cols >= 0) & (cols < n)
    rows, cols = rows[keep], cols[keep]
    row_ptr = torch.from_numpy(np.concatenate([[0], np.cumsum(np.bincount(rows, minlength=n))]).astype(np.int32)).to(DEV)
    col_ind = torch.from_numpy(cols.astype(np.int32)).to(DEV)
    qd, kd, vd = (q * K ** -0.5).to(DEV), k.to(DEV), v.to(DEV)
    plan = capi.Plan.from_device_csr(n, n, len(cols), row_ptr.data_ptr(), col_ind.data_ptr(), K, options=capi.PlanOptions.defaults(spmm_stream=1), keep=(row_ptr, col_ind))
    p, y = torch.empty(len(cols), device=DEV), torch.empty(n, K, device=DEV)
    plan.execute_softmax(0, qd.data_ptr(), kd.data_ptr(), p.data_ptr())
    plan.spmm(p.data_ptr(), vd.data_ptr(), y.data_ptr())
    out, lse = torch.empty(n, K, device=DEV), torch.empty(n, device=DEV)
    d = capi.AttentionDesc.packed(capi.TYPE_F32, 1, 1, 1, K, max_q=n, max_k=n, window_left=half, window_right=half)
    size = capi.attention_workspace_bytes(d)[0]
    ws = torch.empty(size + 256, dtype=torch.uint8, device=DEV)
    q2 = q.to(DEV)
    capi.attention_forward(d, q2.data_ptr(), kd.data_ptr(), vd.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), size)
    torch.cuda.synchronize()
    r = ref.head(q, k, v, half, half, 0, K ** -0.5, 0.0, 0.0)
    assert ((out.cpu().double() - r["out"]).abs() <= r["out_tol"]).all()
    assert ((out - y).abs().cpu().double() <= 2 * r["out_tol"] + 4e-7).all()
