"""sddmm_attention_forward and sddmm_attention_shared against attention in 64 bits."""
import math

import pytest
import torch

import attention_reference as ref
from sddmm_gpu_amd import capi

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODE = {F32: capi.TYPE_F32, BF16: capi.TYPE_BF16, F16: capi.TYPE_F16}


def normal(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


class Case:
    """A batch with results in buffers that are filled with a mark, so that what must not be written can be looked at."""
    MARK = 77.0

    def __init__(self, dtype, lens, heads=2, kv=1, dim=64, left=-1, right=-1, prefix=None, cap=0.0, bias=False, packed=True, shared=0, scale=None, seed=0,
                 slack=3):
        # lens: (rows, keys) of each sequence
        self.dtype, self.lens, self.heads, self.kv, self.dim = dtype, lens, heads, kv, dim
        self.left, self.right, self.cap, self.shared = left, right, cap, shared
        self.prefix = prefix or [0] * len(lens)
        self.scale = scale or dim ** -0.5
        self.slopes = (0.5 ** torch.arange(1, heads + 1).float()) if bias else torch.zeros(heads)
        n, mq, mk = len(lens), max(a for a, _ in lens), max(b for _, b in lens)
        self.packed, self.mq, self.mk = packed, mq, mk
        keep = self.keep = {}
        if packed:
            rq, rk = sum(a for a, _ in lens), sum(b for _, b in lens)
            self.q, self.k, self.v = normal(seed, rq + slack, heads, dim, dtype=dtype), normal(seed + 1, rk + slack, kv, dim, dtype=dtype), normal(seed + 2, rk + slack, kv, dim, dtype=dtype)
            ptr = [torch.tensor([0] + [x[i] for x in lens]).cumsum(0).int() for i in (0, 1)]
            self.where = [(slice(ptr[0][s], ptr[0][s + 1]), slice(ptr[1][s], ptr[1][s + 1])) for s in range(n)]
            # (behind the sequences: rows that nothing may read)
            for x, e in ((self.q, rq), (self.k, rk), (self.v, rk)):
                x[e:] = math.nan
            keep["q_ptr"], keep["k_ptr"] = ptr[0].to(DEV), ptr[1].to(DEV)
            more = dict(q_rows=rq, k_rows=rk)
        else:
            self.q, self.k, self.v = normal(seed, n, mq, heads, dim, dtype=dtype), normal(seed + 1, n, mk, kv, dim, dtype=dtype), normal(seed + 2, n, mk, kv, dim, dtype=dtype)
            self.where = [((s, slice(0, a)), (s, slice(0, b))) for s, (a, b) in enumerate(lens)]
            for s, (a, b) in enumerate(lens):
                self.q[s, a:] = math.nan
                self.k[s, b:] = math.nan
                self.v[s, b:] = math.nan
            keep["q_len"] = torch.tensor([a for a, _ in lens], dtype=torch.int32, device=DEV)
            keep["k_len"] = torch.tensor([b for _, b in lens], dtype=torch.int32, device=DEV)
            more = {}
        if prefix:
            keep["prefix"] = torch.tensor(prefix, dtype=torch.int32, device=DEV)
        if bias:
            keep["slopes"] = self.slopes.to(DEV)
        if shared:
            self.sk, self.sv = normal(seed + 3, shared, kv, dim, dtype=dtype), normal(seed + 4, shared, kv, dim, dtype=dtype)
            more["shared_len"] = shared
        self.desc = capi.AttentionDesc.packed(CODE[dtype], n, heads, kv, dim, max_q=mq, max_k=mk, window_left=left, window_right=right, cap=cap,
                                              scale=self.scale, **more, **{a: b.data_ptr() for a, b in keep.items()})

    def run(self, lse=True, stream=0):
        d = self.desc
        q, k, v = (x.to(DEV) for x in (self.q, self.k, self.v))
        self.out = torch.full_like(q, self.MARK)
        self.lse = torch.full(q.shape[:-1], self.MARK, dtype=F32, device=DEV)
        n = capi.attention_workspace_bytes(d)[0]
        ws = torch.full((n // 4 + 64,), math.nan, device=DEV)
        args = (ws.data_ptr() if n else 0, n, stream)
        if self.shared:
            sk, sv = self.sk.to(DEV), self.sv.to(DEV)
            capi.attention_shared(d, q.data_ptr(), sk.data_ptr(), sv.data_ptr(), k.data_ptr(), v.data_ptr(), self.out.data_ptr(), self.lse.data_ptr() if lse else 0, *args)
        else:
            capi.attention_forward(d, q.data_ptr(), k.data_ptr(), v.data_ptr(), self.out.data_ptr(), self.lse.data_ptr() if lse else 0, *args)
        torch.cuda.synchronize()
        return self

    def operands(self, s, h):
        rq, rk = self.where[s]
        c = h // (self.heads // self.kv)
        at = (lambda x, r, i: x[r][:, i]) if self.packed else (lambda x, r, i: x[r[0], r[1], i])
        k, v = at(self.k, rk, c), at(self.v, rk, c)
        if self.shared:
            k, v = torch.cat([self.sk[:, c], k]), torch.cat([self.sv[:, c], v])
        return at(self.q, rq, h), k, v

    def check(self, lse=True):
        out, ls = self.out.cpu(), self.lse.cpu()
        touched = torch.zeros(out.shape[:-1], dtype=torch.bool)
        for s in range(len(self.lens)):
            rq = self.where[s][0]
            if isinstance(rq, tuple):
                touched[rq[0], rq[1]] = True
            else:
                touched[rq] = True
            for h in range(self.heads):
                q, k, v = self.operands(s, h)
                r = ref.head(q, k, v, self.left, self.right, self.prefix[s], self.scale, self.cap, float(self.slopes[h]))
                got = (out[rq][:, h] if self.packed else out[rq[0], rq[1], h]).double()
                gl = (ls[rq][:, h] if self.packed else ls[rq[0], rq[1], h]).double()
                bad = ~((got - r["out"]).abs() <= r["out_tol"])
                assert not bad.any(), (s, h, int(bad.sum()), float((got - r["out"]).abs().max()), float(r["out_tol"].max()), bad.nonzero()[:4].tolist())
                if lse:
                    none = torch.isinf(r["lse"])
                    assert torch.equal(none, torch.isinf(gl) & (gl < 0))
                    bad = ~((gl - r["lse"]).abs() <= r["lse_tol"]) & ~none
                    assert not bad.any(), (s, h, int(bad.sum()), float((gl - r["lse"])[~none].abs().max()))
        assert (out[~touched] == self.MARK).all(), "rows behind the sequences were written"
        assert (ls[~touched] == self.MARK).all()
        return self


TYPES = [F32, BF16, F16]
# (rows, keys) of the sequences, heads, key heads, head_dim, left, right: one tile and less, borders of tiles of 32, 64, 128 and one
# beyond, rows without keys (more rows than keys under a causal mask), sequences without rows or without keys
SHAPES = [
    ([(1, 1)], 1, 1, 64, -1, 0),
    ([(64, 64), (65, 65), (1, 1), (127, 127)], 2, 1, 64, -1, 0),
    ([(200, 200)], 2, 2, 128, -1, 0),
    ([(129, 260), (31, 33), (0, 40), (5, 0), (40, 20)], 4, 2, 128, -1, 0),
    ([(300, 300)], 3, 1, 96, 20, 33),
    ([(257, 257), (130, 400)], 2, 1, 80, 100, 0),
    ([(150, 90)], 2, 1, 8, -1, -1),
    ([(260, 500)], 1, 1, 128, 0, 0),
    ([(140, 300)], 2, 1, 32, -1, 70),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("lens,heads,kv,dim,left,right", SHAPES)
def test_masks(dtype, packed, lens, heads, kv, dim, left, right):
    Case(dtype, lens, heads, kv, dim, left, right, packed=packed).run().check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (3.0, True)])
@pytest.mark.parametrize("lens,dim,left,right", [([(150, 150), (70, 200)], 64, -1, 0), ([(200, 333)], 128, 90, 40)])
def test_scores(dtype, cap, bias, lens, dim, left, right):
    Case(dtype, lens, 4, 2, dim, left, right, cap=cap, bias=bias).run().check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False])
def test_prefix(dtype, packed):
    Case(dtype, [(200, 200), (90, 90), (100, 160)], 2, 2, 64, -1, 0, prefix=[70, 0, 500], packed=packed).run().check()


# few rows: one tile of (token, head) pairs, caches of uneven lengths, empty ones among them, pieces of keys
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv,dim,left,cap,bias", [
    ([(1, 1)], 1, 1, 64, -1, 0.0, False),
    ([(1, 700), (1, 33), (1, 1), (1, 0), (1, 256)], 8, 2, 128, -1, 0.0, False),
    ([(1, 5000)], 4, 4, 64, -1, 0.0, False),
    ([(4, 900), (3, 2), (0, 50), (1, 400)], 16, 2, 128, -1, 30.0, True),
    ([(1, 3000), (1, 100)], 32, 1, 128, 200, 0.0, False),
    ([(7, 1300), (7, 64)], 4, 1, 80, 64, 0.0, True),
    ([(2, 1000)], 5, 1, 40, -1, 0.0, False),
])
def test_few_rows(dtype, lens, heads, kv, dim, left, cap, bias):
    for packed in (False, True):
        Case(dtype, lens, heads, kv, dim, left, 0, cap=cap, bias=bias, packed=packed).run().check()


# more pairs than one tile of them: pairs packed into tiles of 128
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,heads,kv,dim,left", [([(20, 600), (9, 9), (20, 0)], 8, 2, 64, -1), ([(40, 900), (1, 2)], 6, 2, 128, 300), ([(100, 130)], 12, 4, 128, -1)])
def test_packed_pairs(dtype, lens, heads, kv, dim, left):
    for cap, bias in ((0.0, False), (10.0, True)):
        Case(dtype, lens, heads, kv, dim, left, 0, cap=cap, bias=bias, packed=False).run().check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lens,shared,heads,kv,dim,left,cap,bias,prefix", [
    ([(1, 20), (1, 1), (1, 300)], 500, 8, 2, 64, -1, 0.0, False, None),
    ([(1, 5)], 1, 2, 1, 128, -1, 0.0, False, None),
    ([(1, 50)] * 40, 1100, 8, 1, 128, -1, 20.0, True, None),
    ([(3, 30), (2, 2), (0, 0), (1, 90)], 257, 6, 3, 80, -1, 0.0, True, None),
    ([(2, 40), (2, 700), (1, 1)], 300, 4, 2, 64, 100, 0.0, False, None),   # windows that end inside the shared keys, or behind them
    ([(30, 40), (12, 90)], 200, 4, 1, 64, -1, 0.0, False, [0, 260]),        # many rows; a prefix that reaches into the own keys
    ([(5, 0), (1, 0)], 90, 4, 1, 64, -1, 0.0, False, None),                 # nothing of their own: rows before the end of the shared keys
])
def test_shared(dtype, lens, shared, heads, kv, dim, left, cap, bias, prefix):
    Case(dtype, lens, heads, kv, dim, left, 0, cap=cap, bias=bias, prefix=prefix, packed=False, shared=shared).run().check()


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_of_any_size(dtype):
    """Scores that rise and fall by hundreds along the keys (the running maximum is raised again and again, and never), and a row that one key
    decides: probabilities of 2^-100 beside it."""
    for order in (1, -1):
        c = Case(dtype, [(140, 500)], 2, 1, 64, -1, 0, scale=1.0)
        c.k[:500] = (c.k[:500].float() * torch.linspace(0.1, 6, 500).flip(0 if order < 0 else ())[:, None, None]).to(dtype) if order < 0 else (
            c.k[:500].float() * torch.linspace(0.1, 6, 500)[:, None, None]).to(dtype)
        c.run().check()


@pytest.mark.parametrize("dtype", TYPES)
def test_infinities_and_nans(dtype):
    """Keys that a row does not see may hold anything; a NaN in a key that it sees makes its row NaN and no other."""
    c = Case(dtype, [(200, 200)], 1, 1, 64, -1, 0)
    c.k[150], c.k[160], c.k[199] = math.nan, math.inf, -math.inf
    c.run()
    good = Case(dtype, [(200, 200)], 1, 1, 64, -1, 0).run()
    assert torch.equal(c.out[:150], good.out[:150])
    assert torch.isnan(c.out[150:200]).all()
    # one token: what lies before its window or behind its cache is not read
    for left in (-1, 20):
        c = Case(dtype, [(1, 100)], 2, 1, 64, left, 0, packed=False)
        if left >= 0:
            c.k[0, :100 - 1 - left], c.v[0, :100 - 1 - left] = math.nan, math.inf
        c.run()
        assert torch.isfinite(c.out).all()


def test_broadcast_operands_and_orders():
    """Heads-first arrays, keys of one sequence for all (a stride of 0), one head of q for all."""
    n, mq, mk, heads, kv, dim = 3, 70, 90, 4, 2, 64
    q, k, v = normal(1, n, heads, mq, dim, dtype=BF16), normal(2, kv, mk, dim, dtype=BF16), normal(3, kv, mk, dim, dtype=BF16)
    qd, kd, vd = (x.to(DEV) for x in (q, k, v))
    for one_head in (False, True):
        out = torch.full((n, mq, heads, dim), 5.0, dtype=BF16, device=DEV)
        d = capi.AttentionDesc.packed(capi.TYPE_BF16, n, heads, kv, dim, max_q=mq, max_k=mk, window_right=0, q_seq=heads * mq * dim, q_head=0 if one_head else mq * dim,
                                      q_row=dim, k_seq=0, k_head=mk * dim, k_row=dim, v_seq=0, v_head=mk * dim, v_row=dim)
        ws = torch.empty(capi.attention_workspace_bytes(d)[0] + 256, dtype=torch.uint8, device=DEV)
        capi.attention_forward(d, qd.data_ptr(), kd.data_ptr(), vd.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
        for s in range(n):
            for h in range(heads):
                r = ref.head(q[s, 0 if one_head else h], k[h // 2], v[h // 2], -1, 0, 0, dim ** -0.5, 0.0, 0.0)
                assert ((out[s, :, h].cpu().double() - r["out"]).abs() <= r["out_tol"]).all()


def test_offsets_beyond_32_bits():
    """A cache whose second sequence begins behind 2^32 bytes and 2^31 elements, rows of it 4 MB apart."""
    heads, kv, dim, keys, row = 4, 2, 64, 600, 1 << 21
    k = torch.zeros(2 * keys * row, dtype=BF16, device=DEV)
    some = normal(4, 2, keys, kv, 2, dim, dtype=BF16)
    at = torch.arange(2 * keys, device=DEV).view(2, keys, 1, 1, 1) * row + torch.arange(kv, device=DEV).view(kv, 1, 1) * 2 * dim + torch.arange(2, device=DEV).view(2, 1) * dim + torch.arange(dim, device=DEV)
    k[at.view(-1)] = some.to(DEV).view(-1)
    for mq in (1, 150):
        q = normal(5, 2, mq, heads, dim, dtype=BF16)
        qd, out = q.to(DEV), torch.empty(2, mq, heads, dim, dtype=BF16, device=DEV)
        d = capi.AttentionDesc.packed(capi.TYPE_BF16, 2, heads, kv, dim, max_q=mq, max_k=keys, window_right=0, k_seq=keys * row, k_row=row, k_head=2 * dim, v_seq=keys * row,
                                      v_row=row, v_head=2 * dim)
        ws = torch.empty(capi.attention_workspace_bytes(d)[0] + 256, dtype=torch.uint8, device=DEV)
        capi.attention_forward(d, qd.data_ptr(), k.data_ptr(), k.data_ptr() + 2 * dim, out.data_ptr(), 0, ws.data_ptr(), ws.numel())
        torch.cuda.synchronize()
        for s in range(2):
            for h in range(heads):
                r = ref.head(q[s, :, h], some[s, :, h // 2, 0], some[s, :, h // 2, 1], -1, 0, 0, dim ** -0.5, 0.0, 0.0)
                assert ((out[s, :, h].cpu().double() - r["out"]).abs() <= r["out_tol"]).all()


def test_two_streams_at_once():
    """Calls that overlap in time, a workspace each: the bits of calls one after the other."""
    cases = [Case(BF16, [(1, 3000 + 100 * i), (1, 500)], 8, 2, 128, -1, 0, packed=False, seed=10 * i) for i in range(4)]
    want = [c.run().out.clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    held = []
    for c in cases:
        q, k, v = (x.to(DEV) for x in (c.q, c.k, c.v))
        n = capi.attention_workspace_bytes(c.desc)[0]
        held.append((q, k, v, torch.full_like(q, c.MARK), torch.empty(n, dtype=torch.uint8, device=DEV), n))
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, (q, k, v, out, ws, n) in zip(cases, streams, held):
            capi.attention_forward(c.desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0, ws.data_ptr(), n, s.cuda_stream)
    torch.cuda.synchronize()
    for w, h in zip(want, held):
        assert torch.equal(w, h[3])
