"""sddmm_attention_* on batches that fill the card, for which rows and keys are dealt out in whole tiles: every element type, length of head and form
of the scores, some sequences and heads of each batch against attention in 64 bits."""
import pytest
import torch

import attention_reference as ref
from sddmm_gpu_amd import capi
from test_gpu_attention import BF16, DEV, F16, F32, Case
from test_gpu_attention_backward import backward, pick

pytestmark = pytest.mark.gpu

KINDS = [(t, dim, mod) for t, dims in ((F32, (24, 56, 104)), (BF16, (56, 104)), (F16, (56, 104))) for dim in dims for mod in (False, True)]
kinds = pytest.mark.parametrize("dtype,dim,mod", KINDS)


def lengths(n, rows, keys=None, seed=0):
    """(rows, keys) of n sequences: the longest first, then any below, one without rows and one without keys."""
    g = torch.Generator().manual_seed(seed)
    a = torch.randint(1, rows + 1, (n,), generator=g).tolist()
    b = [x if keys is None else max(x, y) for x, y in zip(a, torch.randint(1, (keys or 1) + 1, (n,), generator=g).tolist())]
    out = list(zip(a, b))
    out[0], out[1] = (rows, keys or rows), (rows, keys or rows)
    if n > 4:
        out[2], out[3] = (0, out[2][1]), (out[3][0], 0)
    return out


def check_some(c, seqs, kvs, grads=True):
    group = c.heads // c.kv
    for name, x in (("out", c.out),) + ((("dq", c.dq), ("dk", c.dk), ("dv", c.dv)) if grads else ()):
        touched = torch.zeros(x.shape[:-2], dtype=torch.bool, device=DEV)
        for rq, rk in c.where:
            touched[rk if name in ("dk", "dv") else rq] = True
        assert (x[~touched] == c.MARK).all(), name + ": rows behind the sequences were written"
        assert torch.isfinite(x).all(), name
    with torch.device(DEV):
        for s in seqs:
            rq, rk = c.where[s]
            for kv in kvs:
                total = {n: 0.0 for n in ("dk", "dv", "dk_tol", "dv_tol")}
                for h in range(kv * group, kv * group + group):
                    q, k, v = (x.to(DEV) for x in c.operands(s, h))
                    r = ref.head(q, k, v, c.left, c.right, c.prefix[s], c.scale, c.cap, float(c.slopes[h]), pick(c, c.dout, rq, h).to(DEV) if grads else None)
                    for name, x in (("out", c.out),) + ((("dq", c.dq),) if grads else ()):
                        bad = ~((pick(c, x, rq, h).double() - r[name]).abs() <= r[name + "_tol"])
                        assert not bad.any(), (name, s, h, int(bad.sum()), bad.nonzero()[:4].tolist())
                    for n in total if grads else ():
                        total[n] = total[n] + r[n]
                for name, x in (("dk", c.dk), ("dv", c.dv)) if grads else ():
                    bad = ~((pick(c, x, rk, kv).double() - total[name]).abs() <= total[name + "_tol"])
                    assert not bad.any(), (name, s, kv, int(bad.sum()), bad.nonzero()[:4].tolist())


def some(c, **kw):
    check_some(c, (0, 2, 3, len(c.lens) // 2, len(c.lens) - 1) if len(c.lens) > 4 else range(len(c.lens)), sorted({0, c.kv - 1}), **kw)


def scores(mod):
    return dict(cap=5.0, bias=True) if mod else {}


@kinds
@pytest.mark.parametrize("packed", [False, True])
def test_tiles_of_128_rows(dtype, dim, mod, packed):
    some(backward(Case(dtype, lengths(66, 170) if not packed else [(170, 170)] * 66, 8, 8, dim, -1, -1, packed=packed, **scores(mod))))


@kinds
@pytest.mark.parametrize("packed", [False, True])
def test_tiles_of_64_rows(dtype, dim, mod, packed):
    some(backward(Case(dtype, lengths(32, 150) if not packed else [(150, 140)] * 32, 8, 8, dim, -1, 0, packed=packed, **scores(mod))))


@kinds
@pytest.mark.parametrize("n", [140, 50])
def test_pairs_of_tokens_and_heads(dtype, dim, mod, n):
    c = Case(dtype, lengths(n, 20, 60), 32, 8, dim, 40, 0, packed=False, **scores(mod))
    some(c.run(), grads=False)


@kinds
@pytest.mark.parametrize("n", [9, 80])
def test_shared_keys(dtype, dim, mod, n):
    c = Case(dtype, lengths(n, 1, 40), 4, 1, dim, 310, 0, packed=False, shared=300, **scores(mod))
    some(c.run(), grads=False)


@kinds
@pytest.mark.parametrize("n,length", [(20, 128), (28, 128), (3, 50)])
def test_few_rows_and_keys(dtype, dim, mod, n, length):
    some(backward(Case(dtype, lengths(n, length, seed=1), 8, 8, dim, -1, 0, prefix=[30] * n, **scores(mod))))


@kinds
def test_many_rows_to_a_key(dtype, dim, mod):
    # whole tiles of keys for heads of any length, and tiles that are cut
    some(backward(Case(dtype, [(1100, 1100)] * 8, 16, 16, dim, -1, -1, packed=False, **scores(mod))))
    check_some(backward(Case(dtype, [(3000, 3000)], 16, 1, dim, -1, -1, **scores(mod))), (0,), (0,))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lens,heads,kv", [([(1, 300), (3, 40), (0, 90), (5, 5)], 8, 2), ([(150, 150), (70, 200), (1, 0)], 4, 4), ([(90, 120)] * 40, 16, 16)])
def test_one_side_packed(dtype, lens, heads, kv):
    """Packed rows against padded caches, and the other way round, forwards and backwards."""
    for q_packed in (True, False):
        a, b = Case(dtype, lens, heads, kv, 64, -1, 0), Case(dtype, lens, heads, kv, 64, -1, 0, packed=False)
        for s in range(len(lens)):  # the same rows in both
            for x, side in (("q", 0), ("k", 1), ("v", 1)):
                getattr(b, x)[b.where[s][side]] = getattr(a, x)[a.where[s][side]]
        rows, keys = (a, b) if q_packed else (b, a)
        d, drop = rows.desc, keys.desc
        mixed = type(d).from_buffer_copy(bytes(d))
        for f in ("k_ptr", "k_len", "k_rows", "k_seq", "v_seq"):
            setattr(mixed, f, getattr(drop, f))
        backward(a)
        q, k, v = rows.q.to(DEV), keys.k.to(DEV), keys.v.to(DEV)
        dout = torch.zeros_like(rows.q)
        for s in range(len(lens)):
            dout[rows.where[s][0]] = a.dout[a.where[s][0]]
        dout = dout.to(DEV)
        out, lse = torch.zeros_like(q), torch.zeros(q.shape[:-1], device=DEV)
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        need = max(capi.attention_workspace_bytes(mixed))
        ws = torch.empty(need + 256, dtype=torch.uint8, device=DEV)
        capi.attention_forward(mixed, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), ws.data_ptr(), need)
        capi.attention_backward(mixed, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(), dout.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                dv.data_ptr(), 0, ws.data_ptr(), need)
        torch.cuda.synchronize()
        mix = Mixed(a, rows, keys, out, dq, dk, dv)
        check_some(mix, range(len(lens)), range(kv) if len(lens) < 10 else (0, kv - 1))


class Mixed:
    """Results laid out as `rows` and `keys` are, read as those of the packed case `a`."""
    def __init__(self, a, rows, keys, out, dq, dk, dv):
        self.__dict__.update(a.__dict__)
        self.operands, self.MARK = a.operands, a.MARK
        for name, x, of, side in (("out", out, rows, 0), ("dq", dq, rows, 0), ("dk", dk, keys, 1), ("dv", dv, keys, 1)):
            like = a.q if side == 0 else a.k
            y = torch.full(like.shape, a.MARK, dtype=x.dtype, device=DEV)
            for s in range(len(a.lens)):
                y[a.where[s][side]] = x[of.where[s][side]]
            setattr(self, name, y)
