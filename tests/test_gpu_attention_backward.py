"""sddmm_attention_backward against the formulas in 64 bits, and against differences."""
import math

import pytest
import torch

import attention_reference as ref
from sddmm_gpu_amd import capi
from test_gpu_attention import BF16, DEV, F16, F32, SHAPES, TYPES, Case, normal

pytestmark = pytest.mark.gpu


def backward(c, seed=50, dslopes=True):
    """The forward and the backward pass of a Case; gradients in marked buffers."""
    c.run()
    dout = normal(seed, *c.q.shape, dtype=c.dtype)
    touched = torch.zeros(dout.shape[:-2], dtype=torch.bool)
    for rq, _ in c.where:
        touched[rq] = True
    dout[~touched] = math.nan
    c.dout = dout
    q, k, v, do = (x.to(DEV) for x in (c.q, c.k, c.v, dout))
    c.dq, c.dk, c.dv = (torch.full_like(x, c.MARK) for x in (q, k, v))
    c.ds = torch.full((c.heads,), c.MARK, device=DEV) if "slopes" in c.keep and dslopes else None
    n = capi.attention_workspace_bytes(c.desc)[1]
    ws = torch.full((n // 4 + 64,), math.nan, device=DEV)
    capi.attention_backward(c.desc, q.data_ptr(), k.data_ptr(), v.data_ptr(), c.out.data_ptr(), c.lse.data_ptr(), do.data_ptr(), c.dq.data_ptr(),
                            c.dk.data_ptr(), c.dv.data_ptr(), c.ds.data_ptr() if c.ds is not None else 0, ws.data_ptr(), n)
    torch.cuda.synchronize()
    return c


def pick(c, x, where, i):
    return x[where][:, i] if c.packed else x[where[0], where[1], i]


def check(c):
    group = c.heads // c.kv
    dq, dk, dv = (x.cpu() for x in (c.dq, c.dk, c.dv))
    slopes, slope_tol = torch.zeros(c.heads, dtype=torch.float64), torch.zeros(c.heads, dtype=torch.float64)
    seen_q, seen_k = torch.zeros(dq.shape[:-2], dtype=torch.bool), torch.zeros(dk.shape[:-2], dtype=torch.bool)
    for s in range(len(c.lens)):
        rq, rk = c.where[s]
        seen_q[rq], seen_k[rk] = True, True
        for kv in range(c.kv):
            total = {n: 0.0 for n in ("dk", "dv", "dk_tol", "dv_tol")}
            for h in range(kv * group, kv * group + group):
                q, k, v = c.operands(s, h)
                r = ref.head(q, k, v, c.left, c.right, c.prefix[s], c.scale, c.cap, float(c.slopes[h]), pick(c, c.dout, rq, h))
                for n in total:
                    total[n] = total[n] + r[n]
                slopes[h] += r["dslope"]
                slope_tol[h] += r["dslope_tol"]
                got = pick(c, dq, rq, h).double()
                bad = ~((got - r["dq"]).abs() <= r["dq_tol"])
                assert not bad.any(), ("dq", s, h, int(bad.sum()), bad.nonzero()[:4].tolist(), float((got - r["dq"]).abs().max()))
            for n, x in (("dk", dk), ("dv", dv)):
                got = pick(c, x, rk, kv).double()
                # (the sum over the heads is rounded once: u |sum| is at most the sum of the heads' u |.|, which the bounds hold)
                bad = ~((got - total[n]).abs() <= total[n + "_tol"])
                assert not bad.any(), (n, s, kv, int(bad.sum()), bad.nonzero()[:4].tolist(), float((got - total[n]).abs().max()))
    assert (dq[~seen_q] == c.MARK).all() and (dk[~seen_k] == c.MARK).all() and (dv[~seen_k] == c.MARK).all(), "rows behind the sequences were written"
    if c.ds is not None:
        assert ((c.ds.cpu().double() - slopes).abs() <= slope_tol).all(), (c.ds.cpu(), slopes, slope_tol)
    return c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("lens,heads,kv,dim,left,right", SHAPES)
def test_masks(dtype, packed, lens, heads, kv, dim, left, right):
    check(backward(Case(dtype, lens, heads, kv, dim, left, right, packed=packed)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap,bias", [(20.0, False), (0.0, True), (3.0, True)])
@pytest.mark.parametrize("lens,dim,left,right", [([(150, 150), (70, 200)], 64, -1, 0), ([(200, 333)], 128, 90, 40)])
def test_scores(dtype, cap, bias, lens, dim, left, right):
    for packed in (True, False):
        check(backward(Case(dtype, lens, 4, 2, dim, left, right, cap=cap, bias=bias, packed=packed)))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("packed", [True, False])
def test_prefix(dtype, packed):
    check(backward(Case(dtype, [(200, 200), (90, 90), (100, 160)], 2, 2, 64, -1, 0, prefix=[70, 0, 500], packed=packed)))


@pytest.mark.parametrize("dtype", TYPES)
def test_many_heads_fill_the_card(dtype):
    # enough workgroups that the rows of a key are not cut into pieces, and few that they are
    check(backward(Case(dtype, [(60, 60)] * 40, 16, 16, 64, -1, 0)))
    check(backward(Case(dtype, [(700, 700)], 8, 1, 128, -1, 0)))


def test_no_rows_and_no_keys():
    for lens in ([(0, 40), (0, 3)], [(33, 0), (2, 0)]):
        for packed in (True, False):
            c = check(backward(Case(BF16, lens, 2, 1, 64, -1, 0, packed=packed, bias=True)))
            assert (c.ds == 0).all()


def test_same_bits_on_every_call():
    c = backward(Case(BF16, [(300, 300), (200, 200)], 8, 2, 128, -1, 0, bias=True))
    first = [x.clone() for x in (c.dq, c.dk, c.dv, c.ds)]
    backward(c)
    for a, b in zip(first, (c.dq, c.dk, c.dv, c.ds)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("cap,bias,left", [(0.0, False, -1), (2.0, True, 40)])
def test_against_differences(cap, bias, left):
    """Gradients along a direction against the central difference of sum(out * dout), fp32.  The difference of step s is off by s^2 of
    the third derivative and by what fp32 leaves of two sums of about 10^4 terms, some 1e-4 / s: with s = 1e-2 both stay under 2e-2 of a
    sum whose terms' root is above 10."""
    base = Case(F32, [(150, 150)], 4, 2, 64, left, 0, cap=cap, bias=bias)
    backward(base)
    dout = base.dout[:150].double()
    for name, grad in (("q", base.dq), ("k", base.dk), ("v", base.dv)):
        x = getattr(base, name)
        step = torch.zeros_like(x)
        step[:150] = normal(9, *x[:150].shape, dtype=F32)
        sums = []
        for sign in (1, -1):
            setattr(base, name, x + sign * 1e-2 * step)
            sums.append(float((base.run().out[:150].cpu().double() * dout).sum()))
        setattr(base, name, x)
        want = (sums[0] - sums[1]) / 2e-2
        got = float((grad[:150].cpu().double() * step[:150].double()).sum())
        size = float((grad[:150].cpu().double() ** 2).sum().sqrt())
        assert abs(got - want) <= 2e-2 * size, (name, got, want, size)
    if bias:
        sums = []
        for sign in (1, -1):
            base.keep["slopes"].copy_(base.slopes * (1 + sign * 1e-2))
            sums.append(float((base.run().out[:150].cpu().double() * dout).sum()))
        want = (sums[0] - sums[1]) / 2e-2
        got = float((base.ds.cpu().double() * base.slopes.double()).sum())
        assert abs(got - want) <= 2e-2 * float((base.ds.cpu().double() ** 2).sum().sqrt() + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [24, 64, 104])
@pytest.mark.parametrize("packed", [True, False])
def test_keys_whose_rows_are_cut(dtype, dim, packed):
    # 16 heads' rows to each of some tiles of 128 keys, and of 32
    check(backward(Case(dtype, [(720, 720), (33, 33)], 16, 1, dim, -1, 0, packed=packed)))
    check(backward(Case(dtype, [(210, 210), (5, 5)], 16, 1, dim, -1, 0, packed=packed)))


@pytest.mark.parametrize("n", [3, 70])
def test_packed_rows_that_begin_later(n):
    for lens, heads in (([(5, 9)] * 3 + [(40, 40)] * n, 2), ([(300, 200)] + [(70, 90)] * n, 4)):
        c = Case(BF16, lens, heads, 1, 64, -1, 0)
        c.desc.q_ptr, c.desc.k_ptr, c.desc.n_seq = c.desc.q_ptr + 4, c.desc.k_ptr + 4, c.desc.n_seq - 1
        c.lens, c.where, c.prefix = c.lens[1:], c.where[1:], c.prefix[1:]
        backward(c)
        c.check()
        check(c)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [0, 66])
def test_pointers_out_of_order_touch_nothing_outside(dtype, n):
    c = Case(dtype, [(40, 40)] * (8 + n), 4, 2, 64, -1, 0)
    c.keep["q_ptr"].copy_(torch.tensor(c.keep["q_ptr"].tolist()[:-8] + [30, 10 ** 9, -5, 2 ** 31 - 1, 200, -2 ** 31, 100, 10 ** 6]))
    c.keep["k_ptr"].copy_(torch.tensor(c.keep["k_ptr"].tolist()[:-8] + [-2 ** 31, 2 ** 31 - 1, -7, 10 ** 9, 90, 50, 10 ** 6, 11]))
    backward(c)
    end = 40 * (8 + n)
    for x in (c.out, c.dq, c.dk, c.dv):
        assert (x[end:] == c.MARK).all()


def test_no_sequences_leave_no_gradient_of_slopes():
    c = Case(BF16, [(4, 4)], 4, 2, 64, bias=True)
    c.desc.n_seq = 0
    ds = torch.full((4,), 5.0, device=DEV)
    assert capi.attention_workspace_bytes(c.desc)[1] == 0
    capi.attention_backward(c.desc, 0, 0, 0, 0, 0, 0, 0, 0, 0, ds.data_ptr(), 0, 0)
    assert (ds == 0).all()
