"""sddmm_rotary and sddmm_rotary_frequencies against complex rotations in 64 bits; refusals and frequencies need no GPU."""
import math

import numpy as np
import pytest
import torch

from sddmm_gpu_amd import capi

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODE = {F32: capi.TYPE_F32, BF16: capi.TYPE_BF16, F16: capi.TYPE_F16}
HALF_STEP = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
HALF, INTERLEAVED = capi.ROTARY_HALF, capi.ROTARY_INTERLEAVED
A = 1 << 20


def turned(x, pos, freq, rot, layout, inverse=False, amplitude=1.0):
    """(x turned, bound of the error): cosine and sine are off by 6 e (e = 2^-24: their series, the angle and its reduction, the
    amplitude), each product and the sum by e more, and the result is rounded to its type."""
    e, half = 2.0 ** -24, rot // 2
    y = x.double().clone()
    first = torch.arange(half) * (1 if layout == HALF else 2)
    second = first + (half if layout == HALF else 1)
    angle = pos.double()[:, None, None] * freq * (-1 if inverse else 1)
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, amplitude), angle)
    size = abs(amplitude) * (y[..., first].abs() + y[..., second].abs())
    tol = torch.zeros_like(y)
    y[..., first], y[..., second] = z.real, z.imag
    tol[..., first] = tol[..., second] = 9 * e * size
    tol[..., :rot] += HALF_STEP[x.dtype] * y[..., :rot].abs() + (2.0 ** -25 if x.dtype == F16 else 1e-38)
    return y, tol


def normal(seed, *shape, dtype):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def run(desc, pos, freq, q, k, q_out, k_out, stream=0):
    freq = torch.as_tensor(freq, dtype=torch.float64).to(DEV)
    p = pos.to(torch.int32).to(DEV) if pos is not None else None
    capi.rotary(desc, p.data_ptr() if p is not None else 0, freq.data_ptr(), q.data_ptr(), q_out.data_ptr(), k.data_ptr() if k is not None else 0,
                k_out.data_ptr() if k_out is not None else 0, stream)
    torch.cuda.synchronize()


# head sizes whose pieces are 16, 8, 4 and 2 bytes wide, parts of heads, one row and many, no keys, more pairs than the table holds
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", [HALF, INTERLEAVED])
@pytest.mark.parametrize("rows,heads,kv,dim,rot", [(1, 1, 0, 2, 2), (1, 32, 8, 128, 128), (37, 4, 2, 64, 32), (5000, 3, 1, 128, 96), (70, 2, 1, 80, 40),
                                                   (9, 2, 2, 50, 50), (33, 3, 1, 41, 26), (4, 2, 1, 12, 4), (3, 1, 1, 4096, 4096), (2, 2, 0, 2100, 2090), (6001, 2, 1, 72, 56), (6001, 1, 0, 40, 32), (3333, 1, 1, 16, 8), (2500, 5, 3, 24, 24)])
def test_rotary(dtype, layout, rows, heads, kv, dim, rot):
    g = torch.Generator().manual_seed(rows)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g)
    pos[0] = 0
    pos[-1] = (1 << 31) - 1 if rows > 4 else 7
    freq, _ = capi.rotary_frequencies(rot)
    f = torch.from_numpy(freq)
    q, k = normal(1, rows, heads, dim, dtype=dtype), normal(2, rows, max(kv, 1), dim, dtype=dtype)
    for inverse, amplitude in ((0, 1.0), (1, 1.25)):
        d = capi.RotaryDesc.packed(CODE[dtype], rows, heads, kv, dim, rot, layout, inverse=inverse, amplitude=amplitude)
        qd, kd = q.to(DEV), k.to(DEV)
        qo, ko = torch.full_like(qd, math.nan), torch.full_like(kd, 5.0)
        run(d, pos, freq, qd, kd, qo, ko)
        # (position 2^31 - 1 in 64 bits: 2^31 radians are known to 2^-22, so the bound of that row is not held to 32 bits' last place)
        far = pos.double()[:, None, None] * 2.0 ** -52
        for x, got in ((q, qo),) + (((k, ko),) if kv else ()):
            want, tol = turned(x, pos, f, rot, layout, inverse, amplitude)
            tol = tol + (x.double().abs().amax() * 4 * far)
            assert ((got.cpu().double() - want).abs() <= tol).all(), float((got.cpu().double() - want).abs().max())
            assert torch.equal(got.cpu()[..., rot:], x[..., rot:])
        if not kv:
            assert (ko == 5.0).all()
        # in place: the same bits
        run(d, pos, freq, qd, kd, qd, kd)
        assert torch.equal(qd, qo) and (not kv or torch.equal(kd, ko))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_a_cache(dtype):
    """q out of a joint projection [row, q heads + 2 kv heads, dim], results in heads-first order and in the rows of a cache."""
    rows, heads, kv, dim, rot = 50, 4, 2, 64, 64
    joint = normal(3, rows, heads + 2 * kv, dim, dtype=dtype).to(DEV)
    qo = torch.full((heads, rows, dim), 9.0, dtype=dtype, device=DEV)
    cache = torch.full((rows, 7, kv, dim), 9.0, dtype=dtype, device=DEV)  # row r: place 5 of sequence r
    d = capi.RotaryDesc.defaults(type=CODE[dtype], n_rows=rows, n_heads=heads, n_kv_heads=kv, head_dim=dim, rot_dim=rot, layout=HALF, first_position=1000,
                                 q_row=(heads + 2 * kv) * dim, q_head=dim, k_row=(heads + 2 * kv) * dim, k_head=dim,
                                 q_out_row=dim, q_out_head=rows * dim, k_out_row=7 * kv * dim, k_out_head=dim)
    freq, _ = capi.rotary_frequencies(rot)
    run(d, None, freq, joint, joint[:, heads:], qo, cache[:, 5])
    pos = torch.arange(rows) + 1000
    for x, got in ((joint[:, :heads].cpu(), qo.permute(1, 0, 2).cpu()), (joint[:, heads:heads + kv].cpu(), cache[:, 5].cpu())):
        want, tol = turned(x, pos, torch.from_numpy(freq), rot, HALF)
        assert ((got.double() - want).abs() <= tol).all()
    assert (cache[:, :5] == 9).all() and (cache[:, 6:] == 9).all()


@pytest.mark.gpu
def test_gradient():
    """inverse gives the gradient: <rotary(x), g> = <x, rotary'(g)>, fp32; both sums have 64 * 3 * 32 terms of size 1."""
    rows, heads, dim, rot = 64, 3, 32, 24
    x, g = normal(5, rows, heads, dim, dtype=F32).to(DEV), normal(6, rows, heads, dim, dtype=F32).to(DEV)
    freq, amplitude = capi.rotary_frequencies(rot, 10000.0, capi.ROTARY_PARTS, 4.0, 8192, 1.0, 32.0)
    y, b = torch.empty_like(x), torch.empty_like(x)
    for inverse, src, dst in ((0, x, y), (1, g, b)):
        d = capi.RotaryDesc.packed(capi.TYPE_F32, rows, heads, 0, dim, rot, INTERLEAVED, inverse=inverse, amplitude=amplitude)
        run(d, torch.arange(rows) * 100, freq, src, None, dst, None)
    left, right = float((y.double() * g.double()).sum()), float((x.double() * b.double()).sum())
    assert abs(left - right) <= 9 * 2.0 ** -24 * 4 * float((x.double().abs() * g.double().abs()).sum() + 1)


def test_frequencies():
    e = np.arange(32)
    plain, a = capi.rotary_frequencies(64)
    assert np.allclose(plain, 10000.0 ** (-e / 32), rtol=1e-14) and a == 1.0
    linear, a = capi.rotary_frequencies(64, 10000.0, capi.ROTARY_LINEAR, 8.0)
    assert np.allclose(linear, plain / 8, rtol=1e-14) and a == 1.0
    wider, a = capi.rotary_frequencies(64, 10000.0, capi.ROTARY_BASE, 8.0)
    assert np.allclose(wider, (10000.0 * 8 ** (64 / 62)) ** (-e / 32), rtol=1e-13) and a == 1.0
    bands, a = capi.rotary_frequencies(64, 500000.0, capi.ROTARY_BANDS, 8.0, 8192, 1.0, 4.0)
    base = 500000.0 ** (-e / 32)
    turns = 8192 * base / (2 * np.pi)
    assert a == 1.0 and np.allclose(bands[turns > 4], base[turns > 4], rtol=1e-14) and np.allclose(bands[turns < 1], base[turns < 1] / 8, rtol=1e-14)
    mixed = (turns >= 1) & (turns <= 4)
    assert mixed.any() and (bands[mixed] < base[mixed]).all() and (bands[mixed] > base[mixed] / 8).all()
    parts, a = capi.rotary_frequencies(64, 10000.0, capi.ROTARY_PARTS, 8.0, 4096, 1.0, 32.0)
    at = [64 * math.log(4096 / (t * 2 * math.pi)) / (2 * math.log(10000.0)) for t in (32.0, 1.0)]
    keep = 1 - np.clip((e - math.floor(at[0])) / (math.ceil(at[1]) - math.floor(at[0])), 0, 1)
    assert np.allclose(parts, plain * (keep + (1 - keep) / 8), rtol=1e-13) and abs(a - (0.1 * math.log(8.0) + 1)) < 1e-15
    assert len(capi.rotary_frequencies(2)[0]) == 1 and capi.rotary_frequencies(2, 10000.0, capi.ROTARY_BASE, 2.0)[0][0] == 1.0


@pytest.mark.parametrize("args,says", [((0,), "rot_dim"), ((7,), "rot_dim"), ((5000,), "rot_dim"), ((64, 1.0), "base"), ((64, math.inf), "base"), ((64, 1e4, 9), "scaling"),
                                       ((64, 1e4, capi.ROTARY_LINEAR, 0.5), "factor"), ((64, 1e4, capi.ROTARY_BASE, math.nan), "factor"),
                                       ((64, 1e4, capi.ROTARY_BANDS, 2.0, 0, 1.0, 4.0), "known_len"), ((64, 1e4, capi.ROTARY_PARTS, 2.0, 100, 4.0, 1.0), "low"),
                                       ((64, 1e4, capi.ROTARY_BANDS, 2.0, 100, 0.0, 1.0), "low")])
def test_frequency_refusals(args, says):
    with pytest.raises(capi.SddmmError, match=says):
        capi.rotary_frequencies(*args)


def desc(**kw):
    d = dict(type=capi.TYPE_BF16, n_rows=10, n_heads=4, n_kv_heads=2, head_dim=64, rot_dim=64, layout=HALF)
    d.update(kw)
    return capi.RotaryDesc.packed(**d)


@pytest.mark.parametrize("kw,says", [(dict(type=5), "type"), (dict(layout=2), "layout"), (dict(layout=-1), "layout"), (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=63), "rot_dim"),
                                     (dict(rot_dim=66), "rot_dim"), (dict(head_dim=1, rot_dim=2), "rot_dim"), (dict(head_dim=8192), "rot_dim"),
                                     (dict(n_heads=0), "heads"), (dict(n_kv_heads=-1), "heads"), (dict(n_rows=-1), "negative"),
                                     (dict(amplitude=math.inf), "amplitude"), (dict(amplitude=math.nan), "amplitude"), (dict(q_row=60), "stride"), (dict(k_out_head=10), "stride"),
                                     (dict(q_head=-64), "stride"), (dict(q_out_row=128), "overlap"), (dict(k_out_row=64, k_out_head=64), "overlap")])
def test_refusals(kw, says):
    with pytest.raises(capi.SddmmError, match=says) as e:
        capi.rotary(desc(**kw), A, A, A, A, A, A)
    assert e.value.code == capi.ERR_ARG


def test_pointer_refusals():
    for i in range(1, 6):
        args = [A] * 6
        args[i] = 0
        with pytest.raises(capi.SddmmError, match="NULL device pointer"):
            capi.rotary(desc(), *args)
    for i, off in ((0, 2), (1, 4), (2, 1), (3, 1), (4, 1), (5, 1)):
        args = [A] * 6
        args[i] += off
        with pytest.raises(capi.SddmmError, match="aligned"):
            capi.rotary(desc(), *args)
    with pytest.raises(capi.SddmmError, match="too many") as e:
        capi.rotary(desc(n_heads=1 << 17), *[A] * 6)
    assert e.value.code == capi.ERR_RANGE
    with pytest.raises(capi.SddmmError, match="NULL description"):
        capi.check(capi.lib().sddmm_rotary(None, A, A, A, A, A, A, None))
    capi.rotary(desc(n_rows=0), 0, 0, 0, 0)  # nothing to do: returns before a launch
