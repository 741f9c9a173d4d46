"""sddmm_attention_paged over codes whose scales are 0, tiny, or far from each other."""
import pytest
import torch

from sddmm_gpu_amd import capi
from tests import attention_reference as ref
from tests import cache_reference as cref
from tests.test_gpu_cache import BF16, DEV, F16, F32, Pages, attend, normal, stream, tables

pytestmark = pytest.mark.gpu

FEW, MANY, MIXED = [2], [70], [90, 1, 1, 1, 1, 1, 1]


def check(dtype, held, n_new, after, v_scales, away=(), cap=0.0, unit=1.0, seed=41):
    """Results against 64 bits.  v_scales(n): the values' scales of the n tokens of a sequence; `away`: tokens that rows see with scores far below the others'.

    Bounds: a row's weights, probabilities times scales, are rounded to 11 bits or more and those below 2^-24 of its largest may be lost (so n * 2^-24 of the largest, times
    the largest code, in all); scores and sums as the reference says of fp32; the result's own rounding.  All in units of `unit`, a power of two about as large as
    the values, since the reference's bounds have an absolute part."""
    page, heads, kv, dim = 32, 4, 2, 64
    table, n_pages = tables(after, page, seed)
    pages = Pages(dtype, held, n_pages, page, 1, kv, dim, False, seed)
    q = normal(seed + 3, sum(n_new), heads, dim).abs().to(dtype)
    k_scale, v_scale = (pages.scales[name].cpu() for name in "kv")
    k_scale[:] = 2.0 ** -5 if held == "i8" else 2.0 ** -7
    codes = pages.cpu["k"][0]
    for s, m in enumerate(after):
        v_of = v_scales(m)
        for j in range(m):
            v_scale[table[s][j // page], :, j % page] = float(v_of[j])
        for j in away:  # (queries are positive: scores of -200 and less)
            codes[table[s][j // page], j % page] = -127.0 if held == "i8" else -448.0
            k_scale[table[s][j // page], :, j % page] = 0.25
    pages._view(pages.gpu["k"]).copy_(codes.to(pages.store) if held == "i8" else codes.float().to(pages.store))
    for name, scale in (("k", k_scale), ("v", v_scale)):
        pages.scales[name].copy_(scale)
        pages.cpu[name] = (pages.cpu[name][0], scale)
    out, _ = attend(dtype, pages, table, n_new, after, heads, q, True, cap=cap)
    at = 0
    for s, (n, m) in enumerate(zip(n_new, after)):
        k, v = (cref.gathered(pages.cpu[name], s, m, table, page, 1, held) for name in "kv")
        steps = v_scales(m).double() / unit
        v = v / unit
        for h in range(heads):
            c = h // 2
            x = q[at: at + n, h].float()
            r = ref.head(x, k[:, c], v[:, c], -1, 0, 0, dim ** -0.5, cap, 0.0)
            pv = ref.head(x, k[:, c], v[:, c].abs(), -1, 0, 0, dim ** -0.5, cap, 0.0)["out"]
            t = q[at: at + n, h].double() @ k[:, c].T * dim ** -0.5
            t = torch.tanh(t / cap) * cap if cap else t
            weights = torch.where(torch.arange(m)[None] <= torch.arange(m - n, m)[:, None], torch.exp(t - r["lse"][:, None]), 0.0) * steps
            lost = 0.0 if dtype == F32 else m * 2.0 ** -24 * weights.amax(1, keepdim=True) * (v[:, c].abs().amax(1) / steps.clamp(min=1e-300)).max()
            tol = r["out_tol"] + lost + (0.0 if dtype == F32 else 2.0 ** -11 * 1.02 * pv)
            tol = tol + ref.HALF[dtype] * (r["out"].abs() + tol) + (2.0 ** -25 / unit if dtype == F16 else 0.0)
            bad = ~((out[at: at + n, h].double() / unit - r["out"]).abs() <= tol)
            assert not bad.any(), (s, h, int(bad.sum()), bad.nonzero()[:3], out[at: at + n, h][bad][:3] / unit, r["out"][bad][:3], tol[bad][:3])
        at += n


def ends(n_new, *lengths):
    """Lengths of the sequences of n_new, the first ones given."""
    return [max(n, lengths[i] if i < len(lengths) else 40 + 30 * i) for i, n in enumerate(n_new)]


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n_new", [FEW, MANY, MIXED])
def test_scales_of_zero(dtype, held, n_new):
    """Values of scale 0 everywhere, in whole tiles of keys before, between and behind others, and in all but one token."""
    one = 2.0 ** -5 if held == "i8" else 2.0 ** -7
    for length in (128, 150, 400):
        for zero in (lambda j: j >= 0, lambda j: j < 64, lambda j: (j >= 64) & (j < 128), lambda j: j >= 64, lambda j: j < 128, lambda j: j != 5):
            check(dtype, held, n_new, ends(n_new, length), lambda n: torch.where(zero(torch.arange(n)), 0.0, one))


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n_new", [FEW, MANY, MIXED, [40], [66]])
def test_tiny_scales(dtype, held, n_new):
    """Values of about 2^-e, in caches that end inside a tile of keys."""
    for length in (40, 64, 66, 130, 150):
        for e in (15, 24, 38, 44, 48, 60, 100):
            check(dtype, held, n_new, ends(n_new, length), lambda n: torch.full((n,), 2.0 ** -e), unit=2.0 ** (5 - e), cap=30.0 if e == 48 else 0.0)


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n_new", [FEW, MANY, MIXED])
def test_scales_far_apart(dtype, held, n_new):
    """Rows whose values are far smaller than others of the tile: of a token behind them, or of one that they hardly see; scales that rise and fall along the cache."""
    for length in (96, 150, 700):
        def last_large(n):
            return torch.where(torch.arange(n) == n - 1, 2.0 ** 60, 2.0 ** -30)

        def first_large(n):
            return torch.where(torch.arange(n) == 0, 2.0 ** 60, 2.0 ** -30)

        def rising(n):
            return torch.ldexp(torch.ones(n), torch.arange(n) * 80 // n - 60)

        check(dtype, held, n_new, ends(n_new, length), last_large, unit=2.0 ** -25)
        check(dtype, held, n_new, ends(n_new, length), first_large, unit=2.0 ** -25, away=(0,))
        check(dtype, held, n_new, ends(n_new, length), first_large, unit=2.0 ** -25, away=(0,), cap=400.0)
        check(dtype, held, n_new, ends(n_new, length), rising, unit=2.0 ** -10)
        check(dtype, held, n_new, ends(n_new, length), lambda n: rising(n).flip(0), unit=2.0 ** -10)


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("n_new", [FEW, MANY, MIXED])
def test_scales_far_apart_in_fp16(held, n_new):
    """The same within the range of fp16: one token of values up to 2^15 that rows hardly see, values of about 2^-10 (2^-2) for the rest."""
    large, small = (2.0 ** 8, 2.0 ** -15) if held == "i8" else (2.0 ** 6, 2.0 ** -17)
    for length in (96, 150, 700):
        for j in (0, 5, 60):
            check(F16, held, n_new, ends(n_new, length), lambda n: torch.where(torch.arange(n) == j, large, small), away=(j,) if j < 40 else (), unit=2.0 ** -5)


def test_scales_in_one_array():
    """Keys' and values' scales one behind the other: as in arrays of their own."""
    n_new, page, block, heads, kv, dim = [9, 30], 16, 8, 4, 2, 64
    after = [20, 30]
    table, n_pages = tables(after, page, 3)
    results = []
    for together in (False, True):
        pages = Pages(BF16, "i8", n_pages, page, block, kv, dim, False, 4)
        if together:
            both = torch.stack([pages.scales["k"], pages.scales["v"]])
            pages.scales = {"k": both[0], "v": both[1]}
        k, v = (normal(6 + i, sum(n_new), kv, dim).to(BF16).to(DEV) * 40 for i in range(2))
        t, length, ptr = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (table, after, [0, 9, 39]))
        desc = capi.AttentionDesc.packed(capi.TYPE_BF16, 2, heads, kv, dim, max_q=30, max_k=30, k_len=length.data_ptr(), q_ptr=ptr.data_ptr(), q_rows=39)
        capi.cache_append(desc, pages.desc(t), 0, 0, k.data_ptr(), v.data_ptr(), stream())
        torch.cuda.synchronize()
        results.append([x.cpu() for name in "kv" for x in (pages.gpu[name], pages.scales[name])])
    assert all(torch.equal(x, y) for x, y in zip(*results))
