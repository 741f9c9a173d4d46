"""sddmm_cache_append and sddmm_attention_paged against their definitions in 64 bits."""
import math

import pytest
import torch

from sddmm_gpu_amd import capi
from tests import attention_reference as ref
from tests import cache_reference as cref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CODE = {F32: capi.TYPE_F32, BF16: capi.TYPE_BF16, F16: capi.TYPE_F16}
HELD = {"i8": (capi.TYPE_I8, torch.int8), "e4m3": (capi.TYPE_E4M3, torch.float8_e4m3fn)}


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


class Pages:
    """A cache on the CPU, [page, token, head, dim] in 64 bits and scales, and on the GPU, in either order, rows padded to 16 bytes and `pad` more elements."""

    def __init__(self, dtype, held, n_pages, page, block, kv, dim, by_token, seed, pad=0, filled=True):
        self.dtype, self.held, self.page, self.block, self.kv, self.dim, self.n_pages = dtype, held, page, block, kv, dim, n_pages
        self.type, self.store = HELD.get(held, (CODE.get(dtype), dtype))
        self.cpu, self.gpu, self.scales = {}, {}, {}
        size = 1 if held != "own" else torch.empty(0, dtype=dtype).element_size()
        wide = -(-dim * size // 16) * 16 // size + pad * 16 // size
        for i, name in enumerate("kv"):
            x = normal(seed + i, n_pages, page, kv, dim)
            if not filled:
                x.zero_()
            x = (x.to(dtype) if held == "own" else (36 * x).round().clamp(-127, 127) if held == "i8" else (100 * x).clamp(-448, 448).to(torch.float8_e4m3fn)).double()
            scale = 2.0 ** torch.randint(-7, -3, (n_pages, kv, page // block), generator=torch.Generator().manual_seed(seed + 7 + i)).float() if held != "own" else None
            self.cpu[name] = (x, scale)
            shape = (n_pages, page, kv, wide) if by_token else (n_pages, kv, page, wide)
            g = torch.zeros(shape, dtype=self.store, device=DEV)
            self.gpu[name] = g
            self._view(g, by_token).copy_(x.to(self.store) if held != "e4m3" else x.float().to(self.store))
            self.scales[name] = scale.to(DEV) if scale is not None else None
        self.by_token, self.wide = by_token, wide

    def _view(self, g, by_token=None):
        by_token = self.by_token if by_token is None else by_token
        return (g if by_token else g.transpose(1, 2))[..., : self.dim]

    def read(self, name):
        return self._view(self.gpu[name]).cpu().float().double(), self.scales[name].cpu() if self.scales[name] is not None else None

    def desc(self, table, **kw):
        d = dict(k=self.gpu["k"].data_ptr(), v=self.gpu["v"].data_ptr(), table=table.data_ptr(), table_row=table.stride(0), block_len=self.block)
        if self.held != "own":
            d.update(k_scale=self.scales["k"].data_ptr(), v_scale=self.scales["v"].data_ptr())
        for n in "kv":
            d[n + "_page"] = self.page * self.kv * self.wide
            d[n + "_row"], d[n + "_head"] = (self.kv * self.wide, self.wide) if self.by_token else (self.wide, self.page * self.wide)
        d.update(kw)
        return capi.CacheDesc.defaults(type=self.type, n_pages=self.n_pages, page_len=self.page, **d)


def tables(after, page, seed, spare=2):
    """(rows of page numbers, count of pages): no two sequences share one."""
    need = [max(1, -(-m // page)) for m in after]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    rows, at = [], 0
    for n in need:
        rows.append(order[at: at + n])
        at += n
    most = max(need, default=1)
    return [r + [-1] * (most - len(r)) for r in rows], sum(need) + spare


def stream():
    return torch.cuda.current_stream().cuda_stream


def check_append(dtype, held, n_new, after, heads, kv, dim, page, block, rot, layout, by_token=False, packed=True, amplitude=1.0, seed=1, pad=0, in_place=False,
                 change=None, queries=True):
    table, n_pages = tables(after, page, seed)
    pages = Pages(dtype, held, n_pages, page, block, kv, dim, by_token, seed + 10, pad)
    total, most = sum(n_new), max(n_new, default=0)
    q, k, v = (normal(seed + 20 + i, total, h, dim).to(dtype) for i, h in enumerate((heads, kv, kv)))
    if change:
        change(k, v)
    freq = torch.tensor([10000.0 ** (-2 * e / max(rot, 1)) for e in range(rot // 2)], dtype=torch.float64)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(n_new, after)]) if total else torch.empty(0)
    want_q = cref.turned(q, pos, freq, rot, layout, amplitude)
    for name, x in (("k", cref.turned(k, pos, freq, rot, layout, amplitude).float()), ("v", v.float())):
        cref.append(pages.cpu[name], x, n_new, after, table, page, block, held, dtype)

    t = torch.tensor(table, dtype=torch.int32, device=DEV)
    length = torch.tensor(after, dtype=torch.int32, device=DEV)
    d_freq = freq.to(DEV)
    more = dict(max_q=most, max_k=max(after), k_len=length.data_ptr())
    if packed:
        ptr = torch.tensor([0] + n_new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV)
        more.update(q_ptr=ptr.data_ptr(), q_rows=total)
        dq, dk, dv = (x.to(DEV) for x in (q, k, v))
    else:
        new = torch.tensor(n_new, dtype=torch.int32, device=DEV)
        more.update(q_len=new.data_ptr(), k_seq=most * kv * dim, v_seq=most * kv * dim)
        at = [sum(n_new[:s]) for s in range(len(n_new))]

        def spread(x):
            y = torch.full((len(n_new), most) + x.shape[1:], float("nan"), dtype=dtype)
            for s, n in enumerate(n_new):
                y[s, :n] = x[at[s]: at[s] + n]
            return y.to(DEV)

        dq, dk, dv = spread(q), spread(k), spread(v)
    desc = capi.AttentionDesc.packed(CODE[dtype], len(n_new), heads, kv, dim, **more)
    out = dq if in_place else torch.full_like(dq, 7.0)
    cache = pages.desc(t, rot_dim=rot, rot_layout=layout, rot_amplitude=amplitude, rot_freq=d_freq.data_ptr() if rot else 0)
    capi.cache_append(desc, cache, dq.data_ptr() if queries else 0, out.data_ptr() if queries else 0, dk.data_ptr(), dv.data_ptr(), stream())
    torch.cuda.synchronize()
    # What is turned into 16 bits: cosine and sine are rounded to fp32 (2^-24 of at most 1), and so are a product and the sum of it and the other one: 4 * 2^-24 of the pair's
    # size at most; then the rounding to the type.  What is turned into fp32 or codes: in 64 bits, rounded to fp32.
    coarse = 0.0 if dtype == F32 else 4 * 2.0 ** -24
    sizes = {"q": coarse * cref.pair_sizes(q, rot, layout, amplitude), "k": 0.0, "v": 0.0}
    if held == "own" and coarse:
        at_cache = torch.zeros_like(pages.cpu["k"][0])
        cref.append((at_cache, None), (coarse * cref.pair_sizes(k, rot, layout, amplitude) * 1.01).float(), n_new, after, table, page, block, "own", F32)
        sizes["k"] = at_cache
    for name in "kv":
        got, scale = pages.read(name)
        want, want_scale = pages.cpu[name]
        if held == "own":
            # (`want` is rounded to the type itself: another half a step)
            tol = 2 * (ref.HALF[dtype] + 2.0 ** -23) * want.abs() + 1e-37 + (2.0 ** -24 if dtype == F16 else 0) + sizes[name]
            same = (got == want) | (got.isnan() & want.isnan())
            assert (same | ((got - want).abs() <= tol)).all(), (name, (got - want).abs().max())
        else:
            assert torch.equal(scale, want_scale), (name, (scale != want_scale).nonzero()[:5], scale[scale != want_scale][:5], want_scale[scale != want_scale][:5])
            bad = (got != want) & ~(got.isnan() & want.isnan())
            assert not bad.any(), (name, bad.nonzero()[:5], got[bad][:5], want[bad][:5])
    if queries:
        o = out.cpu()
        if not packed:
            if not in_place:
                for s, n in enumerate(n_new):
                    assert (o[s, n:] == 7.0).all()  # rows behind a sequence's new ones
            o = torch.cat([o[s, :n] for s, n in enumerate(n_new)])
        tol = (ref.HALF[dtype] + 2.0 ** -23) * want_q.abs() + (2.0 ** -24 if dtype == F16 else 1e-37) + 1e-12 * amplitude * q.double().abs().amax(-1, keepdim=True) + sizes["q"]
        assert ((o.double() - want_q).abs() <= tol).all()


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("page,block", [(16, 1), (16, 2), (32, 4), (16, 8), (64, 16), (32, 32), (64, 64), (256, 32)])
def test_append(dtype, held, page, block):
    check_append(dtype, held, [5, 1, 40, 130], [5, 37, 51, 200], 4, 2, 128, page, block, 128, cref.HALF)
    check_append(dtype, held, [1, 3, 2], [40, 3, 18], 6, 3, 64, page, block, 32, cref.INTERLEAVED, by_token=True, packed=False, amplitude=1.25)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dim,rot,layout", [(8, 8, 0), (16, 0, 0), (24, 24, 0), (40, 40, 0), (40, 6, 1), (72, 72, 0), (72, 20, 1), (80, 80, 0), (96, 48, 0), (104, 104, 1),
                                            (120, 62, 0), (128, 2, 0), (64, 64, 0), (56, 56, 1)])
def test_head_sizes(held, dim, rot, layout):
    for by_token in (False, True):
        check_append(BF16, held, [17, 2], [30, 50], 3, 1, dim, 32, 8, rot, layout, by_token=by_token, pad=by_token, in_place=by_token)
    check_append(F32, held, [3], [3], 2, 2, dim, 16, 16, rot, layout, queries=False)


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("block", [1, 4, 16, 64])
def test_scales(held, block):
    """Larger elements than the block has met, none, zeros alone, infinities and NaNs, and elements near the ends of the range."""
    def large(k, v):
        k[::3] *= 1000.0
        v[::2] *= 3e4

    def small(k, v):
        k *= 1e-30
        v[:] = 0
        k[3] = 0

    def odd(k, v):
        k[1, :, 5], k[2, :, 7], v[0, :, 0], v[4, 0, :] = math.inf, -math.inf, math.nan, math.inf
        v[7] = math.nan

    def ends(k, v):
        k[0], v[1], v[2] = 3e38, -3.3e38, 2e-39

    for change in (large, small, odd, ends):
        check_append(BF16, held, [9, 30, 1], [20, 30, 64], 2, 2, 64, 64, block, 0 if change is odd or change is ends else 64, cref.HALF, change=change)


def test_few_and_many():
    check_append(BF16, "i8", [1], [1], 8, 8, 128, 16, 16, 128, cref.HALF)
    check_append(BF16, "i8", [1], [1], 1, 1, 8, 16, 16, 8, cref.HALF)
    check_append(BF16, "e4m3", [1] * 70, [1 + 3 * i for i in range(70)], 2, 1, 64, 16, 16, 64, cref.HALF)          # more sequences than lanes, packed
    check_append(F16, "i8", [1, 0, 2] * 50, [9 + i for i in range(150)], 2, 1, 64, 32, 4, 64, cref.HALF)
    check_append(BF16, "own", [0, 700, 0, 3], [0, 900, 5, 3], 2, 2, 96, 128, 1, 96, cref.INTERLEAVED)
    check_append(BF16, "i8", [12, 4], [7, 4], 2, 1, 64, 16, 16, 64, cref.HALF)                                       # more new rows than the length counts
    check_append(BF16, "i8", [100], [70000], 2, 1, 64, 4096, 64, 64, cref.HALF)                                      # angles of far positions


def attend(dtype, pages, table, n_new, after, heads, q, packed, left=-1, right=0, prefix=None, cap=0.0, slopes=None, scale=None, lse=True):
    kv, dim = pages.kv, pages.dim
    t = torch.tensor(table, dtype=torch.int32, device=DEV)
    length = torch.tensor(after, dtype=torch.int32, device=DEV)
    total, most = sum(n_new), max(n_new)
    more = dict(max_q=most, max_k=max(after), k_len=length.data_ptr(), window_left=left, window_right=right, cap=cap)
    if scale is not None:
        more["scale"] = scale
    keep = [t, length]
    if prefix is not None:
        keep.append(torch.tensor(prefix, dtype=torch.int32, device=DEV))
        more["prefix"] = keep[-1].data_ptr()
    if slopes is not None:
        keep.append(slopes.to(DEV))
        more["slopes"] = keep[-1].data_ptr()
    if packed:
        keep.append(torch.tensor([0] + n_new, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(DEV))
        more.update(q_ptr=keep[-1].data_ptr(), q_rows=total)
        dq = q.to(DEV)
    else:
        keep.append(torch.tensor(n_new, dtype=torch.int32, device=DEV))
        more["q_len"] = keep[-1].data_ptr()
        dq = torch.full((len(n_new), most, heads, dim), float("nan"), dtype=dtype)
        at = 0
        for s, n in enumerate(n_new):
            dq[s, :n] = q[at: at + n]
            at += n
        dq = dq.to(DEV)
    desc = capi.AttentionDesc.packed(CODE[dtype], len(n_new), heads, kv, dim, **more)
    cache = pages.desc(t)
    out = torch.full_like(dq, 7.0)
    stat = torch.full(dq.shape[:-1], 7.0, dtype=F32, device=DEV)
    n = capi.attention_paged_workspace_bytes(desc, cache)
    ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=DEV)
    capi.attention_paged(desc, cache, dq.data_ptr(), out.data_ptr(), stat.data_ptr() if lse else 0, ws.data_ptr(), n, stream())
    torch.cuda.synchronize()
    out, stat = out.cpu(), stat.cpu()
    if not packed:
        for s, n in enumerate(n_new):
            assert (out[s, n:] == 7.0).all() and (stat[s, n:] == 7.0).all()
        out, stat = (torch.cat([x[s, :n] for s, n in enumerate(n_new)]) for x in (out, stat))
    return out, stat


def lost(dtype, held, n_keys, v):
    """What weights that are rounded to fp16 may be off by in all, where that is more than their share of 2^-11: half of the least step, 2^-25, each, times the values.
    fp16 operands: the largest weight is 1 at least (and scales of values enter it, in units of the largest, a code of up to 16 times the largest value of a key); bf16
    operands over codes, many rows: the running maximum is at most the largest score, and weights are 2^7 times those below it, so the largest is 2^7 at least.
    Results in fp16 are off by half of the least step themselves."""
    if not n_keys or (dtype == BF16 and held == "own") or dtype == F32:
        return 0.0
    each = 2.0 ** -25 * 16 if dtype == F16 else 2.0 ** -32
    return n_keys * each * v.abs().max() + (2.0 ** -25 if dtype == F16 else 0)


def check_attend(dtype, held, n_new, after, heads, kv, dim, page, block, by_token=False, packed=True, seed=5, pad=0, spoil=True, lse=True, **mask):
    table, n_pages = tables(after, page, seed)
    pages = Pages(dtype, held, n_pages, page, block, kv, dim, by_token, seed, pad)
    q = normal(seed + 3, sum(n_new), heads, dim).to(dtype)
    if spoil:  # what lies behind the sequences, in their last pages and in others, is not finite
        used = torch.zeros(n_pages, page, dtype=torch.bool)
        for s, m in enumerate(after):
            for j in range(m):
                used[table[s][j // page], j % page] = True
        for name in "kv":
            g = pages._view(pages.gpu[name])
            if held != "i8":
                y = g.float().cpu()
                y[~used] = float("nan")
                g.copy_(y.to(pages.store))
            if held != "own":
                sc = pages.scales[name].cpu()
                free = ~used.view(n_pages, page // block, block).any(-1)
                sc[free[:, None, :].expand_as(sc)] = float("nan")
                pages.scales[name].copy_(sc)
    out, stat = attend(dtype, pages, table, n_new, after, heads, q, packed, lse=lse, **mask)
    at = 0
    scale = mask.get("scale") or dim ** -0.5
    for s, (n, m) in enumerate(zip(n_new, after)):
        k, v = (cref.gathered(pages.cpu[name], s, m, table, page, block, held) for name in "kv")
        for h in range(heads):
            c = h // (heads // kv)
            pre = mask["prefix"][s] if mask.get("prefix") is not None else 0
            r = ref.head(q[at: at + n, h], k[:, c], v[:, c], mask.get("left", -1), mask.get("right", 0), pre, scale, mask.get("cap", 0.0),
                         float(mask["slopes"][h]) if mask.get("slopes") is not None else 0.0)
            tol = r["out_tol"] + lost(dtype, held, m, v[:, c])
            bad = (out[at: at + n, h].double() - r["out"]).abs() > tol
            assert not bad.any(), (s, h, bad.nonzero()[:4], out[at: at + n, h][bad][:4], r["out"][bad][:4], tol[bad][:4])
            assert not out[at: at + n, h].isnan().any()
            if lse:
                x, y = stat[at: at + n, h].double(), r["lse"]
                assert ((x == y) | ((x - y).abs() <= r["lse_tol"])).all(), (s, h, x, y)
        at += n


SHAPES = [(4, 2, 128), (8, 1, 64), (3, 3, 96), (40, 2, 32), (16, 1, 128)]


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_attend_tokens(dtype, held, heads, kv, dim):
    check_attend(dtype, held, [1, 1, 1, 1], [1, 33, 700, 64], heads, kv, dim, 16, 16)
    check_attend(dtype, held, [1, 0, 2, 3], [300, 5, 2, 47], heads, kv, dim, 64, 4, by_token=True, packed=False)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_masks(dtype, held):
    slopes = torch.tensor([0.5, 0.25, 0.1, 0.03])
    for kw in (dict(left=20), dict(right=-1), dict(left=5, right=3), dict(left=0, right=0), dict(prefix=[10, 0, 70]), dict(cap=5.0), dict(slopes=slopes), dict(cap=20.0, slopes=slopes, left=40)):
        check_attend(dtype, held, [7, 1, 40], [200, 90, 75], 4, 2, 64, 32, 16, **kw)
    # rows that see nothing: more rows than the cache has tokens, and no tokens at all
    check_attend(dtype, held, [9, 3, 1], [4, 1, 0], 4, 2, 64, 16, 1)
    check_attend(dtype, held, [2, 2], [0, 0], 4, 2, 64, 16, 1, lse=False)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 56, 72, 80, 88, 104, 112, 120])
def test_attend_head_sizes(held, dim):
    check_attend(BF16, held, [1, 4], [70, 100], 4, 2, dim, 16, 8, by_token=dim % 16 == 8, pad=1)
    check_attend(F32, held, [1, 20], [70, 100], 2, 1, dim, 16, 8)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("page,block", [(16, 1), (16, 2), (16, 8), (64, 32), (64, 64), (512, 16), (4096, 64)])
def test_attend_pages(held, page, block):
    check_attend(BF16, held, [1, 1, 5], [1023, 129, 2100], 8, 2, 128, page, block)
    check_attend(F16, held, [1, 30], [1500, 31], 2, 2, 64, page, block, by_token=True, left=1000)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_attend_many_rows(dtype, held):
    check_attend(dtype, held, [150, 1, 90, 1, 17], [600, 400, 90, 33, 100], 8, 2, 64, 64, 16)
    check_attend(dtype, held, [130], [390], 4, 4, 128, 32, 1, by_token=True, packed=False)
    check_attend(dtype, held, [65, 64], [65, 300], 2, 1, 128, 16, 16, left=30, cap=10.0)


@pytest.mark.parametrize("held", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n_new,after", [([1, 2], [90, 300]), ([70, 3], [200, 130])])
def test_attend_scales(dtype, held, n_new, after):
    """Scales that are no powers of two, as calibrated ones, some of them far from the others, and far from 1."""
    for low, high, extra in ((0.01, 0.02, 0), (1e-3, 1.0, 0), (2e-9, 4e-9, 0), (0.01, 0.02, 1), (300.0, 400.0, 0)):
        seed = 31
        table, n_pages = tables(after, 32, seed)
        pages = Pages(dtype, held, n_pages, 32, 4, 2, 64, False, seed)
        for i, name in enumerate("kv"):
            g = torch.Generator().manual_seed(seed + 40 + i)
            sc = low * (high / low) ** torch.rand(pages.scales[name].shape, generator=g)
            if extra:
                sc[torch.rand(sc.shape, generator=g) < 0.3] = 0.015625
                if name == "v":
                    sc[torch.rand(sc.shape, generator=g) < 0.1] = 0.0
            pages.scales[name].copy_(sc)
            pages.cpu[name] = (pages.cpu[name][0], sc.float())
        q = normal(seed + 3, sum(n_new), 4, 64).to(dtype)
        scale = 0.125 * 0.015 / high
        out, stat = attend(dtype, pages, table, n_new, after, 4, q, True, scale=scale)
        at = 0
        for s, (n, m) in enumerate(zip(n_new, after)):
            k, v = (cref.gathered(pages.cpu[name], s, m, table, 32, 4, held) for name in "kv")
            for h in range(4):
                r = ref.head(q[at: at + n, h], k[:, h // 2], v[:, h // 2], -1, 0, 0, scale, 0.0, 0.0)
                tol = r["out_tol"] + lost(dtype, held, m, v)
                assert ((out[at: at + n, h].double() - r["out"]).abs() <= tol).all(), (low, high, s, h)
            at += n


@pytest.mark.parametrize("held", ["i8", "e4m3"])
def test_attend_query_ranges(held):
    """bf16 queries of any size, which meet codes in fp16."""
    for size in (1e-30, 1e-4, 1e4, 1e30):
        table, n_pages = tables([150], 16, 3)
        pages = Pages(BF16, held, n_pages, 16, 16, 1, 64, False, 4)
        for n in (2, 130):
            q = (normal(5, n, 2, 64) * size * torch.exp(2 * normal(6, n, 2, 64))).to(BF16)
            q[0, 0] = 0
            out, stat = attend(BF16, pages, table, [n], [150], 2, q, True, scale=min(0.125 / size, 3e38))
            k, v = (cref.gathered(pages.cpu[name], 0, 150, table, 16, 16, held) for name in "kv")
            for h in range(2):
                r = ref.head(q[:, h], k[:, 0], v[:, 0], -1, 0, 0, min(0.125 / size, 3e38), 0.0, 0.0)
                assert ((out[:, h].double() - r["out"]).abs() <= r["out_tol"] + lost(BF16, held, 150, v)).all(), (size, n, h)


@pytest.mark.parametrize("held", ["i8", "e4m3", "own"])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 64), (20, 1, 128), (40, 1, 64)])
def test_attend_mixed(dtype, held, heads, kv, dim):
    """Pieces of prompts beside single tokens, drafts and sequences without new rows."""
    new = [1, 160, 1, 0, 2, 1, 1, 40, 1, 1, 3, 1, 0, 1]
    check_attend(dtype, held, new, [700, 300, 1, 50, 90, 33, 1100, 40, 64, 500, 3, 17, 0, 200], heads, kv, dim, 32, 8)
    check_attend(dtype, held, new, [2000, 1300, 1, 50, 90, 33, 1100, 40, 64, 500, 2, 17, 0, 0], heads, kv, dim, 64, 16, left=300, cap=20.0)
