"""A paged cache of keys and values by its definition in include/sddmm.h (for the tests of sddmm_cache_append and sddmm_attention_paged; all on the CPU)."""
import math

import torch

MOST = {"i8": 127.0, "e4m3": 448.0}
HALF, INTERLEAVED = 0, 1


def code_of(x, held):
    """The nearest code, ties to even, of fp32 values in steps of the scale, as the number that it is."""
    x = x.double()
    if held == "i8":
        return torch.where(x.isnan(), 0.0, torch.round(x).clamp(-127, 127))
    _, e = torch.frexp(x.abs().clamp(max=448.0).nan_to_num(0.0))
    step = torch.ldexp(torch.ones(()).double(), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448, 448)  # (NaN stays NaN)


def least_scale(top, held):
    if top == 0:
        return 2.0 ** -126
    e = max(-126, math.frexp(top / MOST[held])[1] - 2)
    while top > MOST[held] * 2.0 ** e:
        e += 1
    return 2.0 ** e


def turned(x, pos, freq, rot, layout, amplitude):
    """Rows [n, heads, dim] at positions [n], in 64 bits."""
    y = x.double().clone()
    if not rot:
        return y
    half = rot // 2
    first = torch.arange(half) * (1 if layout == HALF else 2)
    second = first + (half if layout == HALF else 1)
    angle = pos.double()[:, None, None] * freq
    z = torch.complex(y[..., first], y[..., second]) * torch.polar(torch.full_like(angle, amplitude), angle)
    y[..., first], y[..., second] = z.real, z.imag
    return y


def pair_sizes(x, rot, layout, amplitude):
    """amplitude * (|x| + |y|) of each turned element's pair, 0 for the others."""
    y = torch.zeros(x.shape, dtype=torch.float64)
    if rot:
        half = rot // 2
        first = torch.arange(half) * (1 if layout == HALF else 2)
        second = first + (half if layout == HALF else 1)
        y[..., first] = y[..., second] = abs(amplitude) * (x[..., first].double().abs() + x[..., second].double().abs())
    return y


def append(cache, rows, n_new, after, table, page, block, held, dtype):
    """Puts rows [n, heads, dim] (fp32; of all sequences one behind the other) into cache = (values or codes [page, token, head, dim] in
    64 bits, scales [page, head, blocks of a page])."""
    values, scales = cache
    at = 0
    for s, (n, m) in enumerate(zip(n_new, after)):
        x = rows[at: at + n]
        at += n
        start = m - n
        if held == "own":
            for i in range(max(0, -start), n):
                p = start + i
                values[table[s][p // page], p % page] = x[i].to(dtype).double()
            continue
        for b in range(max(start, 0) // block, -(-m // block)):
            lo, hi = max(b * block, start, 0), min(b * block + block, m)
            if hi <= lo:
                continue
            p, t = table[s][b * block // page], b * block % page
            kept = max(0, start - b * block)
            for h in range(x.shape[1]):
                new = x[lo - start: hi - start, h]
                finite = new.abs()[new.isfinite()]
                top = float(finite.max()) if finite.numel() else 0.0
                old = float(scales[p, h, t // block]) if kept else 0.0
                scale = old if old > 0 and top <= float(torch.tensor(old * MOST[held], dtype=torch.float32)) else least_scale(top, held)
                if kept and scale != old:
                    stale = (values[p, t: t + kept, h].float() * old).float() / scale
                    values[p, t: t + kept, h] = code_of(stale, held)
                values[p, lo % page: lo % page + hi - lo, h] = code_of(new.float() / scale, held)
                scales[p, h, t // block] = scale


def gathered(cache, s, n_keys, table, page, block, held):
    """The keys or values of sequence s, [n_keys, head, dim] in 64 bits."""
    values, scales = cache
    j = torch.arange(n_keys)
    p = torch.as_tensor(table[s], dtype=torch.long)[j // page]
    x = values[p, j % page]
    return x if held == "own" else x * scales[p][torch.arange(n_keys), :, (j % page) // block][..., None].double()
