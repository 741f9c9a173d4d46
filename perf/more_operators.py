"""Workloads of the paged cache of keys and values: the call that brings new tokens into it and the attention that reads it.

A cache lies in pages of "page" tokens that the sequences take in any order; a table says which.  It is held in the operands' type
("held" = "own") or in 8 bits, "i8" or "e4m3", with a scale for each "block" tokens of a page and key head.  A case is a dict of plain
values.  "op" says which call one pass makes:
  append   the new tokens' keys, turned by their positions ("rot" elements of a head, pairs as in "layout"), and values go into the
           cache; their queries are turned on the way
  attend   the new tokens' rows against the cache, which holds them already
"type" is the element type of queries, new keys and values and results, "heads" query heads share "kv_heads" key heads of "dim"
elements.  "n_seq" sequences bring "tokens" new tokens each, or (0) ragged ones that sum to "total", "singles" of them one token; the
longest sequence has "length" tokens afterwards.  "order": whether a page's rows are those of a head one behind the other ("head") or
those of a token.  "left" bounds the visible keys before a row (-1: no bound), "cap" the bound of the scores' tanh (0: none), "bias" a
bias by distance with a slope for each head.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
MOST = {"i8": 127.0, "e4m3": 448.0}  # the largest value of a code


def listed():
    return [
        # The next token of one user: latency.
        dict(name="append_1", op="append", type="bf16", held="i8", heads=32, kv_heads=8, dim=128, n_seq=1, tokens=1, total=0, singles=0, length=1501,
             page=16, block=16, order="head", rot=128, layout="half"),
        # The next tokens of 64 users.
        dict(name="append_64", op="append", type="bf16", held="i8", heads=32, kv_heads=8, dim=128, n_seq=64, tokens=1, total=0, singles=0, length=2048,
             page=64, block=16, order="head", rot=128, layout="half"),
        # Prompts of uneven lengths, a few of them behind what their sequence has already, into 8 bits.
        dict(name="append_prompts_16k", op="append", type="bf16", held="i8", heads=32, kv_heads=8, dim=128, n_seq=13, tokens=0, total=16384, singles=0, length=9000,
             page=64, block=16, order="head", rot=128, layout="half"),
        # The same with a scale for each token, in fp16, part of a head turned, interleaved pairs, odd lengths.
        dict(name="append_e4m3_6k", op="append", type="f16", held="e4m3", heads=12, kv_heads=12, dim=64, n_seq=3, tokens=0, total=5999, singles=0, length=4000,
             page=32, block=1, order="token", rot=32, layout="interleaved"),
        # A long piece of a prompt into a cache of the operands' type.
        dict(name="append_own_4k", op="append", type="bf16", held="own", heads=16, kv_heads=2, dim=128, n_seq=1, tokens=4096, total=0, singles=0, length=16384,
             page=256, block=1, order="token", rot=128, layout="half"),
        # One token of one user, a short cache: latency.
        dict(name="attend_1", op="attend", type="bf16", held="i8", heads=32, kv_heads=8, dim=128, n_seq=1, tokens=1, total=0, singles=0, length=1501,
             page=16, block=16, order="head", left=-1, cap=0.0, bias=False),
        # One token for each of 64 users with caches of uneven lengths: the caches have to be read.
        dict(name="attend_64", op="attend", type="bf16", held="i8", heads=32, kv_heads=8, dim=128, n_seq=64, tokens=1, total=0, singles=0, length=8192,
             page=64, block=16, order="head", left=-1, cap=0.0, bias=False),
        # A few users with long caches, a scale for each token, in fp16.
        dict(name="attend_long_e4m3", op="attend", type="f16", held="e4m3", heads=16, kv_heads=2, dim=128, n_seq=4, tokens=1, total=0, singles=0, length=32768,
             page=256, block=1, order="token", left=-1, cap=0.0, bias=False),
        # Five drafted tokens for each of 16 users, a window, capped scores, a cache of the operands' type.
        dict(name="attend_drafts_own", op="attend", type="bf16", held="own", heads=16, kv_heads=4, dim=64, n_seq=16, tokens=5, total=0, singles=0, length=6000,
             page=32, block=1, order="token", left=2047, cap=50.0, bias=False),
        # A piece of a prompt behind a long cache, the largest number of operations.
        dict(name="attend_chunk_2k", op="attend", type="bf16", held="i8", heads=16, kv_heads=2, dim=128, n_seq=1, tokens=2048, total=0, singles=0, length=16384,
             page=64, block=16, order="head", left=-1, cap=0.0, bias=False),
        # A serving batch: pieces of three prompts beside the next tokens of 29 users.
        dict(name="attend_mixed_e4m3", op="attend", type="bf16", held="e4m3", heads=32, kv_heads=8, dim=128, n_seq=32, tokens=0, total=1053, singles=29, length=4096,
             page=64, block=32, order="head", left=-1, cap=0.0, bias=False),
        # A small model in fp32, with a bias by distance and capped scores.
        dict(name="attend_bias_f32", op="attend", type="f32", held="i8", heads=4, kv_heads=2, dim=32, n_seq=2, tokens=3, total=0, singles=0, length=1013,
             page=16, block=4, order="token", left=-1, cap=30.0, bias=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))


def draw(rng):
    """One more case of the ranges above, at most the operations and bytes of the largest listed ones."""
    op = rng.choice(["append", "append", "attend", "attend", "attend"])
    case = dict(op=op, type=rng.choice(["bf16", "bf16", "f16", "f32"]), held=rng.choice(["i8", "i8", "e4m3", "e4m3", "own"]))
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
    case["dim"] = rng.choice([32, 64, 64, 80, 96, 128, 128])
    case["page"] = rng.choice([16, 32, 64, 128, 256])
    case["block"] = rng.choice([b for b in (1, 4, 16, 16, 32, 64) if b <= case["page"]])
    case["order"] = rng.choice(["head", "token"])
    kind = rng.choice(["tokens", "tokens", "tokens", "prompts", "mixed"])
    if kind == "tokens":
        n = int(_log_uniform(rng, 1, 64))
        tokens = rng.choice([1, 1, 1, 2, 4, 7])
        most = 32768.0 if op == "attend" else 2048.0
        most = min(most, 64 * 8192 * 8 * 128 / (n * case["kv_heads"] * case["dim"]), 5.0e8 / (n * case["heads"] * tokens))
        case.update(n_seq=n, tokens=tokens, total=0, singles=0, length=int(_log_uniform(rng, 16, most)))
    else:
        n = 1 if kind == "prompts" and rng.random() < 0.3 else rng.randint(2, 24)
        if op == "append":
            most = min(16384.0, 16384.0 * 40 * 128 / ((case["heads"] + case["kv_heads"]) * case["dim"]))
        else:  # (plain scores, all sequences as long as the longest)
            most = math.sqrt(min(1.5e9 / n, 5.0e8) / case["heads"])
        if case["type"] == "f32":
            most = min(most, 4096.0)
        total = int(_log_uniform(rng, max(64, 4 * n), most))
        if n == 1:
            case.update(n_seq=1, tokens=total, total=0, singles=0)
        else:
            case.update(n_seq=n, tokens=0, total=total, singles=rng.randint(1, n - 1) if kind == "mixed" else 0)
        more = min(8192.0, min(1.5e9 / n, 5.0e8) / (case["heads"] * total) - total) if op == "attend" else 4096.0
        case["length"] = total + (int(_log_uniform(rng, 16, more)) if more > 16 and rng.random() < 0.6 else 0)
    if op == "append":
        case.update(rot=rng.choice([0, case["dim"], case["dim"], case["dim"] // 2]), layout=rng.choice(["half", "interleaved"]))
    else:
        case.update(left=int(_log_uniform(rng, 16, 2048)) if rng.random() < 0.2 else -1, cap=rng.choice([0.0, 0.0, 0.0, 50.0]), bias=rng.random() < 0.2)
    return case


# ---------------------------------------------------------------- what follows from a case alone

def _sequences(case):
    """(new tokens, length after them) of each sequence."""
    rng = random.Random("%(n_seq)d %(tokens)d %(total)d %(singles)d %(length)d" % case)
    n = case["n_seq"]
    if case["tokens"]:
        new = [case["tokens"]] * n
    else:
        many = n - case["singles"]
        cuts = sorted(rng.sample(range(1, case["total"] - case["singles"]), many - 1))
        new = [b - a for a, b in zip([0] + cuts, cuts + [case["total"] - case["singles"]])] + [1] * case["singles"]
    after = [max(t, case["length"] if i == 0 else int(case["length"] * rng.random())) for i, t in enumerate(new)]
    if not case["tokens"] and not case["singles"]:  # (prompts: most of them begin their sequence)
        after = [a if i % 4 == 0 else t for i, (t, a) in enumerate(zip(new, after))]
    return list(zip(new, after))


def _pairs(case):
    """(row, key) pairs that are looked at, and keys that have to be read, of all sequences."""
    pairs = read = 0
    for new, after in _sequences(case):
        p = np.arange(after - new, after)
        lo = np.zeros_like(p) if case["left"] < 0 else np.maximum(0, p - case["left"])
        pairs += int((p + 1 - lo).sum())
        read += int(after - lo[0])
    return pairs, read


def work(case):
    size = 4 if case["type"] == "f32" else 2
    held = size if case["held"] == "own" else 1
    rows = sum(new for new, _ in _sequences(case))
    heads, kv, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    if case["op"] == "append":
        scales = 0 if case["held"] == "own" else sum(2 * kv * 4 * (-(-a // block) - (a - t) // block) for t, a in _sequences(case))
        return {"bytes": rows * dim * (2 * size * heads + 2 * (size + held) * kv) + scales, "flops": 3 * rows * (heads + kv) * case["rot"] + 4 * rows * kv * dim}
    pairs, read = _pairs(case)
    scales = 0 if case["held"] == "own" else 2 * 4 * kv * -(-read // block)
    return {"bytes": 2 * size * rows * heads * dim + 2 * held * read * kv * dim + scales, "flops": 4 * dim * pairs * heads}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = TYPES[case["type"]]
    heads, kv, dim, page, block, n = (case[x] for x in ("heads", "kv_heads", "dim", "page", "block", "n_seq"))
    seqs = _sequences(case)
    rows, pages = sum(new for new, _ in seqs), [-(-after // page) for _, after in seqs]
    n_pages, most = sum(pages) + 3, max(pages)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case=case, rows=rows, n_pages=n_pages, most_new=max(new for new, _ in seqs), longest=max(after for _, after in seqs))
    # the pages of the sequences, in no order; entries behind a sequence's last page name none
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    first = np.concatenate([[0], np.cumsum(pages)])
    at = torch.from_numpy(first[:-1, None] + np.arange(most)[None]).cuda()
    there = torch.from_numpy(np.arange(most)[None] < np.array(pages)[:, None]).cuda()
    s["table"] = torch.where(there, order[at.clamp(max=n_pages - 1)], -1).to(torch.int32).contiguous()
    s["len"] = torch.tensor([after for _, after in seqs], dtype=torch.int32, device="cuda")
    s["ptr"] = torch.tensor(np.concatenate([[0], np.cumsum([new for new, _ in seqs])]), dtype=torch.int32, device="cuda")
    s["q"] = normal(rows, heads, dim).to(t)
    shape = (n_pages, kv, page, dim) if case["order"] == "head" else (n_pages, page, kv, dim)
    for name in ("k_cache", "v_cache"):
        x = normal(*shape)
        s[name] = (x.to(t) if case["held"] == "own" else x.mul_(36).round_().clamp_(-127, 127).to(torch.int8) if case["held"] == "i8"
                   else x.mul_(100).clamp_(-448, 448).to(torch.float8_e4m3fn))
        del x
        if case["held"] != "own":  # (36 or 100 steps are values of about 1; 8 bits with a scale for each token are often calibrated ones)
            steps = torch.tensor([0.5, 1.0, 2.0], device="cuda") * (2.0 ** -5 if case["held"] == "i8" else 2.0 ** -7)
            scale = steps[torch.randint(0, 3, (n_pages, kv, page // block), generator=g, device="cuda")]
            if case["op"] == "attend" and block == 1:
                scale = scale * (0.75 + 0.5 * torch.rand(scale.shape, generator=g, device="cuda"))
            s[name[0] + "_scale"] = scale.contiguous()
    if case["op"] == "append":
        # keys have a few large elements at the same places of every token, values do not
        large = 1 + 4 * (torch.rand(kv, dim, generator=g, device="cuda") < 0.03)
        s.update(k=(normal(rows, kv, dim) * large).to(t), v=normal(rows, kv, dim).to(t))
        s["freq"] = torch.tensor(10000.0 ** (-2 * np.arange(case["rot"] // 2, dtype=np.float64) / max(case["rot"], 1)), dtype=torch.float64, device="cuda")
    else:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) if case["bias"] else None
        s["scale"] = dim ** -0.5
    if own:
        _keep(s)
    return s


# ---------------------------------------------------------------- the framework's calls

def _keep(s):
    from sddmm_gpu_amd import capi
    c = s["case"]
    t = {"f32": capi.TYPE_F32, "bf16": capi.TYPE_BF16, "f16": capi.TYPE_F16}[c["type"]]
    more = dict(max_k=s["longest"], k_len=s["len"].data_ptr(), max_q=s["most_new"], window_right=0)
    if not c["tokens"]:
        more.update(q_ptr=s["ptr"].data_ptr(), q_rows=s["rows"])
    if c["op"] == "append":
        more.update(k_seq=c["tokens"] * c["kv_heads"] * c["dim"], v_seq=c["tokens"] * c["kv_heads"] * c["dim"])
    if c["op"] == "attend":
        more.update(window_left=c["left"], cap=c["cap"], scale=s["scale"], slopes=s["slopes"].data_ptr() if c["bias"] else 0)
    s["desc"] = capi.AttentionDesc.packed(t, c["n_seq"], c["heads"], c["kv_heads"], c["dim"], **more)
    s["cache"] = capi.CacheDesc.packed(
        {"own": t, "i8": capi.TYPE_I8, "e4m3": capi.TYPE_E4M3}[c["held"]], s["n_pages"], c["page"], c["kv_heads"], c["dim"],
        by_token=c["order"] == "token", block_len=c["block"], table=s["table"].data_ptr(), table_row=s["table"].shape[1],
        k=s["k_cache"].data_ptr(), v=s["v_cache"].data_ptr(), **({} if c["held"] == "own" else dict(k_scale=s["k_scale"].data_ptr(), v_scale=s["v_scale"].data_ptr())),
        **(dict(rot_dim=c["rot"], rot_layout=capi.ROTARY_HALF if c["layout"] == "half" else capi.ROTARY_INTERLEAVED, rot_freq=s["freq"].data_ptr()) if c["op"] == "append" else {}))
    s["out"] = torch.empty_like(s["q"])
    if c["op"] == "attend":
        s["ws"] = torch.empty(max(capi.attention_paged_workspace_bytes(s["desc"], s["cache"]), 16), dtype=torch.uint8, device="cuda")


def _run_own(s):
    from sddmm_gpu_amd import capi
    stream = torch.cuda.current_stream().cuda_stream
    if s["case"]["op"] == "attend":
        capi.attention_paged(s["desc"], s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), 0, s["ws"].data_ptr(), s["ws"].numel(), stream)
        return dict(out=s["out"])
    capi.cache_append(s["desc"], s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), stream)
    return _updated(s, s["out"])


def _updated(s, q):
    r = dict(q=q, k=s["k_cache"], v=s["v_cache"])
    if s["case"]["held"] != "own":
        r.update(k_scale=s["k_scale"], v_scale=s["v_scale"])
    return r


# ---------------------------------------------------------------- the plain forms

def _by_token(s, cache):
    """The cache as [page, token, head, element], whatever its order."""
    return cache.transpose(1, 2) if s["case"]["order"] == "head" else cache


def _rotate(x, cos, sin, rot, layout):
    y = x.double()
    if layout == "half":
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
    p, q = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).float()


def _append(s):
    c = s["case"]
    rows, page, block = s["rows"], c["page"], c["block"]
    ptr, after = s["ptr"].long(), s["len"].long()
    row = torch.arange(rows, device="cuda")
    of = torch.searchsorted(ptr, row, right=True) - 1  # the sequence of each row
    new = ptr[1:] - ptr[:-1]
    pos = row - ptr[of] + (after - new)[of]
    angle = pos.double()[:, None, None] * s["freq"]
    cos, sin = torch.cos(angle), torch.sin(angle)
    q = _rotate(s["q"], cos, sin, c["rot"], c["layout"]).to(s["q"].dtype)
    k = _rotate(s["k"], cos, sin, c["rot"], c["layout"])
    for x, name in ((k, "k"), (s["v"].float(), "v")):
        cache = _by_token(s, s[name + "_cache"])
        if c["held"] == "own":
            cache[s["table"][of, pos // page].long(), pos % page] = x.to(cache.dtype)
            continue
        # the blocks that new tokens lie in: at most one more than whole ones for each sequence
        begin, first = after - new, (after - new) // block
        count = (after + block - 1) // block - first
        slots = torch.cumsum(count, 0)
        n_slots = rows // block + 2 * c["n_seq"] if block > 1 else rows
        slot = torch.arange(n_slots, device="cuda")
        seq = torch.searchsorted(slots, slot, right=True)
        real = seq < c["n_seq"]
        seq = seq.clamp(max=c["n_seq"] - 1)
        at = (first[seq] + slot - (slots - count)[seq])[:, None] * block + torch.arange(block, device="cuda")  # positions of their tokens
        fresh = real[:, None] & (at >= begin[seq, None]) & (at < after[seq, None])
        kept = real[:, None] & (at < begin[seq, None])
        where = s["table"][seq, torch.where(real, at[:, 0] // page, 0)].long()
        source = torch.where(fresh, ptr[seq, None] + at - begin[seq, None], 0)
        value = torch.where(fresh[..., None, None], x[source], 0.0)  # [block, token, head, element]
        scales = s[name + "_scale"]
        old = torch.where(kept[:, 0, None], scales[where, :, at[:, 0] % page // block], 0.0)  # [block, head]
        top = value.abs().amax((1, 3))
        _, e = torch.frexp(top / MOST[c["held"]])
        e = torch.where(top > 0, e - 1, -126).clamp(min=-126)
        need = ((e + 127) << 23).view(torch.float32)
        need = torch.where(top > need * MOST[c["held"]], need * 2, need)  # the least power of two that holds them
        scale = torch.where((old > 0) & (top <= old * MOST[c["held"]]), old, need)
        stale = cache[where[:, None], at % page].float() * old[:, None, :, None]
        value = torch.where(kept[..., None, None], stale, value) / scale[:, None, :, None]
        code = (value.round().clamp(-127, 127).to(torch.int8) if c["held"] == "i8" else value.to(torch.float8_e4m3fn)).view(torch.uint8)
        seen = (fresh | kept).nonzero(as_tuple=True)
        cache.view(torch.uint8)[where[seen[0]], at[seen] % page] = code[seen]
        some = real.nonzero(as_tuple=True)[0]
        scales[where[some], :, at[some, 0] % page // block] = scale[some]
    return _updated(s, q)


def _attend(s):
    c = s["case"]
    heads, kv, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group, n, most = heads // kv, c["n_seq"], s["most_new"]
    after, table = s["len"].long(), s["table"].long().clamp(min=0)
    keys = table.shape[1] * page

    def read(name):  # [sequence, key head, key, element]
        x = _by_token(s, s[name + "_cache"])[table].float()
        if c["held"] != "own":
            x = x * s[name + "_scale"][table].transpose(2, 3).repeat_interleave(c["block"], 2)[..., None]
        return x.reshape(n, keys, kv, dim).permute(0, 2, 1, 3).contiguous()

    # the rows of each sequence, the last ones of `most`
    new = (s["ptr"][1:] - s["ptr"][:-1]).long()
    i = torch.arange(most, device="cuda")
    there = i >= (most - new)[:, None]
    row = torch.where(there, s["ptr"][1:, None].long() - most + i, 0)
    q = s["q"].float()[row].view(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim)
    pos = (after[:, None] - most + i)[:, :, None]
    j = torch.arange(keys, device="cuda")[None, None, :]
    seen = (j <= pos) & there[:, :, None]
    if c["left"] >= 0:
        seen = seen & (j >= pos - c["left"])
    score = torch.matmul(q, read("k").transpose(2, 3)).mul_(s["scale"]).view(n, kv, group, most, keys)
    if c["cap"]:
        score = score.div_(c["cap"]).tanh_().mul_(c["cap"])
    if c["bias"]:
        score = score - s["slopes"].view(1, kv, group, 1, 1) * (pos - j).abs().float()[:, None, None]
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = score.sub_(torch.where(torch.isfinite(top), top, 0.0)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, 1.0))
    out = torch.matmul(p.view(n, kv, group * most, keys), read("v")).view(n, kv, group, most, dim).permute(0, 3, 1, 2, 4)
    return dict(out=out.reshape(n, most, heads, dim)[there].to(s["q"].dtype))


def run(state):
    if own:
        return _run_own(state)
    return _append(state) if state["case"]["op"] == "append" else _attend(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _power(e):
    """2^e in 64 bits, exactly (as a function it may be off by its last bit)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes(x, held):
    """Values in steps of the scale to the nearest that a code stands for."""
    if held == "i8":
        return torch.sign(x) * torch.where((x.abs() % 1 == 0.5) & (x.abs().floor() % 2 == 0), x.abs().floor(), (x.abs() + 0.5).floor())
    _, e = torch.frexp(x)
    step = _power((e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    half, most = case["rot"] // 2, MOST.get(case["held"], 1.0)
    first = torch.arange(half, device="cuda") * (1 if case["layout"] == "half" else 2)
    second = first + (half if case["layout"] == "half" else 1)
    q, caches = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), {}
    for name in "kv":
        caches[name] = _by_token(s, s[name + "_cache"].double().clone())
        caches[name + "_scale"] = s[name + "_scale"].double().clone() if case["held"] != "own" else None
    begin_row = 0
    for b, (new, after) in enumerate(_sequences(case)):
        at = slice(begin_row, begin_row + new)
        begin_row += new
        angle = torch.arange(after - new, after, device="cuda").double()[:, None, None] * s["freq"]
        unit = torch.polar(torch.ones_like(angle), angle)

        def turned(x):
            y = x.double().clone()
            z = torch.complex(y[..., first], y[..., second]) * unit
            y[..., first], y[..., second] = z.real, z.imag
            return y

        q[at] = turned(s["q"][at])
        for name, x in (("k", turned(s["k"][at]).float().double()), ("v", s["v"][at].double())):
            pages = s["table"][b].long()
            to = torch.arange(after - new, after, device="cuda")
            if case["held"] == "own":
                caches[name][pages[to // case["page"]], to % case["page"]] = x
                continue
            # all of the sequence from the first touched block on, as whole blocks: zeros behind its end
            start = (after - new) // case["block"] * case["block"]
            kept, blocks = after - new - start, -(-(after - start) // case["block"])
            at_all = start + torch.arange(blocks * case["block"], device="cuda")
            page, place = pages[at_all.clamp(max=after - 1) // case["page"]], at_all % case["page"]
            block_page, block_at = page.view(blocks, -1)[:, 0], place.view(blocks, -1)[:, 0] // case["block"]
            full = torch.zeros(blocks * case["block"], case["kv_heads"], case["dim"], dtype=torch.float64, device="cuda")
            full[kept: kept + new] = x
            top = full.view(blocks, case["block"], case["kv_heads"], -1).abs().amax((1, 3))
            part, e = torch.frexp(top / most)
            scale = _power(torch.where(top > 0, torch.where(part == 0.5, e - 1, e), -126).clamp(min=-126))
            if kept:
                before = caches[name + "_scale"][block_page[0], :, block_at[0]]
                full[:kept] = caches[name][page[:kept], place[:kept]] * before[:, None]
                scale[0] = torch.where(top[0] <= before * most, before, scale[0])
            code = _codes(full / scale.repeat_interleave(case["block"], 0)[..., None], case["held"])
            caches[name][page[: kept + new], place[: kept + new]] = code[: kept + new]
            caches[name + "_scale"][block_page, :, block_at] = scale
    r = dict(q=q)
    for name in "kv":
        r[name] = None if case["held"] == "i8" else _by_token(s, caches[name]).contiguous()
        if case["held"] != "own":
            r[name + "_scale"] = caches[name + "_scale"]
    return r


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, s)
    group, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (new, after) in enumerate(_sequences(case)):
        at = slice(begin, begin + new)
        begin += new
        lo = 0 if case["left"] < 0 else max(0, after - new - case["left"])
        j = torch.arange(lo, after, device="cuda")
        pages, place = s["table"][b].long()[j // page], j % page
        p = torch.arange(after - new, after, device="cuda")[:, None]
        hidden = (j > p) | ((j < p - case["left"]) if case["left"] >= 0 else torch.zeros_like(p, dtype=torch.bool))
        for c in range(case["kv_heads"]):
            k, v = (_by_token(s, s[name + "_cache"])[pages, place, c].double() for name in "kv")
            if case["held"] != "own":
                k, v = (x * s[name + "_scale"][pages, c, place // case["block"]].double()[:, None] for x, name in ((k, "k"), (v, "v")))
            for h in range(c * group, c * group + group):
                x = s["q"][at, h].double() @ k.T * s["scale"]
                if case["cap"]:
                    x = torch.tanh(x / case["cap"]) * case["cap"]
                if case["bias"]:
                    x = x - s["slopes"][h].double() * (p - j).abs()
                out[at, h] = torch.softmax(torch.where(hidden, -math.inf, x), 1) @ v
    return dict(out=out)
