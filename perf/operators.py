"""Workloads of the dense attention entry points and of the rotary positions: what a user of this framework has them do.

A case is a dict of plain values.  "op" says which calls one pass makes:
  prompt   attention over the tokens of packed sequences, forward only
  train    the same with log-sum-exp kept, and the gradients of queries, keys, values (and of the bias slopes)
  token    the newest tokens of every sequence against its cache of keys and values (padded caches, a length each)
  shared   the same where all sequences begin with one prefix, whose keys and values exist once
  rotary   rotary positions of queries and keys, "inverse" for their gradients
"type" is the element type, "heads" query heads share "kv_heads" key heads of "dim" elements.  The lengths of "n_seq"
sequences follow from the case alone: all of "length", or ragged ones that sum to "total" (token, shared: cache lengths of up
to "length").  "left" / "right" bound the visible keys around a row (-1: no bound), "prefix" is the share of a sequence's
first keys that all its rows see, "cap" the bound of the scores' tanh (0: none), "bias" a bias by distance with a slope for
each head.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # Local attention as the sparse path has it (16,384 tokens, 128 keys on either side, one head of 64, fp32).
        dict(name="window_f32_16k", op="prompt", type="f32", heads=1, kv_heads=1, dim=64, n_seq=1, length=16384, total=0, left=128, right=128, prefix=0.0, cap=0.0, bias=False),
        # A prompt with capped scores.
        dict(name="prompt_cap_4k", op="prompt", type="bf16", heads=16, kv_heads=4, dim=128, n_seq=1, length=4096, total=0, left=-1, right=0, prefix=0.0, cap=50.0, bias=False),
        # A long prompt, the largest number of operations.
        dict(name="prompt_16k", op="prompt", type="bf16", heads=16, kv_heads=2, dim=128, n_seq=1, length=16384, total=0, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # A training step on packed documents of uneven lengths.
        dict(name="train_documents_8k", op="train", type="bf16", heads=16, kv_heads=4, dim=128, n_seq=13, length=0, total=8192, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # A training step with a bidirectional prefix, in fp16, at odd lengths.
        dict(name="train_prefix_2k", op="train", type="f16", heads=12, kv_heads=12, dim=64, n_seq=3, length=0, total=5999, left=-1, right=0, prefix=0.3, cap=0.0, bias=False),
        # A small training step in fp32: bias by distance whose slopes are learnt, capped scores.
        dict(name="train_bias_f32", op="train", type="f32", heads=4, kv_heads=2, dim=32, n_seq=2, length=0, total=1013, left=-1, right=0, prefix=0.0, cap=30.0, bias=True),
        # One token of one user, a short cache: latency.
        dict(name="token_1", op="token", type="bf16", heads=32, kv_heads=8, dim=128, n_seq=1, tokens=1, length=1501, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # One token for each of 64 users with caches of uneven lengths: the caches have to be read.
        dict(name="tokens_64", op="token", type="bf16", heads=32, kv_heads=8, dim=128, n_seq=64, tokens=1, length=8192, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # A handful of users behind a short common instruction.
        dict(name="shared_4", op="shared", type="f16", heads=16, kv_heads=4, dim=64, n_seq=4, tokens=1, shared=1000, length=250, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # 48 answers to questions on one long document.
        dict(name="shared_48", op="shared", type="bf16", heads=32, kv_heads=8, dim=128, n_seq=48, tokens=1, shared=16000, length=700, left=-1, right=0, prefix=0.0, cap=0.0, bias=False),
        # The rotation of a decoding step: latency.
        dict(name="rotary_tokens", op="rotary", type="bf16", heads=32, kv_heads=8, dim=128, rows=64, rot=128, layout="half", scaling="bands", inverse=False),
        # The rotation of a long prompt, three quarters of each head, interleaved pairs, and the way back.
        dict(name="rotary_16k", op="rotary", type="bf16", heads=32, kv_heads=8, dim=128, rows=16384, rot=96, layout="interleaved", scaling="linear", inverse=True),
    ]


def _log_uniform(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case of the ranges above, at most the operations and bytes of the largest listed ones."""
    op = rng.choice(["prompt", "prompt", "train", "train", "token", "token", "shared", "rotary"])
    case = dict(op=op, type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    case["kv_heads"] = rng.choice([1, 2, 3, 4, 8])
    case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 5, 8])
    case["dim"] = rng.choice([32, 64, 64, 80, 96, 128, 128])
    if op == "rotary":
        rot = rng.choice([case["dim"], case["dim"] // 2])
        case.update(rows=int(_log_uniform(rng, 1, 16384)), rot=rot, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "bands", "parts"]), inverse=rng.random() < 0.4)
        return case
    case.update(left=-1, right=0, prefix=0.0, cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.25)
    if op in ("token", "shared"):
        case.update(n_seq=int(_log_uniform(rng, 1, 64)), tokens=rng.choice([1, 1, 1, 2, 4, 7]))
        # (the caches in elements: at most those of the largest case, and what their plain form holds in 32 bits)
        most = 64 * 8192 * 8 * 128 / (case["n_seq"] * case["kv_heads"] * case["dim"])
        most = min(most, 5.0e8 / (case["n_seq"] * case["heads"] * case["tokens"]), 32768.0)
        if op == "token":
            case["length"] = int(_log_uniform(rng, 16, most))
            if rng.random() < 0.2:
                case["left"] = int(_log_uniform(rng, 16, 1024))
        else:
            case["shared"] = int(_log_uniform(rng, 64, max(128.0, min(16000.0, most))))
            case["length"] = int(_log_uniform(rng, 16, max(32.0, min(700.0, most))))
        return case
    # (plain scores of at most half a billion elements in training, four in a prompt)
    rows_most = min(16384.0, math.sqrt((5.0e8 if op == "train" else 4.0e9) / case["heads"]))
    if case["type"] == "f32":
        rows_most = min(rows_most, 4096.0)
    rows = int(_log_uniform(rng, 64, rows_most))
    if rng.random() < 0.5:
        n_seq = rng.randint(2, max(2, min(24, rows // 32)))
        case.update(n_seq=n_seq, length=0, total=rows)
    else:
        case.update(n_seq=1, length=rows, total=0)
    mask = rng.choice(["causal", "causal", "window", "full", "prefix"])
    if mask == "window":
        case.update(left=int(_log_uniform(rng, 8, 512)), right=rng.choice([0, 0, int(_log_uniform(rng, 8, 512))]))
    elif mask == "full":
        case.update(right=-1)
    elif mask == "prefix":
        case.update(prefix=rng.uniform(0.1, 0.6))
    return case


# ---------------------------------------------------------------- what follows from a case alone

def _lengths(case):
    """Tokens of each sequence (token, shared: of each own cache, the newest tokens among them)."""
    rng = random.Random("%(n_seq)d %(length)d" % case + " %d" % case.get("total", 0))
    n = case["n_seq"]
    if case["op"] in ("token", "shared"):
        least = max(case["tokens"], case["length"] // 64, 1)
        return [case["length"]] + [max(least, int(case["length"] * rng.random())) for _ in range(n - 1)]
    if case["length"]:
        return [case["length"]] * n
    cuts = sorted(rng.sample(range(1, case["total"]), n - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [case["total"]])]


def _prefixes(case, lengths):
    return [int(case["prefix"] * n) for n in lengths]


def _ranges(case, n_rows, n_keys, prefix):
    """Positions of a sequence's rows and the keys each sees, [lo, hi), as numpy arrays."""
    pos = np.arange(n_keys - n_rows, n_keys)
    lo = np.zeros(n_rows, np.int64) if case["left"] < 0 else np.maximum(0, pos - case["left"])
    hi = np.full(n_rows, n_keys) if case["right"] < 0 else np.minimum(n_keys, np.maximum(pos + case["right"] + 1, prefix))
    return pos, lo, hi


def _sequences(case):
    """(rows, keys, prefix) of each sequence; keys count the shared ones."""
    lengths = _lengths(case)
    shared = case.get("shared", 0)
    return [(case.get("tokens") or n, n + shared, p) for n, p in zip(lengths, _prefixes(case, lengths))]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "rotary":
        rotated = case["rows"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * size * rotated * case["dim"] + 4 * case["rows"], "flops": 3 * rotated * case["rot"]}
    rows = keys = pairs = read = 0
    for n_rows, n_keys, prefix in _sequences(case):
        _, lo, hi = _ranges(case, n_rows, n_keys, prefix)
        pairs += int(np.maximum(0, hi - lo).sum())
        rows += n_rows
        keys += n_keys
        read += int(hi.max() - lo.min()) if case["op"] == "token" else n_keys
    if case["op"] == "shared":
        read = keys - (case["n_seq"] - 1) * case["shared"]
    dim, heads, kv = case["dim"], case["heads"], case["kv_heads"]
    passes = (2, 2) if case["op"] != "train" else (4, 4)
    bytes_ = size * dim * (passes[0] * rows * heads + passes[1] * read * kv)
    return {"bytes": bytes_, "flops": (14 if case["op"] == "train" else 4) * dim * pairs * heads}


# ---------------------------------------------------------------- inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    t = TYPES[case["type"]]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(t)

    if case["op"] == "rotary":
        rows = case["rows"]
        # a few sequences at positions of their own, up to those of a long context
        start = torch.randint(0, 120000, (1 + rows // 4096,), generator=g, device="cuda")
        at = torch.arange(rows, device="cuda")
        s = dict(case=case, q=normal(rows, heads, dim), k=normal(rows, kv, dim),
                 positions=(start[at // 4096] + at % 4096).to(torch.int32))
        s["freq"], s["amplitude"] = _frequencies(case)
        if own:
            _keep_rotary(s)
        return s
    lengths = _lengths(case)
    prefixes = _prefixes(case, lengths)
    s = dict(case=case)
    if case["op"] in ("prompt", "train"):
        total = sum(lengths)
        s.update(q=normal(total, heads, dim), k=normal(total, kv, dim), v=normal(total, kv, dim))
        s["ptr"] = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")
        if case["op"] == "train":
            s["grad"] = normal(total, heads, dim)
    else:
        n, tokens = case["n_seq"], case["tokens"]
        s.update(q=normal(n, tokens, heads, dim), k=normal(n, case["length"], kv, dim), v=normal(n, case["length"], kv, dim))
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        if case["op"] == "shared":
            s.update(shared_k=normal(case["shared"], kv, dim), shared_v=normal(case["shared"], kv, dim))
    s["prefix"] = torch.tensor(prefixes, dtype=torch.int32, device="cuda") if case["prefix"] else None
    s["slopes"] = None
    if case["bias"]:  # 2^(-8 h / heads), each a little off as a learnt one is
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, heads + 1, device="cuda") / heads) * (1 + 0.1 * torch.rand(heads, generator=g, device="cuda"))
    s["scale"] = dim ** -0.5
    s["max_len"] = max(lengths)
    if own:
        _keep_attention(s)
    return s


def _frequencies(case):
    """Radians a position of each pair in 64 bits, and the factor of the results, for contexts stretched four times."""
    half = case["rot"] // 2
    e = np.arange(half, dtype=np.float64)
    base, factor, amplitude, known = 10000.0, 4.0, 1.0, 8192.0
    if case["scaling"] == "base":
        base *= factor ** (case["rot"] / max(1, case["rot"] - 2))
    freq = base ** (-2 * e / case["rot"])
    if case["scaling"] == "linear":
        freq = freq / factor
    elif case["scaling"] == "bands":  # turns within the known length: more than 4 kept, fewer than 1 stretched
        mix = np.clip((known * freq / (2 * math.pi) - 1.0) / (4.0 - 1.0), 0, 1)
        freq = freq * (mix + (1 - mix) / factor)
    elif case["scaling"] == "parts":  # a ramp over the pairs between 32 turns and one
        at = [case["rot"] * math.log(known / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        lo, hi = max(0, math.floor(at[0])), min(case["rot"] - 1, math.ceil(at[1]))
        ramp = np.clip((e - lo) / max(hi - lo, 0.001), 0, 1)
        freq = freq * ((1 - ramp) + ramp / factor)
        amplitude = 0.1 * math.log(factor) + 1.0
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), amplitude


# ---------------------------------------------------------------- the framework's calls

def _type_of(case):
    from sddmm_gpu_amd import capi
    return {"f32": capi.TYPE_F32, "bf16": capi.TYPE_BF16, "f16": capi.TYPE_F16}[case["type"]]


def _keep_rotary(s):
    from sddmm_gpu_amd import capi
    c = s["case"]
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    freq, amplitude = capi.rotary_frequencies(c["rot"], 10000.0, dict(none=capi.ROTARY_PLAIN, linear=capi.ROTARY_LINEAR, base=capi.ROTARY_BASE,
                                              bands=capi.ROTARY_BANDS, parts=capi.ROTARY_PARTS)[c["scaling"]], 4.0, 8192,
                                              *dict(bands=(1.0, 4.0), parts=(1.0, 32.0)).get(c["scaling"], (0.0, 0.0)))
    s["own_freq"] = torch.from_numpy(freq).cuda()
    s["desc"] = capi.RotaryDesc.packed(_type_of(c), c["rows"], c["heads"], c["kv_heads"], c["dim"], c["rot"],
                                       capi.ROTARY_HALF if c["layout"] == "half" else capi.ROTARY_INTERLEAVED,
                                       inverse=int(c["inverse"]), amplitude=amplitude)


def _keep_attention(s):
    from sddmm_gpu_amd import capi
    c = s["case"]
    more = dict(window_left=c["left"], window_right=c["right"], scale=s["scale"], cap=c["cap"],
                prefix=s["prefix"].data_ptr() if s["prefix"] is not None else 0,
                slopes=s["slopes"].data_ptr() if s["slopes"] is not None else 0)
    if c["op"] in ("prompt", "train"):
        rows = s["q"].shape[0]
        more.update(q_ptr=s["ptr"].data_ptr(), k_ptr=s["ptr"].data_ptr(), q_rows=rows, k_rows=rows, max_q=s["max_len"], max_k=s["max_len"])
    else:
        more.update(max_q=c["tokens"], max_k=c["length"], k_len=s["lengths"].data_ptr(), shared_len=c.get("shared", 0))
    s["desc"] = d = capi.AttentionDesc.packed(_type_of(c), c["n_seq"], c["heads"], c["kv_heads"], c["dim"], **more)
    s["out"] = torch.empty_like(s["q"])
    need = capi.attention_workspace_bytes(d)[1 if c["op"] == "train" else 0]
    if c["op"] == "train":
        s["lse"] = torch.empty(s["q"].shape[:-1], dtype=torch.float32, device="cuda")
        s["dq"], s["dk"], s["dv"] = (torch.empty_like(s[n]) for n in "qkv")
        s["dslopes"] = torch.empty_like(s["slopes"]) if s["slopes"] is not None else None
        need = max(capi.attention_workspace_bytes(d))
    s["ws"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")


def _run_own(s):
    from sddmm_gpu_amd import capi
    stream = torch.cuda.current_stream().cuda_stream
    op, d = s["case"]["op"], s["desc"]
    if op == "rotary":
        capi.rotary(d, s["positions"].data_ptr(), s["own_freq"].data_ptr(), s["q"].data_ptr(), s["q_out"].data_ptr(),
                    s["k"].data_ptr(), s["k_out"].data_ptr(), stream)
        return dict(q=s["q_out"], k=s["k_out"])
    ws, n = s["ws"].data_ptr(), s["ws"].numel()
    q, k, v, out = s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr()
    if op == "shared":
        capi.attention_shared(d, q, s["shared_k"].data_ptr(), s["shared_v"].data_ptr(), k, v, out, 0, ws, n, stream)
        return dict(out=s["out"])
    if op != "train":
        capi.attention_forward(d, q, k, v, out, 0, ws, n, stream)
        return dict(out=s["out"])
    lse = s["lse"].data_ptr()
    capi.attention_forward(d, q, k, v, out, lse, ws, n, stream)
    more = s["dslopes"].data_ptr() if s["dslopes"] is not None else 0
    capi.attention_backward(d, q, k, v, out, lse, s["grad"].data_ptr(), s["dq"].data_ptr(), s["dk"].data_ptr(), s["dv"].data_ptr(), more, ws, n, stream)
    r = dict(out=s["out"], lse=s["lse"], dq=s["dq"], dk=s["dk"], dv=s["dv"])
    if more:
        r["dslopes"] = s["dslopes"]
    return r


# ---------------------------------------------------------------- the plain forms

def _rotate(x, cos, sin, rot, layout):
    y = x.float()
    if layout == "half":
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
    else:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
    p, q = a * cos - b * sin, a * sin + b * cos
    turned = torch.cat([p, q], -1) if layout == "half" else torch.stack([p, q], -1).flatten(-2)
    return torch.cat([turned, y[..., rot:]], -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freq"]
    sign = -1.0 if c["inverse"] else 1.0
    cos = (torch.cos(angle) * s["amplitude"]).float()[:, None, :]
    sin = (torch.sin(angle) * (sign * s["amplitude"])).float()[:, None, :]
    return dict(q=_rotate(s["q"], cos, sin, c["rot"], c["layout"]), k=_rotate(s["k"], cos, sin, c["rot"], c["layout"]))


def _places(s):
    """(position of each row, position of each key, which keys each row sees), with a leading dimension of the batch."""
    c = s["case"]
    if c["op"] in ("prompt", "train"):
        total, ptr = s["q"].shape[0], s["ptr"].long()
        at = torch.arange(total, device="cuda")
        of = torch.searchsorted(ptr, at, right=True) - 1  # the sequence of each token
        pos = at - ptr[of]
        rows, keys = pos[None, :, None], pos[None, None, :]
        seen = (of[:, None] == of[None, :])[None]
        most = torch.full_like(pos, total) if c["right"] < 0 else pos + c["right"]
        if s["prefix"] is not None:
            most = torch.maximum(most, s["prefix"].long()[of] - 1)
        most = most[None, :, None]
    else:
        shared, n = c.get("shared", 0), s["lengths"].long()
        rows = (shared + n[:, None] - c["tokens"] + torch.arange(c["tokens"], device="cuda"))[:, :, None]
        keys = torch.arange(shared + c["length"], device="cuda")[None, None, :]
        seen = keys < (shared + n)[:, None, None]
        most = rows + c["right"] if c["right"] >= 0 else torch.full_like(rows, shared + c["length"])
    seen = seen & (keys <= most)
    if c["left"] >= 0:
        seen = seen & (keys >= rows - c["left"])
    return rows, keys, seen


def _attention(s):
    c = s["case"]
    heads, kv, dim = c["heads"], c["kv_heads"], c["dim"]
    group = heads // kv
    q, k, v = s["q"], s["k"], s["v"]
    if c["op"] in ("prompt", "train"):
        q, k, v = q[None], k[None], v[None]
    elif c["op"] == "shared":
        k = torch.cat([s["shared_k"][None].expand(c["n_seq"], -1, -1, -1), k], 1)
        v = torch.cat([s["shared_v"][None].expand(c["n_seq"], -1, -1, -1), v], 1)
    n, nq, nk = q.shape[0], q.shape[1], k.shape[1]
    # [sequence, key head, the rows of its query heads, ...]
    q = q.float().reshape(n, nq, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * nq, dim)
    k = k.float().permute(0, 2, 1, 3).contiguous()
    v = v.float().permute(0, 2, 1, 3).contiguous()
    rows, keys, seen = _places(s)
    far = (rows - keys).abs().float()[:, None, None] if c["bias"] else None
    score = torch.matmul(q, k.transpose(2, 3)).mul_(s["scale"]).view(n, kv, group, nq, nk)
    bent = None
    if c["cap"]:
        score = score.div_(c["cap"]).tanh_()
        if c["op"] == "train":
            bent = 1 - score * score
        score = score * c["cap"]
    if c["bias"]:
        score = score - s["slopes"].view(1, kv, group, 1, 1) * far
    score = score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p.view(n, kv, group * nq, nk), v)

    def rows_of(x):
        return x.view(n, kv, group, nq, dim).permute(0, 3, 1, 2, 4).reshape(s["q"].shape).to(s["q"].dtype)

    if c["op"] != "train":
        return dict(out=rows_of(out))
    grad = s["grad"].float().reshape(n, nq, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * nq, dim)
    pf = p.view(n, kv, group * nq, nk)
    dv = torch.matmul(pf.transpose(2, 3), grad)
    ds = torch.matmul(grad, v.transpose(2, 3))
    ds = ds.sub_((grad * out).sum(-1, keepdim=True)).mul_(pf).view(n, kv, group, nq, nk)
    r = dict(out=rows_of(out), lse=(top + total.log())[0, ..., 0].permute(2, 0, 1).reshape(nq, heads).contiguous())
    if c["bias"]:
        r["dslopes"] = -(ds * far).double().sum((0, 3, 4)).reshape(heads).float()
    if bent is not None:
        ds = ds * bent
    ds = ds.mul_(s["scale"]).view(n, kv, group * nq, nk)
    r["dq"] = rows_of(torch.matmul(ds, k))
    r["dk"] = torch.matmul(ds.transpose(2, 3), q)[0].permute(1, 0, 2).to(s["k"].dtype).contiguous()
    r["dv"] = dv[0].permute(1, 0, 2).to(s["v"].dtype).contiguous()
    return r


def run(state):
    if own:
        return _run_own(state)
    return _rotary(state) if state["case"]["op"] == "rotary" else _attention(state)


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rotary(case, s):
    # pairs as complex numbers, turned by a unit number
    half = case["rot"] // 2
    angle = s["positions"].double()[:, None, None] * s["freq"] * (-1 if case["inverse"] else 1)
    unit = torch.polar(torch.full_like(angle, s["amplitude"]), angle)

    def turned(x):
        y = x.double().clone()
        first = torch.arange(half, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (half if case["layout"] == "half" else 1)
        z = torch.complex(y[..., first], y[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        return y

    return dict(q=turned(s["q"]), k=turned(s["k"]))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    heads, group, train = case["heads"], case["heads"] // case["kv_heads"], case["op"] == "train"
    packed = case["op"] in ("prompt", "train")
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if train:
        lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device="cuda")
        dq, dk, dv = (torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv")
        dslopes = torch.zeros(heads, dtype=torch.float64, device="cuda")
    begin = 0
    for b, (n_rows, n_keys, prefix) in enumerate(_sequences(case)):
        pos, lo, hi = (torch.from_numpy(x).cuda()[:, None] for x in _ranges(case, n_rows, n_keys, prefix))
        j = torch.arange(n_keys, device="cuda")[None, :]
        hidden = (j < lo) | (j >= hi)
        far = (pos - j).abs()
        for h in range(heads):
            c = h // group
            if packed:
                at = slice(begin, begin + n_rows)
                q, k, v = s["q"][at, h], s["k"][at, c], s["v"][at, c]
            else:
                q, k, v = s["q"][b, :, h], s["k"][b, : n_keys - case.get("shared", 0), c], s["v"][b, : n_keys - case.get("shared", 0), c]
                if case["op"] == "shared":
                    k, v = torch.cat([s["shared_k"][:, c], k]), torch.cat([s["shared_v"][:, c], v])
            q, k, v = q.double(), k.double(), v.double()
            x = q @ k.T * s["scale"]
            slope = 1.0
            if case["cap"]:
                bent = torch.tanh(x / case["cap"])
                slope, x = 1 - bent ** 2, bent * case["cap"]
            if case["bias"]:
                x = x - s["slopes"][h].double() * far
            x = torch.where(hidden, -math.inf, x)
            z = torch.logsumexp(x, 1, keepdim=True)
            p = torch.exp(x - z)
            o = p @ v
            if not packed:
                out[b, :, h] = o
                continue
            out[at, h] = o
            if train:
                do = s["grad"][at, h].double()
                lse[at, h] = z[:, 0]
                dv[at, c] += p.T @ do
                ds = p * (do @ v.T - (do * o).sum(1, keepdim=True))
                dslopes[h] -= (ds * far).sum()
                ds = ds * slope * s["scale"]
                dq[at, h] = ds @ k
                dk[at, c] += ds.T @ q
        begin += n_rows
    if not train:
        return dict(out=out)
    r = dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)
    if case["bias"]:
        r["dslopes"] = dslopes
    return r
