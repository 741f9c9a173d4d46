"""What sddmm_attention_* refuses, and what it says (no GPU needed: nothing is launched)."""
import pytest

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read


HUGE = dict(q_row=64, q_head=1 << 18, q_seq=1 << 34, o_row=64, o_head=1 << 18, o_seq=1 << 34)  # of 2^18 sequences of 2^12 rows of 65536 heads


def desc(**kw):
    d = dict(type=capi.TYPE_BF16, n_seq=2, n_heads=4, n_kv_heads=2, head_dim=64, max_q=100, max_k=100)
    d.update(kw)
    return capi.AttentionDesc.packed(**d)


def forward(d, q=A, k=A, v=A, out=A, lse=0, ws=A, n=1 << 40):
    capi.attention_forward(d, q, k, v, out, lse, ws, n)


BAD = [
    (dict(type=3), "unknown type"), (dict(type=-1), "unknown type"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=4), "head_dim"), (dict(head_dim=68), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(n_heads=5), "key heads"), (dict(n_heads=0), "key heads"), (dict(n_kv_heads=0), "key heads"), (dict(n_kv_heads=-2), "key heads"),
    (dict(n_seq=-1), "negative"), (dict(max_q=-1, q_seq=0, o_seq=0), "negative"), (dict(max_k=-5, k_seq=0, v_seq=0), "negative"), (dict(shared_len=-1), "negative"),
    (dict(window_left=-2), "window"), (dict(window_right=-7), "window"),
    (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(cap=-1.0), "cap"), (dict(cap=float("inf")), "cap"), (dict(cap=float("nan")), "cap"),
    (dict(cap=1e-16, scale=1.0), "too far apart"), (dict(cap=1e31, scale=1e20), "too far apart"), (dict(cap=1e16, scale=1.0), "too far apart"),
    (dict(q_ptr=A + 2, q_rows=200), "aligned"), (dict(k_len=A + 1), "aligned"), (dict(slopes=A + 2), "aligned"), (dict(prefix=A + 3), "aligned"),
    (dict(q_ptr=A, q_len=A), "lengths beside"), (dict(k_ptr=A, k_len=A), "lengths beside"),
    (dict(q_row=60), "strides"), (dict(k_row=63 * 4 + 1), "strides"), (dict(v_head=12), "strides"), (dict(o_row=1 << 23), "strides"),
    (dict(k_seq=4), "strides"), (dict(q_head=-64), "strides"), (dict(q_seq=-1024), "strides"),
]


@pytest.mark.parametrize("kw,says", BAD)
def test_descriptions(kw, says):
    for call in (forward, capi.attention_workspace_bytes):
        with pytest.raises(capi.SddmmError, match=says) as e:
            call(desc(**kw))
        assert e.value.code == capi.ERR_ARG


def test_sizes_beyond_positions():
    for kw in (dict(max_k=1 << 30, k_seq=64, v_seq=64), dict(n_seq=1 << 20, max_q=1 << 12, q_seq=64, o_seq=64), dict(q_ptr=A, q_rows=1 << 31)):
        with pytest.raises(capi.SddmmError, match="positions") as e:
            forward(desc(**kw))
        assert e.value.code == capi.ERR_RANGE
    with pytest.raises(capi.SddmmError, match="one launch") as e:
        forward(desc(n_seq=1 << 18, max_q=1 << 12, n_heads=65536, n_kv_heads=1, **HUGE))
    assert e.value.code == capi.ERR_RANGE


def test_pointers():
    for kw in (dict(q=0), dict(k=0), dict(v=0), dict(out=0)):
        with pytest.raises(capi.SddmmError, match="NULL device pointer"):
            forward(desc(), **kw)
    for kw in (dict(q=A + 8), dict(k=A + 2), dict(v=A + 4), dict(out=A + 8)):
        with pytest.raises(capi.SddmmError, match="16-byte aligned"):
            forward(desc(), **kw)
    with pytest.raises(capi.SddmmError, match="NULL description"):
        capi.check(capi.lib().sddmm_attention_forward(None, A, A, A, A, None, None, 0, None))


def test_results_must_not_overlap():
    for kw in (dict(o_head=0), dict(o_seq=0), dict(o_row=64), dict(o_seq=64), dict(o_head=32), dict(q_ptr=A, q_rows=200, o_head=0)):
        with pytest.raises(capi.SddmmError, match="overlap"):
            forward(desc(**kw))
    for kw in (dict(q_head=0), dict(k_seq=0), dict(v_head=0), dict(k_row=64), dict(q_seq=64)):
        with pytest.raises(capi.SddmmError, match="rows of a gradient overlap"):
            backward(desc(**kw))
    with pytest.raises(capi.SddmmError, match="lse"):
        forward(desc(), lse=A + 2)
    with pytest.raises(capi.SddmmError, match="lse"):
        backward(desc(), lse=A + 1)


def test_workspace():
    d = desc(n_seq=1, max_q=1, max_k=5000)
    need = capi.attention_workspace_bytes(d)[0]
    assert need > 0
    for kw in (dict(ws=0, n=need), dict(ws=A, n=need - 1), dict(ws=A + 16, n=need)):
        with pytest.raises(capi.SddmmError, match="workspace"):
            forward(d, **kw)
    assert capi.attention_workspace_bytes(desc(n_seq=600, max_q=200))[0] == 0


def test_shared():
    with pytest.raises(capi.SddmmError, match="sddmm_attention_shared"):
        forward(desc(shared_len=10))
    with pytest.raises(capi.SddmmError, match="packed"):
        capi.attention_shared(desc(shared_len=10, q_ptr=A, q_rows=200), A, A, A, A, A, A, 0, A, 1 << 40)
    for bad in ((0, A), (A, 0)):
        with pytest.raises(capi.SddmmError, match="NULL device pointer"):
            capi.attention_shared(desc(shared_len=10), A, *bad, A, A, A, 0, A, 1 << 40)
    with pytest.raises(capi.SddmmError, match="too many rows"):
        capi.attention_shared(desc(shared_len=10, n_seq=1 << 20, max_q=1 << 9, q_seq=64, o_seq=64, n_heads=1 << 12), A, A, A, A, A, A, 0, A, 1 << 40)


def test_nothing_to_do():
    # (returns before a launch, so also without a GPU)
    forward(desc(n_seq=0), q=0, k=0, v=0, out=0)
    forward(desc(max_q=0), q=0, k=0, v=0, out=0)
    forward(desc(q_ptr=A, q_rows=0), q=0, k=0, v=0, out=0)


def backward(d, q=A, k=A, v=A, out=A, lse=A, dout=A, dq=A, dk=A, dv=A, dslopes=0, ws=A, n=1 << 40):
    capi.attention_backward(d, q, k, v, out, lse, dout, dq, dk, dv, dslopes, ws, n)


def test_backward():
    for kw, says in BAD:
        with pytest.raises(capi.SddmmError, match=says):
            backward(desc(**kw))
    for name in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        with pytest.raises(capi.SddmmError, match="NULL device pointer"):
            backward(desc(), **{name: 0})
        if name != "lse":
            with pytest.raises(capi.SddmmError, match="16-byte aligned"):
                backward(desc(), **{name: A + 8})
    with pytest.raises(capi.SddmmError, match="slopes that are not there"):
        backward(desc(), dslopes=A)
    with pytest.raises(capi.SddmmError, match="sddmm_attention_shared"):
        backward(desc(shared_len=5))
    need = capi.attention_workspace_bytes(desc())[1]
    for kw in (dict(ws=0), dict(n=need - 1), dict(ws=A + 128)):
        with pytest.raises(capi.SddmmError, match="workspace"):
            backward(desc(), **kw)
    with pytest.raises(capi.SddmmError, match="one launch"):
        backward(desc(n_seq=1 << 18, max_q=1 << 12, n_heads=65536, n_kv_heads=1, **HUGE), n=1 << 62)
    backward(desc(n_seq=0), *[0] * 9)
    backward(desc(max_q=0, max_k=0), *[0] * 9)


def test_results_in_the_place_of_operands():
    for name in ("q", "k", "v"):
        with pytest.raises(capi.SddmmError, match="in an operand's place"):
            forward(desc(), **dict(dict(q=A, k=A, v=A, out=4 * A), **{name: 4 * A}))
    good = dict(q=A, k=2 * A, v=3 * A, out=4 * A, lse=5 * A, dout=6 * A, dq=7 * A, dk=8 * A, dv=9 * A)
    for result in ("dq", "dk", "dv"):
        for other in good:
            if other != result:
                with pytest.raises(capi.SddmmError, match="gradient's place"):
                    backward(desc(), **dict(good, **{result: good[other]}))
