"""sddmm_attention_* and sddmm_rotary at the most workgroups that a launch holds (less than 2^32 threads), and the refusal of more, before anything is launched."""
import pytest
import torch

from sddmm_gpu_amd import capi

A = 1 << 20  # an address: aligned, never read
FULL = (1 << 24) - 1  # workgroups of 256 threads


def desc(**kw):
    d = dict(type=capi.TYPE_F16, n_seq=1, n_heads=1, n_kv_heads=1, head_dim=8, max_q=1, max_k=1)
    d.update(kw)
    return capi.AttentionDesc.packed(**d)


def forward(d):
    capi.attention_forward(d, A, A, A, 2 * A, 0, A, 1 << 62)


def backward(d, dslopes=0):
    capi.attention_backward(d, A, A, A, A, A, A, 2 * A, 3 * A, 4 * A, dslopes, A, 1 << 62)


def shared(d):
    capi.attention_shared(d, A, A, A, A, A, 2 * A, 0, A, 1 << 62)


@pytest.mark.parametrize("call,d", [
    (forward, desc(n_seq=FULL + 1)), (backward, desc(n_seq=FULL + 1)),           # one row and one key each
    (forward, desc(n_seq=1 << 21, n_heads=8, n_kv_heads=8)),                     # key heads
    (backward, desc(n_seq=FULL + 1, max_q=0)),                                   # dk and dv alone
    (backward, desc(n_seq=FULL + 1, max_k=0)),                                   # dq alone
    (forward, desc(n_seq=1 << 19, max_q=1024, n_heads=4, n_kv_heads=4)),         # whole tiles: 8 of 128 rows
    (forward, desc(n_seq=(1 << 31) - 1)), (backward, desc(n_seq=(1 << 31) - 1, max_q=0, max_k=(1 << 30) - 1, n_heads=65536, n_kv_heads=65536)),
    (shared, desc(n_seq=FULL - 100, shared_len=100000)),                          # those of the sequences, and those of the shared keys beside them
    (shared, desc(n_seq=2, max_q=1 << 28, n_heads=2, shared_len=10)),            # the join of rows and heads
])
def test_more_than_a_launch_holds(call, d):
    with pytest.raises(capi.SddmmError, match="one launch") as e:
        call(d)
    assert e.value.code == capi.ERR_RANGE


def test_rotary_of_more_than_a_launch_holds():
    # (two rows of so many heads to a workgroup)
    for rows in (1 << 25, 1 << 39):
        with pytest.raises(capi.SddmmError, match="one launch") as e:
            capi.rotary(capi.RotaryDesc.packed(capi.TYPE_BF16, rows, 32, 8, 128, 128, capi.ROTARY_HALF), 0, A, A, 2 * A, 3 * A, 4 * A)
        assert e.value.code == capi.ERR_RANGE


@pytest.mark.gpu
def test_the_most_that_a_launch_holds():
    dev = "cuda:0"
    q, k, v, do = (torch.randn(FULL, 1, 1, 8, device=dev).half() for _ in range(4))
    out, dq, dk, dv = (torch.full_like(q, 7.0) for _ in range(4))
    lse = torch.empty(FULL, device=dev)
    d = desc(n_seq=FULL)
    n = max(capi.attention_workspace_bytes(d))
    ws = torch.empty(n + 256, dtype=torch.uint8, device=dev)
    p = [x.data_ptr() for x in (q, k, v, out, lse)]
    capi.attention_forward(d, *p, ws.data_ptr(), n)
    capi.attention_backward(d, *p, do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), 0, ws.data_ptr(), n)
    torch.cuda.synchronize()
    # one key: its probability is 1 and has no gradient but what dp and delta, two sums of the same 8 products in fp32, differ by; the step of fp16 at 0 is
    # 2^-24, half of which the gradient of the score and the results may be off by
    assert torch.equal(out, v) and torch.equal(dv, do)
    e, size = 2.0 ** -24, (do.float() * v.float()).abs().sum(-1, keepdim=True)
    for grad, of in ((dq, k), (dk, q)):
        assert (grad.float().abs() <= (16 * e * size + 2.0 ** -25) * d.scale * of.float().abs() * 1.01 + 2.0 ** -25).all()
