"""attention_f16 takes q, k, v as views with explicit strides: what it reads lies in the tensors' storage, or the call is refused.

The check is on the host and the same for meta tensors, so the refusals are tested there."""
import math

import pytest
import torch

B, H, N, D = 2, 2, 50, 64
C = H * D


def _mi():
    import MultiScaleDeformableAttention  # noqa: F401  (registers the ops)
    return torch.ops.ovis_mi


def _call(q, k, v, q_ld=3 * C, k_ld=3 * C, v_ld=3 * C, Nq=N, Nk=N, batch=B):
    return _mi().attention_f16(q, k, v, batch, H, Nq, Nk, D, Nq * q_ld, q_ld, Nk * k_ld, k_ld, Nk * v_ld, v_ld)


def _meta(*shape):
    return torch.empty(*shape, dtype=torch.float16, device="meta")


def test_views_of_one_buffer_and_copies_of_them_are_taken():
    qkv = _meta(B * N, 3 * C)
    assert _call(qkv, qkv[:, C:], qkv[:, 2 * C:]).shape == (B, N, C)
    assert _call(qkv, qkv[:, C:].clone(), qkv[:, 2 * C:].clone()).shape == (B, N, C)      # dense copies: their own strides
    assert _call(_meta(B * N, C), _meta(B * N, C), _meta(B * N, C), C, C, C).shape == (B, N, C)
    assert _call(_meta(N * (C + 8))[8:].as_strided((N, C), (C + 8, 1), 8), *([_meta(N, C)] * 2), C + 8, C, C, batch=1).shape == (1, N, C)


def test_strides_that_leave_the_storage_are_refused():
    ok = _meta(B * N, C)
    short, flat = _meta(B * N - 1, C), _meta(B * N * C)
    bad = [lambda: _call(short, ok, ok, C, C, C), lambda: _call(ok, short, ok, C, C, C), lambda: _call(ok, ok, short, C, C, C),
           lambda: _call(ok, flat, ok, C, 3 * C, C), lambda: _call(ok, ok, flat[1:], C, C, C), lambda: _call(ok, ok, ok, C, -C, C),
           lambda: _call(ok, ok, ok, C, C, 1 << 40), lambda: _call(ok, ok.float(), ok, C, C, C), lambda: _call(ok, ok, ok, C, C, C, Nk=0),
           lambda: _call(ok, ok, ok, C, C, C, batch=1 << 62), lambda: _call(ok, ok[:, 1:], ok, C, 3 * C, C)]
    for f in bad:
        with pytest.raises(RuntimeError, match="attention_f16"):
            f()


@pytest.mark.gpu
def test_copies_of_views_give_the_views_result():
    """the last copy ends where its storage does: with the buffer's strides the kernel would read 25000 halfs behind it"""
    qkv = torch.randn(B * N, 3 * C, generator=torch.Generator().manual_seed(3)).half().cuda()
    want = _call(qkv, qkv[:, C:], qkv[:, 2 * C:])
    copies = [qkv[:, i * C:].clone() for i in range(3)]
    assert torch.equal(_call(*copies), want)
    q, k, v = (t.double().cpu().view(B, N, H, D).transpose(1, 2) for t in qkv.split(C, 1))
    ref = ((q @ k.transpose(2, 3)) / math.sqrt(D)).softmax(-1) @ v
    # probabilities and the output are rounded to fp16 (2^-11 each, of values of at most 4.5); their f32 sums are far finer
    assert (want.double().cpu().view(B, N, H, D).transpose(1, 2) - ref).abs().max() < 4.5 * 2.0 ** -10 * 1.1
    with pytest.raises(RuntimeError, match="does not hold"):
        _call(qkv[1:], qkv[1:, C:], qkv[1:, 2 * C:])
