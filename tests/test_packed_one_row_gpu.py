"""Calls of one token (or one head) on views whose stride over that one entry no kernel could use: a row of a wider or
broadcast buffer.  The same bits as on contiguous memory, and nothing written beside the row."""

from __future__ import annotations

import pytest
import torch

from helpers import device_ok, need_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()


def rand(*s, seed=0):
    return torch.randn(s, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(torch.bfloat16)


def one_row(row, ld):
    """[1, n] holding ``row`` with token stride ld, and its guarded buffer."""

    buf = torch.full((row.shape[1] + 64,), 7.0, dtype=torch.bfloat16, device="cuda")
    v = buf.as_strided(row.shape, (ld, 1), 0)
    v.copy_(row)
    return v, buf


@pytest.mark.parametrize("ld", [0, 8, 131, 4099])
@pytest.mark.parametrize("n", [1, 3])
def test_adapter_row(ld, n):
    from tfvideo import linear as L

    x, y, A, B = rand(1, 64, seed=1), rand(1, 128, seed=2), rand(n, 8, 64, seed=3), rand(n, 128, 8, seed=4)
    rows = torch.tensor([n - 1], dtype=torch.int32, device="cuda")
    ref = L.adapter_add(y, x, A, B, rows, out=torch.empty_like(y))
    assert not torch.equal(ref, y)
    yv, ybuf = one_row(y, ld)
    ov, obuf = one_row(torch.zeros_like(y), ld)
    assert torch.equal(L.adapter_add(yv, one_row(x, ld)[0], A, B, rows, out=ov), ref) and torch.equal(yv, y)
    assert torch.equal(L.adapter_add(yv, x, A, B, rows), ref)
    assert (ybuf[128:] == 7).all() and (obuf[128:] == 7).all()
    device_ok()


@pytest.mark.parametrize("ld", [0, 8, 131, 4099])
def test_attention_output_row(ld):
    from tfvideo import attention as A

    q, k, v = (rand(1, 4, 128, seed=i) for i in (1, 2, 3))
    out, buf = one_row(torch.zeros((1, 512), dtype=torch.bfloat16, device="cuda"), ld)
    A.bf16_tokens(q, k, v, out)
    assert torch.equal(out, v.view(1, 512)) and (buf[512:] == 7).all()      # one key: its value, bit for bit
    device_ok()


@pytest.mark.parametrize("strides", [(0, 128), (131, 128), (4099, 128), (512, 3)])
def test_norm_and_rotation_of_one_token(strides):
    """Token strides of one token, or a head stride of one head, that are no multiple of four elements."""

    from tfvideo import kernels as K

    S, H = (1, 4) if strides[1] == 128 else (3, 1)
    x = rand(S, H, 128, seed=5)
    w, pos = torch.ones(128, device="cuda"), torch.arange(5, 5 + S, dtype=torch.int32, device="cuda")[:, None]
    e = torch.empty_like(x)
    ref = K.qknorm_rope_axes(x, x.clone(), w, w, pos, (64,), out_q=e, out_k=torch.empty_like(x))[0].clone()
    buf = [torch.full((3 * 512 + 64,), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    q, k, oq, ok = (b.as_strided(x.shape, (*strides, 1), 0) for b in buf)
    q.copy_(x), k.copy_(x)
    K.qknorm_rope_axes(q, k, w, w, pos, (64,), out_q=oq, out_k=ok)
    assert torch.equal(oq, ref) and torch.equal(ok, ref) and torch.equal(q, x)
    K.qknorm_rope_axes(q, k, w, w, pos, (64,))
    assert torch.equal(q, ref) and torch.equal(k, ref)
    reach = (S - 1) * strides[0] + 512 if S == 1 else (S - 1) * strides[0] + 128
    assert all((b[reach:] == 7).all() for b in buf)
    device_ok()
