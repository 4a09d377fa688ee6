"""Argument checks of the packed-batch operators (positions, span masks, adapters): every refusal comes before any CUDA
call, so they run without a GPU, through the Python entry points and through the C ABI."""

from __future__ import annotations

import ctypes

import pytest
import torch

FAKE = 1 << 20   # an aligned address that is never touched


@pytest.fixture(scope="module")
def lib():
    from tfvideo import native
    if not native.LIB_PATH.exists():
        from build import build
        build()
    return native.lib()


def _pos(**kw):
    from tfvideo import native as N

    d = dict(pos=FAKE, type=0, ld=3, axis_stride=1, axes=3, dims=(44, 42, 42), theta=(1e4, 1e4, 1e4))
    d.update(kw)
    p = N.H3Positions(pos=d["pos"], type=d["type"], ld=d["ld"], axis_stride=d["axis_stride"], axes=d["axes"])
    for i, v in enumerate(d["dims"]):
        p.dims[i] = v
    for i, v in enumerate(d["theta"]):
        p.theta[i] = v
    return p


@pytest.mark.parametrize("kw,word", [
    (dict(pos=None), "NULL"), (dict(type=3), "type"), (dict(pos=FAKE + 2), "misaligned"), (dict(axes=0), "axes"),
    (dict(axes=5), "axes"), (dict(dims=(44, 42, 41)), "even"), (dict(dims=(44, 0, 42)), "even"),
    (dict(dims=(64, 64, 2)), "even"), (dict(theta=(1e4, 0.0, 1e4)), "theta"),
    (dict(theta=(1e4, float("inf"), 1e4)), "theta"), (dict(theta=(1e4, float("nan"), 1e4)), "theta"),
])
def test_positions_refused_by_the_library(lib, kw, word):
    from tfvideo import native as N

    assert lib.h3_rope_axes(ctypes.byref(_pos(**kw)), 10, FAKE, None) < 0 and word in N.last_error()


def test_rope_entry_points_check_their_arguments(lib):
    from tfvideo import native as N

    p = ctypes.byref(_pos())
    assert lib.h3_rope_axes(None, 10, FAKE, None) == -1
    assert lib.h3_rope_axes(p, 0, FAKE, None) == -2 and "S" in N.last_error()
    assert lib.h3_rope_axes(p, 10, FAKE + 4, None) == -1 and "aligned" in N.last_error()

    def qk(q=FAKE, ldq=384, S=10, Hq=1, Hk=1, qw=FAKE, pos=p, oq=FAKE, hsq=128):
        return lib.h3_qknorm_rope_axes(q, ldq, hsq, FAKE, 384, 128, S, Hq, Hk, qw, FAKE, pos, 1e-5, oq, 384, 128, FAKE,
                                       384, 128, None)

    assert qk(q=None) == -1 and qk(oq=None) == -1
    assert qk(S=0) == -2 and qk(Hq=0) == -2 and qk(Hk=0) == -2
    assert qk(ldq=386) == -2 and "strides" in N.last_error()
    assert qk(q=FAKE + 4) == -1 and qk(qw=FAKE + 8) == -1
    assert qk(pos=ctypes.byref(_pos(dims=(44, 42, 40)))) == -2 and "multiple of 8" in N.last_error()   # rot 126


def test_outputs_over_other_memory_are_refused(lib):
    from tfvideo import native as N

    p, e = ctypes.byref(_pos()), 2   # bytes an element
    far = FAKE + (1 << 24)

    def qk(q=(FAKE, 768, 128), k=(FAKE + 256 * e, 768, 128), oq=(far, 256, 128), ok=(far + (1 << 20), 256, 128), H=2):
        return lib.h3_qknorm_rope_axes(*q, *k, 10, H, H, FAKE, FAKE, p, 1e-5, *oq, *ok, None)

    q, k = (FAKE, 768, 128), (FAKE + 256 * e, 768, 128)
    for oq, ok in ((k, q), (k, k), (q, q), ((FAKE + 8, 768, 128), k), (q, (far, 0, 128)), (q, (far, 256, 0)),
                   ((FAKE, 256, 128), k), (q, (FAKE + 128 * e, 768, 128)), ((FAKE - 256, 768, 128), k),
                   ((far, 256, 128), (far + 128 * e, 256, 128))):
        assert qk(oq=oq, ok=ok) in (-1, -2) and "overlap" in N.last_error(), (oq, ok)
    q3, k3 = (FAKE, 768, 384), (FAKE + 128 * e, 768, 384)         # q, k and v of a head side by side
    assert qk(q3, k3, q3, (FAKE + 192 * e, 768, 384)) == -1 and "overlap" in N.last_error()

    def attn(out, ldo):
        return lib.h3_attn_bf16(FAKE, 1024, 128, FAKE + 256 * e, 1024, 128, FAKE + 512 * e, 1024, 128, 10, 2, 2, None,
                                None, out, ldo, None, 0, None)

    for at, ldo in ((0, 1024), (256, 1024), (512, 1024), (640, 1024), (0, 256), (896, 1024), (9000, 256)):
        assert attn(FAKE + at * e, ldo) == -1 and "overlap" in N.last_error(), (at, ldo)

    def add(out, ldo, y=FAKE, ldy=512):
        return lib.h3_adapter_add(far, 64, y, ldy, far, far, None, far, 10, 64, 256, 16, 2, out, ldo, far,
                                  lib.h3_adapter_workspace_bytes(10, 16, 2), None)

    for at, ldo in ((0, 256), (8, 512), (248, 512), (4096, 512), (4608, 264)):
        assert add(FAKE + at * e, ldo) == -1 and "overlap" in N.last_error(), (at, ldo)


def test_rope_functions_refuse_bad_arguments():
    from tfvideo import kernels as K

    pos = torch.zeros((10, 3), dtype=torch.int32)
    for bad, dims, theta in ((pos[0], (32, 32, 32), 1e4), (pos.to(torch.int16), (32, 32, 32), 1e4),
                             (pos.double(), (32, 32, 32), 1e4), (pos, (32, 32), 1e4), (pos, (32, 31, 33), 1e4),
                             (pos, (64, 64, 64), 1e4), (pos, (32, 32, 32), 0.0), (pos, (32, 32, 32), (1e4, 1e4)),
                             (torch.zeros((10, 5), dtype=torch.int32), (8,) * 5, 1e4), (pos, (32, -2, 32), 1e4)):
        with pytest.raises(ValueError):
            K.rope_axes(bad, dims, theta)
        with pytest.raises(ValueError):
            K.AxialPositions(bad, dims, theta)
    with pytest.raises(ValueError, match="CUDA device"):
        K.rope_axes(pos, (32, 32, 32))
    with pytest.raises(ValueError, match="out"):
        K.rope_axes(pos, (32, 32, 32), out=torch.empty((10, 48, 2, 2), dtype=torch.float64))
    q = torch.zeros((10, 4, 128), dtype=torch.bfloat16)
    w = torch.ones(128)
    ok = dict(q=q, k=q, qw=w, kw=w, pos=pos, dims=(32, 32, 32))
    for change in (dict(q=q.float()), dict(q=q[:, :, :64]), dict(q=q[0]), dict(k=q[:9]), dict(pos=pos[:9]),
                   dict(dims=(32, 32, 30)), dict(qw=w[:64]), dict(out_q=q[:, :2]), dict(out_k=q.float()),
                   dict(q=torch.zeros((10, 128, 4), dtype=torch.bfloat16).transpose(1, 2)),
                   dict(q=torch.zeros(10 * 4 * 130, dtype=torch.bfloat16).as_strided((10, 4, 128), (520, 130, 1))),
                   dict()):                                                  # the last: CPU tensors
        with pytest.raises(ValueError):
            K.qknorm_rope_axes(**{**ok, **change})


def test_attn_bf16_checks_its_arguments(lib):
    from tfvideo import native as N

    def call(q=FAKE, ldq=384, hsq=128, ldk=384, S=10, Hq=2, Hk=1, lo=None, hi=None, out=FAKE, ldo=256, ws=None, size=0):
        return lib.h3_attn_bf16(q, ldq, hsq, FAKE, ldk, 128, FAKE, 384, 128, S, Hq, Hk, lo, hi, out, ldo, ws, size, None)

    assert call(q=None) == -1 and call(out=None) == -1
    assert call(lo=FAKE) == -1 and "half" in N.last_error()
    assert call(lo=FAKE + 2, hi=FAKE) == -1
    assert call(S=0) == -2 and call(S=262_145) == -2 and call(Hk=0) == -2 and call(Hq=3, Hk=2, ldo=384) == -2
    assert call(Hq=65_536, Hk=1, ldo=65_536 * 128) == -2
    assert call(ldo=128) == -2 and call(ldo=260) == -2
    assert call(ldq=0) == -2 and call(ldq=388) == -2 and call(hsq=-128) == -2 and call(ldk=-8) == -2
    assert call(q=FAKE + 8) == -1 and "16-byte" in N.last_error()
    need = lib.h3_attn_bf16_workspace_bytes(5000, 3)
    assert need >= 3 * 40 * 4 and lib.h3_attn_bf16_workspace_bytes(100, 3) == 0
    assert call(S=5000, Hq=3, Hk=3, ldo=384, ws=FAKE, size=need - 1) == -1 and "workspace" in N.last_error()
    assert call(S=5000, Hq=3, Hk=3, ldo=384, ws=FAKE + 4, size=need) == -1


def test_span_masks():
    from tfvideo import attention as A

    m = A.SpanMask.documents([3, 0, 2], 7, device="cpu")
    assert m.lo.tolist() == [0, 0, 0, 3, 3, 0, 0] and m.hi.tolist() == [3, 3, 3, 5, 5, 0, 0]
    m = A.SpanMask.frames([6, 2], 2, [1, 5], device="cpu")
    assert m.lo.tolist() == [0] * 6 + [6] * 2 and m.hi.tolist() == [1, 3, 3, 5, 5, 6, 8, 8]
    m = A.SpanMask.frames([4], 1, device="cpu")
    assert m.hi.tolist() == [1, 2, 3, 4]
    assert A.SpanMask.documents([], 0, device="cpu").S == 0
    for bad in (dict(lengths=[3, -1]), dict(lengths=[3], S=2)):
        with pytest.raises(ValueError):
            A.SpanMask.documents(**bad, device="cpu")
    for bad in (dict(lengths=[3], frame=-1), dict(lengths=[3], frame=1, prefix=-1), dict(lengths=[3], frame=1, prefix=[1, 2])):
        with pytest.raises(ValueError):
            A.SpanMask.frames(**bad, device="cpu")
    i = torch.zeros(4, dtype=torch.int32)
    for lo, hi in ((i.long(), i), (i, i.float()), (i[:3], i), (i[::2], i[::2]), (i[None], i[None])):
        with pytest.raises(ValueError):
            A.SpanMask(lo, hi)


def test_bf16_attention_refuses_bad_arguments():
    from tfvideo import attention as A

    q = torch.zeros((1, 4, 10, 128), dtype=torch.bfloat16)
    m = A.SpanMask.documents([9], device="cpu")
    for bad in ((q.float(), q, q), (q[0], q, q), (q[..., :64], q[..., :64], q[..., :64]), (q, q[:, :3], q[:, :3]),
                (q, q[:, :, :9], q[:, :, :9]), (q, q, q[:, :2]), (q, q[:, :0], q[:, :0]), (q, q, q, m),
                (q.expand(2, 4, 10, 128), q, q), (q, q, q)):                  # the last: CPU tensors
        with pytest.raises(ValueError):
            A.bf16(*bad)
    r, out = torch.zeros((10, 4, 128), dtype=torch.bfloat16), torch.zeros((10, 512), dtype=torch.bfloat16)
    for bad in ((r[0], r, r, out), (r, r[:9], r[:9], out), (r, r, r[:, :2], out), (r, r[:, :3], r[:, :3], out),
                (r, r, r, out[:, :256]), (r, r, r, out.float()), (r.float(), r, r, out), (r[:, :, :64], r, r, out),
                (r, r, r, out.t().contiguous().t()), (r, r, r, out, m), (r, r, r, out)):   # the last: CPU tensors
        with pytest.raises(ValueError):
            A.bf16_tokens(*bad)


def test_adapter_add_checks_its_arguments(lib):
    from tfvideo import native as N

    def call(x=FAKE, ldx=64, y=FAKE, ldy=64, rows=FAKE, M=10, K=64, N=64, R=16, n=2, out=FAKE, ldo=64, ws=FAKE, size=1 << 20):
        return lib.h3_adapter_add(x, ldx, y, ldy, FAKE, FAKE, None, rows, M, K, N, R, n, out, ldo, ws, size, None)

    for bad in (dict(x=None), dict(y=None), dict(rows=None), dict(out=None), dict(ws=None), dict(x=FAKE + 2),
                dict(out=FAKE + 8), dict(rows=FAKE + 1), dict(size=lib.h3_adapter_workspace_bytes(10, 16, 2) - 1)):
        assert call(**bad) == -1, bad
    for bad in (dict(M=0), dict(K=0), dict(K=60), dict(N=4), dict(R=0), dict(R=12), dict(R=136), dict(n=0), dict(n=2 ** 20 + 1), dict(ldx=56),
                dict(ldx=68), dict(ldy=56), dict(ldo=66)):
        assert call(**bad) == -2, bad
    assert lib.h3_adapter_workspace_bytes(10, 8, 1) >= 320 and lib.h3_adapter_workspace_bytes(0, 8, 1) == 0
    assert lib.h3_act(FAKE, 16, FAKE, 8, 4, 8, 2, None, None) == -2 and lib.h3_act(FAKE, 16, FAKE, 8, 4, 8, 3, None, None) == -1


def test_adapters_refuse_bad_arguments():
    from tfvideo import linear as L

    b = lambda *s: torch.zeros(s, dtype=torch.bfloat16)                     # noqa: E731
    good = dict(y=b(10, 64), x=b(10, 32), A=b(2, 8, 32), B=b(2, 64, 8), rows=torch.zeros(10, dtype=torch.int32))
    for bad in (dict(y=b(9, 64)), dict(y=b(10, 64).float()), dict(x=b(10, 40)), dict(A=b(8, 32)), dict(B=b(2, 64, 16)),
                dict(B=b(3, 64, 8)), dict(rows=torch.zeros(10)), dict(rows=torch.zeros(9, dtype=torch.int32)),
                dict(scale=torch.zeros(3)), dict(scale=torch.zeros(2, dtype=torch.float64)), dict(out=b(10, 72)),
                dict(out=b(10, 64).half()), dict(A=b(2, 4, 32), B=b(2, 64, 4)), dict(A=b(2, 136, 32), B=b(2, 64, 136)),
                dict(y=b(64, 10).t()), dict(y=b(10, 68)[:, :64]), dict(y=b(10, 72)[:, 1:65]),
                dict(out=b(1, 64).expand(10, 64)), dict()):                 # the last: CPU tensors
        with pytest.raises(ValueError):
            L.adapter_add(**{**good, **bad})
    for pairs, scales in (([], None), ([(b(4), b(64, 4))], None), ([(b(4, 32), b(64, 5))], None), ([(b(4, 32), b(64, 4)), (b(4, 40), b(64, 4))], None),
                          ([(b(130, 32), b(64, 130))], None), ([(b(4, 30), b(64, 4))], None), ([(b(4, 32), b(64, 4))], [1, 2])):
        with pytest.raises(ValueError):
            L.AdapterSet(pairs, scales, device="cpu")
    with pytest.raises(ValueError, match="32"):
        L.AdapterSet([(b(4, 32), b(48, 4))], device="cpu").interleaved16()
