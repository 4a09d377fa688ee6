"""Rotation tables and QK-norm + RoPE from multi-axis positions, against the formula in 64 bits.

Tolerances.  A turn is formed in 64 bits and rounded to 32 once: at most 2^-26 of a turn (values up to 1/2) and, for the
sums and products in 64 bits, below 1e-9 of one for the positions here: 9.5e-8 rad.  sincospi is within an ulp of 2^-24
near 1, so a table entry is within 9.5e-8 + 1.2e-7 < 3e-7.  A normed value carries the sum of squares (128 terms in
groups, under 12 roundings), a division, a square root, a division and two products, under 20 x 2^-24 = 1.2e-6
relative; with the rotation's two products, one sum and the table error under 2e-6 of the pair's length.  The result is
rounded to bf16 once: half a step, 2^-8 relative.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import bf16_array, device_ok, need_gpu, to_dev, to_np

pytestmark = pytest.mark.gpu

TABLE_TOL = 3e-7
PAIR_TOL = 2e-6


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()


def angles(pos, dims, theta):
    th = (theta,) * len(dims) if np.isscalar(theta) else theta
    return np.concatenate([pos[:, a:a + 1].astype(np.float64) * th[a] ** (-2.0 * np.arange(d // 2) / d)
                           for a, d in enumerate(dims)], 1)


def grid_positions(S, axes, seed, kind):
    rs = np.random.RandomState(seed)
    if kind == "far":
        return rs.randint(-1_000_000, 1_000_000, (S, axes)).astype(np.int64)
    if kind == "frac":
        return (rs.rand(S, axes) * 1000).astype(np.float32)
    i = np.arange(S)
    return np.stack([i // 63, (i // 9) % 7, i % 9, i % 5], 1)[:, :axes].astype(np.int32)


@pytest.mark.parametrize("S,dims,theta,kind", [
    (1, (44, 42, 42), 10000.0, "grid"), (333, (32, 32, 32), 10000.0, "grid"), (37, (128,), 1e6, "far"),
    (1001, (44, 42, 42), (10000.0, 256.0, 100.0), "frac"), (5, (2,), 10000.0, "far"), (70, (2, 6, 10, 30), 500.0, "frac"),
    (4097, (64, 64), 10000.0, "far"), (37760, (44, 42, 42), 10000.0, "frac"),
])
def test_table(S, dims, theta, kind):
    from tfvideo import kernels as K

    pos = grid_positions(S, len(dims), S, kind)
    got = to_np(K.rope_axes(torch.from_numpy(pos).cuda(), dims, theta)).astype(np.float64)
    a = angles(pos, dims, theta)
    ref = np.stack([np.stack([np.cos(a), -np.sin(a)], -1), np.stack([np.sin(a), np.cos(a)], -1)], -2)
    assert got.shape == ref.shape
    assert np.abs(got - ref).max() <= TABLE_TOL
    device_ok()


def test_table_strided_positions_and_out():
    from tfvideo import kernels as K

    pos = grid_positions(300, 3, 1, "grid")
    ref = K.rope_axes(torch.from_numpy(pos).cuda(), (32, 32, 32))
    wide = torch.from_numpy(np.concatenate([pos, pos + 7], 1).T.copy()).cuda()   # [6, S]: the axes are rows
    out = torch.full((300, 48, 2, 2), 7.0, device="cuda")
    assert K.rope_axes(wide[:3].t(), (32, 32, 32), out=out) is out
    assert torch.equal(out, ref)
    assert torch.equal(K.rope_axes(wide.t()[::2, :3], (32, 32, 32)), ref[::2])
    assert K.rope_axes(wide[:3].t()[:0], (32, 32, 32)).shape == (0, 48, 2, 2)
    for t in (torch.int64, torch.float32):
        assert torch.equal(K.rope_axes(torch.from_numpy(pos).cuda().to(t), (32, 32, 32)), ref)


def norm_rope_ref(x, w, a, eps):
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w.astype(np.float64)
    h = a.shape[1]
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    o = y.copy()
    o[..., :h] = y[..., :h] * c - y[..., h:2 * h] * s
    o[..., h:2 * h] = y[..., :h] * s + y[..., h:2 * h] * c
    size = np.abs(y)
    size[..., :h] = size[..., h:2 * h] = np.hypot(y[..., :h], y[..., h:2 * h])
    return o, size


def check_norm_rope(got, x, w, a, eps):
    ref, size = norm_rope_ref(x, w, a, eps)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + PAIR_TOL * (1 + 2.0 ** -8) * size).all()


@pytest.mark.parametrize("S,Hq,Hk,dims,kind", [
    (1, 1, 1, (128,), "far"), (7, 4, 4, (32, 32, 32), "grid"), (333, 5, 5, (44, 42, 42), "frac"), (130, 20, 5, (64, 64), "grid"),
    (129, 1, 9, (8,), "grid"), (65, 40, 40, (44, 42, 42), "far"), (2049, 3, 2, (16, 24, 24), "frac"),
    (20, 6, 6, (64, 64), "grid"), (19, 7, 7, (32, 32, 32), "far"), (9, 3, 3, (16, 24, 24), "frac"), (4000, 8, 8, (128,), "far"),
    (3, 23, 23, (44, 42, 42), "grid"), (700, 17, 4, (64, 64), "frac"), (77, 2, 31, (32, 32, 32), "grid"),
])
def test_qknorm_rope_axes(S, Hq, Hk, dims, kind):
    from tfvideo import kernels as K

    x = bf16_array((S, Hq + 2 * Hk, 128), seed=S, scale=3.0)
    rs = np.random.RandomState(2)
    qw, kw = (1 + 0.1 * rs.randn(128)).astype(np.float32), (1 + 0.1 * rs.randn(128)).astype(np.float32)
    pos = grid_positions(S, len(dims), S, kind)
    a = angles(pos, dims, 10000.0)
    t, p = to_dev(x), torch.from_numpy(pos).cuda()
    q, k = t[:, :Hq], t[:, Hq:Hq + Hk]
    args = (to_dev(qw, torch.float32), to_dev(kw, torch.float32), p, dims)
    oq, ok = K.qknorm_rope_axes(q, k, *args, out_q=torch.empty_like(q), out_k=torch.empty_like(k))
    assert np.array_equal(to_np(t), x)                                  # inputs left as they were
    check_norm_rope(to_np(oq), x[:, :Hq], qw, a, 1e-5)
    check_norm_rope(to_np(ok), x[:, Hq:Hq + Hk], kw, a, 1e-5)
    iq, ik = K.qknorm_rope_axes(q, k, *args)                            # in place: the same bits, v untouched
    assert iq is q and ik is k
    assert torch.equal(t[:, :Hq], oq) and torch.equal(t[:, Hq:Hq + Hk], ok)
    assert np.array_equal(to_np(t[:, Hq + Hk:]), x[:, Hq + Hk:])
    device_ok()


def test_qknorm_rope_axes_equals_the_table_path():
    """The same norms and rotation as norming with the table that rope_axes makes (h3_qknorm_rope): equal but for a
    rounding where the two order the arithmetic differently, so at most one bf16 step apart."""

    from tfvideo import kernels as K
    from tfvideo import native as N

    S, H, dims = 300, 6, (32, 32, 32)
    x = to_dev(bf16_array((S, 3 * H * 128), seed=4))
    pos = torch.from_numpy(grid_positions(S, 3, 0, "grid")).cuda()
    w = 1 + 0.1 * torch.randn(128, device="cuda")
    oq, ok = K.qknorm_rope_axes(x.view(S, 3 * H, 128)[:, :H], x.view(S, 3 * H, 128)[:, H:2 * H], w, w, pos, dims,
                                out_q=torch.empty((S, H, 128), dtype=torch.bfloat16, device="cuda"),
                                out_k=torch.empty((S, H, 128), dtype=torch.bfloat16, device="cuda"))
    table = K.rope_axes(pos, dims)
    N.qknorm_rope(x[:, :H * 128], x[:, H * 128:], 3 * H * 128, S, H, 96, w, w, table, 1e-5)
    for o, y in ((oq, x.view(S, 3 * H, 128)[:, :H]), (ok, x.view(S, 3 * H, 128)[:, H:2 * H])):
        d = (o.float() - y.float()).abs()
        assert (d <= 2.0 ** -7 * y.float().abs() + 1e-6).all()


def test_parts_of_one_buffer():
    """q, k and v of a head side by side: in place, and into the memory of the third part; [q | k | out] rows."""

    from tfvideo import kernels as K

    S, H, dims = 45, 5, (32, 32, 32)
    x = to_dev(bf16_array((S, H, 3, 128), seed=6))
    pos = torch.from_numpy(grid_positions(S, 3, 0, "grid")).cuda()
    w = 1 + 0.1 * torch.randn(128, device="cuda")
    q, k, v = (x[:, :, i].clone() for i in range(3))
    oq, ok = K.qknorm_rope_axes(q, k, w, w, pos, dims, out_q=torch.empty_like(q), out_k=torch.empty_like(k))
    y = x.clone()
    K.qknorm_rope_axes(y[:, :, 0], y[:, :, 1], w, w, pos, dims)
    assert torch.equal(y, torch.stack([oq, ok, v], 2))
    y = x.clone()
    K.qknorm_rope_axes(y[:, :, 0], y[:, :, 1], w, w, pos, dims, out_q=y[:, :, 2])
    assert torch.equal(y, torch.stack([q, ok, oq], 2))
    y = torch.cat([q, k, v], 1)
    K.qknorm_rope_axes(y[:, :H], y[:, H:2 * H], w, w, pos, dims, out_q=y[:, 2 * H:])
    assert torch.equal(y, torch.cat([q, ok, oq], 1))
    with pytest.raises(RuntimeError, match="overlap"):
        K.qknorm_rope_axes(y[:, :H], y[:, H:2 * H], w, w, pos, dims, out_q=y[:, 1:H + 1])
    assert torch.equal(y, torch.cat([q, ok, oq], 1))


def test_head_major_strides_zero_rows_and_non_finite_rows():
    """[H, S, 128] memory; a zero row stays zero (eps under the root); inf and NaN stay in their own head rows."""

    from tfvideo import kernels as K

    S, H = 50, 3
    x = bf16_array((H, S, 128), seed=9)
    x[1, 4] = 0.0
    t = to_dev(x)
    t[2, 7, 5] = float("nan")
    t[0, 7, 5] = float("inf")
    w = torch.ones(128, device="cuda")
    pos = torch.arange(S, dtype=torch.int32, device="cuda")[:, None]
    q = t.transpose(0, 1)
    oq, ok = K.qknorm_rope_axes(q, q.clone(), w, w, pos, (128,), out_q=torch.empty_like(q))
    assert torch.equal(oq[~torch.isnan(oq)], ok[~torch.isnan(ok)])
    assert (oq[4, 1] == 0).all()
    bad = torch.isnan(oq).any(-1)
    assert bad.nonzero().tolist() == [[7, 0], [7, 2]]
    a = angles(np.arange(S)[:, None], (128,), 10000.0)
    good = to_np(oq)
    ref, size = norm_rope_ref(np.moveaxis(to_np(t), 0, 1), np.ones(128, np.float32), a, 1e-5)
    keep = ~np.isnan(ref).any(-1)
    keep[7, 0] = keep[7, 2] = False
    assert (np.abs(good - ref)[keep] <= (2.0 ** -8 * np.abs(ref) + 3e-6 * size)[keep]).all()


def test_on_a_side_stream_and_in_a_graph():
    from tfvideo import kernels as K

    S, H, dims = 200, 4, (44, 42, 42)
    q, k = (to_dev(bf16_array((S, H, 128), seed=i)) for i in (1, 2))
    pos = torch.from_numpy(grid_positions(S, 3, 0, "frac")).cuda()
    w = torch.ones(128, device="cuda")
    e = dict(dtype=torch.bfloat16, device="cuda")
    ref = K.qknorm_rope_axes(q, k, w, w, pos, dims, out_q=torch.empty((S, H, 128), **e), out_k=torch.empty((S, H, 128), **e))
    tab = K.rope_axes(pos, dims)
    oq, ok, ot = torch.zeros((S, H, 128), **e), torch.zeros((S, H, 128), **e), torch.zeros_like(tab)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        K.rope_axes(pos, dims, out=ot)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(ot, tab)
    with torch.cuda.graph(g):
        K.qknorm_rope_axes(q, k, w, w, pos, dims, out_q=oq, out_k=ok)
        K.rope_axes(pos, dims, out=ot)
    assert not oq.any()
    pos += 3                                    # the graph reads the positions when it is replayed
    g.replay()
    moved = K.qknorm_rope_axes(q, k, w, w, pos, dims, out_q=torch.empty((S, H, 128), **e), out_k=torch.empty((S, H, 128), **e))
    assert torch.equal(oq, moved[0]) and torch.equal(ok, moved[1]) and torch.equal(ot, K.rope_axes(pos, dims))
    assert not torch.equal(oq, ref[0])
