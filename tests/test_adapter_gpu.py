"""Low-rank adapters of several requests beside a projection, against the formula in 64 bits.

Tolerance, element by element: with t = scale A x and its rounding to bf16 (half a step, 2^-8 relative),
|error| <= (2^-8 + 2^-22) sum_r |t_r| |B_nr| + K 2^-24 |scale| sum_r (sum_k |A_rk| |x_k|) |B_nr| (fp32 sums over K)
+ 2^-8 |out| (the result's rounding), times 1 + 2^-7 for the products of these.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from helpers import device_ok, need_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()


def make(M, K, N, R, n, seed=0, kind="runs"):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, f=1.0: (torch.randn(s, generator=g, device="cuda") * f).to(torch.bfloat16)   # noqa: E731
    x, y, A, B = r(M, K), r(M, N), r(n, R, K, f=K ** -0.5), r(n, N, R, f=R ** -0.5)
    scale = torch.rand(n, generator=g, device="cuda") + 0.5
    rs = np.random.RandomState(seed)
    if kind == "one":
        rows = np.full(M, n - 1)
    elif kind == "none":
        rows = np.full(M, -1)
    elif kind == "runs":
        rows = np.sort(rs.randint(-1, n, M))
    elif kind == "back":                            # runs in falling order, and some of an adapter twice
        rows = np.concatenate([np.sort(rs.randint(-1, n, M - M // 3))[::-1], np.sort(rs.randint(-1, n, M // 3))])
    else:                                           # any order, entries outside [0, n) among them
        rows = rs.choice(np.array(list(range(n)) + [-1, -7, n, 2 ** 31 - 1, -2 ** 31]), M)
    return x, y, A, B, torch.from_numpy(rows.astype(np.int32)).cuda(), scale


def check(out, x, y, A, B, rows, scale=None):
    n = A.shape[0]
    K = x.shape[1]
    for i in sorted(set(rows.tolist())):
        at = (rows == i).nonzero()[:, 0]
        if not 0 <= i < n:
            assert torch.equal(out[at].view(torch.int16), y[at].view(torch.int16))
            continue
        s = 1.0 if scale is None else scale[i].double()
        xa, a, b = x[at].double(), A[i].double(), B[i].double()
        t = s * (xa @ a.T)
        ref = y[at].double() + t @ b.T
        size = s * (xa.abs() @ a.abs().T)
        tol = ((2.0 ** -8 + 2.0 ** -22) * (t.abs() @ b.abs().T) + K * 2.0 ** -24 * (size @ b.abs().T)) * (1 + 2.0 ** -7) \
            + 2.0 ** -8 * ref.abs()
        over = (out[at].double() - ref).abs() - tol
        assert (over <= 0).all(), f"adapter {i}: {(over > 0).sum().item()} elements off, worst by {over.max().item():.3g}"


@pytest.mark.parametrize("M,K,N,R,n,kind", [
    (1, 8, 8, 8, 1, "one"), (1, 5120, 15360, 16, 3, "runs"), (5, 72, 136, 24, 2, "any"), (127, 64, 64, 16, 1, "one"),
    (128, 512, 512, 64, 4, "runs"), (129, 520, 264, 128, 3, "any"), (333, 512, 512, 16, 1, "one"), (300, 256, 384, 8, 130, "any"),
    (1000, 1024, 1000, 72, 5, "any"), (640, 2048, 256, 112, 2, "runs"), (500, 128, 200, 40, 3, "none"),
    (4096, 5120, 1280, 64, 4, "runs"), (20000, 512, 384, 32, 7, "any"), (257, 20480, 520, 96, 2, "any"),
    (2048, 64, 72, 8, 2, "any"), (2049, 64, 72, 8, 2, "any"), (5000, 136, 200, 24, 300, "any"), (4100, 64, 64, 16, 5000, "any"),
    (16, 5120, 1024, 64, 6, "any"), (130, 512, 512, 16, 1, "any"), (6000, 256, 136, 40, 3, "runs"), (700, 64, 128, 128, 2, "none"),
    (3000, 200, 264, 16, 3, "back"), (300, 64, 64, 8, 20, "back"), (4500, 72, 136, 16, 9, "back"),
])
def test_adapter_add(M, K, N, R, n, kind):
    from tfvideo import linear as L

    x, y, A, B, rows, scale = make(M, K, N, R, n, seed=M + R, kind=kind)
    before = y.clone()
    out = L.adapter_add(y, x, A, B, rows, scale, out=torch.full_like(y, 7.0))
    assert torch.equal(y, before)
    check(out, x, y, A, B, rows, scale)
    again = L.adapter_add(y, x, A, B, rows, scale, out=torch.empty_like(y))
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    mine = L.adapter_add(y, x, A, B, rows, scale)                 # in place: the same bits
    assert mine is y and torch.equal(y.view(torch.int16), out.view(torch.int16))
    check(L.adapter_add(before, x, A, B, rows, out=torch.empty_like(y)), x, before, A, B, rows)
    device_ok()


def test_rows_without_an_adapter_keep_their_bits():
    from tfvideo import linear as L

    x, y, A, B, rows, scale = make(300, 128, 256, 16, 2, kind="any")
    none = (rows < 0) | (rows >= 2)
    assert none.any() and not none.all()
    bits = y.view(torch.int16)
    bits[none] = torch.randint(-2 ** 15, 2 ** 15, (int(none.sum()), 256), dtype=torch.int16, device="cuda")   # NaN, -0 too
    x[none] = float("nan")
    for out in (torch.empty_like(y), None):
        ref = y.clone()
        o = L.adapter_add(y, x, A, B, rows, scale, out=out)
        assert torch.equal(o.view(torch.int16)[none], ref.view(torch.int16)[none])
        check(o, x, ref, A, B, rows, scale)


def test_requests_do_not_reach_each_other():
    """Non-finite weights, inputs or scales of one adapter's rows leave every other row as it was."""

    from tfvideo import linear as L

    x, y, A, B, rows, scale = make(400, 512, 384, 32, 3, kind="any")
    clean = L.adapter_add(y, x, A, B, rows, scale, out=torch.empty_like(y))
    A2, B2, x2, s2 = A.clone(), B.clone(), x.clone(), scale.clone()
    A2[1], B2[1], s2[1] = float("nan"), float("inf"), float("inf")
    x2[rows == 1] = float("-inf")
    x2[7] = float("nan")
    o = L.adapter_add(y, x2, A2, B2, rows, s2, out=torch.empty_like(y))
    same = rows != 1
    same[7] = False
    assert torch.equal(o[same], clean[same])
    assert torch.isnan(o[rows == 1]).all()


def test_strides_views_and_offsets_past_32_bits():
    from tfvideo import linear as L

    x, y, A, B, rows, scale = make(200, 256, 384, 16, 2)
    ref = L.adapter_add(y, x, A, B, rows, scale, out=torch.empty_like(y))
    wide = torch.full((200, 640), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 128:512] = y
    L.adapter_add(wide[:, 128:512], x, A, B, rows, scale)
    assert torch.equal(wide[:, 128:512], ref) and (wide[:, :128] == 7).all() and (wide[:, 512:] == 7).all()
    odd = torch.empty((200, 260), dtype=torch.bfloat16, device="cuda")[:, 1:257]
    odd.copy_(x)
    t = A.transpose(1, 2).contiguous().transpose(1, 2)
    spread = torch.stack([rows, rows], 1)[:, 0]
    assert torch.equal(L.adapter_add(y, odd, t, B, spread, scale, out=torch.empty_like(y)), ref)
    assert L.adapter_add(y[:0], x[:0], A, B, rows[:0]).shape == (0, 384)
    none = torch.empty_like(y)
    assert torch.equal(L.adapter_add(y, x, A[:0], B[:0], rows, scale[:0], out=none), y)
    M = 150_000                                                    # 2.3 billion elements between first and last row
    big = torch.empty((M, 15_360), dtype=torch.bfloat16, device="cuda")
    x, y, A, B, rows, scale = make(M, 64, 64, 8, 3, kind="any")
    big[:, 15_296:] = y
    L.adapter_add(big[:, 15_296:], x, A, B, rows, scale)
    check(big[:, 15_296:], x, y, A, B, rows, scale)
    device_ok()


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("kind", ["runs", "none", "any"])
def test_out_and_y_may_be_x(n, kind):
    """A square projection's input overwritten, by a call of its own memory or as y: every row's A x comes first."""

    from tfvideo import linear as L

    x, y, A, B, rows, scale = make(20_000, 1024, 1024, 16, n, seed=n, kind=kind)
    ref = L.adapter_add(y, x, A, B, rows, scale, out=torch.empty_like(y))
    over = x.clone()
    assert L.adapter_add(y, over, A, B, rows, scale, out=over) is over and torch.equal(over, ref)
    ref = L.adapter_add(x, x, A, B, rows, scale, out=torch.empty_like(y))
    check(ref, x, x, A, B, rows, scale)
    assert torch.equal(L.adapter_add(x, x, A, B, rows, scale), ref)
    both = torch.empty((400, 2048), dtype=torch.bfloat16, device="cuda")     # y and out side by side in one buffer
    both[:, :1024] = y[:400]
    L.adapter_add(both[:, :1024], y[:400], A, B, rows[:400], scale, out=both[:, 1024:])
    assert torch.equal(both[:, :1024], y[:400])
    check(both[:, 1024:], y[:400], y[:400], A, B, rows[:400], scale)
    device_ok()


def test_sets_of_mixed_ranks_and_interleaved_outputs():
    from tfvideo import linear as L

    g = torch.Generator().manual_seed(0)
    pairs = [(torch.randn((r, 256), generator=g) * 0.05, torch.randn((192, r), generator=g) * 0.2) for r in (4, 16, 9)]
    s = L.AdapterSet(pairs, [1.0, 0.5, -2.0])
    assert s.A.shape == (3, 16, 256) and s.B.shape == (3, 192, 16)
    x, y, _, _, rows, _ = make(300, 256, 192, 8, 3, kind="any")
    out = s.add(y, x, rows, out=torch.empty_like(y))
    check(out, x, y, s.A, s.B, rows, s.scale)
    il = s.interleaved16()
    swap = lambda t: t.view(300, 2, 6, 16).transpose(1, 2).reshape(300, 192).contiguous()    # noqa: E731
    assert torch.equal(il.add(swap(y), x, rows), swap(out))


def test_streams_and_graphs():
    from tfvideo import linear as L

    a, b = make(700, 512, 640, 16, 3, 1, "any"), make(900, 256, 512, 64, 2, 2, "runs")
    call = lambda t: L.adapter_add(t[1], t[0], *t[2:], out=torch.empty_like(t[1]))          # noqa: E731
    ra, rb = call(a), call(b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            oa = call(a)
        with torch.cuda.stream(s2):
            ob = call(b)
    torch.cuda.synchronize()
    assert torch.equal(oa, ra) and torch.equal(ob, rb)
    out = torch.zeros_like(a[1])
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        L.adapter_add(a[1], a[0], *a[2:], out=out)
    out2 = torch.zeros_like(b[1])
    with torch.cuda.graph(g2):
        L.adapter_add(b[1], b[0], *b[2:], out=out2)
    for _ in range(2):
        g1.replay(), g2.replay()
    assert torch.equal(out, ra) and torch.equal(out2, rb)
    a[4].fill_(1)                                                   # the graph reads rows when it is replayed
    g1.replay()
    assert torch.equal(out, call(a)) and not torch.equal(out, ra)
    device_ok()


def test_interleaved_swiglu():
    """act_kind 2 of h3_act: the SwiGLU of 16-column interleaved [gate | up] equals that of the halves, bit for bit."""

    from tfvideo import kernels as K
    from tfvideo import native as N

    g = torch.randn((130, 2, 96), device="cuda").to(torch.bfloat16)
    ref = K.swiglu(g.reshape(130, 192).contiguous())
    il = g.view(130, 2, 6, 16).transpose(1, 2).reshape(130, 192).contiguous()
    out, amax = torch.empty_like(ref), torch.zeros(1, device="cuda")
    N.act(il, out, N.ACT_SWIGLU16, amax.data_ptr())
    assert torch.equal(out, ref) and amax.item() == ref.float().abs().max().item()
