"""bf16 attention under per-token key spans, against softmax attention in 64 bits.

Tolerance, element by element.  With A = sum_j p_j |v_j| (p the exact softmax row): P is rounded to bf16, half a step
2^-8 relative; exp2 is off by at most 7.5e-5 relative (polynomial; the hardware one 2^-22), in P and in the row sum; a
score's fp32 accumulation of 128 products by at most 128 x 2^-24 x sum |q k|, which moves p and the sum by twice that
over sqrt(128); the result is rounded to bf16 once, 2^-8 relative.  So
|error| <= (2^-8 + 2 x 7.5e-5 + 2 x 128 x 2^-24 x max_j sum |q k| / sqrt(128)) A (1 + 2^-7) + 2^-8 |o|.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from helpers import device_ok, need_gpu

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()


def rand(shape, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


def reference(q, k, v, lo=None, hi=None, rows=None):
    """(o, tolerance) float64 [H, rows, 128] for q [1, Hq, S, 128], k / v [1, Hk, S, 128]."""

    Hq, S = q.shape[1], q.shape[2]
    rows = torch.arange(S, device="cuda") if rows is None else rows
    j = torch.arange(S, device="cuda")
    keep = torch.ones((len(rows), S), dtype=torch.bool, device="cuda")
    if lo is not None:
        keep = (j >= lo[rows, None]) & (j < hi[rows, None])
    outs, tols = [], []
    for h in range(Hq):
        kh = h // (Hq // k.shape[1])
        qq, kk, vv = q[0, h, rows].double(), k[0, kh].double(), v[0, kh].double()
        s = (qq @ kk.T) / math.sqrt(128)
        s = torch.where(keep, s, -math.inf)
        p = torch.softmax(s, 1)
        p = torch.where(keep.any(1, keepdim=True), p, 0.0)
        p = torch.where(keep, p, 0.0)
        o, a = p @ vv, p @ vv.abs()
        size = (qq.abs() @ kk.abs().T).amax(1, keepdim=True) / math.sqrt(128)
        outs.append(o)
        tols.append((2.0 ** -8 + 1.5e-4 + 2 * 128 * 2.0 ** -24 * size) * a * (1 + 2.0 ** -7) + 2.0 ** -8 * o.abs())
    return torch.stack(outs), torch.stack(tols)


def check(got, q, k, v, lo=None, hi=None, rows=None):
    o, tol = reference(q, k, v, lo, hi, rows)
    g = got[0].double() if rows is None else got[0][:, rows].double()
    assert torch.isfinite(g).all()
    over = (g - o).abs() - tol
    assert (over <= 0).all(), f"{(over > 0).sum().item()} elements off, worst by {over.max().item():.3g}"


def packed(S, Hq, Hk, seed, scale=1.0):
    """q, k, v as [1, H, S, 128] views of one [S, (Hq + 2 Hk) 128] projection."""

    x = rand((S, Hq + 2 * Hk, 128), seed, scale)
    return (t.transpose(0, 1)[None] for t in (x[:, :Hq], x[:, Hq:Hq + Hk], x[:, Hq + Hk:]))


@pytest.mark.parametrize("S,Hq,Hk", [(1, 1, 1), (2, 3, 3), (63, 2, 1), (64, 1, 1), (127, 4, 2), (128, 2, 2), (129, 2, 2),
                                     (255, 1, 1), (256, 4, 4), (257, 6, 2), (300, 5, 5), (1000, 8, 1), (2500, 2, 2), (4097, 3, 1)])
def test_every_key(S, Hq, Hk):
    from tfvideo import attention as A

    q, k, v = packed(S, Hq, Hk, S)
    o = A.bf16(q, k, v)
    assert o.shape == q.shape
    check(o, q, k, v)
    assert torch.equal(o, A.bf16(q, k, v))
    full = A.SpanMask.documents([S])
    assert torch.equal(o, A.bf16(q, k, v, full))
    assert torch.equal(o, A.get("bf16")(q, k, v)) and torch.equal(o, A.bf16_spans(full)(q, k, v))
    device_ok()


@pytest.mark.parametrize("lengths,S,frame,prefix", [
    ([300], 300, 1, 0), ([1], 5, 0, 0), ([0, 0, 7], 400, 0, 0), ([100, 156], 256, 0, 0), ([129, 1, 127, 255, 64], 576, 0, 0),
    ([333, 77, 0, 519, 1, 68], 1100, 0, 0), ([700, 300], 1000, 1, 77), ([901, 384], 1300, 33, [512, 0]), ([512], 512, 128, 128),
    ([64] * 20, 1280, 0, 0), ([5] * 60, 300, 2, 1), ([], 200, 0, 0),
])
def test_packed_requests(lengths, S, frame, prefix):
    from tfvideo import attention as A

    m = A.SpanMask.frames(lengths, frame, prefix, S)
    q, k, v = packed(S, 4, 2, S + len(lengths))
    o = A.bf16(q, k, v, m)
    check(o, q, k, v, m.lo, m.hi)
    assert (o[0, :, sum(lengths):] == 0).all()
    # each request alone gives what it gives inside the pack, to rounding
    at = 0
    for n, p in zip(lengths, [prefix] * len(lengths) if isinstance(prefix, int) else prefix):
        if n:
            c = slice(at, at + n)
            alone = A.bf16(q[:, :, c], k[:, :, c], v[:, :, c], A.SpanMask.frames([n], frame, p))
            check(o[:, :, c], q[:, :, c], k[:, :, c], v[:, :, c], m.lo[c] - at, m.hi[c] - at)
            check(alone, q[:, :, c], k[:, :, c], v[:, :, c], m.lo[c] - at, m.hi[c] - at)
        at += n
    device_ok()


@pytest.mark.parametrize("kind", ["window", "random", "reversed", "beyond"])
def test_any_spans(kind):
    from tfvideo import attention as A

    S = 777
    i = np.arange(S)
    rs = np.random.RandomState(5)
    if kind == "window":
        lo, hi = i - 40, i + 41
    elif kind == "random":
        lo = rs.randint(-5, S, S)
        hi = lo + rs.randint(-3, 200, S)
    elif kind == "reversed":                                   # far keys only; some rows empty
        lo, hi = S - i - 100, S - i
    else:
        lo, hi = np.full(S, -2 ** 31), np.full(S, 2 ** 31 - 1)
    lo, hi = (torch.from_numpy(x.astype(np.int32)).cuda() for x in (lo, hi))
    q, k, v = packed(S, 3, 3, 11)
    check(A.bf16(q, k, v, A.SpanMask(lo, hi)), q, k, v, lo, hi)
    device_ok()


@pytest.mark.parametrize("kind", ["documents", "frames", "random", "one_key", "none", "every"])
def test_many_tiles_a_cta(kind):
    """440 pairs of query tiles, more than run at once: each CTA works through several of differing lengths, some with no
    keys at all, and what one tile's masked values held must not reach the next."""

    from tfvideo import attention as A

    S, Hq, Hk = 2700, 40, 8
    rs = np.random.RandomState(3)
    if kind == "documents":
        m = A.SpanMask.documents([700, 1, 0, 999, 300], S)                        # the last 700 tokens have no keys
    elif kind == "frames":
        m = A.SpanMask.frames([1500, 1100], 90, [100, 0], S)
    elif kind == "every":
        m = A.SpanMask.documents([S])
    else:
        lo = rs.randint(-5, S, S)
        n = {"random": rs.randint(-300, 300, S), "one_key": np.full(S, 1), "none": np.full(S, 0)}[kind]
        n[1024:1536] = 0                                                          # whole tiles without keys
        m = A.SpanMask(*(torch.from_numpy(x.astype(np.int32)).cuda() for x in (lo, lo + n)))
    q, k, v = (t.clone() for t in packed(S, Hq, Hk, 21))
    o = A.bf16(q, k, v, m)
    check(o, q, k, v, m.lo, m.hi)
    assert torch.equal(o, A.bf16(q, k, v, m))
    if kind in ("documents", "frames"):                                           # padding and one head's first request
        at = 2000 if kind == "documents" else 2600
        for t in (k, v):
            t[:, :, at:] = float("nan")
        v[:, 3, 100, 5] = float("inf")
        bad = A.bf16(q, k, v, m)
        seen = (m.lo <= 100) & (m.hi > 100)
        for h in range(Hq):
            same = torch.ones((S, 128), dtype=torch.bool, device="cuda")
            if h // 5 == 3:
                same[seen, 5] = False
                assert torch.isposinf(bad[0, h, seen, 5]).all()
            assert torch.equal(bad[0, h][same], o[0, h][same])
    device_ok()


def test_many_short_heads():
    from tfvideo import attention as A

    m = A.SpanMask.documents([100, 0, 130, 33], 300)
    q, k, v = packed(300, 200, 50, 22)
    check(A.bf16(q, k, v, m), q, k, v, m.lo, m.hi)
    device_ok()


def test_a_workspace_where_none_is_needed_is_left_alone():
    from tfvideo import attention as A
    from tfvideo import native as N

    S, H = 300, 4
    q, k, v = packed(S, H, H, 23)
    out, ws = torch.empty((S, H * 128), dtype=torch.bfloat16, device="cuda"), torch.full((16,), 7, dtype=torch.int32, device="cuda")
    assert N.attn_bf16_workspace_bytes(S, H) == 0
    ld, hs = q.stride(2), q.stride(1)
    rc = N.lib().h3_attn_bf16(q.data_ptr(), ld, hs, k.data_ptr(), ld, hs, v.data_ptr(), ld, hs, S, H, H, None, None,
                              out.data_ptr(), H * 128, ws.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    torch.cuda.synchronize()
    assert (ws == 7).all()
    assert torch.equal(out.view(S, H, 128).transpose(0, 1)[None], A.bf16(q, k, v))


def test_without_a_workspace():
    """The C entry takes none for any length: every row then keeps a running maximum, and no CTA has a second tile."""

    from tfvideo import attention as A
    from tfvideo import native as N

    S, H = 2500, 24
    q, k, v = packed(S, H, H, 24)
    m = A.SpanMask.documents([900, 0, 1500], S)
    out = torch.empty((S, H * 128), dtype=torch.bfloat16, device="cuda")
    ld, hs = q.stride(2), q.stride(1)
    rc = N.lib().h3_attn_bf16(q.data_ptr(), ld, hs, k.data_ptr(), ld, hs, v.data_ptr(), ld, hs, S, H, H, m.lo.data_ptr(),
                              m.hi.data_ptr(), out.data_ptr(), H * 128, None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    check(out.view(S, H, 128).transpose(0, 1)[None], q, k, v, m.lo, m.hi)
    device_ok()


def test_layouts():
    """Head-major memory, separate buffers, unaligned and strided views (copied when TMA cannot read them), shared
    heads as an expanded view: the same bits as contiguous rows."""

    from tfvideo import attention as A

    S, H = 333, 4
    q, k, v = (rand((1, H, S, 128), i) for i in (1, 2, 3))     # [1, H, S, D] contiguous
    ref = A.bf16(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)))
    check(ref, q, k, v)
    assert torch.equal(A.bf16(q, k, v), ref)
    odd = [torch.empty((S, H * 128 + 4), dtype=torch.bfloat16, device="cuda")[:, 4:].view(S, H, 128) for _ in range(3)]
    for d, s in zip(odd, (q, k, v)):
        d.copy_(s[0].transpose(0, 1))
    assert torch.equal(A.bf16(*(t.transpose(0, 1)[None] for t in odd)), ref)
    spread = [torch.zeros((1, H, S, 256), dtype=torch.bfloat16, device="cuda")[..., ::2] for _ in range(3)]
    for d, s in zip(spread, (q, k, v)):
        d.copy_(s)
    assert torch.equal(A.bf16(*spread), ref)
    one = k[:, :1]
    assert torch.equal(A.bf16(q, one.expand(1, H, S, 128), v), A.bf16(q, one.contiguous().repeat(1, H, 1, 1), v))
    assert torch.equal(A.bf16(q, one, v[:, :1]), A.bf16(q, one.expand(1, H, S, 128), v[:, :1].expand(1, H, S, 128)))
    out = torch.full((S, H * 128 + 64), 7.0, dtype=torch.bfloat16, device="cuda")
    A.bf16_tokens(q[0].transpose(0, 1), k[0].transpose(0, 1), v[0].transpose(0, 1), out[:, :H * 128])
    assert torch.equal(out[:, :H * 128].view(S, H, 128).transpose(0, 1)[None], ref) and (out[:, H * 128:] == 7).all()
    rows = torch.cat([t[0].transpose(0, 1).reshape(S, H * 128) for t in (q, k, v, v)], 1)    # out beside q, k, v
    h = rows.view(S, 4 * H, 128)
    A.bf16_tokens(h[:, :H], h[:, H:2 * H], h[:, 2 * H:3 * H], rows[:, 3 * H * 128:])
    assert torch.equal(h[:, 3 * H:].transpose(0, 1)[None], ref) and torch.equal(h[:, :H].transpose(0, 1)[None], q)
    with pytest.raises(RuntimeError, match="overlap"):
        A.bf16_tokens(h[:, :H], h[:, H:2 * H], h[:, 2 * H:3 * H], rows[:, :H * 128])
    assert A.bf16(q[:, :, :0], k[:, :, :0], v[:, :, :0]).shape == (1, H, 0, 128)
    device_ok()


def test_masked_places_hold_anything():
    """NaN and infinities in keys and values outside a row's span leave the row as it is; inside, they reach exactly
    the rows that see them."""

    from tfvideo import attention as A

    m = A.SpanMask.documents([300, 200, 77], 700)
    q, k, v = (t.clone() for t in packed(700, 2, 2, 3))
    clean = A.bf16(q, k, v, m)
    for t in (k, v):                                            # padding rows, and the middle request's neighbours
        t[:, :, 577:] = float("nan")
        t[:, :, 650:] = float("inf")
    q[:, :, 577:] = float("nan")
    assert torch.equal(A.bf16(q, k, v, m), clean)
    k[:, :, :300] = float("-inf")
    v[:, :, :300] = float("nan")
    o = A.bf16(q, k, v, m)
    assert torch.equal(o[:, :, 300:], clean[:, :, 300:])
    assert torch.isnan(o[:, :, :300]).all()
    # causal: a later token's value in the same tile is hidden from earlier rows only
    q, k, v = (t.clone() for t in packed(200, 1, 1, 4))
    c = A.SpanMask.frames([200], 1)
    clean = A.bf16(q, k, v, c)
    v[0, 0, 70, 5], v[0, 0, 90, 6], v[0, 0, 91, 6] = float("inf"), float("nan"), float("-inf")
    v[0, 0, 100, 7], v[0, 0, 101, 7] = float("inf"), float("-inf")
    o = A.bf16(q, k, v, c)
    assert torch.equal(o[:, :, :70], clean[:, :, :70])
    assert torch.isposinf(o[0, 0, 70:, 5]).all() and torch.equal(o[0, 0, :90, 6], clean[0, 0, :90, 6])
    assert torch.isnan(o[0, 0, 90:, 6]).all()
    assert torch.isposinf(o[0, 0, 100, 7]) and torch.isnan(o[0, 0, 101:, 7]).all()
    rest = [d for d in range(128) if d not in (5, 6, 7)]
    assert torch.equal(o[..., rest], clean[..., rest])
    k[0, 0, 150, 3] = float("nan")                              # a visible NaN key makes its rows NaN
    o2 = A.bf16(q, k, v, c)
    assert torch.equal(o2[:, :, :150, rest], clean[:, :, :150, rest]) and torch.isnan(o2[:, :, 150:]).all()
    device_ok()


def test_visible_non_finite_without_a_mask():
    from tfvideo import attention as A

    q, k, v = (t.clone() for t in packed(300, 1, 1, 8))
    clean = A.bf16(q, k, v)
    v[0, 0, 20, 3] = float("nan")
    q[0, 0, 7, 0] = float("nan")
    o = A.bf16(q, k, v)
    assert torch.isnan(o[0, 0, :, 3]).all() and torch.isnan(o[0, 0, 7]).all()
    rows = [r for r in range(300) if r != 7]
    rest = [d for d in range(128) if d != 3]
    assert torch.equal(o[0, 0, rows][:, rest], clean[0, 0, rows][:, rest])
    k[0, 0, 200] = float("nan")                                 # in the polynomial's places too: every row is NaN
    assert torch.isnan(A.bf16(q, k, v)).all()


@pytest.mark.parametrize("scale", [0.0, 6.0, 40.0])
def test_flat_and_peaked_scores(scale):
    from tfvideo import attention as A

    q, k, v = packed(400, 2, 2, 21)
    q = (q.float() * scale).to(torch.bfloat16)
    check(A.bf16(q, k, v), q, k, v)


def test_a_single_key_gives_its_value():
    """A row that sees one key has that key's value, bit for bit (its P is 1, and so is its sum)."""

    from tfvideo import attention as A

    for S in (1, 300, 2500):
        q, k, v = packed(S, 2, 2, 50 + S, 2.0)
        i = torch.arange(S, dtype=torch.int32, device="cuda")
        assert torch.equal(A.bf16(q, k, v, A.SpanMask(i, i + 1)), v)
        at = (i * 7) % S
        assert torch.equal(A.bf16(q, k, v, A.SpanMask(at, at + 1)), v[:, :, at.long()])


def test_rising_scores_rescale_every_step():
    """Scores that grow along the keys raise each row's maximum in every step."""

    from tfvideo import attention as A

    S = 1500
    q, k, v = packed(S, 2, 2, 22)
    ramp = torch.linspace(0.1, 12, S, device="cuda")[None, None, :, None]
    k = (q[:, :, :1].float() * ramp + 0.3 * k.float()).to(torch.bfloat16)
    q = (q[:, :, :1].float() + 0.1 * q.float()).to(torch.bfloat16)
    check(A.bf16(q, k, v), q, k, v)
    m = A.SpanMask.frames([S], 100, 50)
    check(A.bf16(q, k, v, m), q, k, v, m.lo, m.hi)


@pytest.mark.parametrize("grow", [1.0, 2.5, 6.0])
def test_long_rows_with_and_without_bounded_scores(grow):
    """At 2,048 tokens and more a row of bounded scores keeps its first step's maximum; keys that grow along the
    sequence raise the scores far above it, up to and past the bound (which sends the row to the running maximum)."""

    from tfvideo import attention as A

    S = 2304
    q, k, v = (t.clone() for t in packed(S, 2, 2, 24))
    k = (k.float() * torch.linspace(0.2, grow, S, device="cuda")[None, None, :, None]).to(torch.bfloat16)
    check(A.bf16(q, k, v), q, k, v)
    for m in (A.SpanMask.documents([900, 1, 1300], S), A.SpanMask.frames([S], 200, 77)):
        check(A.bf16(q, k, v, m), q, k, v, m.lo, m.hi)
    k[:, 0, 2000] = float("nan")
    m = A.SpanMask.documents([1900, 404])
    o = A.bf16(q, k, v, m)
    check(o[:, :, :1900], q[:, :, :1900], k[:, :, :1900], v[:, :, :1900])
    assert torch.isnan(o[:, 0, 1900:]).all() and torch.isfinite(o[:, 1]).all()
    device_ok()


def test_values_at_the_type_limits():
    """Masked values of bf16's largest magnitude contribute exactly nothing; visible tiny ones survive."""

    from tfvideo import attention as A

    m = A.SpanMask.documents([100, 100])
    q, k, v = (t.clone() for t in packed(200, 1, 1, 23))
    clean = A.bf16(q, k, v, m)
    v[:, :, 100:] = 3.3e38
    k[:, :, 100:] = 3.3e38
    assert torch.equal(A.bf16(q, k, v, m)[:, :, :100], clean[:, :, :100])
    tiny = torch.full_like(v, 1e-37)
    assert (A.bf16(q, q, tiny).float() > 0.99e-37).all()


def test_long_sequence_and_offsets_past_32_bits():
    """Rows of a 150,000-token projection 15,360 wide (2.3 billion elements), under a window; and 37,760 tokens of two
    requests, sampled rows."""

    from tfvideo import attention as A

    S = 150_000
    x = torch.empty((S, 120, 128), dtype=torch.bfloat16, device="cuda")
    heads = rand((S, 3, 128), 5)
    for i, h in enumerate((39, 79, 119)):
        x[:, h] = heads[:, i]
    i = torch.arange(S, device="cuda", dtype=torch.int32)
    lo, hi = i - 100, i + 50
    q, k, v = (x[:, h:h + 1].transpose(0, 1)[None] for h in (39, 79, 119))
    out = torch.empty((S, 15_360), dtype=torch.bfloat16, device="cuda")
    A.bf16_tokens(x[:, 39:40], x[:, 79:80], x[:, 119:120], out[:, 15_232:], A.SpanMask(lo, hi))
    rows = torch.tensor([0, 1, 99, 100, 75_000, 139_810, 149_000, S - 1], device="cuda")
    check(out[:, 15_232:].view(S, 1, 128).transpose(0, 1)[None], q, k, v, lo, hi, rows)
    del x, out
    S = 37_760
    q, k, v = packed(S, 2, 1, 6)
    m = A.SpanMask.documents([18_907, 18_800], S)
    rows = torch.randint(0, S, (300,), generator=torch.Generator().manual_seed(1)).cuda()
    check(A.bf16(q, k, v, m), q, k, v, m.lo, m.hi, rows)
    device_ok()


def test_streams_and_graphs():
    """Two calls at once on two streams, and a captured call that follows its inputs and its mask."""

    from tfvideo import attention as A

    a, b = list(packed(700, 4, 4, 31)), list(packed(900, 4, 4, 32))
    ra, rb = A.bf16(*a), A.bf16(*b)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            oa = A.bf16(*a)
        with torch.cuda.stream(s2):
            ob = A.bf16(*b)
    torch.cuda.synchronize()
    assert torch.equal(oa, ra) and torch.equal(ob, rb)
    m = A.SpanMask.documents([700])
    q, k, v = (t[0].transpose(0, 1) for t in a)
    out = torch.zeros((700, 512), dtype=torch.bfloat16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        A.bf16_tokens(q, k, v, out, m)
    g.replay()
    assert torch.equal(out.view(700, 4, 128).transpose(0, 1)[None], ra)
    other = A.SpanMask.documents([350, 350])
    m.lo.copy_(other.lo), m.hi.copy_(other.hi)
    g.replay()
    assert torch.equal(out.view(700, 4, 128).transpose(0, 1)[None], A.bf16(*a, other))
    device_ok()
