"""A packed batch of requests through the engine: positions over (time, height, width), a span of keys for every token
and every request's own adapters, together, as a user runs them.

The reference is the block in 32-bit torch with bf16 weights (no quantisation), attention under the mask and the
adapters merged per request.  Bars as for the other block tests: cosine >= 0.998 of the output (the block's bar), and
0.95 of its update, which carries the NVFP4 rounding of four linears.  Two vectors of one length with cosine 0.95 are
sqrt(2 - 2 x 0.95) = 0.316 of that length apart; here the update is small beside x (0.05 to 0.3 of it), so the two
roundings of the bf16 residual, each at most half a step or 2^-8 of its element, have to be counted beside it:
|out - ref| <= 0.316 |ref - x| + 2 x 2^-8 |ref|.
The adapters' part is looked for along its own direction, where rounding noise is spread over 163,840 others: the output
must be nearer to the reference with adapters than to the one without.
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


LENGTHS, S = [150, 0, 90, 61], 320          # three requests (one empty) and 19 padding tokens
DIMS = (32, 32, 32)


def setup(act, layers=1, attn="bf16", adapters=True, seed=3):
    from tfvideo import attention as A
    from tfvideo import kernels as K
    from tfvideo import linear as L
    from tfvideo import minimax_h3 as M

    cfg = M.Config(layers=layers, dim=512, heads=4, head_dim=128, ffn=1024 if act == "gelu" else 512, act=act, t_dim=8)
    weights = list(M.synthetic_weights(cfg, seed=seed, device="cuda"))
    eng = M.MiniMaxH3Engine.from_weights(weights, cfg, device="cuda", attn=attn)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")      # noqa: E731
    x = r(S, 512).to(torch.bfloat16)
    t_emb = r(2, 8)
    segs = [(0, 100, 0), (100, 240, 3), (240, S, 5)]
    i = torch.arange(S, device="cuda")
    p = K.AxialPositions(torch.stack([i // 40, (i // 8) % 5, i % 8], 1).to(torch.int32), DIMS)
    m = A.SpanMask.frames(LENGTHS, 40, 20, S)
    rows = torch.full((S,), -1, dtype=torch.int32, device="cuda")
    rows[:150], rows[240:301] = 1, 0                               # request 2 has no adapter
    sets = {}
    if adapters:
        for b in range(layers):
            for name in ("qkv", "out", "fc1", "fc2"):
                n, k = eng.blocks[b].lins[name].n, eng.blocks[b].lins[name].k
                sets[b, name] = L.AdapterSet([(r(q, k) / math.sqrt(k), r(n, q) * 0.3 / math.sqrt(q)) for q in (8, 20)],
                                             [0.7, 1.3])
    return eng, cfg, weights, x, t_emb, segs, p, m, rows, sets


def reference(cfg, w, x, t_emb, segs, p, m, rows, sets):
    x = x.float()
    idx = torch.zeros(S, dtype=torch.long, device="cuda")
    for a, b, row in segs:
        idx[a:b] = row
    mod = (w["ada_b"] + t_emb @ w["ada_w"].T).view(-1, 6, 512)[idx]

    def norm(t, weight, part):
        t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.eps) * weight
        return t * (1 + mod[:, 3 * part + 1]) + mod[:, 3 * part]

    def linear(t, name):
        y = t @ w[name].float().T
        if (0, name) in sets:
            s = sets[0, name]
            for i in range(s.count):
                on = (rows == i)[:, None]
                y = y + torch.where(on, s.scale[i] * ((t @ s.A[i].float().T) @ s.B[i].float().T), 0.0)
        return y

    qkv = linear(norm(x, w["norm1"], 0), "qkv").view(S, 3, 4, 128)
    ang = torch.cat([p.pos[:, a:a + 1].double() * 10000.0 ** (-2 * torch.arange(16, device="cuda").double() / 32)
                     for a in range(3)], 1)
    c, sn = (f(ang).float()[:, None] for f in (torch.cos, torch.sin))

    def rope(t, weight):
        t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + cfg.qk_eps) * weight
        a, b = t[..., :48], t[..., 48:96]
        return torch.cat([a * c - b * sn, a * sn + b * c, t[..., 96:]], -1)

    q, k, v = rope(qkv[:, 0], w["q_norm"]), rope(qkv[:, 1], w["k_norm"]), qkv[:, 2]
    j = torch.arange(S, device="cuda")
    keep = (j >= m.lo[:, None]) & (j < m.hi[:, None])
    s = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(128)
    pr = torch.softmax(s.masked_fill(~keep, -1e30), -1) * keep
    o = torch.einsum("hij,jhd->ihd", pr, v).reshape(S, 512)
    x = x + linear(o, "out") * mod[:, 2]
    u = linear(norm(x, w["norm2"], 1), "fc1")
    if cfg.act == "gelu":
        a = torch.nn.functional.gelu(u, approximate="tanh")
    else:
        a = torch.nn.functional.silu(u[:, :cfg.ffn]) * u[:, cfg.ffn:]
    return x + linear(a, "fc2") * mod[:, 5]


def cosine(a, b):
    return torch.nn.functional.cosine_similarity(a.double().flatten(), b.double().flatten(), 0).item()


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("names", [("qkv", "out", "fc1", "fc2"), ("fc2",), ("fc1",), ()])
def test_packed_requests_through_a_block(act, names):
    from tfvideo import minimax_h3 as M

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup(act)
    sets = {k: v for k, v in sets.items() if k[1] in names}
    eng.attn_mask = m
    eng.set_adapters(sets, rows if sets else None)
    ref = reference(cfg, w[0], x, t_emb, segs, p, m, rows, sets)
    plain = reference(cfg, w[0], x, t_emb, segs, p, m, rows, {})
    blk = M.EngineBlock(eng, 0)
    for forward in range(3):                                # dynamic scales first, then delayed ones
        out = blk(x.clone(), t_emb, segs, p)
        assert torch.isfinite(out).all()
        assert cosine(out, ref) >= 0.998
        off = (out.float() - ref).norm()
        assert off <= 0.316 * (ref - x.float()).norm() + 2 * 2.0 ** -8 * ref.norm()
        if sets:
            assert off < (out.float() - plain).norm()
    device_ok()


def test_positions_equal_their_table_through_a_block():
    """AxialPositions against the table they make: q and k differ by a bf16 rounding at most, so the outputs do by no
    more than the block's own rounding; and an attention override is handed that table."""

    from tfvideo import minimax_h3 as M

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu", adapters=False)
    eng.attn_mask = m
    blk = M.EngineBlock(eng, 0)
    a = blk(x.clone(), t_emb, segs, p)
    eng.end_run()
    b = blk(x.clone(), t_emb, segs, p.table())
    assert cosine(a, b) >= 0.99999
    seen = []

    def override(h, rope_freqs, transformer_options):
        seen.append(rope_freqs)
        return torch.zeros_like(h)

    blk(x.clone(), t_emb, segs, p, attention=override)
    assert torch.equal(seen[0], p.table()) and seen[0].shape == (1, S, 1, 48, 2, 2)
    with pytest.raises(ValueError, match="tokens"):
        blk(x.clone(), t_emb, segs, p.rows(0, 100))


def test_adapters_through_an_attention_override():
    """An override that projects through AttnFacade gets the adapters of its rows too."""

    from tfvideo import minimax_h3 as M

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu")
    blk = M.EngineBlock(eng, 0)
    h = x.clone()
    base = blk.attn.qkv_proj(h)
    eng.set_adapters(sets, rows)
    with_adapters = blk.attn.qkv_proj(h)
    none = rows < 0
    assert torch.equal(with_adapters[none], base[none]) and not torch.equal(with_adapters[~none], base[~none])
    assert torch.equal(sets[0, "qkv"].add(base.clone(), h, rows), with_adapters)
    with pytest.raises(ValueError, match="tokens"):
        blk.attn.qkv_proj(h[:100])


def test_engine_refusals():
    from tfvideo import attention as A
    from tfvideo import linear as L

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu")
    table = p.table()
    for attn, mask in (("fp8", m), ("sdpa", m), ("bf16", A.TileMask.block_sparse(S)),
                       ("bf16", A.SpanMask.documents([S - 1]))):
        eng.attn, eng.attn_name, eng.attn_mask = A.get(attn), attn, mask
        with pytest.raises(ValueError, match="attn_mask"):
            eng.forward(x.clone(), t_emb, segs, table)
    for bad, r in (({(1, "qkv"): sets[0, "qkv"]}, rows), ({(0, "up"): sets[0, "qkv"]}, rows),
                   ({(0, "out"): sets[0, "qkv"]}, rows), (sets, None), (sets, rows.long()), (sets, rows[::2])):
        with pytest.raises(ValueError):
            eng.set_adapters(bad, r)
    eng.attn, eng.attn_mask = A.bf16, None
    eng.set_adapters(sets, rows[:100].contiguous())
    with pytest.raises(ValueError, match="adapter rows"):
        eng.forward(x.clone(), t_emb, segs, p)
    eng.set_adapters({}, None)
    eng.end_run()
    assert torch.isfinite(eng.forward(x.clone(), t_emb, segs, p)).all()
    device_ok()


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_step_graph_of_a_packed_batch(act):
    """Two blocks captured with positions, mask and adapters replay bit for bit what eager forwards give, and follow
    masks and rows changed in place."""

    from tfvideo import attention as A
    from tfvideo import graph as G

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup(act, layers=2)
    eng.attn_mask = m
    eng.set_adapters(sets, rows)
    xs = [torch.randn((S, 512), generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").to(torch.bfloat16)
          for i in range(4)]
    other = A.SpanMask.documents([200, 120], S)
    own = (m.lo.clone(), m.hi.clone(), eng.adapter_rows.clone())

    def change(back=False):
        m.lo.copy_(own[0] if back else other.lo), m.hi.copy_(own[1] if back else other.hi)
        eng.adapter_rows.copy_(own[2] if back else own[2].roll(50))

    eager = []
    for k, xi in enumerate(xs):
        if k == 3:
            change()
        eager.append(eng.forward(xi.clone(), t_emb, segs, p).clone())
    change(back=True)
    eng.end_run()
    eng.forward(xs[0].clone(), t_emb, segs, p)
    graph = G.StepGraph(eng, xs[1], t_emb, segs, p)
    for k in (1, 2, 3):
        if k == 3:
            change()
        graph.x.copy_(xs[k])
        out = graph.replay()
        assert torch.equal(out, eager[k]), f"replay {k}"
    device_ok()


def test_a_captured_step_keeps_its_mask_and_adapters():
    from tfvideo import attention as A
    from tfvideo import graph as G

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu", layers=2)
    eng.attn_mask = A.SpanMask(m.lo.clone(), m.hi.clone())
    eng.set_adapters(sets, rows.clone())
    eng.forward(x.clone(), t_emb, segs, p)
    ref = eng.forward(x.clone(), t_emb, segs, p).clone()
    eng.end_run()
    eng.forward(x.clone(), t_emb, segs, p)
    graph = G.StepGraph(eng, x, t_emb, segs, p)
    eng.set_adapters({}, None)
    eng.attn_mask = None
    sets.clear()
    waste = [torch.full((n,), -1, dtype=torch.int32, device="cuda") for n in (S, 512, 1 << 12, 1 << 16, 1 << 20) * 8]
    graph.x.copy_(x)
    assert torch.equal(graph.replay(), ref)
    del waste
    device_ok()
