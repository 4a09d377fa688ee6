"""What blocks and captured steps of a packed batch keep: inputs of inference mode, memory that is changed, replaced or
freed between calls.  Every comparison is bit for bit with an eager forward of the same inputs."""

from __future__ import annotations

import pytest
import torch

from helpers import device_ok, need_gpu
from test_packed_block_gpu import S, setup

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    need_gpu()


@pytest.mark.parametrize("use_table", [False, True], ids=["positions", "table"])
def test_blocks_and_captured_steps_in_inference_mode(use_table):
    from tfvideo import graph as G

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu", layers=2)
    eng.attn_mask = m
    eng.set_adapters(sets, rows)
    eng.forward(x.clone(), t_emb, segs, p.table() if use_table else p)
    ref = eng.forward(x.clone(), t_emb, segs, p.table() if use_table else p).clone()
    eng.end_run()
    with torch.inference_mode():
        rope = p.table() if use_table else type(p)(p.pos.clone(), p.dims, p.theta)
        assert (rope if use_table else rope.pos).is_inference()
        eng.forward(x.clone(), t_emb, segs, rope)
        assert torch.equal(eng.forward(x.clone(), t_emb, segs, rope), ref)
        eng.end_run()
        eng.forward(x.clone(), t_emb, segs, rope)
        graph = G.StepGraph(eng, x, t_emb, segs, rope)
        graph.x.copy_(x)
        assert torch.equal(graph.replay(), ref)
    device_ok()


@pytest.mark.parametrize("device", ["cuda", "cpu"])
def test_a_captured_step_follows_positions_changed_in_place(device):
    """The caller's own tensor where it is on the device, ``graph.rope.pos`` in any case."""

    from tfvideo import graph as G

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu", layers=2, adapters=False)
    eng.attn_mask = m
    p = p.to(device)
    moved = type(p)(p.pos.roll(7, 0), p.dims, p.theta)
    eng.forward(x.clone(), t_emb, segs, p)
    refs = [eng.forward(x.clone(), t_emb, segs, q).clone() for q in (p, moved)]
    assert not torch.equal(*refs)
    eng.end_run()
    eng.forward(x.clone(), t_emb, segs, p)
    graph = G.StepGraph(eng, x, t_emb, segs, p)
    if device == "cuda":
        assert graph.rope.pos.data_ptr() == p.pos.data_ptr()
    for k, q in enumerate((p.pos.clone(), moved.pos)):
        (p.pos if device == "cuda" else graph.rope.pos).copy_(q)
        graph.x.copy_(x)
        assert torch.equal(graph.replay(), refs[k]), f"replay {k}"
    device_ok()


def test_a_captured_step_keeps_buffers_weights_and_rows_index():
    """Between replays: a forward of another length (the engine drops its buffers), other weights, a mask and adapters
    that are given other tensors; freed memory is written over each time."""

    from tfvideo import graph as G
    from tfvideo import minimax_h3 as M

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("swiglu", layers=2)
    short = [(0, 128, 3)]
    x2, p2 = x[:128].clone(), p.rows(0, 128)

    def other_length():
        mask, ads, r = eng.attn_mask, eng.adapters, eng.adapter_rows
        eng.attn_mask, eng.adapters, eng.adapter_rows = None, {}, None
        eng.forward(x2.clone(), t_emb, short, p2)
        eng.attn_mask, eng.adapters, eng.adapter_rows = mask, ads, r

    def waste():
        keep = [torch.full((1 << k,), -1, dtype=torch.int8, device="cuda") for k in range(8, 24) for _ in range(8)]
        keep.append([torch.full((1 << k,), -1, dtype=torch.int32) for k in range(6, 16) for _ in range(8)])
        torch.cuda.synchronize()

    eng.attn_mask = m
    eng.set_adapters(sets, rows)
    refs = []
    for k in range(4):
        if k == 2:
            other_length()
        refs.append(eng.forward(x.clone(), t_emb, segs, p).clone())
    eng.end_run()
    eng.forward(x.clone(), t_emb, segs, p)
    graph = G.StepGraph(eng, x, t_emb, list(segs), p)     # (a list no forward has seen)
    assert torch.equal(graph.replay(), refs[1])
    other_length()
    waste()
    graph.x.copy_(x)
    assert torch.equal(graph.replay(), refs[2])
    spare = M.MiniMaxH3Engine.from_weights(M.synthetic_weights(cfg, seed=9, device="cuda"), cfg, device="cuda", attn="bf16")
    eng.replace_blocks(spare.blocks, slots=spare.slots)
    m.lo, m.hi = m.lo * 0, m.hi * 0
    for ad in sets.values():
        ad.A, ad.B, ad.scale = ad.A * 0, ad.B * 0, ad.scale * 0
    eng.set_adapters({}, None)
    eng.attn_mask, eng._idx, eng._idx_key, eng._idx_ref = None, None, None, None
    eng.release_vram()
    waste()
    graph.x.copy_(x)
    assert torch.equal(graph.replay(), refs[3])
    device_ok()


def test_overrides_of_a_forward_share_one_table():
    from tfvideo import minimax_h3 as M

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu", layers=2, adapters=False)
    blocks = [M.EngineBlock(eng, i) for i in range(2)]
    seen = []

    def override(h, rope_freqs, transformer_options):
        seen.append(rope_freqs.clone())
        at.append(rope_freqs.data_ptr())
        return torch.zeros_like(h)

    for moved in range(2):
        if moved:
            p.pos.copy_(p.pos.roll(3, 0))
        at, y = [], x.clone()
        for b in blocks:
            y = b(y, t_emb, segs, p, attention=override)
        assert at[0] == at[1]
        assert torch.equal(seen[-1], p.table()) and torch.equal(seen[-2], p.table())
    assert not torch.equal(seen[0], seen[2])
    device_ok()


@pytest.mark.parametrize("M,R,n", [(700, 16, 64), (4500, 40, 2000), (9000, 128, 3)])
def test_adapter_calls_write_nothing_behind_their_workspace(M, R, n):
    """A tile's part of the workspace ends with its rows: calls whose workspace has a guard behind it, and whose memory
    held NaN before, give what others do."""

    from tfvideo import linear as L
    from tfvideo import native as N
    from test_adapter_gpu import check, make

    x, y, A, B, rows, scale = make(M, 136, 264, R, n, seed=M, kind="any")
    ref = L.adapter_add(y, x, A, B, rows, scale, out=torch.empty_like(y))
    check(ref, x, y, A, B, rows, scale)
    size = N.adapter_workspace_bytes(M, R, n)
    for fill in (0xFF, 0x7F):
        ws = torch.full((size + 4096,), fill, dtype=torch.uint8, device="cuda")
        out = torch.empty_like(y)
        N.launch(0, "h3_adapter_add", 3, x.data_ptr(), 136, y.data_ptr(), 264, A.data_ptr(), B.data_ptr(),
                 scale.data_ptr(), rows.data_ptr(), M, 136, 264, R, n, out.data_ptr(), 264, ws.data_ptr(), size)
        assert torch.equal(out, ref) and (ws[size:] == fill).all()
    device_ok()


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_adapters_changed_in_place(act):
    """Weights and scales of each linear's set, changed in place after set_adapters: forwards and replays use them.  The
    changes are by powers of two, which bf16 takes back without a rounding."""

    from tfvideo import graph as G
    from tfvideo import linear as L

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup(act)
    eng.attn_mask = m

    def forwards(ads):
        eng.set_adapters(ads, rows)
        eng.end_run()
        eng.forward(x.clone(), t_emb, segs, p)
        return eng.forward(x.clone(), t_emb, segs, p).clone()

    def copy(ad):
        c = L.AdapterSet.__new__(L.AdapterSet)
        c.n, c.k, c.count, c.A, c.B, c.scale = ad.n, ad.k, ad.count, ad.A.clone(), ad.B.clone(), ad.scale.clone()
        return c

    forwards(sets)
    eng.end_run()
    eng.forward(x.clone(), t_emb, segs, p)
    graph = G.StepGraph(eng, x, t_emb, segs, p)
    for name in ("qkv", "out", "fc1", "fc2"):
        for what in ("A", "B", "scale"):
            before = forwards({k: copy(ad) for k, ad in sets.items()})
            getattr(sets[0, name], what).mul_(-2)
            ref = forwards({k: copy(ad) for k, ad in sets.items()})
            assert not torch.equal(ref, before)
            eng.set_adapters(sets, rows)               # (as they are now; the next change is made behind it)
            getattr(sets[0, name], what).mul_(-0.5)
            eng.end_run()
            eng.forward(x.clone(), t_emb, segs, p)
            assert torch.equal(eng.forward(x.clone(), t_emb, segs, p), before), (name, what)
            getattr(sets[0, name], what).mul_(-2)
            eng.end_run()
            eng.forward(x.clone(), t_emb, segs, p)
            graph.x.copy_(x)
            assert torch.equal(graph.replay(), ref), (name, what)
    device_ok()


def test_rows_given_on_the_host():
    """A copy of them is what forwards read: ``engine.adapter_rows``, which may be changed in place."""

    eng, cfg, w, x, t_emb, segs, p, m, rows, sets = setup("gelu")
    eng.attn_mask = m

    def second():
        eng.end_run()
        eng.forward(x.clone(), t_emb, segs, p)
        return eng.forward(x.clone(), t_emb, segs, p).clone()

    eng.set_adapters(sets, rows)
    assert eng.adapter_rows is rows
    ref = second()
    rows.copy_(rows.roll(50))
    moved = second()
    assert not torch.equal(moved, ref)
    host = rows.roll(-50).cpu()
    eng.set_adapters(sets, host)
    assert torch.equal(second(), ref)
    eng.adapter_rows.copy_(rows)
    assert torch.equal(second(), moved)
    device_ok()
