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
