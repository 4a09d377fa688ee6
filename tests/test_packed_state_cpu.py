"""What the packed-batch operators and an engine keep between calls (tables, positions, checked arguments), without a GPU."""

from __future__ import annotations

import pytest
import torch


def engine():
    from tfvideo import minimax_h3 as M

    return M.MiniMaxH3Engine([], device="cpu", attn="bf16")


def table(S=6):
    return torch.randn((1, S, 1, 8, 2, 2), generator=torch.Generator().manual_seed(1))


def test_positions_and_tables_of_inference_mode():
    """Tensors made in inference mode count no versions; a sampler's usual ones."""

    from tfvideo import kernels as K

    eng = engine()
    with torch.inference_mode():
        pos = torch.arange(12, dtype=torch.int32).view(6, 2)
        p, t = K.AxialPositions(pos, (8, 8)), table()
        assert t.is_inference() and p.pos.is_inference()
        assert torch.equal(eng.rope_positions(p, 6).pos, pos) and eng.rope_positions(p, 6) is eng.rope_positions(p, 6)
        assert torch.equal(eng.rope_table(t, 6), t.view(6, 8, 2, 2)) and eng.rope_table(t, 6) is eng.rope_table(t, 6)
    assert torch.equal(eng.rope_positions(p, 6).pos, pos)            # outside it too
    assert torch.equal(eng.rope_table(t, 6), t.view(6, 8, 2, 2))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tables_are_kept_by_object_and_version(dtype):
    """Kept while the same object is handed in unchanged; one changed in place, another in its memory, or one that was
    refused is not taken for it."""

    eng = engine()
    t = table().to(dtype)
    ref = lambda x: x.float().reshape(6, 8, 2, 2)      # noqa: E731
    first = eng.rope_table(t, 6)
    assert torch.equal(first, ref(t)) and eng.rope_table(t, 6) is first
    t.mul_(2)
    assert torch.equal(eng.rope_table(t, 6), ref(t))
    for k in range(4):                                 # ids and addresses of freed tables come again
        other = (table() + k).to(dtype)
        assert torch.equal(eng.rope_table(other, 6), ref(other))
        del other
    with pytest.raises(RuntimeError):
        eng.rope_table(t[:, :5], 6)
    assert torch.equal(eng.rope_table(t, 6), ref(t))


def test_an_override_table_is_made_once_a_forward(monkeypatch):
    """Attention overrides of every block are handed one table; positions changed in place, or others, make a new one."""

    from tfvideo import kernels as K

    made = []

    def rope_axes(pos, dims, theta):
        made.append(pos.clone())
        return torch.full((pos.shape[0], 8, 2, 2), float(len(made)))

    monkeypatch.setattr(K, "rope_axes", rope_axes)
    eng = engine()
    p = K.AxialPositions(torch.arange(12, dtype=torch.int32).view(6, 2), (8, 8))
    first = eng.rope_table(p, 6)
    assert eng.rope_table(p, 6) is first and eng.rope_positions(p, 6).pos is p.pos and eng.rope_table(p, 6) is first
    p.pos.add_(1)
    assert eng.rope_table(p, 6) is not first and len(made) == 2 and torch.equal(made[1], p.pos)
    q = K.AxialPositions(p.pos, (8, 8), 50.0)
    assert eng.rope_table(q, 6) is not eng.rope_table(p, 6) and len(made) == 4
    eng._rope_key = None                               # as a new forward does
    t = table()
    assert torch.equal(eng.rope_table(t, 6), t.view(6, 8, 2, 2))


def test_theta_and_dims_are_taken_by_their_values():
    """Tensors and numpy numbers in place of plain ones: as they are when the call is made."""

    import numpy as np
    from tfvideo import kernels as K

    pos = torch.zeros((10, 2), dtype=torch.int32)
    theta, dim = torch.tensor(10000.0), torch.tensor(16)
    for t in (theta, (theta, theta), [theta, 10000.0]):
        theta.fill_(10000.0), dim.fill_(16)
        p = K.AxialPositions(pos, (dim, 16), t)
        assert p.theta == (10000.0, 10000.0) and p.dims == (16, 16) and p.rot == 32
        theta.fill_(50.0), dim.fill_(32)
        p = K.AxialPositions(pos, (dim, 16), t)
        assert p.theta[0] == 50.0 and p.dims == (32, 16) and all(type(x) is float for x in p.theta)
        axes = K._check_positions("rope_axes", pos, (dim, 16), t)
        assert axes[3][0] == 32 and axes[4][0] == 50.0
    p = K.AxialPositions(pos, np.array([16, 24]), np.float32(256))
    assert p.dims == (16, 24) and p.theta == (256.0, 256.0)
    with pytest.raises(ValueError, match="theta"):
        K.AxialPositions(pos, (16, 16), (10000.0,))


@pytest.mark.parametrize("M", [1, 10, 333, 4096, 37_760])
@pytest.mark.parametrize("R", [8, 64, 128])
@pytest.mark.parametrize("n", [1, 2, 100, 1000, 1 << 20])
def test_adapter_workspace_goes_by_the_rows(M, R, n):
    """A x of every row (its rank rounded up to 16, bf16), and 20 bytes a row of lists at the most, however many adapters
    are registered."""

    from tfvideo import native
    if not native.LIB_PATH.exists():
        from build import build
        build()
    size = native.lib().h3_adapter_workspace_bytes(M, R, n)
    t = M * ((R + 15) // 16 * 16) * 2
    assert t <= size <= t + 20 * M + 64
