"""Fused elementwise kernels of a MiniMax H3 block on B200 (libh3b200): each reads its input once, writes once.

Same interface as tfvideo/kernels.py of the reference (:31, :56, :76): ``idx`` (int32 [S]) is each row's
modulation row and ``mod`` (fp32 [R, 6, D]) holds shift_msa, scale_msa, gate_msa, shift_mlp, scale_mlp, gate_mlp.
fp32 inside, bf16 out.  ``gelu_tanh`` is the FFN activation of BASELINE's H3-shaped configs.

``rope_axes`` and ``qknorm_rope_axes`` take positions over several axes (time, height, width) instead of a ready
rotation table; ``AxialPositions`` bundles them for ``EngineBlock`` and ``StepGraph``.
"""

from __future__ import annotations

import ctypes as C
from functools import lru_cache

import torch

from . import native as N


def _check_rows(x: torch.Tensor, name: str) -> None:
    if x.dim() != 2 or x.dtype != torch.bfloat16 or x.stride(1) != 1:
        raise ValueError(f"{name}: expected a row-major bf16 [S, D] tensor, got {tuple(x.shape)} {x.dtype}")


HEAD_DIM = 128


@lru_cache(maxsize=64)
def _axes(what: str, dims: tuple, theta: tuple) -> tuple:
    """Validated (dims, theta per axis, rot, the two as H3Positions holds them) of plain numbers."""

    if not 1 <= len(dims) <= 4 or len(theta) != len(dims):
        raise ValueError(f"{what}: 1 to 4 axes and one theta for each or for all, got dims {dims}, theta {theta}")
    if any(d <= 0 or d % 2 for d in dims) or sum(dims) > HEAD_DIM:
        raise ValueError(f"{what}: each axis rotates an even number of dims, together at most {HEAD_DIM}, got {dims}")
    if any(not 0.0 < t < float("inf") for t in theta):
        raise ValueError(f"{what}: theta must be positive and finite, got {theta}")
    n = len(dims)
    return dims, theta, sum(dims), (N.i32 * 4)(*dims, *(0,) * (4 - n)), (C.c_double * 4)(*theta, *(1.0,) * (4 - n))


def _check_positions(what: str, pos: torch.Tensor, dims, theta) -> tuple:
    # (as plain numbers: a tensor among them would be known by its identity, whatever it comes to hold)
    dims = tuple(map(int, dims))
    axes = _axes(what, dims, tuple(map(float, theta)) if isinstance(theta, (list, tuple)) else (float(theta),) * len(dims))
    if pos.dim() != 2 or pos.dtype not in N.POS_TYPES or pos.shape[1] != len(axes[0]):
        raise ValueError(f"{what}: pos must be an int32, int64 or fp32 [S, {len(axes[0])}] tensor, got "
                         f"{tuple(pos.shape)} {pos.dtype}")
    return axes


def _positions(pos: torch.Tensor, axes: tuple) -> N.H3Positions:
    return N.H3Positions(pos.data_ptr(), N.POS_TYPES[pos.dtype], *pos.stride(), len(axes[0]), axes[3], axes[4])


def rope_axes(pos: torch.Tensor, dims, theta=10000.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """The rotation table fp32 [S, rot/2, 2, 2] ([[cos, -sin], [sin, cos]]) of ``pos`` [S, axes] (int32, int64 or
    fp32, any strides).  Axis a rotates ``dims[a]`` dims (rot = their sum): its j-th pair turns by
    pos[s, a] * theta^(-2j / dims[a]), formed in 64 bits; pairs of the axes one after another.  ``theta``: one number,
    or one per axis."""

    axes = _check_positions("rope_axes", pos, dims, theta)
    S = pos.shape[0]
    shape = (S, axes[2] // 2, 2, 2)
    if out is None:
        out = pos.new_empty(shape, dtype=torch.float32)
    elif out.shape != shape or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError(f"rope_axes: out must be a contiguous fp32 {shape} tensor, got {tuple(out.shape)} {out.dtype}")
    dev = N.one_device("rope_axes", pos, out)
    if S:
        N.launch(dev, "h3_rope_axes", 1, C.byref(_positions(pos, axes)), S, out.data_ptr())
    return out


def qknorm_rope_axes(q: torch.Tensor, k: torch.Tensor, qw: torch.Tensor, kw: torch.Tensor, pos: torch.Tensor, dims,
                     theta=10000.0, eps: float = 1e-5, out_q: torch.Tensor | None = None,
                     out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-head RMSNorm of q [S, Hq, 128] and k [S, Hk, 128] (bf16, head dim contiguous, weights ``qw`` / ``kw``
    [128]) and the split-half rotation of their first rot dims by ``rope_axes``'s angles, in one pass with no table.
    In place, unless ``out_q`` / ``out_k`` name other memory (apart from the inputs).  rot % 8 == 0."""

    axes = _check_positions("qknorm_rope_axes", pos, dims, theta)
    oq, ok = q if out_q is None else out_q, k if out_k is None else out_k
    qs, ks = q.shape, k.shape
    if len(qs) != 3 or len(ks) != 3 or qs[2] != HEAD_DIM or ks[2] != HEAD_DIM or oq.shape != qs or ok.shape != ks \
            or not q.dtype == k.dtype == oq.dtype == ok.dtype == torch.bfloat16:
        raise ValueError(f"qknorm_rope_axes: q, k and their outputs must be bf16 [S, H, {HEAD_DIM}], got "
                         + ", ".join(f"{tuple(t.shape)} {t.dtype}" for t in (q, k, oq, ok)))
    st = []
    for t in (q, k) if out_q is None and out_k is None else (q, k, oq, ok):
        ld, hs, ds = t.stride()
        at = t.data_ptr()
        if ds != 1 or ld & 3 or hs & 3 or at & 7:
            ld, hs = ld if t.shape[0] > 1 else 0, hs if t.shape[1] > 1 else 0   # (of one entry: any)
        if ds != 1 or ld & 3 or hs & 3 or at & 7:
            raise ValueError("qknorm_rope_axes: q, k and their outputs need a contiguous head dim and 8-byte aligned rows, "
                             f"got strides {t.stride()}")
        st += (at, ld, hs)
    if len(st) == 6:
        st += st
    (S, Hq, _), Hk = qs, ks[1]
    if k.shape[0] != S or pos.shape[0] != S:
        raise ValueError(f"qknorm_rope_axes: q has {S} tokens, k {k.shape[0]}, pos {pos.shape[0]}")
    if axes[2] % 8:
        raise ValueError(f"qknorm_rope_axes: the rotated dims must be a multiple of 8, got {axes[0]}")
    if qw.numel() != HEAD_DIM or kw.numel() != HEAD_DIM:
        raise ValueError(f"qknorm_rope_axes: norm weights have {HEAD_DIM} elements")
    if S and (Hq == 0) != (Hk == 0):
        raise ValueError("qknorm_rope_axes: q and k need at least one head each")
    qw, kw = _norm_weight(qw), _norm_weight(kw)
    dev = N.one_device("qknorm_rope_axes", q, k, oq, ok, qw, kw, pos)
    if S and Hq:
        N.launch(dev, "h3_qknorm_rope_axes", 1, *st[:6], S, Hq, Hk, qw.data_ptr(), kw.data_ptr(),
                 C.byref(_positions(pos, axes)), eps, *st[6:])
    return oq, ok


def _norm_weight(w: torch.Tensor) -> torch.Tensor:
    """fp32 [128], contiguous, 16-byte aligned."""

    if w.dtype != torch.float32 or not w.is_contiguous():
        w = w.float().contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


class AxialPositions:
    """Positions of a packed sequence over several axes, in place of a rotation table: ``pos`` [S, axes], the dims
    each axis rotates and theta, as for ``rope_axes``.  ``EngineBlock`` takes one as its ``rope_freqs``."""

    def __init__(self, pos: torch.Tensor, dims, theta=10000.0):
        self.dims, self.theta = _check_positions("AxialPositions", pos, dims, theta)[:2]
        self.pos = pos

    def __len__(self) -> int:
        return self.pos.shape[0]

    @property
    def rot(self) -> int:
        return sum(self.dims)

    def rows(self, a: int, b: int) -> "AxialPositions":
        """The positions of tokens [a, b) (a view)."""

        return AxialPositions(self.pos[a:b], self.dims, self.theta)

    def to(self, device) -> "AxialPositions":
        return AxialPositions(self.pos.to(device), self.dims, self.theta)

    def table(self) -> torch.Tensor:
        """ComfyUI's rope_freqs of these positions: fp32 [1, S, 1, rot/2, 2, 2]."""

        return rope_axes(self.pos, self.dims, self.theta)[None, :, None]


def norm_mod(x: torch.Tensor, w: torch.Tensor, mod: torch.Tensor, part: int, idx: torch.Tensor, eps: float,
             out: torch.Tensor | None = None) -> torch.Tensor:
    """RMSNorm(x) * w * (1 + scale) + shift for x [S, D] bf16; ``part`` 0 = attention (chunks 0, 1), 1 = MLP (3, 4)."""

    _check_rows(x, "norm_mod")
    out = torch.empty_like(x) if out is None else out
    N.norm_mod(x, w.float().contiguous(), mod.float().contiguous(), idx.to(torch.int32).contiguous(), part, eps,
               out=out)
    return out


def gate_add(x: torch.Tensor, y: torch.Tensor, mod: torch.Tensor, part: int, idx: torch.Tensor) -> torch.Tensor:
    """x += y * gate in place (x, y [S, D] bf16); ``part`` 0 = gate_msa (chunk 2), 1 = gate_mlp (chunk 5)."""

    _check_rows(x, "gate_add")
    _check_rows(y, "gate_add")
    N.gate_add(x, y, mod.float().contiguous(), idx.to(torch.int32).contiguous(), part)
    return x


def swiglu(gu: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, 2F] = [gate | up] bf16 -> silu(gate) * up, [M, F] bf16."""

    _check_rows(gu, "swiglu")
    M, F2 = gu.shape
    out = torch.empty((M, F2 // 2), dtype=torch.bfloat16, device=gu.device) if out is None else out
    N.act(gu, out, N.ACT_SWIGLU)
    return out


def gelu_tanh(u: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, F] bf16 -> gelu(u, approximate="tanh"), [M, F] bf16."""

    _check_rows(u, "gelu_tanh")
    out = torch.empty_like(u) if out is None else out
    N.act(u, out, N.ACT_GELU)
    return out
