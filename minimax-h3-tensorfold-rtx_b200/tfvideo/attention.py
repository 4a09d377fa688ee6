"""Attention backends for the full (non-causal) packed sequence: q, k, v [1, H, S, D] bf16 (strided views are fine,
last dim contiguous) -> [1, H, S, D].  Same registry as tfvideo/attention.py of the reference (:44-54).

fp8            libh3b200's tcgen05 FP8 flash attention (Q/K FP8 per row / per 128-key block with K smoothed, P and V
               FP8); the default.  Its output is a [1, H, S, D] view of token-major [S, H, D] memory, which is what
               the block's out-projection reads.
fp8_sparse(m)  the same kernel under a block-sparse mask ``m`` (a TileMask: per 128-token query tile, the 128-token KV
               tiles it attends to).  ``TileMask.block_sparse`` builds the seeded mask of BASELINE's sharded config
               (25% of tiles per query row, diagonal and text tiles always kept).
bf16           libh3b200's tcgen05 bf16 flash attention: q, k, v read as they are, no quantisation; key heads may be
               shared by groups of query heads.
bf16_spans(m)  the same kernel under a SpanMask ``m``: token i attends to the keys [lo_i, hi_i).  Several requests
               packed in one sequence (``SpanMask.documents``), or a prompt with frame-causal video behind it
               (``SpanMask.frames``).
sdpa / cudnn   PyTorch's bf16 backends, kept as the reference's comparison points (not the fast path).
The reference's ``int8`` (comfy-kitchen) and ``fp4`` (Triton, sm_120) backends have no B200 build; asking for them
raises ValueError, like any unknown name.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.nn.attention import SDPBackend, sdpa_kernel

from . import native as N

HEAD_DIM = 128


def sdpa_flash(q, k, v):
    with sdpa_kernel([SDPBackend.FLASH_ATTENTION, SDPBackend.CUDNN_ATTENTION, SDPBackend.EFFICIENT_ATTENTION],
                     set_priority=True):
        return F.scaled_dot_product_attention(q, k, v)


def sdpa_cudnn(q, k, v):
    with sdpa_kernel([SDPBackend.CUDNN_ATTENTION, SDPBackend.FLASH_ATTENTION, SDPBackend.EFFICIENT_ATTENTION],
                     set_priority=True):
        return F.scaled_dot_product_attention(q, k, v)


def _workspace(S: int, H: int, device) -> torch.Tensor:
    n = N.attn_workspace_bytes(S, H)
    return torch.empty(n + 1024, dtype=torch.uint8, device=device)


def aligned_workspace(buf: torch.Tensor) -> torch.Tensor:
    off = (-buf.data_ptr()) % 1024
    return buf[off:]


TILE = 128


class TileMask:
    """Block-sparse attention mask on 128 x 128 tiles, shared by all heads: query tile r (tokens 128 r .. 128 r + 127)
    attends to the KV tiles kv_idx[kv_ptr[r] : kv_ptr[r + 1]].  Held on the device as int32 CSR (the C ABI's form)."""

    def __init__(self, lists, S: int, device="cuda"):
        nt = (S + TILE - 1) // TILE
        if len(lists) != nt:
            raise ValueError(f"TileMask: {len(lists)} rows for {nt} query tiles")
        ptr, idx = [0], []
        for row in lists:
            row = sorted(set(int(c) for c in row))
            if row and (row[0] < 0 or row[-1] >= nt):
                raise ValueError(f"TileMask: KV tile out of range [0, {nt})")
            idx.extend(row)
            ptr.append(len(idx))
        self.S, self.tiles = S, nt
        self.lists = [sorted(set(int(c) for c in row)) for row in lists]
        self.kv_ptr = torch.tensor(ptr, dtype=torch.int32, device=device)
        self.kv_idx = torch.tensor(idx if idx else [0], dtype=torch.int32, device=device)
        self.kept = len(idx)

    @property
    def density(self) -> float:
        return self.kept / float(self.tiles * self.tiles)

    @classmethod
    def block_sparse(cls, S: int, keep: float = 0.25, text_tokens: int = 512, seed: int = 4, device="cuda"):
        """Seeded mask: every query tile keeps its diagonal tile and the text tiles (the first ``text_tokens``
        tokens), then further KV tiles drawn without replacement until ``keep`` of its row is kept."""

        nt = (S + TILE - 1) // TILE
        per_row = max(1, int(round(keep * nt)))
        text = list(range(min(nt, (text_tokens + TILE - 1) // TILE)))
        g = torch.Generator().manual_seed(seed)
        lists = []
        for r in range(nt):
            row = set(text) | {r}
            order = torch.randperm(nt, generator=g).tolist()
            for c in order:
                if len(row) >= per_row:
                    break
                row.add(c)
            lists.append(sorted(row))
        return cls(lists, S, device)


class SpanMask:
    """The keys each token attends to, as one span [lo, hi) a token: int32 [S] device tensors (clipped to [0, S)).  A
    token with an empty span attends to nothing and gets zeros.  Read on the device when the kernel runs, so a captured
    graph follows changes made in place."""

    def __init__(self, lo: torch.Tensor, hi: torch.Tensor):
        for t in (lo, hi):
            if t.dim() != 1 or t.dtype != torch.int32 or not t.is_contiguous() or t.shape != lo.shape:
                raise ValueError("SpanMask: lo and hi must be contiguous int32 [S] tensors, got "
                                 f"{tuple(lo.shape)} {lo.dtype} and {tuple(hi.shape)} {hi.dtype}")
        self.lo, self.hi, self.S = lo, hi, lo.shape[0]

    @classmethod
    def documents(cls, lengths, S: int | None = None, device="cuda") -> "SpanMask":
        """Requests of the given lengths one after another, each token attending to its own request; tokens behind the
        last one (up to ``S``) attend to nothing."""

        return cls.frames(lengths, 0, 0, S, device)

    @classmethod
    def frames(cls, lengths, frame: int, prefix=0, S: int | None = None, device="cuda") -> "SpanMask":
        """Requests as for ``documents``, each a prefix (``prefix`` tokens, one number or one a request) that attends
        to itself, then frames of ``frame`` tokens that attend to the prefix and to every frame up to their own
        (``frame`` 1: causal; 0: no frames, the whole request)."""

        lengths = [int(n) for n in lengths]
        prefix = [int(prefix)] * len(lengths) if isinstance(prefix, int) else [int(p) for p in prefix]
        S = sum(lengths) if S is None else int(S)
        if min(lengths, default=0) < 0 or sum(lengths) > S or frame < 0 or min(prefix, default=0) < 0 \
                or len(prefix) != len(lengths):
            raise ValueError(f"SpanMask: lengths {lengths} (prefix {prefix}, frame {frame}) do not fit {S} tokens")
        lo, hi = torch.zeros(S, dtype=torch.int32), torch.zeros(S, dtype=torch.int32)
        at = 0
        for n, p in zip(lengths, prefix):
            lo[at:at + n] = at
            if frame:
                i = torch.arange(n)
                p = min(p, n)
                hi[at:at + n] = (at + torch.where(i < p, p, p + ((i - p) // frame + 1) * frame).clamp(max=n)).int()
            else:
                hi[at:at + n] = at + n
            at += n
        return cls(lo.to(device), hi.to(device))


def fp8_tokens(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, S: int, H: int, ld: int, hstride: int,
               out: torch.Tensor, workspace: torch.Tensor | None = None, mask: TileMask | None = None) -> torch.Tensor:
    """Low-level form: element (t, h, d) of q / k / v at base + t * ld + h * hstride + d; out [S, H * 128] bf16.
    ``mask`` (a TileMask for this S) selects the block-sparse kernel."""

    ws = aligned_workspace(_workspace(S, H, q.device) if workspace is None else workspace)
    if mask is None:
        N.attn_fp8(q, k, v, ld, hstride, S, H, out, out.stride(0), ws)
    else:
        if mask.S != S:
            raise ValueError(f"TileMask built for S={mask.S}, attention has S={S}")
        N.attn_fp8_sparse(q, k, v, ld, hstride, S, H, mask.kv_ptr, mask.kv_idx, out, out.stride(0), ws)
    return out


def fp8(q, k, v, mask: TileMask | None = None):
    _, H, S, D = q.shape
    if D != HEAD_DIM or not (q.stride(3) == k.stride(3) == v.stride(3) == 1):
        raise ValueError("fp8 attention: head_dim 128 with a contiguous last dim")
    if not (q.stride(1) == k.stride(1) == v.stride(1) and q.stride(2) == k.stride(2) == v.stride(2)):
        q, k, v = (t.contiguous() for t in (q, k, v))
    out = torch.empty((S, H * D), dtype=torch.bfloat16, device=q.device)
    fp8_tokens(q, k, v, S, H, q.stride(2), q.stride(1), out, mask=mask)
    return out.view(1, S, H, D).transpose(1, 2)


def fp8_sparse(mask: TileMask):
    """A backend function (q, k, v) -> o running the FP8 kernel under ``mask``."""

    def run(q, k, v):
        return fp8(q, k, v, mask)

    return run


def bf16_tokens(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                mask: SpanMask | None = None) -> torch.Tensor:
    """Low-level form: q [S, Hq, 128], k and v [S, Hk, 128] bf16 views (token and head strides multiples of 8,
    16-byte aligned); out [S, Hq * 128] bf16, row stride a multiple of 8.  Values and roundings as for ``bf16``."""

    if q.dim() != 3 or k.dim() != 3 or k.shape != v.shape or q.shape[0] != k.shape[0] or k.shape[1] == 0 \
            or q.shape[1] % k.shape[1] or q.shape[2] != HEAD_DIM or k.shape[2] != HEAD_DIM \
            or not q.stride(2) == k.stride(2) == v.stride(2) == 1 \
            or tuple(out.shape) != (q.shape[0], q.shape[1] * HEAD_DIM) or out.stride(1) != 1 \
            or not q.dtype == k.dtype == v.dtype == out.dtype == torch.bfloat16:
        raise ValueError(f"bf16 attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}, out "
                         f"{tuple(out.shape)}: bf16 [S, H, {HEAD_DIM}] rows and [S, Hq * {HEAD_DIM}], query heads a "
                         "multiple of the key heads")
    (S, Hq, _), Hk = q.shape, k.shape[1]
    ldo = out.stride(0) if S > 1 else out.shape[1]      # (one row: any stride)
    _bf16_launch(S, Hq, Hk, q, q.stride(), k, k.stride(), v, v.stride(), out, ldo, mask)
    return out


def _bf16_launch(S, Hq, Hk, q, sq, k, sk, v, sv, out, ldo, mask: SpanMask | None) -> None:
    """``sq``, ``sk``, ``sv``: (token stride, head stride, ...) of q, k and v."""

    if mask is None:
        lo = hi = None
        dev = N.one_device("bf16 attention", q, k, v, out)
    else:
        if mask.S != S:
            raise ValueError(f"SpanMask is for S={mask.S}, attention has S={S}")
        lo, hi = mask.lo.data_ptr(), mask.hi.data_ptr()
        dev = N.one_device("bf16 attention", q, k, v, out, mask.lo, mask.hi)
    if S and Hq:
        size = N.attn_bf16_workspace_bytes(S, Hk)
        ws = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
        N.launch(dev, "h3_attn_bf16", 1 if ws is None else 2 if mask is None else 3, q.data_ptr(), sq[0], sq[1],
                 k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], S, Hq, Hk, lo, hi, out.data_ptr(), ldo,
                 None if ws is None else ws.data_ptr(), size)


def _tma_rows(t: torch.Tensor):
    """t [1, H, S, 128] and its (token stride, head stride); copied when TMA cannot read its rows in place."""

    _, hs, ld, ds = t.stride()
    if ds != 1 or ld & 7 or hs & 7 or ld <= 0 or hs <= 0 or t.data_ptr() & 15:
        _, H, S, _ = t.shape     # (a dimension of one entry has any stride)
        if ds != 1 or t.data_ptr() & 15 or (S > 1 and (ld & 7 or ld <= 0)) or (H > 1 and (hs & 7 or hs <= 0)):
            t = N.aligned16(t)
            _, hs, ld, ds = t.stride()
    return t, (ld, hs)


def bf16(q, k, v, mask: SpanMask | None = None):
    """q [1, H, S, 128], k and v [1, Hk, S, 128] bf16 (any strides; H a multiple of Hk), each token attending to its span
    of ``mask`` (None: to every key).  Scores and sums are in 32 bits; a key's weight is rounded to bf16 for the product
    with V.  Values up to 2^29: sums of larger ones may overflow in long rows (2,048 tokens and more)."""

    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or qs[0] != 1 or ks[0] != 1 or qs[3] != HEAD_DIM or ks[3] != HEAD_DIM \
            or v.shape != ks or not q.dtype == k.dtype == v.dtype == torch.bfloat16:
        raise ValueError(f"bf16 attention: q, k and v must be bf16 [1, H, S, {HEAD_DIM}], k and v alike, got "
                         f"{tuple(qs)} {q.dtype}, {tuple(ks)} {k.dtype}, {tuple(v.shape)} {v.dtype}")
    _, H, S, D = qs
    Hk = ks[1]
    if ks[2] != S or Hk == 0 or H % Hk:
        raise ValueError(f"bf16 attention: q {tuple(qs)}, k and v {tuple(ks)}: one length, and query heads a multiple "
                         "of the key heads")
    (q, sq), (k, sk), (v, sv) = _tma_rows(q), _tma_rows(k), _tma_rows(v)
    out = q.new_empty((1, S, H, D))
    _bf16_launch(S, H, Hk, q, sq, k, sk, v, sv, out, H * D, mask)
    return out.transpose(1, 2)


def bf16_spans(mask: SpanMask):
    """A backend function (q, k, v) -> o running the bf16 kernel under ``mask``."""

    def run(q, k, v):
        return bf16(q, k, v, mask)

    return run


BACKENDS = {"sdpa": sdpa_flash, "cudnn": sdpa_cudnn, "fp8": fp8, "bf16": bf16}
BENCH: dict = {}
DEFAULT = "fp8"


def get(name: str):
    if name == "auto":
        name = DEFAULT
    if name not in BACKENDS:
        raise ValueError(f"attention backend {name!r}: one of {', '.join(['auto', *BACKENDS])}")
    return BACKENDS[name]
