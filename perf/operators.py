"""What the packed-batch operators of ``tfvideo`` are measured on: rotary tables and QK-norm + RoPE from multi-axis
positions, bf16 attention under per-token key spans, and low-rank adapters of several requests beside one projection.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) where ``own`` is false, and
calls the framework where it is true.  Shapes follow the block this framework runs: head_dim 128, 40 heads (5 a GPU on
8 GPUs), hidden 5,120, qkv 15,360 wide, 37,760 tokens (512 text + 1,680 keyframe + 496 audio + 33 x 24 x 44 video),
positions over (time, height, width) with 44 / 42 / 42 or 32 / 32 / 32 rotated dims, theta 10,000.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

HD = 128
EPS = 1e-5


def _tfvideo():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "minimax-h3-tensorfold-rtx_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from tfvideo import attention, kernels, linear
    return attention, kernels, linear


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one still image of 16 x 16 patches behind 77 text tokens: the table of a preview, a latency-bound call
        dict(name="rope_table_still", op="table", s=333, dims="32,32,32", theta=10000.0, frac=False),
        # the whole packed sequence of a video step, fractional time positions (frame rate rescaled)
        dict(name="rope_table_video", op="table", s=37760, dims="44,42,42", theta=10000.0, frac=True),
        # the preview's q / k of a small block (4 heads)
        dict(name="qknorm_still", op="qknorm", s=333, hq=4, hk=4, dims="32,32,32", theta=10000.0, frac=False),
        # one GPU's heads of an 8-GPU step: all tokens, 5 of 40 heads
        dict(name="qknorm_share", op="qknorm", s=37760, hq=5, hk=5, dims="44,42,42", theta=10000.0, frac=False),
        # all heads of the video step on one GPU
        dict(name="qknorm_video", op="qknorm", s=37760, hq=40, hk=40, dims="44,42,42", theta=10000.0, frac=True),
        # two short prompts packed into one small sequence: a latency-bound attention call
        dict(name="attn_pair_small", op="attn", s=256, hq=4, hk=4, docs="156,100", prefix=0, frame=0),
        # several clips of odd lengths, an empty request and padding rows behind the last one, all heads
        dict(name="attn_ragged", op="attn", s=4200, hq=40, hk=40, docs="1333,77,0,2019,1,668", prefix=0, frame=0),
        # frame-causal generation of two clips: a prompt prefix everyone sees, then frames that see the frames before;
        # 4 query heads share each key head
        dict(name="attn_frames", op="attn", s=16385, hq=20, hk=5, docs="9001,7384", prefix=512, frame=330),
        # guided sampling at video length: prompt and negative prompt packed side by side, each full attention
        dict(name="attn_video_guided", op="attn", s=37760, hq=40, hk=40, docs="18907,18853", prefix=0, frame=0),
        # one adapter on the output projection of a preview
        dict(name="adapter_still", op="adapter", m=333, k=512, n=512, r=16, adapters=1, order="runs", none=False),
        # four requests with adapters of their own and one without any, packed at keyframe length
        dict(name="adapter_out_mixed", op="adapter", m=4096, k=5120, n=5120, r=64, adapters=4, order="runs", none=True),
        # two adapters on the qkv projection of the video step
        dict(name="adapter_qkv_video", op="adapter", m=37760, k=5120, n=15360, r=32, adapters=2, order="runs",
             none=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["table", "qknorm", "attn", "adapter"])
    dims = rng.choice(["44,42,42", "32,32,32", "16,24,24", "64,64", "128"])
    theta = rng.choice([10000.0, 10000.0, 256.0, 1000000.0])
    if op == "table":
        return dict(op=op, s=_log(rng, 1, 37760), dims=dims, theta=theta, frac=rng.random() < 0.5)
    if op == "qknorm":
        hk = rng.choice([1, 4, 5, 8, 10, 20, 40])
        hq = hk * rng.choice([1, 1, 2]) if hk <= 20 else hk
        return dict(op=op, s=_log(rng, 1, 37760), hq=hq, hk=hk, dims=dims, theta=theta, frac=rng.random() < 0.5)
    if op == "attn":
        hk = rng.choice([1, 2, 4, 5, 8])
        hq = hk * rng.choice([1, 1, 2, 4])
        s = _log(rng, 1, 12000)
        parts, left = [], s
        for _ in range(rng.randint(1, 5)):
            n = rng.randint(0, left)
            parts.append(n)
            left -= n
        if rng.random() < 0.6:          # no padding rows: the last request takes what is left
            parts.append(left)
        kind = rng.choice(["full", "full", "causal", "frames"])
        return dict(op=op, s=s, hq=hq, hk=hk, docs=",".join(map(str, parts)),
                    prefix=0 if kind == "full" else rng.choice([0, 77, 512]),
                    frame=dict(full=0, causal=1, frames=_log(rng, 16, 1056))[kind])
    return dict(op=op, m=_log(rng, 1, 16384), k=8 * _log(rng, 32, 1200), n=8 * _log(rng, 32, 1200),
                r=8 * rng.randint(1, 16), adapters=rng.randint(1, 6), order=rng.choice(["runs", "runs", "shuffled"]),
                none=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _dims(case):
    return tuple(int(d) for d in case["dims"].split(","))


def _positions(case, rs):
    """[S, axes] positions of a packed sequence: a quarter of text-like tokens (time alone runs on), then patches in
    (time, height, width) order on a grid; ``frac`` stretches time by a frame-rate ratio, in fp32."""

    s, n = case["s"], len(_dims(case))
    text = s // 4
    w = 8 + int(rs.randint(0, 40))
    h = 8 + int(rs.randint(0, 20))
    i = np.arange(s, dtype=np.int64)
    v = np.maximum(i - text, 0)
    t = np.where(i < text, i, text + v // (h * w))
    cols = [t, np.where(i < text, 0, (v // w) % h), np.where(i < text, 0, v % w)][:n]
    pos = np.stack(cols, 1)
    if case["frac"]:
        p = pos.astype(np.float32)
        p[:, 0] *= np.float32(24.0 / (15 + int(rs.randint(0, 15))))
        return torch.from_numpy(p)
    return torch.from_numpy(pos.astype(np.int32))


def _spans(case):
    """int32 [S] first and end key of every token: its request (full attention), or the prefix and the frames up to
    its own; padding rows see nothing."""

    s = case["s"]
    lo, hi = np.zeros(s, np.int32), np.zeros(s, np.int32)
    at = 0
    for n in (int(x) for x in case["docs"].split(",")):
        i = np.arange(n)
        lo[at:at + n] = at
        if case["frame"]:
            p = min(case["prefix"], n)
            seen = np.where(i < p, p, p + ((i - p) // case["frame"] + 1) * case["frame"])
            hi[at:at + n] = at + np.minimum(seen, n)
        else:
            hi[at:at + n] = at + n
        at += n
    return lo, hi


def _rows(case, rs):
    m, n = case["m"], case["adapters"]
    first = -1 if case["none"] else 0
    kinds = np.arange(first, n)
    if case["order"] == "shuffled":
        return rs.choice(kinds, m).astype(np.int32)
    cuts = np.sort(rs.randint(0, m + 1, len(kinds) - 1))
    return np.repeat(kinds, np.diff(np.concatenate([[0], cuts, [m]]))).astype(np.int32)


def prepare(case, seed):
    rs = np.random.RandomState(seed % (1 << 31))
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    if case["op"] == "table":
        st["pos"] = _positions(case, rs).cuda()
    elif case["op"] == "qknorm":
        st["pos"] = _positions(case, rs).cuda()
        s, hq, hk = case["s"], case["hq"], case["hk"]
        qkv = torch.randn((s, (hq + 2 * hk) * HD), generator=g, device="cuda").mul_(2.0).to(torch.bfloat16)
        st["q"] = qkv[:, :hq * HD].view(s, hq, HD)
        st["k"] = qkv[:, hq * HD:(hq + hk) * HD].view(s, hk, HD)
        st["qw"] = 1 + 0.02 * torch.randn(HD, generator=g, device="cuda")
        st["kw"] = 1 + 0.02 * torch.randn(HD, generator=g, device="cuda")
    elif case["op"] == "attn":
        # rows as a block's qkv projection leaves them, q and k of unit variance as after their norms
        s, hq, hk = case["s"], case["hq"], case["hk"]
        qkv = torch.randn((s, (hq + 2 * hk) * HD), generator=g, device="cuda").to(torch.bfloat16)
        cut = [hq * HD, (hq + hk) * HD]
        st["q"] = qkv[:, :cut[0]].view(1, s, hq, HD).transpose(1, 2)
        st["k"] = qkv[:, cut[0]:cut[1]].view(1, s, hk, HD).transpose(1, 2)
        st["v"] = qkv[:, cut[1]:].view(1, s, hk, HD).transpose(1, 2)
        lo, hi = _spans(case)
        st["lo"], st["hi"] = torch.from_numpy(lo).cuda(), torch.from_numpy(hi).cuda()
    else:
        m, k, n, r, a = (case[x] for x in ("m", "k", "n", "r", "adapters"))
        rows = _rows(case, rs)
        st["x"] = torch.randn((m, k), generator=g, device="cuda").to(torch.bfloat16)
        st["y"] = torch.randn((m, n), generator=g, device="cuda").to(torch.bfloat16)
        st["a"] = (torch.randn((a, r, k), generator=g, device="cuda") / math.sqrt(k)).to(torch.bfloat16)
        st["b"] = (torch.randn((a, n, r), generator=g, device="cuda") / math.sqrt(r)).to(torch.bfloat16)
        st["scale"] = torch.rand(a, generator=g, device="cuda") + 0.5
        st["rows"] = torch.from_numpy(rows).cuda()
    return st


# ------------------------------------------------------------------------------------------------ one pass
def _angles(pos, dims, theta):
    parts = [pos[:, i:i + 1].double() * theta ** (-2.0 * torch.arange(d // 2, dtype=torch.float64, device="cuda") / d)
             for i, d in enumerate(dims)]
    return torch.cat(parts, 1)


def _plain_norm_rope(x, w, cos, sin):
    half = cos.shape[1]
    y = x.float()
    y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + EPS) * w
    c, s = cos[:, None, :], sin[:, None, :]
    a, b = y[..., :half], y[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, y[..., 2 * half:]], -1).to(torch.bfloat16)


def _plain_attention(st):
    s, hq, hk = st["s"], st["hq"], st["hk"]
    j = torch.arange(s, device="cuda")
    hidden = (j < st["lo"][:, None]) | (j >= st["hi"][:, None])
    out = torch.empty((s, hq, HD), dtype=torch.bfloat16, device="cuda")
    for h in range(hq):                  # [S, S] scores of one head at a time: all heads' would not fit
        q, k, v = st["q"][0, h].float(), st["k"][0, h * hk // hq].float(), st["v"][0, h * hk // hq].float()
        x = (q @ k.t()).mul_(HD ** -0.5).masked_fill_(hidden, -math.inf)
        top = x.amax(1, keepdim=True).clamp_min_(-1e30)
        p = x.sub_(top).exp_()
        out[:, h] = ((p @ v) / p.sum(1, keepdim=True).clamp_min_(1e-30)).to(torch.bfloat16)
    return out.transpose(0, 1)[None]


def run(state):
    st = state
    if own:
        attention, kernels, linear = _tfvideo()
        if st["op"] == "table":
            return kernels.rope_axes(st["pos"], _dims(st), st["theta"])
        if st["op"] == "qknorm":
            return kernels.qknorm_rope_axes(st["q"], st["k"], st["qw"], st["kw"], st["pos"], _dims(st), st["theta"],
                                            EPS, out_q=torch.empty_like(st["q"], memory_format=torch.contiguous_format),
                                            out_k=torch.empty_like(st["k"], memory_format=torch.contiguous_format))
        if st["op"] == "attn":
            return attention.bf16(st["q"], st["k"], st["v"], attention.SpanMask(st["lo"], st["hi"]))
        return linear.adapter_add(st["y"], st["x"], st["a"], st["b"], st["rows"], st["scale"],
                                  out=torch.empty_like(st["y"]))
    if st["op"] == "table":
        ang = _angles(st["pos"], _dims(st), st["theta"])
        c, s = torch.cos(ang).float(), torch.sin(ang).float()
        return torch.stack([c, -s, s, c], -1).view(st["s"], -1, 2, 2)
    if st["op"] == "qknorm":
        ang = _angles(st["pos"], _dims(st), st["theta"])
        c, s = torch.cos(ang).float(), torch.sin(ang).float()
        return _plain_norm_rope(st["q"], st["qw"], c, s), _plain_norm_rope(st["k"], st["kw"], c, s)
    if st["op"] == "attn":
        return _plain_attention(st)
    n, r, k = st["a"].shape
    t = (st["x"].float() @ st["a"].float().view(n * r, k).t()).view(-1, n, r)
    mine = st["rows"][:, None] == torch.arange(n, device="cuda")
    t = torch.where(mine[:, :, None], t * st["scale"][:, None], torch.zeros((), device="cuda")).view(-1, n * r)
    return (st["y"].float() + t @ st["b"].float().transpose(1, 2).reshape(n * r, -1)).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ the least work
def work(case):
    op = case["op"]
    if op == "table":
        pairs = case["s"] * sum(_dims(case)) // 2
        return {"bytes": pairs * 16 + case["s"] * len(_dims(case)) * 4, "flops": pairs * 3}
    if op == "qknorm":
        n = case["s"] * (case["hq"] + case["hk"]) * HD
        return {"bytes": n * 4 + case["s"] * len(_dims(case)) * 4 + 8 * HD, "flops": n * 7}
    if op == "attn":
        lo, hi = _spans(case)
        seen = int((hi.astype(np.int64) - lo).sum())
        return {"bytes": case["s"] * (2 * case["hq"] + 2 * case["hk"]) * HD * 2 + 8 * case["s"],
                "flops": 4 * HD * case["hq"] * seen}
    m, k, n, r, a = (case[x] for x in ("m", "k", "n", "r", "adapters"))
    on = m * a // (a + 1) if case["none"] else m      # rows that have an adapter, about
    return {"bytes": 2 * (on * k + 2 * m * n + a * r * (k + n)) + 4 * m, "flops": 2 * on * r * (k + n)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _rotations(case, pos):
    """complex128 [S, pairs]: e^(i * position * frequency), pairs of the axes one after another."""

    out = []
    for axis, d in enumerate(_dims(case)):
        f = np.array([math.exp(-math.log(case["theta"]) * (2 * j) / d) for j in range(d // 2)])
        ang = torch.outer(pos[:, axis].to(torch.float64), torch.from_numpy(f).to(pos.device))
        out.append(torch.polar(torch.ones_like(ang), ang))
    return torch.cat(out, 1)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "table":
        z = _rotations(case, st["pos"])
        return torch.view_as_real(torch.stack([z, 1j * z], -1)).transpose(-1, -2).contiguous()
    if op == "qknorm":
        z = _rotations(case, st["pos"])[:, None]
        half = z.shape[-1]

        def one(x, w):
            x, w = x.double(), w.double()
            x = x * w * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / HD + EPS)
            u = torch.complex(x[..., :half], x[..., half:2 * half]) * z
            return torch.cat([u.real, u.imag, x[..., 2 * half:]], -1)

        return one(st["q"], st["qw"]), one(st["k"], st["kw"])
    if op == "attn":
        s, hq, hk = case["s"], case["hq"], case["hk"]
        out = torch.zeros((1, hq, s, HD), dtype=torch.float64, device="cuda")
        lo, hi = _spans(case)
        step = 2048
        for h in range(hq):
            kv = h // (hq // hk)
            q, k, v = (t[0, i].double() for t, i in ((st["q"], h), (st["k"], kv), (st["v"], kv)))
            for a in range(0, s, step):
                b = min(s, a + step)
                live = hi[a:b] > lo[a:b]
                if not live.any():
                    continue
                c, d = int(lo[a:b][live].min()), int(hi[a:b][live].max())
                j = torch.arange(c, d, device="cuda")
                keep = (j >= st["lo"][a:b, None]) & (j < st["hi"][a:b, None])
                x = torch.einsum("id,jd->ij", q[a:b], k[c:d]) / math.sqrt(HD)
                e = torch.where(keep, torch.exp(x - x.max(1, keepdim=True).values), 0.0)
                den = e.sum(1, keepdim=True)
                out[0, h, a:b] = torch.where(den > 0, torch.einsum("ij,jd->id", e, v[c:d]) / den, 0.0)
        return out
    out = st["y"].double()
    rows = st["rows"]
    for i in range(case["adapters"]):
        at = torch.nonzero(rows == i)[:, 0]
        t = st["x"][at].double() @ st["a"][i].double().T
        out[at] += st["scale"][i].double() * (t @ st["b"][i].double().T)
    return out
