"""Worker of tests/test_packed_parallel_gpu.py (run under torchrun): a packed batch (positions over three axes, key spans)
through the Ulysses engine against the single-GPU engine on the same seeded inputs and weights, over three forwards
(dynamic, then delayed scales).  argv: backend (gloo: every rank on GPU 0, exchanges by all-to-all through the host, so
that no kernel waits for another rank's; nccl: a GPU each, exchanges in the producing kernels), attention, tokens."""
import os, sys
from datetime import timedelta
root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(root, "minimax-h3-tensorfold-rtx_b200")); sys.path.insert(0, root)
import torch, torch.distributed as dist
backend, attn, S = sys.argv[1], sys.argv[2], int(sys.argv[3])
rank, world = int(os.environ["RANK"]), int(os.environ["WORLD_SIZE"])
torch.cuda.set_device(rank if backend == "nccl" else 0)
dist.init_process_group(backend, timeout=timedelta(seconds=120))
from tfvideo import attention as A, kernels as K, minimax_h3 as M, native as N
cfg = M.Config(layers=2, dim=512, heads=8, head_dim=128, ffn=1024, act="gelu", t_dim=8)
g = torch.Generator().manual_seed(5)
x = torch.randn(S, cfg.dim, generator=g).to(torch.bfloat16).cuda()
t_emb = torch.randn(2, cfg.t_dim, generator=g).cuda()
segs = [(0, 100, 0), (100, S, 3)]
i = torch.arange(S)
p = K.AxialPositions(torch.stack([i // 40, (i // 8) % 5, i % 8], 1).to(torch.int32), (44, 42, 42))   # on the host
mask = A.SpanMask.frames([S // 2 + 77, 0, S // 2 - 90], 60, 50, S) if attn == "bf16" else None


def engine():
    e = M.MiniMaxH3Engine.synthetic(cfg, seed=1, device="cuda", attn=attn)
    e.attn_mask = mask
    return e


eng, ref = engine(), engine()
ref.sp = None
n = S // world
for f in range(3):
    out = eng.forward(x[rank * n:(rank + 1) * n].clone(), t_emb, segs, p)
    full = ref.forward(x.clone(), t_emb, segs, p)
mine = full[rank * n:(rank + 1) * n]
fused = eng._buf.peers is not None
try:
    eng.set_adapters({(0, "qkv"): None}, None)
    refused = False
except ValueError:
    refused = True
print(f"RESULT rank={rank} world={world} fused={fused} bitwise={torch.equal(out, mine)} moved={not torch.equal(mine, x[rank * n:(rank + 1) * n])} "
      f"refused={refused} status={N.device_status()}", flush=True)
dist.barrier()
dist.destroy_process_group()
