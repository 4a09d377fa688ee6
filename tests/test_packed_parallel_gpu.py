"""A packed batch under Ulysses sequence parallelism: positions and key spans through engines whose tokens are sharded over
two ranks must give exactly the single-GPU engine's rows.

On one GPU the two ranks are processes that exchange by gloo's all-to-all through the host (the engine's path for library
attention and bf16): each rank norms and rotates its own tokens from their positions, the second rank's starting in the
middle of the sequence, and attends over every token with its share of the heads.  The exchanges inside the producing
kernels need two GPUs."""

from __future__ import annotations

import os
import subprocess
import sys

import pytest
import torch

from helpers import need_gpu
from test_parallel_gpu import ROOT, _port

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("backend,attn,S", [("gloo", "bf16", 1024), ("gloo", "bf16", 2304), ("gloo", "fp8", 1024),
                                            ("nccl", "fp8", 1024)])
def test_packed_batch_over_two_ranks(backend, attn, S):
    need_gpu()
    if backend == "nccl" and torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")


    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node", "2", "--master-addr", "127.0.0.1",
           "--master-port", str(_port()), str(ROOT / "tests" / "packed_sp_worker.py"), backend, attn, str(S)]
    r = subprocess.run(cmd, cwd=ROOT, env=dict(os.environ, NCCL_NVLS_ENABLE="0"), capture_output=True, text=True,
                       timeout=300)
    out = r.stdout + r.stderr
    assert r.returncode == 0, out[-3000:]
    lines = sorted(line[line.index("RESULT"):] for line in out.splitlines() if "RESULT" in line)
    assert lines == [f"RESULT rank={k} world=2 fused={backend == 'nccl'} bitwise=True moved=True refused=True status=0"
                     for k in range(2)], lines
