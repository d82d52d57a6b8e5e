"""perf/operators.py beside a torch program: what it returns may be used, and what it was given dropped, by torch work
that waits for nothing.  In a process of its own, which loads torch's HIP runtime before the engine's library."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import gc, sys
import torch
sys.path.insert(0, "perf")
import operators as ops

ops.own = True
for case in ops.listed():
    if case["name"] not in ("cache_long_q4_0", "attn_bank_q8_0", "product_fc1_q8_0"):
        continue
    state = ops.prepare(case, 3)
    for _ in range(3):
        out = ops.run(state)
        out = list(out) if isinstance(out, (list, tuple)) else [out]
        early = [x.clone() for x in out]
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(early, out)), case["name"]
        # the inputs change behind the call, which has them as they were
        for x in out:
            x.zero_()
    keep = early
    out = ops.run(state)
    out = [x.clone() for x in (out if isinstance(out, (list, tuple)) else [out])]
    size = sum(x.numel() * x.element_size() for x in state.values() if isinstance(x, torch.Tensor))
    del state
    gc.collect()
    junk = torch.full((size,), 0xA5, dtype=torch.uint8, device="cuda")  # memory that the state held
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(keep, out)), case["name"]
    del junk
    print(case["name"], "ok", flush=True)
"""


def test_torch_work_follows_the_engines(tmp_path):
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.count(" ok") == 3, (r.returncode, r.stdout[-500:], r.stderr[-1500:])
