"""The paged operators' performance cases beside torch's own work: what a program
enqueues on torch's stream before a pass is seen by it, what it reads after it is
the pass's output, without a synchronization between them."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# (a process of its own: torch brings its HIP runtime, which has to be loaded first)
PROGRAM = """
import torch
from perf import operators as P

P.own = True
a = torch.randn(8192, 8192, device="cuda", dtype=torch.bfloat16)
for case in [c for c in P.listed() if c["name"] in ("append_batch", "decode_token", "prefill_short")]:
    one, two = P.prepare(case, 1), P.prepare(case, 2)
    torch.cuda.synchronize()
    for _ in range(20):
        b = a @ a  # some 20 ms before the new inputs are there
    one["q"].copy_(two["q"])
    got = P.run(one)
    got = (got[0] if isinstance(got, tuple) else got).clone()
    torch.cuda.synchronize()
    want = P.run(one)
    torch.cuda.synchronize()
    want = want[0] if isinstance(want, tuple) else want
    assert torch.equal(got, want), case["name"]
    print(case["name"], "ok", flush=True)
"""


def test_own_calls_are_ordered_with_torch():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=110,
                       env=dict(os.environ, PYTHONPATH=ROOT))
    print(r.stdout, r.stderr[-2000:], flush=True)
    assert r.returncode == 0 and r.stdout.count(" ok") == 3
