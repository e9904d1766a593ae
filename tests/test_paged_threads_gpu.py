"""Other Python threads run while a call of the paged operators waits for its
stream (PERSONA_STRICT_SLOTS=1, which is read once per process)."""

import os
import subprocess
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

CODE = """
import threading, time
import torch
import paged_ref as R
from persona import ops

bt = R.Batch([1, 1], [20, 30], 16, 2, 128, torch.float16)
bt.fill()
q, k = bt.randn(2, 8, 128), bt.randn(2, 2, 128)
p = torch.softmax(bt.randn(2, 50).float(), -1)
tok, acc = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
calls = [lambda: ops.paged_rope_cache(q, k, k, *bt.args(), 1e6, q_out=torch.empty_like(q)),
         lambda: ops.paged_cache_read(*bt.args(), torch.empty_like(k), torch.empty_like(k)),
         lambda: ops.paged_attention(q, *bt.args(), torch.empty_like(q), 0.1),
         lambda: ops.verify_draft(p, tok.clone(), None, bt.indptr, p[:, 0].clone(), p[:, 1].clone(), tok, acc)]
for call in calls:
    call()
torch.cuda.synchronize()
for call in calls:
    torch.cuda._sleep(800_000_000)  # about 0.4 s of the stream, which the call waits for
    ticks, t = 0, threading.Thread(target=call)
    t.start()
    start = time.perf_counter()
    while t.is_alive():
        time.sleep(0.005)
        ticks += 1
    took = time.perf_counter() - start
    print(took, ticks)
    assert took > 0.2 and ticks > 10
"""


def test_a_call_that_waits_lets_other_threads_run():
    env = dict(os.environ, PERSONA_STRICT_SLOTS="1",
               PYTHONPATH=os.pathsep.join([str(ROOT), str(ROOT / "multi-lora-llm-kernel_b200"), str(ROOT / "tests")]))
    r = subprocess.run([sys.executable, "-c", CODE], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
