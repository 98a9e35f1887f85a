"""First calls that come from several threads at once."""
import subprocess
import sys
import threading
import time

import pytest


def test_threads_share_one_default_context(T, monkeypatch):
    from thrml_rs_b200 import engine
    made = []

    class Slow:
        def __init__(self, device_id):
            time.sleep(0.05)  # as the driver's start does, outside the interpreter's lock
            made.append(self)
    monkeypatch.setattr(engine, "Context", Slow)
    monkeypatch.setattr(engine, "_default_ctx", {})
    got = []
    threads = [threading.Thread(target=lambda: got.append(engine.default_context(0))) for _ in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(made) == 1 and all(g is made[0] for g in got) and len(got) == 8


FIRST = """
import threading, torch
import __graft_entry__ as graft
T = graft.load_package()
torch.cuda.init()
x = [torch.randn(m, 512, device="cuda") for m in (1, 30, 64, 700)]
w = torch.randint(-127, 128, (9000, 512), device="cuda", dtype=torch.int8)
ws = torch.rand(9000, device="cuda")
i, t = torch.zeros(700, 2, dtype=torch.int32, device="cuda"), torch.zeros(700, 2, device="cuda")
torch.cuda.synchronize()
results, start = {}, threading.Barrier(8)
def work(n):
    start.wait()
    with torch.cuda.stream(torch.cuda.Stream()):
        out = [T.int8_linear(a, w, ws) for a in x]
        out += [T.adjust_logits(out[3]), T.draw_categories(out[3], 5), *T.distill_step(out[3], i, t)]
        torch.cuda.current_stream().synchronize()
    results[n] = out
threads = [threading.Thread(target=work, args=(n,)) for n in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(results) == 8
for r in results.values():
    assert all(torch.equal(a, b) for a, b in zip(r, results[0]))
print("all the same")
"""


@pytest.mark.gpu
def test_first_readout_calls_from_eight_threads():
    done = subprocess.run([sys.executable, "-c", FIRST], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "all the same" in done.stdout, done.stderr[-2000:]


CLOSED = """
import torch
import __graft_entry__ as graft
T = graft.load_package()
x = torch.ones(2, 32, device="cuda")
T.quantize_rows(x)
torch.cuda.synchronize()
T.default_context(0).close()
try:
    T.quantize_rows(x)
except T.ThrmlError as e:
    print("refused", e)
"""


@pytest.mark.gpu
def test_a_closed_context_is_refused():
    done = subprocess.run([sys.executable, "-c", CLOSED], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "refused" in done.stdout and "null context" in done.stdout, done.stderr[-2000:]
