"""Producer threads of the dataloaders are over before the interpreter ends its threads."""

import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[2]

SCRIPT = """
import atexit, threading

def report():  # registered first, so it runs last
    print("alive", sum(t.is_alive() for t in threading.enumerate() if t is not threading.main_thread()))

atexit.register(report)
import itertools, torch
from mint_b200.data.dist.pretrain import prefetch
batches = prefetch((torch.randint(0, 9, (64, 64)) for _ in itertools.count()), 2)
next(batches)
closed = prefetch(iter([1, 2]), 2)
assert list(closed) == [1, 2]
"""


def test_no_producer_is_left_at_exit():
    run = subprocess.run([sys.executable, "-c", SCRIPT], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr[-2000:]
    assert run.stdout.split() == ["alive", "0"]
