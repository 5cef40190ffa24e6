"""Several host threads, each with a stream of its own, make their first calls of a process at the same time: every thread gets the results of a call on its own."""
import subprocess
import sys

import pytest

from dscuda_b200.library import ROOT

pytestmark = pytest.mark.gpu

PROGRAM = """
import threading
import torch
from dscuda_b200 import flash

def work(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape: torch.randn(*shape, device="cuda", generator=g).bfloat16()
    query, key, value, dout = draw(2, 90 + seed, 8, 128), draw(2, 700, 2, 128), draw(2, 700, 2, 128), draw(2, 90 + seed, 8, 128)
    cache = [torch.zeros(50, 2, 32, 128, dtype=torch.int8, device="cuda") for _ in range(2)] + [torch.zeros(50, 2, device="cuda") for _ in range(2)]
    table, positions = torch.arange(50, device="cuda").int().view(2, 25), torch.arange(180 + 2 * seed, device="cuda").int().view(1, 2, -1)
    lengths = torch.tensor([700, 300 + seed], dtype=torch.int32, device="cuda")
    def step():
        results = []
        for _ in range(8):
            turned, _ = flash.rope(query, None, positions, [64])
            flash.cache_append(*cache, key, value, table, None, lengths)
            results = [turned, *cache, *flash.decode(turned[:, :3].contiguous(), *cache, table, lengths, 0.1)]
            out, lse = flash.cross_forward(turned, key, value, 0.1, lengths)
            results += [out, lse, *flash.cross_forward(turned[:, :1].contiguous(), key, value, 0.1, lengths), *flash.cross_backward(dout, out, lse, turned, key, value, 0.1, lengths)]
        return results
    return step

steps = [work(seed) for seed in range(4)]
torch.cuda.synchronize()
found, ready = [None] * 4, threading.Barrier(4)

def thread(i):
    stream = torch.cuda.Stream()
    ready.wait()
    with torch.cuda.stream(stream):
        found[i] = [x.clone() for x in steps[i]()]
    stream.synchronize()

threads = [threading.Thread(target=thread, args=(i,)) for i in range(4)]
for t in threads:
    t.start()
for t in threads:
    t.join()
for i in range(4):
    alone = steps[i]()
    torch.cuda.synchronize()
    assert len(alone) == 14 and all(torch.equal(a, b) for a, b in zip(found[i], alone)), i
assert flash.device_status() == 0
print("the same")
"""


def test_threads(gpu):
    done = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "the same" in done.stdout, done.stderr[-2000:]
