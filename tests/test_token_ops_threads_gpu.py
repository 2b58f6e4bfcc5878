"""First calls of a process from several threads at once, each on a stream of its own."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import threading
import torch
from sketchpad_b200 import Int4Linear, PagedKVCache

BF, HF, E4M3 = torch.bfloat16, torch.float16, torch.float8_e4m3fn
cuda = dict(device="cuda")
calls = []
for group in (32, 64, 128):
    for zeros in (False, True):
        for sdt in (HF, BF):
            q = torch.randint(0, 256, (96, 128), dtype=torch.uint8, **cuda)
            s = torch.rand(256 // group, 96, **cuda).to(sdt)
            z = torch.randint(0, 16, s.shape, dtype=torch.uint8, **cuda) if zeros else None
            lin = Int4Linear(q, s, z, group_size=group)
            for M in (1, 12, 20):
                x = torch.randn(M, 256, **cuda).to(BF)
                calls.append(lambda lin=lin, x=x: lin(x))
table = torch.arange(4, dtype=torch.int32, **cuda)[None]
lens = torch.full((1,), 50, dtype=torch.int32, **cuda)
for D in (64, 128, 256):
    for dtype, cdt in ((BF, BF), (HF, HF), (BF, E4M3), (HF, E4M3)):
        for page in (16, 20):
            k, v = (torch.randn(4, page, 2, D, **cuda).to(cdt) for _ in range(2))
            sc = (torch.ones(2, **cuda),) * 2 if cdt == E4M3 else ()
            cache, q = PagedKVCache(k, v, *sc), torch.randn(1, 4, D, **cuda).to(dtype)
            calls.append(lambda cache=cache, q=q: cache.attend(q, table, lens))
torch.cuda.synchronize()
N = 6
outs, errors = [[None] * N for _ in calls], []
barrier = threading.Barrier(N)

def work(i):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        for c, call in enumerate(calls):
            barrier.wait(60)
            try:
                outs[c][i] = call()
            except Exception as e:
                errors.append(str(e))
    stream.synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not errors, (len(errors), errors[0])
assert all(torch.equal(o[0], x) for o in outs for x in o)
print("same", len(calls))
"""


def test_first_calls_of_several_threads():
    root = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..")
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=root, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0 and "same" in r.stdout, r.stderr[-1500:]
