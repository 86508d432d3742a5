"""The serving operators captured in a CUDA graph as the first call of a process: the context is
made, and every kernel loaded, inside the capture."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys
import torch
from runtimed_b200 import kv4, sampling

i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
rand = lambda *s: torch.randn(s, device="cuda")
pages, q, k = kv4.alloc_pages(4, 2, 128), rand(64, 16, 128), rand(64, 2, 128)
inv, at, tables = kv4.rope_frequencies(128, 1e4), torch.arange(64, dtype=torch.int32, device="cuda"), kv4.BlockTables(4, 4, 4, 64)
x, u, chunk = rand(64, 5000), torch.rand(64, device="cuda"), rand(300, 16, 128)
table, n, one, many = i32([[0, 1, 2, 3]]), i32([64]), i32([0, 64]), i32([0, 300])
call = dict(plan=lambda: tables.step(tables.length + 3) or tables.tok_pos, append=lambda: kv4.append(q, k, k, inv, at, at, pages),
            read=lambda: torch.stack(kv4.read(pages, at)), attention=lambda: kv4.attention(q, pages, table, one, n, 64, 64),
            chunk=lambda: kv4.attention(chunk, pages, table, many, n, 300, 64, out_dtype=torch.bfloat16),
            sample=lambda: sampling.sample(x, u))[sys.argv[1]]
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    got = call()
g.replay()
got = got.clone()
tables.set_lengths(torch.zeros_like(tables.length))
assert torch.equal(got, call())
print("alike")
"""


@pytest.mark.parametrize("what", ["plan", "append", "read", "attention", "chunk", "sample"])
def test_captured_first(what):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", PROGRAM, what], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip().endswith("alike"), r.stderr[-2000:]
