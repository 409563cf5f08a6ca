"""The operators over caller-owned pages in a process of their own whose first
call of them is captured into a graph: nothing may depend on an eager call."""
import os
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

CHILD = """
import sys
import torch
sys.path[:0] = [{root!r} + "/vibevoice.cpp_b200", {root!r} + "/tests"]
import vvq2
from test_gpu_paged_ops import Chunk, check_weights
op, heads, seqs = {case}
c = Chunk(seqs, heads, torch.float16, seed=71).gpu()
w0 = torch.rand((1, len(seqs), c.nkv, c.max_kv), device="cuda:0")
kl, dst = c.kl, torch.arange(len(seqs), dtype=torch.int32, device="cuda:0")[:, None].contiguous()
k = torch.randn((2 * len(seqs) + 1, c.nkv, 64, c.hd), device="cuda:0").half()
some = vvq2.Pages(k, k.clone(), dst + len(seqs))
lens = torch.full_like(kl, 60)
lse0 = torch.zeros((c.total, c.nq), device="cuda:0")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    if op == "attend":
        out, lse = c.attend()
    elif op == "weigh":
        w = vvq2.attention_key_weights(c.qd, lse0, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    else:
        kept, new_len, w_out = vvq2.pages_evict(some, dst, lens, w0[:, :, :, :60].contiguous(), 20, 2, 5)
for _ in range(2):
    g.replay()
torch.cuda.synchronize()
if op == "attend":
    c.check(out, lse)
elif op == "weigh":
    again = vvq2.attention_key_weights(c.qd, lse0, c.pages, c.qs, c.kl, c.max_q, c.max_kv)
    for s, (_, kv) in enumerate(seqs):
        assert torch.equal(w[s, :, :kv], again[s, :, :kv])
    check_weights(c, lse0, w, None)
else:
    assert new_len.tolist() == [20] * len(seqs) and (kept[..., :2] == torch.arange(2, device="cuda:0")).all()
    assert torch.equal(some.k[:len(seqs)].gather(2, torch.arange(20, device="cuda:0")[None, None, :, None].expand(
        len(seqs), c.nkv, 20, c.hd)), some.k[len(seqs):2 * len(seqs)].gather(2, kept.reshape(
        len(seqs), c.nkv, 20)[..., None].expand(-1, -1, -1, c.hd).long()))
print("captured")
"""

FEW = [(1, 3000), (2, 90)]
LONG = [(300, 300), (5, 2000)]


@pytest.mark.parametrize("case", [("attend", (14, 2, 64), FEW), ("attend", (28, 4, 128), LONG),
                                  ("attend", (14, 2, 64), LONG), ("weigh", (28, 4, 128), FEW),
                                  ("weigh", (128, 1, 64), LONG), ("evict", (14, 2, 64), FEW)],
                         ids=lambda c: f"{c[0]}-{c[1][2]}-{c[2][0][0]}")
def test_the_first_call_may_be_captured(vv, case):
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=str(ROOT), case=repr(case))], capture_output=True,
                       text=True, timeout=200, env=dict(os.environ))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-3000:]
