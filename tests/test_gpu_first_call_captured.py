"""A process whose very first calls of the decoder operators are made under stream capture: they need no warm-up."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

CHILD = r"""
import sys
sys.path[:0] = [sys.argv[1], sys.argv[1] + "/tests"]
import torch
import __graft_entry__ as entry
pkg = entry.load_package()
lib = pkg.load()
import decoder_reference as dr
rows = int(sys.argv[2])
c = dr.Cache(pkg, [(rows, 300), (rows, rows)], page=32, heads=2, dim=64, kv="i8", seed=1)
x = torch.randn((2 * rows, 8 * 64), device="cuda")
n, out, final = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
empty = pkg.LogitsParams()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    st = dr.stream()
    assert lib.htp_b200_add_rms_norm(None, n.data_ptr(), x.data_ptr(), None, None, None, 0, None, 1.0, 1e-5, 512, 2 * rows, 0, st) == 0
    assert lib.htp_b200_kv_append(dr.ref(c.desc()), None, n.data_ptr(), 512, n.data_ptr() + 512, 512, None, 0, None, 0, 0, 0, 0, st) == 0
    assert lib.htp_b200_attn_paged(out.data_ptr(), 512, n.data_ptr(), 512, dr.ref(c.desc()), 8, 0, 0.125, 0, rows, 300, None, 0, st) == 0
    assert lib.htp_b200_logits_process(final.data_ptr(), out.data_ptr(), 512, 2 * rows, 512, dr.ref(empty), st) == 0
graph.replay()
torch.cuda.synchronize()
ref, mass, worst = dr.attention(c, n, 8, 0.125, 0)
assert ((out.double().view_as(ref) - ref).abs() <= dr.attention_bound(ref, mass, worst, True, 300)).all()
assert torch.equal(final, out) and lib.htp_b200_stream_status(torch.cuda.current_stream().cuda_stream) == 0
print("ok")
"""


@pytest.mark.parametrize("rows", [1, 40])
def test_first_calls_under_capture(rows):
    root = Path(__file__).resolve().parents[1]
    done = subprocess.run([sys.executable, "-c", CHILD, str(root), str(rows)],
                          capture_output=True, text=True, timeout=240)
    assert done.returncode == 0 and done.stdout.strip().endswith("ok"), done.stderr[-2000:]
