"""Products captured into a graph in a program whose only call before was another one of the image calls: one call on a device is what the header asks for."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import sys, torch
sys.path.insert(0, {root!r})
import homura_b200 as hm

MX, E, M, K, N = 10, 3, 5, 300, 140
x, w = torch.randn(M, K, device="cuda"), torch.randn(E * N, K, device="cuda")
each = hm.image_bytes(MX, N, K)
xi, wi = torch.zeros(hm.image_bytes(MX, M, K), dtype=torch.uint8, device="cuda"), torch.zeros(E * each, dtype=torch.uint8, device="cuda")
ids = torch.tensor([0, 2, -1, 1, 2], dtype=torch.int32, device="cuda")
plan = torch.zeros(hm.expert_plan_ints(M, E), dtype=torch.int32, device="cuda")
gi = torch.zeros(hm.image_bytes(MX, hm.expert_plan_rows(M, E), K), dtype=torch.uint8, device="cuda")
wt, out = torch.ones(M, device="cuda"), [torch.zeros(M, N, device="cuda") for _ in range(5)]
for i in range(E):
    hm.image_pack((w[i * N :].data_ptr(), N), MX, K=K, image=wi.data_ptr() + i * each, stream=torch.cuda.current_stream().cuda_stream)
torch.cuda.synchronize()


def run():
    st = torch.cuda.current_stream().cuda_stream
    hm.image_pack((x.data_ptr(), M), MX, K=K, image=xi.data_ptr(), stream=st)
    hm.gemm_image((xi.data_ptr(), M), wi.data_ptr(), N, MX, K=K, y=out[0].data_ptr(), stream=st)
    hm.gemv_mx4((x.data_ptr(), M), wi.data_ptr(), N, K=K, y=out[1].data_ptr(), stream=st)
    hm.expert_plan((ids.data_ptr(), M), E, plan=plan.data_ptr(), stream=st)
    hm.image_pack((x.data_ptr(), M), MX, K=K, plan=plan.data_ptr(), pairs=M, experts=E, image=gi.data_ptr(), stream=st)
    hm.expert_gemm(gi.data_ptr(), wi.data_ptr(), plan.data_ptr(), N, MX, pairs=M, experts=E, K=K, y=out[2].data_ptr(), stream=st)
    hm.expert_gemv((x.data_ptr(), M), wi.data_ptr(), ids.data_ptr(), N, top=1, experts=E, K=K, y=out[3].data_ptr(), stream=st)
    hm.expert_sum((out[2].data_ptr(), M), ids.data_ptr(), wt.data_ptr(), top=1, experts=E, width=N, y=out[4].data_ptr(), stream=st)


g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    run()
g.replay()
torch.cuda.synchronize()
got = [y.clone() for y in out]
for y in out:
    y.zero_()
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, out)) and all(a.any() for a in got)
hm.dev_sync()
print("replayed")
"""


def test_products_are_captured_after_one_other_call():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", PROGRAM.format(root=root)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "replayed" in done.stdout, done.stderr[-2000:]
