"""The ring of copies of the norms and activations in bytes, when its waits run out: with no poll to a wait every CTA gives up at its first row, waits for its copies and leaves."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
CODE = """
import torch
from seq2seqsharp_b200 import _native as N
from seq2seqsharp_b200.ops import Ops
T, eps = torch.%(t)s, %(eps)r

def ends(call):
    out = call()
    try:
        N.call("TSB200_Synchronize", 0, 1)
        print("nothing was reported")
    except N.TSB200Error as e:
        print("gave up" if "gave up waiting" in str(e) else e)
    N.call("TSB200_Synchronize", 0, 1)   # reported once

for rows, d, two in ((1203, 1024, False), (1203, 4096, False), (1203, 4096, True), (700, 8192, True), (700, 12288, True), (700, 16384, True)):
    x, r = (torch.randn(rows, d, device="cuda").to(T) for _ in range(2))
    gain = torch.ones(d, device="cuda", dtype=T)
    ends(lambda: Ops.RMSNormInt8(None, x, r if two else None, gain, eps))
    ends(lambda: Ops.RowsInt8(None, x, r if two else None, N.ACT_SILU))
    # the context is as it was: the same rows, a few at a time, which no ring brings
    want = x.double()
    for i in range(0, 300, 100):
        q, scale = Ops.RowsInt8(None, x[i: i + 100])
        v = want[i: i + 100] * 127 / want[i: i + 100].abs().amax(1, keepdim=True)
        assert (q.double() - v).abs().max().item() <= 0.5 + 381 * 2.0 ** -24 and scale.isfinite().all()
    N.call("TSB200_Synchronize", 0, 1)
print("usable", float(torch.ones(4, device="cuda").sum()))
"""


@pytest.mark.parametrize("t", ["float16", "bfloat16"])
@pytest.mark.parametrize("eps", [1e-6, 0.0])
def test_every_ring_reports_a_wait_that_ran_out_and_ends(cuda, t, eps):
    r = subprocess.run([sys.executable, "-c", CODE % dict(t=t, eps=eps)], capture_output=True, text=True, timeout=120,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), env=dict(os.environ, TSB200_WAIT_LIMIT="0"))
    assert r.returncode == 0, r.stderr
    assert r.stdout.split("\n")[:-1] == ["gave up"] * 12 + ["usable 4.0"], r.stdout


@pytest.mark.parametrize("limit", ["x", "-1"])
def test_other_limits_are_no_limit_of_none(cuda, limit):
    code = CODE.split("for rows")[0] % dict(t="float16", eps=1e-6) + "x = torch.randn(1203, 4096, device='cuda').to(T)\nends(lambda: Ops.RowsInt8(None, x))\n"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       env=dict(os.environ, TSB200_WAIT_LIMIT=limit))
    assert r.returncode == 0 and r.stdout == "nothing was reported\n", r.stdout + r.stderr
