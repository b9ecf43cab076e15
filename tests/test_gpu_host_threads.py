"""The fused block operators called from several host threads at once, each on its own stream: the bits of the calls
alone.  The shapes make one kernel ask for different amounts of shared memory (gated_linear's few-rows kernel by the
columns, the norm kernels' by the width), so that first calls raise its limit from several threads."""
import subprocess
import sys
import textwrap
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parent.parent

PROGRAM = textwrap.dedent("""
    import threading
    import torch
    from bee_b200 import tensor_cuda as tc

    def make(i):
        g = torch.Generator().manual_seed(i)
        t = lambda *shape, scale=1.0: (torch.randn(*shape, generator=g) * scale).bfloat16().cuda()
        cols = (16384, 12296)[i % 2]  # both in the 1024-thread block
        d, f = ((512, 2048), (64, 40000))[i % 2]  # one CTA per SM, and two
        return {"h": t(40, cols), "x": t(40, cols), "w": t(cols), "few": t(3, d), "wg": t(f, d, scale=0.05), "wu": t(f, d, scale=0.05),
                "logits": t(20, 9000 + 64 * i, scale=3.0), "targets": torch.arange(20).cuda()}

    def call(s):
        o = {k: torch.empty_like(s["x"]) for k in ("xo", "y", "dh", "dx")} | {k: torch.empty_like(s["w"]) for k in ("dw", "dp")}
        o |= {k: torch.empty(20, device="cuda") for k in ("lp", "ent", "m", "ls")} | {"out": s["few"].new_empty(3, s["wg"].shape[0])}
        for _ in range(3):
            tc.gated_linear(s["few"], s["wg"], s["wu"], o["out"], trans=True)
            tc.norm_gate_residual(s["h"], s["x"], o["xo"], o["y"], w_post=s["w"], w_pre=s["w"])
            tc.norm_gate_residual_backward(s["h"], s["x"], s["x"], s["h"], o["dh"], o["dx"], w_post=s["w"], w_pre=s["w"], dw_post=o["dw"],
                                           dw_pre=o["dp"])
            tc.token_logprobs(s["logits"], s["targets"], o["lp"], o["ent"], o["m"], o["ls"])
        return o

    N = 6
    sets, got, errors, gate = [make(i) for i in range(N)], [None] * N, [], threading.Barrier(N)
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                gate.wait(60)
                got[i] = call(sets[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            errors.append(f"{i}: {e}")

    threads = [threading.Thread(target=work, args=(i,)) for i in range(N)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    for i in range(N):
        want = call(sets[i])
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[i][k], want[k]), (i, k)
    print("threads ok")
""")


def test_first_calls_from_several_threads(cuda):
    r = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "threads ok" in r.stdout, r.stdout + r.stderr
