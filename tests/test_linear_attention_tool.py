"""Linear attention through the command line tool: compiled by the installed ROCm's compiler, not the one that came with torch, on inputs
from files, its results against float64."""
import os
import subprocess

import pytest
import torch

import linear_reference as ref
from test_linear_attention import check_forward, check_gradient, describe, describe_grad, make
from test_linear_attention_schedules import schedules
from test_linear_attention_sources import TOOL

CASES = [
    (("bfloat16", "BSND", 2, 4, 4, 2, 64, 64, "slow", True, None), describe), (("bfloat16", "BSND", 2, 150, 4, 2, 128, 128, "slow", True, None), describe),
    (("float16", "BNSD", 1, 100, 2, 1, 256, 192, "fast", True, None), describe), (("bfloat16", "BSND", 1, 1500, 2, 2, 64, 64, "slow", True, None), describe),
    (("bfloat16", "BSND", 8, 130, 32, 32, 128, 128, "slow", False, None), describe), (("bfloat16", "BSND", 2, 150, 4, 2, 64, 40, "slow", True, None), describe_grad),
    (("float16", "BSND", 1, 70, 4, 4, 64, 64, "slow", False, None), describe_grad), (("bfloat16", "BSND", 1, 70, 2, 2, 256, 256, "mixed", True, None), describe_grad),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case,f", CASES, ids=lambda c: "-".join(str(x) for x in c) if isinstance(c, tuple) else c.__name__)
def test_results_of_the_tool(case, f, tmp_path, monkeypatch):
    t, layout = make(case), case[1]
    text, inputs = f(t, layout, last=case[9]) if f is describe else f(t, layout)
    (tmp_path / "x.info").write_text(text)
    for i, x in enumerate(inputs):
        (tmp_path / ("arg%d.bin" % i)).write_bytes(x.contiguous().view(torch.uint8).numpy().tobytes())
    out = tmp_path / "out"
    out.mkdir()
    env = dict(os.environ, AKG_HIP_NO_CACHE="1")
    command = lambda verb, *more: subprocess.run([TOOL, verb, str(tmp_path / "x.info"), *more], capture_output=True, text=True, timeout=100, env=env)   # noqa: E731
    done = command("run", "-n", "1", "-r", "1", "--inputs", str(tmp_path), "--dump", str(out))
    assert done.returncode == 0, (done.returncode, done.stderr[-500:])
    found = schedules(command("emit").stdout)
    monkeypatch.setattr(ref, "CHUNK", 32 * found[-1][0] if found else ref.CHUNK)   # (which terms are rounded together)
    like = {"q": t["q"], "k": t["k"], "v": t["v"], "out": t["dout"], "state": t.get("state")}
    order = [like[n] for n in (("q", "k", "v", "state") if f is describe_grad else ("out", "state")) if like[n] is not None]
    got = [torch.frombuffer(bytearray((out / ("arg%d.bin" % (len(inputs) + j))).read_bytes()), dtype=x.dtype).view(x.shape) for j, x in enumerate(order)]
    (check_forward if f is describe else check_gradient)(t, layout, got)
