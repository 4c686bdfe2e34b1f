"""Sources of linear attention: they compile with the compiler of the installed ROCm too, which the command line tool uses
(a process that has imported torch uses the one that came with it), and say what they are."""
import os
import subprocess

import pytest

from akg_amd import driver, op_desc
from test_attention_ops import builder
from test_linear_attention import text_of

TOOL = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "akg_amd", "akg-hip")


def described(seq, dim, grad=False, state=True, slots=False, last=True, dtype="bfloat16", batch=2, heads=4, kv=2, lengths=False):
    """Text of a description of `batch` sequences of `seq` tokens."""
    shape = lambda h: (batch, seq, h, dim)   # noqa: E731
    s = ([7 if slots else batch, heads, dim, dim], "float32") if state else None
    more = dict(dout=shape(heads), dstate=s) if grad else dict(last_state=last, slots=([batch], "int32") if slots else None)
    return text_of(dtype=dtype, q=shape(heads), k=shape(kv), v=shape(kv), decay=([heads], "float32"), state=s, lengths=([batch], "int32") if lengths else None,
                   grad=grad, **more)


SOURCES = {
    "few": dict(seq=4, dim=64, slots=True), "one segment": dict(seq=64, dim=64), "one segment of a pool": dict(seq=70, dim=128, slots=True, lengths=True),
    "state given, none left": dict(seq=100, dim=64, last=False), "state left, none given": dict(seq=100, dim=64, state=False),
    "joined": dict(seq=1100, dim=64), "three launches": dict(seq=6000, dim=64), "float16": dict(seq=100, dim=256, dtype="float16"),
    "rows shared": dict(seq=200, dim=256, heads=2), "gradient": dict(seq=70, dim=64, grad=True), "gradient without states": dict(seq=70, dim=64, grad=True, state=False),
    "gradient in segments": dict(seq=1600, dim=64, grad=True), "gradient of wide heads": dict(seq=70, dim=256, grad=True, dtype="float16"),
}


@pytest.mark.parametrize("name", SOURCES)
def test_the_installed_compiler_takes_them(name, tmp_path):
    text = tmp_path / "x.info"
    text.write_text(described(**SOURCES[name]))
    done = subprocess.run([TOOL, "info", str(text)], capture_output=True, text=True, env=dict(os.environ, AKG_HIP_NO_CACHE="1"), timeout=300)
    assert done.returncode == 0 and "linear_attention" in done.stdout, (done.returncode, done.stderr[-500:])


def test_a_source_names_its_family(tmp_path):
    for name, family in (("few", "linear_attention"), ("joined", "linear_attention"), ("gradient", "linear_attention")):
        kernel = driver.HipKernel(described(**SOURCES[name]), out_dir=str(tmp_path))
        assert kernel.family == family and "// family: %s, op: " % family in kernel.source
    b = builder()
    kernel = driver.HipKernel(b.dumps(op_desc.rotary_embedding(b, [b.input([1, 3, 2, 8], "float32")], b.input([3], "int32"))), out_dir=str(tmp_path))
    assert kernel.family == "rotary" and "// family: rotary, op: " in kernel.source
