"""Loads into LDS of the compiled kernels that the compiler does not know of.

They take their address in LDS from m0, which inline assembly writes in front of each. m0 is a reserved register, so the
compiler refuses it among what a statement says it changes; it must have no use for m0 itself then.
"""
import os
import re
import subprocess

import pytest

from test_step_isa import HIPCC, ROOT, _makefile_flags


@pytest.mark.parametrize("source", ["lora", "paged_attention"])
def test_m0_belongs_to_the_inline_assembly(source, tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc not available")
    flags = [f for f in _makefile_flags() if f != "-fPIC"]
    out = tmp_path / "kernels.txt"
    subprocess.run([HIPCC, *flags, "--cuda-device-only", "-S", "-o", str(out),
                    os.path.join(ROOT, "llm-inference_amd", "csrc", source + ".hip")],
                   check=True, capture_output=True, timeout=300)
    asm = out.read_text()
    inline = re.findall(r";#ASMSTART(.*?);#ASMEND", asm, re.S)
    assert sum(bool(re.search(r"\bm0\b", s)) for s in inline) > 10
    rest = re.sub(r";#ASMSTART.*?;#ASMEND", "", asm, flags=re.S)
    assert not re.search(r"\bm0\b", rest)
