"""CPU: the shipped code objects hold no packed fp32 arithmetic.

v_pk_add_f32, v_pk_mul_f32 and v_pk_fma_f32, which the compiler makes of ordinary float code by itself, have given wrong results on these
devices now and then, without an error: csrc/Makefile leaves them out of every file, and this reads the library that is shipped."""
import os
import re
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
import isa_resources  # noqa: E402


def test_no_packed_fp32_arithmetic_in_the_library(tmp_path):
    found, seen = {}, 0
    for k, image in enumerate(isa_resources.code_objects(os.path.join(ROOT, "nncf_amd", "libnncf_hip.so"))):
        co = tmp_path / ("%d.co" % k)
        co.write_bytes(image)
        dis = subprocess.run([os.path.join(isa_resources.LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", str(co)],
                             capture_output=True, text=True, check=True).stdout
        name = "?"
        for line in dis.splitlines():
            m = re.match(r"^[0-9a-f]+ <(\S+)>:", line)
            if m:
                name = m.group(1)
                seen += 1
            elif re.match(r"\s+v_pk_(add|mul|fma)_f32\b", line):
                found[name] = found.get(name, 0) + 1
    assert seen > 150
    assert not found, "%d kernels: %s" % (len(found), sorted(found.items(), key=lambda x: -x[1])[:10])
