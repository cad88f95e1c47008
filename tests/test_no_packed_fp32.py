"""The library holds no packed fp32 arithmetic: some forms of it have given wrong results on this hardware without an error, and the
compiler makes it from ordinary scalar code unless told not to."""
import os
import re
import subprocess

import pytest

from test_kernel_resources import LIB, _code_objects

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="library or llvm-objdump missing")
def test_no_packed_fp32_arithmetic(tmp_path):
    objs = _code_objects(open(LIB, "rb").read())
    assert objs
    for i, (_, code) in enumerate(objs):
        f = tmp_path / f"{i}.o"
        f.write_bytes(code)
        with subprocess.Popen([OBJDUMP, "-d", str(f)], stdout=subprocess.PIPE, text=True) as p:
            found = [line.strip() for line in p.stdout if re.search(r"v_pk_(add|mul|fma)_f32", line)]
        assert p.returncode == 0 and not found, f"code object {i}: {len(found)} of them, first {found[0] if found else None}"
