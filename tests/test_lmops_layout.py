"""The descriptors of ah_linear_ce, ah_orthogonalize and ah_muon_step as the C compiler lays them out, against their ctypes mirror.
CPU only: compiles an offsetof() probe of the header with gcc."""
import ctypes as C
import os
import subprocess

import pytest

from anneal_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("name", ["ah_linear_ce_desc", "ah_orthogonalize_desc", "ah_muon_desc"])
def test_ctypes_mirror_matches_the_c_header(tmp_path, name):
    cls = getattr(L, name)
    fields = [f for f, _ in cls._fields_]
    src = tmp_path / "probe.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "anneal_hip.h"\nint main(void) {\n    printf("%zu\\n", sizeof(' + name + "));\n" +
                   "".join(f'    printf("%zu\\n", offsetof({name}, {f}));\n' for f in fields) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "probe")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "probe")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(cls)] + [getattr(cls, f).offset for f in fields]
