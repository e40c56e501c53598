"""The learning operators' header is plain C."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no C compiler")
def test_header_compiles_as_c11(tmp_path):
    source = tmp_path / "header.c"
    source.write_text('#include "pcu_b200_learn.h"\n'
                      "int kinds(void) { return PCU_B200_F16 + PCU_B200_BF16 + PCU_B200_ACTIVATION_GELU + PCU_B200_DISTILL_TOP_MAX; }\n")
    res = subprocess.run(["gcc", "-std=c11", "-Wall", "-Wextra", "-Werror", "-pedantic", "-fsyntax-only", "-I",
                          os.path.join(ROOT, "include"), str(source)], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
