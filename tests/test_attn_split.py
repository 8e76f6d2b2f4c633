"""How attention's cells are shared out among workgroups (strata-concurrent_amd/csrc/sc_attn_split.hpp), compiled from the
kernels' own header into tests/cpp/bin/attn_split_test and compared with plain loops over the sequences there."""
import subprocess
from pathlib import Path

import pytest

PROGRAM = Path(__file__).resolve().parent / "cpp" / "bin" / "attn_split_test"


@pytest.mark.parametrize("name", ["longest", "ragged"])
def test_attn_split(name):
    run = subprocess.run([str(PROGRAM), name], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
