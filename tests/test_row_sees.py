"""Which cells a sequence's latest queries see (strata-concurrent_amd/csrc/sc_attn_split.hpp), compiled from the kernels' own header into
tests/cpp/bin/row_sees_test and compared with 64-bit arithmetic there."""
import subprocess
from pathlib import Path

PROGRAM = Path(__file__).resolve().parent / "cpp" / "bin" / "row_sees_test"


def test_row_sees():
    run = subprocess.run([str(PROGRAM)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout + run.stderr
