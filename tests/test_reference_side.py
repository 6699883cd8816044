"""Without the reference's sources the suites that need its side are skipped,
not failed, so that a run goes on to the others."""
import os
import subprocess
import sys

import pytest

import oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SUITES = {"test_program_gpu": "integration/libcharlotte_program.so", "test_encoder_program_gpu": "integration/libcharlotte_program.so",
          "test_oracle_pins_gpu": "oracle/_ref/libcharlotte_ref.so"}


@pytest.mark.parametrize("suite", SUITES)
def test_a_suite_without_its_library_is_skipped(suite):
    if oracle.reference_root() is not None or os.path.exists(os.path.join(ROOT, SUITES[suite])):
        pytest.skip("the reference's side is there")
    r = subprocess.run([sys.executable, "-m", "pytest", f"tests/{suite}.py", "-q", "-m", "gpu", "-p", "no:cacheprovider", "-rs"],
                       capture_output=True, text=True, cwd=ROOT, timeout=300)
    last = r.stdout.strip().splitlines()[-1]
    assert r.returncode == 0 and "skipped" in last and "passed" not in last, r.stdout[-2000:]
    assert "the reference sources were absent" in r.stdout
