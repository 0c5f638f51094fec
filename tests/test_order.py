"""The order of a run that ends at its first failure."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(os.path.exists(os.path.join(ROOT, "oracle", "_ref", "gpt2_ref")), reason="the reference's programs are built")
def test_what_needs_the_reference_comes_last():
    r = subprocess.run([sys.executable, "-m", "pytest", "tests/test_distributed.py", "tests/test_rope.py", "-m", "gpu", "--collect-only", "-q"],
                       cwd=ROOT, capture_output=True, text=True, timeout=120)
    ids = [x for x in r.stdout.splitlines() if "::" in x]
    assert r.returncode == 0 and any("test_rope.py" in x for x in ids), r.stderr[-1000:]
    assert ids[-1].endswith("::test_bench_two_ranks_one_gpu_rehearsal")
