"""bench.py's reference arm where the reference's kernels are not built: one line that says so, and exit code 0."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_reference_arm_without_the_reference():
    sys.path.insert(0, str(ROOT))
    from oracle import oracle as O
    if O.load_ref() is not None:
        pytest.skip("the reference's kernels are built here")
    r = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--impl", "reference", "--steps", "1", "--warmup", "3"],
                       capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = [json.loads(ln) for ln in r.stdout.splitlines() if ln.startswith("{")]
    assert len(lines) == 1 and lines[0]["impl"] == "reference" and lines[0]["unavailable"] and set(lines[0]) == {"impl", "unavailable"}
