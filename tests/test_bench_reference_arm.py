"""The bench's reference arm says that the reference cannot run here: a line
without a value, so that no ratio is made against this repository's own port."""
import json
import subprocess
import sys

from tests.conftest import ROOT


def test_reference_arm_is_unavailable_and_says_why():
    out = subprocess.run([sys.executable, "bench.py", "--impl", "reference", "--steps", "1", "--warmup", "1"], cwd=ROOT,
                         capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    lines = out.stdout.strip().splitlines()
    assert len(lines) == 1
    line = json.loads(lines[0])
    assert line["impl"] == "reference" and "Rust" in line["unavailable"] and "\n" not in line["unavailable"]
    assert "value" not in line and "e2e" not in line
