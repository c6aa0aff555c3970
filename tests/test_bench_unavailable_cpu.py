"""bench.py's reference arm where the reference's library is not built: one JSON
line that says so, and no failure."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent

SCRIPT = """
import sys
from pathlib import Path
sys.path.insert(0, {root!r})
import oracle.oracle as o
o.REF_SO = Path({missing!r})
import bench
sys.argv = ["bench.py", "--impl", "reference", "--config", {config!r}, "--steps", "1", "--warmup", "3"]
bench.main()
"""


@pytest.mark.parametrize("config", ["llama3_8b", "oproj_llama3_8b", "attn_block_llama3_8b"])
def test_reference_arm_without_the_reference(tmp_path, config):
    script = SCRIPT.format(root=str(ROOT), missing=str(tmp_path / "libcottus_ref.so"), config=config)
    r = subprocess.run([sys.executable, "-c", script], capture_output=True, text=True, timeout=240, cwd=ROOT)
    assert r.returncode == 0, r.stderr[-2000:]
    lines = r.stdout.splitlines()
    assert len(lines) == 1
    d = json.loads(lines[0])
    assert d["impl"] == "reference" and "libcottus_ref.so" in d["unavailable"] and "\n" not in d["unavailable"]
