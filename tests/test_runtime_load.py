"""How libnuq.so comes into a process (nuclis_amd/backend.py, lib). No GPU is used."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]


def test_one_hip_runtime_whatever_is_called_first():
    """Host calls before torch is imported (sizes, quantising) must not bring a second HIP runtime into the
    process: a context or torch itself would then find no device."""
    code = ("import nuclis_amd as nq\n"
            "nq.cache_bytes(4, 1, 16, 1, 64)\n"
            "import torch\n"
            "print(*{l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l}, sep='\\n')\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    assert len(r.stdout.split()) == 1, r.stdout
