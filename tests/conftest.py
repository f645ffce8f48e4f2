import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: needs an MI355X (runs through libnuq.so on cuda:0)")


# Last, so that a run that stops at the first failure has run all others: its last line takes the rows
# before max_tokens = 2 of four new tokens at a length of 38 for positions 36 and 37. The header's
# positions are 38 - 4 and on, 34 and 35 (test_gpu_attention_calls.py holds those).
LAST = ("test_rows_no_sequence_has_stay_as_they_are",)


def pytest_collection_modifyitems(items):
    items.sort(key=lambda item: item.name in LAST)


def pytest_terminal_summary(terminalreporter):
    try:
        from tests.gpu_util import WORST
    except Exception:
        return
    if not WORST:
        return
    terminalreporter.write_line("worst observed |gpu - oracle| / sum|w*x| per check (bound factor k):")
    for (family, _), (ratio, k, label) in sorted(WORST.items()):
        terminalreporter.write_line(f"  {family:12s} {ratio:.3e}  (k = {k:.0e})  worst: {label}")
