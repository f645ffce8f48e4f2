"""The compiled kernels of the cache, attention and scores: no divergent block of them does nothing
(tests/isa/empty_blocks.py). No GPU is used."""
import subprocess
from pathlib import Path

import pytest

from tests.isa.empty_blocks import empty_blocks

ROOT = Path(__file__).resolve().parents[1]
FLAGS = ["-x", "hip", "--offload-arch=gfx950", "-O3", "-std=c++17", "-I", str(ROOT / "include"), "-Xclang", "-target-feature",
         "-Xclang", "-packed-fp32-ops", "-fno-gpu-flush-denormals-to-zero", "-munsafe-fp-atomics", "--cuda-device-only", "-S"]


@pytest.mark.parametrize("source", ["attention.hip", "attention_prompt.hip", "cache.hip", "logprobs.hip"])
def test_no_divergent_block_is_empty(source, tmp_path):
    out = tmp_path / "kernels.s"
    subprocess.run(["/opt/rocm/bin/hipcc", *FLAGS, str(ROOT / "nuclis_amd" / "csrc" / source), "-o", str(out)],
                   check=True, capture_output=True)
    asm = out.read_text()
    assert asm.count("s_endpgm") >= 4
    assert empty_blocks(asm) == []


def test_a_dropped_move_is_seen():
    def blocks(*body):
        return empty_blocks("_ZN3nuq6kernelE:  ; @k\n" + "\n".join(body) + "\n")

    narrow, restore = "\ts_and_saveexec_b64 s[2:3], s[0:1]", "\ts_or_b64 exec, exec, s[2:3]"
    assert blocks(narrow, "; %bb.60:", restore) == [("_ZN3nuq6kernelE", 2)]
    assert blocks(narrow, "\ts_cbranch_execz .LBB0_2", ".LBB0_2:", restore) == [("_ZN3nuq6kernelE", 2)]
    assert blocks(narrow, "\tv_mov_b32_e32 v75, s60", restore) == []
    assert blocks(narrow, "\ts_branch .LBB0_7", ".LBB0_2:", restore) == []
    assert blocks(narrow, "\ts_or_b64 exec, exec, s[8:9]", restore) == []
