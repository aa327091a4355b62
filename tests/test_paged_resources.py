"""What the assembler reports for the paged chunk kernel: its softmax threads hold 128 scores, and a spill is paid every step."""
import re
import shutil
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent


def test_the_chunk_kernel_keeps_its_registers(tmp_path):
    from vibe_compiler_b200.build import NVCC_FLAGS
    result = subprocess.run([shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc", *NVCC_FLAGS, "-Xptxas", "-v", "-c",
                             str(ROOT / "vibe_compiler_b200/csrc/attention_paged_chunk.cu"), "-o", str(tmp_path / "chunk.o")],
                            check=True, capture_output=True, text=True, timeout=600)
    found = re.findall(r"Compiling entry function '\S*attention_paged_chunk_\w*kernel.*?(\d+) bytes stack frame, (\d+) bytes spill stores", result.stderr, re.S)
    assert len(found) == 8 and all(entry == ("0", "0") for entry in found), found
