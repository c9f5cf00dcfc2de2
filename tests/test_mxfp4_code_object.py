"""CPU test of the built MXFP4 kernels (build products; skipped where nothing is
built or the ROCm LLVM tools are missing): the copies from memory into LDS take
their destination from M0, so each must set it itself, one wait state ahead."""
import re
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
LLVM = Path("/opt/rocm/llvm/bin")
CO = ROOT / "rlx-models_amd" / "lib" / "co" / "mxfp4.co"


def test_every_copy_into_lds_sets_m0(tmp_path):
    tools = [LLVM / "clang-offload-bundler", LLVM / "llvm-objdump"]
    if not CO.exists() or not all(t.exists() for t in tools):
        pytest.skip("no built code object, or no ROCm LLVM tools")
    elf = tmp_path / "mxfp4.elf"
    subprocess.run([tools[0], "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={CO}",
                    f"--output={elf}"], check=True)
    text = subprocess.run([tools[1], "-d", "--mcpu=gfx950", elf], check=True, capture_output=True, text=True).stdout
    ins = [line.split("//")[0].strip() for line in text.splitlines() if line.startswith("\t")]
    copies = [i for i, s in enumerate(ins) if s.startswith("global_load_lds")]
    assert copies
    for i in copies:
        assert ins[i - 1].startswith("s_nop") and re.match(r"s_mov_b32 m0, s\d+", ins[i - 2]), ins[i - 2:i + 1]
