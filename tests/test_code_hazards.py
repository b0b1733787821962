"""What the compiler's hazard recognizer does not see: instructions inside inline
assembly. CPU only: the library's own gfx950 code is disassembled."""
import os
import re
import shutil
import subprocess

import pytest

from hero_amd._lib import LIB_PATH

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """The instructions of every gfx950 code object of the library, in their order."""
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump here")
    folder = tmp_path_factory.mktemp("code")
    shutil.copy(LIB_PATH, folder / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=folder, check=True, capture_output=True)
    objects = sorted(f for f in os.listdir(folder) if f.endswith("gfx950"))
    assert objects
    text = [subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], cwd=folder, check=True, capture_output=True, text=True).stdout for f in objects]
    return [[line.split("//")[0].strip() for line in t.splitlines() if line.startswith("\t")] for t in text]


def test_a_wait_state_between_m0_and_a_load_into_shared_memory(code):
    """A scalar write of M0 needs one wait state before a load that takes its address in shared memory from there:
    without it the load may still see the M0 of before, and its data land elsewhere, with no error."""
    loads, bare = 0, []
    for instructions in code:
        for before, this in zip(instructions, instructions[1:]):
            if re.match(r"(global_load_lds|buffer_load\S* .*\blds\b)", this):
                loads += 1
                if re.match(r"s_\S+ m0\b", before):
                    bare.append(this)
    assert loads > 100
    assert not bare, f"{len(bare)} of {loads}"
