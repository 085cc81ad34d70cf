"""What the compiler does not check of the built kernels: the wait states in front of the copies to LDS, which are
inline assembly (``dma16_opaque`` and its like in csrc/nq_device.hpp)."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from nano_qwen_amd import build

WAIT_STATES = 5    # from a vector instruction's write of a scalar register to a memory instruction that reads it


def scalars(operand):
    m = re.match(r"s\[(\d+):(\d+)\]$", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", operand)
    return {int(m[1])} if m else set()


def early_copies(lines):
    """(copies to LDS, those less than WAIT_STATES behind a vector instruction's write of their descriptor).

    Instructions in order: a copy's own wait states stand right in front of it, where no branch lands."""
    written, at, copies, early = {}, 0, 0, []
    for line in lines:
        text = line.split("//")[0].strip()
        if line.startswith("\t") and text:
            name, _, rest = text.partition(" ")
            ops = [x.strip().split(" ")[0] for x in rest.split(",")]
            if name.startswith("buffer_load") and text.endswith(" lds"):
                copies += 1
                late = [at - written[r] for r in scalars(ops[1]) if r in written]
                if late and min(late) < WAIT_STATES:
                    early.append(text)
            at += int(ops[0], 0) + 1 if name == "s_nop" else 1
            if name.startswith("v_"):
                written.update((r, at) for r in scalars(ops[0]))
            elif name.startswith("s_"):
                for r in scalars(ops[0]):
                    written.pop(r, None)
    return copies, early


def test_early_copies_are_found():
    body = ["\tv_readfirstlane_b32 s6, v9\n", "\ts_mov_b32 m0, s1\n", "\ts_nop {}\n",
            "\tbuffer_load_dwordx4 v8, s[4:7], 0 offen lds\n"]
    for n, early in ((0, 1), (2, 1), (3, 0)):
        copies, found = early_copies(x.format(n) for x in body)
        assert copies == 1 and len(found) == early, n
    assert early_copies([body[0], "\ts_mov_b32 s6, s9\n", body[3]]) == (1, [])


def test_copies_to_lds_wait_for_their_descriptors(tmp_path):
    objdump = Path(build.hipcc()).parent.parent / "llvm" / "bin" / "llvm-objdump"
    if not objdump.exists() or not build.LIB.exists():
        pytest.skip("no built library, or no llvm-objdump beside hipcc")
    lib = shutil.copy(build.LIB, tmp_path)
    subprocess.run([objdump, "--offloading", lib], check=True, capture_output=True, cwd=tmp_path)
    copies = 0
    for code in sorted(tmp_path.glob("*gfx950")):
        out = subprocess.run([objdump, "-d", "--no-show-raw-insn", code], check=True, capture_output=True, text=True).stdout
        for function in re.split(r"\n[0-9a-f]+ <", out):
            n, early = early_copies(function.splitlines())
            assert not early, (function.split(">")[0], early[:3])
            copies += n
    assert copies > 0
