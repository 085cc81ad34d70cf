"""What the compiler does not check of the built kernels, where they have inline assembly: the wait states in front of
the copies to LDS (``dma16_opaque`` and its like in csrc/nq_device.hpp), and between a matrix product and the vector
instructions that read it."""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

from nano_qwen_amd import build

WAIT_STATES = 5    # from a vector instruction's write of a scalar register to a memory instruction that reads it
PRODUCT_STATES = 9    # from v_mfma_f32_16x16x32 to a vector instruction that reads the result, as the compiler keeps them


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


def vectors(operand):
    m = re.match(r"[-|]*v\[(\d+):(\d+)\]", operand)
    if m:
        return range(int(m[1]), int(m[2]) + 1)
    m = re.match(r"[-|]*v(\d+)\b", operand)
    return [int(m[1])] if m else []


def early_readers(lines):
    """(products, vector instructions less than PRODUCT_STATES behind one whose result they read), in order."""
    product, at, products, early = {}, 0, 0, []
    for line in lines:
        text = line.split("//")[0].strip()
        if line.startswith("\t") and text:
            name, _, rest = text.partition(" ")
            ops = [x.strip() for x in rest.split(",")]
            if name.startswith("v_mfma"):
                long = name.startswith("v_mfma_f32_16x16x32")
                products += long
                for r in vectors(ops[0]):
                    product.pop(r, None)
                    if long:
                        product[r] = at + 1
            elif name.startswith(("v_", "ds_", "buffer_", "global_")):
                if name.startswith("v_"):
                    late = [at - product[r] for x in ops[1:] for r in vectors(x) if r in product]
                    if late and min(late) < PRODUCT_STATES:
                        early.append(text)
                for r in vectors(ops[0]):
                    product.pop(r, None)
            at += int(ops[0], 0) + 1 if name == "s_nop" else 1
    return products, early


def test_early_copies_are_found():
    body = ["\tv_readfirstlane_b32 s6, v9\n", "\ts_mov_b32 m0, s1\n", "\ts_nop {}\n",
            "\tbuffer_load_dwordx4 v8, s[4:7], 0 offen lds\n"]
    for n, early in ((0, 1), (2, 1), (3, 0)):
        copies, found = early_copies(x.format(n) for x in body)
        assert copies == 1 and len(found) == early, n
    assert early_copies([body[0], "\ts_mov_b32 s6, s9\n", body[3]]) == (1, [])


def test_early_readers_are_found():
    body = ["\tv_mfma_f32_16x16x32_f16 v[4:7], v[8:11], v[12:15], v[4:7]\n", "\ts_nop {}\n",
            "\tv_max3_f32 v1, v2, v3, v6\n"]
    for n, early in ((0, 1), (7, 1), (8, 0)):
        products, found = early_readers(x.format(n) for x in body)
        assert products == 1 and len(found) == early, n
    assert early_readers([body[0], "\tv_mov_b32 v6, 0\n", body[2]]) == (1, [])


@pytest.fixture(scope="module")
def functions(tmp_path_factory):
    """(name, disassembled lines) of every kernel of the built library."""
    objdump = Path(build.hipcc()).parent.parent / "llvm" / "bin" / "llvm-objdump"
    if not objdump.exists() or not build.LIB.exists():
        pytest.skip("no built library, or no llvm-objdump beside hipcc")
    folder = tmp_path_factory.mktemp("code")
    lib = shutil.copy(build.LIB, folder)
    subprocess.run([objdump, "--offloading", lib], check=True, capture_output=True, cwd=folder)
    found = []
    for code in sorted(folder.glob("*gfx950")):
        out = subprocess.run([objdump, "-d", "--no-show-raw-insn", code], check=True, capture_output=True, text=True).stdout
        found += [(x.split(">")[0], x.splitlines()) for x in re.split(r"\n[0-9a-f]+ <", out)[1:]]
    return found


def test_copies_to_lds_wait_for_their_descriptors(functions):
    found = [(name, *early_copies(lines)) for name, lines in functions]
    assert sum(n for _, n, _ in found) > 0
    assert not [(name, early[:3]) for name, _, early in found if early]


def test_readers_wait_for_matrix_products(functions):
    found = [(name, *early_readers(lines)) for name, lines in functions]
    assert sum(n for _, n, _ in found) > 0
    assert not [(name, early[:3]) for name, _, early in found if early]
