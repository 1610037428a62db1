"""CPU tier: hazards that neither the hardware nor, inside inline assembly, the compiler takes care of, looked for in
the disassembly of the built library's gfx950 code."""
import os
import re
import subprocess

import pytest

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """[(function, [instructions])] of libsmla.so."""
    from smla import _lib
    _lib.lib()      # raises where nothing is built
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    at = tmp_path_factory.mktemp("code")
    os.symlink(_lib.LIB_PATH, at / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=at, check=True, capture_output=True)
    functions = []
    for f in sorted(at.glob("lib.so.*gfx950")):
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", f], check=True, capture_output=True, text=True).stdout
        for line in text.split("\n"):
            name = re.match(r"[0-9a-f]+ <(.*)>:$", line)
            line = line.split("//")[0].strip()
            if name:
                functions.append((name.group(1), []))
            elif line and functions and not line.endswith(":"):
                functions[-1][1].append(line)
    assert functions
    return functions


def _sgprs(text):
    regs = {int(r) for r in re.findall(r"\bs(\d+)\b", text)}
    for a, b in re.findall(r"\bs\[(\d+):(\d+)\]", text):
        regs |= set(range(int(a), int(b) + 1))
    return regs


def _walk(body):
    """(instruction, operands, wait states before it) of a function, in the order of the code."""
    at = 0
    for line in body:
        op, _, args = line.partition(" ")
        yield op, args.strip(), at
        at += int(args, 0) + 1 if op == "s_nop" else 1


def test_copies_to_lds_wait_for_m0(code):
    """A copy from memory to LDS takes its LDS address from M0, a wait state after the write of it at the earliest."""
    copies, bad = 0, []
    for name, body in code:
        written = None
        for op, args, at in _walk(body):
            if op.startswith(("global_load_lds", "buffer_load")) and (op.startswith("global_load_lds") or " lds" in args):
                copies += 1
                if written is not None and at - written < 2:
                    bad.append(name)
            if op.startswith("s_") and args.split(",")[0] == "m0":
                written = at
    assert copies > 100 and not bad, f"{len(bad)} of {copies} copies in {sorted(set(bad))}"


def test_scalar_addresses_wait_for_vector_writes(code):
    """A scalar register that a vector instruction wrote is read as an address five wait states later at the earliest."""
    bad = []
    for name, body in code:
        written = {}
        for op, args, at in _walk(body):
            if op.startswith(("global_", "buffer_", "flat_", "scratch_")):
                bad += [name for r in _sgprs(args) if at - written.get(r, -99) < 6]
            for r in _sgprs(args.split(",")[0]):
                if op.startswith(("v_readlane", "v_readfirstlane", "v_cmp")):
                    written[r] = at
                elif op.startswith("s_"):
                    written.pop(r, None)
    assert not bad, sorted(set(bad))
