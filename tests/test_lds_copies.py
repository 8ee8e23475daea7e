"""Copies from memory straight to LDS have landed when a barrier publishes them: read from the built library's own kernels.

A wave waits for such copies with ``s_waitcnt vmcnt(0)`` and then meets the others at ``s_barrier``; a barrier alone orders LDS
accesses only.  A kernel that misses the wait on one path is right nearly always, so its results show nothing: the instructions
do."""
import collections
import re
import shutil
import subprocess

import pytest

from mpnn_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]+):.*?(?:<(\S+?)(?:\+0x([0-9a-f]+))?>)?$")


def kernels(listing):
    """{name: [(address, mnemonic, operands, branch target)]} of a disassembly."""
    found, name, start = collections.OrderedDict(), None, {}
    for line in listing.splitlines():
        head = re.match(r"^([0-9a-f]+) <(\S+)>:$", line)
        if head:
            name = head.group(2)
            start[name], found[name] = int(head.group(1), 16), []
            continue
        m = LINE.match(line)
        if m and name:
            target = (m.group(4), int(m.group(5) or "0", 16)) if m.group(4) else None
            found[name].append((int(m.group(3), 16), m.group(1), m.group(2), target))
    return {k: [(a, op, args, start[t[0]] + t[1] if t else None) for a, op, args, t in v] for k, v in found.items()}


def loose_copies(code):
    """Addresses of barriers (and ends of the program) that a wave can reach with copies to LDS on their way."""
    at = {a: i for i, (a, _, _, _) in enumerate(code)}
    seen, work, loose = {}, [(0, False)], set()
    while work:
        i, out = work.pop()
        while i < len(code) and not (seen.get(i, -1) >= int(out)):
            seen[i] = int(out)
            address, op, args, target = code[i]
            if "_load_lds_" in op or ("buffer_load" in op and re.search(r"\blds\b", args)):
                out = True
            elif op == "s_waitcnt" and "vmcnt(0)" in args:
                out = False
            elif op in ("s_barrier", "s_endpgm") and out:
                loose.add(address)
            if op == "s_endpgm":
                break
            if op.startswith("s_cbranch"):
                work.append((at[target], out))
            elif op == "s_branch":
                i = at[target]
                continue
            i += 1
    return loose


def listing_of(*lines):
    """A disassembly's text of instructions of 4 bytes; a number in place of an operand is the instruction branched to."""
    text = ["0000000000001000 <k>:"]
    for i, (op, arg) in enumerate(lines):
        to = f" <k+0x{4 * arg:x}>" if isinstance(arg, int) else ""
        text.append(f"\t{op} {'' if isinstance(arg, int) else arg}  // {0x1000 + 4 * i:012X}: 00000000{to}")
    return "\n".join(text)


def test_the_reading_of_a_listing():
    copy, wait = ("global_load_lds_dwordx4", "v[2:3], off"), ("s_waitcnt", "vmcnt(0) lgkmcnt(0)")
    lds, bar, end = ("s_waitcnt", "lgkmcnt(0)"), ("s_barrier", ""), ("s_endpgm", "")
    # the loop that was built without its wait: the copies of one round are still on their way at the next round's barrier
    loop = lambda w: kernels(listing_of(copy, wait, w, bar, ("ds_read_b128", "v[0:3], v4"), copy, ("s_cbranch_scc1", 2), wait, end))["k"]
    assert loose_copies(loop(lds)) == {0x100c} and not loose_copies(loop(wait))
    assert loose_copies(kernels(listing_of(copy, ("s_waitcnt", "vmcnt(1)"), bar, wait, end))["k"]) == {0x1008}
    assert loose_copies(kernels(listing_of(copy, end))["k"]) == {0x1004}
    assert not loose_copies(kernels(listing_of(("s_cbranch_execz", 4), copy, wait, bar, end))["k"])
    assert loose_copies(kernels(listing_of(copy, ("s_branch", 3), wait, bar, end))["k"]) == {0x100c, 0x1010}


@pytest.mark.skipif(not shutil.which(OBJDUMP), reason="no disassembler")
def test_every_barrier_of_the_library_waits_for_the_copies_before_it(tmp_path):
    lib = shutil.copy(_lib.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, capture_output=True, cwd=tmp_path)
    with_copies = 0
    for part in sorted(tmp_path.glob("lib.so.*gfx950")):
        listing = subprocess.run([OBJDUMP, "-d", str(part)], check=True, capture_output=True, text=True).stdout
        if "load_lds" not in listing and " lds" not in listing:
            continue
        for name, code in kernels(listing).items():
            if any("_load_lds_" in op for _, op, _, _ in code):
                with_copies += 1
                assert any(op == "s_barrier" for _, op, _, _ in code), name
                assert not loose_copies(code), name
    assert with_copies >= 4
