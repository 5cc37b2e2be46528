"""The compiled kernels, without a GPU: no register is saved or brought back at the head of a block before the lanes that skipped the region ahead of it are
let in again.

With vector and accumulation registers all in use the compiler has put such saves, of registers that all lanes live on, between the label that those lanes
jump to and the instruction that restores their execution mask: they lose what is saved, addresses among it. Where it does so hangs on the source around it and on
the compiler, so every build is searched."""
import os
import re
import subprocess

import pytest

from lmserve_amd import _lib

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
SAVES = re.compile(r"v_accvgpr_(write|read|mov)|scratch_(store|load)")
RESTORES = re.compile(r"s_or_b64 exec, exec,")
LINE = re.compile(r"^\t(\S.*?)\s*// ([0-9A-F]+):")
FUNCTION = re.compile(r"^[0-9a-f]+ <(\S+)>:")
TARGET = re.compile(r"<(\S+?)\+0x([0-9a-f]+)>\s*$")


def saves_ahead_of_exec(listing):
    """[(function, address, instructions)] of the blocks that begin at a jump's target, where a save stands before the mask is restored."""
    functions, name = {}, None
    for line in listing.splitlines():
        m = FUNCTION.match(line)
        if m:
            name = m.group(1)
            functions[name] = []
            continue
        m = LINE.match(line)
        if m and name:
            to = TARGET.search(line) if m.group(1).startswith(("s_cbranch", "s_branch")) else None
            functions[name].append((int(m.group(2), 16), m.group(1), int(to.group(2), 16) if to else None))
    bad = []
    for name, code in functions.items():
        if not code:
            continue
        start = code[0][0]
        targets = {start + to for _, _, to in code if to is not None}
        block, entered = [], False
        for at, text, _ in code:
            if at in targets:
                block, entered, first = [], True, at
            if entered:
                if RESTORES.match(text):
                    if any(SAVES.match(x) for x in block):
                        bad.append((name, hex(first), [x for x in block if SAVES.match(x)]))
                    entered = False
                elif text.startswith(("s_cbranch", "s_branch", "s_endpgm")):
                    entered = False
                else:
                    block.append(text)
    return bad


def test_the_search_finds_them():
    """A listing with one: written by hand, as the compiler's would be."""
    kernel = """
0000000000000100 <kernel>:
\ts_and_saveexec_b64 s[2:3], vcc                             // 000000000100: BE82206A
\ts_cbranch_execz 2                                          // 000000000104: BF880002 <kernel+0x10>
\tv_accvgpr_write_b32 a1, v9                                 // 000000000108: D3D94001
\tglobal_load_dword v2, v[4:5], off                          // 00000000010C: DC508000
%s\ts_or_b64 exec, exec, s[2:3]                                // 000000000118: 87FE7E02
\tv_accvgpr_write_b32 a2, v8                                 // 00000000011C: D3D94002
\ts_endpgm                                                   // 000000000120: BF810000
"""
    save = "\tv_accvgpr_write_b32 a0, v7                                 // 000000000110: D3D94000\n"
    keep = "\tv_mov_b32_e32 v3, 0                                        // 000000000110: 7E060280\n"
    assert saves_ahead_of_exec(kernel % keep) == []
    assert [x[1:] for x in saves_ahead_of_exec(kernel % save)] == [("0x110", ["v_accvgpr_write_b32 a0, v7"])]


def test_no_kernel_has_saves_ahead_of_the_mask(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("no llvm-objdump")
    library = tmp_path / "libkvcache.so"
    library.write_bytes(open(_lib.lib()._name, "rb").read())
    subprocess.run([OBJDUMP, "--offloading", library.name], cwd=tmp_path, check=True, capture_output=True, timeout=120)
    objects = sorted(p for p in tmp_path.iterdir() if "gfx950" in p.name and p.stat().st_size)
    assert objects
    kernels, bad = 0, []
    for o in objects:
        listing = subprocess.run([OBJDUMP, "-d", str(o)], check=True, capture_output=True, text=True, timeout=120).stdout
        kernels += sum(bool(FUNCTION.match(x)) for x in listing.splitlines())
        bad += saves_ahead_of_exec(listing)
    print(f"{kernels} functions in {len(objects)} objects")
    assert kernels > 100
    assert not bad, bad[:5]
