"""What the compiler made of regions that only some lanes run: at their end the lanes that stood aside come back (`s_or_b64 exec, exec, ..`), and nothing
may be saved, copied or reloaded in front of that, since it would be for some lanes only.  The register allocator has put such a copy there in a
kernel whose scalar and vector registers were both full; rows were then stored to the places of others.  This reads the device code of the built
library, every kernel of it."""
import os
import re
import shutil
import subprocess

import pytest

from rustingbrain_amd import _lib as L

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
LABEL = r"(?:[0-9a-f]{8,} )?<?(\.?\w+)>?:$"
# scalar instructions and lane accesses go by no mask
UNMASKED = ("s_", "v_readlane", "v_readfirstlane", "v_writelane")


def early(lines):
    """[(number, instruction)] of masked instructions between the end of a region and the return of its lanes."""
    code = [l.split("//")[0].split(";")[0].strip() for l in lines]
    targets = {c.split()[1] for c in code if c.startswith("s_cbranch_execz")}
    found = []
    for i, c in enumerate(code):
        label = re.match(LABEL, c)
        if not (label and label[1] in targets) and not c.startswith("s_cbranch_execnz"):  # (behind a loop that lanes leave one by one)
            continue
        seen = []
        for j in range(i + 1, len(code)):
            c = code[j]
            if re.match(r"s_or_b64 exec, exec,|s_xor_b64 exec,|s_(or|andn2)_saveexec_b64", c):
                found += seen
                break
            if not c or re.match(LABEL, c) or c.startswith(("s_cbranch", "s_branch", "s_and_saveexec", "s_endpgm")) or re.match(r"s_\w+ exec", c):
                if not c:
                    continue
                break
            if not c.startswith(UNMASKED):
                seen.append((j, c))
    return found


def test_the_reader_finds_them():
    good = ["s_and_saveexec_b64 s[4:5], vcc", "s_cbranch_execz L1", "global_load_dword v1, v[2:3], off", "<L1>:", "s_mov_b32 s1, s2", "v_writelane_b32 v255, s1, 0",
            "s_or_b64 exec, exec, s[4:5]", "v_accvgpr_write_b32 a72, v144"]
    assert not early(good)
    assert early(good[:4] + [good[-1]] + good[4:-1]) == [(4, good[-1])]
    loop = ["<L2>:", "s_andn2_b64 exec, exec, s[0:1]", "s_cbranch_execnz L2", "s_or_b64 exec, exec, s[0:1]", "scratch_store_dword off, v1, off"]
    assert not early(loop)
    assert early(loop[:3] + [loop[-1]] + [loop[3]]) == [(3, loop[-1])]


def test_nothing_stands_in_front_of_the_lanes_return(tmp_path):
    if not os.path.exists(OBJDUMP):
        pytest.skip("needs llvm-objdump")
    L.load()  # (built if it is not)
    library = shutil.copy(L.LIB_PATH, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(library)], check=True, capture_output=True, cwd=tmp_path)  # (extracts beside it)
    bad, kernels = {}, 0
    for f in sorted(os.listdir(tmp_path)):
        if "gfx950" not in f or not os.path.getsize(tmp_path / f):
            continue
        text = subprocess.run([OBJDUMP, "-d", "--symbolize-operands", "--no-show-raw-insn", str(tmp_path / f)], check=True, capture_output=True, text=True).stdout
        parts = re.split(r"^[0-9a-f]+ <(_Z\w+)>:$", text, flags=re.M)
        for name, body in zip(parts[1::2], parts[2::2]):
            kernels += 1
            got = early(body.split("\n"))
            if got:
                bad[name] = got[:5]
    assert kernels > 200, kernels
    assert not bad, bad
