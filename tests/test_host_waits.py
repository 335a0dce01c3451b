"""The wait states that the hardware leaves to the program, in the built library's own gfx950 code: a copy from memory to LDS
reads M0 at the earliest two instructions after the scalar write of it (gfx9: one wait state), and nothing but those copies uses
M0, so that inline assembly may set it without the compiler's knowledge."""
import os
import re
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen38-megakernel_amd")
LIB, OBJDUMP = os.path.join(PKG, "libqwen38_kv.so"), "/opt/rocm/llvm/bin/llvm-objdump"
M0 = re.compile(r"\bm0\b")


def early_copies(lines):
    """Instructions of a listing -> (copies to LDS, those right behind a write of M0, other uses of M0)."""
    copies, early, other, set_m0 = 0, [], [], False
    for line in lines:
        text = line.split("//")[0].strip()
        if not text or text.endswith(":"):
            continue
        if "_lds_" in text.split()[0]:  # global_load_lds_*, buffer_load_lds_*
            copies += 1
            if set_m0:
                early.append(text)
        elif M0.search(text) and not text.startswith("s_mov_b32 m0, "):
            other.append(text)
        set_m0 = text.startswith("s_mov_b32 m0, ")
    return copies, early, other


def test_reader():
    """The reader finds a missing wait state and another user of M0 (planted in a listing of its own)."""
    bad = ["\ts_mov_b32 m0, s2", "\tglobal_load_lds_dwordx4 v1, s[4:5]", "\ts_mov_b32 m0, s3  // 0000: BE", "\ts_nop 0", "\tglobal_load_lds_dwordx4 v1, s[4:5]",
           "\tglobal_load_lds_dwordx4 v1, s[4:5] offset:1024", "\ts_mov_b32 s4, m0"]
    assert early_copies(bad) == (3, ["global_load_lds_dwordx4 v1, s[4:5]"], ["s_mov_b32 s4, m0"])


@pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(OBJDUMP)), reason="no built library, or no disassembler")
def test_lds_copies_wait_for_m0(tmp_path):
    os.symlink(LIB, tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", "lib.so"], cwd=tmp_path, check=True, capture_output=True)
    objs = sorted(f for f in os.listdir(tmp_path) if f.endswith("gfx950"))
    assert objs
    total = 0
    for f in objs:
        p = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", f], cwd=tmp_path, stdout=subprocess.PIPE, text=True)
        copies, early, other = early_copies(p.stdout)
        assert p.wait() == 0
        assert not early, (f, len(early), early[:3])
        assert not other, (f, other[:3])
        total += copies
    assert total > 0
