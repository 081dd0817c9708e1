"""What the compiler may not make of the sources, read from the built library without a GPU."""
import os
import re
import shutil
import subprocess
import tempfile

import pytest

from test_code_object import LIB, LLVM, kernel_table

ROOT = os.path.join(os.path.dirname(__file__), "..")

pytestmark = pytest.mark.skipif(not (os.path.exists(LIB) and os.path.exists(f"{LLVM}/llvm-objdump")), reason="library or llvm tools not present")


def test_no_packed_fp32_arithmetic():
    """The compiler makes it from ordinary float code unless the build says otherwise; some forms have given wrong results."""
    with tempfile.TemporaryDirectory() as tmp:
        lib = shutil.copy(LIB, tmp)
        subprocess.run([f"{LLVM}/llvm-objdump", "--offloading", lib], check=True, capture_output=True, cwd=tmp)
        objects = [os.path.join(tmp, name) for name in sorted(os.listdir(tmp)) if "amdgcn" in name]
        assert len(objects) > 20
        for path in objects:
            with subprocess.Popen([f"{LLVM}/llvm-objdump", "-d", "--no-show-raw-insn", path], stdout=subprocess.PIPE, text=True) as p:
                found = sorted({m.group(0) for m in map(re.compile(r"\bv_pk_(add|mul|fma)_f32\b").search, p.stdout) if m})
            assert p.returncode == 0 and not found, (os.path.basename(path), found)


def test_every_hip_build_switches_it_off():
    for path in ("wavenet_amd/csrc/Makefile", "tools/ubench/Makefile", "tools/build_variant.sh"):
        text = open(os.path.join(ROOT, path)).read()
        defined = dict(re.findall(r"^(\w+)\s*[:?]?=\s*(.*)$", text, re.M))

        def expand(line):
            for _ in range(4):
                line = re.sub(r"\$[({]?(\w+)[)}]?", lambda m: defined.get(m.group(1), ""), line)
            return line

        lines = [expand(l) for l in text.splitlines() if re.search(r"\$\(HIPCC\)|/hipcc ", l) and not re.search(r"^\w+\s*\??=|-shared", l)]
        assert lines, path
        for line in lines:
            assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in line, (path, line)


@pytest.mark.parametrize("taps", [4, 8, 16])
def test_train64_keeps_no_low_pass_values_in_scratch_memory(taps):
    """Held across the cost they take 1012, 852 and 1136 bytes per lane."""
    found = [private for name, (private, _) in kernel_table().items() if re.search(r"9k_train64ILi%dE" % taps, name)]
    assert len(found) == 1 and found[0] <= 692, found
