"""CPU: how csrc/build.sh compiles.  hipcc's packed fp32 forms (v_pk_add / mul / fma_f32) have given wrong results on gfx950 now and then: no source is compiled with
them, no built kernel holds one, and an object that was compiled with other flags is compiled again."""
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "videoitg_amd", "csrc")
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"
OBJDUMP = "/opt/rocm/lib/llvm/bin/llvm-objdump"


@pytest.fixture
def tree(tmp_path):
    """the sources beside a compiler that writes down its arguments and touches its output"""
    src = tmp_path / "videoitg_amd" / "csrc"
    src.mkdir(parents=True)
    for f in os.listdir(CSRC):
        if f.endswith((".hip", ".h", ".sh")):
            shutil.copy(os.path.join(CSRC, f), src / f)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    log, cc = tmp_path / "log", tmp_path / "cc"
    cc.write_text(f'#!/bin/bash\necho "$*" >> {log}\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && touch "$2"; shift; done\n')
    cc.chmod(0o755)

    def build(*args):
        log.write_text("")
        subprocess.run(["bash", str(src / "build.sh"), *args], check=True, capture_output=True, env={**os.environ, "HIPCC": str(cc), "VITG_CLEAN": "0"})
        return [line for line in log.read_text().splitlines() if " -c " in f" {line} "]
    build.src = src
    return build


@pytest.mark.parametrize("flavour", [(), ("--profiling",), ("--exp", "x")])
def test_every_source_is_compiled_without_packed_fp32(tree, flavour):
    lines = tree(*flavour)
    assert len(lines) >= 15
    for line in lines:
        assert FLAG in line, line


def test_objects_follow_the_build_script(tree):
    everything = len(tree())
    assert tree() == []
    os.utime(tree.src / "build.sh", (os.path.getmtime(tree.src / "gemm.hip") + 1e6,) * 2)
    assert len(tree()) == everything


def test_the_built_library_holds_no_packed_fp32(tmp_path):
    lib = os.path.join(ROOT, "videoitg_amd", "libvideoitg_hip.so")
    if not os.path.exists(lib) or not os.path.exists(OBJDUMP):
        pytest.skip("library not built, or no llvm-objdump")
    local = tmp_path / "lib.so"
    shutil.copy(lib, local)
    subprocess.run([OBJDUMP, "--offloading", str(local)], check=True, capture_output=True, cwd=tmp_path)
    code = [f for f in os.listdir(tmp_path) if "gfx950" in f]
    assert code
    kernels = 0
    for f in code:
        text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", "--mcpu=gfx950", str(tmp_path / f)], check=True, capture_output=True, text=True).stdout
        kernels += len(re.findall(r"^[0-9a-f]+ <_ZN4vitg", text, flags=re.M))
        found = re.findall(r"\bv_pk_(?:add|mul|fma)_f32\b", text)
        assert not found, (f, len(found))
    assert kernels > 100
