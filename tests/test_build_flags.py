"""Every build of the kernels uses the flags of tools/build_native.py, which keep packed FP32 instructions out (some of their
forms have returned wrong values, without an error), and a change of them rebuilds what is there.  CPU only: the library that is
loaded is taken apart into its gfx950 code objects and read."""
import os
import re
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT / "tools"))
import build_native  # noqa: E402

LIB = ROOT / "distributed_tensorflow_amd" / "_lib" / "libdtf_kernels.so"
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
needs_rocm = pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no ROCm tools")


def test_flags_for_scripts():
    r = subprocess.run([sys.executable, str(ROOT / "tools" / "build_native.py"), "--flags"], capture_output=True, text=True, check=True)
    assert r.stdout.split() == build_native.HIP_FLAGS and "-packed-fp32-ops" in build_native.HIP_FLAGS
    assert f"--offload-arch={build_native.ARCH}" in build_native.HIP_FLAGS


def test_no_tool_has_flags_of_its_own():
    """A tool that compiles kernels names the shared list; nobody else spells the target out (linking needs no device flags)."""
    own = []
    for f in sorted((ROOT / "tools").rglob("*")):
        if f.suffix not in (".py", ".sh", ".hip") or f.name == "build_native.py":
            continue
        for k, line in enumerate(f.read_text().split("\n"), 1):
            if "--offload-arch" in line and "-shared -fPIC -o" not in line:
                own.append(f"{f.relative_to(ROOT)}:{k}")
    assert not own, own


@needs_rocm
@pytest.mark.skipif(not LIB.exists(), reason="library not built")
def test_no_packed_fp32_instruction_is_shipped(tmp_path):
    shutil.copy(LIB, tmp_path / "k.so")
    subprocess.run([OBJDUMP, "--offloading", "k.so"], cwd=tmp_path, check=True, capture_output=True)
    objects = sorted(tmp_path.glob("k.so.*gfx950"))
    assert len(objects) >= 10
    kernels = 0
    for o in objects:
        text = subprocess.run([OBJDUMP, "-d", str(o)], check=True, capture_output=True, text=True).stdout
        kernels += text.count("s_endpgm")
        found = re.findall(r"v_pk_(?:add|mul|fma)_f32\b.*", text)
        assert not found, (o.name, len(found), found[0])
    assert kernels >= 50


@needs_rocm
def test_the_gemm_pipelines_waits_as_shipped(tmp_path, monkeypatch):
    """The wait-placement guard on the code that is shipped: the same check, compiled with the library's flags."""
    import test_gemm_isa
    run = subprocess.run
    monkeypatch.setattr(test_gemm_isa.subprocess, "run", lambda cmd, **kw: run([cmd[0], *build_native.DEVICE_FLAGS, *cmd[1:]], **kw))
    test_gemm_isa.test_lds_dma_pipeline_waits_are_exactly_the_pipelines_own(tmp_path)


# ------------------------------------------------------------------------------------------------ what is rebuilt
@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of two kernels; commands are noted and make their output file."""
    for d in ("csrc/kernels", "csrc/runtime"):
        (tmp_path / d).mkdir(parents=True)
    for name in ("a", "b"):
        (tmp_path / "csrc" / "kernels" / f"{name}.hip").write_text("//")
    commands = []

    def run(cmd):
        commands.append(cmd)
        Path(cmd[cmd.index("-o") + 1]).write_text("built")

    monkeypatch.setattr(build_native, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(build_native, "OUT", tmp_path / "lib")
    monkeypatch.setattr(build_native, "BUILD", tmp_path / "build")
    monkeypatch.setattr(build_native, "_hipcc", lambda: "hipcc")
    monkeypatch.setattr(build_native, "_run", run)
    return commands


def compiled(commands):
    return sorted(Path(c[c.index("-c") + 1]).stem for c in commands if "-c" in c)


def test_a_change_of_flags_rebuilds_every_object(tree, monkeypatch):
    build_native.build_kernels(verbose=False)
    assert compiled(tree) == ["a", "b"] and "-shared" in tree[-1]
    del tree[:]
    build_native.build_kernels(verbose=False)
    assert tree == []                                        # nothing to do
    monkeypatch.setattr(build_native, "HIP_FLAGS", build_native.HIP_FLAGS + ["-DX=1"])
    build_native.build_kernels(verbose=False)
    assert compiled(tree) == ["a", "b"] and "-shared" in tree[-1] and all("-DX=1" in c for c in tree if "-c" in c)
    del tree[:]
    build_native.build_kernels(verbose=False)
    assert tree == []


def test_an_object_whose_flags_are_unknown_is_rebuilt(tree):
    build_native.build_kernels(verbose=False)
    for f in build_native.BUILD.glob("a*"):
        if f.suffix != ".o":
            f.unlink()
    del tree[:]
    build_native.build_kernels(verbose=False)
    assert compiled(tree) == ["a"]
