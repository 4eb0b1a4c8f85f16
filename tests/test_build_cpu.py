"""What build.sh compiles again: with stand-ins for the compilers that note their calls."""
import os
import shutil
import subprocess
import time

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COMPILER = """#!/bin/bash
if [ "$1" = --version ]; then echo "$(basename $0) $COMPILER_IS"; exit; fi
echo "$(basename $0) $*" >> "$CALLS"
[ -n "$FAILS" ] && case "$*" in *"$FAILS"*) exit 1;; esac
while [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done
exit 0
"""
FILES = {"norm", "adamw", "gemm", "bind"}


@pytest.fixture
def build(tmp_path):
    """build(**environment): runs the script in a small tree and returns the sources it compiled."""
    shutil.copy(os.path.join(ROOT, "build.sh"), tmp_path)
    src, tools = tmp_path / "reid_gan_amd" / "csrc", tmp_path / "bin"
    src.mkdir(parents=True), tools.mkdir(), (tmp_path / "include").mkdir()
    old = time.time() - 100
    for name in ("norm.hip", "adamw.hip", "gemm.hip", "bind.cpp", "common.h", "../../include/ried_gan.h"):
        (src / name).write_text("")
        os.utime(src / name, (old, old))
    for name, text in (("hipcc", COMPILER), ("g++", COMPILER), ("python3", '#!/bin/bash\necho "/torch $TORCH_IS 3.10 /include"\n')):
        (tools / name).write_text(text)
        (tools / name).chmod(0o755)

    def run(*args, fails="", **env):
        calls = tmp_path / "calls"
        calls.write_text("")
        env = {**os.environ, "PATH": f"{tools}:{os.environ['PATH']}", "CALLS": str(calls), "COMPILER_IS": "1", "TORCH_IS": "2", "FAILS": fails, **env}
        rc = subprocess.run(["bash", str(tmp_path / "build.sh"), *args], env=env, capture_output=True).returncode
        assert (rc != 0) == bool(fails)
        words = calls.read_text().split()
        return {w.rsplit(".", 1)[0] for w in words if w.endswith((".hip", ".cpp"))}
    run.tree, run.src = tmp_path, src
    return run


def test_builds_everything_once(build):
    assert build() == FILES
    assert build() == set()
    assert (build.tree / "reid_gan_amd" / "libried_gan.so").exists()


def test_builds_again_what_a_source_changed(build):
    build()
    new = time.time() + 10
    os.utime(build.src / "norm.hip", (new, new))
    assert build() == {"norm"}
    build.src.joinpath("norm.o").touch(), os.utime(build.src / "norm.o", (new + 1, new + 1))
    os.utime(build.tree / "include" / "ried_gan.h", (new, new))
    assert build() == FILES - {"norm"}


def test_builds_everything_again_with_other_flags_or_compilers(build):
    build()
    assert build(COMPILER_IS="9") == FILES
    assert build(COMPILER_IS="9") == set()
    assert build() == FILES
    script = build.tree / "build.sh"
    script.write_text(script.read_text().replace('FLAGS="-O3', 'FLAGS="-O3 -DOTHER', 1))
    assert build() == FILES - {"bind"}
    script.write_text(script.read_text().replace('BIND_FLAGS="-O2', 'BIND_FLAGS="-O1', 1))
    assert build() == {"bind"}


def test_builds_the_binding_again_for_another_torch(build):
    build()
    assert build(TORCH_IS="3") == {"bind"}


def test_an_interrupted_build_is_not_taken_for_a_whole_one(build):
    build()
    script = build.tree / "build.sh"
    script.write_text(script.read_text().replace('FLAGS="-O3', 'FLAGS="-O3 -DOTHER', 1))
    build(fails="adamw.hip")
    assert build() == FILES


def test_builds_everything_when_told_to(build):
    build()
    assert build("-f") == FILES


def test_packed_fp32_instructions_are_off():
    text = open(os.path.join(ROOT, "build.sh")).read()
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in text
