"""CPU-only: what the build needs and where it writes.  The compiler is a stand-in that records its command lines and writes
the file after -o, so that the makefiles run whole in a moment."""
import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

PKG = "dynamic-reward-rl-vae_amd"
WRITABLE = (f"{PKG}/csrc/", f"{PKG}/drlvae/", "tests/native/")
HIPCC = """#!/bin/sh
echo "$PWD: $*" >> "$HIPCC_LOG"
case "$*" in *"$HIPCC_FAILS_AT"*) echo "stand-in: cannot do $*" >&2; exit 3 ;; esac
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then echo made > "$2" || exit 4; fi
  shift
done
"""


@pytest.fixture
def tree(tmp_path):
    """A copy of the sources and a PATH that has make, python3 and what a shell needs, and no compiler but the stand-in."""
    root = tmp_path / "tree"
    for d in (f"{PKG}/csrc", f"{PKG}/drlvae", "include", "tools", "tests/native"):
        shutil.copytree(os.path.join(ROOT, d), root / d, ignore=shutil.ignore_patterns("*.so", "*.o", "obj", "_build", "__pycache__", "formats"))
    shutil.copy(os.path.join(ROOT, "__graft_entry__.py"), root)
    path = tmp_path / "bin"
    path.mkdir()
    for tool in ("make", "sh", "mkdir", "rm", "cat", "env"):
        os.symlink(shutil.which(tool), path / tool)
    os.symlink(sys.executable, path / "python3")
    fake = path / "hipcc"
    fake.write_text(HIPCC)
    fake.chmod(0o755)
    env = {"PATH": str(path), "HIPCC": str(fake), "HIPCC_LOG": str(tmp_path / "log"), "HIPCC_FAILS_AT": "no such thing", "HOME": str(tmp_path)}
    return root, env, tmp_path / "log"


def files(root):
    return {os.path.relpath(os.path.join(d, f), root) for d, _, fs in os.walk(root) for f in fs}


def make(root, env, where, *args):
    return subprocess.run(["make", "-C", str(root / where), *args], env=env, capture_output=True, text=True)


@pytest.mark.parametrize("where", [f"{PKG}/csrc", "tests/native"])
def test_hipcc_is_the_only_compiler_and_nothing_is_written_elsewhere(tree, where):
    root, env, log = tree
    before = files(root)
    r = make(root, env, where)
    assert r.returncode == 0, r.stdout + r.stderr
    new = files(root) - before
    assert new and all(f.startswith(WRITABLE) for f in new), new
    lines = log.read_text().splitlines()
    assert all(sum(a.endswith((".hip", ".cpp")) for a in x.split()) <= 1 for x in lines), "one source to a command"
    # no part of the make is a make of its own, with jobs of its own
    assert "make[1]" not in r.stdout and "-j" not in r.stdout


@pytest.mark.parametrize("where", [f"{PKG}/csrc", "tests/native"])
def test_every_source_is_a_prerequisite(tree, where):
    root, env, log = tree
    assert make(root, env, where).returncode == 0
    assert make(root, env, where, "-q").returncode == 0, "up to date"
    sources = [f"{PKG}/csrc/{f}" for f in sorted(os.listdir(root / PKG / "csrc")) if f.endswith((".hip", ".h", ".cpp"))] + ["include/drlvae.h"]
    assert len(sources) > 12
    for s in sources:
        old = os.stat(root / s)
        later = max(os.stat(os.path.join(d, f)).st_mtime for d, _, fs in os.walk(root) for f in fs) + 5
        os.utime(root / s, (later, later))
        assert make(root, env, where, "-q").returncode == 1, s
        os.utime(root / s, (old.st_atime, old.st_mtime))


def test_a_failing_build_says_what_failed(tree):
    root, env, _ = tree
    env["HIPCC_FAILS_AT"] = "sequence.hip"
    r = subprocess.run(["python3", "-c", "import __graft_entry__ as g\ntry:\n    g.build()\nexcept Exception as e:\n    print('RAISED', e)"], env=env,
                       cwd=root, capture_output=True, text=True)
    said = r.stdout[r.stdout.index("RAISED"):]
    assert "make" in said and "stand-in: cannot do" in said and "sequence.hip" in said, r.stdout + r.stderr
