"""The kernel library's Makefile: what has changed is compiled again, the compiler's flags included (a library linked from
objects of older flags would carry the identity of the current sources)."""
import os
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "symbolic-music-generation_amd")


@pytest.fixture
def built(tmp_path):
    """A tree of empty sources in which everything is up to date."""
    csrc = tmp_path / "csrc"
    (csrc / "build").mkdir(parents=True)
    (tmp_path / "mgen").mkdir()
    shutil.copy(os.path.join(PKG, "csrc", "Makefile"), csrc)
    shutil.copy(os.path.join(PKG, "mgen", "_srcid.py"), tmp_path / "mgen")
    names = [f for f in os.listdir(os.path.join(PKG, "csrc")) if f.endswith((".hip", ".h"))]
    for f in [*names, "Makefile"]:
        (csrc / f).touch()
        os.utime(csrc / f, (1000, 1000))
    objects = [f[:-4] + ".o" for f in names if f.endswith(".hip")]
    for f in objects:
        (csrc / "build" / f).touch()
        os.utime(csrc / "build" / f, (2000, 2000))
    (tmp_path / "mgen" / "libmgen_hip.so").touch()
    return csrc, objects


def compiled(csrc):
    """Objects that make would compile."""
    out = subprocess.run(["make", "-n", "-C", str(csrc)], check=True, capture_output=True, text=True).stdout
    return {line.split(" -o build/")[1].split()[0] for line in out.splitlines() if " -c " in line}


def test_nothing_to_do(built):
    assert compiled(built[0]) == set()


@pytest.mark.parametrize("changed", ["Makefile", "common.h"])
def test_flags_and_headers_reach_every_object(built, changed):
    csrc, objects = built
    os.utime(csrc / changed, (3000, 3000))
    assert compiled(csrc) == set(objects)


def test_a_source_reaches_its_object_and_the_identity(built):
    csrc, _ = built
    os.utime(csrc / "kvmx.hip", (3000, 3000))
    assert compiled(csrc) == {"kvmx.o", "runtime.o"}


def test_no_packed_fp32():
    """Some forms of these instructions give wrong results on these GPUs: the compiler is told not to make them, and no
    source writes one by hand."""
    with open(os.path.join(PKG, "csrc", "Makefile")) as f:
        text = f.read()
    assert "-Xclang -target-feature -Xclang -packed-fp32-ops" in text and "$(NO_PK_F32)" in text
    root = os.path.join(PKG, "..")
    for top in (os.path.join(PKG, "csrc"), os.path.join(root, "tools")):
        for folder, _, names in os.walk(top):
            for name in names:
                if name.endswith((".hip", ".h")) or (name.endswith(".s") and os.path.basename(folder) == "build"):
                    with open(os.path.join(folder, name)) as f:
                        assert not any(f"v_pk_{op}_f32" in line for line in f for op in ("add", "mul", "fma")), name
