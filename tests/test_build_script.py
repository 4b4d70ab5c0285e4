"""The build script needs hipcc alone for the C library: without torch the Python module is left out, and a module that does
not compile leaves the library built (a copy of the script, with stand-ins for the compilers; no GPU needed)."""
import os
import shutil
import subprocess

from conftest import PKG, ROOT

STAND_IN = """#!/bin/sh
while [ $# -gt 0 ]; do [ "$1" = -o ] && echo built > "$2"; shift; done
"""


def run(tmp_path, torch, gxx):
    """(status, message, what was built) of the script with a python3 that has torch or not and a g++ that works or not."""
    csrc, tools = tmp_path / "pkg" / "csrc", tmp_path / "tools"
    for d in (csrc, tmp_path / "pkg" / "uwc_amd", tmp_path / "include", tools):
        d.mkdir(parents=True)
    shutil.copy(os.path.join(PKG, "csrc", "build.sh"), csrc)
    shutil.copy(os.path.join(ROOT, "include", "uwc.h"), tmp_path / "include")
    for f in ("uwc_one.hip", "uwc_two.hip", "uwc_kv_bind.cpp"):
        (csrc / f).write_text("")
    python = "#!/bin/sh\necho /somewhere\n" if torch else "#!/bin/sh\nexit 1\n"
    for name, text in (("hipcc", STAND_IN), ("g++", STAND_IN if gxx else "#!/bin/sh\nexit 1\n"), ("python3", python)):
        (tools / name).write_text(text)
        (tools / name).chmod(0o755)
    env = dict(os.environ, PATH=f"{tools}:{os.environ['PATH']}", HIPCC=str(tools / "hipcc"))
    r = subprocess.run(["sh", str(csrc / "build.sh")], env=env, capture_output=True, text=True)
    return r.returncode, r.stderr, sorted(os.listdir(tmp_path / "pkg" / "uwc_amd"))


def test_library_and_module(tmp_path):
    assert run(tmp_path, True, True)[::2] == (0, ["_kv.so", "libuwc_hip.so"])


def test_without_torch_the_library_alone(tmp_path):
    status, err, built = run(tmp_path, False, True)
    assert status == 0 and built == ["libuwc_hip.so"] and "no torch" in err


def test_a_module_that_does_not_compile(tmp_path):
    status, err, built = run(tmp_path, True, False)
    assert status == 1 and built == ["libuwc_hip.so"] and "the library is built" in err
