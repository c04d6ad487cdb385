"""CPU: every command of this repository that compiles HIP sources leaves the packed fp32 instructions out (some of their forms have given wrong
results now and then), and no source asks for them by name."""
import os
import pathlib
import re
import subprocess
import sys

import pytest

ROOT = pathlib.Path(__file__).resolve().parent.parent
FLAG = "-Xclang -target-feature -Xclang -packed-fp32-ops"


def files(*kinds):
    return [p for top in ("swat_amd", "tools", "include") for p in sorted((ROOT / top).rglob("*")) if p.suffix in kinds]


def test_scripts_and_recipes():
    seen = set()
    for path in files(".sh", ".py"):
        for line in path.read_text().splitlines():
            # (what links objects into a library compiles nothing)
            if "--offload-arch" in line and (line.startswith("FLAGS=") or " -c " in line or re.search(r"\w\.hip\b", line)):
                seen.add(path.name)
                assert FLAG in line, f"{path}: {line}"
    assert {"build.sh", "build_asan.sh", "variant.sh", "adamw_beside.py"} <= seen, seen


def test_no_source_names_them():
    for path in files(".hip", ".hpp", ".h"):
        assert not re.search(r"v_pk_(add|mul|fma)_f32", path.read_text()), path


def test_the_generated_code_of_the_librarys_own_flags(tmp_path):
    """The build that runs has none of them, and its register-carried weight stages are untouched while in flight (the walk over the generated
    code that is made elsewhere for a build without the flag)."""
    hipcc, csrc = "/opt/rocm/bin/hipcc", ROOT / "swat_amd" / "csrc"
    if not os.path.exists(hipcc):
        pytest.skip("no hipcc")
    flags = re.search(r'^FLAGS="(.*)"$', (csrc / "build.sh").read_text(), re.M).group(1).split()
    out = tmp_path / "vit_mega.s"
    subprocess.check_call([hipcc, *flags, "--cuda-device-only", "-S", "-o", str(out), str(csrc / "vit_mega.hip")], stderr=subprocess.DEVNULL)
    assert not re.search(r"v_pk_(add|mul|fma)_f32", out.read_text())
    r = subprocess.run([sys.executable, str(ROOT / "tools" / "micro" / "check_inflight_regs.py"), str(out), "mega2"], stdout=subprocess.PIPE, text=True)
    assert r.returncode == 0 and "register-stage loads, 0 violations" in r.stdout and " 0 register-stage loads" not in r.stdout, r.stdout[-1000:]
