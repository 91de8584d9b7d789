"""Which built files count as current."""
import os

import pytest
import torch

from cverl_b200 import _build
from cverl_b200 import _native as nv


@pytest.fixture
def builds(monkeypatch, tmp_path):
    """Output paths of the compilations that build_torch_ext starts, in a folder of its own."""
    made = []

    def run(cmd, log_path=None):
        out = cmd[cmd.index("-o") + 1]
        made.append(out)
        open(out, "w").close()

    monkeypatch.setattr(_build, "LIB_DIR", tmp_path)
    monkeypatch.setattr(_build, "_run", run)
    return made


def test_the_extension_is_built_once(builds):
    first = _build.build_torch_ext()
    assert builds == [str(first)] and first == _build.torch_ext_path()
    assert _build.build_torch_ext() == first and len(builds) == 1
    os.utime(first, (0, 0))                                        # older than its sources
    assert _build.build_torch_ext() == first and len(builds) == 2


def test_another_torch_or_python_takes_another_extension(builds, monkeypatch):
    first = _build.build_torch_ext()
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    second = _build.build_torch_ext()
    assert second != first and len(builds) == 2
    monkeypatch.setattr(_build.sysconfig, "get_config_var", lambda name: "cpython-399-other")
    assert _build.build_torch_ext() not in (first, second) and len(builds) == 3


def test_an_extension_of_another_torch_is_not_loaded(monkeypatch):
    monkeypatch.setattr(nv, "_torch_ext", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9+other")
    monkeypatch.setenv("CVERL_B200_NO_AUTOBUILD", "1")
    with pytest.raises(RuntimeError, match="native extension missing"):
        nv.torch_ext()


def test_8_bit_launchers_are_declared_once_and_bound_as_declared():
    """The header that the kernels and the extension are compiled against, letter by letter against the ctypes binding."""
    import re
    text = re.sub(r"//.*", "", (_build.PKG / "cuda" / "fp8_launch.h").read_text())
    letters = {"int": "i", "long long": "l", "float": "f"}
    declared = {}
    for name, args in re.findall(r"\bint (cvb_fp8_\w+)\(([^)]*)\);", text):
        kinds = [re.sub(r"\s*\w+$", "", a.strip()) for a in args.split(",") if a.strip() not in ("", "void")]
        declared[name] = "".join("p" if k.endswith("*") else letters[k] for k in kinds)
    bound = {n: c.replace(" ", "") for n, c in nv._CUDA_PROTOS.items() if n.startswith("cvb_fp8_")}
    assert set(bound) <= set(declared) and {n: declared[n] for n in bound} == bound
    for path in [*(_build.PKG / "cuda").glob("fp8_*.cu"), *(_build.PKG / "torch_ext").glob("*.cc")]:
        assert '#include "fp8_launch.h"' in path.read_text(), path.name


def test_the_extension_is_built_anew_when_a_launcher_changes(builds):
    first = _build.build_torch_ext()
    at = (_build.PKG / "cuda" / "fp8_launch.h").stat().st_mtime
    os.utime(first, (at - 1, at - 1))
    assert _build.build_torch_ext() == first and len(builds) == 2


def test_the_extension_is_built_anew_when_its_recipe_changes(builds):
    first = _build.build_torch_ext()
    at = os.stat(_build.__file__).st_mtime
    os.utime(first, (at - 1, at - 1))
    assert _build.build_torch_ext() == first and len(builds) == 2


def test_errors_of_the_extension_are_python_exceptions():
    """Messages with numbers in them end the process where the extension brings a C++ runtime of its own beside torch's."""
    import subprocess
    import sys
    code = ("import torch; from cverl_b200 import _native as nv\n"
            "try: nv.torch_ext().view8(torch.zeros(5, dtype=torch.uint8), 3, 7, 0)\n"
            "except ValueError as e: print(e)")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=_build.ROOT)
    assert r.returncode == 0 and "[3, 7] matrix" in r.stdout, (r.returncode, r.stderr[-500:])
