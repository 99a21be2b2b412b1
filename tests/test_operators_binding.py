"""CPU-side checks of the operators' binding (asr_amd/_torch_ops.so) and of the build."""
import os
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _python(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr


def test_modules_without_bound_operators_import_without_the_binding():
    """Attention, layer norm and the dropout epoch need the C library only; dropout_add says what is missing."""
    _python("""
import sys
sys.modules["asr_amd._torch_ops"] = None  # what a missing or unloadable binding does to its import
import asr_amd.attention, asr_amd.layernorm, asr_amd.harness, asr_amd.parallel, asr_amd.dropout, torch
try:
    asr_amd.dropout.dropout_add(torch.zeros(2, 8), None, 0.0)
except ImportError:
    pass
else:
    raise SystemExit("dropout_add ran without the binding")
""")


def test_a_binding_of_another_abi_is_refused():
    _python("""
import sys, types
from asr_amd import _lib
for version in (_lib.ABI_VERSION - 1, None):  # (a binding from before it carried its version)
    stub = types.ModuleType("asr_amd._torch_ops")
    stub.entries, stub.bind = ("",), lambda at: None
    if version is not None:
        stub.abi_version = version
    sys.modules["asr_amd._torch_ops"] = stub
    sys.modules.pop("asr_amd._call", None)
    try:
        import asr_amd._call
    except ImportError as e:
        assert "ABI version" in str(e), e
    else:
        raise SystemExit(f"a binding of ABI version {version} was bound")
""")


def test_the_binding_carries_the_library_s_abi_version():
    from asr_amd import _call, _lib

    assert _call.ops.abi_version == _lib.ABI_VERSION == _lib.lib.lmufft_abi_version()


@pytest.mark.skipif(shutil.which("make") is None, reason="needs make")
def test_a_change_of_the_build_flags_rebuilds_every_object():
    csrc = os.path.join(ROOT, "asr_amd", "csrc")
    plan = subprocess.run(["make", "-C", csrc, "-n", "-W", os.path.join(csrc, "Makefile")], capture_output=True, text=True, check=True).stdout
    for name in sorted(os.listdir(csrc)):
        if name.endswith(".hip"):
            assert f"build/{name[:-4]}.o " in plan, name
