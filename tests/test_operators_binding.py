"""CPU-side checks of the operators' binding (asr_amd/_torch_ops.so)."""
import os
import subprocess
import sys

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
