"""What the package gives where torch is not installed: everything but the calls on torch tensors."""
import pathlib
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parent.parent


def run(code):
    return subprocess.run([sys.executable, "-c", code], cwd=str(ROOT), capture_output=True, text=True)


def test_all_names_without_torch():
    r = run("import sys; sys.modules['torch'] = None\n"   # (as an import of it sees a package that is not there)
            "from annembed_amd import *\n"
            "import annembed_amd as A; assert KGraph is A.KGraph and callable(to_proba_edges) and 'Points8' not in dir()\n"
            "try:\n    A.Points8\nexcept ImportError:\n    print('said so')")
    assert r.returncode == 0 and r.stdout.strip() == "said so", r.stderr


def test_all_names_with_torch():
    r = run("from annembed_amd import *\nassert Points8 and teacher_loss and teacher_grad and KGraph")
    assert r.returncode == 0, r.stderr


def test_all_names_with_a_torch_that_nobody_found():
    """a module put into sys.modules by hand has no spec"""
    r = run("import sys, types; sys.modules['torch'] = types.ModuleType('torch')\nimport annembed_amd as A\nassert 'Points8' in A.__all__ and A.KGraph")
    assert r.returncode == 0, r.stderr
