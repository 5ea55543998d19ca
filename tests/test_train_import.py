"""A checkout that is not built yet: the training operators' modules are imported and their tests collected without the
library, which a call then asks for."""
import os
import shutil
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def clean(tmp_path):
    shutil.copytree(os.path.join(ROOT, "indecis_b200"), tmp_path / "indecis_b200",
                    ignore=shutil.ignore_patterns("*.so", "_build", "__pycache__", "csrc"))
    return tmp_path


def run(at, *args):
    env = {k: v for k, v in os.environ.items() if k != "PYTHONPATH"}
    return subprocess.run([sys.executable, *args], cwd=at, env=env, capture_output=True, text=True, timeout=300)


def test_modules(tmp_path):
    code = """
import torch
from indecis_b200 import _capi, layers, optim
x = torch.zeros(2, 8)
m = optim.new_moment(x, 8)
for call in (lambda: layers.layer_norm(x), lambda: layers.gated_ff(x, x, x), lambda: optim.AdamW([x]).step([x])):
    try:
        call()
    except _capi.LibraryMissing as e:
        assert "_torch_ops.so is not built" in str(e) and "indecis_b200.build" in str(e), e
    else:
        raise AssertionError("expected LibraryMissing")
"""
    r = run(clean(tmp_path), "-c", code)
    assert r.returncode == 0, r.stderr


def test_collection(tmp_path):
    at = clean(tmp_path)
    os.mkdir(at / "tests")
    for name in ("conftest.py", "test_train_args.py"):
        shutil.copy(os.path.join(ROOT, "tests", name), at / "tests" / name)
    r = run(at, "-m", "pytest", "--collect-only", "-q", "-p", "no:cacheprovider", "tests")
    assert r.returncode == 0, r.stdout + r.stderr
