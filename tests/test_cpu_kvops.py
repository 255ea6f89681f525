"""The KV-cache operators' refusal of a second HIP runtime, which torch brings."""

import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _run(code):
    env = dict(os.environ, PYTHONPATH=os.path.join(ROOT, "fish-s2pro_amd"))
    return subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)


def test_torch_after_the_library_is_refused():
    r = _run("from s2hip import KvOps, _lib\n_lib.load()\nimport torch\nassert len(_lib.hip_runtimes()) == 2\nKvOps(8, 2, 64)")
    assert r.returncode and "two HIP runtimes" in r.stderr and "import torch before" in r.stderr


def test_torch_before_the_library_shares_its_runtime():
    r = _run("import torch\nfrom s2hip import _lib\n_lib.load()\nprint(len(_lib.hip_runtimes()))")
    assert r.returncode == 0 and r.stdout.strip() == "1", r.stderr
