"""The status word of the 4-bit cache where its first call comes in inference mode."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
PROGRAM = """
import torch
from nanoquantization_b200 import _lib
from nanoquantization_b200.layers import kv4
kc, vc = kv4.new_cache(2, 16, 1, "cuda")
with torch.inference_mode():
    kv4.load(kc, vc, torch.tensor([1000], device="cuda"), torch.float16)
for outside in range(2):
    try:
        _lib.check_cache_status()
        print("nothing")
    except RuntimeError as e:
        print(e)
"""


def test_a_status_that_was_made_in_inference_mode():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, cwd=root)
    assert got.returncode == 0, got.stderr
    first, second = got.stdout.splitlines()
    assert "outside its buffer" in first and second == "nothing"
