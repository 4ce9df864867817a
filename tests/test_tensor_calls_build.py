"""The calls that take tensors are built in where torch has what they need; elsewhere the module is built without them."""
import os
import subprocess

import pytest

from tests.test_native_calls_build import CSRC


def words(torch_dir):
    out = subprocess.run(["make", "-n", "-B", "-C", CSRC] + ([f"TORCH={torch_dir}"] if torch_dir else []), capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr
    (line,) = [x for x in out.stdout.splitlines() if x.strip().startswith("g++")]
    return line.split()


def test_with_this_torch():
    assert {"tensorcalls.cpp", "-DSPD_TORCH", "-lc10_cuda"} <= set(words(None))


@pytest.mark.parametrize("files", [[], ["include/ATen/ATen.h", "lib/libc10.so"], ["include/ATen/ATen.h", "include/ATen/cuda/EmptyTensor.h"]])
def test_without_cuda(tmp_path, files):
    for f in files:
        os.makedirs(os.path.dirname(tmp_path / f), exist_ok=True)
        (tmp_path / f).write_text("")
    got = words(tmp_path)
    assert "pycalls.cpp" in got and not {"tensorcalls.cpp", "-DSPD_TORCH", "-lc10_cuda"} & set(got)
