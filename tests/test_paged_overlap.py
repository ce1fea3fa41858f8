"""Which tensors the attention operators' checks take to share memory, without a GPU."""

import os
import subprocess

from libcertex_amd import _capi as C


def test_shared_elements(tmp_path):
    """csrc/attention/overlap.hpp: small strided tensors against every pair of their elements, and large ones."""
    here = os.path.dirname(__file__)
    exe = tmp_path / "shared_elements"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I",
                    os.path.join(os.path.dirname(C.__file__), "csrc"), os.path.join(here, "c", "shared_elements.cpp"), "-o",
                    str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout
