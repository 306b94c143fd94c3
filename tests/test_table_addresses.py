"""Bounds of addresses that kernels of the 4-bit table form, on the CPU: the header they share with the kernels, compiled for the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_read_as_they_lie_stay_inside(tmp_path):
    exe = str(tmp_path / "addresses")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", os.path.join(ROOT, "tests", "cpp", "test_table4_address.cpp"), "-o", exe])
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout
