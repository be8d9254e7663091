"""The plans of few-row products on the host: tests/cpp/test_few_rows_plan.cpp includes the planner that the library is built with."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_plan_is_one_that_can_be_launched(tmp_path):
    binary = str(tmp_path / "few_rows_plan")
    res = subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "swiftrt_b200", "csrc"), "-o", binary,
                          os.path.join(ROOT, "tests", "cpp", "test_few_rows_plan.cpp")], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([binary], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout
