"""A refused launch is the call's error, with a text, and nobody else's: tests/cpp/test_launch_status.cpp, without a device."""
import os
import re
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "swiftrt_b200", "csrc")


def test_a_refused_launch_leaves_no_error_behind(tmp_path):
    import importlib.util
    spec = importlib.util.spec_from_file_location("_srt_b200_build", os.path.join(ROOT, "swiftrt_b200", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.nvcc_path()))), "include")
    binary = str(tmp_path / "launch_status")
    res = subprocess.run(["g++", "-std=c++17", "-O2", "-I" + CSRC, "-I" + os.path.join(ROOT, "include"), "-I" + cuda, "-o", binary,
                          os.path.join(ROOT, "tests", "cpp", "test_launch_status.cpp")], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    res = subprocess.run([binary], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout


def test_every_extended_launch_reports_through_it():
    for name in os.listdir(CSRC):
        if name.endswith(".cu"):
            text = open(os.path.join(CSRC, name)).read()
            for m in re.finditer(r"cudaLaunchKernelEx\(", text):
                line = text[text.rfind("\n", 0, m.start()) + 1:text.find("\n", m.start())]
                assert "launch_status(" in line, f"{name}: {line.strip()}"
