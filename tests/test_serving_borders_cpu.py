"""The serving step at the borders of what it takes, without a GPU: the walk over a part's sequences."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_part_walk(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "part_walk_check.cpp"), "-o", exe])
    assert subprocess.run([exe], capture_output=True, text=True, timeout=60).stdout == "ok\n"
