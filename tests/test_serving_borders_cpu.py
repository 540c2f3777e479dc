"""The serving step at the borders of what it takes, without a GPU: the walk over a part's sequences, scales that fp32 has no room for."""
import math
import os
import subprocess

import pytest

import test_serving_cpu as T

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_part_walk(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=address,undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "include"),
                           os.path.join(ROOT, "tests", "part_walk_check.cpp"), "-o", exe])
    assert subprocess.run([exe], capture_output=True, text=True, timeout=60).stdout == "ok\n"


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38, -3e38, 2.0 ** 101, 2.0 ** -101, -1e-40])
def test_attention_scales_that_are_refused(scale):
    T.refused("gp_launch_paged_attention", T.attend(scale=scale), "scale")


@pytest.mark.parametrize("scale", [3e38, 2.0 ** 101, 2.0 ** -101, 1e-40, -0.5, -math.inf])
def test_scales_of_logits_that_are_refused(scale):
    T.refused("gp_launch_token_logprobs", T.logprobs(scale=scale), "scale")
