"""The ring of cached rows of the absorbed latent attention on the CPU: whatever order its copies land in, no step is taken before its rows have come.  CPU only."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    exe = str(tmp_path_factory.mktemp("ring") / "ring")
    subprocess.run(["g++", "-std=c++17", "-O1", os.path.join(ROOT, "tests", "host", "latent_ring_check.cpp"), "-o", exe], check=True, capture_output=True, timeout=300)
    return lambda *a: tuple(map(int, subprocess.run([exe, *map(str, a)], check=True, capture_output=True, text=True, timeout=300).stdout.split()))


@pytest.mark.parametrize("slots", range(3, 9))
def test_no_step_before_its_rows(run, slots):
    assert run(slots, 400, "step") == (0, 0, 0)


def test_too_few_slots(run):
    """a group asks again once it has the step behind: with two slots that one is never asked for (latent_attn.cu asserts that there are more)"""
    early, _, stuck = run(2, 400, "step")
    assert early == 0 and stuck > 0


@pytest.mark.parametrize("slots", [3, 5, 7])
def test_the_model_sees_a_late_copy(run, slots):
    """a barrier a slot, whose steps are the two groups' by turns: a wait succeeds on the phase before the step's own"""
    assert run(slots, 400, "slot")[0] > 0
