"""What the kernels of the latent attention wait for, on the CPU: whatever order the copies of cached rows land in, no step is taken before its rows have come; and warps whose waits run out
stay for the barriers that the others pass.  CPU only."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(folder, name):
    exe = str(folder / name)
    subprocess.run(["g++", "-std=c++17", "-O1", os.path.join(ROOT, "tests", "host", name + ".cpp"), "-o", exe], check=True, capture_output=True, timeout=300)
    return lambda *a: tuple(map(int, subprocess.run([exe, *map(str, a)], check=True, capture_output=True, text=True, timeout=300).stdout.split()))


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    return build(tmp_path_factory.mktemp("ring"), "latent_ring_check")


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


def test_warps_stay_for_the_others(tmp_path):
    run = build(tmp_path, "latent_rounds_check")
    assert run("rounds") == (0, 0, 0)
    assert run("leave")[0] > 0
