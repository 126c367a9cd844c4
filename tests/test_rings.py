"""The rings of the epilogue products, walked on the host in random order with the kernels' own size and turn rules: no wait
passes for another use of its slot, no slot is refilled while it is read, and every walk ends."""
import os
import subprocess

import pytest

from loom_skills_b200 import build as B

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    tmp = str(tmp_path_factory.mktemp("walk"))
    B._write_iq3s_grid(tmp)                     # the table that the formats' header includes
    exe = os.path.join(tmp, "ring_walk")
    subprocess.check_call([B.NVCC, "-O2", "-std=c++17", "--expt-relaxed-constexpr", "-gencode",
                           "arch=compute_100a,code=sm_100a", "-I", tmp, "-I", B.CSRC,
                           os.path.join(HERE, "ring_walk.cu"), "-o", exe])
    return lambda *a: subprocess.run([exe, *a], capture_output=True, text=True, timeout=600)


def test_decode_rings(walk):
    r = walk("mvx")
    assert r.returncode == 0, r.stdout


def test_the_walk_finds_groups_that_do_not_follow_each_other(walk):
    r = walk("mvx", "alone")
    assert r.returncode == 1 and "another use" in r.stdout, r.stdout


def test_prefill_rings(walk):
    r = walk("gemmx")
    assert r.returncode == 0, r.stdout


def test_the_walk_finds_a_short_last_chunk_of_one_group(walk):
    r = walk("gemmx", "whole")
    assert r.returncode == 1 and "another use" in r.stdout, r.stdout


def test_epilogue_warps_meet_after_a_wait_gave_up(walk):
    r = walk("epilogue")
    assert r.returncode == 0, r.stdout
