"""The give-up logic of the kernels' bounded waits, built for the host from the kernels' own headers."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MS = 1000 * 1000


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("no g++")
    out = str(tmp_path_factory.mktemp("protocol") / "libprotocol.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + os.path.join(ROOT, "cubert_b200", "csrc", "kernels"),
                    os.path.join(ROOT, "tests", "window_protocol_host.cpp"), "-o", out], check=True)
    return C.CDLL(out)


def over_at(host, readings):
    a = np.array(readings, dtype=np.uint64)
    return host.wait_over_at(a.ctypes.data_as(C.c_void_p), len(a))


def test_a_wait_ends_after_its_time(host):
    every = 50 * 1000                                            # 64 polls
    readings = [10 ** 18 + every * i for i in range(10000)]
    assert over_at(host, readings) == 200 * MS // every + 2      # the first reading past 0.2 s


@pytest.mark.parametrize("away", [250 * MS, 10 ** 12])
@pytest.mark.parametrize("at", [1, 100, 3990])
def test_time_off_the_sm_does_not_end_a_wait(host, at, away):
    """A block that comes back after the deadline has had no chance to look: it goes on for what is left of its 0.2 s,
    less a millisecond."""
    every = 50 * 1000
    readings = [10 ** 18 + every * i + (away if i >= at else 0) for i in range(10000)]
    # a gap of 20 readings' time: 19 readings fewer, or the first one back where less than that was left
    assert over_at(host, readings) == max(200 * MS // every + 2 - 19, at + 1)


def test_every_wait_ends(host):
    """However often a block is taken off, 201 gaps are enough."""
    assert over_at(host, [10 ** 18 + 10 ** 10 * i for i in range(1000)]) == 202
