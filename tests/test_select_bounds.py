"""Host-side check of the bounded cache's selection (no GPU): the keys that share
the wanted first digit fit the words that they are set apart in, also where more
slots are among the newest positions than the cache keeps, so that the digit is
that of the slots past the end too; the form that sets those apart must be caught."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
SRC = ROOT / "tests" / "host" / "select_check.cpp"
INC = ROOT / "spikingbrain-cpu_amd" / "csrc"


@pytest.fixture(scope="module")
def checker(tmp_path_factory):
    exe = tmp_path_factory.mktemp("select") / "select_check"
    subprocess.run(["g++", "-O1", "-std=c++17", "-Wall", "-I", str(INC), str(SRC), "-o", str(exe)], check=True)
    return exe


def run(checker, *args):
    r = subprocess.run([str(checker), *map(str, args)], capture_output=True, text=True)
    return r.returncode, [int(x) for x in r.stdout.split()]


@pytest.mark.parametrize("n", [4097, 8192, 8193, 9000, 12287, 12288, 12289, 16384, 16385, 20480, 24576, 28672, 32767, 32768])
def test_keys_set_apart_fit(checker, n):
    for recent in (0, 1, 600, 2047, 2048, 2049, n):
        rc, (counted, apart) = run(checker, n, recent)
        assert rc == 0 and apart <= min(counted, recent)


@pytest.mark.parametrize("n,counted,apart", [(12288, 600, 4696), (20480, 600, 12888), (24576, 600, 8792)])
def test_slots_past_the_end_would_not_fit(checker, n, counted, apart):
    assert run(checker, n, 600, "unmasked") == (1, [counted, apart])
