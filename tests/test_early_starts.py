"""The switches that make kernels start strictly after their predecessors hold for every library and every launch in it."""
import glob
import os
import re
import subprocess
import sys

import pytest

from tokenizer_b200.kernels import build


def early_starts(env, libraries):
    """What the libraries say in a process with these switches."""
    code = ("import ctypes, sys\n"
            "for path in sys.argv[1:]: print(ctypes.CDLL(path).tokb200_early_starts())")
    plain = {k: v for k, v in os.environ.items() if not k.startswith("TOKB200_PDL")}
    done = subprocess.run([sys.executable, "-c", code, *libraries], env={**plain, **env}, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    return [int(x) for x in done.stdout.split()]


@pytest.mark.parametrize("env, want", [
    ({}, [1, 1, 1]), ({"TOKB200_PDL": "0"}, [0, 0, 0]), ({"TOKB200_PDL": "1"}, [1, 1, 1]),
    ({"TOKB200_PDL_OFF": "sample_filtered"}, [0, 1, 1]), ({"TOKB200_PDL_OFF": "nothing,shared_prefix_tcgen05"}, [1, 0, 1]),
    ({"TOKB200_PDL_OFF": "pages,sample_filtered"}, [0, 1, 0]), ({"TOKB200_PDL_OFF": ""}, [1, 1, 1])])
def test_a_library_knows_both_switches(env, want):
    libraries = [build.compile_library("sample_filtered.cu"), build.compile_library("shared_prefix_tcgen05.cu", ("HEAD_DIM=64",)),
                 build.compile_library("pages.cu")]
    assert early_starts(env, libraries) == want


def test_every_early_start_asks_them():
    """No launch reads the environment for itself, and what allows an early start is always that answer."""
    for path in glob.glob(os.path.join(build.CSRC, "*.cu")) + glob.glob(os.path.join(build.CSRC, "*.cuh")):
        text = open(path).read()
        if os.path.basename(path) != "common.cuh":
            assert "TOKB200_PDL" not in text, path
        for value in re.findall(r"programmaticStreamSerializationAllowed = ([^;]*);", text):
            assert "tokb200_early_starts()" in value, path
