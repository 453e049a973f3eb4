"""Kernels that may exist while the kernel before them still writes what they will read must not read it by the path for data that nobody writes meanwhile, whose
loads the compiler may also move over the wait."""
import os
import re

import pytest

from tests.conftest import ROOT

CSRC = os.path.join(ROOT, "smallframework_b200", "csrc")
EARLY = sorted(f for f in os.listdir(CSRC) if f.endswith(".cu") and "narrow_types.cuh" in open(os.path.join(CSRC, f)).read())


def code(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


def test_which_files_start_early():
    assert EARLY == ["dense_f8.cu", "logprobs.cu", "quantize_f8.cu"]


@pytest.mark.parametrize("name", EARLY + ["narrow_types.cuh"])
def test_no_loads_by_the_read_only_path(name):
    found = re.findall(r"__ldg|__ldlu|__restrict__|ld\.global(?:\.\w+)*\.nc|ld\.global\.nc", code(name))
    assert not found


def test_only_these_files_start_early():
    """Launch, whose attribute lets a kernel start before the end of the one before it, is used nowhere else."""
    others = [f for f in sorted(os.listdir(CSRC)) if f not in EARLY + ["narrow_types.cuh"] and "ProgrammaticStreamSerialization" in code(f)]
    assert not others
