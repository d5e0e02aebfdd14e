"""Kernels launched with launch_overlapped start while the kernel before them in the stream still runs, which may write anything
they read. Loads through the read-only path are only defined for data that nobody writes while the kernel exists."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dace_onnx_b200", "csrc")


def code(path):
    text = open(path).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


OVERLAPPED = sorted(p for p in glob.glob(os.path.join(CSRC, "*.cu")) if "launch_overlapped(" in code(p))


def test_there_are_overlapped_kernels():
    assert {os.path.basename(p) for p in OVERLAPPED} >= {"rows_quant.cu", "gemm_scaled.cu"}


@pytest.mark.parametrize("path", OVERLAPPED, ids=os.path.basename)
def test_no_read_only_loads(path):
    for p in (path, os.path.join(CSRC, "typed.cuh")):
        assert not re.findall(r"__ldg\w*|ld\.global\.nc\S*|ld_stream4|__restrict__", code(p))


@pytest.mark.parametrize("path", OVERLAPPED, ids=os.path.basename)
def test_every_overlapped_kernel_waits(path):
    kernels = re.split(r"\b__global__\b", code(path))[1:]
    assert kernels
    for k in kernels:
        assert "wait_previous();" in k.split("template <")[0]
