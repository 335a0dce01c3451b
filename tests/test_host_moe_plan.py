"""What the experts' kernels take for granted of their plan (parts of k that have work, whole groups of tokens, LDS that a CU has), without a
GPU: over the shapes that the entry points accept."""
import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
PLAN = os.path.join(os.path.dirname(HERE), "qwen38-megakernel_amd", "csrc", "step_moe_plan.h")
UNITS = 3


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plan") / "m.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-w", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-D__forceinline__=inline", f'-DPLAN="{PLAN}"', "-I/opt/rocm/include",
                    os.path.join(HERE, "moe_plan_model.cpp"), "-o", so], check=True)
    m = ctypes.CDLL(so)
    m.model_sweep.restype = ctypes.c_longlong
    return m


@pytest.mark.parametrize("rows", [*range(1, 20), 24, 31, 32, 33, 47, 48, 49, 56, 63, 64])
def test_every_form(model, rows):
    bad = (ctypes.c_int * 8)()
    for e in (1, 2, 3, 5, 8, 16, 17, 60, 64, 128, 200, 256, 512, 1024):
        assert model.model_sweep(rows, e, 1 + rows * 1024 + e, bad) > 0, list(bad)


def test_every_length(model):
    """All numbers of blocks of dim and of inner."""
    for rows, e, top in ((1, 8, 2), (3, 8, 2), (16, 128, 8), (47, 8, 2), (64, 2, 2), (64, 256, 8)):
        for nb in range(1, 1025):
            for gsh, mins, xform in ((0, 0, UNITS), (1, 1, 0), (2, 0, 1), (2, 1, 2), (0, 1, 0)):
                assert model.model_holds(rows, 32 * min(nb, 512), 32 * (1025 - nb), e, top, gsh, mins, xform), (rows, e, top, nb, gsh, mins, xform)
                assert model.model_holds(rows, 32 * min(nb, 512), 32 * nb, e, top, gsh, mins, xform), (rows, e, top, nb, gsh, mins, xform)


def test_what_does_not_hold(model):
    """A wave without a run, a chunk of one run a wave in front of another, more at a time than there are."""
    assert model.model_parts(4, 4, 2) and model.model_parts(9, 8, 0) and model.model_parts(16, 8, 2) and model.model_parts(12, 8, 2)
    assert not model.model_parts(3, 3, 2)
    assert not model.model_parts(9, 8, 2)  # (the last chunk has one run for four waves)
    assert not model.model_parts(8, 4, 2)
    assert not model.model_parts(4, 8, 0) and not model.model_parts(4, 0, 0)
