"""The step operators on a machine of two devices, without a GPU (step_devices.cpp): buffers and a stream of the current device
run, one of the other device's is refused before any launch."""
import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
API = os.path.join(os.path.dirname(HERE), "qwen38-megakernel_amd", "csrc", "step_api.cpp")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    import qkv
    so = str(tmp_path_factory.mktemp("step") / "m.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-D__HIP_PLATFORM_AMD__", f'-DSTEP_API="{API}"', "-I/opt/rocm/include",
                    os.path.join(HERE, "step_devices.cpp"), "-o", so], check=True)
    m = ctypes.CDLL(so)
    for name in ("mk_norm_q32", "mk_w4_units", "mk_w4_rows", "mk_verify_ws", "mk_verify_drafts"):
        f = getattr(m, name)
        f.restype, f.argtypes = qkv.SIGNATURES[name]
    m.model_message.restype = ctypes.c_char_p
    return m


def buf(device, i=0):
    return ((device + 1) << 32) + (i << 12)


def stream(device):
    return 16 * (device + 1)


# calls of one row each: p(i) is the i-th buffer
CALLS = {
    "norm": (8, lambda m, p, s: m.mk_norm_q32(p(0), 64, p(1), 64, p(2), 1, 64, 1e-6, 0, p(3), 64, p(4), 64, p(5), p(6), p(7), s)),
    "units": (7, lambda m, p, s: m.mk_w4_units(1, 16, 64, 32, p(0), p(1), p(2), p(3), p(4), p(5), p(6), 16, s)),
    "rows": (5, lambda m, p, s: m.mk_w4_rows(1, 16, 64, 32, p(0), p(1), p(2), p(3), 64, 1, p(4), 16, s)),
    "verify": (10, lambda m, p, s: m.mk_verify_drafts(1, 2, 100, p(0), 100, 0, 0, p(1), p(2), p(3), p(4), p(5), p(6), p(7), p(8), p(9), 1 << 20, s)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("device", [0, 1])
def test_current_device(model, name, device):
    n, call = CALLS[name]
    model.model_device(device)
    for s in (0, stream(device)):
        before = model.model_launches()
        assert call(model, lambda i: buf(device, i), s) == 0, model.model_message()
        assert model.model_launches() == before + 1


@pytest.mark.parametrize("name", CALLS)
def test_a_buffer_elsewhere(model, name):
    n, call = CALLS[name]
    model.model_device(0)
    before = model.model_launches()
    for k in range(n):
        for there, msg in ((buf(1, k), b"memory of device 1"), (1 << 20, b"not device memory")):
            assert call(model, lambda i: there if i == k else buf(0, i), 0) == -1
            assert msg in model.model_message()
    assert model.model_launches() == before


@pytest.mark.parametrize("name", CALLS)
def test_a_stream_elsewhere(model, name):
    """The kernels would run on the stream's device, on buffers of another."""
    n, call = CALLS[name]
    for device in (0, 1):
        model.model_device(device)
        before = model.model_launches()
        assert call(model, lambda i: buf(device, i), stream(1 - device)) == -1
        assert f"stream is of device {1 - device}, the current device is {device}".encode() in model.model_message()
        assert call(model, lambda i: buf(device, i), stream(5)) == -1
        assert model.model_launches() == before
