"""The adapters, the router and the experts on a machine of two devices, without a GPU (step_mix_devices.cpp): buffers and a stream of the
current device run, one of the other device's is refused before any launch."""
import ctypes
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
API = os.path.join(os.path.dirname(HERE), "qwen38-megakernel_amd", "csrc", "step_mix_api.cpp")


@pytest.fixture(scope="module")
def model(tmp_path_factory):
    import qkv
    so = str(tmp_path_factory.mktemp("mix") / "m.so")
    subprocess.run(["g++", "-O1", "-std=c++17", "-w", "-fPIC", "-shared", "-Wl,-Bsymbolic", "-D__HIP_PLATFORM_AMD__", f'-DSTEP_API="{API}"', "-I/opt/rocm/include",
                    os.path.join(HERE, "step_mix_devices.cpp"), "-o", so], check=True)
    m = ctypes.CDLL(so)
    for name in ("mk_lora_rows", "mk_lora_units", "mk_moe_route", "mk_moe_rows", "mk_moe_units", "mk_moe_layer"):
        f = getattr(m, name)
        f.restype, f.argtypes = qkv.SIGNATURES[name]
    m.model_message.restype = ctypes.c_char_p
    return m


def buf(device, i=0):
    return ((device + 1) << 32) + (i << 12)


def stream(device):
    return 16 * (device + 1)


SIZE = 1 << 20
# calls of one row each, their buffers and launches: p(i) is the i-th buffer
CALLS = {
    "lora": (9, 1, lambda m, p, s: m.mk_lora_rows(1, 16, 64, 2, 8, p(0), p(1), 2, p(2), p(3), p(4), p(5), 64, 0, p(6), 16, p(7), 16, p(8), SIZE, s)),
    "lora_units": (11, 1, lambda m, p, s: m.mk_lora_units(1, 16, 64, 2, 8, p(0), p(1), 2, p(2), p(3), p(4), p(5), p(6), p(7), p(8), 16, p(9), 16, p(10), SIZE, s)),
    "route": (7, 1, lambda m, p, s: m.mk_moe_route(1, 64, 8, 2, p(0), 64, 0, p(1), 0, p(2), 2, 1.0, p(3), p(4), p(5), p(6), SIZE, s)),
    "rows": (11, 1, lambda m, p, s: m.mk_moe_rows(1, 64, 64, 8, 2, 32, p(0), p(1), p(2), p(3), p(4), p(5), p(6), 64, 0, p(7), p(8), p(9), 64, p(10), SIZE, s)),
    "units": (13, 1, lambda m, p, s: m.mk_moe_units(1, 64, 64, 8, 2, 32, p(0), p(1), p(2), p(3), p(4), p(5), p(6), p(7), p(8), p(9), p(10), p(11), 64, p(12), SIZE, s)),
    "layer": (14, 2, lambda m, p, s: m.mk_moe_layer(1, 64, 64, 8, 2, 32, p(0), p(1), p(2), p(3), p(4), p(5), p(6), 64, 0, p(7), 0, p(8), 3, 1.0, p(9), p(10), p(11), p(12), 64,
                                                    p(13), SIZE, s)),
}


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("device", [0, 1])
def test_current_device(model, name, device):
    n, launches, call = CALLS[name]
    model.model_device(device)
    for s in (0, stream(device)):
        before = model.model_launches()
        assert call(model, lambda i: buf(device, i), s) == 0, model.model_message()
        assert model.model_launches() == before + launches


@pytest.mark.parametrize("name", CALLS)
def test_a_buffer_elsewhere(model, name):
    n, _, call = CALLS[name]
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
    n, _, call = CALLS[name]
    for device in (0, 1):
        model.model_device(device)
        before = model.model_launches()
        assert call(model, lambda i: buf(device, i), stream(1 - device)) == -1
        assert f"stream is of device {1 - device}, the current device is {device}".encode() in model.model_message()
        assert call(model, lambda i: buf(device, i), stream(5)) == -1
        assert model.model_launches() == before
