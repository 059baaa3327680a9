"""The host side of the low-precision entry points without a GPU: which stream outputs belong to, what import needs."""
import contextlib
import ctypes
import os
import subprocess
import sys

import pytest
import torch

import pto_isa_mirror_b200 as pto
from pto_isa_mirror_b200 import _capi, build

gemm = sys.modules["pto_isa_mirror_b200.gemm"]  # the package's `gemm` is the function


class OnDevice:
    """Stands for a CUDA tensor."""

    def __init__(self, shape, dtype, events):
        self.shape, self.dtype, self.events = torch.Size(shape), dtype, events

    def stride(self):
        return (self.shape[1], 1)

    def data_ptr(self):
        return 4096

    def get_device(self):
        return 0

    def new_empty_strided(self, size, stride, dtype):
        self.events.append("allocate")
        return OnDevice(size, dtype, self.events)


class Stream:
    def __init__(self, device_index):
        self.device_index, self.cuda_stream = device_index, 77


@pytest.fixture
def events(monkeypatch):
    seen = []

    @contextlib.contextmanager
    def on(stream):
        seen.append("enter")
        yield
        seen.append("leave")

    class Lib:
        @staticmethod
        def pto_b200_mx_quantize_e4m3_src(stream, *args):
            seen.append(("launch", stream))
            return 0

    inside = lambda: seen.count("enter") - seen.count("leave")  # noqa: E731
    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(gemm, "_raw_stream", lambda device: 77 if inside() else 5)
    monkeypatch.setattr(gemm, "_require_cuda_2d", lambda t, name: None)
    monkeypatch.setattr(_capi, "load", lambda: Lib)
    return seen


def test_the_mx_quantisers_outputs_belong_to_the_stream_it_launches_on(events):
    # blocks of the current stream's pool may still be used by work queued there, which the other stream does not wait for
    pto.mx_quantize_e4m3(OnDevice((4, 64), torch.bfloat16, events), stream=Stream(0))
    assert events == ["enter", "allocate", "allocate", ("launch", 77), "leave"]
    events.clear()
    pto.mx_quantize_e4m3(OnDevice((4, 64), torch.bfloat16, events))
    assert events == ["allocate", "allocate", ("launch", 5)]


def test_the_mx_quantiser_refuses_a_stream_of_another_device(events):
    with pytest.raises(ValueError, match="another device"):
        pto.mx_quantize_e4m3(OnDevice((4, 64), torch.bfloat16, events), stream=Stream(1))
    assert events == []


@pytest.mark.parametrize("transpose", [0, 1])
@pytest.mark.parametrize("rows", [4, 1 << 20])
def test_a_quantisers_maximum_and_tensor_scale_are_two_places(rows, transpose):
    build.build()
    lib = _capi.load()
    buf = (ctypes.c_uint8 * 4096)()
    p = (ctypes.addressof(buf) + 63) & ~63
    before = lib.pto_b200_launch_count()
    tail = (rows, 64, 64, 1 << 20, _capi.BF16, transpose)  # rows, k, ld_src, ld_data, source type
    assert lib.pto_b200_nvfp4_quantize(None, p, p + 512, p + 256, p + 1024, p + 256, *tail) == _capi.EINVAL
    assert lib.pto_b200_nvfp4_quantize_dynamic(None, p, p + 512, p + 256, p + 256, p + 1024, *tail) == _capi.EINVAL
    assert lib.pto_b200_launch_count() == before


@pytest.mark.parametrize("shape", [(1, 1), (1, 3), (1, 36), (5, 4), (130, 33), (2, 12), (0, 8), (3, 0)])
def test_codes_to_dequantise_come_in_whole_blocks(monkeypatch, shape):
    # the kernel reads whole words of codes, and a row's scale tiles are counted from its blocks
    nvfp4 = sys.modules["pto_isa_mirror_b200.nvfp4"]
    launches = []

    class Lib:
        pto_b200_nvfp4_dequantize = staticmethod(lambda *args: launches.append(args) or 0)

    monkeypatch.setattr(nvfp4, "_require_cuda_2d", lambda t, name: None)
    monkeypatch.setattr(nvfp4, "_require_scales", lambda *args: None)
    monkeypatch.setattr(nvfp4, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(nvfp4, "_elsewhere", lambda device, stream: None)
    monkeypatch.setattr(_capi, "load", lambda: Lib)
    scales = OnDevice((1, 1, 512), torch.uint8, [])
    with pytest.raises(ValueError, match="blocks of 16"):
        pto.nvfp4_dequantize(OnDevice(shape, torch.uint8, []), scales)
    assert launches == []
    assert pto.nvfp4_dequantize(OnDevice((1, 40), torch.uint8, []), scales).shape == (1, 80)
    assert len(launches) == 1 and launches[0][5:9] == (1, 80, 40, 80)  # rows, k, ld_data, ld_out


def test_the_weight_gradients_scales_are_e8m0_bytes(monkeypatch):
    wgrad = sys.modules["pto_isa_mirror_b200.wgrad"]
    launches = []

    class Lib:
        pto_b200_gemm_wgrad_mx = staticmethod(lambda *args: launches.append(args) or 0)

    monkeypatch.setattr(wgrad, "_require_cuda_2d", lambda t, name: None)
    monkeypatch.setattr(wgrad, "_raw_stream", lambda device: 5)
    monkeypatch.setattr(wgrad, "_elsewhere", lambda device, stream: None)
    monkeypatch.setattr(_capi, "load", lambda: Lib)
    call = lambda dtype: pto.gemm_wgrad_mx(  # noqa: E731
        OnDevice((8, 16), torch.bfloat16, []), OnDevice((8, 64), torch.uint8, []), OnDevice((8, 2), dtype, []))
    for dtype in (torch.bool, torch.int8, torch.float8_e4m3fn, torch.float8_e5m2):
        with pytest.raises(ValueError, match="e8m0"):
            call(dtype)
    assert launches == []
    for dtype in (torch.uint8, torch.float8_e8m0fnu):
        assert call(dtype).shape == (16, 64)
    assert len(launches) == 2


def test_the_package_imports_with_a_torch_built_without_cuda():
    code = """
import torch
del torch._C._cuda_getCurrentRawStream  # what such a build lacks
import pto_isa_mirror_b200 as pto
from pto_isa_mirror_b200 import build, gen_data
try:
    pto.gemm(torch.zeros((4, 4)), torch.zeros((4, 4)))
except ValueError as e:
    print("refused:", e)
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    got = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=600)
    assert got.returncode == 0 and got.stdout.startswith("refused:"), got.stderr
