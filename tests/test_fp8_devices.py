"""Where the 8-bit layer's Python functions run: their tensors' device and stream.  Nothing is launched here."""
import importlib

import pytest
import torch

import tensorvia_amd as tv

mm = importlib.import_module("tensorvia_amd.matmul")  # the package has a function of that name
ENTRIES = ["tv_hip_quantize_fp8", "tv_hip_rms_norm_fp8", "tv_hip_gemm_fp8", "tv_hip_route", "tv_hip_experts_fp8"]
F8 = torch.float8_e4m3fn


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


CALLS = {
    "quantize": lambda: tv.quantize_fp8(_t(4, 8)),
    "quantize_weights": lambda: tv.quantize_fp8(_t(4, 8), 128),
    "norm": lambda: tv.rms_norm_fp8(_t(4, 8), _t(8), _t(4, 8), normed=True),
    "gemm": lambda: tv.gemm_fp8(_t(4, 8, dtype=F8), _t(4, 1), _t(8, 8, dtype=F8), _t(1, 1)),
    "route": lambda: tv.route(_t(4, 8), 2),
    "experts": lambda: tv.experts_fp8(_t(4, 8, dtype=F8), _t(4, 1), _t(2, 2, 4, 8, dtype=F8), _t(2, 2, 1, 1), _t(2, 8, 4, dtype=F8),
                                      _t(2, 1, 1), _t(4, 2), _t(4, 2, dtype=torch.int32)),
}


@pytest.mark.parametrize("name", CALLS)
def test_host_tensors_are_refused(monkeypatch, name):
    """Arguments that fit together but for their place: a kernel would read host addresses.  The library is not called."""
    called = []
    monkeypatch.setattr(mm, "_entries", {e: lambda *args: called.append(args) or 0 for e in ENTRIES})
    with pytest.raises(RuntimeError, match="must be on a GPU, got cpu"):
        CALLS[name]()
    assert not called
