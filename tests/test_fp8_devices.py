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


class Placed:
    """What the checks read of a tensor on a GPU that this machine need not have."""

    def __init__(self, dtype, *shape, device=1):
        self.dtype, self.shape, self.device = dtype, torch.Size(shape), torch.device("cuda", device)

    def dim(self):
        return len(self.shape)

    def is_contiguous(self):
        return True

    def stride(self):
        return torch.empty(self.shape, device="meta").stride()

    def data_ptr(self):
        return 4096


class Machine:
    """A current device and a current stream for each, as torch keeps them; the entry points record where they are called."""

    def __init__(self, monkeypatch):
        self.current, self.calls = 0, []
        machine = self

        class Switch:
            def __init__(self, device):
                self.device = device.index if isinstance(device, torch.device) else device

            def __enter__(self):
                self.before, machine.current = machine.current, self.device

            def __exit__(self, *exc):
                machine.current = self.before
        monkeypatch.setattr(torch.cuda, "device", Switch)
        monkeypatch.setattr(mm, "_current_device", lambda: machine.current, raising=False)
        monkeypatch.setattr(mm, "_current_stream", lambda: 100 + machine.current)
        monkeypatch.setattr(mm, "_entries", {e: self.entry for e in ENTRIES + ["tv_hip_gemm"]})

    def entry(self, args, stream):
        self.calls.append((self.current, stream))
        return 0


@pytest.mark.parametrize("device", [0, 1])
@pytest.mark.parametrize("stream", [None, 7])
def test_calls_run_on_their_tensors_device(monkeypatch, device, stream):
    """The current device is the tensors' own during the call, and the stream its current one; afterwards it is what it was."""
    machine = Machine(monkeypatch)
    f32, bf16, i32 = torch.float32, torch.bfloat16, torch.int32

    def t(dtype, *shape):
        return Placed(dtype, *shape, device=device)
    tv.quantize_fp8(t(bf16, 4, 8), q=t(F8, 4, 8), scale=t(f32, 4, 1), stream=stream)
    tv.rms_norm_fp8(t(bf16, 4, 8), t(bf16, 8), q=t(F8, 4, 8), scale=t(f32, 4, 1), stream=stream)
    tv.gemm_fp8(t(F8, 4, 8), t(f32, 4, 1), t(F8, 8, 8), t(f32, 1, 1), out=t(bf16, 4, 8), stream=stream)
    tv.route(t(f32, 4, 8), 2, weights=t(f32, 4, 2), ids=t(i32, 4, 2), stream=stream)
    tv.experts_fp8(t(F8, 4, 8), t(f32, 4, 1), t(F8, 2, 2, 4, 8), t(f32, 2, 2, 1, 1), t(F8, 2, 8, 4), t(f32, 2, 1, 1), t(f32, 4, 2),
                   t(i32, 4, 2), out=t(bf16, 4, 8), stream=stream)
    tv.gemm(t(bf16, 4, 8), t(bf16, 8, 4), out=t(bf16, 4, 4), stream=stream)
    assert machine.calls == [(device, 100 + device if stream is None else stream)] * 6
    assert machine.current == 0
