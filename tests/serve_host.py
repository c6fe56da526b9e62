"""Runs the host side of glt_b200.serve without a GPU: tensors of host memory that say they lie on a
CUDA device, and a library whose launches a test replaces.  Nothing follows their pointers."""
import torch

from glt_b200 import _lib, serve


class DeviceTensor(torch.Tensor):
    """A host tensor that passes for one on the CUDA device `index` (views and copies of it too)."""
    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))

    def get_device(self):
        return self.index


class SecondDeviceTensor(DeviceTensor):
    index = 1


def on(t: torch.Tensor, index: int = 0) -> torch.Tensor:
    return t.as_subclass(SecondDeviceTensor if index else DeviceTensor)


class Host:
    """What serve runs on: the current device and stream, and every launch in order."""

    def __init__(self, monkeypatch):
        self.current, self.stream, self.calls = 0, 0, []
        monkeypatch.setattr(serve, "torch", self)
        monkeypatch.setattr(serve, "lib", self)
        monkeypatch.setattr(serve, "_raw_stream", lambda index: self.stream)
        monkeypatch.setattr(serve, "_capturing", lambda: False)
        monkeypatch.setattr(serve, "_current_device", lambda: self.current, raising=False)
        monkeypatch.setattr(torch.cuda, "device", lambda index: on_device(self, index))

    # -- torch
    def empty(self, *shape, dtype=torch.float32, device=None):
        device = torch.device(device)
        return on(torch.empty(*shape, dtype=dtype), self.current if device.index is None else device.index)

    # -- both: a launch is noted with the current device, everything else is the real one
    def __getattr__(self, name):
        if name.startswith("glt_"):
            real = getattr(_lib.lib, name)
            if name.endswith(("_workspace", "_bytes")):
                return real

            def launch(*args):
                self.calls.append((name, self.current, args))
                return self.launched(name, args)
            return launch
        return getattr(torch, name)

    def launched(self, name, args):
        return 0


class on_device:
    """torch.cuda.device for a Host: launches note the device that is current."""

    def __init__(self, host, index):
        self.host, self.index = host, index if isinstance(index, int) else index.index

    def __enter__(self):
        self.before, self.host.current = self.host.current, self.index

    def __exit__(self, *_):
        self.host.current = self.before
