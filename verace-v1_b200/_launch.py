"""The launch path of the decode step's small calls, where the host's share of a call is longer
than the kernel: the current stream's handle without the Python objects of
``torch.cuda.stream`` (``raw_stream(index)``), and the current device's index (``current()``)
to skip the device guard where it changes nothing.  A torch without these two names (one built
without CUDA, for which the package still imports) goes through ``torch.cuda``."""
import torch


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)
current = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
