"""The launch path of the decode step's small calls: the current stream's handle and the
device guard without the Python objects of ``torch.cuda.stream`` / ``torch.cuda.device``
(which cost more than these kernels' launches)."""
import torch

_raw_stream = torch._C._cuda_getCurrentRawStream
_current = torch._C._cuda_getDevice


def launch(device: torch.device, entry, *args) -> int:
    """entry(*args, stream) on `device`'s current stream; returns the entry's status."""
    index = device.index
    if index == _current():
        return entry(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return entry(*args, _raw_stream(index))
